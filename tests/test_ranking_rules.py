"""Rules of the ranking layer that no run on one GPU can show, from its sources and with stand-ins for streams."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "culsh_b200", "csrc")


def source(name):
    return open(os.path.join(CSRC, name)).read()


def test_results_are_waited_for_by_an_event_of_their_own():
    """A query in flight waits for `counted`: another thread that ranks an earlier result must not record that."""
    text = source("ranking.cu")
    assert "counted" not in text
    body = text[text.index("int culsh_candidates_after("):]
    body = body[:body.index("\n}\n")]
    lock, record, wait = (body.index(x) for x in ("lock_guard", "cudaEventRecord(c->ctx->read_by", "cudaStreamWaitEvent(c->ctx->stream, c->ctx->read_by"))
    assert body.index("cudaStreamIsCapturing") < lock < record < wait
    others = [f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")) and f != "ranking.cu" and re.search(r"(Record|Wait\w*|Synchronize)\([^;]*\bread_by\b", source(f))]
    assert not others


def test_a_receive_buffer_is_waited_for_on_the_device_that_reads_it(monkeypatch):
    """Results of an exchange lie in a buffer that other processes write next: the stream that read it is waited for, whatever device is current."""
    import torch

    from culsh_b200 import ranking
    waited = []

    class Stream:
        def __init__(self, device):
            self.device = device

        def synchronize(self):
            waited.append(self.device)

    class Result:
        _ptr, _keepalive, n_queries, n_total_candidates = 1, object(), 3, 7
        _h = type("Handle", (), {"device": 1})

        def empty(self):
            return False

        def device_pointers(self):
            return 16, 16, 16

    after = []
    lib = type("Lib", (), {"culsh_candidates_after": lambda self, *a: after.append(a) or 0})()
    handle = type("Handle", (), {"lib": lib, "ptr": 5})()
    monkeypatch.setattr(ranking, "Candidates", Result)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(device))
    lists = ranking._Lists(Result(), torch.device("cuda", 1))
    lists.done(handle, 77)
    assert after == [(5, 1, 77)] and waited == [torch.device("cuda", 1)]
    Result._keepalive = None
    lists.done(handle, 77)
    assert len(after) == 2 and len(waited) == 1


class Functions:
    """Bodies of the functions and structs of a source by their names."""

    def __init__(self, name):
        self.text = source(name)

    def __getitem__(self, name):
        m = re.search(r"^(?:__global__|__device__|struct|inline)[^\n]*?\b%s\b[^;{]*\{\n" % name, self.text, re.M)
        return self.text[m.end():re.compile(r"^\}", re.M).search(self.text, m.end()).start()]


def test_kernels_launched_early_read_by_l2():
    """A kernel that is launched early begins while those in front still write: what it reads of theirs must not come from a line that L1 already has, nor by
    loads that take memory for constant."""
    rows, score, lp = (Functions(f) for f in ("mx_rows.cuh", "mx_score.cuh", "log_probs.cuh"))
    used = [rows["EightOf"], rows["mx_quantize_kernel"], score["mx_slices_kernel"]]
    used += [lp[n] for n in ("LpRows", "lp_load", "lp_chunks", "LpFind", "lp_first_named", "lp_find_in_any_order", "lp_finish", "log_probs_unit_kernel", "log_probs_join_kernel")]
    early = lp["log_probs_unit_kernel"] + lp["log_probs_join_kernel"]
    assert "EARLY ? __ldcg(x + p) : x[p]" in lp["lp_load"] and "<false" not in early and "LpFind<>" not in early
    assert not re.search(r"\.(?:begin|end)\(", early) and early.count("rows.begin<true>(") >= 4
    assert re.search(r"if constexpr \(EARLY\) return __ldcg\(p\);", lp["lp_get"])
    for body in used:
        body = body.replace("EARLY ? __ldcg(x + p) : x[p]", "")
        assert "__ldg" not in body
        assert not re.search(r"(?<![\w.])(?:x|q|X|Q|ids|names|targets|offsets)\[(?!32\b)", body), body
        assert not re.search(r"= a\.\w+\[", body), body
    assert "__ldg" not in source("mx_product.cuh")
    # the kernel that gathers scales by L1 is launched as usual
    assert re.search(r"\bmx_score_tc_kernel<<<", score["mx_score"]) and "KernelBefore" not in source("mx_score.cuh").split("mx_score_tc_kernel(")[1].split("{")[0]


def test_a_kernel_that_gives_up_waits_for_what_it_has_in_flight():
    """Where a bounded wait ran out, loads and tensor-core work may still be on their way to memory that the CTA is about to give back: behind the barrier at which all
    roles are done, and before tensor memory is freed, both are waited for, without regard to the flag that ends the other waits."""
    for name, kernel in (("mx_product.cuh", "mx_product_kernel"), ("mx_score.cuh", "mx_score_tc_kernel")):
        text = source(name)
        end = text[text.index(kernel + "("):]
        end = end[:end.index("tcgen05.dealloc")]
        last = end[end.rindex("tc_fence_before"):]
        assert re.search(r"__syncthreads\(\);.*if \(\*s_abort\) \{.*mbar_wait_landed\(\w*full, .*tc_commit_warp\(drained\);\s*mbar_wait_landed\(drained, 1, 1\);.*__syncthreads\(\);", last, re.S), name
        assert end.count("++fills;") == 1 and "*s_fills = fills;" in end
    wait = source("mx_product.cuh")
    wait = wait[wait.index("void mbar_wait_landed("):]
    wait = wait[:wait.index("\n}\n")]
    assert "TC_WAIT_CYCLES" in wait and "abort" not in wait


def test_loads_that_landed_are_told_from_their_number(tmp_path):
    """The phase of a ring's barrier that its last load ends: loads go to the slots in turn, a phase for each."""
    from native import run_native
    body = source("mx_product.cuh")
    line = re.search(r"const uint32_t of_this = ([^;]+);", body).group(1)
    parity = re.search(r"mbar_try_wait\(&bars\[s\], ([^)]*\)[^)]*)\)\)", body).group(1)
    out = run_native(tmp_path, """
#include <cstdint>
#include <cstdio>
#include <vector>
int main() {
    for (uint32_t n = 1; n <= 12; ++n)
        for (uint32_t fills = 0; fills < 40; ++fills) {
            std::vector<uint32_t> phases(n, 0);
            for (uint32_t i = 0; i < fills; ++i) ++phases[i %% n];
            for (uint32_t s = 0; s < n; ++s) {
                const uint32_t of_this = %s;
                if (of_this != phases[s]) return 1;
                if (of_this && (%s) != ((phases[s] - 1) %% 2)) return 2;
            }
        }
    puts("ok");
}
""" % (line, parity))
    assert out == "ok\n"


def test_temperatures_that_no_float_divides_by_are_refused():
    """Between them and the ones whose reciprocal is no float either, ties came out as NaN."""
    import pytest
    import torch

    import culsh_b200 as culsh
    s, one = torch.zeros(2, 2), torch.zeros(2)
    for t in (4.2e-39, 3.5e-39, 1e-39, 1e-300):
        with pytest.raises(ValueError, match="too small"):
            culsh.log_probs(s, temperature=t)
        with pytest.raises(ValueError, match="too small"):
            culsh.log_probs_backward(s, None, one, one, temperature=t)
