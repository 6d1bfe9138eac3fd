"""Instructions that want all lanes of a warp at the same place (tcgen05.ld and .st, .sync.aligned): where lanes may have gone their own way in front of them, the warp comes together first."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "culsh_b200", "csrc")
POLICIES = ("ce_fused.cuh", "cross_entropy.cuh", "int8_product.cuh", "tc_gemm.cuh")  # whose tiles end inside a warp


def _code(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_tensor_memory_is_read_by_warps_that_have_come_together():
    for name in POLICIES:
        text = _code(name)
        for m in re.finditer(r"\btc_ld(16|32)\(", text):
            assert re.search(r"__syncwarp\(\);\s*$", text[:m.start()]), (name, text[m.start() - 80:m.end() + 40])


def test_lanes_do_not_leave_a_pass_of_a_loop_that_reads_tensor_memory():
    """`continue` by a lane's own row, in front of the next pass's read."""
    for name in POLICIES + ("mx_product.cuh",):
        text = _code(name)
        for m in re.finditer(r"\b(?:tg_read|ce_with_own|t[cg]_ld(?:16|32))\(", text):
            behind = text[m.end():m.end() + 400]
            assert not re.search(r"if \((?:row|at) >= a\.\w+\) continue;", behind), (name, behind)


def test_rows_of_four_bits_too():
    text = _code("mx_product.cuh")
    loop = text[text.index("for (int q0 = 0; q0 < a.nq; q0 += 16)"):]
    assert loop.index("__syncwarp();") < loop.index("tc_ld16(")
