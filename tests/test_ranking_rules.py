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
