"""The paged 8-bit K/V cache without a GPU: what its kernels' sources promise, and what the tolerances of the GPU tests can see."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "decide_b200" / "csrc"


def code_of(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def test_the_lanes_of_a_warp_agree_on_every_wait():
    """The lanes of one warp that part at a wait that ran out would wait for one another without a limit. So the waits of the tcgen05 form go through
    warp_wait, which takes a vote, but for the last one of all, whose answer nothing branches on."""
    code = code_of("kv8_attn_tc.cu")
    assert re.search(r"bool warp_wait\([^)]*\) \{\s*return __all_sync\(0xffffffffu, mbar_wait\([^;]*\)\);\s*\}", code)
    calls = [m for m in re.finditer(r"(?<!\w)mbar_wait\(", code)]
    assert len(calls) == 2
    last = code[:calls[1].start()].rstrip()
    assert last.endswith((";", "{", "}")), "the answer of a wait that takes no vote is used"
    assert len(re.findall(r"warp_wait\(", code)) >= 8
