"""The paged 8-bit K/V cache without a GPU: what its kernels' sources promise, and what the tolerances of the GPU tests can see."""
import re
from pathlib import Path

import numpy as np

from oracle import kv8

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


def test_the_tolerance_of_few_rows_sees_a_missing_second_part():
    """The weights of few rows are two fp16 parts. In numpy, with one part the outputs leave the tolerance that the GPU tests hold few rows to, with
    both they keep well inside it."""
    rng = np.random.RandomState(0)
    n, hd = 16, 128
    c = kv8.Cache(1, 1, 1, hd, 1, 1, 16)
    c.extend([n])
    c.append(0, rng.randn(n, 1, hd) * 0.2, rng.randn(n, 1, hd), [0, n])
    q = rng.randn(1, 8, hd).astype(np.float16).astype(np.float64)
    want, tol = c.attention(0, q, None, [0, 1], None, 0.0, False, weight=2.0 ** -22, least=2.0 ** -32)
    (kc, ks), (vc, vs) = c.tokens(0, 0, 0, c.k, c.k_scale), c.tokens(0, 0, 0, c.v, c.v_scale)
    off = {1: 0.0, 2: 0.0}
    for h in range(8):
        t = (kc * ks[:, None]) @ q[0, h] * hd ** -0.5 / np.log(2) + np.log2(vs)
        w = 2.0 ** (t - t.max() + 7)
        high = w.astype(np.float16).astype(np.float64)
        low = (w - high).astype(np.float16).astype(np.float64)
        cols = slice(h * hd, (h + 1) * hd)
        for parts, weight in ((1, high), (2, high + low)):
            got = weight @ vc / (w / vs).sum()
            off[parts] = max(off[parts], (np.abs(got - want[0, cols]) / tol[0, cols]).max())
    assert off[1] > 2 and off[2] < 0.5, off
