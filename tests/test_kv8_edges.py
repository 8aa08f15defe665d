"""The paged 8-bit K/V cache without a GPU: what its kernels' sources promise, and what the tolerances of the GPU tests can see."""
import re
from pathlib import Path

import numpy as np

from oracle import kv8

CSRC = Path(__file__).resolve().parents[1] / "decide_b200" / "csrc"


def code_of(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def test_no_wait_parts_the_lanes_of_a_warp():
    """Lanes of one warp that part at a wait that ran out would wait for one another without a limit. So the waits of the tcgen05 form give no answer that
    anything could branch on; the one look at the flag that says whether one of them ran out is a vote of the whole warp, but for the wait loop itself and
    the teardown behind the last barrier."""
    code = code_of("kv8_attn_tc.cu")
    assert re.search(r"void await\(uint64_t", code) and len(re.findall(r"(?<!\w)await\(&?\w", code)) >= 8
    waits = [code[:m.start()].rstrip()[-1] for m in re.finditer(r"(?<!\w)mbar_wait\(", code)]
    assert waits == [";"], "the answer of a wait is used"
    looks = [code[:m.end()].splitlines()[-1].strip() for m in re.finditer(r"\*abort_flag\b(?! = 1u| = 0u;)", code)]
    looks = [x for x in looks if not x.endswith("volatile uint32_t* abort_flag")]
    assert looks == ["if (*abort_flag", "if (__all_sync(0xffffffffu, *abort_flag", "if (*abort_flag"], looks


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
