"""The paged 8-bit K/V cache on the GPU against the numpy model of oracle/kv8.py. Codes, scales, tables, lengths and counts are exact;
attention is held to the tolerance that the model derives from the kernel's arithmetic."""
import numpy as np
import pytest
import torch

from decide_b200.kernels import Engine, Family, KernelError, Kv8Cache
from oracle import kv8

pytestmark = pytest.mark.gpu

SENTINEL = 7.0


class Pair:
    """A cache on the GPU and its model, filled alike. What no sequence holds starts as codes for NaN."""

    def __init__(self, k, layers=1, n_pages=12, nkv=2, hd=128, n_seqs=3, max_pages=8, page=16, token_major=False):
        self.ops, self.dev = k.kv8, k.dev
        self.model = kv8.Cache(layers, n_pages, nkv, hd, n_seqs, max_pages, page)
        self.model.k[:], self.model.v[:] = 0x7F, 0x7F
        self.model.k_scale[:], self.model.v_scale[:] = np.nan, np.nan
        shape = (layers, n_pages, page, nkv, hd) if token_major else (layers, n_pages, nkv, page, hd)
        codes = [torch.full(shape, 0x7F, dtype=torch.uint8, device="cuda") for _ in range(2)]
        codes = [c.transpose(2, 3) if token_major else c for c in codes]
        scales = [torch.full((layers, n_pages, nkv), float("nan"), device="cuda") for _ in range(2)]
        self.gpu = Kv8Cache(*codes, *scales, torch.zeros(n_seqs, max_pages, dtype=torch.int32, device="cuda"),
                            torch.zeros(n_seqs, dtype=torch.int32, device="cuda"), torch.zeros(n_pages, dtype=torch.int32, device="cuda"))

    def same(self):
        for name in ("k", "v"):
            assert np.array_equal(getattr(self.gpu, name).cpu().numpy(), getattr(self.model, name)), name
        for name in ("k_scale", "v_scale", "table", "lens", "refs"):
            assert np.array_equal(getattr(self.gpu, name).cpu().numpy(), getattr(self.model, name), equal_nan=name.endswith("scale")), name

    def ints(self, values):
        return torch.tensor(np.array(values, dtype=np.int64).astype(np.uint32).view(np.int32), device="cuda")

    def extend(self, add):
        self.ops.extend(None, self.gpu, self.ints(add))
        self.model.extend(add)

    def fork(self, src, dst, deep):
        self.ops.fork(None, self.gpu, self.ints(src), self.ints(dst), len(src), deep)
        self.model.fork(src, dst, deep)

    def free(self, seqs):
        self.ops.free(None, self.gpu, self.ints(seqs), len(seqs))
        self.model.free(seqs)

    def compact(self):
        live = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.ops.compact(None, self.gpu, live)
        assert self.model.compact() == int(live)

    def append(self, counts, size=1.0, seed=0, pad=0, layer=0, spoil=None):
        """`counts` new rows a sequence, `pad` columns between the rows, two rows behind the last."""
        start = np.concatenate([[0], np.cumsum(counts)])
        rows, nkv, hd = int(start[-1]), self.gpu.nkv, self.gpu.hd
        gen = torch.Generator().manual_seed(seed)
        new = [(torch.randn(rows + 2, nkv * hd + pad, generator=gen) * size).to(self.dev.act_torch) for _ in range(2)]
        if spoil:
            spoil(new)
        on = [x.cuda() for x in new]
        ld = nkv * hd + pad
        self.ops.append(None, self.gpu, layer, *on, ld, ld, self.ints(start), rows, max(counts))
        self.model.append(layer, *(x[:rows, :nkv * hd].double().numpy().reshape(rows, nkv, hd) for x in new), start)
        return on, start, rows

    def attend(self, counts, nq, qpos=None, gate=True, seed=0, layer=0, pad=0, size=1.5, max_len=None, stream=None, spoil=None):
        start = np.concatenate([[0], np.cumsum(counts)])
        rows, hd = int(start[-1]), self.gpu.hd
        width, act = nq * hd, self.dev.act_torch
        gen = torch.Generator().manual_seed(seed + 100)
        q = (torch.randn(rows + 2, width + pad, generator=gen) * size).to(act)
        if spoil:
            spoil(q)
        g = torch.randn(rows + 2, width + 4, generator=gen) if gate else None
        y = torch.full((rows + 2, width + 8), SENTINEL, dtype=act, device="cuda")
        at = None if qpos is None else self.ints(list(qpos) + [0, 0])
        longest = int(self.model.lens.max()) if max_len is None else max_len
        self.ops.attention(stream, self.gpu, layer, q.cuda(), g.cuda() if gate else None, self.ints(start), at, y, rows, width + pad, width + 4, width + 8, nq,
                           max(counts), longest)
        got = y.double().cpu().numpy()
        want, tol = self.model.attention(layer, q[:rows, :width].double().numpy().reshape(rows, nq, hd), g[:rows, :width].double().numpy() if gate else None,
                                         start, None if qpos is None else np.array(qpos), torch.finfo(act).eps / 2, act == torch.bfloat16)
        assert (got[:, width:] == SENTINEL).all() and (got[rows:] == SENTINEL).all(), "written past the rows"
        got = got[:rows, :width]
        assert np.array_equal(np.isnan(got), np.isnan(want)), "NaN where there should be none, or the other way round"
        fine = ~np.isnan(want)
        off = np.abs(got - want)[fine] - tol[fine]
        assert off.size == 0 or off.max() <= 0, f"off by {np.abs(got - want)[fine][off.argmax()]:.3e}, allowed {tol[fine][off.argmax()]:.3e}"
        return y


LAYOUTS = [dict(page=16, hd=128, nkv=1), dict(page=32, hd=256, nkv=2, token_major=True), dict(page=64, hd=128, nkv=3), dict(page=128, hd=256, nkv=1),
           dict(page=128, hd=128, nkv=2, token_major=True)]


# ---------------------------------------------------------------- pages

@pytest.mark.parametrize("deep", [False, True])
def test_fork_extend_free_compact(k, deep):
    p = Pair(k, layers=2, n_pages=14, n_seqs=5, page=16)
    p.extend([40, 16, 0, 1, 0])
    p.append([40, 16, 0, 1, 0], seed=1)
    p.append([40, 16, 0, 1, 0], seed=2, layer=1)
    p.same()
    p.fork([0, 1, 0], [2, 4, 3], deep)      # a destination that held a page, two copies of one sequence, one that ends with its page
    p.same()
    p.extend([0, 0, 9, 16, 1])
    p.same()
    p.free([0, 4, 0])                       # named twice, and its pages shared (deep: not)
    p.same()
    p.compact()
    p.same()
    p.compact()                             # nothing left to move
    p.same()
    p.fork([2], [0], True)
    p.free([2, 3])
    p.compact()
    p.same()
    p.dev.check_status()


def test_pages_random_walk(k):
    """A few hundred calls, every state compared; calls that do not fit change nothing."""
    rng = np.random.RandomState(3)
    p = Pair(k, layers=2, n_pages=28, nkv=1, n_seqs=9, max_pages=6, page=16)
    refused = 0
    for step in range(200):
        try:
            what = rng.randint(4)
            if what == 0:
                add = rng.randint(0, 60, 9) * (rng.rand(9) < 0.6)
                p.extend([int(a) for a in add])
            elif what == 1:
                order = [int(x) for x in rng.permutation(9)]
                n = rng.randint(1, 4)
                p.fork([order[rng.randint(4, 9)] for _ in range(n)], order[:n], bool(rng.randint(2)))
            elif what == 2:
                p.free([int(x) for x in rng.randint(0, 9, rng.randint(1, 4))])
            else:
                p.compact()
        except kv8.Violation:
            refused += 1
            with pytest.raises(KernelError):
                p.dev.check_status()
        p.same()
    assert 10 < refused < 150
    p.dev.check_status()


def test_many_sequences_and_pages(k):
    """More sequences and pages than the deciding CTA has threads."""
    rng = np.random.RandomState(4)
    p = Pair(k, n_pages=9000, nkv=1, n_seqs=2500, max_pages=5, page=16)
    p.extend([int(x) for x in rng.randint(0, 60, 2500)])
    p.same()
    order = [int(x) for x in rng.permutation(2500)]
    p.fork(order[1250:], order[:1250], False)
    p.free(order[100:1900])
    p.same()
    p.compact()
    p.same()
    p.fork(order[1900:2500], order[100:700], True)
    p.same()
    p.dev.check_status()


@pytest.mark.parametrize("call,word", [
    (lambda p: p.extend([100, 0, 0]), "too few free"), (lambda p: p.extend([0, 129, 0]), "longer"), (lambda p: p.extend([0, 0xFFFFFFFF, 0]), "longer"),
    (lambda p: p.fork([0], [0], False), "sequence"), (lambda p: p.fork([0, 0], [1, 1], False), "sequence"), (lambda p: p.fork([0], [3], False), "sequence"),
    (lambda p: p.fork([0xFFFFFFFF], [1], True), "sequence"), (lambda p: p.fork([0, 0], [1, 2], True), "too few free"),
    (lambda p: p.fork([0, 1], [1, 2], False), "sequence"), (lambda p: p.free([7]), "sequence"),
])
def test_violations_change_nothing(k, call, word):
    p = Pair(k, n_pages=9, max_pages=13 if word == "too few free" else 8)
    p.extend([70, 3, 1])
    p.append([70, 3, 1])
    with pytest.raises(kv8.Violation):
        call(p)
    with pytest.raises(KernelError, match=word):
        p.dev.check_status()
    p.same()
    p.dev.check_status()


def test_corrupt_tables_are_reported(k):
    """A page id outside the pool, a length past the table, a page that nobody holds: reported, nothing outside the arrays touched."""
    for spoil, word, calls in (
            (lambda p: p.gpu.table.__setitem__((0, 1), 9), "outside the pool", "fork copy free compact append attend"),
            (lambda p: p.gpu.table.__setitem__((0, 1), -1), "outside the pool", "fork copy free compact append attend"),
            (lambda p: p.gpu.lens.__setitem__(0, 129), "longer", "extend fork copy free compact append attend"),
            (lambda p: p.gpu.refs.__setitem__(0, 0), "freed more often", "drop free"),
            (lambda p: p.gpu.refs.__setitem__(1, 2), "several", "append")):
        for call in calls.split():
            p = Pair(k, n_pages=9)
            p.extend([30, 3, 0])
            p.append([30, 3, 0])
            spoil(p)
            one = p.ints([0])
            x = torch.zeros(40, 256, dtype=k.dev.act_torch, device="cuda")
            if call == "extend":
                p.ops.extend(None, p.gpu, p.ints([1, 0, 0]))
            elif call in ("fork", "copy"):
                p.ops.fork(None, p.gpu, one, p.ints([2]), 1, call == "copy")
            elif call == "drop":
                p.ops.fork(None, p.gpu, p.ints([1]), one, 1, False)
            elif call == "free":
                p.ops.free(None, p.gpu, one, 1)
            elif call == "compact":
                p.ops.compact(None, p.gpu)
            elif call == "append":
                p.ops.append(None, p.gpu, 0, x, x, 256, 256, p.ints([0, 20, 20, 20]), 20, 20)
            else:
                y = torch.full((1, 512), SENTINEL, dtype=k.dev.act_torch, device="cuda")
                p.ops.attention(None, p.gpu, 0, x, None, p.ints([0, 1, 1, 1]), None, y, 1, 512, 0, 512, 4, 1, 0)
                assert (torch.isnan(y) if word != "longer" else y == SENTINEL).all()
            with pytest.raises(KernelError, match=word):
                k.dev.check_status()
    k.dev.check_status()


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
def test_append(k, act, layout):
    """Rows for some sequences and none for others, in several steps whose sizes make scales rise, pages in the middle and at their ends."""
    page = layout["page"]
    p = Pair(k, n_pages=16, n_seqs=4, max_pages=6, **layout)
    for step, (counts, size) in enumerate([([1, page, 0, page + 1], 0.01), ([1, 1, 0, 2 * page - 1], 0.01), ([page - 2, 0, 3, 1], 3.0), ([1, 5, 1, 0], 400.0), ([2 * page, 0, 0, 0], 1e-4)]):
        p.extend(counts)
        on, start, rows = p.append(counts, size, seed=step, pad=8 * step)
        p.same()
        ld = p.gpu.nkv * p.gpu.hd + 8 * step
        p.ops.append(None, p.gpu, 0, *on, ld, ld, p.ints(start), rows, max(counts))      # the same rows again
        p.same()
    k.dev.check_status()


def test_append_extreme_values(k, act):
    """Zeros, the type's largest and smallest magnitudes, each as the first rows of a page and joining one."""
    top, low = torch.finfo(act).max, torch.finfo(act).smallest_normal
    tiny = low * torch.finfo(act).eps
    for values in ([0.0, 1.0], [1.0, 0.0], [top, -top], [tiny, -tiny], [tiny, top], [1.75, 1.7578125], [448.0, 450.0], [-0.0, 0.0]):
        p = Pair(k, nkv=1, n_seqs=1)
        for i, x in enumerate(values):
            p.extend([3])
            p.append([3], seed=i, spoil=lambda new: [n.fill_(x) for n in new])
            p.same()
    k.dev.check_status()


def test_append_non_finite_poisons_its_page_and_head_alone(k, act):
    for bad in (float("nan"), float("inf"), -float("inf")):
        p = Pair(k, nkv=2, n_seqs=2, page=16)
        p.extend([20, 5])
        p.append([20, 5])
        p.extend([3, 1])

        def spoil(new, bad=bad):
            new[0][1, 130] = bad        # K, head 1, the second new row of sequence 0
            new[1][3, 5] = bad          # V, head 0, the new row of sequence 1
        p.append([3, 1], seed=1, spoil=spoil)
        p.same()
        assert int(np.isnan(p.model.k_scale[0, p.model.table[0, :2]]).sum()) == 1
        p.extend([14, 1])               # into the poisoned pages, and a fresh one
        p.append([14, 1], seed=2)
        p.same()
        p.attend([20, 3], nq=4)         # rows before the bad token's page attend it not at all
    k.dev.check_status()


def test_a_cache_elsewhere_is_refused(k):
    """The context's device and the cache's have to be the same."""
    p = Pair(k)
    cpu = Kv8Cache.empty(1, 4, 2, 128, 3, 4, 16, device="cpu")
    for call in (lambda: p.ops.extend(None, cpu, p.ints([0, 0, 0])), lambda: p.ops.compact(None, cpu), lambda: p.ops.free(None, cpu, p.ints([0]), 1)):
        with pytest.raises(KernelError, match="device"):
            call()


def test_append_refusals(k):
    p = Pair(k)
    x = torch.zeros(4, 264, dtype=k.dev.act_torch, device="cuda")
    start = p.ints([0, 1, 2, 3])
    p.ops.append(None, p.gpu, 0, x, x, 256, 256, start, 0, 0)       # no rows
    for args in ((1, x, x, 256, 256, start, 3, 1), (0, None, x, 256, 256, start, 3, 1), (0, x, x, 248, 256, start, 3, 1), (0, x, x, 256, 260, start, 3, 1),
                 (0, (x, 2), x, 256, 256, start, 3, 1), (0, x, x, 256, 256, None, 3, 1)):
        with pytest.raises(KernelError):
            p.ops.append(None, p.gpu, *args)
    p.extend([3, 3, 3])
    for start, rows, most in (([0, 4, 4, 4], 4, 4), ([0, 2, 1, 3], 3, 3), ([0, 1, 2, 5], 4, 3), ([0, 3, 3, 3], 3, 2)):
        before = p.gpu.k.clone()
        p.ops.append(None, p.gpu, 0, x, x, 256, 256, p.ints(start), rows, most)
        with pytest.raises(KernelError, match="offsets"):
            k.dev.check_status()
        assert int((before != p.gpu.k).any(-1).sum()) <= 2 * 2 * 2      # only sequences whose offsets hold: two of two rows, two heads
    k.dev.check_status()


# ---------------------------------------------------------------- attention

ATTENTION = [
    # lens, rows a sequence, query heads, kv heads, hd, page
    dict(lens=[1], counts=[1], nq=4, nkv=1, hd=128, page=16),
    dict(lens=[16, 17, 15], counts=[1, 1, 1], nq=8, nkv=2, hd=128, page=16),
    dict(lens=[100, 0, 33], counts=[1, 1, 0], nq=6, nkv=2, hd=128, page=32),
    dict(lens=[64, 5, 130], counts=[3, 5, 1], nq=2, nkv=2, hd=256, page=64, token_major=True),
    dict(lens=[129, 200, 7], counts=[9, 2, 7], nq=5, nkv=1, hd=128, page=128),
    dict(lens=[255, 256, 257], counts=[1, 2, 1], nq=16, nkv=1, hd=256, page=16),
    dict(lens=[300, 1, 90], counts=[17, 1, 33], nq=6, nkv=2, hd=128, page=64, token_major=True),
    dict(lens=[90, 40, 31], counts=[33, 40, 1], nq=3, nkv=1, hd=256, page=32),
    # whole tiles of pairs
    dict(lens=[130], counts=[130], nq=1, nkv=1, hd=128, page=16),
    dict(lens=[300, 40, 700], counts=[100, 40, 70], nq=8, nkv=2, hd=128, page=16),
    dict(lens=[1000, 0, 5], counts=[64, 3, 5], nq=3, nkv=1, hd=128, page=32),
    dict(lens=[2600], counts=[65], nq=2, nkv=2, hd=128, page=64, token_major=True),
    dict(lens=[129, 257, 128, 1], counts=[20, 33, 16, 1], nq=16, nkv=1, hd=128, page=128),
    dict(lens=[129], counts=[129], nq=1, nkv=1, hd=256, page=16),
    dict(lens=[300, 40, 700], counts=[50, 40, 70], nq=8, nkv=2, hd=256, page=16),
    dict(lens=[1000, 0, 5], counts=[64, 3, 5], nq=3, nkv=1, hd=256, page=32, token_major=True),
    dict(lens=[65, 64, 63, 1], counts=[20, 33, 16, 1], nq=16, nkv=1, hd=256, page=128),
]


# A table with room for this many tokens a sequence, and no length given, makes 64 and more (row, head) pairs of a kv head a call for whole
# tiles of the tensor cores, however short the sequences are.
ROOM = 65536


def _filled(k, lens, nkv, hd, page, token_major=False, size=1.0, seed=0, room=0):
    pages = [-(-n // page) for n in lens]
    p = Pair(k, n_pages=sum(pages) + 2, nkv=nkv, hd=hd, n_seqs=len(lens), max_pages=max(max(pages) + 1, room // page), page=page, token_major=token_major)
    step = [n // 2 for n in lens]       # in two steps, so that the sequences' pages interleave
    for part in (step, [n - s for n, s in zip(lens, step)]):
        p.extend(part)
        if sum(part):
            p.append(part, size, seed)
    return p


@pytest.mark.parametrize("case", ATTENTION, ids=str)
def test_attention(k, act, case):
    c = dict(case)
    counts, nq = c.pop("counts"), c.pop("nq")
    p = _filled(k, **c)
    p.attend(counts, nq, gate=False)
    p.attend(counts, nq, gate=True, pad=8, seed=1)
    rng = np.random.RandomState(0)
    qpos = [kv8.NO_KEYS if n == 0 or rng.rand() < 0.2 else rng.randint(n) for n, m in zip(c["lens"], counts) for _ in range(m)]
    p.attend(counts, nq, qpos=qpos, seed=2, max_len=0)
    k.dev.check_status()
    if max(counts) * (nq // c["nkv"]) >= 64:
        p = _filled(k, room=ROOM, **c)
        p.attend(counts, nq, gate=False, max_len=0)
        p.attend(counts, nq, gate=True, pad=8, seed=1, max_len=0)
        p.attend(counts, nq, qpos=qpos, seed=2, max_len=0)
        k.dev.check_status()


@pytest.mark.parametrize("lens,counts,hd", [([5000, 2049, 1], [1, 1, 1], 128), ([2500], [6], 128), ([1200, 700], [1, 2], 256), ([3500, 1500, 300], [40, 20, 30], 128), ([2100, 900], [40, 33], 256)])
def test_attention_in_chunks(k, act, lens, counts, hd):
    """Sequences cut over several CTAs, whose parts are joined."""
    for room in (0, ROOM) if max(counts) >= 16 else (0,):
        p = _filled(k, lens, 1, hd, 64, room=room)
        max_len = 0 if room else None
        p.attend(counts, 4, max_len=max_len)
        p.attend(counts, 4, qpos=[n // (i + 1) - 1 if n > 1 else 0 for n, m in zip(lens, counts) for i in range(m)], seed=1, max_len=max_len)
        k.dev.check_status()


def test_attention_long_sequences_whole(k):
    """So many sequences that none is cut: a warp's share of the long ones is more tiles than it remembers pages of at a time."""
    p = _filled(k, [9000, 4500] + [5] * 90, 1, 128, 32)
    p.attend([1] * 92, 2)
    p = _filled(k, [2400] + [7] * 320, 1, 256, 128)
    p.attend([1] * 321, 9)
    k.dev.check_status()


def test_attention_few_rows_of_many_heads(k, act):
    """16 heads a kv head: rows whose heads lie in two tiles of pairs."""
    for hd, counts in ((128, [1, 2]), (128, [1, 5]), (256, [2, 3])):
        p = _filled(k, [70, 300], 2, hd, 32)
        p.attend(counts, 32)
    k.dev.check_status()


@pytest.mark.parametrize("hd", [128, 256])
def test_attention_repeats_bit_for_bit(k, hd):
    """The same call many times, with the GPU to itself and behind other calls: the same bits, and no wait that runs out."""
    p = _filled(k, [129, 257, 128, 1, 900], 1, hd, 128, room=ROOM)
    counts, nq = [20, 33, 16, 1, 24], 16
    first = [p.attend(counts, nq, max_len=0), p.attend(counts, nq, seed=1, max_len=400 * 128)]
    rows, width = sum(counts), nq * hd
    gen = torch.Generator().manual_seed(100)
    q = (torch.randn(rows + 2, width, generator=gen) * 1.5).to(k.dev.act_torch).cuda()
    g = torch.randn(rows + 2, width + 4, generator=gen).cuda()
    start = p.ints(np.concatenate([[0], np.cumsum(counts)]))
    y = torch.empty_like(first[0])
    for i in range(200):
        y.fill_(SENTINEL)
        p.ops.attention(None, p.gpu, 0, q, g, start, None, y, rows, width, width + 4, width + 8, nq, max(counts), 0 if i % 2 else 300 * 128)
        if i % 3 == 0:
            torch.cuda.synchronize()
        if i % 2:
            assert torch.equal(y, first[0]), i
    k.dev.check_status()


def test_attention_engines_agree(k):
    """dc_set_engine keeps a call off tcgen05; what scratch_bytes says is what the call takes, on either."""
    p = _filled(k, [1500, 700], 2, 128, 32, room=ROOM)
    counts, nq = [60, 33], 8
    try:
        for engine in (Engine.Tcgen05, Engine.MmaSync):
            k.dev.set_engine(Family.Attn, engine)
            k.dev.reserve_workspace(p.ops.attention_scratch_bytes(p.gpu, nq, 60, 0))
            k.dev.set_workspace_frozen(True)
            before = k.dev.launches
            p.attend(counts, nq, max_len=0)
            assert k.dev.launches - before == (2 if engine == Engine.Tcgen05 else 1)      # cut in chunks there, whole or joined in place here
            k.dev.set_workspace_frozen(False)
        k.dev.check_status()
    finally:
        k.dev.set_workspace_frozen(False)
        k.dev.set_engine(Family.Attn, Engine.Tcgen05)


def test_attention_one_key_is_its_value(k):
    """A row that sees one key gets that key's V: codes times scale, exactly (they fit fp16)."""
    p = _filled(k, [1], 2, 128, 16)
    q = torch.ones(1, 512, dtype=torch.float16, device="cuda")
    y = torch.empty(1, 512, dtype=torch.float16, device="cuda")
    p.ops.attention(None, p.gpu, 0, q, None, p.ints([0, 1]), None, y, 1, 512, 0, 512, 4, 1, 1)
    want = np.repeat(kv8.DECODE[p.model.v[0, p.model.table[0, 0], :, 0]] * p.model.v_scale[0, p.model.table[0, 0]][:, None], 2, axis=0)
    # the division by the sum of one weight (exactly 1) and the weight 2^0: nothing rounds
    assert np.array_equal(y.double().cpu().numpy().reshape(4, 128), want)


def test_attention_scales_far_apart(k, act):
    """Pages whose K and V scales differ by many powers of two; a page of large values that a row weighs as nothing."""
    p = Pair(k, n_pages=8, nkv=1, n_seqs=1, page=16)
    for i, size in enumerate([1e-3, 30.0, 1.0, 2e-2]):
        p.extend([16])

        def spoil(new, size=size, i=i):
            new[1].mul_(size)
            new[0].mul_(1 if i != 1 else 0.1)
        p.append([16], 1.0, seed=i, spoil=spoil)
    p.attend([9], 4)
    p.attend([1], 4, size=20.0)
    p.attend([3], 4, size=0.0)
    k.dev.check_status()


def test_attention_queries_at_the_ends_of_their_type(k, act):
    p = _filled(k, [40], 1, 128, 16, size=1e-4 if act == torch.float16 else 1.0)
    top = torch.finfo(act).max
    p.attend([2], 4, spoil=lambda q: q.copy_(q.sign() * (top / 8 if act == torch.float16 else 1.0)))
    p.attend([2], 4, spoil=lambda q: q.mul_(torch.finfo(act).smallest_normal * 4))
    if act == torch.bfloat16:       # a few large elements among very small ones
        p.attend([1], 4, spoil=lambda q: q[:, 3:].mul_(1e-30))
    bad = torch.full((1, 512), 1.0, dtype=act, device="cuda")
    bad[0, 5] = float("nan")
    bad[0, 128 + 9] = -float("inf")
    bad[0, 256 + 9] = float("inf")
    y = torch.empty(1, 512, dtype=act, device="cuda")
    p.ops.attention(None, p.gpu, 0, bad, None, p.ints([0, 1]), None, y, 1, 512, 0, 512, 4, 1, 40)
    assert torch.isnan(y[0, :384]).all() and torch.isfinite(y[0, 384:]).all()      # each head of its own
    k.dev.check_status()


def test_attention_layers_and_forked_sequences(k):
    """Three sequences that share pages, in the second of two layers."""
    p = Pair(k, layers=2, n_pages=12, nkv=2, n_seqs=3, page=16)
    p.extend([37, 0, 0])
    p.append([37, 0, 0], seed=5, layer=0)
    p.append([37, 0, 0], seed=6, layer=1)
    p.fork([0, 0], [1, 2], False)
    p.extend([0, 1, 20])
    p.append([0, 1, 20], seed=7, layer=1)
    p.same()
    p.attend([1, 1, 20], 4, layer=1)
    k.dev.check_status()


def test_attention_positions_past_the_end_are_reported(k):
    p = _filled(k, [20], 1, 128, 16)
    q = torch.ones(2, 128, dtype=k.dev.act_torch, device="cuda")
    y = torch.empty(2, 128, dtype=k.dev.act_torch, device="cuda")
    p.ops.attention(None, p.gpu, 0, q, None, p.ints([0, 2]), p.ints([20, 19]), y, 2, 128, 0, 128, 1, 2, 20)
    with pytest.raises(KernelError, match="position"):
        k.dev.check_status()
    assert torch.equal(y[0], y[1])
    p.ops.attention(None, p.gpu, 0, q, None, p.ints([0, 2]), None, y, 2, 128, 0, 128, 1, 2, 10)
    with pytest.raises(KernelError, match="max_len"):
        k.dev.check_status()
    for start, rows, most in (([0, 3], 2, 2), ([1, 0], 2, 2), ([0, 2], 2, 1)):
        y.fill_(SENTINEL)
        p.ops.attention(None, p.gpu, 0, q, None, p.ints(start), None, y, rows, 128, 0, 128, 1, most, 20)
        with pytest.raises(KernelError, match="offsets"):
            k.dev.check_status()
        assert (y == SENTINEL).all()


def test_attention_refusals(k):
    p = _filled(k, [20], 2, 128, 16)
    q = torch.ones(2, 1024, dtype=k.dev.act_torch, device="cuda")
    g = torch.ones(2, 1024, device="cuda")
    y = torch.empty(2, 1024, dtype=k.dev.act_torch, device="cuda")
    s = p.ints([0, 1])
    good = dict(layer=0, q=q, gate=g, q_start=s, qpos=None, y=y, rows=1, ldq=1024, ldg=1024, ldy=1024, nq=8, max_q=1, max_len=20)
    p.ops.attention(None, p.gpu, **good)
    p.ops.attention(None, p.gpu, **{**good, "rows": 0})
    p.ops.attention(None, p.gpu, **{**good, "max_q": 0})
    for bad in ({"layer": 1}, {"q": None}, {"q_start": None}, {"y": None}, {"nq": 7}, {"nq": 0}, {"nq": 34}, {"ldq": 1016}, {"ldq": 1028}, {"ldy": 1020}, {"ldg": 1022},
                {"ldg": 512}, {"q": (q, 8)}, {"y": (y, 2)}, {"gate": (g, 4)}, {"max_q": 1 << 27}):
        with pytest.raises(KernelError):
            p.ops.attention(None, p.gpu, **{**good, **bad})
    k.dev.check_status()


def test_another_stream_a_graph_and_a_frozen_workspace(k):
    """The whole round on a side stream, then captured and replayed, with the workspace reserved and frozen: same bits."""
    p = _filled(k, [2900, 10], 2, 128, 64)
    nq, width = 8, 1024
    q = torch.randn(2, width, device="cuda").to(k.dev.act_torch)
    x = torch.randn(2, 2, 256, device="cuda").to(k.dev.act_torch)
    start, add = p.ints([0, 1, 2]), p.ints([1, 1])
    y = torch.empty(2, width, dtype=k.dev.act_torch, device="cuda")
    k.dev.reserve_workspace(max(p.ops.attention_scratch_bytes(p.gpu, nq, 1, 2950), p.ops.pages_scratch_bytes(p.gpu)))
    k.dev.set_workspace_frozen(True)
    try:
        def step(stream):
            p.ops.extend(stream, p.gpu, add)
            p.ops.append(stream, p.gpu, 0, x[0], x[1], 256, 256, start, 2, 1)
            p.ops.attention(stream, p.gpu, 0, q, None, start, None, y, 2, width, 0, width, nq, 1, 2950)

        side = torch.cuda.Stream()
        saved = [t.clone() for t in (p.gpu.k, p.gpu.v, p.gpu.k_scale, p.gpu.v_scale, p.gpu.table, p.gpu.lens, p.gpu.refs)]
        side.wait_stream(torch.cuda.current_stream())
        step(side)
        side.synchronize()
        first = y.clone()

        def restore():
            for t, s in zip((p.gpu.k, p.gpu.v, p.gpu.k_scale, p.gpu.v_scale, p.gpu.table, p.gpu.lens, p.gpu.refs), saved):
                t.copy_(s)
        restore()
        allocs = k.dev.alloc_count
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(side)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, y) and k.dev.alloc_count == allocs
        graph.replay()      # another token each
        torch.cuda.synchronize()
        assert p.gpu.lens.tolist() == [2902, 12] and not torch.equal(first, y)
        k.dev.check_status()
    finally:
        k.dev.set_workspace_frozen(False)


def test_a_graph_keeps_its_workspace(k):
    """Scratch that grows after a capture, used by other calls in between, leaves the graph's own alone; a capture that would allocate is refused."""
    from decide_b200.kernels import Device, Kernels
    dev = Device(0)
    fresh = Kernels(dev)
    p = _filled(fresh, [2900, 10], 2, 128, 64)
    nq, width = 8, 1024
    q = torch.randn(2, width, device="cuda").to(dev.act_torch)
    start = p.ints([0, 1, 2])
    y, z = (torch.empty(2, width, dtype=dev.act_torch, device="cuda") for _ in range(2))
    dev.reserve_workspace(p.ops.pages_scratch_bytes(p.gpu))
    need = p.ops.attention_scratch_bytes(p.gpu, nq, 1, 2950)
    assert need > dev.workspace_bytes

    def attend(out):
        p.ops.attention(None, p.gpu, 0, q, None, start, None, out, 2, width, 0, width, nq, 1, 2950)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q.mul_(1)
        with pytest.raises(KernelError, match="during a capture"):
            attend(y)
    before = dev.workspace_bytes
    dev.reserve_workspace(need)
    assert dev.workspace_bytes == need > before
    attend(z)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(y)
    dev.reserve_workspace(need + (8 << 20))
    filler = [torch.full((need // 4 + 64,), float("nan"), device="cuda") for _ in range(8)]   # what the old block's memory would hold by now
    for _ in range(3):
        y.zero_()
        graph.replay()
        attend(z)
        torch.cuda.synchronize()
        assert torch.equal(y, z)
    dev.check_status()
    del graph, filler
    dev.close()


def test_follow_up_questions_share_a_state(k):
    """As they would be used: a request's state is written once, three questions fork it, each adds its rows and attends; one ends, the
    cache closes up, the others go on a token at a time and see what they saw before."""
    p = Pair(k, layers=2, n_pages=30, nkv=2, n_seqs=4, max_pages=10, page=16)
    nq = 8
    p.extend([75, 0, 0, 0])
    for layer in range(2):
        p.append([75, 0, 0, 0], seed=layer, layer=layer)
        p.attend([75, 0, 0, 0], nq, seed=layer, layer=layer)
    p.fork([0, 0, 0], [1, 2, 3], False)
    rows = [0, 18, 5, 33]
    p.extend(rows)
    for layer in range(2):
        p.append(rows, seed=10 + layer, layer=layer)
        p.attend(rows, nq, seed=10 + layer, layer=layer)
    p.same()
    again = p.attend([0, 1, 0, 1], nq, seed=20)
    p.free([2])
    p.compact()
    p.same()
    assert torch.equal(p.attend([0, 1, 0, 1], nq, seed=20), again)      # pages have moved: not a bit changes
    for step in range(3):
        p.extend([0, 1, 0, 1])
        for layer in range(2):
            p.append([0, 1, 0, 1], seed=30 + step, layer=layer)
            p.attend([0, 1, 0, 1], nq, seed=30 + step, layer=layer)
    p.same()
    k.dev.check_status()
