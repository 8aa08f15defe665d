"""The paged 8-bit K/V cache on the GPU at the ends of what its entry points allow: terms far below a row's largest, what a row does not
attend, page bookkeeping that is wrong. Each case runs on the forms of the attention that it concerns: few rows, two sets of eight (row, head)
pairs, whole tiles of the tensor cores. The numpy model and its tolerances are those of oracle/kv8.py."""
import functools

import numpy as np
import pytest
import torch

from decide_b200.kernels import KernelError, Kv8Cache
from oracle import kv8
from tests.test_kv8_gpu import ROOM, Pair

pytestmark = pytest.mark.gpu

# What the weights of the V product may be off by, numerator and total together, and what a small one may be off by of the row's largest
# term: two fp16 parts each take half of 2^-11 of what the one before left; 11 bits in both sums, 2^-10 apart at most. A row's largest
# weight is at least 2^7, so that half a step of the smallest fp16 numbers, 2^-25, is 2^-32 of it.
TWO_PARTS = dict(weight=2.0 ** -22, least=2.0 ** -32)
ONE_PART = dict(weight=2 * 2.0 ** -11, least=2.0 ** -32)
# rows that the last sequence brings, query heads and sequences for the three forms: up to eight pairs a tile, sixteen, 128 or 256
FORMS = {"rows": dict(rows=1, nq=4, seqs=1), "pairs": dict(rows=5, nq=4, seqs=120), "tiles": dict(rows=33, nq=4, seqs=1)}


def filled(k, form, n, hd, k_rows, v_rows, page=16):
    """A cache whose last sequence holds n tokens with the K and V that k_rows(x), v_rows(x) make of normal numbers x [n, hd], written a page at a
    time; the sequences before it hold one token each."""
    f = FORMS[form]
    p = Pair(k, n_pages=f["seqs"] - 1 + n // page + 2, nkv=1, hd=hd, n_seqs=f["seqs"], max_pages=max(n // page + 1, ROOM // page if form == "tiles" else 0), page=page)
    p.model.attention = functools.partial(p.model.attention, **(TWO_PARTS if form == "rows" else ONE_PART))
    counts = [1] * (f["seqs"] - 1) + [n]

    def spoil(new):
        for x, rows in zip(new, (k_rows, v_rows)):
            at = len(x) - 2 - n
            x[at:at + n, :hd] = rows(x[at:at + n, :hd].float()).to(x.dtype)
    p.extend(counts)
    p.append(counts, spoil=spoil)
    return p, [1] * (f["seqs"] - 1) + [f["rows"]], f["nq"]


def attend(p, form, counts, nq, **kw):
    return p.attend(counts, nq, max_len=0 if form == "tiles" else None, **kw)


# ---------------------------------------------------------------- terms far below the largest

@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("gap", [12, 16, 20, 24, 26])
@pytest.mark.parametrize("form", FORMS)
def test_a_key_that_takes_nearly_all_the_weight_hides_nothing(k, act, form, gap, hd):
    """The first key weighs 2^gap as much as any other, and its V is zero: what is left is the others' V, 2^-gap of it each."""
    n = 700

    def k_rows(x):
        x = x * 0.01
        x[:, 0] = 0
        x[0, 0] = gap * np.log(2) * hd ** 0.5 / 8
        return x

    def v_rows(x):
        x = (x.abs() + 0.25) * 1024
        x[0] = 0
        return x
    p, counts, nq = filled(k, form, n, hd, k_rows, v_rows)

    def spoil(q):
        q.mul_(0.01)
        q.view(len(q), -1, hd)[:, :, 0] = 8
    attend(p, form, counts, nq, gate=False, spoil=spoil)
    k.dev.check_status()


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("gap", [8, 16, 18, 20])
@pytest.mark.parametrize("form", FORMS)
def test_a_page_of_one_large_value_hides_nothing(k, act, form, gap, hd):
    """One value of the first page raises the page's V scale to 2^gap times the others'; in the other columns that page's codes are zeros. All
    keys behind it have one score, so that what their weights are rounded by does not average out. V is positive, so that errors are relative to the
    sums: half a step of the output's type (2^-8 for bf16, 2^-11 for fp16), 2^-10 for weights of 11 bits in product and total, and 2^-14 for scores
    below 1 (18 steps of 2^-22) and exponents below 2^5 (2^-21 of them, twice): together less than half a step and 2^-9."""
    n = 700
    size = 2.0 ** -10 if act == torch.float16 else 1.0

    def k_rows(x):
        x = x * 0
        x[:16, 0] = 0.3 * hd ** 0.5 / 8
        return x

    def v_rows(x):
        x = (x.abs() + 0.25).clamp(max=3.5) * size      # scales of 2^-7, the first page's 2^(gap - 7)
        x[:16, 1:] = 0
        x[3, 0] = 3.5 * size * 2.0 ** gap
        return x
    p, counts, nq = filled(k, form, n, hd, k_rows, v_rows)

    def spoil(q):
        q.mul_(0)
        q.view(len(q), -1, hd)[:, :, 0] = 8
    y = attend(p, form, counts, nq, gate=False, spoil=spoil)
    q_rows, j = FORMS[form]["rows"], len(counts) - 1
    got = y[j:j + q_rows, :nq * hd].double().cpu().numpy().reshape(q_rows, nq, hd)[:, :, 1:]
    codes, scales = p.model.tokens(0, j, 0, p.model.v, p.model.v_scale)
    key, key_scale = p.model.tokens(0, j, 0, p.model.k, p.model.k_scale)
    weight = np.exp(key[:, 0] * key_scale * 8 / hd ** 0.5)
    for i in range(q_rows):
        see = n - q_rows + i + 1
        want = weight[:see] @ (codes[:see] * scales[:see, None])[:, 1:] / weight[:see].sum()
        assert (np.abs(got[i] - want) < (torch.finfo(act).eps / 2 + 2.0 ** -9) * want).all()
    k.dev.check_status()


# ---------------------------------------------------------------- strides

@pytest.mark.parametrize("page,stride", [(128, 40_000_000), (64, 95_000_000)])
def test_tokens_farther_apart_than_32_bits(k, page, stride):
    """Tokens outermost: a page's last tokens lie more than 2^32 bytes behind its first. The same bits as from a cache that is contiguous."""
    memory = torch.empty(page * stride, dtype=torch.uint8, device="cuda")
    for hd in (128, 256):
        n, rows, nq = 2 * page + page // 2 + 3, 33, 4
        plain, far = (Pair(k, n_pages=5, nkv=1, hd=hd, n_seqs=1, max_pages=ROOM // page, page=page) for _ in range(2))
        view = [memory.as_strided((1, 5, 1, page, hd), (0, hd, 0, stride, 1), at) for at in (0, 1 << 20)]
        far.gpu = type(far.gpu)(*view, far.gpu.k_scale, far.gpu.v_scale, far.gpu.table, far.gpu.lens, far.gpu.refs)
        y = []
        for p in (plain, far):
            p.extend([n])
            p.append([n], seed=1)
            y.append([p.attend([1], nq), p.attend([rows], nq, max_len=0)])
        assert all(torch.equal(a, b) for a, b in zip(*y))
        for name in ("k", "v"):
            ids = plain.gpu.table[0, :3].long()
            for i, q in enumerate(ids.tolist()):
                held = min(page, n - i * page)
                assert torch.equal(getattr(plain.gpu, name)[0, q, 0, :held], getattr(far.gpu, name)[0, q, 0, :held])
    k.dev.check_status()
    del memory, view, far, p
    torch.cuda.empty_cache()


# ---------------------------------------------------------------- what a row does not attend

def spread(k, form, hd, spare=0):
    """The form's last sequence over 300 tokens, with rows at the places `at`; pages 0 and 1 are free and hold the codes for NaN. `spare` tokens more are
    its own but not written."""
    f = FORMS[form]
    rows, n = max(f["rows"], 2), 300
    p = Pair(k, n_pages=f["seqs"] + n // 16 + spare // 16 + 6, nkv=2, hd=hd, n_seqs=f["seqs"] + 1, max_pages=ROOM // 16 if form == "tiles" else 30, page=16)
    p.extend([20] + [1] * (f["seqs"] - 1) + [0])
    p.append([20] + [1] * (f["seqs"] - 1) + [0])
    p.extend([0] * f["seqs"] + [n])
    p.append([0] * f["seqs"] + [n], seed=1)
    p.free([0])
    p.gpu.k[:, :2], p.gpu.v[:, :2], p.model.k[:, :2], p.model.v[:, :2] = 0x7F, 0x7F, 0x7F, 0x7F
    if spare:
        p.extend([0] * f["seqs"] + [spare])
    at = [(i * 23 + 3) % 60 for i in range(rows)]       # within the first four pages
    return p, [0] + [1] * (f["seqs"] - 1) + [rows], [0] * (f["seqs"] - 1) + at, f["nq"]


def call(p, counts, nq, qpos, seed=5):
    """The attention call as it is, without the model: outputs [rows, nq * hd] in float64."""
    start, hd, act = np.concatenate([[0], np.cumsum(counts)]), p.gpu.hd, p.dev.act_torch
    rows, width = int(start[-1]), nq * hd
    q = torch.randn(rows, width, generator=torch.Generator().manual_seed(seed)).to(act)
    y = torch.full((rows, width), 7.0, dtype=act, device="cuda")
    p.ops.attention(None, p.gpu, 0, q.cuda(), None, p.ints(start), p.ints(qpos), y, rows, width, 0, width, nq, max(counts), 0)
    want, tol = p.model.attention(0, q.double().numpy().reshape(rows, nq, hd), None, start, np.array(qpos), torch.finfo(act).eps / 2, act == torch.bfloat16)
    return y.double().cpu().numpy(), want, tol


@pytest.mark.parametrize("spare", [1, 4, 40])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_tokens_that_are_not_written_yet_reach_no_row(k, act, form, hd, spare):
    """A sequence that has been lengthened but not written to: its memory holds the codes for NaN, its new pages' scales are NaN. Rows that see all the
    written tokens, in the middle of a page, and rows that see few."""
    p, counts, qpos, nq = spread(k, form, hd, spare)
    qpos[-1] = 299
    got, want, tol = call(p, counts, nq, qpos)
    assert (np.abs(got - want) <= tol).all()
    k.dev.check_status()


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_a_bad_page_reaches_the_rows_that_attend_it_alone(k, act, form, hd):
    p, counts, qpos, nq = spread(k, form, hd)
    last = len(qpos) - 1
    qpos[last] = 299                                        # attends the page that is spoilt below; the others do not
    j = len(counts) - 1
    first = last - counts[j] + 1                            # the sequence's first row
    for bad in (p.gpu.n_pages, -1):
        for column in (6, 18):                              # in the middle, and where the sequence ends
            good = int(p.gpu.table[j, column])
            p.gpu.table[j, column] = bad
            got, want, tol = call(p, counts, nq, qpos)
            p.gpu.table[j, column] = good
            assert np.isnan(got[last]).all()
            assert (np.abs(got[:last] - want[:last]) <= tol[:last]).all()
            with pytest.raises(KernelError, match="outside the pool"):
                k.dev.check_status()
    got, want, tol = call(p, counts, nq, qpos)
    assert (np.abs(got - want) <= tol).all()
    k.dev.check_status()
    # the first page: all that attend anything are NaN, a row that attends nothing is zero
    qpos[first] = kv8.NO_KEYS
    p.gpu.table[j, 0] = p.gpu.n_pages
    got, want, tol = call(p, counts, nq, qpos)
    assert (got[first] == 0).all() and np.isnan(got[first + 1:]).all() and (np.abs(got[:first] - want[:first]) <= tol[:first]).all()
    with pytest.raises(KernelError, match="outside the pool"):
        k.dev.check_status()


@pytest.mark.parametrize("scale", [-3.0, 0.0, float("inf"), float("nan")])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_scales_of_pages_nobody_holds_are_not_used(k, act, form, hd, scale):
    """Keys are taken sixteen, and scores 64, at a time: what lies past the last key that any row attends has no page."""
    p, counts, qpos, nq = spread(k, form, hd)
    qpos = [i % 40 for i in qpos]
    for s in (p.gpu.k_scale, p.gpu.v_scale):
        s[:, :2] = scale
    got, want, tol = call(p, counts, nq, qpos)
    assert (np.abs(got - want) <= tol).all()
    k.dev.check_status()


# ---------------------------------------------------------------- pages that are wrong

def test_a_page_freed_too_often_ends_at_none(k):
    """Two hundred sequences that all name one page, of which the counts know fewer, freed in one call: no count falls below zero."""
    for holders in (0, 1, 3, 199, 200):
        for _ in range(10):
            p = Pair(k, n_pages=300, nkv=1, n_seqs=200, max_pages=2, page=16)
            p.extend([20] * 100 + [0] * 100)
            p.gpu.lens[100:] = 3
            p.gpu.table[:, 0] = 250
            p.gpu.refs[250] = holders
            p.ops.free(None, p.gpu, p.ints(range(200)), 200)
            assert int(p.gpu.refs[250]) == 0 and p.gpu.lens.tolist() == [0] * 200
            assert int(p.gpu.refs.sum()) == 100         # what the table no longer names
            if holders < 200:
                with pytest.raises(KernelError, match="freed more often"):
                    k.dev.check_status()
            else:
                k.dev.check_status()


# ---------------------------------------------------------------- the forms on inputs that are not easy

def grown(k, form, hd, sizes, page=16, nkv=2, layers=1, spoil=None, bits=True):
    """The form's last sequence, written a page at a time with K and V of the sizes given; the ones before it hold 7 tokens."""
    f = FORMS[form]
    n = page * len(sizes)
    p = Pair(k, layers=layers, n_pages=f["seqs"] - 1 + len(sizes) + 3, nkv=nkv, hd=hd, n_seqs=f["seqs"], max_pages=max(len(sizes) + 1, ROOM // page if form == "tiles" else 0), page=page)
    if bits:
        p.model.attention = functools.partial(p.model.attention, **(TWO_PARTS if form == "rows" else ONE_PART))
    for i, (k_size, v_size) in enumerate(sizes):
        counts = [7 if i == 0 else 0] * (f["seqs"] - 1) + [page]
        p.extend(counts)

        def scaled(new, i=i):
            new[0].mul_(k_size)
            new[1].mul_(v_size)
            if spoil:
                spoil(i, new)
        p.append(counts, seed=i, spoil=scaled)
    rows = max(f["rows"], 3)
    return p, [1] * (f["seqs"] - 1) + [rows], f["nq"] if form != "rows" else 2, n


def places(counts, at):
    """Positions: the first sequences' last tokens, then `at` over and over."""
    return [6] * (len(counts) - 1) + [at[i % len(at)] for i in range(counts[-1])]


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_scores_and_scales_that_keep_growing(k, act, form, hd):
    """Each page's scores are larger than the last one's by more than the running maximum may lag, and V's scales rise and fall by powers of two: the
    sums are scaled again and again, in registers and in tensor memory."""
    sizes = [(0.05 * 1.45 ** i, (1.0, 0.02, 30.0, 0.5)[i % 4]) for i in range(20)]
    p, counts, nq, n = grown(k, form, hd, sizes)
    attend(p, form, counts, nq, gate=False)
    attend(p, form, counts, nq, qpos=places(counts, [n - 1, 0, 200, kv8.NO_KEYS, 77, 63, 64]), seed=1)
    p, counts, nq, n = grown(k, form, hd, sizes[::-1])
    attend(p, form, counts, nq, seed=2)
    attend(p, form, counts, nq, qpos=places(counts, [n - 1, 0, 200, kv8.NO_KEYS, 77, 63, 64]), seed=3)
    k.dev.check_status()


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_poisoned_pages_reach_the_rows_that_attend_them_alone(k, act, form, hd):
    """A K that is not finite in one head's page, a V in another's: NaN for the rows of that head that attend the page."""
    for bad, (page_k, page_v) in ((float("nan"), (17, 18)), (float("inf"), (3, 18)), (-float("inf"), (18, 4)), (float("nan"), (0, 18))):
        def spoil(i, new):
            if i == page_k:
                new[0][-3, hd + 5] = bad        # the page's last token, the second kv head
            if i == page_v:
                new[1][-3, 9] = bad             # the first
        p, counts, nq, n = grown(k, form, hd, [(1.0, 1.0)] * 19, spoil=spoil)
        assert int(np.isnan(p.model.k_scale[0, p.model.table[-1, :19]]).sum()) == 1
        attend(p, form, counts, nq, qpos=places(counts, [n - 1, 40, 3, kv8.NO_KEYS, 16 * 17 + 2, 16 * 17 - 1, 47, 48]))
        attend(p, form, counts, nq, qpos=places(counts, [15, 40, 3, kv8.NO_KEYS]), gate=False)
    k.dev.check_status()


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_scales_far_apart(k, act, form, hd):
    """Pages of zeros, of very small and of large values side by side."""
    top = 2.0 ** 12 if act == torch.float16 else 2.0 ** 40
    sizes = [(1e-3, 1.0), (1.0, 1e-4), (0.0, 0.0), (0.1, 30.0), (1.0, 0.0), (0.5, 1 / top), (0.0, 1.0), (1.0, 1e-3)] * 3
    p, counts, nq, n = grown(k, form, hd, sizes)
    attend(p, form, counts, nq)
    attend(p, form, counts, nq, qpos=places(counts, [n - 1, 15, 16, kv8.NO_KEYS, 31, 47, 200]), seed=1)
    attend(p, form, counts, nq, size=0.0, seed=2)
    p, counts, nq, n = grown(k, form, hd, [(1.0, 0.0)] * 6)      # V of zeros: zeros
    y = attend(p, form, counts, nq)
    assert (y[:sum(counts), :nq * hd] == 0).all()
    k.dev.check_status()


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_queries_at_the_ends_of_their_type(k, act, form, hd):
    small = 1e-4 if act == torch.float16 else 1.0
    top = torch.finfo(act).max
    p, counts, nq, n = grown(k, form, hd, [(small, 1.0)] * 6)
    attend(p, form, counts, nq, spoil=lambda q: q.copy_(q.sign() * (top / 8 if act == torch.float16 else 1.0)))
    attend(p, form, counts, nq, spoil=lambda q: q.mul_(torch.finfo(act).smallest_normal * 4))
    attend(p, form, counts, nq, spoil=lambda q: q.zero_())
    if act == torch.bfloat16:
        attend(p, form, counts, nq, spoil=lambda q: q[:, 3:].mul_(1e-30))
        p, counts, nq, n = grown(k, form, hd, [(2.0 ** -50, 1.0)] * 6)
        attend(p, form, counts, nq, spoil=lambda q: q.mul_(2.0 ** 50))
    # values that are not finite: their own row and head, and not where it attends nothing
    start = np.concatenate([[0], np.cumsum(counts)])
    rows, width = int(start[-1]), nq * hd
    for bad in (float("nan"), float("inf"), -float("inf")):
        q = torch.ones(rows, width, dtype=act, device="cuda")
        row = rows - 2
        q[row, hd + 9] = bad
        q[rows - 1, 5] = bad
        y = torch.empty(rows, width, dtype=act, device="cuda")
        p.ops.attention(None, p.gpu, 0, q, None, p.ints(start), p.ints(places(counts, [n - 1])[:-1] + [kv8.NO_KEYS]), y, rows, width, 0, width, nq, max(counts), 0)
        nan = torch.isnan(y)
        assert nan[row, hd:2 * hd].all() and int(nan.sum()) == hd and (y[rows - 1] == 0).all()
    k.dev.check_status()


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_violations_of_a_call_skip_what_they_concern(k, act, form, hd):
    """Positions past the end attend all there is; rows of offsets that do not hold and sequences longer than said are not written, others are."""
    p, counts, nq, n = grown(k, form, hd, [(1.0, 1.0)] * 6)
    start = np.concatenate([[0], np.cumsum(counts)])
    rows, width, first = int(start[-1]), nq * hd, int(start[-2])
    gen = torch.Generator().manual_seed(9)
    q = torch.randn(rows + 1, width, generator=gen).to(act).cuda()

    def run(start, qpos, rows, most, max_len=0):
        y = torch.full((len(q), width), 7.0, dtype=act, device="cuda")
        p.ops.attention(None, p.gpu, 0, q, None, p.ints(start), None if qpos is None else p.ints(qpos), y, rows, width, 0, width, nq, most, max_len)
        return y
    last = places(counts, [n - 1])
    want = run(start, last, rows, max(counts))
    exact, tol = p.model.attention(0, q[:rows].double().cpu().numpy().reshape(rows, nq, hd), None, start, np.array(last), torch.finfo(act).eps / 2, act == torch.bfloat16)
    k.dev.check_status()
    got = run(start, last[:-2] + [n, 0x7FFFFFFF], rows, max(counts))
    with pytest.raises(KernelError, match="position"):
        k.dev.check_status()
    assert torch.equal(got, want)
    for s, r, most, word in ((start, rows - 1, max(counts), "offsets"), (start, rows, max(counts) - 1, "offsets"),
                             (list(start[:-1]) + [max(int(start[-2]) - 1, 0) if len(counts) > 1 else 0xFFFFFFFF], rows, max(counts), "offsets")):
        got = run(s, last, r, most)
        with pytest.raises(KernelError, match=word):
            k.dev.check_status()
        assert (got[first:] == 7).all() and (np.abs(got[:first].double().cpu().numpy() - exact[:first]) <= tol[:first]).all()    # (another `most` may cut the rows otherwise)
    if form != "tiles":     # max_len is what keeps the call on its form there
        got = run(start, last, rows, max(counts), n - 1)
        with pytest.raises(KernelError, match="max_len"):
            k.dev.check_status()
        assert (got[first:] == 7).all() and torch.equal(got[:first], want[:first])
    else:
        p.gpu.lens[-1] = p.gpu.max_pages * 16 + 1
        got = run(start, last, rows, max(counts))
        with pytest.raises(KernelError, match="longer"):
            k.dev.check_status()
        assert (got[first:] == 7).all()
    k.dev.check_status()


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_forked_sequences_in_the_second_layer(k, act, form, hd):
    """Two forks of one sequence grow apart and attend their own tokens behind the pages they share."""
    p = Pair(k, layers=2, n_pages=40, nkv=2, hd=hd, n_seqs=3, max_pages=ROOM // 16 if form == "tiles" else 12, page=16)
    nq, m = 4, {"rows": 1, "pairs": 7, "tiles": 33}[form]
    p.extend([101, 0, 0])
    for layer in range(2):
        p.append([101, 0, 0], seed=5 + layer, layer=layer)
    p.fork([0, 0], [1, 2], False)
    p.extend([0, 1, m])
    for layer in range(2):
        p.append([0, 1, m], seed=7 + layer, layer=layer)
    p.same()
    for layer in range(2):
        attend(p, form, [1, 1, m], nq, layer=layer, seed=layer)
        attend(p, form, [m, m, m], nq, layer=layer, seed=3)
    p.free([0])
    p.compact()
    p.same()
    attend(p, form, [0, 1, m], nq, layer=1, seed=4)
    k.dev.check_status()


def test_both_parts_of_a_weight_count(k):
    """Few rows over few keys, with small scores: the second fp16 part of the weights is what keeps fp32's accuracy."""
    for hd, n in ((128, 5), (128, 16), (256, 9), (128, 40)):
        p, counts, nq = filled(k, "rows", n, hd, lambda x: x * 0.2, lambda x: x)
        p.attend(counts, nq, gate=False, size=1.0)
        p.attend(counts, nq, gate=False, size=0.5, seed=1)
    k.dev.check_status()


@pytest.mark.parametrize("hd", [128, 256])
def test_the_same_call_gives_the_same_bits(k, hd):
    """Two calls that cut the keys differently, in turn and behind one another, each compared with its own first result."""
    p, counts, nq, n = grown(k, "tiles", hd, [(0.3 * 1.2 ** i, 1.0) for i in range(40)])
    rows, width = sum(counts), nq * hd
    q = torch.randn(rows, width, generator=torch.Generator().manual_seed(4)).to(k.dev.act_torch).cuda()
    start = p.ints(np.concatenate([[0], np.cumsum(counts)]))
    y = torch.empty(rows, width, dtype=k.dev.act_torch, device="cuda")
    first = {}
    for i in range(120):
        max_len = (0, n, ROOM // 2)[i % 3]
        y.fill_(7)
        p.ops.attention(None, p.gpu, 0, q, None, start, None, y, rows, width, 0, width, nq, max(counts), max_len)
        if i % 4 == 0:
            torch.cuda.synchronize()
        assert torch.equal(y, first.setdefault(max_len, y.clone())), (i, max_len)
    k.dev.check_status()


# ---------------------------------------------------------------- the largest and the smallest, captured calls

def test_the_largest_pool(k):
    """2^21 pages and 65,535 sequences: every page handed out, taken back, and the last of them (K and V beyond 2^32 bytes) written and attended to
    the bit as the first ones are."""
    n_pages, n_seqs, width, hd = 1 << 21, 65535, 32, 256
    cache = Kv8Cache(*(torch.empty(1, n_pages, 1, 16, hd, dtype=torch.uint8, device="cuda") for _ in range(2)), *(torch.ones(1, n_pages, 1, device="cuda") for _ in range(2)),
                     torch.zeros(n_seqs, width, dtype=torch.int32, device="cuda"), torch.zeros(n_seqs, dtype=torch.int32, device="cuda"),
                     torch.zeros(n_pages, dtype=torch.int32, device="cuda"))
    ops, dev = k.kv8, k.dev

    def ints(x):
        return torch.as_tensor(np.asarray(x, dtype=np.int32), device="cuda")
    ops.extend(None, cache, ints(np.full(n_seqs, 512)))
    dev.check_status()
    assert torch.equal(cache.table.view(-1).long(), torch.arange(n_seqs * width, device="cuda")) and int(cache.refs.sum()) == n_seqs * width
    ops.extend(None, cache, ints(np.eye(1, n_seqs, 3)[0]))
    with pytest.raises(KernelError, match="longer"):
        dev.check_status()
    ops.fork(None, cache, ints(np.arange(0, 65534, 2)), ints(np.arange(1, 65535, 2)), 32767, True)     # copies of the even ones in the odd ones' place
    dev.check_status()
    assert int(cache.refs.sum()) == n_seqs * width and int(cache.refs.max()) == 1
    ops.fork(None, cache, ints(np.arange(0, 65534, 2)), ints(np.arange(1, 65535, 2)), 32767, False)    # and shared
    dev.check_status()
    shared = torch.zeros(n_pages, dtype=torch.long, device="cuda").index_add_(0, cache.table.view(-1).long(), torch.ones(n_seqs * width, dtype=torch.long, device="cuda"))
    assert torch.equal(cache.refs.long(), shared) and int(shared.max()) == 2
    keep = [0, n_seqs - 1]
    ops.free(None, cache, ints(np.arange(1, n_seqs - 1)), n_seqs - 2)
    dev.check_status()
    assert int(cache.refs.sum()) == 2 * width and cache.lens[keep].tolist() == [512, 512]
    gen = torch.Generator().manual_seed(8)
    new = torch.randn(2, 512, hd, generator=gen).to(dev.act_torch).cuda().repeat(1, 2, 1)
    start = np.zeros(n_seqs + 1)
    start[1:] = 512
    start[-1] = 1024
    ops.append(None, cache, 0, new[0], new[1], hd, hd, ints(start), 1024, 512)
    for rows, nq in ((1, 4), (64, 4)):
        start[1:], start[-1] = rows, 2 * rows
        q = torch.randn(rows, nq * hd, generator=gen).to(dev.act_torch).cuda().repeat(2, 1)
        y = torch.empty_like(q)
        ops.attention(None, cache, 0, q, None, ints(start), None, y, 2 * rows, nq * hd, 0, nq * hd, nq, rows, 512)
        dev.check_status()
        assert torch.equal(y[:rows], y[rows:]) and torch.isfinite(y).all()
    before = y.clone()
    live = ints([0])
    ops.compact(None, cache, live)
    assert int(live) == 2 * width and int(cache.table[n_seqs - 1].max()) < 2 * width
    ops.attention(None, cache, 0, q, None, ints(start), None, y, 2 * rows, nq * hd, 0, nq * hd, nq, rows, 512)
    dev.check_status()
    assert torch.equal(y, before)
    del cache, before
    torch.cuda.empty_cache()


def test_the_smallest_pool(k):
    """One page, one sequence, one token; nothing in use."""
    p = Pair(k, n_pages=1, nkv=1, n_seqs=1, max_pages=1, page=16)
    p.compact()
    p.extend([0])
    p.free([0])
    p.attend([1], 1)                # an empty sequence: zero
    p.extend([1])
    p.append([1])
    p.attend([1], 1)
    p.attend([1], 16, qpos=[0])
    p.extend([15])
    p.append([15])
    p.attend([16], 16)
    p.compact()
    p.same()
    p.free([0])
    p.compact()
    p.same()
    k.dev.check_status()


def test_offsets_that_do_not_start_at_zero(k, act):
    """Rows before the first sequence's are nobody's: not read, not written."""
    p = Pair(k, nkv=1, n_seqs=2, page=16)
    p.extend([20, 3])
    gen = torch.Generator().manual_seed(1)
    new = torch.randn(2, 30, 128, generator=gen).to(act)
    new[:, :5] = float("nan")
    p.ops.append(None, p.gpu, 0, new[0].cuda(), new[1].cuda(), 128, 128, p.ints([5, 25, 28]), 28, 20)
    p.model.append(0, *(x[5:28].double().numpy().reshape(23, 1, 128) for x in new), [0, 20, 23])
    p.same()
    q = torch.randn(9, 128, generator=gen).to(act)
    y = torch.full((9, 128), 7.0, dtype=act, device="cuda")
    p.ops.attention(None, p.gpu, 0, q.cuda(), None, p.ints([4, 6, 8]), None, y, 8, 128, 0, 128, 1, 2, 20)
    want, tol = p.model.attention(0, q[4:8].double().numpy().reshape(4, 1, 128), None, [0, 2, 4], None, torch.finfo(act).eps / 2, act == torch.bfloat16)
    got = y.double().cpu().numpy()
    assert (got[:4] == 7).all() and (got[8:] == 7).all() and (np.abs(got[4:8] - want) <= tol).all()
    k.dev.check_status()


@pytest.mark.parametrize("form", FORMS)
def test_a_captured_round_of_every_call(k, form):
    """Fork, extend, append, attention, free and compact in one graph, replayed over restored and over changed caches: what the same calls give without
    a graph, and the graph's rows follow the lengths of the moment."""
    p, counts, nq, n = grown(k, form, 128, [(1.0, 1.0)] * 20)
    seqs, page, m = len(counts), 16, counts[-1]
    cache = Kv8Cache.empty(1, p.gpu.n_pages + 40, 2, 128, seqs + 2, p.gpu.max_pages, page)
    for name in ("k", "v", "k_scale", "v_scale"):
        getattr(cache, name)[:, :p.gpu.n_pages] = getattr(p.gpu, name).view(getattr(cache, name).dtype) if name in "kv" else getattr(p.gpu, name)
    cache.table[:seqs], cache.lens[:seqs], cache.refs[:p.gpu.n_pages] = p.gpu.table, p.gpu.lens, p.gpu.refs
    k.kv8.extend(None, cache, p.ints([0] * (seqs + 1) + [20]))      # what is freed below
    state = (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.table, cache.lens, cache.refs)
    saved = [t.clone() for t in state]
    gen = torch.Generator().manual_seed(6)
    start = p.ints([0] * (seqs + 1) + [m, m])
    add = p.ints([0] * seqs + [m, 0])
    new = torch.randn(2, m, 256, generator=gen).to(k.dev.act_torch).cuda()
    q = torch.randn(m, nq * 128, generator=gen).to(k.dev.act_torch).cuda()
    y, live = torch.zeros_like(q), p.ints([0])
    src, dst, gone = p.ints([seqs - 1]), p.ints([seqs]), p.ints([seqs + 1])
    max_len = 0 if form == "tiles" else 400
    k.dev.reserve_workspace(max(k.kv8.attention_scratch_bytes(cache, nq, m, max_len), k.kv8.pages_scratch_bytes(cache)))

    def round_of_calls():
        k.kv8.fork(None, cache, src, dst, 1)
        k.kv8.extend(None, cache, add)
        k.kv8.append(None, cache, 0, new[0], new[1], 256, 256, start, m, m)
        k.kv8.attention(None, cache, 0, q, None, start, None, y, m, nq * 128, 0, nq * 128, nq, m, max_len)
        k.kv8.free(None, cache, gone, 1)
        k.kv8.compact(None, cache, live)

    def restore():
        for t, s in zip(state, saved):
            t.copy_(s)
    round_of_calls()
    k.dev.check_status()
    want = [t.clone() for t in (*state, y, live)]
    restore()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        round_of_calls()
    for _ in range(3):
        restore()
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        k.dev.check_status()
        for a, b in zip((*state, y, live), want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))      # bits: free pages' scales are NaN
    graph.replay()          # over what the last one left: the fork is made again
    torch.cuda.synchronize()
    k.dev.check_status()
    assert torch.equal(y, want[-2]) and int(cache.lens[seqs]) == n + m
    del graph


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_tiny_queries_of_huge_keys(k, act, form, hd):
    """Queries at the small end of their type against keys at its large end, and the other way round: scores of an ordinary size."""
    up = 2.0 ** 13 if act == torch.float16 else 2.0 ** 124
    down = 2.0 ** -13 if act == torch.float16 else 2.0 ** -125
    p, counts, nq, n = grown(k, form, hd, [(up, 1.0)] * 6)
    attend(p, form, counts, nq, size=down)
    p, counts, nq, n = grown(k, form, hd, [(2.0 ** -13 if act == torch.float16 else 2.0 ** -50, 1.0)] * 6)
    attend(p, form, counts, nq, size=2.0 ** 13 if act == torch.float16 else 2.0 ** 50)
    k.dev.check_status()


def test_part_of_a_caches_sequences(k, act):
    """Calls over views of the table: the one sequence that brings many rows and the others that bring one each, apart."""
    p = Pair(k, n_pages=60, nkv=2, n_seqs=4, max_pages=ROOM // 16, page=16)
    p.extend([200, 33, 340, 1])
    p.append([200, 33, 340, 1])
    nq, counts = 8, [1, 1, 40, 1]
    start = np.concatenate([[0], np.cumsum(counts)])
    rows, width = int(start[-1]), nq * 128
    q = torch.randn(rows, width, generator=torch.Generator().manual_seed(2)).to(act)
    y = torch.full((rows, width), 7.0, dtype=act, device="cuda")
    g, on = p.gpu, q.cuda()
    many = Kv8Cache(g.k, g.v, g.k_scale, g.v_scale, g.table[2:3], g.lens[2:3], g.refs)
    p.ops.attention(None, many, 0, on, None, p.ints(start[2:4]), None, y, rows, width, 0, width, nq, 40)
    p.ops.attention(None, g, 0, on, None, p.ints([0, 1, 2, 2, 2]), None, y, rows, width, 0, width, nq, 1, 400)
    last = Kv8Cache(g.k, g.v, g.k_scale, g.v_scale, g.table[3:], g.lens[3:], g.refs)
    p.ops.attention(None, last, 0, on, None, p.ints(start[3:]), None, y, rows, width, 0, width, nq, 1, 400)
    want, tol = p.model.attention(0, q.double().numpy().reshape(rows, nq, 128), None, start, None, torch.finfo(act).eps / 2, act == torch.bfloat16)
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()
    k.dev.check_status()
