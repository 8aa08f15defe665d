"""What is measured of the paged 8-bit K/V cache: the write of new rows, the attention that reads it, and the page operations.

Each operator has a plain form here (elementary torch operations) and the call a user makes of the framework. The cache holds
e4m3 codes in pages of `page` tokens, one power-of-two fp32 scale per (page, kv head) for K and one for V: value = code * scale.
A sequence is a row of the page table and a length. The scale of a page is the least power of two 2^e with 448 * 2^e >= the
largest finite magnitude the page has held (e >= -60); it never falls while the page is in use, and when it rises the codes
already there are rounded again. A page that has taken in a value that is not finite has the scale NaN from then on.
"""
from __future__ import annotations

import random

import torch

own = False

SCALE_EXP_MIN = -60      # least exponent of a page's scale: a page of zeros has 2^-60
NO_KEYS = -1             # qpos of a padding row (0xFFFFFFFF as u32): it attends nothing
_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases

def listed():
    base = {"nkv": 8, "hd": 128, "page": 64, "token_major": False}
    return [
        # every running request adds one token to its cache
        dict(base, name="append, a token each", op="append", dtype="f16", seqs=64, rows=1, length=2307, ragged=False),
        # a follow-up question's rows join the state of a 2,491-token request, in the middle of a page
        dict(base, name="append, a follow-up", op="append", dtype="bf16", seqs=1, rows=178, length=2491, ragged=False, token_major=True),
        # the benchmark batch: 64 requests of 603 tokens, written whole
        dict(base, name="append, a batch", op="append", dtype="f16", seqs=64, rows=603, length=603, ragged=False),
        # one token of one short request: latency
        dict(base, name="attention, one token", op="attention", dtype="f16", nq=32, seqs=1, rows=1, length=603, ragged=False, gate=True, scattered=False),
        # one token for each of 64 running requests of unlike lengths
        dict(base, name="attention, a token each", op="attention", dtype="f16", nq=32, seqs=64, rows=1, length=2307, ragged=True, gate=True, scattered=False),
        # one token over one very long history
        dict(base, name="attention, long history", op="attention", dtype="bf16", nq=32, seqs=1, rows=1, length=131071, ragged=False, gate=False, scattered=False),
        # the six answer rows of each of 16 requests, at their places in the request
        dict(base, name="attention, answer rows", op="attention", dtype="f16", nq=32, seqs=16, rows=6, length=603, ragged=False, gate=True, scattered=True),
        # a follow-up question's rows over the shared state
        dict(base, name="attention, a follow-up", op="attention", dtype="f16", nq=32, seqs=1, rows=178, length=2491, ragged=False, gate=True, scattered=False),
        # a chunk of a long request's prefill
        dict(base, name="attention, a chunk", op="attention", dtype="f16", nq=32, seqs=1, rows=2048, length=8191, ragged=False, gate=False, scattered=False),
        # a few dozen rows for each of eight requests; heads of 256, small pages
        dict(base, name="attention, wide heads", op="attention", dtype="bf16", nq=16, nkv=4, hd=256, page=16, seqs=8, rows=64, length=1500, ragged=True, gate=True, scattered=False),
        # eight follow-up questions fork one state in all nine attention layers, grow, half of them end, the cache closes up
        dict(base, name="pages, eight follow-ups", op="pages", layers=9, parents=2, children=8, length=2491, grow=178, deep=False, free=4, compact=True),
        # independent copies of four requests' states in all nine attention layers
        dict(base, name="pages, copies", op="pages", layers=9, parents=4, children=4, length=2307, grow=0, deep=True, free=0, compact=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    case = {"op": rng.choice(["append", "attention", "attention", "pages"]), "page": rng.choice([16, 32, 64, 128]), "hd": rng.choice([128, 128, 256]),
            "nkv": rng.choice([1, 2, 4, 8]), "token_major": rng.random() < 0.25}
    if case["op"] == "append":
        seqs = _log_int(rng, 1, 64)
        rows = _log_int(rng, 1, 38592 // seqs)
        return dict(case, dtype=rng.choice(["f16", "bf16"]), seqs=seqs, rows=rows, length=rows + _log_int(rng, 1, 2048) - 1, ragged=rng.random() < 0.7)
    if case["op"] == "attention":
        group = rng.choice([1, 2, 3, 4, 4, 6, 8, 16])
        seqs = _log_int(rng, 1, 64)
        length = _log_int(rng, 1, min(131072, 2 ** 19 // (seqs * case["nkv"])))
        # at most the work of the largest listed case, and no more scores than 2^28 in the plain form
        rows = _log_int(rng, 1, max(1, min(2048, length, 2 ** 28 // (seqs * length * case["nkv"] * group))))
        rows = 1 if rng.random() < 0.4 else rows
        return dict(case, dtype=rng.choice(["f16", "bf16"]), nq=case["nkv"] * group, seqs=seqs, rows=rows, length=length, ragged=rng.random() < 0.7,
                    gate=rng.random() < 0.5, scattered=rng.random() < 0.3)
    parents = _log_int(rng, 1, 8)
    children = _log_int(rng, 1, 16)
    layers = rng.choice([1, 3, 9])
    length = _log_int(rng, 1, min(4096, 2 ** 18 // (layers * (parents + children))))
    return dict(case, layers=layers, parents=parents, children=children, length=length, grow=rng.choice([0, 1, 178, 603]), deep=rng.random() < 0.3,
                free=rng.randint(0, children), compact=rng.random() < 0.6)


def _rows(case):
    """Rows that each sequence brings: all alike, or from none to the most (the first has the most)."""
    rng = random.Random(17 * case["seqs"] + case["rows"])
    return [case["rows"] if not case["ragged"] or not j or case["rows"] == 1 else rng.randint(0, case["rows"]) for j in range(case["seqs"])]


def _lengths(case):
    """Tokens that each sequence holds, the new rows among them (the first has the most)."""
    rng = random.Random(31 * case["seqs"] + case["length"])
    return [case["length"] if not case["ragged"] or not j else max(m, rng.randint(case["length"] // 4, case["length"])) for j, m in enumerate(_rows(case))]


def _pages_of(length, page):
    return -(-length // page)


def _positions(case):
    """The query rows' positions where they are scattered: spread over the sequence, the last of several a padding row."""
    return [NO_KEYS if case["seqs"] == 1 and m > 1 and i == m - 1 else (i + 1) * n // (m + 1) for m, n in zip(_rows(case), _lengths(case)) for i in range(m)]


def work(case):
    token = case["nkv"] * case["hd"]                      # values of K, and of V, that a token has in one layer
    if case["op"] == "append":
        rows = sum(_rows(case))
        pages = sum(_pages_of(n, case["page"]) - (n - m) // case["page"] for m, n in zip(_rows(case), _lengths(case)) if m)
        return {"bytes": rows * token * 2 * (2 + 1) + pages * (4 + case["nkv"] * 2 * 4), "flops": rows * token * 2 * 3}
    if case["op"] == "attention":
        rows, lengths = _rows(case), _lengths(case)
        positions = _positions(case) if case["scattered"] else [n - m + i for m, n in zip(rows, lengths) for i in range(m)]
        first = [sum(rows[:j]) for j in range(len(rows))]
        seen = [max((p + 1 for p in positions[a:a + m]), default=0) for a, m in zip(first, rows)]
        pages = sum(_pages_of(n, case["page"]) for n in seen)
        pairs = sum(p + 1 for p in positions)
        return {"bytes": sum(seen) * token * 2 + pages * (4 + case["nkv"] * 2 * 4) + sum(rows) * case["nq"] * case["hd"] * (2 + 2 + (4 if case["gate"] else 0)),
                "flops": 4 * pairs * case["nq"] * case["hd"]}
    page_bytes = case["layers"] * 2 * case["nkv"] * (case["page"] * case["hd"] + 4)
    held, full = _pages_of(case["length"], case["page"]), case["length"] // case["page"]
    copied = case["children"] * (held if case["deep"] else held - full)
    table = case["children"] * _pages_of(case["length"] + case["grow"], case["page"])
    moved = 0
    if case["compact"]:     # what the children that stay own moves into the places of what the freed ones owned
        each = _pages_of(case["length"] + case["grow"], case["page"]) - (0 if case["deep"] else full)
        stay = case["children"] - case["free"]
        moved = min(case["free"], stay) * each
    return {"bytes": 2 * (copied + moved) * page_bytes + 2 * 4 * table + 4 * _pool(case), "flops": 0}


def _pool(case):
    most = _pages_of(case["length"] + case["grow"], case["page"])
    return (case["parents"] + case["children"]) * most + 3


# ---------------------------------------------------------------- inputs

def _exponent(amax):
    """Least e >= SCALE_EXP_MIN with 448 * 2^e >= amax (448 = 0.875 * 2^9), exactly."""
    mantissa, exponent = torch.frexp(amax)
    e = exponent - 9 + (mantissa > 0.875).to(torch.int32)
    return torch.where(amax > 0, e, torch.full_like(e, SCALE_EXP_MIN)).clamp(min=SCALE_EXP_MIN)


def _values(shape, gen, spread):
    """Rows as a projection with a few strong columns and heads of unlike size makes them: [..., head, token, dim]."""
    x = torch.randn(shape, generator=gen, device="cuda")
    column = 1 + 7 * (torch.rand(shape[-1], generator=gen, device="cuda") < 0.03).float()
    head = torch.exp2(spread * torch.randn(shape[-3], generator=gen, device="cuda"))
    return x * column * head[:, None, None]


def _ragged_table(counts, n_pages, gen):
    """A page table whose pages lie in no order: row j holds counts[j] pages, the rest of it page 0."""
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(counts), max(max(counts), 1), dtype=torch.int32, device="cuda")
    at = 0
    for j, c in enumerate(counts):
        table[j, :c] = order[at:at + c]
        at += c
    return table


def _codes(layers, n_pages, case, gen, spread):
    """Filled pages of one kind (K or V) and their scales."""
    shape = (layers, n_pages, case["nkv"], case["page"], case["hd"])
    codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    if case["token_major"]:
        codes = torch.empty((layers, n_pages, case["page"], case["nkv"], case["hd"]), dtype=torch.float8_e4m3fn, device="cuda").transpose(2, 3)
    scales = torch.empty(shape[:3], device="cuda")
    for i in range(layers):
        x = _values(shape[1:], gen, spread)
        s = torch.exp2(_exponent(x.abs().amax((-1, -2))).float())
        scales[i] = s
        codes[i] = (x / s[..., None, None]).to(torch.float8_e4m3fn)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "pages":
        return _prepare_pages(case, gen)
    dtype, rows, lengths = _DTYPES[case["dtype"]], _rows(case), _lengths(case)
    counts = [_pages_of(n, case["page"]) for n in lengths]
    n_pages = sum(counts) + 2
    kc, ks = _codes(1, n_pages, case, gen, 0.5)
    vc, vs = _codes(1, n_pages, case, gen, 0.5)
    table = _ragged_table(counts, n_pages, gen)
    # what lies behind a sequence's last token is left over from an earlier owner of the page, here as the code for NaN
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    tail = torch.arange(case["page"], device="cuda")[None, :] >= ((lens - 1) % case["page"] + 1)[:, None]
    last = table.gather(1, ((lens.clamp(min=1) - 1) // case["page"]).long()[:, None])[:, 0].long()
    seq, off = tail.nonzero(as_tuple=True)
    kc.view(torch.uint8)[0, last[seq], :, off] = 0x7F
    vc.view(torch.uint8)[0, last[seq], :, off] = 0x7F
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[table[torch.arange(table.shape[1], device="cuda")[None, :] < torch.tensor(counts, device="cuda")[:, None]].long()] = 1
    start = torch.tensor([0] + rows, device="cuda").cumsum(0).to(torch.int32)
    total, nkv, hd = sum(rows), case["nkv"], case["hd"]
    state = {"case": case, "k": kc, "v": vc, "k_scale": ks, "v_scale": vs, "table": table, "lens": lens, "refs": refs, "start": start, "rows": total}
    if case["op"] == "append":
        # two rows behind the last sequence's: a padded batch
        new = torch.stack([_values((nkv, total + 2, hd), gen, 0.5), _values((nkv, total + 2, hd), gen, 0.5)])
        new = new.transpose(1, 2).to(dtype).contiguous()
        return dict(state, k_new=new[0], v_new=new[1], most=max(rows))
    q = torch.randn(total + 2, case["nq"], hd, generator=gen, device="cuda") * 1.5
    gate = torch.randn(total + 2, case["nq"] * hd, generator=gen, device="cuda") if case["gate"] else None
    qpos = torch.tensor(_positions(case) + [0, 0], dtype=torch.int32, device="cuda") if case["scattered"] else None
    y = torch.full((total + 2, case["nq"] * hd), 7.0, dtype=dtype, device="cuda")
    return dict(state, q=q.to(dtype), gate=gate, qpos=qpos, y=y, most=max(rows), longest=max(lengths))


def _prepare_pages(case, gen):
    parents, children = case["parents"], case["children"]
    n_pages, held = _pool(case), _pages_of(case["length"], case["page"])
    kc, ks = _codes(case["layers"], n_pages, case, gen, 0.5)
    vc, vs = _codes(case["layers"], n_pages, case, gen, 0.5)
    n_seqs, most = parents + children, _pages_of(case["length"] + case["grow"], case["page"])
    table = torch.zeros(n_seqs, most, dtype=torch.int32, device="cuda")
    # the parents hold the first pages of the pool, each in an order of its own
    table[:parents, :held] = torch.randperm(parents * held, generator=gen, device="cuda").to(torch.int32).view(parents, held)
    lens = torch.zeros(n_seqs, dtype=torch.int32, device="cuda")
    lens[:parents] = case["length"]
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[:parents * held] = 1
    # the children's rows of the table in an order that the seed makes
    dst = parents + torch.randperm(children, generator=gen, device="cuda").to(torch.int32)
    src = torch.randint(0, parents, (children,), generator=gen, device="cuda").to(torch.int32)
    add = torch.zeros(n_seqs, dtype=torch.int32, device="cuda")
    add[parents:] = case["grow"]
    gone = dst[torch.randperm(children, generator=gen, device="cuda")[:case["free"]]].contiguous()
    live = torch.zeros(1, dtype=torch.int32, device="cuda")
    return {"case": case, "k": kc, "v": vc, "k_scale": ks, "v_scale": vs, "table": table, "lens": lens, "refs": refs, "src": src, "dst": dst, "add": add, "gone": gone, "live": live}


# ---------------------------------------------------------------- the framework's calls

_kernels = {}


def _handles(state):
    """The context's operators and the cache object, which a program makes once and keeps."""
    if "cache" not in state:
        from decide_b200.kernels import Act, Device, Kernels, Kv8Cache

        dtype = state["case"].get("dtype", "f16")
        if dtype not in _kernels:
            _kernels[dtype] = Kernels(Device(0))
            _kernels[dtype].dev.set_activation_dtype(Act.F16 if dtype == "f16" else Act.BF16)
        state["cache"] = Kv8Cache(state["k"], state["v"], state["k_scale"], state["v_scale"], state["table"], state["lens"], state["refs"])
        state["kernels"] = _kernels[dtype]
    return state["kernels"].kv8, state["cache"]


def _run_own(state):
    case = state["case"]
    kv8, cache = _handles(state)
    if case["op"] == "append":
        row = case["nkv"] * case["hd"]
        kv8.append(None, cache, 0, state["k_new"], state["v_new"], row, row, state["start"], state["rows"], state["most"])
    elif case["op"] == "attention":
        row = case["nq"] * case["hd"]
        kv8.attention(None, cache, 0, state["q"], state["gate"], state["start"], state["qpos"], state["y"], state["rows"], row, row, row, case["nq"],
                      state["most"], state["longest"])
    else:
        kv8.fork(None, cache, state["src"], state["dst"], case["children"], case["deep"])
        if case["grow"]:
            kv8.extend(None, cache, state["add"])
        if case["free"]:
            kv8.free(None, cache, state["gone"], case["free"])
        if case["compact"]:
            kv8.compact(None, cache, state["live"])
    return _outputs(state)


def _outputs(state):
    case = state["case"]
    if case["op"] == "append":
        return {"k": state["k"], "v": state["v"], "k_scale": state["k_scale"], "v_scale": state["v_scale"]}
    if case["op"] == "attention":
        return {"y": state["y"]}
    return {"k": state["k"], "v": state["v"], "k_scale": state["k_scale"], "v_scale": state["v_scale"], "table": state["table"], "lens": state["lens"],
            "refs": state["refs"], "live": state["live"]}


# ---------------------------------------------------------------- the plain forms

def _owner(state):
    """For each packed row: its sequence, and how many rows of that sequence come before it."""
    start = state["start"].long()
    row = torch.arange(state["rows"], device="cuda")
    seq = torch.searchsorted(start, row, right=True) - 1
    return seq, row - start[seq], start[1:] - start[:-1]


def _append_one(codes, scales, new, page, offset, first, page_size):
    """`new` [rows, nkv, hd] goes to `offset` of `page` row by row; first [n_pages]: the least offset written now, page_size where none is."""
    n_pages, nkv = scales.shape
    x = new.float()
    size = x.abs()
    finite = torch.isfinite(size)
    where = page[:, None].expand(-1, nkv)
    amax = torch.zeros(n_pages, nkv, device="cuda").scatter_reduce_(0, where, torch.where(finite, size, 0.0).amax(-1), "amax")
    bad = torch.zeros(n_pages, nkv, device="cuda").scatter_reduce_(0, where, (~finite).any(-1).float(), "amax") > 0
    touched, fresh = (first < page_size)[:, None], (first == 0)[:, None]
    fits = torch.exp2(_exponent(amax).float())
    scale = torch.where(fresh, fits, torch.maximum(scales, fits))       # a NaN that the page has stays
    scale = torch.where(bad, torch.full_like(scale, float("nan")), scale)
    grown = touched & ~fresh & (scale > scales)
    at_page, at_head = grown.nonzero(as_tuple=True)
    held = torch.arange(page_size, device="cuda")[None, :, None] < first[at_page][:, None, None]
    old = codes.view(torch.uint8)[at_page, at_head].view(torch.float8_e4m3fn).float()
    again = (old * (scales / scale)[at_page, at_head][:, None, None]).to(torch.float8_e4m3fn)
    codes.view(torch.uint8)[at_page, at_head] = torch.where(held, again.view(torch.uint8), codes.view(torch.uint8)[at_page, at_head])
    s = scale[page][..., None]
    code = torch.where(torch.isnan(s), torch.zeros_like(x), x / s).to(torch.float8_e4m3fn)
    codes.view(torch.uint8)[page, :, offset] = code.view(torch.uint8)
    scales.copy_(torch.where(touched, scale, scales))


def _run_append(state):
    case = state["case"]
    seq, index, count = _owner(state)
    position = state["lens"].long()[seq] - count[seq] + index
    page = state["table"].long()[seq, position // case["page"]]
    offset = position % case["page"]
    first = torch.full((state["refs"].shape[0],), case["page"], dtype=torch.long, device="cuda").scatter_reduce_(0, page, offset, "amin")
    _append_one(state["k"][0], state["k_scale"][0], state["k_new"][:state["rows"]], page, offset, first, case["page"])
    _append_one(state["v"][0], state["v_scale"][0], state["v_new"][:state["rows"]], page, offset, first, case["page"])


def _gathered(codes, scales, table, held, page_size):
    """The tokens of every sequence, [seq, head, token, dim] in fp32, zero where the sequence has none."""
    token = torch.arange(held.shape[1], device="cuda")
    page, offset = table.long()[:, token // page_size], (token % page_size)[None, :].expand(table.shape[0], -1)
    x = codes.view(torch.uint8)[page, :, offset].view(torch.float8_e4m3fn).float() * scales[page][..., None]
    return torch.where(held[:, :, None, None], x, 0.0).transpose(1, 2)


def _run_attention(state):
    case = state["case"]
    nkv, hd, group, n, total = case["nkv"], case["hd"], case["nq"] // case["nkv"], case["seqs"], state["rows"]
    seq, index, count = _owner(state)
    lens = state["lens"].long()
    position = lens[seq] - count[seq] + index if state["qpos"] is None else state["qpos"][:total].long()
    token = torch.arange(state["longest"], device="cuda")
    held = token[None, :] < lens[:, None]
    k = _gathered(state["k"][0], state["k_scale"][0], state["table"], held, case["page"])
    v = _gathered(state["v"][0], state["v_scale"][0], state["table"], held, case["page"])
    most = state["most"]
    q = torch.zeros(n, most, nkv, group, hd, device="cuda")
    q[seq, index] = state["q"][:total].float().view(total, nkv, group, hd)
    sees = torch.full((n, most), NO_KEYS, dtype=torch.long, device="cuda")
    sees[seq, index] = torch.minimum(position, lens[seq] - 1)
    score = q.permute(0, 2, 1, 3, 4).reshape(n, nkv, most * group, hd) @ k.transpose(2, 3)
    score = score.view(n, nkv, most, group, -1) * hd ** -0.5
    score.masked_fill_((token > sees[:, :, None])[:, None, :, None, :], float("-inf"))
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    whole = score.sum(-1, keepdim=True)
    out = score.view(n, nkv, most * group, -1) @ v
    out = torch.where(whole == 0, 0.0, out.view(n, nkv, most, group, hd) / whole)
    out = out.permute(0, 2, 1, 3, 4)[seq, index].reshape(total, -1)
    if state["gate"] is not None:
        out = out / (1 + torch.exp(-state["gate"][:total]))
    state["y"][:total] = out.to(state["y"].dtype)


def _release(state, seqs):
    table, lens, refs = state["table"], state["lens"], state["refs"]
    held = torch.arange(table.shape[1], device="cuda")[None, :] < (-(-lens[seqs] // state["case"]["page"]))[:, None]
    refs -= torch.bincount(table[seqs][held], minlength=refs.shape[0]).to(torch.int32)
    lens[seqs] = 0


def _copy_pages(state, src, dst):
    state["k"].view(torch.uint8)[:, dst] = state["k"].view(torch.uint8)[:, src]
    state["v"].view(torch.uint8)[:, dst] = state["v"].view(torch.uint8)[:, src]
    state["k_scale"][:, dst] = state["k_scale"][:, src]
    state["v_scale"][:, dst] = state["v_scale"][:, src]


def _lowest_free(refs, count):
    return (refs == 0).nonzero()[:count, 0]


def _run_fork(state):
    case, table, lens, refs = state["case"], state["table"], state["lens"], state["refs"]
    src, dst, page = state["src"].long(), state["dst"].long(), state["case"]["page"]
    _release(state, dst)
    column = torch.arange(table.shape[1], device="cuda")[None, :]
    held, full = (-(-lens[src] // page))[:, None], (lens[src] // page)[:, None]
    shared = column < (full * (0 if case["deep"] else 1))
    refs += torch.bincount(table[src][shared], minlength=refs.shape[0]).to(torch.int32)
    copied = (column < held) & ~shared
    at_seq, at_column = copied.nonzero(as_tuple=True)
    new = _lowest_free(refs, at_seq.shape[0])
    old = table[src[at_seq], at_column].long()
    rows = torch.where(column < held, table[src], table[dst])
    rows[at_seq, at_column] = new.to(torch.int32)
    table[dst] = rows
    refs[new] = 1
    lens[dst] = lens[src]
    _copy_pages(state, old, new)


def _run_extend(state):
    table, lens, refs, page = state["table"], state["lens"], state["refs"], state["case"]["page"]
    column = torch.arange(table.shape[1], device="cuda")[None, :]
    before, after = -(-lens // page), -(-(lens + state["add"]) // page)
    at_seq, at_column = ((column >= before[:, None]) & (column < after[:, None])).nonzero(as_tuple=True)
    new = _lowest_free(refs, at_seq.shape[0])
    table[at_seq, at_column] = new.to(torch.int32)
    refs[new] = 1
    lens += state["add"]


def _run_compact(state):
    table, lens, refs, page = state["table"], state["lens"], state["refs"], state["case"]["page"]
    held = refs > 0
    live = held.sum()
    index = torch.arange(refs.shape[0], device="cuda")
    src, dst = (held & (index >= live)).nonzero()[:, 0], (~held & (index < live)).nonzero()[:, 0]
    _copy_pages(state, src, dst)
    moved = index.clone()
    moved[src] = dst
    refs[dst] = refs[src]
    refs[src] = 0
    column = torch.arange(table.shape[1], device="cuda")[None, :]
    table.copy_(torch.where(column < (-(-lens // page))[:, None], moved[table.long()].to(torch.int32), table))
    state["live"].copy_(live)


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "append":
        _run_append(state)
    elif case["op"] == "attention":
        _run_attention(state)
    else:
        _run_fork(state)
        if case["grow"]:
            _run_extend(state)
        if case["free"]:
            _release(state, state["gone"].long())
        if case["compact"]:
            _run_compact(state)
    return _outputs(state)


# ---------------------------------------------------------------- from the definition, in 64 bits

def _to_e4m3(x):
    """The nearest value that e4m3 has, ties to the even code, of x with |x| <= 448: in float64."""
    size = x.abs()
    # 3 bits behind the leading one; below 2^-6 the steps stay at 2^-9
    step = torch.exp2(torch.floor(torch.log2(size.clamp(min=2.0 ** -6))) - 3)
    return torch.copysign(torch.round(size / step) * step, x)


def exact(case, seed):
    if case["op"] == "pages":
        return None         # pages are moved and counted: nothing is computed
    state = prepare(case, seed)
    table, page = state["table"].tolist(), case["page"]
    starts, lengths, nkv, hd = state["start"].tolist(), state["lens"].tolist(), case["nkv"], case["hd"]
    if case["op"] == "append":
        out = {}
        for name in ("k", "v"):
            codes, scales = state[name][0].double(), state[name + "_scale"][0].double()
            new = state[name + "_new"].double()
            for j, length in enumerate(lengths):
                begin = length - (starts[j + 1] - starts[j])
                for b in range(begin // page, _pages_of(length, page) if begin < length else 0):
                    lo, hi = max(begin, b * page), min(length, (b + 1) * page)
                    x = new[starts[j] + lo - begin:starts[j] + hi - begin].transpose(0, 1)      # [head, token, dim]
                    need = torch.ceil(torch.log2(x.abs().amax((1, 2)) / 448)).clamp(min=SCALE_EXP_MIN)
                    p, o = table[j][b], lo - b * page
                    scale = torch.exp2(need) if o == 0 else torch.maximum(torch.exp2(need), scales[p])
                    codes[p, :, :o] = _to_e4m3(codes[p, :, :o] * (scales[p] / scale)[:, None, None])
                    codes[p, :, o:o + hi - lo] = _to_e4m3(x / scale[:, None, None])
                    scales[p] = scale
            out[name], out[name + "_scale"] = codes[None], scales[None]
        return out
    out, row = state["y"].double(), 0
    for j, length in enumerate(lengths):
        pages = torch.tensor(table[j][:_pages_of(length, page)], device="cuda")
        m = starts[j + 1] - starts[j]
        if not m:
            continue
        at = list(range(length - m, length)) if state["qpos"] is None else state["qpos"][row:row + m].tolist()
        hidden = torch.arange(length, device="cuda")[None, :] > torch.tensor(at, device="cuda")[:, None]
        for h in range(nkv):
            k, v = ((state[n].view(torch.uint8)[0][:, h][pages].view(torch.float8_e4m3fn).double() * state[n + "_scale"][0][:, h][pages].double()[:, None, None]).reshape(-1, hd)[:length] for n in ("k", "v"))
            group = case["nq"] // nkv
            for g in range(h * group, (h + 1) * group):
                s = (state["q"][row:row + m, g].double() @ k.T * hd ** -0.5).masked_fill(hidden, float("-inf"))
                w = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)     # a row that sees nothing is zero
                o = w @ v
                if state["gate"] is not None:
                    o = o * torch.sigmoid(state["gate"][row:row + m, g * hd:(g + 1) * hd].double())
                out[row:row + m, g * hd:(g + 1) * hd] = o
        row += m
    return {"y": out}
