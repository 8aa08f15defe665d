"""The context's scratch workspace under captured graphs: a graph replays into the block it was captured with, so that block stays allocated whatever
later calls of the context ask for. What the driver has free says whether it did before any replay runs."""
import numpy as np
import pytest
import torch

from decide_b200.kernels import Device, KernelError, Kernels, Kv8Cache
from decide_b200.synth import synth_batch, synth_state_dict
from tests.test_model_gpu import SMALL

pytestmark = pytest.mark.gpu

PAGE, NQ, NKV, HD, MAX_LEN = 16, 32, 8, 128, 4096


class Follow:
    """A cache and a call of its attention whose key chunks need some 20 MB of scratch: 64 rows over 4,000 keys."""

    def __init__(self, k):
        self.k, pages = k, MAX_LEN // PAGE
        self.cache = Kv8Cache.empty(1, pages, NKV, HD, 1, pages, PAGE)
        k.kv8.extend(None, self.cache, torch.tensor([4000], dtype=torch.int32, device="cuda"))
        gen = torch.Generator().manual_seed(1)
        rows = torch.randn(2, 4000, NKV * HD, generator=gen).to(k.dev.act_torch).cuda()
        k.kv8.append(None, self.cache, 0, rows[0], rows[1], NKV * HD, NKV * HD, torch.tensor([0, 4000], dtype=torch.int32, device="cuda"), 4000, 4000)
        self.q = torch.randn(64, NQ * HD, generator=gen).to(k.dev.act_torch).cuda()
        self.start = torch.tensor([0, 64], dtype=torch.int32, device="cuda")
        self.y = torch.empty(64, NQ * HD, dtype=k.dev.act_torch, device="cuda")
        self.need = k.kv8.attention_scratch_bytes(self.cache, NQ, 64, MAX_LEN)

    def attend(self, k=None):
        k = k or self.k
        k.kv8.attention(None, self.cache, 0, self.q, None, self.start, None, self.y, 64, NQ * HD, 0, NQ * HD, NQ, 64, MAX_LEN)


def grows_beside(dev, call, need):
    """`call` makes the workspace grow to `need` bytes and the old block stays allocated. Returns blocks that the old one's memory would have gone to."""
    old = dev.workspace_bytes
    assert old >= 4 << 20 and need > old, "the sizes tell a block that stays from one that goes"
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    call()
    torch.cuda.synchronize()
    assert dev.workspace_bytes == need
    assert before - torch.cuda.mem_get_info()[0] > need - old // 2, "the old workspace was freed under a graph that replays into it"
    return [torch.full((old // 4,), float("nan"), device="cuda") for _ in range(4)]


def test_a_models_graph_keeps_its_workspace(k):
    """An engine whose forward replays from a graph, on a context that then serves a larger attention over the 8-bit cache: the graph's scratch stays
    its own, and the engine's answers the same."""
    from decide_b200.engine import Engine
    first = Follow(k)
    first.attend()                                  # kernels are loaded (which takes device memory) before anything is measured
    want = first.y.clone()
    dev = Device(0)
    eng = Engine(SMALL, synth_state_dict(SMALL, 5), dev=dev, max_rows=256, max_seqs=1, max_answers=4, max_cand=8)
    batch = synth_batch(SMALL, 1, 150, seed=6, n_answers=2, n_cand=8, max_cand=8)
    logits = eng.logits(batch)
    assert np.array_equal(eng.logits(batch), logits) and eng.graph_count == 1
    own = Kernels(dev)
    fillers = grows_beside(dev, lambda: first.attend(own), first.need)
    assert torch.equal(first.y, want)
    for _ in range(3):
        assert np.array_equal(eng.logits(batch), logits)
        first.attend(own)
        torch.cuda.synchronize()
        assert torch.equal(first.y, want)
    assert all(torch.isnan(f).all() for f in fillers), "the graph wrote memory that is not its own"
    dev.check_status()
    eng.close()
    dev.close()


def test_graphs_of_every_kind_of_call_keep_their_workspace(k):
    """Packed attention, captured; then a page operation, captured; each time the workspace grows afterwards. A capture that would have to allocate is
    refused and the capture goes on."""
    follow = Follow(k)
    follow.attend()
    want_follow = follow.y.clone()
    dev = Device(0)
    own = Kernels(dev)
    n, nq, nkv = 20000, 4, 2
    gen = torch.Generator().manual_seed(3)
    q, kc, vc = (torch.randn(n, w * 128, generator=gen).to(dev.act_torch).cuda() for w in (nq, nkv, nkv))
    y, z = (torch.zeros(n, nq * 128, dtype=dev.act_torch, device="cuda") for _ in range(2))
    start = torch.tensor([0, n // 2, n], dtype=torch.int32, device="cuda")
    pos = torch.cat([torch.arange(n // 2), torch.arange(n - n // 2)]).to(torch.int32).cuda()

    def packed(out):
        own.attn.attention(None, q, kc, vc, None, pos, out, n, 0, nq, nkv, 128, start, 2, n // 2)

    k.attn.attention(None, q, kc, vc, None, pos, z, n, 0, nq, nkv, 128, start, 2, n // 2)     # loaded, on the other context
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q.mul_(1)
        with pytest.raises(KernelError, match="during a capture"):
            packed(y)
    packed(z)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        packed(y)
    fillers = grows_beside(dev, lambda: follow.attend(own), follow.need)

    src, dst = (torch.tensor([i], dtype=torch.int32, device="cuda") for i in (0, 1))
    small = Kv8Cache.empty(1, 8, 1, 128, 2, 4, 16)
    own.kv8.extend(None, small, torch.tensor([20, 0], dtype=torch.int32, device="cuda"))
    pages = torch.cuda.CUDAGraph()
    with torch.cuda.graph(pages):
        own.kv8.fork(None, small, src, dst, 1)
    fillers += grows_beside(dev, lambda: dev.reserve_workspace(64 << 20), 64 << 20)
    for i in range(3):
        y.zero_()
        graph.replay()
        pages.replay()
        follow.y.zero_()
        follow.attend(own)
        torch.cuda.synchronize()
        assert torch.equal(y, z) and torch.equal(follow.y, want_follow)
        assert small.lens.tolist() == [20, 20] and small.refs.tolist() == [2, 1, 1, 0, 0, 0, 0, 0]
    assert all(torch.isnan(f).all() for f in fillers), "a graph wrote memory that is not its own"
    dev.check_status()
    del graph, pages
    dev.close()


def test_growing_under_graphs_has_no_limit(k):
    """Forty captures, each followed by a larger demand."""
    dev = Device(0)
    own = Kernels(dev)
    small = Kv8Cache.empty(1, 8, 1, 128, 2, 4, 16)
    add = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    graphs = []
    dev.reserve_workspace(4096)
    for i in range(40):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            own.kv8.extend(None, small, add)
        dev.reserve_workspace(dev.workspace_bytes + 4096)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert small.lens.tolist() == [40, 0] and small.refs.tolist() == [1, 1, 1, 0, 0, 0, 0, 0]
    dev.check_status()
    del graphs
    dev.close()
