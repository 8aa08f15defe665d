"""The paged 8-bit K/V cache without a GPU: the numpy model's own behaviour (codes, scales, pages, refusals) and the refusals that the
library and the Python binding make before anything runs."""
import ctypes
import math

import numpy as np
import pytest
import torch

from decide_b200 import _lib
from decide_b200.kernels import KernelError, Kv8Cache, _Kv8Struct
from oracle import kv8


def test_codes_are_e4m3():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(t, kv8.DECODE, equal_nan=True)
    x = np.concatenate([np.random.RandomState(0).randn(20000) * s for s in (1e-3, 0.02, 1, 60)] + [np.linspace(-448, 448, 200001)])
    x = np.clip(x.astype(np.float32), -448, 448)
    assert np.array_equal(kv8.encode(x.astype(np.float64)), torch.tensor(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


@pytest.mark.parametrize("amax,scale", [(0.0, 2.0 ** -60), (448.0, 1.0), (448.5, 2.0), (224.0, 0.5), (1e-30, 2.0 ** -60), (65504.0, 256.0), (447.0, 1.0)])
def test_scale_is_the_least_power_of_two(amax, scale):
    assert kv8.scale_for(amax) == scale


def test_model_pages():
    c = kv8.Cache(1, 8, 1, 128, 4, 4, 16)
    c.extend([20, 0, 0, 0])
    assert c.table[0, :2].tolist() == [0, 1] and c.refs.tolist() == [1, 1, 0, 0, 0, 0, 0, 0]
    c.fork([0, 0], [1, 2], False)
    assert c.table[1, :2].tolist() == [0, 2] and c.table[2, :2].tolist() == [0, 3] and c.refs[:4].tolist() == [3, 1, 1, 1]
    c.free([0, 1])
    assert c.refs[:4].tolist() == [1, 0, 0, 1] and c.compact() == 2 and c.table[2, :2].tolist() == [0, 1]
    with pytest.raises(kv8.Violation):
        c.extend([0, 0, 200, 0])
    with pytest.raises(kv8.Violation):
        c.fork([2], [2], False)
    with pytest.raises(kv8.Violation):
        c.fork([2, 2], [0, 0], False)
    c.table[2, 1] = 8
    with pytest.raises(kv8.Violation):
        c.free([2])


def test_model_scale_rises_and_codes_round_again():
    c = kv8.Cache(1, 2, 1, 128, 1, 2, 16)
    c.extend([1])
    c.append(0, np.full((1, 1, 128), 17.0), np.full((1, 1, 128), 1.0), [0, 1])
    # 17 / 2^-4 = 272 lies half way between 256 = 1.000b * 2^8 and 288 = 1.001b * 2^8: the even code is that of 256
    assert c.k_scale[0, 0, 0] == 2.0 ** -4 and kv8.DECODE[c.k[0, 0, 0, 0, 0]] == 256
    c.extend([1])
    c.append(0, np.full((1, 1, 128), 1e4), np.full((1, 1, 128), math.inf), [0, 1])
    assert c.k_scale[0, 0, 0] == 32.0 and kv8.DECODE[c.k[0, 0, 0, 0, 0]] == 0.5
    assert math.isnan(c.v_scale[0, 0, 0]) and c.v[0, 0, 0, 1].max() == 0


def _struct(**changes):
    fields = dict(k=1 << 20, v=1 << 21, k_scale=1 << 22, v_scale=1 << 23, table=1 << 24, lens=1 << 25, refs=1 << 26, layer_stride=4 * 8 * 16 * 128,
                  page_stride=8 * 16 * 128, head_stride=16 * 128, token_stride=128, layers=2, n_pages=4, nkv=8, page_size=16, hd=128, n_seqs=3, max_pages=4, reserved=0)
    return _Kv8Struct(**{**fields, **changes})


@pytest.mark.parametrize("changes,code,word", [
    ({}, 0, ""), ({"k": 0}, 1, "null"), ({"refs": 0}, 1, "null"), ({"v": (1 << 21) + 8}, 1, "aligned"), ({"lens": (1 << 25) + 2}, 1, "aligned"),
    ({"hd": 64}, 3, "hd"), ({"page_size": 48}, 3, "page_size"), ({"page_size": 256}, 3, "page_size"), ({"nkv": 0}, 1, "at least 1"), ({"n_seqs": 0}, 1, "at least 1"),
    ({"max_pages": 0}, 1, "at least 1"), ({"n_seqs": 65536}, 3, "65535"), ({"n_pages": 0x200001, "layers": 1}, 3, "2^21"),
    ({"max_pages": 1 << 27}, 3, "2^31"), ({"reserved": 1}, 1, "reserved"), ({"token_stride": 136}, 1, "multiples"), ({"token_stride": 64}, 1, "overlap"),
    ({"token_stride": 1 << 28, "layers": 1, "n_pages": 1, "nkv": 1}, 3, "2^28"),
    ({"page_stride": 7 * 16 * 128}, 1, "overlap"), ({"head_stride": 0}, 1, "overlap"), ({"layer_stride": 1 << 47, "layers": 65535}, 1, "2^48"),
    # the same bytes with a token's heads side by side, and a view with holes
    ({"head_stride": 128, "token_stride": 8 * 128}, 0, ""), ({"token_stride": 256, "head_stride": 32 * 128, "page_stride": 1 << 20, "layer_stride": 1 << 30}, 0, ""),
    # a stride that nothing steps along says nothing
    ({"layers": 1, "layer_stride": 3}, 0, ""),
])
def test_descriptions_are_checked_without_a_gpu(changes, code, word):
    lib = _lib.load()
    err = ctypes.create_string_buffer(160)
    s = _struct(**changes)
    assert lib.dc_kv8_check(ctypes.addressof(s), err, len(err)) == code
    assert word in err.value.decode() and (code == 0) == (err.value == b"")
    assert lib.dc_kv8_check(ctypes.addressof(s), None, 0) == code


def test_null_cache_and_null_context():
    lib = _lib.load()
    s = _struct()
    ref = ctypes.addressof(s)
    assert lib.dc_kv8_check(None, None, 0) == 1
    assert lib.dc_kv8_extend(None, None, ref, None) == 1
    assert lib.dc_kv8_fork(None, None, ref, None, None, 1, 0) == 1
    assert lib.dc_kv8_free(None, None, ref, None, 1) == 1
    assert lib.dc_kv8_compact(None, None, ref, None) == 1
    assert lib.dc_kv8_append(None, None, ref, 0, None, None, 0, 0, None, 0, 0) == 1
    assert lib.dc_kv8_attention(None, None, ref, 0, None, None, None, None, None, 0, 0, 0, 0, 0, 0, 0) == 1
    assert lib.dc_kv8_attention_scratch_bytes(None, ref, 8, 1, 0) == 0
    assert lib.dc_kv8_pages_scratch_bytes(None) == 0 and lib.dc_kv8_pages_scratch_bytes(ref) > 0


def test_the_binding_checks_its_tensors():
    good = Kv8Cache.empty(2, 4, 2, 128, 3, 4, 16, device="cpu")
    assert (good.layers, good.n_pages, good.nkv, good.page_size, good.hd, good.n_seqs, good.max_pages) == (2, 4, 2, 16, 128, 3, 4)
    parts = dict(k=good.k, v=good.v, k_scale=good.k_scale, v_scale=good.v_scale, table=good.table, lens=good.lens, refs=good.refs)
    wide = torch.zeros(2, 4, 16, 2, 128, dtype=torch.uint8).transpose(2, 3)     # a token's heads side by side
    other = Kv8Cache(**{**parts, "k": wide, "v": wide.clone(memory_format=torch.preserve_format)})
    assert (other.struct.head_stride, other.struct.token_stride) == (128, 256)
    for bad in ({"k": good.k.view(torch.uint8).to(torch.int32)}, {"v": good.v[:, :3]}, {"k": wide}, {"k_scale": good.k_scale.double()}, {"k_scale": good.k_scale[:1]},
                {"lens": good.lens[:2]}, {"refs": good.refs.long()}, {"table": good.table[0]}, {"table": good.table.t().contiguous().t()}):
        with pytest.raises((KernelError, IndexError)):
            Kv8Cache(**{**parts, **bad})
    with pytest.raises(KernelError):
        Kv8Cache.empty(1, 4, 2, 64, 3, 4, 16, device="cpu")
