"""Refusals of the 8-bit KV cache and shared-prefix entry points, before anything is launched."""
import ctypes as C

import numpy as np
import pytest
import torch

import kv8_ref as R
from kvasir_b200 import _lib as L

F = C.c_void_p(0x1000)  # never dereferenced: the checks fail first


def _refused(st, *words):
    msg = L.lib().kvb_last_error().decode()
    assert st == L.KVB_ERR_SHAPE, (st, msg)
    assert all(w in msg for w in words), msg


def _append(**k):
    a = dict(qkv=F, qkv_len=2 * 3 * 12 * 64, n_seq=2, t=3, pos=F, cos=F, sin=F, table=16 * 32, kc=F,
             vc=F, ks=F, vs=F, stride=2 * 16 * 64, cache=2 * 2 * 16 * 64, scales=2 * 2 * 16, n_q=8,
             n_kv=2, hd=64, max_seq=16, fmt=0, dtype=0)
    a.update(k)
    return L.lib().kvb_rope_kv_append_q8(None, *a.values())


def test_append_refusals():
    _refused(_append(fmt=2), "KV format")
    _refused(_append(dtype=5), "dtype")
    _refused(_append(hd=63), "")
    _refused(_append(hd=0), "head_dim")
    _refused(_append(hd=258), "head_dim")
    _refused(_append(n_kv=0), "n_kv")
    _refused(_append(qkv_len=100), "qkv has")
    _refused(_append(stride=2 * 16 * 64 - 64), "seq_stride")
    _refused(_append(stride=2 * 16 * 64 + 32), "seq_stride")
    _refused(_append(cache=2 * 2 * 16 * 64 - 64, scales=2 * 2 * 16 - 1), "too small")
    _refused(_append(scales=63), "scales")
    _refused(_append(table=16 * 32 + 1), "table")
    _refused(_append(sin=None), "cos / sin")
    _refused(_append(pos=None), "null")
    _refused(_append(kc=None), "null")
    _refused(_append(max_seq=1 << 31, stride=1 << 40, cache=1 << 41, scales=1 << 35), "i32")
    # a cache so large that its size would wrap
    _refused(_append(n_seq=3, qkv_len=3 * 3 * 12 * 64, stride=1 << 62, cache=1 << 40, scales=1 << 34),
             "too small")
    assert _append(n_seq=0, qkv_len=0) == 0  # nothing to do
    assert _append(t=0, qkv_len=0) == 0


def test_paged_append_refusals():
    def call(**k):
        a = dict(qkv=F, qkv_len=2 * 12 * 64, n_seq=2, t=1, pos=F, cos=F, sin=F, table=16 * 32, kc=F,
                 vc=F, ks=F, vs=F, pool=5 * 2 * 16 * 64, scales=5 * 2 * 16, bt=F, mb=3, bs=16, n_q=8,
                 n_kv=2, hd=64, fmt=1, dtype=1)
        a.update(k)
        return L.lib().kvb_rope_kv_append_q8_paged(None, *a.values())
    _refused(call(pool=5 * 2 * 16 * 64 + 64), "whole number")
    _refused(call(scales=5), "scales")
    _refused(call(bs=0), "block_size")
    _refused(call(bt=None), "block table")
    _refused(call(mb=1 << 30), "i32")
    _refused(call(fmt=-1), "KV format")


def test_read_refusals():
    def call(**k):
        a = dict(kc=F, vc=F, ks=F, vs=F, stride=2 * 16 * 64, cache=2 * 2 * 16 * 64, scales=64, pos=F,
                 n_seq=2, t=3, n_kv=2, hd=64, max_seq=16, ko=F, vo=F, out_len=2 * 2 * 4 * 64, rows=4,
                 fmt=0, dtype=0)
        a.update(k)
        return L.lib().kvb_kv_read_q8(None, *a.values())
    _refused(call(t=5), "rows into")
    _refused(call(out_len=10), "outputs of")
    _refused(call(ko=None), "null")
    _refused(call(scales=63), "scales")
    assert call(t=0) == 0


def test_decode_refusals():
    def call(**k):
        a = dict(q=F, qs=8 * 64, kc=F, vc=F, ks=F, vs=F, stride=2 * 16 * 64, cache=2 * 2 * 16 * 64,
                 scales=64, lens=F, n_seq=2, max_len=16, n_q=8, n_kv=2, hd=64, max_seq=16, scale=0.125,
                 out=F, os=8 * 64, ws=None, wl=0, fmt=0, dtype=0)
        a.update(k)
        return L.lib().kvb_attention_decode_q8(None, *a.values())
    _refused(call(max_len=17), "max_len")
    _refused(call(n_q=7), "multiple")
    _refused(call(n_q=0), "multiple")
    _refused(call(hd=257), "head_dim")
    _refused(call(qs=511), "q_row_stride")
    _refused(call(os=511), "out_row_stride")
    _refused(call(lens=None), "null")
    _refused(call(scales=65), "scales")
    _refused(call(fmt=7), "KV format")
    assert call(n_seq=0) == 0

    def paged(**k):
        a = dict(q=F, qs=8 * 64, kc=F, vc=F, ks=F, vs=F, pool=5 * 2 * 16 * 64, scales=5 * 32, bt=F, mb=3,
                 bs=16, lens=F, n_seq=2, max_len=48, n_q=8, n_kv=2, hd=64, scale=0.125, out=F, os=8 * 64,
                 ws=None, wl=0, fmt=0, dtype=0)
        a.update(k)
        return L.lib().kvb_attention_decode_q8_paged(None, *a.values())
    _refused(paged(max_len=49), "exceeds")
    _refused(paged(pool=7), "whole number")
    _refused(paged(bt=None), "block table")


def test_shared_refusals():
    def call(**k):
        a = dict(q=F, qs=8 * 64, pk=F, pv=F, prefix=10, rows=12, kc=F, vc=F, stride=2 * 16 * 64,
                 cache=2 * 2 * 16 * 64, lens=F, n_seq=2, max_len=16, n_q=8, n_kv=2, hd=64, max_seq=16,
                 scale=0.125, out=F, os=8 * 64, ws=None, wl=0, dtype=0)
        a.update(k)
        return L.lib().kvb_attention_decode_shared(None, *a.values())
    _refused(call(prefix=13), "prefix")
    _refused(call(max_len=17), "max_len")
    _refused(call(pk=None), "null")
    _refused(call(stride=2 * 16 * 64 + 8), "seq_stride")
    _refused(call(cache=64), "too small")
    _refused(call(n_kv=3), "multiple")
    assert call(n_seq=0) == 0

    def paged(**k):
        a = dict(q=F, qs=8 * 64, kc=F, vc=F, pool=5 * 2 * 16 * 64, bt=F, mb=3, bs=16, shared=20, lens=F,
                 n_seq=2, max_len=48, n_q=8, n_kv=2, hd=64, scale=0.125, out=F, os=8 * 64, ws=None, wl=0,
                 dtype=0)
        a.update(k)
        return L.lib().kvb_attention_decode_shared_paged(None, *a.values())
    _refused(paged(shared=49), "shared_len")
    _refused(paged(max_len=49), "exceeds")
    _refused(paged(pool=7), "whole number")
    _refused(paged(bt=None), "block table")


def test_decoder_refusals():
    lib = L.lib()
    _refused(lib.kvb_decoder_use_q8_cache(None, F, F, F, F, 0), "null")
    _refused(lib.kvb_decoder_use_q8_paged_cache(None, F, F, F, F, 64, F, 1, 16, 0), "null")


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_reference_quantisation_is_within_half_a_step(fmt):
    """The tests' own reference: within half a step of the row, exact at the row's maximum."""
    rng = np.random.default_rng(0)
    x = (rng.normal(0, 1, (200, 64)) * 2.0 ** rng.integers(-30, 30, (200, 1))).astype(np.float32)
    codes, scale = R.quantise(x, fmt)
    v = R.values(codes, fmt)
    step = 0.5 if fmt == "int8" else np.maximum(np.abs(v) * 2.0 ** -4 * 1.07, 2.0 ** -10)
    assert np.all(np.abs(v - x / scale[:, None].astype(np.float64)) <= step + 1e-4)
    assert np.all(np.abs(v).max(-1) == R.TOP[fmt])


def test_buffers_on_the_cpu_are_refused():
    from kvasir_b200.gpu import ShapeError, kv_format
    assert kv_format(torch.zeros(1, dtype=torch.int8)) == L.KVB_KV_INT8
    assert kv_format(torch.zeros(1, dtype=torch.float8_e4m3fn)) == L.KVB_KV_E4M3
    with pytest.raises(ShapeError):
        kv_format(torch.zeros(1, dtype=torch.uint8))
