"""The 8-bit KV cache: append (codes and scales bit-exact against the definition in numpy),
read back, and decode attention over it against f64."""
import numpy as np
import pytest
import torch

import kv8_ref as R
from gpu_util import dev, host_bits, normal16
from oracle import oracle as O

pytestmark = pytest.mark.gpu

# One weight of the softmax is rounded to f16 in the tensor-core kernel: half a step, 2^-11.
W_EPS = 2.0 ** -11


@pytest.fixture(scope="module")
def g():
    from kvasir_b200 import Gpu
    return Gpu(0)


def _tables(hd, rows):
    cos, sin = O.cos_sin_table(hd, rows, **O.LLAMA3_ROPE)
    return cos, sin


def _rotated(bits, cos, sin, pos, t, n_q, n_kv, hd, dtype):
    """qkv bits [n_seq, t, heads, hd] after RoPE: f32 multiplies and adds, one rounding."""
    x = O.to_f32(bits.ravel(), dtype).astype(np.float32).reshape(bits.shape).copy()
    half = hd // 2
    for b in range(bits.shape[0]):
        c = cos.reshape(-1, half)[pos[b]:pos[b] + t][:, None]
        s = sin.reshape(-1, half)[pos[b]:pos[b] + t][:, None]
        lo, hi = x[b, :, :n_q + n_kv, :half].copy(), x[b, :, :n_q + n_kv, half:].copy()
        x[b, :, :n_q + n_kv, :half] = lo * c - hi * s
        x[b, :, :n_q + n_kv, half:] = hi * c + lo * s
    out = O.from_f32(x.ravel(), dtype).reshape(bits.shape)
    out[:, :, n_q + n_kv:] = bits[:, :, n_q + n_kv:]
    return out


SHAPES = [  # n_seq, t, n_q, n_kv, hd
    (1, 1, 32, 8, 64), (32, 1, 32, 8, 64), (3, 517, 32, 8, 64), (2, 5, 6, 2, 128),
    (2, 700, 4, 4, 128), (3, 4, 2, 1, 80), (2, 3, 3, 3, 256), (2, 3, 0, 2, 6), (1, 2, 16, 1, 2),
    (2, 3, 64, 8, 128), (1, 5, 32, 33, 64),  # more chunks in a row than a CTA has threads
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("fmt,dtype", [("int8", "bf16"), ("e4m3", "bf16"), ("int8", "f16"),
                                       ("e4m3", "f16")])
@pytest.mark.parametrize("block", [0, 16, 24])
def test_append_and_read_are_exact(g, shape, fmt, dtype, block):
    n_seq, t, n_q, n_kv, hd = shape
    rng = np.random.default_rng(n_seq * 1000 + t * 10 + hd)
    heads = n_q + 2 * n_kv
    max_seq = t + 40
    pos = rng.integers(0, 40, n_seq).astype(np.int32)
    bits = normal16(rng, n_seq * t * heads * hd, dtype=dtype).reshape(n_seq, t, heads, hd)
    cos, sin = _tables(hd, max_seq)
    want = _rotated(bits, cos, sin, pos, t, n_q, n_kv, hd, dtype)
    rows = O.to_f32(want.ravel(), dtype).astype(np.float32).reshape(want.shape)
    qkv = dev(bits.ravel(), dtype)
    gap = 0 if block else 3  # rows between the sequences' caches
    seq_rows = n_kv * max_seq + gap
    # contiguous reference of both caches, sentinels where nothing is written
    kc = np.full((n_seq, seq_rows, hd), 0x55, np.int8)
    vc, ks, vs = kc.copy(), np.full((n_seq, seq_rows), 7.5, np.float32), None
    vs = ks.copy()
    wk, wv, wks, wvs = kc.copy(), vc.copy(), ks.copy(), vs.copy()
    for b in range(n_seq):
        for h in range(n_kv):
            at = slice(h * max_seq + pos[b], h * max_seq + pos[b] + t)
            wk[b, at], wks[b, at] = R.quantise(rows[b, :, n_q + h], fmt)
            wv[b, at], wvs[b, at] = R.quantise(rows[b, :, n_q + n_kv + h], fmt)
    dpos = torch.from_numpy(pos).cuda()
    dcos, dsin = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    tdt = R.TDT[dtype]
    ko = torch.full((n_seq, n_kv, t + 2, hd), 3.0, dtype=tdt, device="cuda")
    vo = ko.clone()
    if not block:
        ckc, cvc = R.to_dev(kc, fmt), R.to_dev(vc, fmt)
        cks, cvs = torch.from_numpy(ks).cuda(), torch.from_numpy(vs).cuda()
        g.rope_kv_append_q8(qkv, n_seq, t, dpos, dcos, dsin, ckc, cvc, cks, cvs, seq_rows * hd, n_q,
                            n_kv, hd, max_seq)
        g.kv_read_q8(ckc, cvc, cks, cvs, seq_rows * hd, dpos, n_seq, t, n_kv, hd, max_seq, ko, vo,
                     t + 2)
        got = [x.view(torch.int8).cpu().numpy() for x in (ckc, cvc)]
        gots = [x.cpu().numpy() for x in (cks, cvs)]
        wants, wantss = [wk, wv], [wks, wvs]
    else:
        shp = (n_seq, n_kv, max_seq)
        table = None
        pools = []
        for x in (kc, vc, ks, vs, wk, wv, wks, wvs):
            pool, table = R.page(np.random.default_rng(5), x.reshape(*shp, *x.shape[2:]), block,
                                 table=table)
            pools.append(pool)
        ckc, cvc = R.to_dev(pools[0], fmt), R.to_dev(pools[1], fmt)
        cks, cvs = torch.from_numpy(pools[2]).cuda(), torch.from_numpy(pools[3]).cuda()
        dt = torch.from_numpy(table).cuda()
        g.rope_kv_append_q8_paged(qkv, n_seq, t, dpos, dcos, dsin, ckc, cvc, cks, cvs, dt,
                                  table.shape[1], block, n_q, n_kv, hd)
        g.kv_read_q8_paged(ckc, cvc, cks, cvs, dt, table.shape[1], block, dpos, n_seq, t, n_kv, hd,
                           ko, vo, t + 2)
        got = [x.view(torch.int8).cpu().numpy() for x in (ckc, cvc)]
        gots = [x.cpu().numpy() for x in (cks, cvs)]
        wants, wantss = pools[4:6], pools[6:8]
    assert g.device_error() == 0
    assert np.array_equal(host_bits(qkv).reshape(want.shape), want)
    for a, w in zip(got, wants):
        assert np.array_equal(a, w)
    for a, w in zip(gots, wantss):
        assert np.array_equal(a.view(np.uint32), w.view(np.uint32))
    # read back: code * scale in f32, rounded once; rows past t untouched
    for out, first in ((ko, n_q), (vo, n_q + n_kv)):
        codes, scale = R.quantise(rows[:, :, first:first + n_kv], fmt)
        val = R.values(codes, fmt).astype(np.float32) * scale[..., None]
        w16 = torch.from_numpy(val.transpose(0, 2, 1, 3).copy()).to(tdt)
        assert torch.equal(out[:, :, :t].cpu(), w16)
        assert bool((out[:, :, t:] == 3.0).all())
        # and within half a step of the row: int8 scale / 2, e4m3 2^-4 relative (2^-10 scale
        # below its normal range), plus the f32 steps of the product and the rounding
        x = rows[:, :, first:first + n_kv].astype(np.float64)
        step = scale[..., None] * 0.5 if fmt == "int8" else np.maximum(
            np.abs(x) * 2.0 ** -4, scale[..., None] * 2.0 ** -10)
        assert np.all(np.abs(R.values(codes, fmt) * scale[..., None] - x) <=
                      step + np.abs(x).max(-1, keepdims=True) * 2.0 ** -21)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_special_rows(g, fmt):
    """Zero rows, subnormal rows, rows at the tiny threshold, the largest finite value, and
    rows with a NaN or an infinity; no rotation tables."""
    n_kv, hd = 4, 64
    rng = np.random.default_rng(0)
    rows = []
    for special in (0.0, 2.0 ** -130, 2.0 ** -119, 2.0 ** -120, 3.38e38, np.nan, np.inf, -np.inf, 1.0):
        x = rng.normal(0, 1, (2 * n_kv, hd)).astype(np.float32)
        x = x * np.float32(special) if np.isfinite(special) and special < 1e38 else x
        if not (np.isfinite(special) and special < 1e38):
            x[:, 5] = special
        rows.append(x)
    t = len(rows)
    bits = O.from_f32(np.stack(rows).ravel())
    x = O.to_f32(bits).astype(np.float32).reshape(t, 2 * n_kv, hd)
    kc = torch.zeros(n_kv, t, hd, dtype=torch.int8, device="cuda").view(R.CODE[fmt])
    vc, ks = kc.clone(), torch.zeros(n_kv, t, device="cuda")
    vs = ks.clone()
    g.rope_kv_append_q8(dev(bits), 1, t, torch.zeros(1, dtype=torch.int32, device="cuda"), None,
                        None, kc, vc, ks, vs, n_kv * t * hd, 0, n_kv, hd, t)
    ko = torch.empty(n_kv, t, hd, dtype=torch.bfloat16, device="cuda")
    vo = torch.empty_like(ko)
    g.kv_read_q8(kc, vc, ks, vs, n_kv * t * hd, torch.zeros(1, dtype=torch.int32, device="cuda"), 1,
                 t, n_kv, hd, t, ko, vo, t)
    assert g.device_error() == 0
    for c, s, out, part in ((kc, ks, ko, x[:, :n_kv]), (vc, vs, vo, x[:, n_kv:])):
        codes, scale = R.quantise(part.transpose(1, 0, 2), fmt)
        assert np.array_equal(c.view(torch.int8).cpu().numpy(), codes)
        got = s.cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(scale))
        assert np.array_equal(got[~np.isnan(scale)], scale[~np.isnan(scale)])
        nan = torch.from_numpy(np.isnan(scale))[..., None].expand(-1, -1, hd)
        assert torch.equal(out.cpu().isnan(), nan)


def test_append_reports_bad_positions_and_blocks(g):
    n_seq, n_kv, hd, max_seq = 5, 2, 64, 32
    rng = np.random.default_rng(1)
    bits = normal16(rng, n_seq * 2 * n_kv * hd)
    pos = torch.tensor([3, -1, 32, 40, 0], dtype=torch.int32, device="cuda")
    kc = torch.full((n_seq, n_kv, max_seq, hd), 9, dtype=torch.int8, device="cuda")
    vc, ks = kc.clone(), torch.full((n_seq, n_kv, max_seq), 9.0, device="cuda")
    vs = ks.clone()
    g.rope_kv_append_q8(dev(bits), n_seq, 1, pos, None, None, kc, vc, ks, vs, n_kv * max_seq * hd,
                        0, n_kv, hd, max_seq)
    assert g.device_error() == 4
    for b in (1, 2, 3):
        assert bool((kc[b] == 9).all()) and bool((vs[b] == 9.0).all())
    assert not bool((kc[0, :, 3] == 9).all()) and not bool((vc[4, :, 0] == 9).all())
    # paged: an entry of -1 and one past the pool
    table = torch.tensor([[0, 1], [-1, 2], [6, 3], [4, 5], [1, 0]], dtype=torch.int32, device="cuda")
    kp = torch.full((6, n_kv, 16, hd), 9, dtype=torch.int8, device="cuda")
    vp, sp = kp.clone(), torch.full((6, n_kv, 16), 9.0, device="cuda")
    sv = sp.clone()
    pos = torch.tensor([3, 0, 15, 17, 5], dtype=torch.int32, device="cuda")
    g.rope_kv_append_q8_paged(dev(bits), n_seq, 1, pos, None, None, kp, vp, sp, sv, table, 2, 16, 0,
                              n_kv, hd)
    assert g.device_error() == 4
    written = (sp != 9.0).nonzero().tolist()
    assert sorted(set((a, c) for a, _, c in written)) == [(0, 3), (1, 5), (5, 1)]
    ko = torch.ones(n_seq, n_kv, 1, hd, dtype=torch.bfloat16, device="cuda")
    vo = torch.ones_like(ko)
    g.kv_read_q8_paged(kp, vp, sp, sv, table, 2, 16, pos, n_seq, 1, n_kv, hd, ko, vo, 1)
    assert g.device_error() == 4
    assert bool((ko[1:3] == 0).all()) and bool((ko[[0, 3, 4]] != 0).any())


# ---------------------------------------------------------------------- decode attention
LENS = [0, 1, 15, 16, 17, 63, 64, 65, 255, 256, 257, 700, 1301]


def _decode_case(rng, lens, n_q, n_kv, hd, fmt, dtype, row_scale=None, q_std=1.0):
    n_seq, max_seq = len(lens), max(lens) + 3
    q = normal16(rng, n_seq * n_q * hd, std=q_std, dtype=dtype)
    qf = O.to_f32(q, dtype).astype(np.float64).reshape(n_seq, n_q, hd)
    lead = (n_seq, n_kv)
    rs = [None, None] if row_scale is None else row_scale
    kc, ks = R.cache(rng, lead, max_seq, hd, fmt, rs[0])
    vc, vs = R.cache(rng, lead, max_seq, hd, fmt, rs[1])
    for b, n in enumerate(lens):  # what lies past the length must not matter
        kc[b, :, n:], vc[b, :, n:] = 0x7F, -1
        ks[b, :, n:], vs[b, :, n:] = np.nan, np.inf

    def kv_of(b, h):
        n = lens[b]
        return (R.values(kc[b, h, :n], fmt) * ks[b, h, :n, None].astype(np.float64),
                R.values(vc[b, h, :n], fmt) * vs[b, h, :n, None].astype(np.float64))
    return q, qf, (kc, vc, ks, vs), kv_of, max_seq


def _run_decode(g, q, cache, lens, n_q, n_kv, hd, max_seq, fmt, dtype, block=0, workspace=True,
                table=None):
    n_seq, max_len = len(lens), max(lens)
    out = torch.empty(n_seq, n_q * hd, dtype=R.TDT[dtype], device="cuda")
    ws = torch.empty(max(16, g.attention_decode_q8_workspace_bytes(n_seq, max_len, n_q, n_kv, hd)),
                     dtype=torch.uint8, device="cuda") if workspace else None
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kc, vc, ks, vs = cache
    if block:
        pools = []
        for x in (kc, vc, ks, vs):
            pool, table = R.page(np.random.default_rng(3), x, block, table=table)
            pools.append(pool)
        t = table.copy()
        for b, n in enumerate(lens):  # entries past the last key are never used
            t[b, -(-n // block):] = -1
        g.attention_decode_q8_paged(dev(q, dtype), n_q * hd, R.to_dev(pools[0], fmt),
                                    R.to_dev(pools[1], fmt), torch.from_numpy(pools[2]).cuda(),
                                    torch.from_numpy(pools[3]).cuda(), torch.from_numpy(t).cuda(),
                                    t.shape[1], block, ld, max_len, n_q, n_kv, hd, out, n_q * hd,
                                    workspace=ws)
    else:
        g.attention_decode_q8(dev(q, dtype), n_q * hd, R.to_dev(kc, fmt), R.to_dev(vc, fmt),
                              torch.from_numpy(ks).cuda(), torch.from_numpy(vs).cuda(),
                              n_kv * max_seq * hd, ld, max_len, n_q, n_kv, hd, max_seq, out,
                              n_q * hd, workspace=ws)
    return out


@pytest.mark.parametrize("n_q,n_kv,hd,block", [
    (32, 8, 64, 0), (32, 8, 64, 16), (32, 8, 64, 64), (4, 4, 64, 48), (6, 2, 64, 0), (14, 2, 64, 32),
    (16, 1, 64, 0), (20, 1, 64, 0), (8, 2, 128, 0), (8, 1, 128, 16), (16, 1, 128, 128),
    (3, 3, 128, 0), (4, 2, 80, 0), (4, 2, 80, 24), (2, 1, 256, 0), (4, 2, 64, 8), (5, 5, 5, 0)])
@pytest.mark.parametrize("fmt,dtype", [("int8", "bf16"), ("e4m3", "bf16"), ("int8", "f16"),
                                       ("e4m3", "f16")])
def test_decode_against_f64(g, n_q, n_kv, hd, block, fmt, dtype):
    rng = np.random.default_rng(n_q * 100 + hd + block)
    q, qf, cache, kv_of, max_seq = _decode_case(rng, LENS, n_q, n_kv, hd, fmt, dtype)
    out = _run_decode(g, q, cache, LENS, n_q, n_kv, hd, max_seq, fmt, dtype, block)
    assert g.device_error() == 0
    assert bool((out[0] == 0).all())  # no keys: zeros
    R.check_attention(out, qf, kv_of, n_kv, R.default_scale(hd), dtype, W_EPS, q_eps=R.Q_EPS[fmt])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("n_seq,n", [(1, 513), (1, 5000), (1, 70000), (3, 16384), (150, 300)])
def test_decode_splits_agree_with_f64(g, fmt, n_seq, n):
    """One long sequence (keys split over CTAs), many short ones, with and without workspace."""
    rng = np.random.default_rng(n)
    n_q, n_kv, hd = 8, 2, 64
    lens = [n - 7 * i for i in range(n_seq)] if n_seq < 10 else [n - i for i in range(n_seq)]
    q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, fmt, "bf16")
    for ws in (True, False):
        out = _run_decode(g, q, cache, lens, n_q, n_kv, hd, max_seq, fmt, "bf16", workspace=ws)
        again = _run_decode(g, q, cache, lens, n_q, n_kv, hd, max_seq, fmt, "bf16", workspace=ws)
        assert g.device_error() == 0
        assert torch.equal(out, again)
        R.check_attention(out, qf, kv_of, n_kv, R.default_scale(hd), "bf16", W_EPS, q_eps=R.Q_EPS[fmt])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_decode_with_scales_of_many_magnitudes(g, fmt):
    """K rows over 2^12 and V rows over 2^24 in magnitude, peaked softmax: a key with a small
    V scale that takes all the weight must keep its precision."""
    rng = np.random.default_rng(9)
    n_q, n_kv, hd, lens = 8, 2, 64, [700, 64, 33]
    shape = (3, n_kv, 703)
    rs = [2.0 ** rng.integers(-10, 3, shape), 2.0 ** rng.integers(-20, 5, shape)]
    q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, fmt, "bf16", rs, q_std=4.0)
    out = _run_decode(g, q, cache, lens, n_q, n_kv, hd, max_seq, fmt, "bf16")
    R.check_attention(out, qf, kv_of, n_kv, R.default_scale(hd), "bf16", W_EPS, q_eps=R.Q_EPS[fmt])


@pytest.mark.parametrize("hd", [64, 128, 80])
def test_decode_nan_rows_stay_in_their_head(g, hd):
    rng = np.random.default_rng(4)
    n_q, n_kv, lens = 8, 2, [300, 300]
    q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, "int8", "bf16")
    clean = _run_decode(g, q, cache, lens, n_q, n_kv, hd, max_seq, "int8", "bf16")
    cache[2][0, 1, 130] = np.nan  # a K row of sequence 0, KV head 1
    cache[3][1, 0, 7] = np.nan    # a V row of sequence 1, KV head 0
    out = _run_decode(g, q, cache, lens, n_q, n_kv, hd, max_seq, "int8", "bf16").view(2, 2, -1)
    clean = clean.view(2, 2, -1)
    assert bool(out[0, 1].isnan().all()) and bool(out[1, 0].isnan().all())
    assert torch.equal(out[0, 0], clean[0, 0]) and torch.equal(out[1, 1], clean[1, 1])


@pytest.mark.parametrize("hd", [64, 128, 80])
def test_decode_strides_and_untouched_columns(g, hd):
    """q inside qkv rows, out rows wider than the result, caches further apart than needed."""
    rng = np.random.default_rng(6)
    n_q, n_kv, lens = 8, 2, [90, 5, 130]
    q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, "e4m3", "f16")
    want = _run_decode(g, q, cache, lens, n_q, n_kv, hd, max_seq, "e4m3", "f16")
    qs, os_ = (n_q + 2 * n_kv) * hd, n_q * hd + 8
    wide = torch.full((3, qs), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, :n_q * hd] = dev(q, "f16").view(3, -1)
    gap = 5
    seq_rows = n_kv * max_seq + gap

    def spread(x):
        flat = x.reshape(3, n_kv * max_seq, *x.shape[3:])
        y = np.zeros((3, seq_rows, *x.shape[3:]), x.dtype)
        y[:, :n_kv * max_seq] = flat
        return y
    kc, vc, ks, vs = (spread(x) for x in cache)
    out = torch.full((3, os_), 7.0, dtype=torch.float16, device="cuda")
    g.attention_decode_q8(wide, qs, R.to_dev(kc, "e4m3"), R.to_dev(vc, "e4m3"),
                          torch.from_numpy(ks).cuda(), torch.from_numpy(vs).cuda(), seq_rows * hd,
                          torch.tensor(lens, dtype=torch.int32, device="cuda"), max(lens), n_q, n_kv,
                          hd, max_seq, out, os_,
                          workspace=torch.empty(max(16, g.attention_decode_q8_workspace_bytes(
                              3, max(lens), n_q, n_kv, hd)), dtype=torch.uint8, device="cuda"))
    assert g.device_error() == 0
    assert torch.equal(out[:, :n_q * hd], want)
    assert bool((out[:, n_q * hd:] == 7.0).all())


@pytest.mark.parametrize("hd", [64, 80])
def test_decode_bad_lengths_and_blocks_are_reported(g, hd):
    rng = np.random.default_rng(8)
    n_q, n_kv, lens = 4, 1, [40, 40, 40]
    q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, "e4m3", "bf16")
    kc, vc, ks, vs = cache
    out = torch.empty(3, n_q * hd, dtype=torch.bfloat16, device="cuda")
    args = (R.to_dev(kc, "e4m3"), R.to_dev(vc, "e4m3"), torch.from_numpy(ks).cuda(),
            torch.from_numpy(vs).cuda(), n_kv * max_seq * hd)
    g.attention_decode_q8(dev(q), n_q * hd, *args,
                          torch.tensor([-5, 41, 40], dtype=torch.int32, device="cuda"), 40, n_q, n_kv,
                          hd, max_seq, out, n_q * hd)
    assert g.device_error() == 2
    want = _run_decode(g, q, cache, [0, 40, 40], n_q, n_kv, hd, max_seq, "e4m3", "bf16")
    assert torch.equal(out, want)
    # paged: a bad entry reads as zero keys and values
    pools = [R.page(np.random.default_rng(3), x, 16)[0] for x in cache]
    table = R.page(np.random.default_rng(3), kc, 16)[1]
    bad = table.copy()
    bad[0, 1], bad[2, 0] = -1, pools[0].shape[0]
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    g.attention_decode_q8_paged(dev(q), n_q * hd, R.to_dev(pools[0], "e4m3"),
                                R.to_dev(pools[1], "e4m3"), torch.from_numpy(pools[2]).cuda(),
                                torch.from_numpy(pools[3]).cuda(), torch.from_numpy(bad).cuda(),
                                bad.shape[1], 16, ld, 40, n_q, n_kv, hd, out, n_q * hd)
    assert g.device_error() == 4

    def zeroed(b, h):
        k, v = kv_of(b, h)
        for i in range(3):
            if bad[b, i] != table[b, i]:
                k[16 * i:16 * i + 16], v[16 * i:16 * i + 16] = 0, 0
        return k, v
    R.check_attention(out, qf, zeroed, n_kv, R.default_scale(hd), "bf16", W_EPS)


def test_decode_in_graph_and_on_another_stream(g):
    from kvasir_b200 import Gpu
    rng = np.random.default_rng(11)
    n_q, n_kv, hd, lens, fmt = 32, 8, 64, [700, 1, 300], "int8"
    cases = [_decode_case(rng, lens, n_q, n_kv, hd, fmt, "bf16") for _ in range(2)]
    max_seq = cases[0][4]
    want = [_run_decode(g, c[0], c[2], lens, n_q, n_kv, hd, max_seq, fmt, "bf16") for c in cases]
    s = torch.cuda.Stream()
    gs = Gpu(0, stream=s)
    q = dev(cases[0][0]).clone()
    kc, vc = (R.to_dev(x, fmt) for x in cases[0][2][:2])
    ks, vs = (torch.from_numpy(x).cuda() for x in cases[0][2][2:])
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.empty(3, n_q * hd, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(max(16, g.attention_decode_q8_workspace_bytes(3, 700, n_q, n_kv, hd)),
                     dtype=torch.uint8, device="cuda")

    def call():
        gs.attention_decode_q8(q, n_q * hd, kc, vc, ks, vs, n_kv * max_seq * hd, ld, 700, n_q, n_kv,
                               hd, max_seq, out, n_q * hd, workspace=ws)
    torch.cuda.synchronize()
    call()
    s.synchronize()
    assert torch.equal(out, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        call()
    for i in (1, 0):
        for t, x in zip((kc, vc), cases[i][2][:2]):
            t.view(torch.int8).copy_(torch.from_numpy(x))
        ks.copy_(torch.from_numpy(cases[i][2][2]))
        vs.copy_(torch.from_numpy(cases[i][2][3]))
        q.copy_(dev(cases[i][0]))
        out.fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
    assert g.device_error() == 0


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("block", [0, 64])
def test_prefill_then_decode_steps_on_one_cache(g, fmt, block):
    """As a server runs them: a prompt's rows appended, read back and prefilled over, then
    decode steps that append one row per sequence and attend.  The prefill equals
    attention_prefill on the f64-checked read-back rows; each step is checked against f64 on
    what the cache holds."""
    n_q, n_kv, hd, n_seq, t, steps = 8, 2, 64, 3, 70, 3
    max_seq, dtype = 128, "bf16"
    rng = np.random.default_rng(21)
    heads = n_q + 2 * n_kv
    cos, sin = _tables(hd, max_seq)
    dcos, dsin = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    per = max_seq // block if block else 0
    lead = (n_seq * per, n_kv, block) if block else (n_seq, n_kv, max_seq)
    kc = torch.zeros(*lead, hd, dtype=torch.int8, device="cuda").view(R.CODE[fmt])
    vc, ks = kc.clone(), torch.zeros(*lead, device="cuda")
    vs = ks.clone()
    table = torch.from_numpy(rng.permutation(n_seq * max(per, 1)).astype(np.int32)).cuda().view(
        n_seq, -1)

    def append(bits, t, pos):
        qkv = dev(bits)
        p = torch.full((n_seq,), pos, dtype=torch.int32, device="cuda")
        if block:
            g.rope_kv_append_q8_paged(qkv, n_seq, t, p, dcos, dsin, kc, vc, ks, vs, table, per, block,
                                      n_q, n_kv, hd)
        else:
            g.rope_kv_append_q8(qkv, n_seq, t, p, dcos, dsin, kc, vc, ks, vs, n_kv * max_seq * hd,
                                n_q, n_kv, hd, max_seq)
        return qkv

    def read(n):
        k = torch.zeros(n_seq, n_kv, max_seq, hd, dtype=torch.bfloat16, device="cuda")
        v, p = torch.zeros_like(k), torch.zeros(n_seq, dtype=torch.int32, device="cuda")
        if block:
            g.kv_read_q8_paged(kc, vc, ks, vs, table, per, block, p, n_seq, n, n_kv, hd, k, v, max_seq)
        else:
            g.kv_read_q8(kc, vc, ks, vs, n_kv * max_seq * hd, p, n_seq, n, n_kv, hd, max_seq, k, v,
                         max_seq)
        return k, v

    def exact_rows():
        """f64 values of the cache, [n_seq, n_kv, max_seq, hd]."""
        got = []
        for c, s in ((kc, ks), (vc, vs)):
            x = R.values(c.view(torch.int8).cpu().numpy(), fmt) * s.cpu().numpy().astype(
                np.float64)[..., None]
            if block:
                x = x[table.cpu().numpy()].transpose(0, 2, 1, 3, 4).reshape(n_seq, n_kv, max_seq, hd)
            got.append(x)
        return got

    qkv = append(normal16(rng, n_seq * t * heads * hd), t, 0)
    k16, v16 = read(t)
    out = torch.empty(n_seq * t, n_q * hd, dtype=torch.bfloat16, device="cuda")
    g.attention_prefill(qkv, k16, v16, out, n_seq, t, 0, n_q, n_kv, hd, max_seq)
    q = O.to_f32(host_bits(qkv)).astype(np.float64).reshape(n_seq, t, heads, hd)[:, :, :n_q]
    k, v = (x.float().cpu().numpy().astype(np.float64) for x in (k16, v16))
    got = out.view(n_seq, t, -1)
    for i in (0, 1, 33, t - 1):
        R.check_attention(got[:, i], q[:, i], lambda b, h: (k[b, h, :i + 1], v[b, h, :i + 1]), n_kv,
                          R.default_scale(hd), dtype, 2.0 ** -15, f"row {i}")
    for i in range(steps):
        qkv = append(normal16(rng, n_seq * heads * hd), 1, t + i)
        n = t + i + 1
        ld = torch.full((n_seq,), n, dtype=torch.int32, device="cuda")
        step = torch.empty(n_seq, n_q * hd, dtype=torch.bfloat16, device="cuda")
        if block:
            g.attention_decode_q8_paged(qkv, heads * hd, kc, vc, ks, vs, table, per, block, ld, n, n_q,
                                        n_kv, hd, step, n_q * hd)
        else:
            g.attention_decode_q8(qkv, heads * hd, kc, vc, ks, vs, n_kv * max_seq * hd, ld, n, n_q,
                                  n_kv, hd, max_seq, step, n_q * hd)
        kx, vx = exact_rows()
        qx = O.to_f32(host_bits(qkv)).astype(np.float64).reshape(n_seq, heads, hd)[:, :n_q]
        R.check_attention(step, qx, lambda b, h: (kx[b, h, :n], vx[b, h, :n]), n_kv,
                          R.default_scale(hd), dtype, W_EPS, f"step {i}", R.Q_EPS[fmt])
    assert g.device_error() == 0


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_decode_query_magnitudes(g, fmt, dtype):
    """Heads of q from 2^-20 to 2^7 in magnitude, one of zeros, elements spread over 2^10 within
    a head; a NaN and an infinity make their own head's row NaN and no other."""
    rng = np.random.default_rng(31)
    n_q, n_kv, hd, lens = 16, 2, 64, [300, 65]
    q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, fmt, dtype)
    x = qf * 2.0 ** rng.integers(-10, 1, qf.shape) * 2.0 ** np.linspace(-20, 4, n_q)[None, :, None]
    x[0, 5] = 0
    q = O.from_f32(x.astype(np.float32).ravel(), dtype)
    qf = O.to_f32(q, dtype).astype(np.float64).reshape(x.shape)
    out = _run_decode(g, q, cache, lens, n_q, n_kv, hd, max_seq, fmt, dtype)
    R.check_attention(out, qf, kv_of, n_kv, R.default_scale(hd), dtype, W_EPS, q_eps=R.Q_EPS[fmt])
    x[0, 2, 7], x[1, 9, 0] = np.nan, np.inf
    bad = _run_decode(g, O.from_f32(x.astype(np.float32).ravel(), dtype), cache, lens, n_q, n_kv, hd,
                      max_seq, fmt, dtype).view(2, n_q, hd)
    rows = torch.zeros(2, n_q, dtype=torch.bool)
    rows[0, 2] = rows[1, 9] = True
    assert torch.equal(bad.isnan().all(-1).cpu(), rows)
    keep = ~rows.cuda()
    assert torch.equal(bad[keep], out.view(2, n_q, hd)[keep])


@pytest.mark.parametrize("n_q,n_kv,hd,block", [
    (32, 8, 64, 0), (32, 8, 64, 16), (6, 2, 64, 48), (16, 1, 64, 64), (8, 2, 128, 0), (16, 1, 128, 32),
    (3, 3, 128, 16)])
@pytest.mark.parametrize("fmt,dtype", [("int8", "bf16"), ("e4m3", "bf16"), ("int8", "f16"),
                                       ("e4m3", "f16")])
@pytest.mark.parametrize("workspace", [True, False])
def test_fused_step_equals_append_then_decode(g, n_q, n_kv, hd, block, fmt, dtype, workspace):
    """rope_attention_decode_q8: out, codes and scales bit for bit, at lengths around tiles and
    chunks; qkv stays as it was.  The last sequence's position lies outside the RoPE tables."""
    rng = np.random.default_rng(hd + block + n_q)
    lens = [1, 2, 32, 33, 64, 65, 128, 129, 256, 257, 512, 513, 900, 1301, 1400]
    n_seq, max_seq = len(lens), 1408
    heads = n_q + 2 * n_kv
    qkv = dev(normal16(rng, n_seq * heads * hd, dtype=dtype), dtype).view(n_seq, -1)
    cos, sin = _tables(hd, 1399)
    dcos, dsin = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    kc, ks = R.cache(rng, (n_seq, n_kv), max_seq, hd, fmt)
    vc, vs = R.cache(rng, (n_seq, n_kv), max_seq, hd, fmt)
    table = None
    arrays = [kc, vc, ks, vs]
    if block:
        pools = []
        for x in arrays:
            pool, table = R.page(np.random.default_rng(3), x, block, table=table)
            pools.append(pool)
        arrays = pools
        dt = torch.from_numpy(table).cuda()

    def caches():
        return [R.to_dev(arrays[0], fmt), R.to_dev(arrays[1], fmt), torch.from_numpy(arrays[2]).cuda(),
                torch.from_numpy(arrays[3]).cuda()]
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = torch.empty(max(16, g.attention_decode_q8_workspace_bytes(n_seq, max_seq, n_q, n_kv, hd)),
                     dtype=torch.uint8, device="cuda") if workspace else None
    want = torch.empty(n_seq, n_q * hd, dtype=R.TDT[dtype], device="cuda")
    got = torch.empty_like(want)
    a, b = caches(), caches()
    rot = qkv.clone()
    stride = n_kv * max_seq * hd
    if block:
        g.rope_kv_append_q8_paged(rot, n_seq, 1, ld - 1, dcos, dsin, *a, dt, dt.shape[1], block, n_q, n_kv,
                                  hd)
        assert g.device_error() == 4
        g.attention_decode_q8_paged(rot, heads * hd, *a, dt, dt.shape[1], block, ld, max_seq, n_q, n_kv, hd,
                                    want, n_q * hd, workspace=ws)
        before = qkv.clone()
        g.rope_attention_decode_q8_paged(qkv, dcos, dsin, *b, dt, dt.shape[1], block, ld, max_seq, n_q,
                                         n_kv, hd, got, n_q * hd, workspace=ws)
    else:
        g.rope_kv_append_q8(rot, n_seq, 1, ld - 1, dcos, dsin, *a, stride, n_q, n_kv, hd, max_seq)
        assert g.device_error() == 4
        g.attention_decode_q8(rot, heads * hd, *a, stride, ld, max_seq, n_q, n_kv, hd, max_seq, want,
                              n_q * hd, workspace=ws)
        before = qkv.clone()
        g.rope_attention_decode_q8(qkv, dcos, dsin, *b, stride, ld, max_seq, n_q, n_kv, hd, max_seq, got,
                                   n_q * hd, workspace=ws)
    assert g.device_error() == 4
    assert torch.equal(qkv, before)
    assert torch.equal(got, want)
    for x, y in zip(a, b):
        if x.dtype == torch.float32:
            assert torch.equal(x.view(torch.int32), y.view(torch.int32))
        else:
            assert torch.equal(x.view(torch.int8), y.view(torch.int8))


def test_fused_step_reports_bad_blocks_and_refuses_other_shapes(g):
    from kvasir_b200.gpu import ShapeError, UnsupportedError
    n_q, n_kv, hd = 4, 2, 64
    rng = np.random.default_rng(2)
    qkv = dev(normal16(rng, 2 * 8 * hd)).view(2, -1)
    cos, sin = (torch.from_numpy(x).cuda() for x in _tables(hd, 64))
    kp = torch.full((4, n_kv, 16, hd), 9, dtype=torch.int8, device="cuda")
    vp, sk = kp.clone(), torch.full((4, n_kv, 16), 1.0, device="cuda")
    sv = sk.clone()
    table = torch.tensor([[0, -1], [1, 9]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([20, 17], dtype=torch.int32, device="cuda")
    out = torch.empty(2, n_q * hd, dtype=torch.bfloat16, device="cuda")
    g.rope_attention_decode_q8_paged(qkv, cos, sin, kp, vp, sk, sv, table, 2, 16, lens, 32, n_q, n_kv, hd,
                                     out, n_q * hd)
    assert g.device_error() == 4
    assert bool((kp == 9).all()) and bool((vp == 9).all()) and bool((sk == 1).all())
    # 16 keys of value 9 with scale 1, then keys that read as zeros: between 0 and 9
    assert bool(((out >= 0) & (out <= 9)).all())
    with pytest.raises(UnsupportedError):
        g.rope_attention_decode_q8_paged(qkv, cos, sin, kp, vp, sk, sv, table.view(2, 2), 2, 8, lens, 16,
                                         n_q, n_kv, hd, out, n_q * hd)
    with pytest.raises(ShapeError):
        g.rope_attention_decode_q8_paged(qkv[:, :-1].contiguous(), cos, sin, kp, vp, sk, sv, table, 2, 16,
                                         lens, 32, n_q, n_kv, hd, out, n_q * hd)
    with pytest.raises(ShapeError):
        g.attention_decode_q8_paged(qkv.float(), n_q * hd, kp, vp, sk, sv, table, 2, 16, lens, 32, n_q,
                                    n_kv, hd, out, n_q * hd)


@pytest.mark.parametrize("hd", [64, 128])
def test_unaligned_buffers_take_the_general_kernels(g, hd):
    """Views that start one element (or one code) past an aligned address: the append gives the
    same bits, the attention the f64 result."""
    rng = np.random.default_rng(17)
    n_q, n_kv, fmt, dtype, t, max_seq = 4, 2, "int8", "bf16", 3, 40
    heads = n_q + 2 * n_kv
    bits = normal16(rng, t * heads * hd)
    cos, sin = (torch.from_numpy(x).cuda() for x in _tables(hd, max_seq))
    pos = torch.tensor([30], dtype=torch.int32, device="cuda")
    got = []
    for shift in (0, 1):
        q = torch.empty(t * heads * hd + 1, dtype=torch.bfloat16, device="cuda")[shift:shift + bits.size]
        q.copy_(dev(bits))
        cs = [torch.zeros(n_kv * max_seq * hd + 1, dtype=torch.int8, device="cuda")[shift:][
            :n_kv * max_seq * hd] for _ in range(2)]
        sc = [torch.zeros(n_kv * max_seq, device="cuda") for _ in range(2)]
        g.rope_kv_append_q8(q, 1, t, pos, cos, sin, *cs, *sc, n_kv * max_seq * hd, n_q, n_kv, hd, max_seq)
        ko = torch.empty(2 * n_kv * t * hd + 1, dtype=torch.bfloat16, device="cuda")[shift:]
        kv = ko[:n_kv * t * hd], ko[n_kv * t * hd:2 * n_kv * t * hd]
        g.kv_read_q8(*cs, *sc, n_kv * max_seq * hd, pos, 1, t, n_kv, hd, max_seq, *kv, t)
        got.append([q.clone(), *[x.clone() for x in cs], *sc, *[x.clone() for x in kv]])
    assert all(torch.equal(x, y) for x, y in zip(*got))
    lens = [33, 7]
    q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, fmt, dtype)
    kc, vc, ks, vs = cache
    shifted = []
    for x in (kc, vc):
        y = torch.empty(x.size + 1, dtype=torch.int8, device="cuda")[1:]
        y.copy_(torch.from_numpy(x.ravel()))
        shifted.append(y)
    qs = torch.empty(q.size + 1, dtype=torch.bfloat16, device="cuda")[1:]
    qs.copy_(dev(q))
    out = torch.empty(2, n_q * hd, dtype=torch.bfloat16, device="cuda")
    g.attention_decode_q8(qs, n_q * hd, *shifted, torch.from_numpy(ks).cuda(), torch.from_numpy(vs).cuda(),
                          n_kv * max_seq * hd, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                          max(lens), n_q, n_kv, hd, max_seq, out, n_q * hd)
    R.check_attention(out, qf, kv_of, n_kv, R.default_scale(hd), dtype, W_EPS, q_eps=R.Q_EPS[fmt])
    assert g.device_error() == 0


def test_calls_on_two_streams_at_once(g):
    """Two handles on two streams, each with a workspace of its own, many calls in flight."""
    from kvasir_b200 import Gpu
    rng = np.random.default_rng(41)
    n_q, n_kv, hd, fmt = 32, 8, 64, "e4m3"
    jobs = []
    for lens in ([700, 1301, 64], [5, 2000, 900]):
        q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, fmt, "bf16")
        want = _run_decode(g, q, cache, lens, n_q, n_kv, hd, max_seq, fmt, "bf16")
        h = Gpu(0, stream=torch.cuda.Stream())
        ws = torch.empty(max(16, h.attention_decode_q8_workspace_bytes(3, max(lens), n_q, n_kv, hd)),
                         dtype=torch.uint8, device="cuda")
        args = (dev(q), n_q * hd, R.to_dev(cache[0], fmt), R.to_dev(cache[1], fmt),
                torch.from_numpy(cache[2]).cuda(), torch.from_numpy(cache[3]).cuda(), n_kv * max_seq * hd,
                torch.tensor(lens, dtype=torch.int32, device="cuda"), max(lens), n_q, n_kv, hd, max_seq)
        jobs.append((h, args, want, ws))
    torch.cuda.synchronize()
    outs = [[torch.empty_like(want) for _ in range(20)] for _, _, want, _ in jobs]
    torch.cuda.synchronize()
    for i in range(20):
        for (h, args, _, ws), o in zip(jobs, outs):
            h.attention_decode_q8(*args, o[i], n_q * hd, workspace=ws)
    torch.cuda.synchronize()
    for (_, _, want, _), o in zip(jobs, outs):
        assert all(torch.equal(x, want) for x in o)
    assert g.device_error() == 0


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("scale", [0.0, -0.125])
def test_decode_scale_of_either_sign(g, fmt, scale):
    rng = np.random.default_rng(3)
    n_q, n_kv, hd, lens = 8, 2, 64, [70, 300]
    q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, fmt, "bf16")
    kc, vc, ks, vs = cache
    out = torch.empty(2, n_q * hd, dtype=torch.bfloat16, device="cuda")
    g.attention_decode_q8(dev(q), n_q * hd, R.to_dev(kc, fmt), R.to_dev(vc, fmt),
                          torch.from_numpy(ks).cuda(), torch.from_numpy(vs).cuda(), n_kv * max_seq * hd,
                          torch.tensor(lens, dtype=torch.int32, device="cuda"), max(lens), n_q, n_kv, hd,
                          max_seq, out, n_q * hd, scale=scale)
    R.check_attention(out, qf * (-1 if scale < 0 else 1), kv_of, n_kv, abs(scale), "bf16", W_EPS,
                      q_eps=R.Q_EPS[fmt])


@pytest.mark.parametrize("hd", [64, 80])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_rows_past_32_bit_offsets(g, fmt, hd):
    """The second sequence's rows lie more than 2^32 codes behind the first's, contiguous and in
    blocks of a pool: append, read back, decode and the one-launch step as on a small cache, bit
    for bit (hd 80: the general kernels)."""
    n_q, n_kv, rows, t, block = 8, 2, 80, 70, 16
    heads = n_q + 2 * n_kv
    rng = np.random.default_rng(51)
    cos, sin = (torch.from_numpy(x).cuda() for x in _tables(hd, rows))
    qkv0 = dev(normal16(rng, 2 * t * heads * hd)).view(2 * t, -1)
    step0 = dev(normal16(rng, 2 * heads * hd)).view(2, -1)
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    lens = torch.full((2,), t + 1, dtype=torch.int32, device="cuda")
    per = n_kv * rows * hd
    per_block = n_kv * block * hd
    blocks = rows // block

    def run(stride, n, table=None):
        kc, vc = (torch.empty(n, dtype=torch.int8, device="cuda").view(R.CODE[fmt]) for _ in range(2))
        ks, vs = (torch.empty(n // hd, device="cuda") for _ in range(2))
        qkv, step = qkv0.clone(), step0.clone()
        ko, vo = (torch.empty(2, n_kv, t, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        out, out2 = (torch.empty(2, n_q * hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        if table is None:
            g.rope_kv_append_q8(qkv, 2, t, zero, cos, sin, kc, vc, ks, vs, stride, n_q, n_kv, hd, rows)
            g.kv_read_q8(kc, vc, ks, vs, stride, zero, 2, t, n_kv, hd, rows, ko, vo, t)
            g.attention_decode_q8(step, heads * hd, kc, vc, ks, vs, stride, lens - 1, t, n_q, n_kv, hd,
                                  rows, out, n_q * hd)
            if hd == 64:
                g.rope_attention_decode_q8(step, cos, sin, kc, vc, ks, vs, stride, lens, t + 1, n_q, n_kv,
                                           hd, rows, out2, n_q * hd)
        else:
            tab = (table, table.shape[1], block)
            g.rope_kv_append_q8_paged(qkv, 2, t, zero, cos, sin, kc, vc, ks, vs, *tab, n_q, n_kv, hd)
            g.kv_read_q8_paged(kc, vc, ks, vs, *tab, zero, 2, t, n_kv, hd, ko, vo, t)
            g.attention_decode_q8_paged(step, heads * hd, kc, vc, ks, vs, *tab, lens - 1, t, n_q, n_kv, hd,
                                        out, n_q * hd)
            if hd == 64:
                g.rope_attention_decode_q8_paged(step, cos, sin, kc, vc, ks, vs, *tab, lens, t + 1, n_q,
                                                 n_kv, hd, out2, n_q * hd)
        assert g.device_error() == 0
        return (ko, vo, out) + ((out2,) if hd == 64 else ())

    far = (2 ** 32 // hd + 5) * hd
    want = run(per, 2 * per)
    for x, y in zip(run(far, far + per), want):
        assert torch.equal(x, y)
    n_blocks = 2 ** 32 // per_block + 9
    table = torch.arange(2 * blocks, dtype=torch.int32, device="cuda").view(2, blocks)
    table[1] += n_blocks - 2 * blocks
    for x, y in zip(run(0, n_blocks * per_block, table), want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("hd", [64, 128, 80])
def test_int8_codes_of_minus_128(g, hd):
    """A cache written by something else may hold -128, which the append never does."""
    rng = np.random.default_rng(52)
    n_q, n_kv, lens = 8, 2, [100, 37]
    q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, "int8", "bf16")
    kc, vc, ks, vs = cache
    for x in (kc, vc):
        x[rng.random(x.shape) < 0.3] = -128
    out = _run_decode(g, q, cache, lens, n_q, n_kv, hd, max_seq, "int8", "bf16")
    R.check_attention(out, qf, kv_of, n_kv, R.default_scale(hd), "bf16", W_EPS, q_eps=R.Q_EPS["int8"])
    ko, vo = (torch.empty(2, n_kv, 30, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g.kv_read_q8(R.to_dev(kc, "int8"), R.to_dev(vc, "int8"), torch.from_numpy(ks).cuda(),
                 torch.from_numpy(vs).cuda(), n_kv * max_seq * hd,
                 torch.zeros(2, dtype=torch.int32, device="cuda"), 2, 30, n_kv, hd, max_seq, ko, vo, 30)
    for got, c, s in ((ko, kc, ks), (vo, vc, vs)):
        want = torch.from_numpy(c[:, :, :30].astype(np.float32) * s[:, :, :30, None]).to(torch.bfloat16)
        assert torch.equal(got.cpu(), want)
    assert g.device_error() == 0


@pytest.mark.parametrize("chunks", [1, 2, 3, 7])
@pytest.mark.parametrize("hd", [64, 128])
def test_decode_smaller_workspaces(g, chunks, hd):
    """A workspace for fewer chunks than the call would take: longer ones, the same attention, and
    nothing behind the workspace is written."""
    rng = np.random.default_rng(72)
    n_q, n_kv, lens = 8, 2, [5000, 0, 4400, 63]
    q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, "int8", "bf16")
    n = len(lens) * n_kv * chunks * ((4 * (hd + 2) + 3) // 4 * 4) * 4
    assert n < g.attention_decode_q8_workspace_bytes(len(lens), max(lens), n_q, n_kv, hd)
    whole = torch.full((n + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    out = torch.empty(len(lens), n_q * hd, dtype=torch.bfloat16, device="cuda")
    kc, vc, ks, vs = cache
    g.attention_decode_q8(dev(q), n_q * hd, R.to_dev(kc, "int8"), R.to_dev(vc, "int8"),
                          torch.from_numpy(ks).cuda(), torch.from_numpy(vs).cuda(), n_kv * max_seq * hd,
                          torch.tensor(lens, dtype=torch.int32, device="cuda"), max(lens), n_q, n_kv, hd,
                          max_seq, out, n_q * hd, workspace=whole[:n])
    R.check_attention(out, qf, kv_of, n_kv, R.default_scale(hd), "bf16", W_EPS, q_eps=R.Q_EPS["int8"])
    assert bool((whole[n:] == 0xA5).all())
    assert g.device_error() == 0


@pytest.mark.parametrize("hd", [64, 128, 80])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("ratio", [2.0 ** 12, 2.0 ** 13, 2.0 ** 30, 2.0 ** 45, 2.0 ** 100])
@pytest.mark.parametrize("group", [4, 12])
def test_a_large_v_row_without_weight(g, hd, fmt, ratio, group):
    """A V row far above the others leaves them their precision: where no head gives its key weight,
    and where one head of the group does and the others do not.  The f64 bound per head."""
    rng = np.random.default_rng(group)
    n_kv, lens = 2, [700, 64, 33, 3000]
    n_q = n_kv * group
    for heads_on in (0, 1):
        q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, fmt, "bf16")
        x = np.abs(qf) + 0.5
        x[:, ::group] *= -1 if heads_on else 1  # the first head of each group
        q = O.from_f32(x.astype(np.float32).ravel())
        qf = O.to_f32(q).astype(np.float64).reshape(x.shape)
        kc, vc, ks, vs = cache
        for b, n in enumerate(lens):
            for key in (5, n // 2, n - 1):
                kc[b, :, key] = R.quantise(np.full((1, hd), -8.0, np.float32), fmt)[0]
                ks[b, :, key] = R.quantise(np.full((1, hd), -8.0, np.float32), fmt)[1]
                vs[b, :, key] *= np.float32(ratio)
        for ws in (True, False):
            out = _run_decode(g, q, cache, lens, n_q, n_kv, hd, max_seq, fmt, "bf16", workspace=ws)
            assert g.device_error() == 0
            R.check_attention(out, qf, kv_of, n_kv, R.default_scale(hd), "bf16", W_EPS,
                              f"heads_on {heads_on}", q_eps=R.Q_EPS[fmt])


@pytest.mark.parametrize("hd", [64, 128, 80])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_scores_of_minus_infinity(g, fmt, hd):
    """Scores that overflow to -infinity: NaN where a row has no other (whatever the workspace),
    and no weight beside finite ones."""
    rng = np.random.default_rng(92)
    n_q, n_kv, lens = 8, 2, [5000, 40, 0]
    q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, fmt, "bf16")
    x = (np.abs(qf) + 0.5) * 2.0 ** 60
    q = O.from_f32(x.astype(np.float32).ravel())
    kc, vc, ks, vs = cache
    one = R.quantise(np.full((1, hd), -1.0, np.float32), fmt)[0]
    kc[0, :], ks[0, :] = one, 2.0 ** 90  # every key of sequence 0
    kc[1, 0, :33], ks[1, 0, :33] = one, 2.0 ** 90  # KV head 0 of sequence 1: keys 33 .. 39 are left
    ks[1] = np.where(ks[1] < 1e10, ks[1] * np.float32(2.0 ** -60), ks[1])  # those score as usual

    def left(b, h):
        k, v = kv_of(b, h)
        return (k[33:], v[33:]) if h == 0 else (k, v)
    qs = O.to_f32(q).astype(np.float64).reshape(x.shape)
    for ws in (True, False):
        out = _run_decode(g, q, cache, lens, n_q, n_kv, hd, max_seq, fmt, "bf16", workspace=ws)
        assert g.device_error() == 0
        assert bool(out[0].isnan().all()) and bool((out[2] == 0).all())
        R.check_attention(out[1:2], qs[1:2], lambda b, h: left(1, h), n_kv, R.default_scale(hd), "bf16",
                          W_EPS, q_eps=R.Q_EPS[fmt])


@pytest.mark.parametrize("hd,block", [(64, 0), (128, 0), (64, 16)])
def test_fused_step_with_lengths_out_of_range(g, hd, block):
    """Lengths past max_len and past the cache, and negative ones: reported, and no row that is in
    the cache is lost -- the step writes what the append writes at lens - 1, and attends as the
    attention does."""
    rng = np.random.default_rng(93)
    n_q, n_kv, max_seq, max_len, fmt = 8, 2, 96, 50, "int8"
    lens = [51, 50, 80, 97, 120, -2, -2 ** 31, 2 ** 31 - 1, 7]
    n_seq, heads = len(lens), n_q + 2 * n_kv
    qkv = dev(normal16(rng, n_seq * heads * hd)).view(n_seq, -1)
    dcos, dsin = (torch.from_numpy(x).cuda() for x in _tables(hd, 88))
    arrays = [x for _ in range(2) for x in R.cache(rng, (n_seq, n_kv), max_seq, hd, fmt)]
    arrays = [arrays[0], arrays[2], arrays[1], arrays[3]]
    table = None
    if block:
        pools = []
        for x in arrays:
            pool, table = R.page(np.random.default_rng(3), x, block, table=table)
            pools.append(pool)
        arrays, table = pools, torch.from_numpy(table).cuda()
    a, b = ([R.to_dev(arrays[0], fmt), R.to_dev(arrays[1], fmt), torch.from_numpy(arrays[2]).cuda(),
             torch.from_numpy(arrays[3]).cuda()] for _ in range(2))
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    pos = torch.tensor([max(n - 1, -2 ** 31) for n in lens], dtype=torch.int32, device="cuda")
    want, got = (torch.empty(n_seq, n_q * hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    rot, stride = qkv.clone(), n_kv * max_seq * hd
    if block:
        tab = (table, table.shape[1], block)
        g.rope_kv_append_q8_paged(rot, n_seq, 1, pos, dcos, dsin, *a, *tab, n_q, n_kv, hd)
        g.attention_decode_q8_paged(rot, heads * hd, *a, *tab, ld, max_len, n_q, n_kv, hd, want, n_q * hd)
        assert g.device_error() == 6
        g.rope_attention_decode_q8_paged(qkv, dcos, dsin, *b, *tab, ld, max_len, n_q, n_kv, hd, got,
                                         n_q * hd)
    else:
        g.rope_kv_append_q8(rot, n_seq, 1, pos, dcos, dsin, *a, stride, n_q, n_kv, hd, max_seq)
        g.attention_decode_q8(rot, heads * hd, *a, stride, ld, max_len, n_q, n_kv, hd, max_seq, want,
                              n_q * hd)
        assert g.device_error() == 6
        g.rope_attention_decode_q8(qkv, dcos, dsin, *b, stride, ld, max_len, n_q, n_kv, hd, max_seq, got,
                                   n_q * hd)
    assert g.device_error() == 6
    for x, y in zip(a, b):
        kind = torch.int32 if x.dtype == torch.float32 else torch.int8
        assert torch.equal(x.view(kind), y.view(kind))
    assert torch.equal(got, want)


def test_decode_over_a_cache_without_rows(g):
    """max_len 0 on a cache of no rows, contiguous and paged: zero rows."""
    import ctypes as C
    one = torch.zeros(64, device="cuda")  # never read
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    table = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = torch.ones(2, 512, dtype=torch.bfloat16, device="cuda")
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    s = C.c_void_p(g.stream.cuda_stream)
    for paged in (False, True):
        out = torch.ones(2, 512, dtype=torch.bfloat16, device="cuda")
        if paged:
            st = g._lib.kvb_attention_decode_q8_paged(
                s, p(q), 512, p(one), p(one), p(one), p(one), 0, 0, p(table), 0, 16, p(lens), 2, 0, 8, 2, 64,
                0.125, p(out), 512, None, 0, 0, 0)
        else:
            st = g._lib.kvb_attention_decode_q8(s, p(q), 512, p(one), p(one), p(one), p(one), 0, 0, 0, p(lens),
                                                2, 0, 8, 2, 64, 0, 0.125, p(out), 512, None, 0, 0, 0)
        assert st == 0
        torch.cuda.synchronize()
        assert bool((out == 0).all())
    assert g.device_error() == 0


@pytest.mark.parametrize("hd,counts", [(64, [4, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129]),
                                       (128, [4, 8, 9, 16, 17, 32, 33, 64, 65, 140])])
@pytest.mark.parametrize("n_q", [1, 5])
def test_every_form_of_the_join(g, hd, counts, n_q):
    """Part counts on both sides of each number of warps a row and loads a lane, with sequences of
    fewer parts, of one part and of none beside them: some warps of a row have no part then."""
    unit = 256 if hd == 64 else 128  # a chunk of one tile for each warp
    part = (n_q * (hd + 2) + 3) // 4 * 4 * 4
    for parts in counts:
        lens = [unit * parts - 5, unit * (parts // 3) + 1, 7, 0][:3 if parts > 100 else 4]
        n = g.attention_decode_q8_workspace_bytes(len(lens), max(lens), n_q, 1, hd)
        if parts <= 3 * 148 // len(lens):  # of 148 SMs
            assert n == len(lens) * parts * part
        rng = np.random.default_rng(parts)
        q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, 1, hd, "int8", "bf16")
        out = _run_decode(g, q, cache, lens, n_q, 1, hd, max_seq, "int8", "bf16")
        assert g.device_error() == 0
        R.check_attention(out, qf, kv_of, 1, R.default_scale(hd), "bf16", W_EPS, f"{parts} parts",
                          R.Q_EPS["int8"])
        if len(lens) == 4:
            assert bool((out[3] == 0).all())


def test_inputs_rewritten_between_captured_calls(g):
    """Several split calls in one graph, q and lengths rewritten on the stream before each: every
    call and its join read what was written last."""
    from kvasir_b200 import Gpu
    rng = np.random.default_rng(103)
    n_q, n_kv, hd, fmt, lens = 8, 2, 64, "int8", [3000, 900, 2100]
    q, _, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, fmt, "bf16")
    kc, vc, ks, vs = R.to_dev(cache[0], fmt), R.to_dev(cache[1], fmt), *(torch.from_numpy(x).cuda()
                                                                        for x in cache[2:])
    qs = [normal16(rng, 3 * n_q * hd) for _ in range(4)]
    ns = [[int(rng.integers(0, n + 1)) for n in lens] for _ in qs]
    ns[1] = [5, 900, 0]  # one chunk, all of the keys, none
    s = torch.cuda.Stream()
    gs = Gpu(0, stream=s)
    dq, dn = [dev(x) for x in qs], [torch.tensor(n, dtype=torch.int32, device="cuda") for n in ns]
    cq, cn = torch.empty_like(dq[0]), torch.empty_like(dn[0])
    outs = [torch.empty(3, n_q * hd, dtype=torch.bfloat16, device="cuda") for _ in qs]
    ws = torch.empty(g.attention_decode_q8_workspace_bytes(3, 3000, n_q, n_kv, hd), dtype=torch.uint8,
                     device="cuda")
    assert ws.numel() > 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        for i in range(4):
            cq.copy_(dq[i])
            cn.copy_(dn[i])
            gs.attention_decode_q8(cq, n_q * hd, kc, vc, ks, vs, n_kv * max_seq * hd, cn, 3000, n_q, n_kv, hd,
                                   max_seq, outs[i], n_q * hd, workspace=ws)
    for _ in range(5):
        for o in outs:
            o.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i in range(4):
            qf = O.to_f32(qs[i]).astype(np.float64).reshape(3, n_q, hd)
            R.check_attention(outs[i], qf, lambda b, h: tuple(x[:ns[i][b]] for x in kv_of(b, h)), n_kv,
                              R.default_scale(hd), "bf16", W_EPS, f"call {i}", R.Q_EPS[fmt])
    assert g.device_error() == 0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_a_large_v_row_beside_nan(g, fmt, hd):
    """V rows far apart with a NaN in one head's q, or in one KV head's V: the other heads keep the
    f64 bound, those are NaN."""
    rng = np.random.default_rng(104)
    n_q, n_kv, lens = 8, 2, [900, 70]
    rs = [None, np.where(rng.random((2, n_kv, 903)) < 0.02, 2.0 ** 40, 1.0)]
    q, qf, cache, kv_of, max_seq = _decode_case(rng, lens, n_q, n_kv, hd, fmt, "bf16", rs)
    x = qf.copy()
    x[0, 2, 5] = np.nan
    cache[3][1, 1, 33] = np.nan
    out = _run_decode(g, O.from_f32(x.astype(np.float32).ravel()), cache, lens, n_q, n_kv, hd, max_seq, fmt,
                      "bf16").view(2, n_q, hd)
    assert bool(out[0, 2].isnan().all()) and bool(out[1, 4:].isnan().all())
    keep = {0: [0, 1, 3, 4, 5, 6, 7], 1: [0, 1, 2, 3]}
    for b, heads in keep.items():
        for h in heads:
            R.check_attention(out[b:b + 1, h].contiguous(), qf[b:b + 1, h:h + 1],
                              lambda _, __: kv_of(b, h // 4), 1, R.default_scale(hd), "bf16", W_EPS,
                              f"sequence {b} head {h}", R.Q_EPS[fmt])
    assert g.device_error() == 0
