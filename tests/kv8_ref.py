"""Plain restatements of the 8-bit KV cache and of decode attention in 64 bits, for the
tests: the row quantisation in numpy's f32 (the definition, bit for bit) and attention in
f64 with the bound that its f32 / 16-bit evaluation has to stay within."""
import math

import numpy as np
import torch

TOP = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TDT = {"bf16": torch.bfloat16, "f16": torch.float16}
TINY = np.float32(2.0 ** -119)


def quantise(x, fmt):
    """f32 rows [..., hd] -> (code bytes as int8 bit patterns, f32 scales)."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        amax = np.abs(x).max(-1)
        bad = ~np.isfinite(x).all(-1)
        zero = ~bad & (amax < TINY)
        one = np.where(bad | zero, np.float32(1), amax)
        top = np.float32(TOP[fmt])
        y = x * (top / one)[..., None]
        scale = np.where(bad, np.float32(np.nan), np.where(zero, np.float32(0), one / top))
        y = np.where((bad | zero)[..., None], np.float32(0), y)
    if fmt == "int8":
        codes = np.rint(y).astype(np.int8)
    else:
        codes = torch.from_numpy(np.ascontiguousarray(y)).to(torch.float8_e4m3fn).view(
            torch.int8).numpy()
    return codes, scale.astype(np.float32)


def values(codes, fmt):
    """The numbers that code bytes (int8 patterns) stand for, without their scale, f64."""
    t = torch.from_numpy(np.ascontiguousarray(codes))
    return t.view(CODE[fmt]).to(torch.float32).numpy().astype(np.float64)


def cache(rng, lead, rows, hd, fmt, row_scale=None):
    """Codes (int8 patterns) and scales of unit normal rows."""
    x = rng.normal(0, 1, (*lead, rows, hd)).astype(np.float32)
    if row_scale is not None:
        x *= row_scale[..., None].astype(np.float32)
    return quantise(x, fmt)


def to_dev(codes, fmt):
    return torch.from_numpy(np.ascontiguousarray(codes)).cuda().view(CODE[fmt])


def page(rng, x, block, spare=3, table=None):
    """[n_seq, n_kv, rows, ...] -> (pool [n_blocks, n_kv, block, ...], table): rows padded to
    whole blocks, blocks scattered, unused blocks filled with a pattern."""
    n_seq, n_kv, rows = x.shape[:3]
    per = -(-rows // block)
    if table is None:
        table = rng.permutation(n_seq * per + spare)[:n_seq * per].reshape(n_seq, per).astype(np.int32)
    pool = np.zeros((n_seq * per + spare, n_kv, block, *x.shape[3:]), x.dtype)
    pool[:] = 0x7F if x.dtype == np.int8 else np.nan if x.dtype.kind == "f" else 0x7FFF
    for b in range(n_seq):
        for i in range(per):
            part = x[b, :, i * block:(i + 1) * block]
            pool[table[b, i], :, :part.shape[1]] = part
    return pool, table


def attention(q, k, v, scale):
    """One KV head in f64: q [G, hd], k and v [n, hd] -> (out [G, hd], sum_k p_k |v_k|,
    the largest sum_d |q_d k_d| * scale of each row, the largest |q_d| sum_d |k_d| * scale).
    No keys: zeros."""
    if k.shape[0] == 0:
        z = np.zeros(q.shape)
        return z, z, np.zeros(q.shape[0]), np.zeros(q.shape[0])
    s = q @ k.T * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return (p @ v, p @ np.abs(v), (np.abs(q) @ np.abs(k).T * scale).max(-1),
            np.abs(q).max(-1) * np.abs(k).sum(-1).max() * scale)


# An int8 cache's scores use Q as 16-bit integers, 32639 for a head's largest element: each
# element is off by at most half an integer (and the f32 steps of the scaling).
Q_EPS = {"int8": 0.5 / 32639 * (1 + 2.0 ** -6), "e4m3": 0.0}


def check_attention(got, q, kv_of, n_kv, scale, dtype, weight_eps, name="", q_eps=0.0):
    """got [n_seq, n_q * hd] (16-bit) against f64; kv_of(b, h) -> (k, v) rows in f64.

    Bound per element, o the exact value and A = sum_k p_k |v_k|:
      half a step of the output type            eps / 2 * |o|  (and its smallest step)
      weights rounded to weight_eps each        weight_eps * A
      scores summed in f32 over hd terms: each off by d <= (hd + 4) 2^-24 max_k sum|q k| scale,
        which moves a normalised weight by at most exp(2 d) - 1; d also has q_eps max |q| sum |k|
        scale for elements of q that are each off by q_eps of the head's largest
      exp and the sums over up to 2^11 terms in a row: 2^-13 * A
    """
    n_seq, hd = q.shape[0], q.shape[-1]
    group = q.shape[1] // n_kv
    fin = torch.finfo(TDT[dtype])
    got = got.float().cpu().numpy().astype(np.float64).reshape(n_seq, n_kv, group, hd)
    worst = 0.0
    for b in range(n_seq):
        for h in range(n_kv):
            k, v = kv_of(b, h)
            o, A, s, s_max = attention(q[b, h * group:(h + 1) * group], k, v, scale)
            d = (hd + 4) * 2.0 ** -24 * s[:, None] + q_eps * s_max[:, None]
            tol = fin.eps / 2 * np.abs(o) + fin.smallest_normal * fin.eps + A * (
                weight_eps + np.expm1(2 * d) + 2.0 ** -13)
            err = np.abs(got[b, h] - o)
            bad = ~(err <= tol)
            assert not bad.any(), (f"{name} sequence {b} head {h} keys {k.shape[0]}: {bad.sum()} of "
                                   f"{bad.size} off, worst {np.nanmax(err / np.maximum(tol, 1e-300)):.3g} x bound")
            worst = max(worst, float(np.max(err / np.maximum(tol, 1e-300))))
    return worst


def default_scale(hd):
    return 1.0 / math.sqrt(hd)
