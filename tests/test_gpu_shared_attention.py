"""Decode attention of sequences that share a prefix, contiguous and paged, against f64."""
import numpy as np
import pytest
import torch

import kv8_ref as R
from gpu_util import dev, normal16
from oracle import oracle as O

pytestmark = pytest.mark.gpu

# Weights of the softmax: head + remainder in bf16 (16 bits: 2^-15 with the truncated head),
# one f16 for f16 inputs (half a step, 2^-11).
W_EPS = {"bf16": 2.0 ** -15, "f16": 2.0 ** -11}


@pytest.fixture(scope="module")
def g():
    from kvasir_b200 import Gpu
    return Gpu(0)


def _f64(bits, dtype, *shape):
    return O.to_f32(bits, dtype).astype(np.float64).reshape(shape)


class Case:
    """Prefix rows [n_kv, P, hd], own rows [n_seq, n_kv, own_max, hd], as bits and f64."""

    def __init__(self, rng, prefix, lens, n_q, n_kv, hd, dtype, q_std=1.0):
        self.prefix, self.lens, self.n_q, self.n_kv, self.hd, self.dtype = prefix, lens, n_q, n_kv, hd, dtype
        self.n_seq, self.max_seq = len(lens), max(lens) + 5
        nan = 0x7FFF
        self.q = normal16(rng, self.n_seq * n_q * hd, std=q_std, dtype=dtype)
        self.rows = prefix + 3  # rows past the prefix hold garbage
        self.pk, self.pv = (normal16(rng, n_kv * self.rows * hd, dtype=dtype).reshape(n_kv, self.rows, hd)
                            for _ in range(2))
        self.kc, self.vc = (normal16(rng, self.n_seq * n_kv * self.max_seq * hd, dtype=dtype).reshape(
            self.n_seq, n_kv, self.max_seq, hd) for _ in range(2))
        self.qf = _f64(self.q, dtype, self.n_seq, n_q, hd)
        self.f = [_f64(x.ravel(), dtype, *x.shape) for x in (self.pk, self.pv, self.kc, self.vc)]
        for x in (self.pk, self.pv):
            x[:, prefix:] = nan
        for x in (self.kc, self.vc):
            for b, n in enumerate(lens):
                x[b, :, n:] = nan
        self.ld = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def kv_of(self, b, h):
        p, n = self.prefix, self.lens[b]
        return tuple(np.concatenate([self.f[i][h, :p], self.f[i + 2][b, h, :n]]) for i in (0, 1))

    def out(self):
        return torch.full((self.n_seq, self.n_q * self.hd), 9.0, dtype=R.TDT[self.dtype], device="cuda")

    def ws(self, g, own):
        n = g.attention_decode_shared_workspace_bytes(self.n_seq, self.prefix, own, self.n_q, self.n_kv,
                                                      self.hd)
        return torch.empty(max(16, n), dtype=torch.uint8, device="cuda")

    def contiguous(self, g, workspace=True):
        d, out = self.dtype, self.out()
        g.attention_decode_shared(dev(self.q, d), self.n_q * self.hd, dev(self.pk, d), dev(self.pv, d),
                                  self.prefix, self.rows, dev(self.kc, d), dev(self.vc, d),
                                  self.n_kv * self.max_seq * self.hd, self.ld, max(self.lens), self.n_q,
                                  self.n_kv, self.hd, self.max_seq, out, self.n_q * self.hd,
                                  workspace=self.ws(g, max(self.lens)) if workspace else None)
        return out

    def pools(self, block, seed=3):
        """One pool: the prefix's whole blocks once, the rest of each sequence by itself."""
        whole = self.prefix // block
        total = self.prefix + self.max_seq
        per = -(-total // block)
        rng = np.random.default_rng(seed)
        n_blocks = whole + self.n_seq * (per - whole) + 3
        ids = rng.permutation(n_blocks).astype(np.int32)
        table = np.empty((self.n_seq, per), np.int32)
        table[:, :whole] = ids[:whole]
        table[:, whole:] = ids[whole:whole + self.n_seq * (per - whole)].reshape(self.n_seq, -1)
        pools = []
        for p, own in ((self.pk, self.kc), (self.pv, self.vc)):
            pool = np.full((n_blocks, self.n_kv, block, self.hd), 0x7FFF, np.uint16)
            for b in range(self.n_seq):
                x = np.full((self.n_kv, per * block, self.hd), 0x7FFF, np.uint16)
                x[:, :self.prefix] = p[:, :self.prefix]
                x[:, self.prefix:total] = own[b]
                for i in range(per):
                    pool[table[b, i]] = x[:, i * block:(i + 1) * block]
            pools.append(pool)
        for b, n in enumerate(self.lens):
            table[b, -(-(self.prefix + n) // block):] = -1
        return pools, table

    def paged(self, g, block, workspace=True):
        d, out = self.dtype, self.out()
        (kp, vp), table = self.pools(block)
        g.attention_decode_shared_paged(dev(self.q, d), self.n_q * self.hd, dev(kp, d), dev(vp, d),
                                        torch.from_numpy(table).cuda(), table.shape[1], block,
                                        self.prefix, self.ld + self.prefix,
                                        self.prefix + max(self.lens), self.n_q, self.n_kv, self.hd, out,
                                        self.n_q * self.hd,
                                        workspace=self.ws(g, max(self.lens)) if workspace else None)
        return out

    def check(self, out, name=""):
        R.check_attention(out, self.qf, self.kv_of, self.n_kv, R.default_scale(self.hd), self.dtype,
                          W_EPS[self.dtype], name)


@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 65, 96, 300, 1000])
@pytest.mark.parametrize("n_q,n_kv,hd", [(32, 8, 64), (4, 4, 64), (6, 2, 64), (14, 2, 64), (16, 1, 64),
                                         (20, 1, 64), (4, 2, 128), (4, 2, 80)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_against_f64(g, prefix, n_q, n_kv, hd, dtype):
    c = Case(np.random.default_rng(prefix + n_q), prefix, [1, 0, 64, 65, 200, 31, 7], n_q, n_kv, hd, dtype)
    for ws in (True, False):
        c.check(c.contiguous(g, ws), "contiguous")
        c.check(c.paged(g, 64, ws), "paged")
    assert g.device_error() == 0


@pytest.mark.parametrize("n_seq", [1, 2, 31, 32, 33, 64, 100])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_batch_sizes(g, n_seq, dtype):
    """Row tiles with one row left over, filled exactly, and less than one."""
    rng = np.random.default_rng(n_seq)
    c = Case(rng, 700, [int(x) for x in rng.integers(0, 90, n_seq)] or [1], 8, 2, 64, dtype)
    c.check(c.contiguous(g), "contiguous")
    c.check(c.paged(g, 128), "paged")
    assert g.device_error() == 0


@pytest.mark.parametrize("block", [8, 16, 32, 64, 96, 256])
def test_block_sizes(g, block):
    c = Case(np.random.default_rng(block), 515, [1, 100, 40], 8, 2, 64, "bf16")
    c.check(c.paged(g, block))
    assert g.device_error() == 0


def test_long_prefix_and_peaked_rows(g):
    """Keys split over CTAs and joined; large scores (a few keys take all the weight)."""
    for q_std, dtype in ((1.0, "bf16"), (6.0, "bf16"), (6.0, "f16")):
        c = Case(np.random.default_rng(5), 9000, [500, 0, 3, 1500], 8, 2, 64, dtype, q_std)
        out = c.contiguous(g)
        c.check(out)
        assert torch.equal(out, c.contiguous(g))
        paged = c.paged(g, 64)
        c.check(paged)
        assert torch.equal(paged, c.paged(g, 64))
    assert g.device_error() == 0


def test_empty_rows(g):
    """No prefix and no keys: zeros."""
    c = Case(np.random.default_rng(6), 0, [0, 5, 0], 8, 2, 64, "bf16")
    for out in (c.contiguous(g), c.paged(g, 64)):
        assert bool((out[[0, 2]] == 0).all())
        c.check(out)


def test_no_keys_at_all(g):
    """No prefix and max_len 0, with and without a workspace: zeros, and no report although the
    lengths are written right before the call."""
    c = Case(np.random.default_rng(6), 0, [0, 0, 0], 8, 2, 64, "bf16")
    for ws in (True, False):
        c.ld.fill_(7)
        c.ld.zero_()
        assert bool((c.contiguous(g, ws) == 0).all())
    assert g.device_error() == 0


@pytest.mark.parametrize("hd", [64, 80])
def test_paged_lengths_below_the_prefix(g, hd):
    """A sequence shorter than shared_len attends to its own first keys only; 0 gives zeros."""
    c = Case(np.random.default_rng(7), 300, [10, 20, 30, 40], 8, 2, hd, "bf16")
    (kp, vp), table = c.pools(64)
    short = [0, 1, 130, 299]
    out = c.out()
    g.attention_decode_shared_paged(dev(c.q), c.n_q * hd, dev(kp), dev(vp), torch.from_numpy(table).cuda(),
                                    table.shape[1], 64, 300,
                                    torch.tensor(short, dtype=torch.int32, device="cuda"), 340, c.n_q,
                                    c.n_kv, hd, out, c.n_q * hd, workspace=c.ws(g, 40))
    assert g.device_error() == 0
    R.check_attention(out, c.qf, lambda b, h: (c.f[0][h, :short[b]], c.f[1][h, :short[b]]), c.n_kv,
                      R.default_scale(hd), "bf16", W_EPS["bf16"])
    assert bool((out[0] == 0).all())


@pytest.mark.parametrize("hd", [64, 80])
def test_bad_lengths_and_blocks_are_reported(g, hd):
    c = Case(np.random.default_rng(8), 128, [64, 64, 64], 4, 1, hd, "bf16")
    good = c.contiguous(g)
    c.ld = torch.tensor([-1, 64, 70], dtype=torch.int32, device="cuda")
    out = c.contiguous(g)
    assert g.device_error() == 2
    assert torch.equal(out[1:], good[1:])
    R.check_attention(out[:1], c.qf[:1], lambda b, h: (c.f[0][h, :128], c.f[1][h, :128]), c.n_kv,
                      R.default_scale(hd), "bf16", W_EPS["bf16"])
    # paged: a bad entry among the prefix's and one among a sequence's own
    (kp, vp), table = c.pools(64)
    table[0, 1], table[2, 2] = kp.shape[0], -7
    out = c.out()
    g.attention_decode_shared_paged(dev(c.q), c.n_q * hd, dev(kp), dev(vp), torch.from_numpy(table).cuda(),
                                    table.shape[1], 64, 128,
                                    torch.full((3,), 192, dtype=torch.int32, device="cuda"), 192, c.n_q,
                                    c.n_kv, hd, out, c.n_q * hd, workspace=c.ws(g, 64))
    assert g.device_error() == 4

    def zeroed(b, h):
        k, v = c.kv_of(b, h)
        k[64:128], v[64:128] = 0, 0
        if b == 2:
            k[128:], v[128:] = 0, 0
        return k, v
    R.check_attention(out, c.qf, zeroed, c.n_kv, R.default_scale(hd), "bf16", W_EPS["bf16"])


def test_equals_decode_over_the_same_keys(g):
    """attention_decode on caches that hold prefix and own keys together, to the bound twice."""
    c = Case(np.random.default_rng(12), 320, [100, 50, 1, 200], 32, 8, 64, "bf16")
    shared = c.contiguous(g)
    max_seq = 320 + c.max_seq
    k, v = (np.concatenate([np.broadcast_to(p[None, :, :320], (4, 8, 320, 64)), own], 2)
            for p, own in ((c.pk, c.kc), (c.pv, c.vc)))
    out = c.out()
    g.attention_decode(dev(c.q), 32 * 64, dev(k), dev(v), 8 * max_seq * 64, c.ld + 320, 520, 32, 8, 64,
                       max_seq, out, 32 * 64)
    c.check(shared)
    c.check(out)


@pytest.mark.parametrize("hd", [64, 80])
def test_strides_graph_and_stream(g, hd):
    from kvasir_b200 import Gpu
    c = Case(np.random.default_rng(13), 500, [70, 3, 64], 8, 2, hd, "bf16")
    want = c.contiguous(g)
    n_q = c.n_q
    qs, os_ = (n_q + 2 * c.n_kv) * hd, n_q * hd + 8
    q = torch.full((3, qs), float("nan"), dtype=torch.bfloat16, device="cuda")
    q[:, :n_q * hd] = dev(c.q).view(3, -1)
    out = torch.full((3, os_), 7.0, dtype=torch.bfloat16, device="cuda")
    s = torch.cuda.Stream()
    gs = Gpu(0, stream=s)
    pk, pv, kc, vc, ws = dev(c.pk), dev(c.pv), dev(c.kc), dev(c.vc), c.ws(g, 70)

    def call():
        gs.attention_decode_shared(q, qs, pk, pv, 500, c.rows, kc, vc, c.n_kv * c.max_seq * hd, c.ld, 70,
                                   n_q, c.n_kv, hd, c.max_seq, out, os_, workspace=ws)
    torch.cuda.synchronize()
    call()
    s.synchronize()
    assert torch.equal(out[:, :n_q * hd], want) and bool((out[:, n_q * hd:] == 7.0).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        call()
    for _ in range(2):
        out.fill_(1.0)
        ws.fill_(255)  # what an earlier call left in the workspace does not matter
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:, :n_q * hd], want) and bool((out[:, n_q * hd:] == 1.0).all())
    assert g.device_error() == 0


def test_two_streams_at_once_and_negative_scale(g):
    from kvasir_b200 import Gpu
    jobs = []
    for seed, prefix, lens in ((1, 900, [70, 3, 640]), (2, 2000, [1, 0, 200])):
        c = Case(np.random.default_rng(seed), prefix, lens, 32, 8, 64, "bf16")
        want = c.contiguous(g)
        h = Gpu(0, stream=torch.cuda.Stream())
        t = [dev(x) for x in (c.q, c.pk, c.pv, c.kc, c.vc)]
        jobs.append((c, h, t, want, c.ws(g, max(lens))))
    outs = [[torch.empty_like(j[3]) for _ in range(10)] for j in jobs]
    torch.cuda.synchronize()
    for i in range(10):
        for (c, h, (q, pk, pv, kc, vc), _, ws), o in zip(jobs, outs):
            h.attention_decode_shared(q, 2048, pk, pv, c.prefix, c.rows, kc, vc, 8 * c.max_seq * 64, c.ld,
                                      max(c.lens), 32, 8, 64, c.max_seq, o[i], 2048, workspace=ws)
    torch.cuda.synchronize()
    for (c, *_, want, _), o in zip(jobs, outs):
        assert all(torch.equal(x, want) for x in o)
    c, _, (q, pk, pv, kc, vc), _, ws = jobs[0]
    for scale in (-0.125, 0.0):
        out = c.out()
        g.attention_decode_shared(q, 2048, pk, pv, c.prefix, c.rows, kc, vc, 8 * c.max_seq * 64, c.ld,
                                  max(c.lens), 32, 8, 64, c.max_seq, out, 2048, scale=scale, workspace=ws)
        # scores of -scale against -q are those of scale against q
        R.check_attention(out, c.qf * (-1 if scale < 0 else 1), c.kv_of, 8, abs(scale), "bf16",
                          W_EPS["bf16"])
    assert g.device_error() == 0


@pytest.mark.parametrize("n_q,n_kv", [(8, 8), (21, 3), (26, 2), (16, 1)])
def test_groups_that_do_not_fill_a_tile(g, n_q, n_kv):
    """Group sizes 1, 7, 13 and 16 over enough sequences for several CTAs of row tiles."""
    rng = np.random.default_rng(n_q)
    c = Case(rng, 200, [int(x) for x in rng.integers(0, 70, 300)], n_q, n_kv, 64, "bf16")
    c.check(c.contiguous(g))
    c.check(c.paged(g, 64))
    assert g.device_error() == 0


@pytest.mark.parametrize("hd", [64, 80])
def test_rows_past_32_bit_offsets(g, hd):
    """Own keys more than 2^32 elements apart, contiguous and in blocks of a pool: as on a small
    cache, bit for bit."""
    n_q, n_kv, prefix, own, block = 8, 2, 128, 128, 64
    rng = np.random.default_rng(61)
    q = dev(normal16(rng, 2 * n_q * hd)).view(2, -1)
    rows = [dev(normal16(rng, n_kv * n * hd)).view(n_kv, n, hd) for n in (prefix, prefix, own, own, own, own)]
    pk, pv, own_kv = rows[0], rows[1], (rows[2:4], rows[4:6])
    lens = torch.tensor([100, 77], dtype=torch.int32, device="cuda")
    ws = torch.empty(max(16, g.attention_decode_shared_workspace_bytes(2, prefix, own, n_q, n_kv, hd)),
                     dtype=torch.uint8, device="cuda")
    per, per_block = n_kv * own * hd, n_kv * block * hd

    def contiguous(stride):
        out = torch.empty(2, n_q * hd, dtype=torch.bfloat16, device="cuda")
        kc, vc = (torch.empty(stride + per, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        for b in (0, 1):
            for x, r in zip((kc, vc), own_kv[b]):
                x[b * stride:b * stride + per].view(n_kv, own, hd).copy_(r)
        g.attention_decode_shared(q, n_q * hd, pk, pv, prefix, prefix, kc, vc, stride, lens, 100, n_q, n_kv,
                                  hd, own, out, n_q * hd, workspace=ws)
        assert g.device_error() == 0
        return out

    def paged(n_blocks):
        out = torch.empty(2, n_q * hd, dtype=torch.bfloat16, device="cuda")
        kp, vp = (torch.empty(n_blocks, n_kv, block, hd, dtype=torch.bfloat16, device="cuda")
                  for _ in range(2))
        last = n_blocks - 1  # the prefix: the first and the last block; own keys: near both ends
        table = torch.tensor([[0, last, 1, last - 1], [0, last, 2, last - 2]], dtype=torch.int32)
        for x, p, i in ((kp, pk, 0), (vp, pv, 1)):
            for j in (0, 1):
                x[table[0, j]] = p[:, j * block:(j + 1) * block]
                for b in (0, 1):
                    x[table[b, 2 + j]] = own_kv[b][i][:, j * block:(j + 1) * block]
        g.attention_decode_shared_paged(q, n_q * hd, kp, vp, table.cuda(), 4, block, prefix, lens + prefix,
                                        prefix + 100, n_q, n_kv, hd, out, n_q * hd, workspace=ws)
        assert g.device_error() == 0
        return out

    assert torch.equal(contiguous((2 ** 32 // hd + 3) * hd), contiguous(per))
    assert torch.equal(paged(2 ** 32 // per_block + 9), paged(8))


@pytest.mark.parametrize("parts", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("paged", [False, True])
def test_smaller_workspaces(g, parts, paged):
    """A workspace of fewer parts than the call would take: fewer slices and longer chunks, the same
    attention; nothing behind the workspace is written.  Too small for one part of each: the
    general kernel."""
    c = Case(np.random.default_rng(71), 5000, [1500, 0, 700, 3, 64], 8, 2, 64, "bf16")
    part = (4 * (64 + 2) + 3) // 4 * 4 * 4  # bytes of O, m, l of a group of 4 heads
    n = c.n_seq * c.n_kv * parts * part
    assert n < g.attention_decode_shared_workspace_bytes(c.n_seq, c.prefix, 1500, 8, 2, 64)
    whole = torch.full((n + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    c.ws = lambda *_: whole[:n]
    c.check(c.paged(g, 64) if paged else c.contiguous(g))
    assert bool((whole[n:] == 0xA5).all())
    assert g.device_error() == 0


@pytest.mark.parametrize("prefix,max_len", [(256, 256), (300, 340), (300, 150), (5000, 5003)])
@pytest.mark.parametrize("n_seq", [5, 40, 80])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_paged_lengths_below_the_prefix_ignore_later_values(g, prefix, max_len, n_seq, dtype):
    """NaN and infinities in V (and NaN in K) past a sequence's length do not reach it, wherever in
    the prefix it ends, with one, two and four row tiles to a CTA, and with the general kernel;
    the sequences that attend to such a V row are NaN."""
    rng = np.random.default_rng(prefix + n_seq)
    c = Case(rng, prefix, [40] * n_seq, 8, 2, 64, dtype)
    bad = prefix // 2 + 3  # in the middle of a tile
    (kp, vp), table = c.pools(64)
    blk, at = table[0, bad // 64], bad % 64
    vp[blk, :, at] = 0x7FFF
    if bad + 30 < prefix:
        vp[table[0, (bad + 30) // 64], :, (bad + 30) % 64] = 0x7F80 if dtype == "bf16" else 0x7C00
    last = table[0, prefix // 64 - 1]
    kp[last, :, 63] = 0x7FFF  # the last key of the prefix's last whole tile
    short = [0, 1, 63, 64, 65, bad - 1, bad, bad + 1, prefix // 64 * 64 - 1, max_len]
    short = [min(short[3 * i % len(short)], max_len) for i in range(n_seq)]
    clean = [i for i, n in enumerate(short) if n <= bad]
    lens = torch.tensor(short, dtype=torch.int32, device="cuda")
    for ws in (c.ws(g, max(max_len - prefix, 0)), None):
        out = c.out()
        g.attention_decode_shared_paged(dev(c.q, dtype), 512, dev(kp, dtype), dev(vp, dtype),
                                        torch.from_numpy(table).cuda(), table.shape[1], 64, prefix, lens,
                                        max_len, 8, 2, 64, out, 512, workspace=ws)
        assert g.device_error() == 0
        R.check_attention(out[clean], c.qf[clean],
                          lambda i, h: (c.f[0][h, :short[clean[i]]], c.f[1][h, :short[clean[i]]]), c.n_kv,
                          R.default_scale(64), dtype, W_EPS[dtype])
        rest = [i for i in range(n_seq) if i not in clean]
        assert bool(out[rest].isnan().all())


def test_f16_weights_far_below_the_largest(g):
    """One key 17 above 16384 others whose V rows have one sign, in a single slice of the prefix.
    A weight is one f16 of at most 2^15 (the reference is within 2^8 of the row's maximum, and
    here equals it): half a step is 2^-11 of the weight, or 2^-25 below 2^-14, which is 2^-32 of
    the largest weight for each key.  Scores: multiples of 1/8, exact."""
    n_q, n_kv, hd, n = 4, 2, 64, 16384
    q = np.zeros((1, n_q, hd), np.float32)
    q[:, :, 0] = 17.0
    k = np.zeros((n_kv, n, hd), np.float32)
    k[:, 0, 0] = 8.0
    v = np.abs(np.random.default_rng(81).normal(1.0, 0.1, (n_kv, n, hd))).astype(np.float32)
    v[:, 0] = 0.0
    qb, kb, vb = (O.from_f32(x.ravel(), "f16") for x in (q, k, v))
    vf = _f64(vb, "f16", n_kv, n, hd)
    own = torch.zeros(1, n_kv, 1, hd, dtype=torch.float16, device="cuda")
    out = torch.empty(1, n_q * hd, dtype=torch.float16, device="cuda")
    ws = torch.empty(n_kv * 2 * (hd + 2) * 4, dtype=torch.uint8, device="cuda")  # one part: O, m, l
    g.attention_decode_shared(dev(qb, "f16"), n_q * hd, dev(kb, "f16").view(n_kv, n, hd),
                              dev(vb, "f16").view(n_kv, n, hd), n, n, own, own, n_kv * hd,
                              torch.zeros(1, dtype=torch.int32, device="cuda"), 0, n_q, n_kv, hd, 1, out,
                              n_q * hd, workspace=ws)
    p = np.full(n, np.exp(-17.0))
    p[0] = 1.0
    p /= p.sum()
    want = np.stack([p @ vf[h // 2] for h in range(n_q)])
    A = want  # all terms have one sign
    tol = (2.0 ** -11 + 2.0 ** -11 + 2.0 ** -13 + np.expm1(2 * 68 * 2.0 ** -24 * 17)) * A + \
        2.0 ** -32 * np.abs(vf).sum(1)[[h // 2 for h in range(n_q)]]
    err = np.abs(out.float().cpu().numpy().astype(np.float64).reshape(n_q, hd) - want)
    assert np.all(err <= tol), np.max(err / tol)
    assert g.device_error() == 0


@pytest.mark.parametrize("hd", [64, 80])
def test_scores_of_minus_infinity(g, hd):
    """Keys whose scores are all -infinity have no weight beside others, in the prefix or among a
    sequence's own; a row that has keys and no other scores is NaN, one without keys zeros; the
    same with and without a workspace."""
    rng = np.random.default_rng(91)
    for prefix, own, inf_prefix, inf_own in ((300, 200, 300, 200), (300, 200, 300, 0), (300, 200, 0, 200),
                                             (300, 200, 64, 70), (0, 200, 0, 200), (0, 200, 0, 130)):
        c = Case(rng, prefix, [own, 0, own - 3], 8, 2, hd, "bf16")
        c.q = O.from_f32(np.abs(O.to_f32(c.q)) + np.float32(0.5))
        c.qf = _f64(c.q, "bf16", 3, 8, hd)
        c.pk[:, :inf_prefix] = c.kc[:, :, :inf_own] = 0xFF80
        want = c.qf * 0
        for b in range(3):
            n = c.lens[b]
            for h in range(2):
                k = np.concatenate([c.f[0][h, inf_prefix:prefix], c.f[2][b, h, min(inf_own, n):n]])
                v = np.concatenate([c.f[1][h, inf_prefix:prefix], c.f[3][b, h, min(inf_own, n):n]])
                want[b, 4 * h:4 * h + 4] = R.attention(c.qf[b, 4 * h:4 * h + 4], k, v,
                                                       R.default_scale(hd))[0] if len(k) else \
                    (np.nan if prefix + n else 0.0)
        for ws in (True, False):
            for out in (c.contiguous(g, ws), c.paged(g, 64, ws)):
                got = out.float().cpu().numpy().reshape(want.shape)
                # half a bf16 step is 2^-8 of a value; the averages of unit normals here are below 4, and the
                # weights (2^-15 of each) and f32 sums far below 2^-8
                np.testing.assert_allclose(got, want, rtol=2.0 ** -8, atol=2.0 ** -8, equal_nan=True)
    assert g.device_error() == 0


def test_paged_over_a_pool_without_blocks(g):
    """Sequences of length 0 on an empty pool: zero rows; longer ones are reported (their keys read
    as zeros)."""
    import ctypes as C
    one = torch.zeros(64, device="cuda")  # never read
    q = torch.ones(2, 512, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(2, dtype=torch.int32, device="cuda")
    n = g.attention_decode_shared_workspace_bytes(2, 64, 0, 8, 2, 64)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    for length, err in ((0, 0), (64, 4)):
        lens = torch.full((2,), length, dtype=torch.int32, device="cuda")
        out = torch.ones(2, 512, dtype=torch.bfloat16, device="cuda")
        st = g._lib.kvb_attention_decode_shared_paged(
            C.c_void_p(g.stream.cuda_stream), p(q), 512, p(one), p(one), 0, p(table), 1, 64, 64, p(lens), 2,
            64, 8, 2, 64, 0.125, p(out), 512, p(ws), n, 0)
        assert st == 0
        assert g.device_error() == err
        assert bool((out == 0).all())


@pytest.mark.parametrize("paged", [False, True])
def test_inputs_rewritten_between_captured_calls(g, paged):
    """Several calls in one graph, q, lengths and block table rewritten on the stream before each:
    every call reads what was written last, although its launches start before their own waits."""
    from kvasir_b200 import Gpu
    rng = np.random.default_rng(101)
    cases = [Case(rng, 640, [int(n) for n in rng.integers(0, 300, 6)], 8, 2, 64, "bf16") for _ in range(4)]
    c0 = cases[0]
    for c in cases:  # the same caches for all
        c.pk, c.pv, c.kc, c.vc, c.f, c.max_seq, c.rows = c0.pk, c0.pv, c0.kc, c0.vc, c0.f, c0.max_seq, c0.rows
        c.lens = [min(n, m) for n, m in zip(c.lens, c0.lens)]
        c.ld = torch.tensor(c.lens, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    gs = Gpu(0, stream=s)
    n = max(c0.lens)
    (kp, vp), table = c0.pools(64)
    kp, vp, pk, pv, kc, vc = (dev(x) for x in (kp, vp, c0.pk, c0.pv, c0.kc, c0.vc))
    # every call's table: the sequences' rows in another order, their lengths and q with them
    orders = [np.roll(np.arange(6), i) for i in range(4)]
    tables = [torch.from_numpy(table[o]).cuda() for o in orders]
    for t in tables:  # row 0 holds the prefix in every order
        assert torch.equal(t[0, :10], t[1, :10])
    order = (lambda i: torch.from_numpy(orders[i]).cuda()) if paged else (lambda i: torch.arange(6).cuda())
    qs = [dev(c.q).view(6, 512)[order(i)].contiguous() for i, c in enumerate(cases)]
    lens = [(c.ld + (640 if paged else 0))[order(i)].contiguous() for i, c in enumerate(cases)]
    q, ld, tab = torch.empty_like(qs[0]), torch.empty_like(lens[0]), torch.empty_like(tables[0])
    outs, ws = [c.out() for c in cases], c0.ws(g, n)

    def calls():
        for i in range(4):
            q.copy_(qs[i])
            ld.copy_(lens[i])
            tab.copy_(tables[i])
            if paged:
                gs.attention_decode_shared_paged(q, 512, kp, vp, tab, tab.shape[1], 64, 640, ld, 640 + n, 8, 2,
                                                 64, outs[i], 512, workspace=ws)
            else:
                gs.attention_decode_shared(q, 512, pk, pv, 640, c0.rows, kc, vc, 2 * c0.max_seq * 64, ld, n, 8,
                                           2, 64, c0.max_seq, outs[i], 512, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        calls()
    for _ in range(5):
        for o in outs:
            o.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, c in enumerate(cases):
            got = torch.empty_like(outs[i])
            got[order(i)] = outs[i]
            c.check(got, f"call {i}")
    assert g.device_error() == 0
