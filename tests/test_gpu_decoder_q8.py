"""The decode-step driver on an 8-bit KV cache: the step is the composition of the Gpu calls,
bit for bit, and the cache halves without moving the logits further than its codes do."""
import numpy as np
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu


def _cfg(head_dim=64, heads=8, kv=2):
    from kvasir_b200.config import LlamaConfig
    return LlamaConfig(hidden_size=512, intermediate_size=512, num_layers=2, num_heads=heads,
                       num_kv_heads=kv, head_dim=head_dim, vocab_size=1000, rms_norm_eps=1e-5,
                       rope_theta=500000.0, max_position_embeddings=4096)


def _step(g, dec, ids, pos, block):
    """One step through the Gpu methods, on the decoder's own weights, tables and cache clones."""
    cfg, w, n = dec.cfg, dec.w, dec.n_seq
    H, I, nq, nkv, hd = (cfg.hidden_size, cfg.intermediate_size, cfg.num_heads, cfg.num_kv_heads,
                         cfg.head_dim)
    e = lambda *s: torch.empty(*s, dtype=dec.dtype, device="cuda")  # noqa: E731
    x, h, qkv, attn, o, act = e(n, H), e(n, H), e(n, cfg.qkv_dim), e(n, cfg.q_dim), e(n, H), e(n, I)
    lens, max_seq = pos + 1, dec.max_seq
    ws = torch.empty(max(16, g.attention_decode_q8_workspace_bytes(n, max_seq, nq, nkv, hd)),
                     dtype=torch.uint8, device="cuda")
    g.embedding_rmsnorm(ids, w["embed"], w["attn_norm"][0], x, h, H, cfg.rms_norm_eps)
    for l in range(cfg.num_layers):
        g.linear_rows(h, w["w_qkv"][l], qkv, n, H, cfg.qkv_dim)
        kc, vc, ks, vs = dec.kc[l], dec.vc[l], dec.ks[l], dec.vs[l]
        if block:
            mb = dec.block_table.shape[1]
            g.rope_kv_append_q8_paged(qkv, n, 1, pos, dec.cos, dec.sin, kc, vc, ks, vs,
                                      dec.block_table, mb, block, nq, nkv, hd)
            g.attention_decode_q8_paged(qkv, cfg.qkv_dim, kc, vc, ks, vs, dec.block_table, mb, block,
                                        lens, max_seq, nq, nkv, hd, attn, cfg.q_dim, workspace=ws)
        else:
            stride = nkv * max_seq * hd
            g.rope_kv_append_q8(qkv, n, 1, pos, dec.cos, dec.sin, kc, vc, ks, vs, stride, nq, nkv, hd,
                                max_seq)
            g.attention_decode_q8(qkv, cfg.qkv_dim, kc, vc, ks, vs, stride, lens, max_seq, nq, nkv, hd,
                                  max_seq, attn, cfg.q_dim, workspace=ws)
        g.linear_rows(attn, w["w_o"][l], o, n, cfg.q_dim, H)
        g.add_rmsnorm(x, o, w["mlp_norm"][l], h, n, H, cfg.rms_norm_eps)
        g.linear_silu_mul(h, w["w_gu"][l], act, n, H, I)
        g.linear_rows(act, w["w_down"][l], o, n, I, H)
        last = l + 1 == cfg.num_layers
        g.add_rmsnorm(x, o, w["final_norm"] if last else w["attn_norm"][l + 1], h, n, H,
                      cfg.rms_norm_eps)
    out = torch.empty(n, dtype=torch.int32, device="cuda")
    g.lm_head_argmax(h, w["embed"], n, H, cfg.vocab_size, out)
    return out


@pytest.mark.parametrize("head_dim,heads,kv", [(64, 8, 2), (128, 4, 2), (64, 8, 8)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("block", [0, 16, 24])
def test_step_equals_the_composition(head_dim, heads, kv, fmt, block):
    from kvasir_b200 import Gpu
    from kvasir_b200.decoder import Decoder
    g = Gpu(0)
    cfg = _cfg(head_dim, heads, kv)
    n_seq, max_seq = 3, 600
    dec = Decoder(cfg, n_seq, max_seq, seed=7, paged_block_size=block or None, kv_dtype=R.CODE[fmt])
    ref = Decoder(cfg, n_seq, max_seq, weights=dec.w, seed=7, paged_block_size=block or None,
                  kv_dtype=R.CODE[fmt])
    dec.set_row_projections(True)
    dec.set_fused_lm_head(True)
    dec.fill_kv_normal(seed=3)
    for a, b in ((ref.kc, dec.kc), (ref.vc, dec.vc)):
        a.view(torch.int8).copy_(b.view(torch.int8))
    ref.ks.copy_(dec.ks)
    ref.vs.copy_(dec.vs)
    pos = torch.tensor([0, 63, 590], dtype=torch.int32, device="cuda")
    dec.set_lengths(pos.cpu().numpy())
    ids = torch.tensor([1, 500, 999], dtype=torch.int32, device="cuda")
    dec.ids_in.copy_(ids)
    for _ in range(4):
        dec.step()
        ids = _step(g, ref, ids, pos, block)
        assert torch.equal(dec.ids_out, ids)
        for a, b in ((ref.kc, dec.kc), (ref.vc, dec.vc)):
            assert torch.equal(a.view(torch.int8), b.view(torch.int8))
        assert torch.equal(ref.ks, dec.ks) and torch.equal(ref.vs, dec.vs)
        pos = pos + 1
    assert g.device_error() == 0
    own, lib = dec.launches_per_step()
    assert own > 0 and lib == 0
    dec.close()
    ref.close()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_logits_stay_with_the_read_back_cache(fmt):
    """Against the 16-bit decoder on the same rows read back to 16 bits: the caches differ by
    that rounding (2^-9 of a value) and by the new token's codes (half a step: 1/254 of a row's
    largest value, or 2^-4 of an element).  One new key of 300 carries about 1/300 of the weight,
    so the logits differ by rounding alone: a few bf16 steps through two layers (bar: 0.03 of
    the largest logit, the bar of the 16-bit step against its oracle)."""
    from kvasir_b200 import Gpu
    from kvasir_b200.decoder import Decoder
    g = Gpu(0)
    cfg = _cfg()
    n_seq, max_seq, cur = 4, 320, 300
    q8 = Decoder(cfg, n_seq, max_seq, seed=9, kv_dtype=R.CODE[fmt])
    b16 = Decoder(cfg, n_seq, max_seq, weights=q8.w, seed=9)
    q8.fill_kv_normal(seed=4)
    pos = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
    for l in range(cfg.num_layers):
        g.kv_read_q8(q8.kc[l], q8.vc[l], q8.ks[l], q8.vs[l], q8.kc[l, 0].numel(), pos, n_seq, max_seq,
                     cfg.num_kv_heads, cfg.head_dim, max_seq, b16.kc[l], b16.vc[l], max_seq)
    ids = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    for d in (q8, b16):
        d.set_lengths(cur)
        d.ids_in.copy_(ids)
        d.step()
    torch.cuda.synchronize()
    want, got = b16.logits.cpu().numpy(), q8.logits.cpu().numpy()
    assert np.abs(got - want).max() <= 0.03 * np.abs(want).max() + 0.02
    # a paged 16-bit cache afterwards replaces the 8-bit one
    bs = 64
    pools = torch.zeros(cfg.num_layers, n_seq * 5, cfg.num_kv_heads, bs, cfg.head_dim,
                        dtype=torch.bfloat16, device="cuda")
    vpools = torch.zeros_like(pools)
    table = torch.arange(n_seq * 5, dtype=torch.int32, device="cuda").view(n_seq, 5)
    for l in range(cfg.num_layers):
        for src, dst in ((b16.kc, pools), (b16.vc, vpools)):
            dst[l].view(n_seq, 5, cfg.num_kv_heads, bs, cfg.head_dim).copy_(
                src[l].view(n_seq, cfg.num_kv_heads, 5, bs, cfg.head_dim).transpose(1, 2))
    q8.use_paged_cache(pools, vpools, table, 5, bs)
    q8.set_lengths(cur)
    q8.ids_in.copy_(ids)
    q8.step()
    torch.cuda.synchronize()
    assert np.abs(q8.logits.cpu().numpy() - want).max() <= 0.03 * np.abs(want).max() + 0.02
    for d in (q8, b16):
        d.close()


def test_rows_past_two_to_the_31():
    """Caches of more than 2^31 codes: append, read back and decode in the last sequence give
    the bits of the same calls on a cache of one sequence."""
    from kvasir_b200 import Gpu
    g = Gpu(0)
    n_q, n_kv, hd, max_seq, n_seq = 8, 8, 64, 16400, 260
    stride = n_kv * max_seq * hd
    assert n_seq * stride > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(5)
    t = 300
    heads = n_q + 2 * n_kv
    qkv = torch.randn(t, heads * hd, generator=gen, device="cuda").to(torch.bfloat16)
    big = torch.zeros(2, n_seq, n_kv, max_seq, hd, dtype=torch.int8, device="cuda")
    scales = torch.zeros(2, n_seq, n_kv, max_seq, device="cuda")
    small = torch.zeros(2, 1, n_kv, max_seq, hd, dtype=torch.int8, device="cuda")
    sscales = torch.zeros(2, 1, n_kv, max_seq, device="cuda")
    start = max_seq - t
    rows = torch.empty(n_seq, heads * hd, dtype=torch.bfloat16, device="cuda")
    pos = torch.full((n_seq,), start, dtype=torch.int32, device="cuda")
    for i in range(t):  # one row a call for all sequences; only the last one's matter
        rows.copy_(qkv[i].expand(n_seq, -1))
        g.rope_kv_append_q8(rows, n_seq, 1, pos + i, None, None, big[0], big[1], scales[0], scales[1],
                            stride, n_q, n_kv, hd, max_seq)
    g.rope_kv_append_q8(qkv, 1, t, pos[:1], None, None, small[0], small[1], sscales[0], sscales[1],
                        stride, n_q, n_kv, hd, max_seq)
    assert torch.equal(big[:, -1], small[:, 0]) and torch.equal(scales[:, -1], sscales[:, 0])
    ko = torch.empty(n_seq, n_kv, 2, hd, dtype=torch.bfloat16, device="cuda")
    vo, k1 = torch.empty_like(ko), torch.empty(1, n_kv, 2, hd, dtype=torch.bfloat16, device="cuda")
    v1 = torch.empty_like(k1)
    g.kv_read_q8(big[0], big[1], scales[0], scales[1], stride, pos, n_seq, 2, n_kv, hd, max_seq, ko, vo, 2)
    g.kv_read_q8(small[0], small[1], sscales[0], sscales[1], stride, pos[:1], 1, 2, n_kv, hd, max_seq, k1,
                 v1, 2)
    assert torch.equal(ko[-1:], k1) and torch.equal(vo[-1:], v1)
    lens = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
    lens[-1] = max_seq
    out = torch.empty(n_seq, n_q * hd, dtype=torch.bfloat16, device="cuda")
    out1 = torch.empty(1, n_q * hd, dtype=torch.bfloat16, device="cuda")
    q = qkv[:1, :n_q * hd].contiguous()
    # without a workspace both calls take one chunk per (sequence, head): the same sums
    g.attention_decode_q8(q.expand(n_seq, -1).contiguous(), n_q * hd, big[0], big[1], scales[0], scales[1],
                          stride, lens, max_seq, n_q, n_kv, hd, max_seq, out, n_q * hd)
    g.attention_decode_q8(q, n_q * hd, small[0], small[1], sscales[0], sscales[1], stride, lens[-1:],
                          max_seq, n_q, n_kv, hd, max_seq, out1, n_q * hd)
    assert torch.equal(out[-1:], out1) and bool((out[:-1] == 0).all())
    assert g.device_error() == 0


@pytest.mark.parametrize("block", [None, 16])
@pytest.mark.parametrize("first_seq", [None, 0])
def test_fill_after_the_switch_to_a_16_bit_pool(block, first_seq):
    """fill_kv_normal fills the cache that the steps read: after use_paged_cache, the pools given
    there, as it fills a 16-bit decoder's own."""
    from kvasir_b200.decoder import Decoder
    cfg, n_seq, max_seq, bs = _cfg(), 3, 150, 64
    ref = Decoder(cfg, n_seq, max_seq, seed=9, paged_block_size=bs)
    ref.fill_kv_normal(seed=4, first_seq=first_seq)
    dec = Decoder(cfg, n_seq, max_seq, weights=ref.w, seed=9, paged_block_size=block, kv_dtype=torch.int8)
    dec.fill_kv_normal(seed=2)
    kp, vp = torch.zeros_like(ref.kc), torch.zeros_like(ref.vc)
    dec.use_paged_cache(kp, vp, ref.block_table, ref.block_table.shape[1], bs)
    dec.fill_kv_normal(seed=4, first_seq=first_seq)
    assert torch.equal(kp, ref.kc) and torch.equal(vp, ref.vc)
    ids = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    for d in (ref, dec):
        d.set_lengths(100)
        d.ids_in.copy_(ids)
        d.step()
    torch.cuda.synchronize()
    assert torch.equal(ref.logits, dec.logits)
    for d in (ref, dec):
        d.close()
