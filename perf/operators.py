"""Cases that measure the 8-bit KV cache and the shared-prefix decode attention.

Three kinds of pass, each as a serving program makes it:

  kv      RoPE of a chunk's qkv rows, their K and V quantised into an 8-bit cache as they
          are written, and the same rows read back as 16-bit values (what a prefill over
          the chunk reads)
  decode  one decode step's attention over an 8-bit cache, one query row per sequence
  shared  one decode step's attention of sequences that share a prefix, the prefix's keys
          read once for all of them (16-bit caches)

An 8-bit row (one position of one KV head) is head_dim codes, int8 or e4m3, and one f32
scale: scale = amax / 127 (int8) or amax / 448 (e4m3), code = round(x * (127 or 448) / amax).

`run` with own = False is the plain form in elementary torch operations; with own = True it
calls the framework.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
TINY = 2.0 ** -119  # rows whose largest magnitude is below this are stored as zeros

_gpu = None


def _handle():
    global _gpu
    if _gpu is None:
        from kvasir_b200 import Gpu
        _gpu = Gpu(0)
    return _gpu


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one sequence, one token at position 512 of a Llama-3.2-1B layer: launch latency
        dict(name="kv_one_token", op="kv", n_seq=1, t=1, pos=512, n_q=32, n_kv=8, hd=64,
             dtype="bf16", fmt="int8", block=0),
        # a decode batch of 32 into a paged cache of small blocks, each at a position of its own
        dict(name="kv_decode_paged", op="kv", n_seq=32, t=1, pos=1087, n_q=32, n_kv=8, hd=64,
             dtype="bf16", fmt="e4m3", block=16),
        # the prefill batch of 4 x 2048 tokens
        dict(name="kv_prefill", op="kv", n_seq=4, t=2048, pos=0, n_q=32, n_kv=8, hd=64,
             dtype="bf16", fmt="int8", block=0),
        # an odd chunk of a long prompt, head_dim 128, f16, paged
        dict(name="kv_chunk_odd", op="kv", n_seq=3, t=4001, pos=777, n_q=8, n_kv=2, hd=128,
             dtype="f16", fmt="e4m3", block=64),
        # one sequence over 513 positions: the smallest attention of the chain
        dict(name="decode_one", op="decode", n_seq=1, lo=513, hi=513, n_q=32, n_kv=8, hd=64,
             dtype="bf16", fmt="int8", block=0),
        # 64 sequences, context lengths uniform in [1, 4096]
        dict(name="decode_ragged", op="decode", n_seq=64, lo=1, hi=4096, n_q=32, n_kv=8, hd=64,
             dtype="bf16", fmt="e4m3", block=0),
        # a decode batch of 32 near context 1024 on a paged cache
        dict(name="decode_paged", op="decode", n_seq=32, lo=900, hi=1088, n_q=32, n_kv=8, hd=64,
             dtype="f16", fmt="int8", block=16),
        # head_dim 128, an odd batch, empty sequences among them
        dict(name="decode_hd128", op="decode", n_seq=37, lo=0, hi=5003, n_q=14, n_kv=2, hd=128,
             dtype="bf16", fmt="int8", block=0),
        # one GPU's long-context step: 256 sequences x 16384 tokens
        dict(name="decode_long", op="decode", n_seq=256, lo=16384, hi=16384, n_q=32, n_kv=8, hd=64,
             dtype="bf16", fmt="int8", block=0),
        # a few answers to one short instruction
        dict(name="shared_few", op="shared", n_seq=4, prefix=513, lo=1, hi=100, n_q=32, n_kv=8,
             hd=64, dtype="bf16", block=0),
        # a batch on a common system prompt, paged
        dict(name="shared_batch", op="shared", n_seq=32, prefix=4096, lo=1, hi=512, n_q=32, n_kv=8,
             hd=64, dtype="bf16", block=64),
        # a full batch over one long document
        dict(name="shared_long", op="shared", n_seq=256, prefix=16384, lo=1, hi=1000, n_q=32,
             n_kv=8, hd=64, dtype="f16", block=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["kv", "decode", "decode", "shared"])
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16"]))
    n_kv = rng.choice([1, 2, 4, 8, 8])
    group = rng.choice([1, 2, 3, 4, 4, 7, 8, 16])
    hd = 64 if op == "shared" else rng.choice([64, 64, 128])
    c.update(n_q=n_kv * group, n_kv=n_kv, hd=hd)
    if op == "kv":
        n_seq = _log(rng, 1, 128)
        t = _log(rng, 1, max(1, 12000 // n_seq))
        c.update(n_seq=n_seq, t=t, pos=rng.randint(0, 4000), fmt=rng.choice(["int8", "e4m3"]),
                 block=rng.choice([0, 16, 48, 64, 128]))
    elif op == "decode":
        n_seq = _log(rng, 1, 128)
        hi = _log(rng, 1, min(20000, 400000 // n_seq))
        c.update(n_seq=n_seq, lo=rng.choice([0, 1, hi]), hi=hi, fmt=rng.choice(["int8", "e4m3"]),
                 block=rng.choice([0, 0, 16, 32, 64, 256]))
    else:
        n_seq = _log(rng, 1, 200)
        prefix = _log(rng, 1, min(16000, 100_000_000 // (n_seq * n_kv * group)))
        hi = _log(rng, 1, min(4000, 100000 // n_seq))
        c.update(n_seq=n_seq, prefix=prefix, lo=rng.choice([0, 1, hi]), hi=hi,
                 block=rng.choice([0, 0, 64, 128]))
    return c


# ------------------------------------------------------------------------------ inputs
def _quantise(x, fmt):
    """f32 rows [..., hd] -> (codes, scales), the definition in f32.  The divisors are
    tensors so that both divisions are divisions."""
    amax = x.abs().amax(-1)
    top = torch.full_like(amax, TOP[fmt])
    zero = amax < TINY
    inv = torch.where(zero, torch.zeros_like(amax), top / amax)
    scale = torch.where(zero, torch.zeros_like(amax), amax / top)
    y = x * inv[..., None]
    if fmt == "int8":
        return y.round().clamp(-127, 127).to(torch.int8), scale
    return y.to(torch.float8_e4m3fn), scale


def _rows(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _q8_cache(g, lead, rows, hd, dtype, fmt):
    """Codes [lead..., rows, hd] and scales [lead..., rows] of unit normal rows."""
    codes = torch.empty(*lead, rows, hd, dtype=CODE[fmt], device="cuda")
    scales = torch.empty(*lead, rows, dtype=torch.float32, device="cuda")
    step = max(1, (1 << 26) // (lead[1] * rows * hd))
    for i in range(0, lead[0], step):
        x = _rows(g, (min(step, lead[0] - i), *lead[1:], rows, hd), dtype).float()
        codes[i:i + step], scales[i:i + step] = _quantise(x, fmt)
    return codes, scales


def _table(rng, n_seq, per_seq, spare, device="cuda"):
    n = n_seq * per_seq + spare
    return torch.randperm(n, generator=rng, device=device)[:n_seq * per_seq].to(
        torch.int32).reshape(n_seq, per_seq), n


def prepare(case, seed):
    c, dt = case, DT[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    n_seq, n_q, n_kv, hd, block = c["n_seq"], c["n_q"], c["n_kv"], c["hd"], c["block"]
    s = dict(case=dict(c))
    if c["op"] == "kv":
        t = c["t"]
        max_seq = c["pos"] + t + 5
        s["qkv"] = _rows(g, (n_seq * t, (n_q + 2 * n_kv) * hd), dt)
        # positions below and up to pos, as sequences of one batch have
        low = 0 if t == 1 else c["pos"]
        s["pos"] = torch.randint(low, c["pos"] + 1, (n_seq,), generator=g, device="cuda").int()
        ang = torch.arange(max_seq, device="cuda", dtype=torch.float64)[:, None] * (
            500000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd))
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        if block:
            per = -(-max_seq // block)
            s["table"], n_blocks = _table(g, n_seq, per, 3)
            lead, rows = (n_blocks, n_kv), block
        else:
            lead, rows = (n_seq, n_kv), max_seq
        for k in ("k", "v"):
            s[k + "c"] = torch.zeros(*lead, rows, hd, dtype=torch.int8, device="cuda").view(
                CODE[c["fmt"]])
            s[k + "s"] = torch.zeros(*lead, rows, device="cuda")
            s[k + "_out"] = torch.empty(n_seq, n_kv, t, hd, dtype=dt, device="cuda")
        s["max_seq"] = max_seq
    else:
        s["q"] = _rows(g, (n_seq, n_q * hd), dt)
        lens = torch.randint(c["lo"], c["hi"] + 1, (n_seq,), generator=g, device="cuda").int()
        if c["op"] == "decode":
            max_seq = c["hi"] + 1
            if block:
                per = -(-max_seq // block)
                s["table"], n_blocks = _table(g, n_seq, per, 3)
                lead, rows = (n_blocks, n_kv), block
            else:
                lead, rows = (n_seq, n_kv), max_seq
            s["kc"], s["ks"] = _q8_cache(g, lead, rows, hd, dt, c["fmt"])
            s["vc"], s["vs"] = _q8_cache(g, lead, rows, hd, dt, c["fmt"])
            s["max_len"] = c["hi"]
        else:
            if block:  # one pool; every table begins with the prefix's blocks
                max_seq = c["prefix"] + c["hi"] + 1
                per, pre = -(-max_seq // block), c["prefix"] // block
                table, n_blocks = _table(g, n_seq, per, 3)
                table[:, :pre] = table[:1, :pre]
                s["table"] = table
                s["kc"] = _rows(g, (n_blocks, n_kv, block, hd), dt)
                s["vc"] = _rows(g, (n_blocks, n_kv, block, hd), dt)
                r = c["prefix"] - pre * block
                if r:  # the prefix ends inside a block: each sequence holds its own copy of it
                    for x in (s["kc"], s["vc"]):
                        x[table[:, pre].long(), :, :r] = x[table[0, pre].long(), :, :r].clone()
                lens = lens + c["prefix"]
                s["max_len"] = c["prefix"] + c["hi"]
            else:
                max_seq = c["hi"] + 1
                s["pk"] = _rows(g, (n_kv, c["prefix"], hd), dt)
                s["pv"] = _rows(g, (n_kv, c["prefix"], hd), dt)
                s["kc"] = _rows(g, (n_seq, n_kv, max_seq, hd), dt)
                s["vc"] = _rows(g, (n_seq, n_kv, max_seq, hd), dt)
                s["max_len"] = c["hi"]
        s["lens"], s["max_seq"] = lens, max_seq
        s["out"] = torch.empty(n_seq, n_q * hd, dtype=dt, device="cuda")
    if own:  # the handle and the workspace that a serving program keeps
        s["gpu"] = _handle()
        n = 0
        if c["op"] == "decode":
            n = s["gpu"].attention_decode_q8_workspace_bytes(n_seq, c["hi"], n_q, n_kv, hd)
        elif c["op"] == "shared":
            n = s["gpu"].attention_decode_shared_workspace_bytes(n_seq, c["prefix"], c["hi"], n_q,
                                                                 n_kv, hd)
        s["ws"] = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    return (_run_own if own else _run_plain)[c["op"]](s, c)


def _positions(s, c):
    """Index of each new row: [n_seq, t] positions."""
    return s["pos"].long()[:, None] + torch.arange(c["t"], device="cuda")


def _plain_kv(s, c):
    n_seq, t, n_q, n_kv, hd, dt = c["n_seq"], c["t"], c["n_q"], c["n_kv"], c["hd"], DT[c["dtype"]]
    x = s["qkv"].view(n_seq, t, n_q + 2 * n_kv, hd)
    p = _positions(s, c)
    cos, sin = s["cos"][p][:, :, None], s["sin"][p][:, :, None]
    a, b = x[:, :, :n_q + n_kv, :hd // 2].float(), x[:, :, :n_q + n_kv, hd // 2:].float()
    x[:, :, :n_q + n_kv] = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(dt)
    got = [s["qkv"]]
    for name, first in (("k", n_q), ("v", n_q + n_kv)):
        codes, scales = _quantise(x[:, :, first:first + n_kv].float(), c["fmt"])
        where = _where(s, c, p)
        _bytes(s[name + "c"])[where] = codes.view(torch.int8)
        s[name + "s"][where] = scales
        back = _bytes(s[name + "c"])[where].view(CODE[c["fmt"]]).float() * s[name + "s"][where][..., None]
        s[name + "_out"].copy_(back.to(dt).transpose(1, 2))
        got.append(s[name + "_out"])
    return got


def _bytes(x):
    return x.view(torch.int8)


def _where(s, c, p):
    """Index of positions p [n_seq, t] in the cache, all heads: [n_seq, t, n_kv] of them."""
    h = torch.arange(c["n_kv"], device="cuda")
    b = torch.arange(c["n_seq"], device="cuda")[:, None]
    if c["block"]:
        return (s["table"].long()[b, p // c["block"]][..., None], h, (p % c["block"])[..., None])
    return (b[..., None], h, p[..., None])


def _unpaged(x, s, c):
    """[n_seq, n_kv, rows, ...] of a cache that may be in blocks."""
    if not c["block"]:
        return x
    y = x[s["table"].long()].transpose(1, 2)  # [n_seq, n_kv, blocks, block, ...]
    return y.reshape(y.shape[0], y.shape[1], y.shape[2] * y.shape[3], *y.shape[4:])


def _softmax(z):
    """Rows of scores, -inf where masked; a row with nothing left is zeros."""
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(m.isinf(), torch.zeros_like(m), m))
    return e / e.sum(-1, keepdim=True).clamp_min(torch.finfo(z.dtype).tiny)


def _plain_decode(s, c):
    n_seq, n_q, n_kv, hd = c["n_seq"], c["n_q"], c["n_kv"], c["hd"]
    q = s["q"].view(n_seq, n_kv, n_q // n_kv, hd).float()
    fmt = CODE[c["fmt"]]
    k = _unpaged(_bytes(s["kc"]), s, c).view(fmt).float() * _unpaged(s["ks"], s, c)[..., None]
    z = q @ k.transpose(-1, -2) * (1 / math.sqrt(hd))
    del k
    free = torch.arange(z.shape[-1], device="cuda") >= s["lens"][:, None]
    p = _softmax(z.masked_fill(free[:, None, None], -math.inf))
    v = _unpaged(_bytes(s["vc"]), s, c).view(fmt).float() * _unpaged(s["vs"], s, c)[..., None]
    s["out"].copy_((p @ v).reshape(n_seq, n_q * hd).to(s["out"].dtype))
    return s["out"]


def _plain_shared(s, c):
    n_seq, n_q, n_kv, hd, n_pre = c["n_seq"], c["n_q"], c["n_kv"], c["hd"], c["prefix"]
    q = s["q"].view(n_seq, n_kv, n_q // n_kv, hd).float()
    k, v = _unpaged(s["kc"], s, c), _unpaged(s["vc"], s, c)
    lens = s["lens"]
    if c["block"]:
        pk, pv, k, v = k[0, :, :n_pre], v[0, :, :n_pre], k[:, :, n_pre:], v[:, :, n_pre:]
        lens = lens - n_pre
    else:
        pk, pv = s["pk"], s["pv"]
    # the prefix once for all: the sequences' rows of one KV head against its keys
    rows = q.transpose(0, 1).reshape(n_kv, -1, hd)
    z0 = (rows @ pk.float().transpose(-1, -2)).view(n_kv, n_seq, -1, n_pre).transpose(0, 1)
    z1 = q @ k.float().transpose(-1, -2)
    free = torch.arange(z1.shape[-1], device="cuda") >= lens[:, None]
    p = _softmax(torch.cat([z0, z1.masked_fill(free[:, None, None], -math.inf)], -1) *
                 (1 / math.sqrt(hd)))
    o = p[..., :n_pre].transpose(0, 1).reshape(n_kv, -1, n_pre) @ pv.float()
    o = o.view(n_kv, n_seq, -1, hd).transpose(0, 1) + p[..., n_pre:] @ v.float()
    s["out"].copy_(o.reshape(n_seq, n_q * hd).to(s["out"].dtype))
    return s["out"]


def _own_kv(s, c):
    g, n_seq, t, n_q, n_kv, hd = s["gpu"], c["n_seq"], c["t"], c["n_q"], c["n_kv"], c["hd"]
    if c["block"]:
        mb = s["table"].shape[1]
        g.rope_kv_append_q8_paged(s["qkv"], n_seq, t, s["pos"], s["cos"], s["sin"], s["kc"], s["vc"],
                                  s["ks"], s["vs"], s["table"], mb, c["block"], n_q, n_kv, hd)
        g.kv_read_q8_paged(s["kc"], s["vc"], s["ks"], s["vs"], s["table"], mb, c["block"], s["pos"],
                           n_seq, t, n_kv, hd, s["k_out"], s["v_out"], t)
    else:
        stride = n_kv * s["max_seq"] * hd
        g.rope_kv_append_q8(s["qkv"], n_seq, t, s["pos"], s["cos"], s["sin"], s["kc"], s["vc"],
                            s["ks"], s["vs"], stride, n_q, n_kv, hd, s["max_seq"])
        g.kv_read_q8(s["kc"], s["vc"], s["ks"], s["vs"], stride, s["pos"], n_seq, t, n_kv, hd,
                     s["max_seq"], s["k_out"], s["v_out"], t)
    return [s["qkv"], s["k_out"], s["v_out"]]


def _own_decode(s, c):
    g, n_q, n_kv, hd = s["gpu"], c["n_q"], c["n_kv"], c["hd"]
    if c["block"]:
        g.attention_decode_q8_paged(s["q"], n_q * hd, s["kc"], s["vc"], s["ks"], s["vs"], s["table"],
                                    s["table"].shape[1], c["block"], s["lens"], s["max_len"], n_q,
                                    n_kv, hd, s["out"], n_q * hd, workspace=s["ws"])
    else:
        g.attention_decode_q8(s["q"], n_q * hd, s["kc"], s["vc"], s["ks"], s["vs"],
                              n_kv * s["max_seq"] * hd, s["lens"], s["max_len"], n_q, n_kv, hd,
                              s["max_seq"], s["out"], n_q * hd, workspace=s["ws"])
    return s["out"]


def _own_shared(s, c):
    g, n_q, n_kv, hd = s["gpu"], c["n_q"], c["n_kv"], c["hd"]
    if c["block"]:
        g.attention_decode_shared_paged(s["q"], n_q * hd, s["kc"], s["vc"], s["table"],
                                        s["table"].shape[1], c["block"], c["prefix"], s["lens"],
                                        s["max_len"], n_q, n_kv, hd, s["out"], n_q * hd,
                                        workspace=s["ws"])
    else:
        g.attention_decode_shared(s["q"], n_q * hd, s["pk"], s["pv"], c["prefix"], c["prefix"],
                                  s["kc"], s["vc"], n_kv * s["max_seq"] * hd, s["lens"],
                                  s["max_len"], n_q, n_kv, hd, s["max_seq"], s["out"], n_q * hd,
                                  workspace=s["ws"])
    return s["out"]


_run_plain = dict(kv=_plain_kv, decode=_plain_decode, shared=_plain_shared)
_run_own = dict(kv=_own_kv, decode=_own_decode, shared=_own_shared)


# -------------------------------------------------------------------------- its cost
def work(case):
    c = case
    n_seq, n_q, n_kv, hd = c["n_seq"], c["n_q"], c["n_kv"], c["hd"]
    if c["op"] == "kv":
        rows = n_seq * c["t"]
        kv = 2 * rows * n_kv
        # q and k heads read and written, v heads read, the tables' rows; codes and scales
        # written, 16-bit rows written
        b = (rows * (n_q + n_kv) * hd * 4 + rows * n_kv * hd * 2 + rows * hd * 4 +
             kv * (hd + 4) + kv * hd * 2)
        return dict(bytes=b, flops=rows * (n_q + n_kv) * hd * 3 + kv * hd * 4)
    keys = n_seq * (c["lo"] + c["hi"]) / 2
    io = 2 * n_seq * n_q * hd * 2
    if c["op"] == "decode":
        return dict(bytes=keys * n_kv * 2 * (hd + 4) + io, flops=keys * n_q * hd * 4)
    return dict(bytes=(keys + c["prefix"]) * n_kv * hd * 4 + io,
                flops=(keys + n_seq * c["prefix"]) * n_q * hd * 4)


# ------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c = case
    n_seq, n_q, n_kv, hd, block = c["n_seq"], c["n_q"], c["n_kv"], c["hd"], c["block"]
    if c["op"] == "kv":
        t, half = c["t"], hd // 2
        x = s["qkv"].double().reshape(n_seq, t, n_q + 2 * n_kv, hd)
        for b in range(n_seq):
            p = int(s["pos"][b])
            co, si = s["cos"][p:p + t].double()[:, None], s["sin"][p:p + t].double()[:, None]
            rot = x[b, :, :n_q + n_kv]
            lo, hi = rot[..., :half].clone(), rot[..., half:].clone()
            rot[..., :half] = lo * co - hi * si
            rot[..., half:] = lo * si + hi * co
        heads = x[:, :, n_q:].to(DT[c["dtype"]]).double()  # the cache holds 16-bit rows' codes
        big = heads.abs().max(-1, keepdim=True).values
        y = heads / big * TOP[c["fmt"]]
        if c["fmt"] == "int8":
            y = torch.round(y)
        else:  # three mantissa bits, exponents down to 2^-6
            e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6)))
            y = torch.round(y * 2 ** (3 - e)) * 2 ** (e - 3)
        y = (y * big / TOP[c["fmt"]]).permute(0, 2, 1, 3)
        return [x.reshape(n_seq * t, -1), y[:, :n_kv].contiguous(), y[:, n_kv:].contiguous()]
    group = n_q // n_kv
    out = torch.zeros(n_seq, n_q * hd, dtype=torch.float64, device="cuda")
    lens = s["lens"].tolist()
    for b in range(n_seq):
        if block:
            rows = s["table"][b].long()
            pick = lambda x: x[rows].transpose(0, 1).flatten(1, 2)  # noqa: E731
        else:
            pick = lambda x: x[b]  # noqa: E731
        if c["op"] == "decode":
            k, v = (_code_values(pick(_bytes(s[n + "c"]))[:, :lens[b]], c["fmt"]) *
                    pick(s[n + "s"])[:, :lens[b], None].double() for n in ("k", "v"))
        else:
            k, v = (pick(s[n])[:, :lens[b]].double() for n in ("kc", "vc"))
            if not block:
                k = torch.cat([s["pk"].double(), k], 1)
                v = torch.cat([s["pv"].double(), v], 1)
        if k.shape[1] == 0:
            continue
        q = s["q"][b].double().view(n_kv, group, hd)
        w = torch.softmax(torch.einsum("hgd,hkd->hgk", q, k) / math.sqrt(hd), -1)
        out[b] = torch.einsum("hgk,hkd->hgd", w, v).reshape(-1)
    return out


def _code_values(x, fmt):
    return x.view(CODE[fmt]).to(torch.float32).double()
