"""The 8-bit paged KV cache and shared-prefix attention, as measured passes.

Four operators of one serving path over a paged KV cache:

  rope_kv_append_paged_quant  RoPE(q, k), then K and V written as 8-bit codes (int8 or e4m3) with
                              one fp32 scale for each (token, kv head)
  paged_kv_dequant            the contexts read back into dense 16-bit K and V, as a prefill takes them
  paged_attention_quant       decode attention (one query token a sequence) over the 8-bit cache
  paged_attention_prefix      decode attention of a batch whose sequences share a long prefix, over
                              16-bit or 8-bit caches

`run` computes a case in plain torch operations (own = False) or through the framework's entry
points (own = True); both start from what `prepare` returns.
"""

from __future__ import annotations

import functools
import math
import random
import sys
from pathlib import Path

import torch

own = False

QMAX = {"int8": 127.0, "e4m3": 448.0}
SCALE_FLOOR = 1e-12
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


# ------------------------------------------------------------------------ cases
def _case(name, kind, dtype, cache, B, ctx_lo, ctx_hi, Hq=32, Hkv=8, bs=16, new=0, prefix=0):
    c = dict(kind=kind, dtype=dtype, cache=cache, B=B, ctx_lo=ctx_lo, ctx_hi=ctx_hi, Hq=Hq, Hkv=Hkv, D=128, bs=bs,
             new=new, prefix=prefix)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one new token of one short sequence: what a single call costs
        _case("write_read_1tok_int8", "write_read", "bf16", "int8", 1, 17, 17, new=1),
        # chunked prefill: four sequences each bring 509 more tokens, and their contexts are read back for the
        # chunk's attention; lengths that end inside a page
        _case("write_read_chunk_e4m3", "write_read", "bf16", "e4m3", 4, 2000, 4001, new=509),
        # a whole prefill batch of 16384 tokens written and read back (fp16)
        _case("write_read_prefill_int8", "write_read", "fp16", "int8", 8, 2048, 2048, new=2048),
        # decode of one sequence with a short context: latency
        _case("decode_1seq_e4m3", "decode", "bf16", "e4m3", 1, 67, 67),
        # the decode step of a full batch, ragged contexts
        _case("decode_64seq_int8", "decode", "bf16", "int8", 64, 512, 8192),
        # the same batch with fewer and larger pages, eight query heads a kv head, e4m3, fp16
        _case("decode_48seq_g8_e4m3", "decode", "fp16", "e4m3", 48, 1, 8191, Hq=32, Hkv=4, bs=32),
        # few sequences with very long contexts: the work has to be split over the tokens
        _case("decode_3seq_long_int8", "decode", "bf16", "int8", 3, 90001, 131072),
        # two sequences behind a short system prompt: latency
        _case("prefix_2seq_bf16", "prefix", "bf16", "same", 2, 1, 33, prefix=130),
        # a full batch behind a long shared prompt
        _case("prefix_64seq_bf16", "prefix", "bf16", "same", 64, 1, 512, prefix=8192),
        # many samples of one prompt: compute counts as much as bandwidth
        _case("prefix_250seq_fp16", "prefix", "fp16", "same", 250, 1, 256, prefix=4091),
        # the full batch over the 8-bit cache
        _case("prefix_64seq_int8", "prefix", "bf16", "int8", 64, 1, 512, prefix=8192),
        # few sequences behind a document
        _case("prefix_12seq_e4m3", "prefix", "fp16", "e4m3", 12, 16, 2000, Hq=64, prefix=50001),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["write_read", "decode", "decode", "prefix", "prefix"])
    dtype = rng.choice(["bf16", "fp16"])
    bs = rng.choice([16, 16, 32])
    Hkv = rng.choice([1, 2, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 4, 8])
    if kind == "write_read":
        B = _log_int(rng, 1, 32)
        hi = _log_int(rng, 2, min(8192, 32768 // B))
        lo = _log_int(rng, 1, hi)
        new = min(lo, _log_int(rng, 1, max(1, 16384 // B)))
        return _case(None, kind, dtype, rng.choice(["int8", "e4m3"]), B, lo, hi, Hq, Hkv, bs, new=new)
    if kind == "decode":
        B = _log_int(rng, 1, 96)
        hi = _log_int(rng, 1, min(131072, 278528 // B))
        return _case(None, kind, dtype, rng.choice(["int8", "e4m3"]), B, _log_int(rng, 1, hi), hi, Hq, Hkv, bs)
    B = _log_int(rng, 1, 256)
    hi = _log_int(rng, 1, min(2048, 65536 // B))
    prefix = _log_int(rng, 1, min(50000, 1048576 // B))
    return _case(None, kind, dtype, rng.choice(["same", "int8", "e4m3"]), B, _log_int(rng, 1, hi), hi, Hq, Hkv, bs,
                 prefix=prefix)


# ----------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _contexts(case, seed):
    g = torch.Generator().manual_seed(seed + 17)
    return torch.randint(case["ctx_lo"], case["ctx_hi"] + 1, (case["B"],), generator=g, dtype=torch.int64)


def _quantise(x, kind):
    """Codes and scales of the last axis: fp32 in, scale = max(amax / qmax, floor)."""
    amax = x.abs().amax(-1)
    # (a division by a tensor: one by a Python number may run as a product with its rounded reciprocal)
    s = torch.clamp(amax / torch.full_like(amax, QMAX[kind]), min=SCALE_FLOOR)
    y = x / s.unsqueeze(-1)
    y = torch.clamp(torch.round(y) if kind == "int8" else y, -QMAX[kind], QMAX[kind])
    return y.to(_CODES[kind]), s


def _kv_rows(shape, D, g, keys):
    """Keys have a few loud channels, values differ in loudness from token to token."""
    x = torch.randn(*shape, D, generator=g, device="cuda")
    if keys:
        x *= 1.0 + 3.0 * (torch.rand(D, generator=g, device="cuda") < 0.05).float()
    else:
        x *= torch.exp(0.5 * torch.randn(*shape, 1, generator=g, device="cuda"))
    return x


def _cache(case, num_blocks, g, dtype):
    """K and V caches [num_blocks, bs, Hkv, D]; 8-bit ones with scales [num_blocks, Hkv, bs]."""

    def fill(keys):
        x = _kv_rows((num_blocks, case["bs"], case["Hkv"]), case["D"], g, keys)
        if case["cache"] == "same":
            return x.to(dtype), None
        c, s = _quantise(x, case["cache"])
        return c, s.transpose(1, 2).contiguous()

    (kc, ks), (vc, vs) = fill(True), fill(False)
    return kc, vc, ks, vs


def prepare(case, seed):
    dtype, bs, B, D = _DTYPES[case["dtype"]], case["bs"], case["B"], case["D"]
    g = _gen(seed)
    ctx = _contexts(case, seed)
    pages = -(-case["ctx_hi"] // bs)
    n_prefix = -(-case["prefix"] // bs)
    num_blocks = B * pages + n_prefix + 8
    perm = torch.randperm(num_blocks, generator=g, device="cuda")
    table = perm[: B * pages].reshape(B, pages).to(torch.int32).contiguous()
    kc, vc, ks, vs = _cache(case, num_blocks, g, dtype)
    s = dict(kind=case["kind"], cache=case["cache"], dtype=dtype, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs,
             block_table=table, context_len=ctx.to("cuda", torch.int32), max_len=case["ctx_hi"])
    if case["kind"] == "write_read":
        new = case["new"]
        T = B * new
        pos = (ctx.unsqueeze(1) - new + torch.arange(new)).to("cuda")  # the last `new` tokens of each context
        blk = torch.gather(table.long(), 1, pos // bs)
        s["slots"] = (blk * bs + pos % bs).reshape(T).contiguous()
        s["positions"] = pos.reshape(T).contiguous()
        ang = torch.outer(torch.arange(case["ctx_hi"], dtype=torch.float64),
                          1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
        ang = torch.cat((ang, ang), dim=-1)
        s["cos"], s["sin"] = ang.cos().float().to("cuda"), ang.sin().float().to("cuda")
        s["q"] = torch.randn(T, case["Hq"], D, generator=g, device="cuda").to(dtype)
        s["k"] = _kv_rows((T, case["Hkv"]), D, g, True).to(dtype)
        s["v"] = _kv_rows((T, case["Hkv"]), D, g, False).to(dtype)
    else:
        s["q"] = torch.randn(B, case["Hq"], D, generator=g, device="cuda").to(dtype)
    if case["kind"] == "prefix":
        s["prefix_table"] = perm[B * pages: B * pages + n_prefix].to(torch.int32).contiguous()
        s["prefix_len"] = torch.tensor([case["prefix"]], dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------ plain forms
def _rotate(x, c, s):
    h = x.shape[-1] // 2
    x1, x2 = x[..., :h].float(), x[..., h:].float()
    return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1)


def _pages(codes, scale, ids):
    """fp32 rows [..., pages * bs, Hkv, D] of the pages `ids` [..., pages]."""
    x = codes[ids].float()
    if scale is not None:
        x = x * scale[ids].transpose(-1, -2).unsqueeze(-1)
    return x.flatten(-4, -3)


def _plain_write(s):
    h = s["q"].shape[-1] // 2
    c = s["cos"][s["positions"], :h].unsqueeze(1)
    sn = s["sin"][s["positions"], :h].unsqueeze(1)
    q_out = _rotate(s["q"], c, sn).to(s["dtype"])
    bs = s["k_cache"].shape[1]
    blk, off = s["slots"] // bs, s["slots"] % bs
    kq, ksc = _quantise(_rotate(s["k"], c, sn), s["cache"])
    vq, vsc = _quantise(s["v"].float(), s["cache"])
    # (8-bit floating types are indexed through their bytes)
    s["k_cache"].view(torch.uint8)[blk, off] = kq.view(torch.uint8)
    s["v_cache"].view(torch.uint8)[blk, off] = vq.view(torch.uint8)
    s["k_scale"][blk, :, off] = ksc
    s["v_scale"][blk, :, off] = vsc
    return q_out


def _plain_read(s):
    ids = s["block_table"].long()
    live = torch.arange(s["max_len"], device="cuda") < s["context_len"].unsqueeze(1)
    live = live[:, :, None, None]

    def dense(codes, scale):
        x = _pages(codes, scale, ids)[:, : s["max_len"]]
        return torch.where(live, x, torch.zeros_like(x)).transpose(1, 2).to(s["dtype"]).contiguous()

    return dense(s["k_cache"], s["k_scale"]), dense(s["v_cache"], s["v_scale"])


def _plain_attend(s):
    q = s["q"].float()
    B, Hq, D = q.shape
    Hkv = s["k_cache"].shape[2]
    G = Hq // Hkv
    q = q.reshape(B, Hkv, G, D) / math.sqrt(D)
    ids = s["block_table"].long()
    K = _pages(s["k_cache"], s["k_scale"], ids).transpose(1, 2)  # [B, Hkv, S, D]
    V = _pages(s["v_cache"], s["v_scale"], ids).transpose(1, 2)
    live = torch.arange(K.shape[2], device="cuda") < s["context_len"].unsqueeze(1)
    x = torch.matmul(q, K.transpose(2, 3))  # [B, Hkv, G, S]
    x = x.masked_fill(~live[:, None, None, :], -math.inf)
    m = x.amax(-1, keepdim=True)
    if s["kind"] == "prefix":
        n = s["prefix_len"].long()
        pids = s["prefix_table"].long()
        Kp = _pages(s["k_cache"], s["k_scale"], pids).transpose(0, 1)  # [Hkv, P, D]
        Vp = _pages(s["v_cache"], s["v_scale"], pids).transpose(0, 1)
        plive = torch.arange(Kp.shape[1], device="cuda") < n
        qp = q.transpose(0, 1).reshape(Hkv, B * G, D)
        xp = torch.matmul(qp, Kp.transpose(1, 2)).masked_fill(~plive, -math.inf)
        mp = xp.amax(-1, keepdim=True).reshape(Hkv, B, G, 1).transpose(0, 1)
        m = torch.maximum(m, mp)
        pp = torch.exp(xp - m.transpose(0, 1).reshape(Hkv, B * G, 1))
        lp = pp.sum(-1, keepdim=True).reshape(Hkv, B, G, 1).transpose(0, 1)
        op = torch.matmul(pp, Vp).reshape(Hkv, B, G, D).transpose(0, 1)
    p = torch.exp(x - m)
    l, o = p.sum(-1, keepdim=True), torch.matmul(p, V)
    if s["kind"] == "prefix":
        l, o = l + lp, o + op
    return (o / l).reshape(B, Hq, D).to(s["dtype"])


@functools.lru_cache(maxsize=None)
def _ops():
    root = str(Path("triton-agent_b200").resolve())
    if root not in sys.path:
        sys.path.insert(0, root)
    from b200ops.runtime import ops

    return ops


def run(state):
    s = state
    if s["kind"] == "write_read":
        if own:
            K = _ops()
            q_out = K.rope_kv_append_paged_quant(s["q"], s["k"], s["v"], s["positions"], s["cos"], s["sin"],
                                                 s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
            k, v = K.paged_kv_dequant(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"],
                                      s["context_len"], s["max_len"], dtype=s["dtype"])
        else:
            q_out = _plain_write(s)
            k, v = _plain_read(s)
        return {"q_out": q_out, "k": k, "v": v}
    if not own:
        return _plain_attend(s)
    if s["kind"] == "decode":
        return _ops().paged_attention_quant(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                                            s["block_table"], s["context_len"])
    return _ops().paged_attention_prefix(s["q"], s["k_cache"], s["v_cache"], s["prefix_table"], s["prefix_len"],
                                         s["block_table"], s["context_len"], k_scale=s["k_scale"],
                                         v_scale=s["v_scale"])


# ------------------------------------------------------------------------- work
def work(case):
    B, Hq, Hkv, D, bs = case["B"], case["Hq"], case["Hkv"], case["D"], case["bs"]
    ctx = B * (case["ctx_lo"] + case["ctx_hi"]) / 2
    row = D * 2 if case["cache"] == "same" else D + 4  # one cached row of one head, scale included
    table = 4 * ctx / bs + 4 * B
    if case["kind"] == "write_read":
        T = B * case["new"]
        moved = T * (2 * Hq * D * 2 + 2 * Hkv * D * 2 + D * 4 + 16)  # q in and out, k and v in, cos/sin, position, slot
        moved += T * 2 * Hkv * row  # the new rows
        moved += 2 * (ctx - T) * Hkv * row + table  # the older rows
        moved += 2 * B * case["ctx_hi"] * Hkv * D * 2  # dense K and V
        return {"bytes": moved, "flops": 6 * T * (Hq + Hkv) * D / 2}
    tokens = ctx + case["prefix"]
    moved = 2 * tokens * Hkv * row + 2 * B * Hq * D * 2 + table + 4 * case["prefix"] / bs
    return {"bytes": moved, "flops": 4 * (ctx + B * case["prefix"]) * Hq * D}


# ------------------------------------------------------------------------ exact
def _exact_rows(s, which, ids, n):
    """Rows [n, Hkv, D] of the pages `ids` in float64."""
    c = s[which + "_cache"][ids].double()
    if s[which + "_scale"] is not None:
        c = c * s[which + "_scale"][ids].double().permute(0, 2, 1)[..., None]
    return c.reshape(-1, *c.shape[2:])[:n]


def _exact_codes(x, kind):
    """What 8 bits keep of the rows of x (float64): nearest code times scale."""
    s = (x.abs().max(-1, keepdim=True).values / QMAX[kind]).clamp(min=SCALE_FLOOR)
    y = x / s
    if kind == "int8":
        return y.round().clamp(-127, 127) * s
    # e4m3: three bits behind the leading one, exponents from -6 up
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return (torch.round(y / step) * step).clamp(-448, 448) * s


def exact(case, seed):
    s = prepare(case, seed)
    bs, B, Hkv, D = case["bs"], case["B"], case["Hkv"], case["D"]
    lens = [int(x) for x in s["context_len"].cpu()]
    if case["kind"] == "write_read":
        h, new = D // 2, case["new"]
        pos = s["positions"].double()
        inv = 1e4 ** (-2.0 * torch.arange(h, device="cuda", dtype=torch.float64) / D)
        ang = pos[:, None] * inv
        # the tables hold the angles' cosines and sines in 32 bits; they are inputs
        c = ang.cos().float().double()[:, None]
        sn = ang.sin().float().double()[:, None]

        def turn(x):
            a, b = x.double().split(h, dim=-1)
            return torch.cat((a * c - b * sn, b * c + a * sn), -1)

        fresh = {"k": _exact_codes(turn(s["k"]), case["cache"]), "v": _exact_codes(s["v"].double(), case["cache"])}
        out = {"q_out": turn(s["q"])}
        for w in ("k", "v"):
            dense = torch.zeros(B, Hkv, s["max_len"], D, dtype=torch.float64, device="cuda")
            for b, n in enumerate(lens):
                rows = _exact_rows(s, w, s["block_table"][b, : -(-n // bs)].long(), n)
                rows[n - new: n] = fresh[w][b * new: (b + 1) * new]
                dense[b, :, :n] = rows.transpose(0, 1)
            out[w] = dense
        return out
    G = case["Hq"] // Hkv
    out = torch.empty(B, case["Hq"], D, dtype=torch.float64, device="cuda")
    n0 = case["prefix"]
    head = [None, None]
    if n0:
        head = [_exact_rows(s, w, s["prefix_table"].long(), n0) for w in ("k", "v")]
    for b, n in enumerate(lens):
        ids = s["block_table"][b, : -(-n // bs)].long()
        k, v = _exact_rows(s, "k", ids, n), _exact_rows(s, "v", ids, n)
        if n0:
            k, v = torch.cat((head[0], k)), torch.cat((head[1], v))
        for j in range(Hkv):
            qj = s["q"][b, j * G:(j + 1) * G].double()
            w = torch.softmax(qj @ k[:, j].T / math.sqrt(D), dim=-1)
            out[b, j * G:(j + 1) * G] = w @ v[:, j]
    return out
