"""64-bit restatements of the 8-bit cache operators and the error bounds their
tests use.

Bounds count roundings (u = half a step: bf16 2^-8, fp16 2^-11, fp32 2^-24):
  a logit is a sum of D fp32 products: off by (D + 8) 2^-24 sum|q k| scale,
  and a weight by as much, relatively (plus 2^-18 for exp2, log2 and the
  scales' products); a weight enters the second product rounded to 16 bits (u_p
  relative, 2^-25 absolute where f16 is subnormal); the sums over n tokens add
  n 2^-23; the result is rounded once (u of its type).
8-bit caches: the streaming kernel's weights are relative to the largest of 32
tokens and off by 2^-13 of themselves or 2^-17 of that largest, where a weight is p_t vs_t (vs
the value's scale) and meets a code c_td: with |c| vs <= the token's largest |v|,
one element is off by at most 2^-17 n max_t(p_t max_d |v_td|) / sum p on top."""

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rows64(codes, scale, table, n):
    """Token rows [n', Hkv, D] (float64) of the valid blocks of `table`, at most n."""
    nb, bs = codes.shape[:2]
    n = max(int(n), 0)
    ids = [int(i) for i in table[: (n + bs - 1) // bs] if 0 <= int(i) < nb]
    ids = torch.tensor(ids, dtype=torch.long, device=codes.device)
    if codes.element_size() == 1:
        x = codes.view(torch.uint8)[ids].view(codes.dtype).float().double()
        x = x * scale[ids].double().transpose(1, 2).unsqueeze(-1)
    else:
        x = codes[ids].double()
    return x.reshape(-1, *codes.shape[2:])[:n]


def attend64(q, K, V, out_dtype, p_dtype, scale=None, code=False):
    """(out, bound) of softmax(scale q K^T) V for q [Hq, D], K, V [n, Hkv, D]."""
    Hq, D = q.shape
    n = K.shape[0]
    if n == 0:
        z = torch.zeros(Hq, D, dtype=torch.float64, device=q.device)
        return z, z
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    G = Hq // K.shape[1]
    k = K.transpose(0, 1).repeat_interleave(G, 0)
    v = V.transpose(0, 1).repeat_interleave(G, 0)
    qd = q.double()
    x = torch.einsum("hd,hld->hl", qd, k) * scale
    w = torch.softmax(x, -1)
    out = torch.einsum("hl,hld->hd", w, v)
    mean = torch.einsum("hl,hld->hd", w, v.abs())
    terms = torch.einsum("hd,hld->hl", qd.abs(), k.abs()).amax(-1, keepdim=True) * scale
    rel = U[p_dtype] + 2 * ((D + 8) * 2.0 ** -24 * terms) + 2.0 ** -18 + n * 2.0 ** -23
    bound = mean * rel + v.abs().amax((1, 2))[:, None] * n * 2.0 ** -25
    if code:
        bound = bound + (w * v.abs().amax(-1)).amax(-1, keepdim=True) * n * 2.0 ** -17
    return out, bound * (1 + 2.0 ** -7) + U[out_dtype] * (out.abs() + bound) + 1e-30


def check_rows(got, q, k_cache, v_cache, k_scale, v_scale, table, ctx, prefix_table=None, prefix_len=0, scale=None):
    """Every row of an attention result within its bound."""
    p_dtype = torch.float16 if k_cache.element_size() == 1 else q.dtype
    worst = 0.0
    for b in range(q.shape[0]):
        K, V = (rows64(c, s, table[b], ctx[b]) for c, s in ((k_cache, k_scale), (v_cache, v_scale)))
        if prefix_table is not None:
            Kp, Vp = (rows64(c, s, prefix_table, prefix_len) for c, s in ((k_cache, k_scale), (v_cache, v_scale)))
            K, V = torch.cat((Kp, K)), torch.cat((Vp, V))
        want, bound = attend64(q[b], K, V, q.dtype, p_dtype, scale, k_cache.element_size() == 1)
        off = (got[b].double() - want).abs()
        assert torch.isfinite(got[b]).all(), f"row {b}"
        worst = max(worst, float((off / bound.clamp(min=1e-30)).max()))
        assert (off <= bound).all(), f"row {b} (context {int(ctx[b])}): {float((off / bound.clamp(min=1e-30)).max())} bounds"
    return worst
