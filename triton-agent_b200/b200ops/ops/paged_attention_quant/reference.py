"""Paged decode attention over an 8-bit cache: reference in plain PyTorch.
paged_attention of the values code * scale (fp32); a sequence without tokens
gives zeros.
"""

import math

import torch

from b200ops.ops.paged_kv_dequant.reference import dense_rows


def attend(q, K, V):
    """softmax(q K^T / sqrt(D)) V for q [Hq, D], K and V [n, Hkv, D], in fp32."""
    G = q.shape[0] // K.shape[1]
    k = K.transpose(0, 1).repeat_interleave(G, 0)
    v = V.transpose(0, 1).repeat_interleave(G, 0)
    w = torch.softmax(torch.einsum("hd,hld->hl", q.float(), k) / math.sqrt(q.shape[1]), dim=-1)
    return torch.einsum("hl,hld->hd", w, v)


def paged_attention_quant(q, k_cache, v_cache, k_scale, v_scale, block_table, context_len):
    bs = k_cache.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
    for b in range(q.shape[0]):
        ctx = int(context_len[b])
        ids = block_table[b, : max(0, (ctx + bs - 1) // bs)]
        K = dense_rows(k_cache, k_scale, ids, max(ctx, 0))
        if K.shape[0]:
            out[b] = attend(q[b], K, dense_rows(v_cache, v_scale, ids, ctx))
    return out.to(q.dtype)


def generate_test_inputs(B: int = 8, H: int = 32, D: int = 128, num_blocks: int = 256, block_size: int = 16,
                         max_blocks: int = 32, ctx_len: int = 500, H_kv: int = 8, e4m3: int = 0,
                         dtype: torch.dtype = torch.bfloat16, device: str = "cuda", seed: int = 0):
    from b200ops.workloads import quant_cache

    g = torch.Generator(device=device).manual_seed(seed)
    q = torch.randn(B, H, D, generator=g, device=device).to(dtype)
    c = quant_cache(num_blocks, block_size, H_kv, D, torch.float8_e4m3fn if e4m3 else torch.int8, device, seed)
    table = torch.randint(0, num_blocks, (B, max_blocks), generator=g, device=device)
    ctx = torch.full((B,), ctx_len, dtype=torch.long, device=device)
    return q, c.k_cache, c.v_cache, c.k_scale, c.v_scale, table, ctx
