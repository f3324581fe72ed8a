"""Decode attention of a batch that shares a prefix: reference in plain PyTorch.
Sequence b attends to the first prefix_len tokens of the prefix's blocks and
to its own context_len[b] tokens behind them, one softmax over both, in fp32.
Caches in q's dtype (scales None) or 8-bit with scales.
"""

import torch

from b200ops.ops.paged_attention_quant.reference import attend
from b200ops.ops.paged_kv_dequant.reference import dense_rows


def paged_attention_prefix(q, k_cache, v_cache, prefix_table, prefix_len, block_table, context_len, k_scale=None,
                           v_scale=None):
    bs = k_cache.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float32, device=q.device)

    def rows(codes, scale, table, n):
        n = max(int(n), 0)
        return dense_rows(codes, scale, table[: (n + bs - 1) // bs], n)

    Kp, Vp = rows(k_cache, k_scale, prefix_table, prefix_len), rows(v_cache, v_scale, prefix_table, prefix_len)
    for b in range(q.shape[0]):
        K = torch.cat((Kp, rows(k_cache, k_scale, block_table[b], context_len[b])))
        if K.shape[0]:
            out[b] = attend(q[b], K, torch.cat((Vp, rows(v_cache, v_scale, block_table[b], context_len[b]))))
    return out.to(q.dtype)


def generate_test_inputs(B: int = 8, H: int = 32, D: int = 128, num_blocks: int = 512, block_size: int = 16,
                         prefix: int = 1000, max_blocks: int = 8, ctx_len: int = 100, H_kv: int = 8, quant: int = 0,
                         e4m3: int = 0, dtype: torch.dtype = torch.bfloat16, device: str = "cuda", seed: int = 0):
    from b200ops.workloads import paged_cache, quant_cache

    g = torch.Generator(device=device).manual_seed(seed)
    q = torch.randn(B, H, D, generator=g, device=device).to(dtype)
    table = torch.randint(0, num_blocks, (B, max_blocks), generator=g, device=device)
    ptable = torch.randint(0, num_blocks, ((prefix + block_size - 1) // block_size,), generator=g, device=device)
    plen = torch.full((1,), prefix, dtype=torch.long, device=device)
    ctx = torch.full((B,), ctx_len, dtype=torch.long, device=device)
    if quant or e4m3:
        c = quant_cache(num_blocks, block_size, H_kv, D, torch.float8_e4m3fn if e4m3 else torch.int8, device, seed)
        return q, c.k_cache, c.v_cache, ptable, plen, table, ctx, c.k_scale, c.v_scale
    c = paged_cache(num_blocks, block_size, H_kv, D, dtype, device, seed)
    return q, c.k_cache, c.v_cache, ptable, plen, table, ctx
