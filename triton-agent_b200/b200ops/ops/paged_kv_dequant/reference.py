"""Contexts of an 8-bit paged cache as dense 16-bit K and V: reference in plain
PyTorch.  Row s of sequence b is code * scale (fp32, rounded once) of its
token s; ids outside [0, num_blocks) are dropped and later blocks move up;
rows at or past the context are zero.
"""

import torch


def dense_rows(codes, scale, ids, n):
    """fp32 rows [n', Hkv, D], n' <= n, of the valid blocks among ids."""
    ids = ids[(ids >= 0) & (ids < codes.shape[0])].long()
    x = codes.view(torch.uint8)[ids].view(codes.dtype).float()
    if scale is not None:
        x = x * scale[ids].transpose(1, 2).unsqueeze(-1)
    return x.reshape(-1, *codes.shape[2:])[:n]


def paged_kv_dequant(k_cache, v_cache, k_scale, v_scale, block_table, context_len, max_len, dtype=torch.bfloat16):
    nb, bs, Hkv, D = k_cache.shape
    outs = []
    for codes, scale in ((k_cache, k_scale), (v_cache, v_scale)):
        out = torch.zeros(block_table.shape[0], Hkv, max_len, D, dtype=dtype, device=codes.device)
        for b in range(block_table.shape[0]):
            ctx = int(context_len[b])
            if ctx > 0:
                rows = dense_rows(codes, scale, block_table[b, : (ctx + bs - 1) // bs], min(ctx, max_len))
                out[b, :, : rows.shape[0]] = rows.transpose(0, 1).to(dtype)
        outs.append(out)
    return tuple(outs)


def generate_test_inputs(B: int = 4, Hkv: int = 8, D: int = 128, num_blocks: int = 256, block_size: int = 16,
                         max_blocks: int = 32, ctx_len: int = 500, max_len: int = 512, e4m3: int = 0,
                         dtype: torch.dtype = torch.bfloat16, device: str = "cuda", seed: int = 0):
    from b200ops.workloads import quant_cache

    g = torch.Generator(device=device).manual_seed(seed)
    c = quant_cache(num_blocks, block_size, Hkv, D, torch.float8_e4m3fn if e4m3 else torch.int8, device, seed)
    table = torch.randint(0, num_blocks, (B, max_blocks), generator=g, device=device)
    ctx = torch.full((B,), ctx_len, dtype=torch.long, device=device)
    return c.k_cache, c.v_cache, c.k_scale, c.v_scale, table, ctx, max_len, dtype
