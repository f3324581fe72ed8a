"""RoPE(q, k) + append into an 8-bit paged cache: reference in plain PyTorch.

A cached row x (rotated k, or v; fp32) becomes codes and one scale:
scale = max(max|x| / qmax, 1e-12); int8 code = clamp(round(x / scale), -127,
127), e4m3 code = the nearest e4m3 value to x / scale.  Every operation is
rounded on its own in fp32.  Returns (q_out, k_cache', v_cache', k_scale',
v_scale') as new tensors; 8-bit floating caches as fp16 values of their codes
(exact).
"""

import torch

QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
SCALE_FLOOR = 1e-12


def quantise_rows(x, code_dtype):
    """Codes and scales of the last axis of x (fp32)."""
    amax = x.abs().amax(-1)
    s = torch.clamp(amax / torch.full_like(amax, QMAX[code_dtype]), min=SCALE_FLOOR)
    y = x / s.unsqueeze(-1)
    y = torch.clamp(torch.round(y) if code_dtype == torch.int8 else y, -QMAX[code_dtype], QMAX[code_dtype])
    return y.to(code_dtype), s


def rotate(x, c, s):
    h = x.shape[-1] // 2
    a, b = x[..., :h].float(), x[..., h:].float()
    return torch.cat((a * c - b * s, b * c + a * s), dim=-1)


def rope_kv_append_paged_quant(q, k, v, positions, cos, sin, slot_mapping, k_cache, v_cache, k_scale, v_scale):
    h = k.shape[-1] // 2
    c = cos[positions, :h].float().unsqueeze(1)
    s = sin[positions, :h].float().unsqueeze(1)
    q_out = rotate(q, c, s).to(q.dtype)
    kq, ks = quantise_rows(rotate(k, c, s), k_cache.dtype)
    vq, vs = quantise_rows(v.float(), v_cache.dtype)
    nb, bs = k_cache.shape[:2]
    kc, vc = k_cache.view(torch.uint8).clone(), v_cache.view(torch.uint8).clone()
    ksc, vsc = k_scale.clone(), v_scale.clone()
    for t in range(k.shape[0]):
        slot = int(slot_mapping[t])
        if 0 <= slot < nb * bs:
            kc[slot // bs, slot % bs] = kq[t].view(torch.uint8)
            vc[slot // bs, slot % bs] = vq[t].view(torch.uint8)
            ksc[slot // bs, :, slot % bs] = ks[t]
            vsc[slot // bs, :, slot % bs] = vs[t]
    return q_out, codes_as_values(kc.view(k_cache.dtype)), codes_as_values(vc.view(v_cache.dtype)), ksc, vsc


def codes_as_values(c):
    return c if c.dtype == torch.int8 else c.half()


def generate_test_inputs(T: int = 64, Hq: int = 32, Hkv: int = 8, D: int = 128, num_blocks: int = 4096,
                         block_size: int = 16, max_pos: int = 4096, e4m3: int = 0,
                         dtype: torch.dtype = torch.bfloat16, device: str = "cuda", seed: int = 0):
    from b200ops.workloads import quant_cache, rope_tables

    g = torch.Generator(device=device).manual_seed(seed)
    q = torch.randn(T, Hq, D, generator=g, device=device).to(dtype)
    k = torch.randn(T, Hkv, D, generator=g, device=device).to(dtype)
    v = torch.randn(T, Hkv, D, generator=g, device=device).to(dtype)
    positions = torch.randint(0, max_pos, (T,), generator=g, device=device)
    cos, sin = rope_tables(max_pos, D, device=device)
    slots = torch.randperm(num_blocks * block_size, generator=g, device=device)[:T].contiguous()
    c = quant_cache(num_blocks, block_size, Hkv, D, torch.float8_e4m3fn if e4m3 else torch.int8, device, seed)
    return q, k, v, positions, cos, sin, slots, c.k_cache, c.v_cache, c.k_scale, c.v_scale
