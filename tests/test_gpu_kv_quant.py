"""The 8-bit paged KV cache on the GPU: codes and scales bit for bit against
the plain form and within half a code step of 64 bits, the read-back bit for
bit, attention within bounds derived in kv8_ref, and the operators together."""

import pytest
import torch
from click.testing import CliRunner

from b200ops import cli
from b200ops import workloads as WL
from b200ops.ops.paged_kv_dequant import reference as RD
from b200ops.ops.rope_kv_append_paged_quant import reference as RA
from b200ops.runtime import lib as L
from b200ops.runtime import ops as K
from kv8_ref import U, attend64, check_rows, rows64

pytestmark = pytest.mark.gpu
CODES = [torch.int8, torch.float8_e4m3fn]


def bits(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def append_inputs(T, Hq, Hkv, D, dtype, nb, bs, code, cs_dtype=torch.float32, seed=0, max_pos=600):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(T, Hq, D, generator=g).to(dtype) if Hq else None
    k, v = (torch.randn(T, Hkv, D, generator=g).to(dtype) for _ in range(2))
    pos = torch.randint(0, max_pos, (T,), generator=g)
    cos, sin = WL.rope_tables(max_pos, D, device="cpu")
    slots = torch.randperm(nb * bs, generator=g)[:T]
    c = WL.quant_cache(nb, bs, Hkv, D, code, "cpu", seed)
    return q, k, v, pos, cos.to(cs_dtype), sin.to(cs_dtype), slots, c


def run_append(x, dev, cfg=None):
    q, k, v, pos, cos, sin, slots, c = x
    d = [t.to(dev) if t is not None else None for t in (q, k, v, pos, cos, sin, slots)]
    cache = [t.to(dev).clone() for t in (c.k_cache, c.v_cache, c.k_scale, c.v_scale)]
    q_out = K.rope_kv_append_paged_quant(*d, *cache, cfg=cfg)
    torch.cuda.synchronize()
    return q_out, cache


def expect_append(x):
    """The plain form token by token, tokens out of range left out (CPU)."""
    q, k, v, pos, cos, sin, slots, c = x
    P, n = cos.shape[0], c.k_cache.shape[0] * c.k_cache.shape[1]
    ok = (pos >= 0) & (pos < P)
    sl = torch.where(ok & (slots >= 0) & (slots < n), slots, torch.full_like(slots, -1))
    safe = torch.where(ok, pos, torch.zeros_like(pos))
    q_in = q if q is not None else k[:, :1]
    want = RA.rope_kv_append_paged_quant(q_in, k, v, safe, cos, sin, sl, c.k_cache, c.v_cache, c.k_scale, c.v_scale)
    q_out = torch.where(ok[:, None, None], want[0], torch.zeros_like(want[0])) if q is not None else None
    return (q_out, *want[1:])


def same(got, want):
    q_out, cache = got
    if want[0] is None:
        assert q_out is None
    else:
        assert torch.equal(q_out.cpu(), want[0])
    for a, b in zip(cache, want[1:]):
        a = a.cpu()
        assert torch.equal(RA.codes_as_values(a) if a.element_size() == 1 else a, b)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,Hq,Hkv,D,bs", [(1, 32, 8, 128, 16), (5, 8, 8, 128, 8), (64, 32, 8, 128, 16),
                                           (513, 16, 2, 128, 32), (700, 0, 3, 128, 16), (33, 4, 1, 64, 16),
                                           (3, 7, 7, 6, 5), (530, 2, 2, 80, 16)])
def test_append_bit_exact(T, Hq, Hkv, D, bs, dtype, code, cuda_device):
    x = append_inputs(T, Hq, Hkv, D, dtype, 64 if T < 100 else 1000 // bs + 80, bs, code, seed=T)
    want = expect_append(x)
    for cfg in (None, {"rows_per_cta": 1}, {"rows_per_cta": 6}):
        same(run_append(x, cuda_device, cfg), want)


@pytest.mark.parametrize("code", CODES)
def test_append_16_bit_tables(code, cuda_device):
    x = append_inputs(40, 8, 4, 128, torch.bfloat16, 32, 16, code, cs_dtype=torch.bfloat16)
    same(run_append(x, cuda_device), expect_append(x))


@pytest.mark.parametrize("T", [9, 300, 900])
def test_append_collisions_and_tokens_out_of_range(T, cuda_device):
    """The last token that writes a slot wins, whether later slots are scanned
    or looked up; tokens out of range neither write nor hide earlier ones."""
    x = list(append_inputs(T, 4, 2, 128, torch.bfloat16, 100, 16, torch.int8, seed=T))
    g = torch.Generator().manual_seed(T)
    slots = x[6].clone()
    slots[torch.randperm(T, generator=g)[: T // 3]] = int(slots[0])  # many tokens, one slot
    slots[1], slots[2], slots[T // 2] = -1, 1600, 1 << 40
    slots[T - 2] = slots[T - 1] = slots[3]
    pos = x[3].clone()
    pos[T - 1], pos[4] = 600, -3
    x[6], x[3] = slots, pos
    want = expect_append(x)
    same(run_append(x, cuda_device), want)
    assert torch.count_nonzero(want[0][T - 1]) == 0


@pytest.mark.parametrize("code", CODES)
def test_codes_within_half_a_step_of_64_bits(code, cuda_device):
    """|code * s - x| <= half a code step (int8: s / 2; e4m3: 2^-4 of the value,
    at least 2^-10 s), plus the fp32 roundings of x, s and the quotient: 8 u
    of the row's largest element."""
    x = append_inputs(50, 2, 4, 128, torch.bfloat16, 64, 16, code, seed=5)
    _, k, v, pos, cos, sin, slots, _ = x
    _, (kc, vc, ks, vs) = run_append(x, cuda_device)
    h = 64
    c, s = (t[pos, :h].double()[:, None] for t in (cos, sin))
    kd = k.double()
    rot = torch.cat((kd[..., :h] * c - kd[..., h:] * s, kd[..., h:] * c + kd[..., :h] * s), -1)
    for cache, scale, want in ((kc, ks, rot), (vc, vs, v.double())):
        sc = scale.cpu()[slots // 16, :, slots % 16].double()[..., None]
        got = bits(cache.cpu())[slots // 16, slots % 16].view(code).float().double() * sc
        step = sc / 2 if code == torch.int8 else torch.maximum(want.abs() * 2.0 ** -4, sc * 2.0 ** -10)
        slack = want.abs().amax(-1, keepdim=True) * 8 * 2.0 ** -24
        assert ((got - want).abs() <= step * (1 + 2.0 ** -20) + slack).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("D", [128, 64])
def test_rows_of_zeros_tiny_and_non_finite_values(D, code, cuda_device):
    x = append_inputs(6, 2, 2, D, torch.float16, 8, 16, code, seed=8)
    _, k, v, pos, _, _, slots, _ = x
    v[0] = 0
    v[1] = 2.0 ** -24  # below the scale floor's reach: codes of a tiny row
    v[2, 0, 5] = float("inf")
    v[3, 1, D - 1] = float("nan")
    k[4, 0, 3] = float("-inf")
    _, (kc, vc, ks, vs) = run_append(x, cuda_device)
    want = expect_append(x)
    at = lambda t, i: t.cpu()[slots[i] // 16, :, slots[i] % 16]  # noqa: E731
    assert torch.equal(at(vs, 0), torch.full((2,), 1e-12))
    assert torch.equal(at(vs, 1), want[4][slots[1] // 16, :, slots[1] % 16])
    assert torch.isnan(at(vs, 2)).tolist() == [True, False] and torch.isnan(at(vs, 3)).tolist() == [False, True]
    assert torch.isnan(at(ks, 4)).tolist() == [True, False]
    table = (slots[:4] // 16).to(cuda_device).reshape(4, 1)
    kd, vd = K.paged_kv_dequant(kc, vc, ks, vs, table, torch.full((4,), 16, device=cuda_device), 16,
                                dtype=torch.float16)
    off = slots % 16
    assert torch.count_nonzero(vd[0, :, off[0]]) == 0
    assert torch.isnan(vd[2, 0, off[2]]).all() and torch.isfinite(vd[2, 1, off[2]]).all()
    assert torch.isnan(vd[3, 1, off[3]]).all()


# ------------------------------------------------------------------- read back
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hkv,D,bs,index", [(8, 128, 16, torch.int32), (1, 128, 32, torch.int64),
                                            (3, 64, 8, torch.int32), (2, 20, 5, torch.int64)])
def test_read_back_bit_exact(Hkv, D, bs, index, dtype, code, cuda_device):
    nb, maxb = 60, 14
    c = WL.quant_cache(nb, bs, Hkv, D, code, cuda_device, seed=D)
    g = torch.Generator().manual_seed(D)
    bt = torch.randint(0, nb, (8, maxb), generator=g)
    cl = torch.tensor([0, 1, bs - 1, bs, bs + 1, 9 * bs + 3, maxb * bs, maxb * bs + 50])
    bt[5, 2], bt[6, 0], bt[6, 7] = -1, nb, -9  # dropped: later blocks move up
    for max_len in (1, 4 * bs + 1, maxb * bs + 7):
        want = RD.paged_kv_dequant(*(t.cpu() for t in (c.k_cache, c.v_cache, c.k_scale, c.v_scale)), bt, cl, max_len,
                                   dtype)
        outs = [torch.full((8, Hkv, max_len, D), float("nan"), dtype=dtype, device=cuda_device) for _ in range(2)]
        got = K.paged_kv_dequant(c.k_cache, c.v_cache, c.k_scale, c.v_scale, bt.to(index).to(cuda_device),
                                 cl.to(index).to(cuda_device), max_len, dtype=dtype, k_out=outs[0], v_out=outs[1])
        for a, b in zip(got, want):
            assert torch.equal(a.cpu(), b)


# ------------------------------------------------------------------- attention
def attention_case(dev, B, Hq, Hkv, D, bs, dtype, code, ctx, nb=None, index=torch.int32, seed=0, extra=0):
    maxb = max(1, max((c + bs - 1) // bs for c in ctx)) + extra
    nb = nb or B * maxb + 3
    g = torch.Generator(device=dev).manual_seed(seed)
    if code is None:
        c = WL.paged_cache(nb, bs, Hkv, D, dtype, dev, seed)
        cache = (c.k_cache, c.v_cache, None, None)
    else:
        c = WL.quant_cache(nb, bs, Hkv, D, code, dev, seed)
        cache = (c.k_cache, c.v_cache, c.k_scale, c.v_scale)
    q = torch.randn(B, Hq, D, generator=g, device=dev).to(dtype)
    table = torch.randperm(nb, generator=g, device=dev)[: B * maxb].reshape(B, maxb).to(index)
    return q, cache, table, torch.tensor(ctx, device=dev, dtype=index)


CTX = [1, 15, 16, 17, 0, 33, 200, 511]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,bs", [(32, 8, 128, 16), (8, 8, 128, 16), (8, 4, 128, 32), (8, 1, 128, 16),
                                         (6, 3, 128, 16), (48, 12, 128, 48), (4, 2, 128, 128), (8, 8, 128, 256),
                                         (2, 1, 128, 8), (9, 3, 128, 16), (6, 2, 64, 16), (4, 4, 200, 5)])
def test_decode_attention(Hq, Hkv, D, bs, dtype, code, cuda_device):
    q, cache, bt, cl = attention_case(cuda_device, len(CTX), Hq, Hkv, D, bs, dtype, code, CTX, seed=Hq + bs)
    out = K.paged_attention_quant(q, *cache, bt, cl)
    again = K.paged_attention_quant(q, *cache, bt, cl)
    torch.cuda.synchronize()
    assert K.read_device_error() == 0
    assert torch.equal(out, again)
    assert torch.count_nonzero(out[4]) == 0
    check_rows(out, q, *cache, bt, cl)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("cfg", [None, {"stages": 2}, {"stages": 6}, {"rows_per_cta": 4}, {"rows_per_cta": 1},
                                 {"flags": 8}, {"flags": 1}])
def test_decode_attention_launch_parameters(cfg, code, cuda_device):
    ctx = [3000, 1, 777, 64, 2049, 0, 16]
    q, cache, bt, cl = attention_case(cuda_device, len(ctx), 16, 8, 128, 16, torch.bfloat16, code, ctx, index=torch.int64)
    out = K.paged_attention_quant(q, *cache, bt, cl, cfg=cfg)
    torch.cuda.synchronize()
    assert K.read_device_error() == 0
    check_rows(out, q, *cache, bt, cl)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("Hkv,bs", [(8, 16), (2, 16), (1, 8)])
def test_dropped_ids_and_garbage_behind_the_context(Hkv, bs, code, cuda_device):
    """Ids outside the pool are dropped (later blocks move up); slots behind the
    context hold NaN codes and NaN, infinite and negative scales."""
    ctx = [40, 100, 5, 320, 1, 250]
    q, cache, bt, cl = attention_case(cuda_device, len(ctx), 2 * Hkv, Hkv, 128, bs, torch.bfloat16, code, ctx, extra=2)
    kc, vc, ks, vs = cache
    for b, c in enumerate(ctx):
        last, off = int(bt[b, (c - 1) // bs]), (c - 1) % bs + 1
        bits(kc)[last, off:] = 127  # e4m3: NaN
        bits(vc)[last, off:] = 127
        ks[last, :, off:] = float("nan")
        vs[last, :, off:] = float("inf")
        if off + 1 < bs:
            vs[last, :, off + 1:] = -1.0
    check_rows(K.paged_attention_quant(q, *cache, bt, cl), q, *cache, bt, cl)
    bt[1, 1], bt[3, 0], bt[3, 9], bt[4, 0] = -1, kc.shape[0], -(1 << 30), -2
    # the kept blocks now end where garbage-free pages follow
    clean = WL.quant_cache(kc.shape[0], bs, Hkv, 128, code, cuda_device, seed=77)
    cache = (clean.k_cache, clean.v_cache, clean.k_scale, clean.v_scale)
    out = K.paged_attention_quant(q, *cache, bt, cl)
    check_rows(out, q, *cache, bt, cl)
    assert torch.count_nonzero(out[4]) == 0  # its only block was dropped


def test_context_longer_than_the_table(cuda_device):
    q, cache, bt, _ = attention_case(cuda_device, 2, 8, 2, 128, 16, torch.float16, torch.int8, [64, 64])
    cl = torch.tensor([10000, -5], dtype=torch.int32, device=cuda_device)
    out = K.paged_attention_quant(q, *cache, bt, cl)
    check_rows(out, q, *cache, bt, torch.tensor([64, 0]))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("B,Hkv,bs,pages", [(1, 8, 16, 10), (1, 8, 16, 11), (9, 2, 32, 3), (40, 16, 16, 24),
                                            (75, 16, 16, 8), (148, 4, 16, 1)])
def test_short_tables(B, Hkv, bs, pages, code, cuda_device):
    """Tables of few entries, with sequences of every length down to none, some
    without a valid block; and the same batch in a table of many columns."""
    ctx = [pages * bs - (7 * b) % (pages * bs + 1) for b in range(B)]
    q, cache, bt, cl = attention_case(cuda_device, B, 2 * Hkv, Hkv, 128, bs, torch.bfloat16, code, ctx)
    bt = bt[:, :pages].contiguous()
    cl[B // 2] = -3
    bt[B // 3] = -1
    out = K.paged_attention_quant(q, *cache, bt, cl)
    check_rows(out, q, *cache, bt, cl)
    wide = torch.full((B, 60), -1, dtype=bt.dtype, device=cuda_device)
    wide[:, :pages] = bt
    check_rows(K.paged_attention_quant(q, *cache, wide, cl), q, *cache, wide, cl)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("Hkv", [8, 2, 3])
def test_value_scales_of_every_size(Hkv, code, cuda_device):
    """Value scales from 2^-90 to 2^60 side by side, unwritten (zero) scales and
    queries of very different size: every row stays within its bound."""
    ctx = [300, 64, 17]
    q, cache, bt, cl = attention_case(cuda_device, 3, Hkv * 4, Hkv, 128, 16, torch.bfloat16, code, ctx, seed=4)
    g = torch.Generator(device=cuda_device).manual_seed(9)
    for b, (lo, hi) in enumerate(((-12, 2), (-90, -80), (50, 60))):
        ids = bt[b].long()
        e = torch.randint(lo, hi + 1, cache[3][ids].shape, generator=g, device=cuda_device)
        cache[3][ids] *= torch.exp2(e.float())
    cache[2][bt[0, 1].long(), :, 3] = 0.0
    cache[3][bt[0, 1].long(), :, 3] = 0.0
    bits(cache[0])[bt[0, 1].long(), 3] = 0
    bits(cache[1])[bt[0, 1].long(), 3] = 0
    q[1] *= 1e-30
    q[2] *= 40.0
    q[0, :, :64] *= 2.0 ** -20
    small = cache[3].clone()
    out = K.paged_attention_quant(q, *cache, bt, cl)
    # the 2^60 row overflows fp16-like ranges but not bf16: finite
    check_rows(out, q, *cache, bt, cl)
    assert torch.equal(small, cache[3])


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("flags", [0, 1])
def test_nan_reaches_the_output_that_reads_it(flags, code, cuda_device):
    q, cache, bt, cl = attention_case(cuda_device, 3, 16, 4, 128, 16, torch.bfloat16, code, [50, 20, 70])
    cache[2][bt[0, 1].long(), 1, 4] = float("nan")
    cache[3][bt[1, 0].long(), 2, 19 - 16] = float("nan")
    q[2, 5, 7] = float("nan")
    out = K.paged_attention_quant(q, *cache, bt, cl, cfg={"flags": flags})
    bad = torch.isnan(out).all(-1).cpu()
    want = torch.zeros(3, 16, dtype=torch.bool)
    want[0, 4:8] = want[1, 8:12] = want[2, 5] = True
    assert torch.equal(bad, want)
    assert torch.equal(torch.isnan(out).any(-1).cpu(), want)


def test_batch_of_more_segments_than_a_launch_takes(cuda_device):
    B, Hkv = 300, 64  # eight head groups a sequence: 2400 segments
    ctx = [int(c) for c in torch.randint(0, 40, (B,), generator=torch.Generator().manual_seed(1))]
    q, cache, bt, cl = attention_case(cuda_device, B, Hkv, Hkv, 128, 16, torch.float16, torch.int8, ctx, nb=1000)
    out = K.paged_attention_quant(q, *cache, bt, cl, cfg={"flags": 8})
    torch.cuda.synchronize()
    assert K.read_device_error() == 0
    for b in (0, 1, 100, 255, 256, 257, 299):
        check_rows(out[b:b + 1], q[b:b + 1], *cache, bt[b:b + 1], cl[b:b + 1])


def test_long_context_offsets_beyond_32_bits(cuda_device):
    """Two caches of 4.3 GB: pages at byte offsets above 2^32."""
    nb, bs, Hkv = 262400, 16, 8
    kc = torch.zeros(nb, bs, Hkv, 128, dtype=torch.int8, device=cuda_device)
    vc = torch.zeros_like(kc)
    ks = torch.full((nb, Hkv, bs), 0.01, device=cuda_device)
    vs = ks.clone()
    g = torch.Generator(device=cuda_device).manual_seed(0)
    ids = torch.cat((torch.arange(nb - 40, nb, device=cuda_device), torch.arange(20, device=cuda_device)))
    for c in (kc, vc):
        c[ids] = torch.randint(-127, 128, (60, bs, Hkv, 128), generator=g, device=cuda_device, dtype=torch.int8)
    bt = ids.reshape(2, 30).to(torch.int32)
    cl = torch.tensor([480, 471], dtype=torch.int32, device=cuda_device)
    q = torch.randn(2, 32, 128, generator=g, device=cuda_device).bfloat16()
    out = K.paged_attention_quant(q, kc, vc, ks, vs, bt, cl)
    check_rows(out, q, kc, vc, ks, vs, bt, cl)
    kd, _ = K.paged_kv_dequant(kc, vc, ks, vs, bt, cl, 480)
    assert torch.equal(kd[0].cpu(), (rows64(kc, ks, bt[0], 480)).transpose(0, 1).to(torch.bfloat16).cpu())
    x = [torch.randn(1, h, 128, generator=g, device=cuda_device).bfloat16() for h in (32, 8, 8)]
    cos, sin = WL.rope_tables(8, 128, device=cuda_device)
    slot = torch.tensor([nb * bs - 5], device=cuda_device)
    K.rope_kv_append_paged_quant(*x, torch.zeros(1, dtype=torch.long, device=cuda_device), cos, sin, slot, kc, vc, ks, vs)
    want, _ = RA.quantise_rows(x[2].float().cpu(), torch.int8)
    assert torch.equal(vc[nb - 1, bs - 5].cpu(), want[0])


# -------------------------------------------------------------- the shared prefix
@pytest.mark.parametrize("code", [None, *CODES])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,bs,B", [(32, 8, 128, 16, 5), (8, 8, 128, 16, 3), (8, 1, 128, 32, 70),
                                           (16, 8, 128, 64, 40), (6, 3, 128, 16, 9), (64, 8, 128, 128, 33),
                                           (8, 2, 128, 256, 3), (9, 3, 128, 16, 4), (4, 2, 64, 16, 3), (2, 2, 40, 6, 3)])
def test_prefix_attention(Hq, Hkv, D, bs, B, dtype, code, cuda_device):
    g = torch.Generator().manual_seed(B)
    ctx = [int(c) for c in torch.randint(0, 120, (B,), generator=g)]
    ctx[0], ctx[1] = 0, 1
    n_prefix = (1000 + bs - 1) // bs
    q, cache, bt, cl = attention_case(cuda_device, B, Hq, Hkv, D, bs, dtype, code, ctx, seed=B,
                                      nb=B * 16 + n_prefix + 40, index=torch.int32)
    pt = torch.randperm(cache[0].shape[0], generator=torch.Generator().manual_seed(B))[:n_prefix].to(
        cuda_device, torch.int32)
    for n in (0, 1, bs, 130, 1000):
        pl = torch.tensor([n], dtype=torch.int32, device=cuda_device)
        out = K.paged_attention_prefix(q, cache[0], cache[1], pt, pl, bt, cl, cache[2], cache[3])
        torch.cuda.synchronize()
        assert K.read_device_error() == 0
        check_rows(out, q, *cache, bt, cl, pt, n)
        if n == 0:
            assert torch.count_nonzero(out[0]) == 0


@pytest.mark.parametrize("code", [None, *CODES])
@pytest.mark.parametrize("B,Hq,prefix_pages,pages", [(40, 32, 600, 24), (6, 32, 600, 200), (150, 16, 9, 60),
                                                     (20, 64, 2500, 2)])
def test_prefix_lengths_far_from_the_tables(B, Hq, prefix_pages, pages, code, cuda_device):
    """The SMs are shared out by the tables' sizes; the lengths follow later."""
    q, cache, bt, cl = attention_case(cuda_device, B, Hq, 8, 128, 16, torch.bfloat16, code, [pages * 16] * B, seed=B,
                                      nb=B * pages + 100)
    g = torch.Generator().manual_seed(B)
    pt = torch.randint(0, cache[0].shape[0], (prefix_pages,), generator=g).to(cuda_device, torch.int32)
    some = torch.randint(0, pages * 16 + 1, (B,), generator=g).to(cuda_device, torch.int32)
    for n, ctx in ((0, some), (37, torch.zeros_like(cl)), (prefix_pages * 16 - 3, torch.zeros_like(cl)), (1, cl),
                   (prefix_pages * 16 + 99, torch.ones_like(cl))):
        pl = torch.tensor([n], dtype=torch.int32, device=cuda_device)
        out = K.paged_attention_prefix(q, cache[0], cache[1], pt, pl, bt, ctx, cache[2], cache[3])
        torch.cuda.synchronize()
        assert K.read_device_error() == 0
        check_rows(out, q, *cache, bt, ctx, pt, min(n, prefix_pages * 16))


@pytest.mark.parametrize("code", [None, *CODES])
@pytest.mark.parametrize("bs", [16, 8])
def test_prefix_dropped_ids_garbage_and_no_own_tokens(bs, code, cuda_device):
    B, n = 20, 515
    q, cache, bt, cl = attention_case(cuda_device, B, 16, 4, 128, bs, torch.bfloat16, code, [7] * B, nb=400, index=torch.int64)
    # blocks of the prefix alone (garbage behind its last token must not be a sequence's live token)
    free = torch.ones(400, dtype=torch.bool, device=cuda_device)
    free[bt.flatten()] = False
    pt = torch.nonzero(free).flatten().flip(0)[: (n + bs - 1) // bs + 3].clone()
    last, off = int(pt[(n - 1) // bs]), (n - 1) % bs + 1
    for c in cache[:2]:
        if code is None:
            c[last, off:] = float("nan")
        else:
            bits(c)[last, off:] = 127
    if code is not None:
        cache[2][last, :, off:] = float("inf")
        cache[3][last, :, off:] = float("nan")
    pl = torch.tensor(n, device=cuda_device)  # 0-d is taken too
    run = lambda t, c, l: K.paged_attention_prefix(q, cache[0], cache[1], pt, l, t, c, cache[2], cache[3])  # noqa: E731
    check_rows(run(bt, cl, pl), q, *cache, bt, cl, pt, n)
    none = torch.zeros_like(cl)
    check_rows(run(bt, none, pl), q, *cache, bt, none, pt, n)
    check_rows(run(bt[:, :0].contiguous(), none, pl), q, *cache, bt, none, pt, n)  # no table of own blocks
    pt[2], pt[10] = -1, 400
    if code is None:
        for c in cache[:2]:
            c[last] = 0.5
    else:
        cache[2][last], cache[3][last] = 0.1, 0.1
        bits(cache[0])[last], bits(cache[1])[last] = 3, 5
    n2 = torch.tensor([n], device=cuda_device)
    check_rows(run(bt, cl, n2), q, *cache, bt, cl, pt, n)
    too_long = torch.tensor([1 << 20], device=cuda_device)
    check_rows(run(bt, cl, too_long), q, *cache, bt, cl, pt, pt.numel() * bs)


@pytest.mark.parametrize("code", [None, *CODES])
def test_prefix_equals_attention_over_the_joined_tables(code, cuda_device):
    """A prefix of whole blocks followed by each sequence's own blocks is one
    table: both ways within twice the bound of one."""
    B, bs, P = 30, 16, 64
    ctx = [int(c) for c in torch.randint(1, 300, (B,), generator=torch.Generator().manual_seed(3))]
    q, cache, bt, cl = attention_case(cuda_device, B, 32, 8, 128, bs, torch.bfloat16, code, ctx, nb=1200)
    pt = torch.arange(1100, 1100 + P, device=cuda_device, dtype=torch.int32)
    out = K.paged_attention_prefix(q, cache[0], cache[1], pt, torch.tensor([P * bs], device=cuda_device, dtype=torch.int32),
                                   bt, cl, cache[2], cache[3])
    joined = torch.cat((pt.expand(B, P), bt), 1).contiguous()
    both = cl + P * bs
    one = K.paged_attention(q, cache[0], cache[1], joined, both) if code is None else \
        K.paged_attention_quant(q, *cache, joined, both)
    for b in range(B):
        _, bound = attend64(q[b], rows64(cache[0], cache[2], joined[b], both[b]),
                            rows64(cache[1], cache[3], joined[b], both[b]), q.dtype,
                            torch.bfloat16 if code is None else torch.float16, code=code is not None)
        assert ((out[b].double() - one[b].double()).abs() <= 2 * bound).all()


# ---------------------------------------------------------------- used together
@pytest.mark.parametrize("code", CODES)
def test_prefill_then_decode_steps_then_read_back(code, cuda_device):
    """A serving run: prompts appended, read back for flash_attn, then decode
    steps that append and attend; each step against 64 bits over the cache it
    left."""
    B, Hq, Hkv, D, bs, prompt, steps = 3, 16, 16, 128, 16, 130, 4
    nb, dev = 64, cuda_device
    kc = torch.zeros(nb, bs, Hkv, D, dtype=code, device=dev)
    vc = torch.zeros_like(kc)
    ks, vs = (torch.zeros(nb, Hkv, bs, device=dev) for _ in range(2))
    cos, sin = WL.rope_tables(256, D, device=dev)
    g = torch.Generator(device=dev).manual_seed(0)
    table = torch.randperm(nb, generator=g, device=dev)[: B * 10].reshape(B, 10).to(torch.int32)
    slot_of = lambda b, p: table[b].long()[p // bs] * bs + p % bs  # noqa: E731
    rand = lambda n, h: torch.randn(n, h, D, generator=g, device=dev).bfloat16()  # noqa: E731

    def append(pos):
        n = B * pos.numel()
        slots = torch.cat([slot_of(b, pos) for b in range(B)])
        x = rand(n, Hq), rand(n, Hkv), rand(n, Hkv)
        return K.rope_kv_append_paged_quant(*x, pos.repeat(B), cos, sin, slots, kc, vc, ks, vs)

    append(torch.arange(prompt, device=dev))
    cl = torch.full((B,), prompt, dtype=torch.int32, device=dev)
    for step in range(steps):
        q = append(torch.tensor([prompt + step], device=dev))
        cl += 1
        out = K.paged_attention_quant(q, kc, vc, ks, vs, table, cl, cfg={"flags": 8})
        check_rows(out, q, kc, vc, ks, vs, table, cl)
    n = prompt + steps
    kd, vd = K.paged_kv_dequant(kc, vc, ks, vs, table, cl, n)
    o = K.flash_attn(q.reshape(B, Hq, 1, D), kd, vd)  # the last step's query over the dense context
    for b in range(B):
        want, bound = attend64(q[b], kd[b].transpose(0, 1).double(), vd[b].transpose(0, 1).double(), q.dtype,
                               torch.bfloat16)
        assert ((o[b, :, 0].double() - want).abs() <= bound).all()


def test_two_graphs_and_two_streams(cuda_device):
    """Two captured steps and eager calls on other streams run at once: no
    scratch is shared, results stay those of a call alone."""
    dev = cuda_device
    cases = []
    for i in range(2):
        ctx = [int(c) for c in torch.randint(1, 2500, (24,), generator=torch.Generator().manual_seed(i))]
        cases.append(attention_case(dev, 24, 32, 8, 128, 16, torch.bfloat16, CODES[i], ctx, seed=i))
    pt = torch.arange(40, device=dev, dtype=torch.int32)
    pl = torch.tensor([630], dtype=torch.int32, device=dev)

    def both(c):
        q, cache, bt, cl = c
        return (K.paged_attention_quant(q, *cache, bt, cl),
                K.paged_attention_prefix(q, cache[0], cache[1], pt, pl, bt, cl, cache[2], cache[3]))

    want = [tuple(t.clone() for t in both(c)) for c in cases]
    torch.cuda.synchronize()
    graphs = []
    for c in cases:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = both(c)
        graphs.append((gr, outs))
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(5):
        eager = []
        for s, (gr, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        for i, s in enumerate(streams[2:]):
            with torch.cuda.stream(s):
                eager.append(both(cases[i]))
        torch.cuda.synchronize()
        assert K.read_device_error() == 0
        for i in range(2):
            for a, b, w in zip(graphs[i][1], eager[i], want[i]):
                assert torch.equal(a, w) and torch.equal(b, w)


def test_captured_step_follows_its_inputs(cuda_device):
    """Append + attention captured once, replayed with new tokens and longer contexts."""
    dev, B = cuda_device, 4
    q, cache, bt, cl = attention_case(dev, B, 8, 2, 128, 16, torch.bfloat16, torch.int8, [90, 17, 200, 64], extra=1)
    cos, sin = WL.rope_tables(512, 128, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    x = [torch.randn(B, h, 128, generator=g, device=dev).bfloat16() for h in (8, 2, 2)]
    pos = cl.long().clone()
    slots = torch.empty(B, dtype=torch.long, device=dev)
    put = lambda: slots.copy_(torch.gather(bt.long(), 1, (pos // 16)[:, None])[:, 0] * 16 + pos % 16)  # noqa: E731
    put()
    cl += 1

    def step():
        qr = K.rope_kv_append_paged_quant(*x, pos, cos, sin, slots, *cache)
        return qr, K.paged_attention_quant(qr, *cache, bt, cl)

    step()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        qr, out = step()
    for _ in range(3):
        pos += 1
        cl += 1
        put()
        for t in x:
            t.copy_(torch.randn(t.shape, generator=g, device=dev))
        gr.replay()
        torch.cuda.synchronize()
        check_rows(out, qr, *cache, bt, cl)


@pytest.mark.parametrize("op,shape,dtype", [
    ("rope_kv_append_paged_quant", "T=16", "bf16"), ("rope_kv_append_paged_quant", "T=20,e4m3=1", "fp16"),
    ("paged_kv_dequant", "", "bf16"), ("paged_kv_dequant", "e4m3=1,D=64", "fp16"),
    ("paged_attention_quant", "", "bf16"), ("paged_attention_quant", "B=3,H=8,H_kv=2,e4m3=1", "fp16"),
    ("paged_attention_prefix", "", "bf16"), ("paged_attention_prefix", "quant=1", "fp16"),
    ("paged_attention_prefix", "e4m3=1,B=70", "bf16")])
def test_correctness_gate(op, shape, dtype, tmp_path):
    res = CliRunner().invoke(cli.main, ["verify-correctness", op, "--shape", shape, "--dtype", dtype])
    assert res.exit_code == 0, res.output


# --------------------------------------------------------------------- refusals
def refused(code, fn, *a, **kw):
    with pytest.raises(L.B200OpsError) as e:
        fn(*a, **kw)
    assert e.value.code == code


def test_refusals(cuda_device):
    dev = cuda_device
    q, cache, bt, cl = attention_case(dev, 2, 8, 2, 128, 16, torch.bfloat16, torch.int8, [20, 30])
    kc, vc, ks, vs = cache
    att = K.paged_attention_quant
    refused(L.ERR_NO_DEVICE, att, q.cpu(), *cache, bt, cl)
    refused(L.ERR_BAD_ARG, att, q, kc, vc, ks.transpose(1, 2), vs, bt, cl)
    refused(L.ERR_BAD_ARG, att, q, kc, vc, ks.half(), vs, bt, cl)
    refused(L.ERR_BAD_ARG, att, q, kc, vc.view(torch.float8_e4m3fn), ks, vs, bt, cl)
    refused(L.ERR_UNSUPPORTED, att, q, kc.bfloat16(), vc.bfloat16(), ks, vs, bt, cl)
    refused(L.ERR_BAD_ARG, att, q[:, :7].contiguous(), *cache, bt, cl)
    refused(L.ERR_BAD_ARG, att, q.transpose(0, 1).contiguous().transpose(0, 1), *cache, bt, cl)
    refused(L.ERR_UNSUPPORTED, att, q.float(), *cache, bt, cl)
    refused(L.ERR_UNSUPPORTED, att, q, *cache, bt.float(), cl)
    refused(L.ERR_BAD_ARG, att, q, *cache, bt, cl[:1])
    refused(L.ERR_BAD_ARG, att, q, *cache, bt, cl, out=torch.empty_like(q).half())
    refused(L.ERR_BAD_ARG, att, q, *cache, bt[:, :0], cl)
    pre = K.paged_attention_prefix
    pt, pl = bt[0].clone(), cl[:1]
    refused(L.ERR_BAD_ARG, pre, q, kc, vc, pt, pl, bt, cl)  # scales missing
    refused(L.ERR_BAD_ARG, pre, q, kc.bfloat16(), vc.bfloat16(), pt, pl, bt, cl, ks, vs)
    refused(L.ERR_BAD_ARG, pre, q, kc.half(), vc.half(), pt, pl, bt, cl)
    refused(L.ERR_BAD_ARG, pre, q, kc, vc, pt, cl, bt, cl, ks, vs)  # one length, not two
    refused(L.ERR_BAD_ARG, pre, q, kc, vc, pt[:0], pl, bt, cl, ks, vs)
    x = append_inputs(4, 8, 2, 128, torch.bfloat16, 32, 16, torch.int8)
    d = [t.to(dev) for t in x[:7]]
    app = K.rope_kv_append_paged_quant
    refused(L.ERR_UNSUPPORTED, app, *d[:6], d[6].int(), *cache)
    refused(L.ERR_BAD_ARG, app, *d[:6], d[6][:3], *cache)
    refused(L.ERR_BAD_ARG, app, d[0], d[1][:, :1].contiguous(), *d[2:], *cache)
    refused(L.ERR_BAD_ARG, app, d[0][:2], *d[1:], *cache)
    refused(L.ERR_UNSUPPORTED, app, *(t.float() for t in d[:3]), *d[3:], *cache)
    refused(L.ERR_UNSUPPORTED, app, *d[:4], d[4].half(), d[5].half(), d[6], *cache)
    refused(L.ERR_BAD_ARG, K.paged_kv_dequant, *cache, bt, cl, -1)
    refused(L.ERR_BAD_ARG, K.paged_kv_dequant, *cache, bt, cl, 8, k_out=torch.empty(2, 2, 9, 128, device=dev).bfloat16())
    refused(L.ERR_UNSUPPORTED, K.paged_kv_dequant, *cache, bt, cl, 8, dtype=torch.float32)


def test_empty_calls(cuda_device):
    dev = cuda_device
    q, cache, bt, cl = attention_case(dev, 2, 8, 2, 128, 16, torch.bfloat16, torch.int8, [20, 30])
    assert K.paged_attention_quant(q[:0], *cache, bt[:0], cl[:0]).shape == (0, 8, 128)
    k, v = K.paged_kv_dequant(*cache, bt, cl, 0)
    assert k.shape == v.shape == (2, 2, 0, 128)
    x = append_inputs(4, 8, 2, 128, torch.bfloat16, 32, 16, torch.int8)
    d = [t.to(dev)[:0] if i not in (4, 5) else t.to(dev) for i, t in enumerate(x[:7])]
    before = [t.clone() for t in cache]
    assert K.rope_kv_append_paged_quant(*d, *cache).shape == (0, 8, 128)
    assert all(torch.equal(a, b) for a, b in zip(before, cache))
