"""The 8-bit cache and shared-prefix operators at the edges of what their
documentation allows: lengths at the ends of their type, weights and queries
spread over many powers of two, and the rarer launch paths."""

import pytest
import torch

from b200ops import workloads as WL
from b200ops.ops.rope_kv_append_paged_quant import reference as RA
from b200ops.runtime import ops as K
from kv8_ref import check_rows, rows64
from test_gpu_kv_quant import CODES, append_inputs, attention_case, expect_append, run_append, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,flags", [(128, 0), (128, 1), (64, 0)])
def test_lengths_at_the_ends_of_64_bits(D, flags, cuda_device):
    """A length past the table means the whole table, up to 2^63 - 1; a negative one none."""
    top = 2 ** 63 - 1
    q, cache, bt, _ = attention_case(cuda_device, 4, 8, 2, D, 16, torch.bfloat16, torch.int8, [50] * 4, index=torch.int64)
    cl = torch.tensor([top, top - 7, -top - 1, 49], device=cuda_device)
    n = [64, 64, 0, 49]
    out = K.paged_attention_quant(q, *cache, bt, cl, cfg={"flags": flags})
    check_rows(out, q, *cache, bt, torch.tensor(n))
    pt, pl = bt[3].clone(), torch.tensor([top], device=cuda_device)
    out = K.paged_attention_prefix(q, cache[0], cache[1], pt, pl, bt, cl, cache[2], cache[3], cfg={"flags": flags})
    check_rows(out, q, *cache, bt, torch.tensor(n), pt, 64)
    kd, _ = K.paged_kv_dequant(*cache, bt, cl, 70)
    for b in range(4):
        want = torch.zeros(2, 70, D, dtype=torch.float64, device=cuda_device)
        want[:, : n[b]] = rows64(cache[0], cache[2], bt[b], n[b]).transpose(0, 1)
        assert torch.equal(kd[b], want.to(torch.bfloat16))


@pytest.mark.parametrize("T,Hq,Hkv,D,bs,code", [(900, 3, 2, 64, 16, torch.int8), (900, 0, 3, 80, 5, torch.float8_e4m3fn),
                                                (600, 240, 12, 128, 16, torch.int8), (700, 4, 140, 128, 32, torch.int8),
                                                (2600, 8, 2, 128, 16, torch.float8_e4m3fn)])
def test_colliding_slots_of_many_tokens(T, Hq, Hkv, D, bs, code, cuda_device):
    """More than 512 tokens with shared slots: other head dims (general kernel), more
    rows a token than a CTA holds (264 and 284), and many shared slots: the last token
    that writes a slot is found in it, tokens out of range hide nothing."""
    nb = (T + bs - 1) // bs + 10
    x = list(append_inputs(T, Hq, Hkv, D, torch.bfloat16, nb, bs, code, seed=T))
    g = torch.Generator().manual_seed(T)
    slots, pos = x[6].clone(), x[3].clone()
    slots[torch.randperm(T, generator=g)[: T // 4]] = int(slots[0])  # a quarter of the tokens, one slot
    half = torch.randperm(T, generator=g)[: T // 2]
    slots[half] = slots[half.flip(0)]  # pairs
    slots[5], slots[T // 3] = -1, nb * bs
    slots[T - 2] = slots[T - 1] = slots[3]
    pos[T - 1], pos[T // 2] = 600, -3
    x[6], x[3] = slots, pos
    same(run_append(x, cuda_device), expect_append(x))


def test_unaligned_append_of_many_tokens(cuda_device):
    """K at 2 bytes past an aligned address: the general kernel, with shared slots."""
    x = list(append_inputs(700, 2, 2, 128, torch.float16, 60, 16, torch.int8, seed=3))
    x[6][100:140] = x[6][600:640].clone()
    flat = torch.empty(x[1].numel() + 1, dtype=torch.float16, device=cuda_device)
    k = flat[1:].view_as(x[1]).copy_(x[1])
    assert k.data_ptr() % 16 == 2
    q, _, v, pos, cos, sin, slots, c = x
    d = [t.to(cuda_device) for t in (q, k, v, pos, cos, sin, slots)]
    d[1] = k
    cache = [t.to(cuda_device).clone() for t in (c.k_cache, c.v_cache, c.k_scale, c.v_scale)]
    same((K.rope_kv_append_paged_quant(*d, *cache), cache), expect_append(x))


@pytest.mark.parametrize("code", [None, torch.int8])
def test_prefix_batch_of_more_segments_than_a_launch_takes(code, cuda_device):
    """Eight head groups a sequence, 2400 segments: the call runs in slices of 256
    sequences that share a workspace, prefix, own pages and join in turn."""
    B, Hkv, n = 300, 64, 200
    g = torch.Generator().manual_seed(2)
    ctx = [int(c) for c in torch.randint(0, 40, (B,), generator=g)]
    q, cache, bt, cl = attention_case(cuda_device, B, Hkv, Hkv, 128, 16, torch.float16, code, ctx, nb=1000)
    pt = torch.randint(0, 1000, (13,), generator=g).to(cuda_device, torch.int32)
    pl = torch.tensor([n], dtype=torch.int32, device=cuda_device)
    run = lambda: K.paged_attention_prefix(q, cache[0], cache[1], pt, pl, bt, cl, cache[2], cache[3])  # noqa: E731
    out = run()
    torch.cuda.synchronize()
    assert K.read_device_error() == 0
    for b in (0, 1, 100, 255, 256, 257, 299):
        check_rows(out[b:b + 1], q[b:b + 1], *cache, bt[b:b + 1], cl[b:b + 1], pt, n)
    assert torch.equal(out, run())


def loud_key_case(dev, code, dtype, B, n, at, Hkv=8, G=4, bs=16):
    """n tokens of which one (at) has a logit that leaves the others weights of 2^-20 to
    2^-31 of its own, by head, and a value only in dim 0 (16-bit caches: none): dims 1..
    of the output are the flat tail alone.  Tail keys are zero (their logits are exactly
    0), tail values' largest element is the loud one's.  The same pages for every sequence."""
    D, Hq = 128, Hkv * G
    g = torch.Generator().manual_seed(n)
    k, v = torch.zeros(n, Hkv, D), 100 * torch.rand(n, Hkv, D, generator=g) - 30
    v[:, :, 0], v[:, :, 1] = 0, 100
    k[at, :, 0], v[at] = 8, 0
    if code is not None:
        v[at, :, 0] = 100
    want_bits = torch.linspace(20.3, 31.3, Hq)  # log2 of loud over tail
    q = torch.zeros(B, Hq, D)
    q[:, :, 0] = want_bits * (D ** 0.5 / 1.4426950408889634 / 8)
    nb = (n + bs - 1) // bs
    pad = lambda t: torch.cat((t, torch.zeros(nb * bs - n, *t.shape[1:]))).reshape(nb, bs, Hkv, D)  # noqa: E731
    if code is None:
        cache = (pad(k).to(dtype).to(dev), pad(v).to(dtype).to(dev), None, None)
    else:
        (kc, ks), (vc, vs) = (RA.quantise_rows(pad(t), code) for t in (k, v))
        cache = tuple(t.to(dev).contiguous() for t in (kc, vc, ks.transpose(1, 2), vs.transpose(1, 2)))
    table = torch.arange(nb, dtype=torch.int32, device=dev)
    return q.to(dtype).to(dev), cache, table


def check_tail(out, q, cache, table, n):
    """Dims 1.. of every row against 64 bits.  A weight w_t (the largest is in [2^7, 2^15]
    where it is held) rounds to f16: 2^-11 of itself, or 2^-25 where it is subnormal, which is
    2^-32 of the largest; times at most 100 and n of them over a sum of that largest or more.
    The logits are one product each (fp32, up to 31 in log2 units: 31 * 4 roundings of 2^-24),
    exponentials and scale factors 2^-18 relative, sums n 2^-23; the output rounds once more (fp16:
    at least 2^-25 absolute)."""
    K64, V64 = rows64(cache[0], cache[2], table, n), rows64(cache[1], cache[3], table, n)
    G = q.shape[1] // K64.shape[1]
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[q.dtype]
    x = torch.einsum("hd,nhd->hn", q[0].double(), K64.repeat_interleave(G, 1)) / 128 ** 0.5
    want = torch.einsum("hn,nhd->hd", torch.softmax(x, -1), V64.repeat_interleave(G, 1))[:, 1:]
    mean = torch.einsum("hn,nhd->hd", torch.softmax(x, -1), V64.abs().repeat_interleave(G, 1))[:, 1:]
    bound = mean * (2.0 ** -11 + 2.0 ** -17 + 2.0 ** -18 + n * 2.0 ** -23) + 100 * n * 2.0 ** -32
    bound = bound * (1 + 2.0 ** -7) + u * (want.abs() + bound) + 2.0 ** -25
    off = (out[:, :, 1:].double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())


TAIL = [(None, torch.float16), (torch.float8_e4m3fn, torch.float16), (torch.float8_e4m3fn, torch.bfloat16)]


@pytest.mark.parametrize("at", [0, 150, 299])
@pytest.mark.parametrize("code,dtype", [*TAIL, (torch.int8, torch.float16)])
def test_flat_tail_behind_a_loud_key_in_the_prefix(code, dtype, at, cuda_device):
    """Weights that the second product takes as f16: a tail far below the largest keeps
    its bits (16-bit prefix in fp16, 8-bit prefixes)."""
    n = 300
    for B in (20, 70):  # one row tile of query rows, and three
        q, cache, pt = loud_key_case(cuda_device, code, dtype, B, n, at)
        pl = torch.tensor([n], dtype=torch.int32, device=cuda_device)
        none = torch.zeros(B, dtype=torch.int32, device=cuda_device)
        bt = torch.zeros(B, 1, dtype=torch.int32, device=cuda_device)
        check_tail(K.paged_attention_prefix(q, cache[0], cache[1], pt, pl, bt, none, cache[2], cache[3]), q, cache, pt, n)


@pytest.mark.parametrize("at", [0, 150, 299])
@pytest.mark.parametrize("code,dtype", TAIL)
def test_flat_tail_behind_a_loud_key_in_own_pages(code, dtype, at, cuda_device):
    """The same in the streaming kernel: own pages beside an empty prefix, and (8-bit) a decode."""
    n, B = 300, 150
    q, cache, table = loud_key_case(cuda_device, code, dtype, B, n, at)
    bt = table.expand(B, -1).contiguous()
    cl = torch.full((B,), n, dtype=torch.int32, device=cuda_device)
    zero = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    check_tail(K.paged_attention_prefix(q, cache[0], cache[1], table, zero, bt, cl, cache[2], cache[3]), q, cache, table, n)
    if code is not None:
        for b in (20, B):  # a CTA a segment, and ranges
            check_tail(K.paged_attention_quant(q[:b], *cache, bt[:b], cl[:b]), q, cache, table, n)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype,loud", [(torch.float16, 3e4), (torch.bfloat16, 1e5), (torch.bfloat16, 1e6)])
@pytest.mark.parametrize("Hkv,G,rows", [(8, 4, "one"), (2, 8, "all"), (1, 1, "all")])
def test_loud_query_element_over_silent_key_channels(Hkv, G, rows, dtype, loud, code, cuda_device):
    """Query rows with one element far above the others, over key channels that hold
    zeros: the logits are those of the other elements, which keep their bits.  Few
    tokens, so that a logit's error is the output's (bounds of kv8_ref, which count no
    term of the row's largest element); other rows of the batch without such an element."""
    B, D = 6, 128
    ctx = [2, 3, 2, 5, 2, 40]
    g = torch.Generator().manual_seed(int(loud))
    k, v = (torch.randn(60, 16, Hkv, D, generator=g) for _ in range(2))
    k[..., 17] = 0
    (kc, ks), (vc, vs) = (RA.quantise_rows(t, code) for t in (k, v))
    cache = [t.to(cuda_device).contiguous() for t in (kc, vc, ks.transpose(1, 2), vs.transpose(1, 2))]
    q = torch.randn(B, Hkv * G, D, generator=g).to(dtype)
    if rows == "one":
        q[0, 2, 17], q[3, Hkv * G - 1, 17] = loud, -loud
    else:
        q[..., 17] = loud
    q = q.to(cuda_device)
    bt = torch.randperm(60, generator=g)[: B * 3].reshape(B, 3).to(cuda_device, torch.int32)
    cl = torch.tensor(ctx, dtype=torch.int32, device=cuda_device)
    check_rows(K.paged_attention_quant(q, *cache, bt, cl), q, *cache, bt, cl)
    wide = torch.cat((bt, torch.full((B, 60), -1, dtype=torch.int32, device=cuda_device)), 1)  # (ranges and a join)
    check_rows(K.paged_attention_quant(q, *cache, wide, cl), q, *cache, wide, cl)
    pt, pl = bt[5].clone(), cl[5:].clone()
    check_rows(K.paged_attention_prefix(q, cache[0], cache[1], pt, pl, bt, cl, cache[2], cache[3]), q, *cache, bt, cl, pt,
               40)
