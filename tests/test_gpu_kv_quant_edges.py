"""The 8-bit cache and shared-prefix operators at the edges of what their
documentation allows: lengths at the ends of their type, weights and queries
spread over many powers of two, and the rarer launch paths."""

import pytest
import torch

from b200ops import workloads as WL
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
