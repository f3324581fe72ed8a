"""sm_100a CUDA variant of rope_kv_append_paged_quant (libb200ops.so through ctypes).

`sm100(**compile_args)` returns kernel_fn(*inputs) for the inputs produced by
reference.generate_test_inputs, the calling convention of the reference's
Triton templates; compile_args may carry b200_launch_cfg fields chosen by the
tuner.  There is no fallback: without the library or a GPU the call raises.
"""

import torch as _torch  # noqa: F401

from b200ops.ops._variant import make_factory as _make_factory
from b200ops.runtime import ops as _K


def _run(q, k, v, positions, cos, sin, slot_mapping, k_cache, v_cache, k_scale, v_scale, cfg=None):
    q_out = _K.rope_kv_append_paged_quant(q, k, v, positions, cos, sin, slot_mapping, k_cache, v_cache, k_scale,
                                          v_scale, cfg=cfg)

    def values(c):  # codes of an 8-bit floating cache as fp16 values (exact)
        return c if c.dtype == _torch.int8 else c.half()

    return q_out, values(k_cache), values(v_cache), k_scale, v_scale


sm100 = _make_factory(_run, uses_threads=False)
