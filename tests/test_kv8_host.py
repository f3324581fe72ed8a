"""The 8-bit cache and shared-prefix entries on the host: refusals that need
no GPU, and their contracts."""

import ctypes

import pytest
import torch

from b200ops import cli
from b200ops.runtime import lib as L
from b200ops.runtime import ops as K

OPS = ["rope_kv_append_paged_quant", "paged_kv_dequant", "paged_attention_quant", "paged_attention_prefix"]


def test_kv8_bad_arguments_rejected_on_host():
    """The 8-bit cache and shared-prefix entries refuse before any launch."""
    lib = L.load()
    p = ctypes.c_void_p(1 << 20)  # an address that is never read

    def append(T=4, Hq=8, Hkv=2, D=128, nb=16, bs=16, dt=L.BF16, cs=L.F32, code=L.I8, ws=None, ws_bytes=0, q=p, k=p,
               cs_rows=10):
        return lib.b200_rope_kv_append_paged_quant(q, k, p, p, p, p, cs_rows, p, q, p, p, p, p, T, Hq, Hkv, D, nb, bs,
                                                   dt, cs, code, ws, ws_bytes, None, None)

    assert append(D=127) == L.ERR_BAD_ARG and append(cs_rows=0) == L.ERR_BAD_ARG and append(T=-1) == L.ERR_BAD_ARG
    assert append(k=None) == L.ERR_BAD_ARG
    assert append(code=L.BF16) == L.ERR_UNSUPPORTED and append(dt=L.F32) == L.ERR_UNSUPPORTED
    assert append(cs=L.F16) == L.ERR_UNSUPPORTED
    assert append(T=513) == L.ERR_WORKSPACE  # many tokens need the claim table
    need = lib.b200_rope_kv_append_paged_quant_workspace_size(513)
    assert need > 0 and lib.b200_rope_kv_append_paged_quant_workspace_size(512) == 0
    assert append(T=513, ws=p, ws_bytes=need - 1) == L.ERR_WORKSPACE
    assert append(T=0) == L.OK

    def attend(B=2, Hq=8, Hkv=2, D=128, bs=16, maxb=4, dt=L.BF16, code=L.I8, ix=L.I32, ks=p, ws=None, n=0):
        return lib.b200_paged_attention_quant(p, p, p, ks, p, p, p, p, B, Hq, Hkv, D, 16, bs, maxb, 0.0, dt, code, ix,
                                              ws, n, None, None)

    assert attend(Hq=9) == L.ERR_BAD_ARG and attend(maxb=0) == L.ERR_BAD_ARG and attend(ks=None) == L.ERR_BAD_ARG
    assert attend(code=L.BF16) == L.ERR_UNSUPPORTED and attend(dt=L.F32) == L.ERR_UNSUPPORTED
    assert attend(ix=L.I8) == L.ERR_UNSUPPORTED and attend(D=257 * 2) == L.ERR_UNSUPPORTED
    assert attend(maxb=40) == L.ERR_WORKSPACE
    need = lib.b200_paged_attention_quant_workspace_size(2, 8, 2, 128, 16, 16, 40, None)
    assert need > 0 and lib.b200_paged_attention_quant_workspace_size(2, 8, 2, 128, 16, 16, 4, None) == 0  # short tables
    assert attend(maxb=40, ws=p, n=need - 1) == L.ERR_WORKSPACE
    assert attend(maxb=40, ws=ctypes.c_void_p((1 << 20) + 8), n=need) == L.ERR_ALIGNMENT
    assert attend(B=0) == L.OK

    def prefix(B=2, P=4, maxb=4, dt=L.BF16, code=L.BF16, table=p):
        return lib.b200_paged_attention_prefix(p, p, p, None, None, table, p, p, p, p, B, 8, 2, 128, 16, 16, P, maxb,
                                               0.0, dt, code, L.I32, None, 0, None, None)

    assert prefix(P=0) == L.ERR_BAD_ARG and prefix(table=None) == L.ERR_BAD_ARG and prefix(maxb=-1) == L.ERR_BAD_ARG
    assert prefix(code=L.F16) == L.ERR_UNSUPPORTED and prefix(code=L.I8) == L.ERR_BAD_ARG  # scales missing
    assert prefix(B=0) == L.OK

    def dequant(max_len=4, code=L.I8, dt=L.BF16, out=p):
        return lib.b200_paged_kv_dequant(p, p, p, p, p, p, out, p, 2, 2, 128, 16, 16, 4, max_len, dt, code, L.I32, None,
                                         None)

    assert dequant(max_len=-1) == L.ERR_BAD_ARG and dequant(out=None) == L.ERR_BAD_ARG
    assert dequant(code=L.F16) == L.ERR_UNSUPPORTED and dequant(dt=L.F32) == L.ERR_UNSUPPORTED
    assert dequant(max_len=0) == L.OK


def test_discovered_with_contract_and_reference():
    for op in OPS:
        assert list(cli.load_templates(op)) == ["cuda_v1.sm100"]
        ref, gen = cli.load_reference(op)
        assert callable(ref) and callable(gen)
        assert L.config_space(op)["op"] == op


def test_no_cpu_path():
    t = torch.zeros(2, 16, 2, 128, dtype=torch.int8)
    s = torch.zeros(2, 2, 16)
    i = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(L.B200OpsError) as e:
        K.paged_attention_quant(torch.zeros(1, 4, 128).bfloat16(), t, t, s, s, i, i[0, :1])
    assert e.value.code == L.ERR_NO_DEVICE


def test_host_fault_injection(monkeypatch):
    lib, p = L.load(), ctypes.c_void_p(1 << 20)
    monkeypatch.setenv("B200OPS_INJECT_ERROR", "paged_attention_quant")
    assert lib.b200_paged_attention_quant(p, p, p, p, p, p, p, p, 1, 1, 1, 128, 1, 16, 1, 0.0, L.BF16, L.I8, L.I32,
                                          None, 0, None, None) == L.ERR_INJECTED
