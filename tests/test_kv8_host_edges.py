"""The 8-bit cache and shared-prefix entries on the host: calls at the edges of
what their documentation allows."""

import ctypes
import importlib.util
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from b200ops.runtime import lib as L
from b200ops.runtime import ops as K


class Recorder:
    """Stands in for the loaded library: keeps the arguments of each entry and answers
    workspace queries with `size` (a number, or a function of the arguments)."""

    def __init__(self, size=0):
        self.size, self.calls = size, {}

    def __getattr__(self, name):
        def entry(*a):
            self.calls.setdefault(name, []).append(a)
            if name.endswith("_workspace_size"):
                return self.size(*a) if callable(self.size) else self.size
            return L.OK

        return entry


@pytest.fixture
def recorder(monkeypatch):
    """CPU tensors taken as if they were on device 0, entries recorded instead of run."""
    r = Recorder()
    monkeypatch.setattr(L, "load", lambda: r)
    monkeypatch.setattr(K, "_on_one_device", lambda op, *t: 0)
    monkeypatch.setattr(K, "_need_cuda", lambda op, *t: torch.device("cuda", 0))
    monkeypatch.setattr(K, "_elsewhere", lambda dev: False)
    monkeypatch.setattr(K, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(K, "_stream", lambda dev: None)
    monkeypatch.setattr(K.WORKSPACES, "get", lambda dev, n, tag: torch.empty(max(n, 1), dtype=torch.uint8))
    K._scratch_bytes.cache_clear()
    yield r
    K._scratch_bytes.cache_clear()


def decode_args(B=2, pages=4, index=torch.int32, D=128, Hkv=2, code=torch.int8, nb=16, bs=16):
    cache = [torch.zeros(nb, bs, Hkv, D, dtype=code) for _ in range(2)]
    scale = [torch.zeros(nb, Hkv, bs) for _ in range(2)] if code.itemsize == 1 else []
    return (torch.zeros(B, 8, D).bfloat16(), *cache, *scale, torch.zeros(B, pages, dtype=index),
            torch.ones(B, dtype=index))


def test_prefix_workspace_alignment():
    """Piece rows of the prefix are stored 32 bytes at a time: a workspace at 16
    modulo 32 is refused before any launch (a decode's may be there)."""
    lib = L.load()
    p = ctypes.c_void_p(1 << 20)  # an address that is never read
    for code in (L.BF16, L.I8, L.F8E4M3):
        scale = None if code == L.BF16 else p
        need = lib.b200_paged_attention_prefix_workspace_size(2, 8, 2, 128, 16, 16, 8, 4, code, None)
        assert need > 0
        for off in (8, 16, 48):
            assert lib.b200_paged_attention_prefix(
                p, p, p, scale, scale, p, p, p, p, p, 2, 8, 2, 128, 16, 16, 8, 4, 0.0, L.BF16, code, L.I32,
                ctypes.c_void_p((1 << 20) + off), need, None, None) == L.ERR_ALIGNMENT


def launch_flags(arg):
    return arg._obj.flags if arg is not None else 0


@pytest.mark.parametrize("as_struct", [False, True])
@pytest.mark.parametrize("entry", ["b200_paged_attention_quant", "b200_paged_attention"])
def test_rewritten_lengths_and_tables_are_waited_for(entry, as_struct, recorder):
    """Launch flag 8 reads table and lengths before the previous kernel is over.
    Where the wrapper converts or compacts one of them, its own kernel is the
    previous one: the flag is taken off; the other parameters and the caller's stay."""
    quant = entry.endswith("quant")
    op, pos = (K.paged_attention_quant, -2) if quant else (K.paged_attention, -2)
    *front, bt, cl = decode_args(code=torch.int8 if quant else torch.bfloat16)
    cfg = {"flags": 9, "stages": 6}
    if as_struct:
        cfg = L.LaunchCfg.from_dict(cfg)

    def flags(table, lengths):
        op(*front, table, lengths, cfg=cfg)
        got = recorder.calls[entry][-1][pos]
        assert got._obj.stages == 6
        return launch_flags(got)

    assert flags(bt, cl) == 9
    assert flags(bt, cl.long()) == 1
    assert flags(bt, torch.ones(4, dtype=torch.int32)[::2]) == 1
    if quant:
        assert flags(torch.zeros(2, 9, dtype=torch.int32)[:, :4], cl) == 1
    assert flags(bt, cl) == 9
    op(*front, bt, cl.long())
    assert recorder.calls[entry][-1][pos] is None


def test_workspace_of_each_device(monkeypatch, recorder):
    """Workspace sizes follow the current device's SM count: the size of one device is
    not given to a call on another (here: 1000 bytes on device 0, 2000 on 1)."""
    at = [0]
    monkeypatch.setattr(K, "_on_one_device", lambda op, *t: at[0])
    recorder.size = lambda *a: 1000 * (at[0] + 1)
    args = decode_args()
    q, kc, vc, ks, vs, bt, cl = args
    for at[0] in (0, 1, 0):
        K.paged_attention_quant(*args)
        K.paged_attention_prefix(q, kc, vc, bt[0], cl[:1], bt, cl, ks, vs)
        for entry in ("b200_paged_attention_quant", "b200_paged_attention_prefix"):
            assert recorder.calls[entry][-1][-3] == 1000 * (at[0] + 1)


def test_64_bit_lengths_and_ids_beside_a_32_bit_table():
    """Lengths and ids beyond 32 bits stay beyond every table and pool when they
    are brought to the table's type (2^32 + 3 is no length of 3, nor block 3)."""
    far = torch.tensor([5, 0, -7, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 3, -(2 ** 32) + 3, 2 ** 63 - 1, -(2 ** 63)])
    got = K._index("op", "x", far, torch.int32, far.shape)
    top = 2 ** 31 - 1
    assert got.dtype == torch.int32 and got.tolist() == [5, 0, -1, top, top, top, -1, top, -1]
    near = torch.tensor([3, -9], dtype=torch.int32)
    assert K._index("op", "x", near, torch.int64, near.shape).tolist() == [3, -9]
    assert K._index("op", "x", near, torch.int32, near.shape) is near


def test_flash_attn_refuses_keys_of_other_heads(recorder):
    """K and V with fewer heads (as a grouped cache is read back), other sizes or
    another type would be read out of range: refused before the launch."""
    q = torch.zeros(2, 8, 4, 128).bfloat16()
    good = torch.zeros(2, 8, 6, 128).bfloat16()
    K.flash_attn(q, good, good)
    bad = [good[:, :2].contiguous(), good[:1], good[..., :64].contiguous(), good.half(), good[:, :, :5].contiguous()]
    for k, v in [(b, good) for b in bad] + [(good, b) for b in bad]:
        with pytest.raises(L.B200OpsError) as e:
            K.flash_attn(q, k, v)
        assert e.value.code == L.ERR_BAD_ARG
    assert len(recorder.calls["b200_flash_attn"]) == 1


def test_build_refuses_too_few_registers_for_the_split():
    """The prefix kernel's register split waits for good with fewer registers at
    launch than it hands out: the build reads ptxas's report and stops."""
    spec = importlib.util.spec_from_file_location("lib_build", Path(K.__file__).resolve().parents[2] / "build.py")
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    entry = ("ptxas info    : Compiling entry function '_ZN4b20018prefix_attn_kernelI{0}EEv' for 'sm_100a'\n"
             "ptxas info    : Function properties for _ZN4b20018prefix_attn_kernelI{0}EEv\n"
             "    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads\n"
             "ptxas info    : Used {1} registers, used 2 barriers\n")
    other = entry.replace("18prefix_attn_kernel", "24paged_attn_pieces_kernel").format("x", 90)
    for src, need in (("kv_attn_16.cu", 168), ("kv_attn_i8.cu", 128), ("kv_attn_e4m3.cu", 128)):
        b.check_registers(src, other + entry.format("6__half", need) + other + entry.format("13__nv_bfloat16", need + 8))
        with pytest.raises(RuntimeError, match="registers"):
            b.check_registers(src, entry.format("6__half", need) + other + entry.format("13__nv_bfloat16", need - 8))
        with pytest.raises(RuntimeError, match="no register report"):
            b.check_registers(src, other)


GRANT_RACE = r"""
#include <cuda_runtime.h>
#include <atomic>
#include <cstdio>
#include <thread>
static std::atomic<int> attribute{49152}, asked{0};
static cudaError_t fake_device(int* d) { *d = 0; return cudaSuccess; }
// the first two requests meet here, the larger one takes effect first
template <typename K>
static cudaError_t fake_set(K, cudaFuncAttribute, int bytes) {
  const int n = asked.fetch_add(1);
  if (n < 2) for (int i = 0; i < 500 && asked.load() < 2; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
  if (n < 2 && bytes < 200000) std::this_thread::sleep_for(std::chrono::milliseconds(200));
  attribute.store(bytes);
  return cudaSuccess;
}
#define cudaGetDevice fake_device
#define cudaFuncSetAttribute fake_set
#include "common.cuh"
static void kernel() {}
int main() {
  static b200::SmemGrant grant;
  std::thread a([] { grant(kernel, 100000); }), b([] { grant(kernel, 200000); });
  a.join(), b.join();
  const int first = attribute.load();
  if (grant(kernel, 200000) != cudaSuccess) return 3;
  std::printf("%d %d\n", first, attribute.load());
  return attribute.load() >= 200000 ? 0 : 1;
}
"""


def test_shared_memory_grants_of_two_threads(tmp_path):
    """Two threads' first calls of one kernel ask for different sizes at once: the
    kernel's limit ends at or above both (against a fake of the CUDA calls)."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(nvcc).exists():
        pytest.skip("no nvcc")
    csrc = Path(K.__file__).resolve().parents[2] / "csrc"
    src, exe = tmp_path / "grant.cu", tmp_path / "grant"
    src.write_text(GRANT_RACE)
    subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", str(csrc), "-o", str(exe),
                    str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
