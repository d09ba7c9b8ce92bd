"""Calls whose workgroups have more threads together than a launch can count (2^32), from a host without a GPU:
the runtime's devices and launches are those of a small library that is loaded first, in a process of its own. A
launch there is noted, or fails if it has too many threads, as the runtime's does."""
import subprocess
import sys

import pytest

STUB = r"""
#include <hip/hip_runtime_api.h>
#include <stdint.h>
#include <string.h>
static uint64_t grids[512], args0[512];
static int n;
static hipError_t last = hipSuccess;
extern "C" hipError_t hipGetDeviceCount(int* c) { *c = 1; return hipSuccess; }
extern "C" hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
extern "C" hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
  memset(p, 0, sizeof(*p));
  strcpy(p->gcnArchName, "gfx950:sramecc+:xnack-");
  p->multiProcessorCount = 256;
  return hipSuccess;
}
static dim3 grid, block;
extern "C" hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t, hipStream_t) {
  grid = g, block = b;
  return hipSuccess;
}
extern "C" hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, hipStream_t* stream) {
  *g = grid, *b = block, *lds = 0, *stream = nullptr;
  return hipSuccess;
}
extern "C" hipError_t hipLaunchKernel(const void*, dim3 g, dim3 b, void** args, size_t, hipStream_t) {
  if ((uint64_t)g.x * b.x > UINT32_MAX) return last = hipErrorInvalidConfiguration;
  if (n < 512) {
    memcpy(&args0[n], args[0], 8);
    grids[n++] = (uint64_t)g.x << 16 | b.x;
  }
  return hipSuccess;
}
extern "C" hipError_t hipGetLastError() { const hipError_t e = last; last = hipSuccess; return e; }
extern "C" int noted(uint64_t* out) {  // grid << 16 | threads and the first eight bytes of the arguments
  for (int i = 0; i < n; ++i) out[2 * i] = grids[i], out[2 * i + 1] = args0[i];
  const int c = n;
  n = 0;
  return c;
}
"""

PROGRAM = """
import ctypes, sys
S = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
sys.path[:0] = [sys.argv[2], sys.argv[3]]
import mi_gemm as mi
import test_serve_abi as t

def launches():
    out = (ctypes.c_uint64 * 1024)()
    n = S.noted(out)
    return [(out[2 * i] >> 16, out[2 * i] & 0xffff, out[2 * i + 1]) for i in range(n)]

print(eval(sys.argv[4]))
"""


@pytest.fixture(scope="module")
def ask(mi, tmp_path_factory):
    import os

    d = tmp_path_factory.mktemp("stub")
    (d / "stub.cpp").write_text(STUB)
    subprocess.run(["g++", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", str(d / "stub.cpp"), "-o",
                    str(d / "stub.so")], check=True)

    def f(what):
        out = subprocess.run([sys.executable, "-c", PROGRAM, str(d / "stub.so"), os.path.dirname(mi.LIB_PATH),
                              os.path.dirname(os.path.abspath(__file__)), what], check=True, capture_output=True, text=True,
                             timeout=100)
        return eval(out.stdout)

    return f


@pytest.mark.parametrize("rows,dtype,es", [(1, 1, 2), (300, 1, 2), (8388607, 1, 2), (8388608, 1, 2), (2 ** 31 - 1, 0, 4)])
def test_rows_of_the_sampler(ask, rows, dtype, es):
    st, got = ask(f"t.sample(mi, rows={rows}, V=3, ld=5, dtype={dtype}), launches()")
    assert st == 0
    at = 0
    for grid, threads, logits in got:
        assert grid * threads < 2 ** 32 and logits == (1 << 20) + at * 5 * es
        at += grid
    assert at == rows and len(got) == -(-rows // 8388607)


@pytest.mark.parametrize("tokens", [1, 2 ** 28 - 16, 2 ** 28 - 15, 2 ** 31 - 1])
def test_tokens_of_a_rotation(ask, tokens):
    st, got = ask(f"t.rope(mi, B=1, T={tokens}, d=2, heads=1, rot=t.rotary(mi, rot_dim=2)), launches()")
    assert st == 0
    assert all(g * b < 2 ** 32 for g, b, _ in got)
    each = 16 if tokens > 1 else 1
    assert sum(g for g, _, _ in got) == -(-tokens // each) and len(got) == -(-tokens // (each * (2 ** 24 - 1)))


def test_rows_and_tiles_of_the_attention(ask):
    # one new token of each of many sequences: a workgroup for each and each KV head
    st, got = ask("t.attend(mi, s=t.seqs(mi, n_seqs=(1 << 23) - 1, total_q=(1 << 23) - 1, q_start=0), mq=1), launches()")
    assert st == 0 and [g for g, _, _ in got] == [2 * ((1 << 23) - 1)]
    st, got, text = ask("t.attend(mi, s=t.seqs(mi, n_seqs=1 << 23, total_q=1 << 23, q_start=0), mq=1), launches(), t._msg(mi)")
    assert st == 1 and not got and "workgroups" in text
    # a million times more rows than max_q_len says: right, and not cut into pieces that nothing could join
    st, got = ask("t.attend(mi, s=t.seqs(mi, n_seqs=1, total_q=5 << 20), mq=1, mk=1 << 20, ws=1 << 20, wsb=1 << 50), launches()")
    assert st == 0 and len(got) == 1 and got[0][0] * got[0][1] < 2 ** 32
