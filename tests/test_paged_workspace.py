"""Bytes of mi_paged_attn_workspace_size, without a GPU. The HIP runtime's answers about devices are
replaced by those of a small library that is loaded first, in a process of its own."""
import subprocess
import sys

import pytest

STUB = r"""
#include <hip/hip_runtime_api.h>
#include <string.h>
extern "C" hipError_t hipGetDeviceCount(int* n) { *n = 1; return hipSuccess; }
extern "C" hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
#undef hipGetDeviceProperties
extern "C" hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
  memset(p, 0, sizeof(*p));
  strcpy(p->gcnArchName, "gfx950:sramecc+:xnack-");
  p->multiProcessorCount = CUS;
  return hipSuccess;
}
"""

PROGRAM = """
import ctypes, sys
ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
L = ctypes.CDLL(sys.argv[2])
f = L.mi_paged_attn_workspace_size
f.restype, f.argtypes = ctypes.c_size_t, [ctypes.c_int64] * 7
shapes = [(8, 2, 128, 1, 1, 1, 32768), (16, 4, 128, 64, 64, 1, 8000), (16, 4, 128, 1, 512, 512, 32768)]
if sys.argv[3] == "later":  # another query has looked at the devices before
    L.mi_gemm_workspace_size.restype = ctypes.c_size_t
    i = ctypes.c_int64(256)
    L.mi_gemm_workspace_size(0, 0, i, i, i, 1, 0, ctypes.c_int64(1))
print([f(*s) for s in shapes])
"""


def sizes(cus):
    """Bytes for a device of that many CUs, from the layout of the workspace: pieces of [rows][heads][d + 1]
    floats, or shares, two parts of [heads][d + 1] each, and a sum for each sequence and one more."""
    pieces = cus // 2                     # a workgroup a CU of the 2 KV heads
    share = 2 * cus // 4                  # two a CU, of 4 KV heads
    rows = 512 * 16 // 4 // 128 * 4       # row tiles and KV heads of the prompt
    many = -(-2 * cus // rows)            # two a CU
    return [pieces * 8 * 129 * 4, 2 * share * 16 * 129 * 4 + 65 * 4, many * 512 * 16 * 129 * 4]


@pytest.mark.parametrize("cus", [128, 256])
def test_bytes_follow_the_device_from_the_first_call_on(mi, tmp_path, cus):
    src, lib = tmp_path / "stub.cpp", tmp_path / "stub.so"
    src.write_text(STUB)
    subprocess.run(["g++", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", f"-DCUS={cus}", "-I/opt/rocm/include",
                    str(src), "-o", str(lib)], check=True)

    def ask(how):
        out = subprocess.run([sys.executable, "-c", PROGRAM, str(lib), mi.LIB_PATH, how], check=True, capture_output=True,
                             text=True, timeout=100)
        return eval(out.stdout)

    assert ask("later") == sizes(cus)
    assert ask("first") == sizes(cus)


def test_bytes_without_a_device(mi):
    """Those of 256 CUs."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    f = mi.paged_attn_workspace_size
    assert [f(8, 2, 128, 1, 1, 1, 32768), f(16, 4, 128, 64, 64, 1, 8000), f(16, 4, 128, 1, 512, 512, 32768)] == sizes(256)
    # one piece, nothing to join
    assert f(16, 4, 128, 1, 1, 1, 512) == 0 and f(16, 4, 128, 64, 64, 1, 1000) == 0
    # refused by the call
    for bad in ((16, 3, 128, 4, 4, 1, 100), (0, 1, 128, 4, 4, 1, 100), (16, 4, 0, 4, 4, 1, 100), (16, 4, 128, 4, 0, 1, 100),
                (16, 4, 128, 1, 1 << 31, 1, 100), (1 << 16, 1, 128, 1, 1 << 15, 1 << 15, 100)):
        assert f(*bad) == 0, bad


def test_where_even_shares_begin(mi):
    """1024 keys for each piece that a sequence would be cut into, 2048 at least."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    f = mi.paged_attn_workspace_size
    parts = lambda share, S: 2 * share * 16 * 129 * 4 + (S + 1) * 4  # noqa: E731
    for S, pieces in ((64, 1), (256, 1), (32, 2), (16, 4)):
        border = 1024 * max(pieces, 2)
        assert f(16, 4, 128, S, S, 1, border) == (pieces * S * 16 * 129 * 4 if pieces > 1 else 0)
        assert f(16, 4, 128, S, S, 1, border + 1) == max(parts(128, S), pieces * S * 16 * 129 * 4 if pieces > 1 else 0)
    assert f(16, 4, 128, 1, 1, 1, 10 ** 6) == 64 * 16 * 129 * 4  # one sequence: pieces


def test_rows_that_no_join_could_be_launched_for(mi):
    """The call does not cut them, whatever max_q_len says, and asks for no room to."""
    f = mi.paged_attn_workspace_size
    assert f(16, 4, 128, 1, 1 << 20, 1, 1 << 20) == 0
    assert f(16, 4, 128, 1, (1 << 20) - 1, 1, 1 << 20) > 0
