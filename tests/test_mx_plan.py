"""What tcg_mx_linear launches, on the CPU: the object file of its kernels is linked with a stand-in for the CUDA runtime
that records launches (grid, block, cluster, shared memory) and runs nothing."""
import ctypes as C
import os
import subprocess

import pytest

import tcg

PKG = os.path.dirname(os.path.dirname(tcg.LIB_PATH))
OBJECT = os.path.join(PKG, "_build", "cuda", "mx_linear.o")
P = 1 << 20                          # a pointer that nothing reads
SMS, MOST_SMEM = 148, 227 * 1024

RUNTIME = r"""
#include "tcg_common.cuh"

#include <cuda.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

struct Launch { int grid, block, cluster, smem; };
static Launch last;
static int device, at_once[64], asked;
static char message[256];

namespace tcg {
int g_pdl = 1;
Ctx &ctx()
{
    static thread_local Ctx c;
    c.ready = true, c.device = device, c.sms = 148;
    return c;
}
bool need_ctx() { return true; }
bool fail(const char *fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(message, sizeof message, fmt, ap);
    va_end(ap);
    return false;
}
bool cuda_fail(cudaError_t e, const char *what, const char *, int) { return fail("%s: %d", what, (int)e); }
}

static CUresult encode(CUtensorMap *map, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                       const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill)
{
    memset(map, 0, sizeof *map);
    return CUDA_SUCCESS;
}

extern "C" {
void **__cudaRegisterFatBinary(void *) { static void *handle; return &handle; }
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
void __cudaRegisterFunction(void **, const char *, char *, const char *, int, void *, void *, void *, void *, int *) {}
cudaError_t __cudaPopCallConfiguration(dim3 *, dim3 *, size_t *, void *) { return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaGetDevice(int *d) { *d = device; return cudaSuccess; }
cudaError_t cudaGetDriverEntryPoint(const char *, void **fn, unsigned long long, cudaDriverEntryPointQueryResult *r)
{
    *fn = (void *)encode, *r = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaLaunchKernel(const void *, dim3, dim3, void **, size_t, cudaStream_t) { return cudaErrorUnknown; }
cudaError_t cudaOccupancyMaxActiveClusters(int *n, const void *, const cudaLaunchConfig_t *)
{
    asked++;
    *n = at_once[device];
    return cudaSuccess;
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t *lc, const void *, void **)
{
    last = Launch{ (int)lc->gridDim.x, (int)lc->blockDim.x, 1, (int)lc->dynamicSmemBytes };
    for (unsigned i = 0; i < lc->numAttrs; i++)
        if (lc->attrs[i].id == cudaLaunchAttributeClusterDimension) last.cluster = (int)lc->attrs[i].val.clusterDim.x;
    return cudaSuccess;
}
void set_device(int d, int clusters) { device = d, at_once[d] = clusters; }
int times_asked() { return asked; }
Launch last_launch() { return last; }
const char *last_message() { return message; }
}
"""


class Launch(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("grid", "block", "cluster", "smem")]


@pytest.fixture()
def plan(tmp_path):
    """A fresh copy of the operator's host code, which has seen no device."""
    if not os.path.exists(OBJECT):
        subprocess.run(["make", "-s", "-C", PKG, os.path.relpath(OBJECT, PKG)], check=True)
    src, so = tmp_path / "runtime.cc", tmp_path / "plan.so"
    src.write_text(RUNTIME)
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc"))), "include")
    inc = [cuda, os.path.join(PKG, "csrc", "cuda"), os.path.join(PKG, "csrc"), os.path.join(os.path.dirname(PKG), "include")]
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wl,-Bsymbolic", *("-I" + i for i in inc), "-o", str(so), str(src), OBJECT],
                   check=True)
    lib = C.CDLL(str(so))
    lib.last_launch.restype, lib.last_message.restype = Launch, C.c_char_p
    lib.tcg_mx_linear.restype = C.c_bool
    lib.tcg_mx_linear.argtypes = [C.c_void_p, C.POINTER(tcg.Mx), C.POINTER(tcg.Mx), C.c_void_p, C.c_int64, C.c_int]

    def launch(rows, cols, outs, bits, t=tcg.F32):
        x, w = tcg.Mx(P, P, rows, cols, bits), tcg.Mx(P, P, outs, cols, 4)
        if not lib.tcg_mx_linear(P, C.byref(x), C.byref(w), None, outs, t):
            raise tcg.TcgError(lib.last_message().decode())
        return lib.last_launch()

    launch.device, launch.asked = lib.set_device, lib.times_asked
    return launch


def test_each_device_has_its_own_clusters(plan):
    """How many clusters run at once is the device's: what one has answered is not taken for another."""
    plan.device(0, 1000)
    a = plan(1, 14336, 4096, 8)
    assert a.cluster > 1 and a.grid == 32 * a.cluster                    # 32 tiles, K split
    plan.device(1, 5)                                                    # fewer at once than tiles: undivided
    b = plan(1, 14336, 4096, 8)
    assert b.cluster == 1 and b.grid == 32
    plan.device(0, 1000)
    asked = plan.asked()
    again = plan(1, 14336, 4096, 8)
    assert (again.cluster, again.grid) == (a.cluster, a.grid) and plan.asked() == asked


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("t", [tcg.F32, tcg.BF16])
def test_launches_over_the_range(plan, bits, t):
    """One row to many, one column to 2^24, one output to 2^30: grids of whole clusters or pairs, within shared memory."""
    plan.device(0, 15)
    for rows in (1, 8, 9, 16, 17, 32, 33, 64, 65, 127, 128, 129, 300, 1000, 5000, 1 << 20, 1 << 30):
        for cols in (1, 128, 129, 257, 1100, 4096, 14336, 70000, 1 << 24):
            for outs in (1, 100, 128, 129, 4096, 5003, 60000, 1 << 30):
                if rows * outs > 1 << 44:
                    continue
                p = plan(rows, cols, outs, bits, t)
                assert p.grid > 0 and p.smem <= MOST_SMEM and 1 <= p.cluster <= 8 and p.grid % p.cluster == 0
                assert p.block in (256, 576) and (p.block == 256 or (p.grid % 2 == 0 and p.grid <= SMS))
                if p.cluster > 1:
                    assert p.grid <= SMS and p.grid // p.cluster <= 15


def test_sizes_of_too_many_tiles_are_refused(plan):
    plan.device(0, 15)
    with pytest.raises(tcg.TcgError, match="too many"):
        plan(1 << 30, 128, 1 << 30, 8)
