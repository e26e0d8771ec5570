"""What the C entries set up on the host before a launch, with the CUDA runtime's calls replaced by counting fakes (no GPU, no launch)."""
import json
import os
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest

from torchft_b200 import _build

FAKE = r"""
#include <cuda.h>
#include <cuda_runtime_api.h>
#include <string.h>
#include <unistd.h>
static __thread int device = 0;
static int attributes[8], launches[8];
static CUresult encode(void) { return CUDA_SUCCESS; }
void fake_device(int d) { device = d; }
int fake_attributes(int d) { return attributes[d]; }
int fake_launches(int d) { return launches[d]; }
cudaError_t cudaGetDriverEntryPoint(const char* name, void** f, unsigned long long flags, enum cudaDriverEntryPointQueryResult* q) {
  usleep(100000);  /* long enough for another thread to come here */
  *f = (void*)encode;
  *q = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}
cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, enum cudaDeviceAttr a, int d) { *v = 148; return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void* f, enum cudaFuncAttribute a, int v) { __sync_fetch_and_add(&attributes[device], 1); return cudaSuccess; }
cudaError_t cudaFuncGetAttributes(struct cudaFuncAttributes* a, const void* f) {
  memset(a, 0, sizeof *a);
  a->numRegs = 255;
  return cudaSuccess;
}
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void* f, const cudaLaunchConfig_t* c) { *n = 36; return cudaSuccess; }
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
cudaError_t cudaMemsetAsync(void* p, int v, size_t n, cudaStream_t s) { return cudaSuccess; }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void** a) { __sync_fetch_and_add(&launches[device], 1); return cudaSuccess; }
cudaError_t cudaLaunchKernel(const void* f, dim3 g, dim3 b, void** a, size_t m, cudaStream_t s) { __sync_fetch_and_add(&launches[device], 1); return cudaSuccess; }
"""

# The fakes are in the process before the library; no pointer is followed.
RUN = r"""
import ctypes, json, sys, threading
fakes = ctypes.CDLL(sys.argv[1])
lib = ctypes.CDLL(sys.argv[2])
P, I, L, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
at = 1 << 20
tensors = lambda n: [P(at)] * n
sizes = [I(1), I(512), I(2), I(1), I(128)]
entries = {
    "attention_fwd": [*tensors(5), *sizes, *[L(256)] * 4, F(0.1), I(1), P(at), None],
    "attention_fwd2": [*tensors(5), *sizes, *[L(256)] * 4, F(0.1), I(1), I(0), P(at), None],
    "attention_bwd": [*tensors(10), *sizes, *[L(256)] * 8, F(0.1), I(1), None, P(at), None],
    "attention_masked_fwd": [*tensors(5), None, None, None, None, *sizes, *[L(256)] * 4, F(0.1), F(30.0), I(1), P(at), None],
    "attention_masked_bwd": [*tensors(10), None, None, None, None, *sizes, *[L(256)] * 8, F(0.1), F(30.0), I(1), None, P(at), None],
    "gemm_bf16": [*tensors(3), I(256), I(256), I(64), I(0), I(0), L(64), L(64), L(256), I(0), P(at), I(0), None],
    "gemm_bf16_2cta": [*tensors(3), I(256), I(256), I(64), I(0), I(0), L(64), L(64), L(256), I(0), P(at), I(0), None],
    "layernorm_bwd": [*tensors(5), None, *tensors(4), L(8), I(64), I(0), I(0), P(at), None],
}
name, what = sys.argv[3], sys.argv[4]
call = lambda: getattr(lib, "ftb200_" + name)(*entries[name])
if what == "threads":
    codes = []
    start = threading.Barrier(4)
    def work():
        start.wait()
        codes.append(call())
    many = [threading.Thread(target=work) for _ in range(4)]
    [t.start() for t in many]
    [t.join() for t in many]
    print(json.dumps(codes))
else:
    seen = []
    for device in (0, 1, 1, 0, 2):
        fakes.fake_device(device)
        assert call() == 0
        seen.append([fakes.fake_attributes(device), fakes.fake_launches(device)])
    print(json.dumps(seen))
"""

ENTRIES = ["attention_fwd", "attention_fwd2", "attention_bwd", "attention_masked_fwd", "attention_masked_bwd", "gemm_bf16", "gemm_bf16_2cta",
           "layernorm_bwd"]


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    where = tmp_path_factory.mktemp("fakes")
    (where / "fakes.c").write_text(FAKE)
    so = where / "fakes.so"
    cmd = ["gcc", "-shared", "-fPIC", "-O1", f"-I{_build._cuda_home()}/include", str(where / "fakes.c"), "-o", str(so)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr
    import nvidia.cuda_runtime  # the runtime that torch brings

    runtime = str(Path(list(nvidia.cuda_runtime.__path__)[0]) / "lib")
    library = _build.build_kernels()

    def one(name, what):
        env = {**os.environ, "LD_PRELOAD": str(so), "CUDA_VISIBLE_DEVICES": "", "LD_LIBRARY_PATH": runtime + ":" + os.environ.get("LD_LIBRARY_PATH", "")}
        proc = subprocess.run([sys.executable, "-c", textwrap.dedent(RUN), str(so), str(library), name, what], capture_output=True, text=True,
                              timeout=120, env=env)
        assert proc.returncode == 0, proc.stderr
        return json.loads(proc.stdout)

    return one


@pytest.mark.parametrize("name", [e for e in ENTRIES if e != "layernorm_bwd"])
def test_first_calls_of_several_threads(run, name):
    """None of them sees another's search for the driver's entry point half done."""
    assert run(name, "threads") == [0, 0, 0, 0]


@pytest.mark.parametrize("name", ENTRIES)
def test_attributes_are_set_on_every_device(run, name):
    """A kernel's limit of shared memory belongs to a device: set once on each that is used, and not at every call."""
    first, other, again, back, third = run(name, "devices")
    assert first[0] == other[0] == third[0] > 0  # of each device
    assert again[0] == other[0] and back[0] == first[0]
    assert again[1] == 2 * other[1] and back[1] == 2 * first[1] and first[1] > 0
