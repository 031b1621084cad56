"""The context's buffers when memory runs out: csrc/context.cu, compiled for the host with a runtime of this file in CUDA's place."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# A runtime with a limited memory.  What is allocated is host memory, so that a use after free or a null pointer would show.
RUNTIME = r"""
#include "context.cu"

#include <map>

static std::map<void*, size_t> blocks;
static size_t room = 0;
static int copies = 0;
static cudaError_t last = cudaSuccess;
static cudaError_t said(cudaError_t e) { if (e != cudaSuccess) last = e; return e; }

extern "C" {
cudaError_t cudaMalloc(void** p, size_t n) {
    size_t used = 0;
    for (auto& b : blocks) used += b.second;
    if (used + n > room) return said(cudaErrorMemoryAllocation);
    *p = ::malloc(n);
    blocks[*p] = n;
    return cudaSuccess;
}
cudaError_t cudaFree(void* p) {
    if (!p) return cudaSuccess;
    if (!blocks.erase(p)) return said(cudaErrorInvalidValue);
    ::free(p);
    return cudaSuccess;
}
cudaError_t cudaGetLastError() { const cudaError_t e = last; last = cudaSuccess; return e; }
const char* cudaGetErrorString(cudaError_t e) { return e == cudaErrorMemoryAllocation ? "out of memory" : "error"; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaGetDeviceCount(int* n) { *n = 1; return cudaSuccess; }
cudaError_t cudaGetDeviceProperties_v2(cudaDeviceProp*, int) { return cudaErrorInvalidValue; }
cudaError_t cudaMemset(void*, int, size_t) { return cudaSuccess; }
cudaError_t cudaMemsetAsync(void*, int, size_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaMemcpyAsync(void*, const void*, size_t, cudaMemcpyKind, cudaStream_t) { copies++; return cudaSuccess; }
cudaError_t cudaHostAlloc(void**, size_t, unsigned) { return cudaErrorInvalidValue; }
cudaError_t cudaFreeHost(void*) { return cudaSuccess; }
cudaError_t cudaStreamCreateWithFlags(cudaStream_t*, unsigned) { return cudaErrorInvalidValue; }
cudaError_t cudaStreamDestroy(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaEventCreate(cudaEvent_t*) { return cudaErrorInvalidValue; }
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaEventSynchronize(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventElapsedTime(float*, cudaEvent_t, cudaEvent_t) { return cudaErrorInvalidValue; }
cudaError_t cudaMemGetInfo(size_t*, size_t*) { return cudaErrorInvalidValue; }
cudaError_t cudaProfilerStart() { return cudaSuccess; }
cudaError_t cudaProfilerStop() { return cudaSuccess; }
}

#define SAY(what) do { if (!(what)) { fprintf(stderr, "line %d: %s\n", __LINE__, #what); return 1; } } while (0)
"""

BUFFER = r"""
    // a call that needs too much fails, and leaves nothing behind that a smaller one would use
    b2_ctx ctx;
    void* at = nullptr;
    room = 64 << 20;
    SAY(GET(&ctx, 1 << 20, &at) == B2_OK && blocks.count(at) && blocks[at] >= 1 << 20);
    SAY(GET(&ctx, 1 << 10, &at) == B2_OK && blocks.count(at) && blocks.size() == 1);
    SAY(GET(&ctx, 1 << 30, &at) == B2_ERR_CUDA);
    SAY(GET(&ctx, 1 << 20, &at) == B2_OK && blocks.count(at) && blocks[at] >= 1 << 20);
    SAY(GET(&ctx, 8 << 20, &at) == B2_OK && blocks.count(at) && blocks[at] >= 8 << 20 && blocks.size() == 1);
    return 0;
"""

CASES = {
    "stage": "#define GET b2_ctx_stage\nint main() {" + BUFFER + "}",
    "scratch": "#define GET b2_ctx_scratch\nint main() {" + BUFFER + "}",
    # prefill's parts of rows, which the calls over 16-bit and 4-bit pages share, and the projections' partial sums
    "parts": r"""
static int32_t GET(b2_ctx* ctx, size_t bytes, void** out) {
    B2_CHECK(b2_ctx_grow(ctx, &ctx->pf_part, &ctx->pf_part_bytes, bytes));
    *out = ctx->pf_part;
    return B2_OK;
}
int main() {""" + BUFFER + "}",
    "partial sums": r"""
static int32_t GET(b2_ctx* ctx, size_t bytes, void** out) {
    B2_CHECK(b2_ctx_grow(ctx, &ctx->tc_partial, &ctx->tc_partial_bytes, bytes));
    *out = ctx->tc_partial;
    return B2_OK;
}
int main() {""" + BUFFER + "}",
    # the error belongs to the call that failed: a kernel's launch after it asks for the last error
    "last error": r"""
int main() {
    b2_ctx ctx;
    void* at = nullptr;
    SAY(b2_malloc(&ctx, 1 << 10, &at) == B2_ERR_CUDA);
    SAY(std::string(b2_last_error()).find("out of memory") != std::string::npos);
    SAY(cudaGetLastError() == cudaSuccess);
    return 0;
}""",
}


@pytest.mark.parametrize("name", CASES)
def test_memory_that_runs_out(tmp_path, name):
    from mlx_llm_b200 import build

    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    src, exe = tmp_path / "case.cpp", tmp_path / "case"
    src.write_text(RUNTIME + CASES[name])
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(build._nvcc()))), "include")
    subprocess.run([cxx, "-std=c++17", "-O1", "-w", "-I", build.CSRC, "-I", cuda, str(src), "-o", str(exe), "-ldl"], check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
