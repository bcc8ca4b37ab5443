"""The launches of the library's entry points at their largest sizes, without a
GPU: a program that puts its own functions in place of HIP's notes every launch
instead of making it."""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

PROGRAM = r"""
#include <hip/hip_runtime_api.h>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>
#include <vector>
#include "myl_hip.h"

// ---- HIP, as far as the entry points ask for it ----
struct Launch { dim3 grid, block; size_t lds; };
static std::vector<Launch> launches;
static Launch next;
extern "C" {
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t) { return next = {grid, block, lds}, hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, hipStream_t* s) {
    return *grid = next.grid, *block = next.block, *lds = next.lds, *s = nullptr, hipSuccess;
}
hipError_t hipLaunchKernel(const void*, dim3 grid, dim3 block, void**, size_t lds, hipStream_t) {
    launches.push_back({grid, block, lds});
    return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipGetDeviceCount(int* n) { return *n = 1, hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
    std::memset((void*)p, 0, sizeof *p);
    p->multiProcessorCount = 256;
    return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) { return *v = 256, hipSuccess; }
hipError_t hipStreamCreate(hipStream_t* s) { return *s = (hipStream_t)0x10, hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipGetSymbolAddress(void** p, const void*) { return *p = (void*)0x100000, hipSuccess; }
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipOccupancyMaxActiveBlocksPerMultiprocessor(int* n, const void*, int, size_t) { return *n = 1, hipSuccess; }
hipError_t hipMalloc(void** p, size_t) { return *p = (void*)0x200000, hipSuccess; }
hipError_t hipFree(void*) { return hipSuccess; }
hipError_t hipMemset(void*, int, size_t) { return hipSuccess; }
}

static long calls = 0, bad = 0;
static void check(const std::string& what, int rc, bool accepted = true) {
    ++calls;
    if ((rc == 0) != accepted) ++bad, std::printf("%s: status %d\n", what.c_str(), rc);
    if (accepted && launches.empty()) ++bad, std::printf("%s: no launch\n", what.c_str());
    if (!accepted && !launches.empty()) ++bad, std::printf("%s: refused behind a launch\n", what.c_str());
    for (const Launch& l : launches) {
        const uint64_t threads = (uint64_t)l.block.x * l.block.y * l.block.z;
        if (l.grid.x == 0 || l.grid.y == 0 || l.grid.z == 0 || l.grid.x * (uint64_t)l.block.x >= (1ull << 32) || l.grid.y > 65535 ||
            l.grid.z > 65535 || threads == 0 || threads > 1024 || l.lds > 160 * 1024) {
            ++bad;
            std::printf("%s: grid %u x %u x %u of %llu threads, %zu bytes\n", what.c_str(), l.grid.x, l.grid.y, l.grid.z, (unsigned long long)threads, l.lds);
        }
    }
    launches.clear();
}
template <class T>
static T* at(size_t n) { return reinterpret_cast<T*>(n); }  // never read on the host

int main() {
    myl_ctx* c = nullptr;
    if (myl_init(0, &c) != MYL_OK) return 2;
    launches.clear();
    const int16_t* x = at<int16_t>(1 << 20);
    const uint8_t* sh = at<uint8_t>(1 << 21);
    int16_t* out = at<int16_t>(1 << 22);
    void* ws = at<void>(1 << 23);
    for (size_t M : {(size_t)1, (size_t)2, (size_t)33, (size_t)65535, (size_t)65536, (size_t)65600, (size_t)131071, (size_t)1 << 20, (size_t)1 << 23})
        for (size_t K : {(size_t)1, (size_t)33, (size_t)64, (size_t)80, (size_t)128, (size_t)131072})
            for (size_t N : {(size_t)1, (size_t)40})
                for (size_t W : {(size_t)0x1000000, (size_t)0x1000001}) {
                    const std::string size = std::to_string(M) + " x " + std::to_string(N) + " x " + std::to_string(K) + (W & 1 ? ", odd weights" : "");
                    for (size_t n : {(size_t)0, (size_t)1, (size_t)300}) {
                        const size_t bytes = myl_linear_w8a16_adapters_workspace(c, M, N, K, 16, n);
                        check("adapters " + std::to_string(n) + ", " + size,
                              myl_linear_w8a16_adapters_dev(c, x, M, K, at<int8_t>(W), N, K, sh, 10, 10, nullptr, at<int32_t>(64), at<int8_t>(64), sh, 10,
                                                            at<int8_t>(64), sh, n, 16, out, N, ws, bytes));
                    }
                    check("projection " + size, myl_linear_w8a16_dev(c, x, M, K, at<int8_t>(W), N, K, sh, 10, 10, nullptr, out, N));
                    check("multipliers " + size, myl_linear_w8a16_mult_dev(c, x, M, K, at<int8_t>(W), N, K, at<int32_t>(64), sh, out, N));
                    if (M <= 1 << 20) {
                        check("head " + size, myl_logits_dev(c, x, M, K, at<void>(W), 8, N, K, sh, 10, 6, at<int32_t>(64), N));
                        check("16-bit head " + size, myl_logits_dev(c, x, M, K, at<void>(W & ~(size_t)1), 16, N, K, sh, 10, 6, at<int32_t>(64), N));
                        check("sums " + size, myl_dot_i8_i16_dev(c, x, M, K, at<int8_t>(W), N, K, at<int64_t>(64), N));
                    }
                }
    check("too many rows", myl_linear_w8a16_adapters_dev(c, x, ((size_t)1 << 23) + 1, 64, at<int8_t>(64), 1, 64, sh, 10, 10, nullptr, at<int32_t>(64),
                                                         at<int8_t>(64), sh, 10, at<int8_t>(64), sh, 1, 16, out, 1, ws, ~(size_t)0), false);
    struct { size_t seqs, rows, heads, kvh, prefix, tail; } shapes[] = {
        {65535, 1, 64, 1, 1, 1}, {65535, 1, 64, 64, 65535, 1}, {1, 65535, 64, 8, 100, 65436}, {255, 257, 64, 64, 40000, 2000}, {1, 1, 65535, 65535, 65536, 0},
        {1, 1, 65535, 1, 0, 65536}, {64, 1, 28, 4, 30000, 2000}, {1, 1, 1, 1, 1, 0}, {1024, 1, 8, 1, 160, 160}, {3, 1, 8, 8, 0, 0}};
    for (auto& s : shapes)
        for (size_t hd : {(size_t)64, (size_t)128})
            for (size_t lut : {(size_t)1, (size_t)2662, (size_t)16385, (size_t)32768}) {
                const size_t bytes = myl_attention_prefix_workspace(c, s.seqs, s.rows, s.heads, s.kvh, hd, s.prefix, s.tail), ld = s.heads * hd;
                check("attention " + std::to_string(s.seqs) + " x " + std::to_string(s.rows) + " x " + std::to_string(s.heads) + ", " + std::to_string(lut),
                      myl_attention_prefix_dev(c, x, s.seqs, s.rows, ld, s.heads, s.kvh, hd, x, x, s.prefix, s.prefix * hd, x, x, s.seqs,
                                               s.kvh * s.tail * hd, s.tail * hd, s.tail, nullptr, at<int32_t>(64), 2896, 21, x, lut, 6, 14, out, ld, ws, bytes));
            }
    struct { size_t seqs, k, vocab, lut; } drafts[] = {{65535, 0, (size_t)1 << 20, 32768}, {31, 1024, (size_t)1 << 20, 32768}, {21845, 1, 1, 1}, {1, 4, 32001, 2662},
                                                       {65535, 0, 8193, 0}, {31, 1024, 152064, 0}};
    for (auto& s : drafts)
        for (const int32_t* draft : {(const int32_t*)nullptr, at<const int32_t>(64)}) {
            const size_t bytes = myl_verify_drafts_workspace(c, s.seqs, s.k, s.vocab, s.lut);
            check("drafts " + std::to_string(s.seqs) + " x " + std::to_string(s.k) + " of " + std::to_string(s.vocab),
                  myl_verify_drafts_dev(c, at<int32_t>(64), s.vocab, draft, s.vocab, s.seqs, s.k, s.vocab, at<int64_t>(64), nullptr, at<uint64_t>(64),
                                        s.lut ? x : nullptr, s.lut, at<int32_t>(64), at<int64_t>(64), ws, bytes));
        }
    std::printf("calls %ld bad %ld\n", calls, bad);
    return bad != 0;
}
"""


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc absent")
def test_grids_at_the_largest_sizes(tmp_path):
    """The second and third dimension of a grid are at most 65535, the threads of the first below 2^32."""
    from myelith_amd._lib import lib
    lib()
    so = ROOT / "myelith_amd" / "libmyl_hip.so"
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PROGRAM)
    subprocess.run([HIPCC, "-O1", "-std=c++17", "-I", str(ROOT / "include"), str(src), f"-L{so.parent}", f"-l:{so.name}", f"-Wl,-rpath,{so.parent}", "-Wl,--export-dynamic",
                    "-o", str(exe)], check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.stdout[-3000:], r.stderr[-1000:])
    assert int(re.match(r"calls (\d+) bad 0", r.stdout.strip().splitlines()[-1]).group(1)) > 1000
