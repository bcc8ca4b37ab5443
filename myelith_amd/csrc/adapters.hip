// adapters.hip -- low-rank adapters of many requests beside a shared W8A16
// projection: myl_linear_w8a16_adapters_dev.  Each step is a reference
// primitive (linear.rs:43-119):
//   u[m] = linear_w8a16(x[m], A[id], a_shifts[id], act_frac, mid_frac)   [rank]
//   d[m] = linear_w8a16(u[m], B[id], b_shifts[id], mid_frac, out_frac)   [N]
//   out[m] = clamp_i16(linear_w8a16(x[m], W, w_shifts, act_frac, out_frac) + d[m])
// with id = ids[m]; a row whose id is outside [0, n_adapters) has d = 0.
#include "abi_internal.h"
#include "gemm_dispatch.h"

#include <algorithm>
#include <string>

namespace myl {

// One wave per (row, rank index).
__global__ __launch_bounds__(64) void adapters_down_kernel(const int16_t* __restrict__ x, int ldx, int K,
                                                           const int32_t* __restrict__ ids, int n_adapters, int rank,
                                                           const int8_t* __restrict__ A,
                                                           const uint8_t* __restrict__ a_shifts, uint8_t act_frac,
                                                           uint8_t mid_frac, int16_t* __restrict__ u) {
    const int m = blockIdx.x, j = blockIdx.y;
    const int id = ids[m];
    if (id < 0 || id >= n_adapters) return;
    const int16_t* xr = x + (size_t)m * ldx;
    const int8_t* a = A + ((size_t)id * rank + j) * K;
    int64_t acc = 0;
    for (int k = threadIdx.x; k < K; k += 64) acc += (int32_t)xr[k] * (int32_t)a[k];
    acc = wave_sum_i64(acc);
    if (threadIdx.x == 0)
        u[(size_t)m * rank + j] =
            clamp_i16_i64(rescale64(acc, (uint8_t)(a_shifts[(size_t)id * rank + j] + act_frac), mid_frac));
}

// One thread per output.
__global__ __launch_bounds__(256) void adapters_up_kernel(const int16_t* __restrict__ u, const int32_t* __restrict__ ids,
                                                          int n_adapters, int rank, const int8_t* __restrict__ B,
                                                          const uint8_t* __restrict__ b_shifts, uint8_t mid_frac,
                                                          uint8_t out_frac, const uint8_t* __restrict__ out_frac_pc,
                                                          int N, int16_t* __restrict__ out, int ldo) {
    const int m = blockIdx.y, n = blockIdx.x * 256 + threadIdx.x;
    const int id = ids[m];
    if (n >= N || id < 0 || id >= n_adapters) return;
    const int8_t* b = B + ((size_t)id * N + n) * rank;
    int32_t acc = 0;
    for (int j = 0; j < rank; ++j) acc += (int32_t)u[(size_t)m * rank + j] * (int32_t)b[j];
    const int16_t d = clamp_i16_i64(rescale64(acc, (uint8_t)(b_shifts[(size_t)id * N + n] + mid_frac),
                                              out_frac_pc ? out_frac_pc[n] : out_frac));
    int16_t* o = out + (size_t)m * ldo + n;
    *o = clamp_i16((int32_t)*o + (int32_t)d);
}

__global__ __launch_bounds__(256) void adapters_clear_kernel(unsigned long long* __restrict__ p, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) p[i] = 0;
}

namespace {

constexpr size_t kMaxRank = 256;               // |sum B u| <= 2^7 2^15 2^8 = 2^30
constexpr size_t kAccElems = (size_t)512 << 10;  // products with more outputs do not split K

// The workspace: the shared product's byte planes and split-K sums, and u.
struct Space {
    int8_t* planes = nullptr;
    unsigned long long* acc = nullptr;
    size_t planes_bytes = 0, acc_elems = 0, bytes = 0;
    int16_t* u = nullptr;
    static Space of(void* base, size_t M, size_t N, size_t K, size_t rank) {
        Carve c{(char*)base};
        Space s;
        if (M >= 2) {
            s.planes_bytes = 2 * M * K;
            s.acc_elems = M * N <= kAccElems ? M * N : 0;
            s.planes = c.take<int8_t>(s.planes_bytes);
            s.acc = c.take<unsigned long long>(std::max<size_t>(s.acc_elems, 1));
        }
        s.u = c.take<int16_t>(M * rank);
        s.bytes = c.used ? c.used : 256;  // 0 stands for sizes that a call refuses
        return s;
    }
};

}  // namespace
}  // namespace myl

using namespace myl;

extern "C" {

size_t myl_linear_w8a16_adapters_workspace(const myl_ctx* ctx, size_t M, size_t N, size_t K, size_t rank) {
    if (!ctx || !fits_int(M) || !fits_int(N) || !fits_int(K) || rank > kMaxRank) return 0;
    return Space::of(nullptr, M, N, K, rank).bytes;
}

int myl_linear_w8a16_adapters_dev(myl_ctx* ctx, const int16_t* x, size_t M, size_t ldx, const int8_t* W, size_t N,
                                  size_t K, const uint8_t* w_shifts, uint8_t act_frac, uint8_t out_frac,
                                  const uint8_t* out_frac_pc, const int32_t* ids, const int8_t* A,
                                  const uint8_t* a_shifts, uint8_t mid_frac, const int8_t* B, const uint8_t* b_shifts,
                                  size_t n_adapters, size_t rank, int16_t* out, size_t ldo, void* workspace,
                                  size_t workspace_bytes) {
    if (!ctx) return MYL_E_INVALID;
    const char* what = "linear_w8a16_adapters_dev";
    auto bad = [&](const char* why) { return ctx->fail(MYL_E_INVALID, std::string(what) + ": " + why); };
    if (K == 0) return bad("K must be > 0");
    if (ldx < K || ldo < N) return bad("leading dimension too small");
    if (!fits_int(M) || !fits_int(N) || !fits_int(K) || !fits_int(ldx) || !fits_int(ldo) || !fits_int(n_adapters))
        return bad("shape too large");
    if (n_adapters > 0 && (rank == 0 || rank > kMaxRank)) return bad("rank must be 1 to 256");
    if (M == 0 || N == 0) return MYL_OK;
    if (!x || !W || !w_shifts || !out) return bad("null operand");
    if (n_adapters > 0 && (!ids || !A || !a_shifts || !B || !b_shifts)) return bad("null adapter operand");
    if (n_adapters == 0) rank = 0;
    const Space s = Space::of(workspace, M, N, K, rank);
    if (!workspace || workspace_bytes < s.bytes) return bad("workspace too small (myl_linear_w8a16_adapters_workspace)");
    if ((uintptr_t)workspace & 15) return bad("workspace must be 16-byte aligned");
    const DeviceGuard guard(ctx->device);
    const hipStream_t st = ctx->stream;
    MmCtx mm;
    mm.cus = ctx->prop.multiProcessorCount > 0 ? ctx->prop.multiProcessorCount : 1;
    mm.planes = s.planes;
    mm.planes_bytes = s.planes_bytes;
    mm.acc = s.acc;
    mm.acc_elems = s.acc_elems;
    if (s.acc_elems) {
        adapters_clear_kernel<<<(unsigned)std::min<size_t>((s.acc_elems + 255) / 256, 1024), 256, 0, st>>>(s.acc, s.acc_elems);
        if (int rc = ctx->hip(hipGetLastError(), what)) return rc;
    }
    int rc = ctx->hip(linear_w8a16(x, (int)M, (int)ldx, W, (int)N, (int)K, w_shifts, act_frac, out_frac, out_frac_pc, out,
                                   (int)ldo, st, &mm), what);
    if (rc || n_adapters == 0) return rc;
    for (size_t m0 = 0; m0 < M; m0 += 65535) {  // the grid's y range
        const int rows = (int)std::min<size_t>(M - m0, 65535);
        adapters_down_kernel<<<dim3(rows, (unsigned)rank), 64, 0, st>>>(x + m0 * ldx, (int)ldx, (int)K, ids + m0, (int)n_adapters,
                                                                        (int)rank, A, a_shifts, act_frac, mid_frac,
                                                                        s.u + m0 * rank);
        adapters_up_kernel<<<dim3((unsigned)((N + 255) / 256), rows), 256, 0, st>>>(
            s.u + m0 * rank, ids + m0, (int)n_adapters, (int)rank, B, b_shifts, mid_frac, out_frac, out_frac_pc, (int)N,
            out + m0 * ldo, (int)ldo);
    }
    return ctx->hip(hipGetLastError(), what);
}

}  // extern "C"
