// verify.hip -- drafted tokens checked against the target's probabilities with
// given random numbers: myl_verify_drafts_dev.
//
// A logit row z has the weights of the integer log-softmax (fixed.h):
// p_j = exp_lut[(max z - z_j) << 2], 0 past the table; P = sum p_j.  The draft's
// row gives q_j and Q the same way (without draft logits q is 1 at the drafted
// token and 0 elsewhere).  Draft i of a sequence is accepted when its random
// number r_i satisfies r_i / 2^64 < (p_t / P) / (q_t / Q), that is
//   floor(r_i q_t P / 2^64) < p_t Q.
// Where the first draft is rejected the next token follows the weights
// w_j = max(0, p_j Q - q_j P); behind the last accepted draft, w_j = p_j.  With
// W = sum w_j and the sequence's last random number r the token is the first j
// with floor(r W / 2^64) < w_0 + ... + w_j.
//
// Table entries are below 2^15 and vocabularies at most 2^20, so P, Q < 2^35,
// w_j < 2^50, and only W and its running sums pass 64 bits (< 2^70).
//
// Bound by reading the rows.  P needs the row's maximum first; as the logits are whole
// numbers, a chunk of a row is read once and leaves its own maximum and how many of its
// values lie k below it (verify_count_kernel), from which the row's maximum and P
// follow (verify_sum_kernel).  Many blocks share a row, so that few rows fill the chip too.
// The row that decides the next token is read a second time, chunk by chunk
// (verify_weight_kernel), and the group of 256 values with the token a third
// (verify_pick_kernel).  24 sequences of up to 5 drafts (about 150 rows, 88 MB), vocabulary
// 152064: 19.4 us for the count (4.5 TB/s), 5.6, 9.5 and 5.9 for the others, 40 in all; one
// block per row, with a pass for the maximum and one for the sum, took 355.
#include "abi_internal.h"
#include "ops.h"
#include "serve_plan.h"
#include "wave.h"

#include <string>

namespace myl {
namespace {

struct Verify {
    const int32_t *target, *draft;  // draft may be null
    const int64_t* tokens;
    const int32_t* n_draft;  // may be null
    const uint64_t* randoms;
    const int16_t* lut;  // null: greedy
    int32_t* accepted;
    int64_t* out;
    size_t ldt, ldd;
    SmallDiv k1, kd;  // k + 1, k
    int B, k, V, chunks;
    uint32_t bins, words;  // table entries a logit step apart; pairs of them
    // the workspace
    struct RowStat* stat;  // [rows]
    int32_t* cmax;         // [rows][chunks]
    uint32_t* counts;      // [rows][chunks][words]
    uint64_t* sums;        // [sequences][chunks][kVerifyChunk / 256]
    uint64_t* keys;        // greedy: [rows][chunks]
    int32_t* first;        // [sequences] accepted drafts
};

struct RowStat {
    int32_t m;   // the maximum
    int32_t pad;
    uint64_t s;  // the sum of the weights
};

constexpr int kBlk = 256, kWeightThreads = 1024;
template <int THREADS>
constexpr int kGroups = kVerifyChunk / (4 * THREADS);  // quads of a thread in a chunk

// Four consecutive values of a row: rows start at any 4-byte address.
typedef int32_t RowQuad __attribute__((ext_vector_type(4), aligned(4)));

constexpr uint32_t kPerLogit = 1u << (MYL_TV_EXP_INPUT_FRAC - MYL_TV_LOGIT_FRAC_BITS);  // table entries per logit step
__device__ inline uint32_t weight_below(const Verify& a, uint32_t below) {
    return below < a.bins ? (uint32_t)max(0, (int32_t)a.lut[below * kPerLogit]) : 0u;
}
__device__ inline uint32_t weight(const Verify& a, int32_t m, int32_t z) {  // z <= m
    return weight_below(a, (uint32_t)m - (uint32_t)z);
}

__device__ inline uint64_t max_key(int32_t v, uint32_t idx) {  // by value, then by the smaller index
    return ((uint64_t)((uint32_t)v ^ 0x80000000u) << 32) | (uint64_t)(0xFFFFFFFFu - idx);
}

__device__ inline int drafts_of(const Verify& a, int b) { return a.n_draft ? min(max(a.n_draft[b], 0), a.k) : a.k; }

// Row r of the target's B (k + 1) rows, then the draft's B k; null past the sequence's drafts.
__device__ inline const int32_t* row_of(const Verify& a, int r) {
    const int T = a.B * (a.k + 1);
    const bool t = r < T;
    int rem;
    const int b = divmod(t ? a.k1 : a.kd, t ? r : r - T, rem);
    const int n = drafts_of(a, b);
    if (t) return rem <= n ? a.target + (size_t)r * a.ldt : nullptr;
    return rem < n ? a.draft + (size_t)(r - T) * a.ldd : nullptr;
}

// A thread's quads of a chunk, 4 THREADS values apart, and how many values of each lie in the row.
template <int THREADS>
__device__ inline void load_chunk(const int32_t* __restrict__ z, int V, int c0, RowQuad (&v)[kGroups<THREADS>], int (&n)[kGroups<THREADS>]) {
#pragma unroll
    for (int q = 0; q < kGroups<THREADS>; ++q) {
        const int i = c0 + q * 4 * THREADS + 4 * (int)threadIdx.x;
        n[q] = min(max(V - i, 0), 4);
        if (n[q] == 4) v[q] = *reinterpret_cast<const RowQuad*>(z + i);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) v[q][e] = e < n[q] ? z[i + e] : INT32_MIN;
    }
}

__global__ __launch_bounds__(kBlk) void verify_count_kernel(Verify a) {
    extern __shared__ uint32_t cnt[];
    __shared__ int32_t red[kBlk / 64];
    const int c = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
    const int32_t* z = row_of(a, r);
    if (!z) return;
    RowQuad v[kGroups<kBlk>];
    int n[kGroups<kBlk>];
    load_chunk<kBlk>(z, a.V, c * kVerifyChunk, v, n);
    for (uint32_t i = tid; i < a.words * 2; i += kBlk) cnt[i] = 0;
    int32_t mx = INT32_MIN;
#pragma unroll
    for (int q = 0; q < kGroups<kBlk>; ++q) mx = max(max(mx, max(v[q][0], v[q][1])), max(v[q][2], v[q][3]));
    mx = block_max_i32_dpp(mx, red);  // its barrier also publishes the cleared counters
#pragma unroll
    for (int q = 0; q < kGroups<kBlk>; ++q) {
        // a value that fills the wave's quads is counted once: the lanes' adds to one counter follow one another
        const int32_t first = __builtin_amdgcn_readfirstlane(v[q][0]);
        if (__all(n[q] == 4 && v[q][0] == first && v[q][1] == first && v[q][2] == first && v[q][3] == first)) {
            const uint32_t below = (uint32_t)mx - (uint32_t)first;
            if (below < a.bins && (tid & 63) == 0) atomicAdd(&cnt[below], 256u);
            continue;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t below = (uint32_t)mx - (uint32_t)v[q][e];
            if (below < a.bins && e < n[q]) atomicAdd(&cnt[below], 1u);
        }
    }
    __syncthreads();
    // counts are at most kVerifyChunk: 16 bits each
    uint32_t* out = a.counts + ((size_t)r * a.chunks + c) * a.words;
    for (uint32_t i = tid; i < a.words; i += kBlk) out[i] = cnt[2 * i] | (cnt[2 * i + 1] << 16);
    if (tid == 0) a.cmax[(size_t)r * a.chunks + c] = mx;
}

// The weights of the bins in LDS, by a block of THREADS: the first entries are on their way
// while the block loads what else it needs.  A barrier follows before they are read.
template <int THREADS>
struct BinWeights {
    static constexpr int kEach = 1024 / THREADS;
    uint32_t w[kEach];
    __device__ inline void load(const Verify& a) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) w[i] = weight_below(a, threadIdx.x + i * THREADS);
    }
    __device__ inline void store(const Verify& a, uint16_t* wt) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (threadIdx.x + i * THREADS < a.bins) wt[threadIdx.x + i * THREADS] = (uint16_t)w[i];
        for (uint32_t i = threadIdx.x + 1024; i < a.bins; i += THREADS) wt[i] = (uint16_t)weight_below(a, i);
    }
};

// A wave per chunk: its counts against the table, shifted by how far its maximum is below the row's.
// 16 waves: with four, 19 chunks of a row came one after another (13.7 us for 264 rows of 152064, now 5.8).
constexpr int kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void verify_sum_kernel(Verify a) {
    extern __shared__ uint16_t wt[];
    __shared__ uint64_t red[kSumThreads / 64];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    if (!row_of(a, r)) return;
    const int32_t* cm = a.cmax + (size_t)r * a.chunks;
    BinWeights<kSumThreads> bw;
    bw.load(a);
    int32_t mx = INT32_MIN;
    for (int c = lane; c < a.chunks; c += 64) mx = max(mx, cm[c]);
    bw.store(a, wt);
    mx = wave_max_i32(mx);
    __syncthreads();
    uint64_t s = 0;
    for (int c = w; c < a.chunks; c += kSumThreads / 64) {
        const uint32_t d = (uint32_t)mx - (uint32_t)cm[c];
        if (d >= a.bins) continue;
        const uint32_t* n = a.counts + ((size_t)r * a.chunks + c) * a.words;
        for (uint32_t i0 = lane; i0 < a.words; i0 += 8 * 64) {
            uint32_t two[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) two[k] = i0 + 64 * k < a.words ? n[i0 + 64 * k] : 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t at = d + 2 * (i0 + 64 * k);
                if (two[k] & 0xFFFFu) s += (uint64_t)(two[k] & 0xFFFFu) * (at < a.bins ? wt[at] : 0u);
                if (two[k] >> 16) s += (uint64_t)(two[k] >> 16) * (at + 1 < a.bins ? wt[at + 1] : 0u);
            }
        }
    }
    s = wave_sum_u64(s);
    if (lane == 0) red[w] = s;
    __syncthreads();
    if (w == 0) {
        s = wave_sum_u64(lane < kSumThreads / 64 ? red[lane] : 0);
        if (lane == 0) a.stat[r] = RowStat{mx, 0, s};
    }
}

// How a sequence's drafts end: the accepted ones, and the weights of the next
// token, w_j = max(0, p_j Q - q_j P) (q_j = 0 where qrow is null, but 1 at `not_j`).
struct Ending {
    int n;
    const int32_t *prow, *qrow;
    int32_t pm, qm;
    uint64_t P, Q;
    int64_t not_j;
};

// The first draft that fails, all tested at once by the whole block.
__device__ inline int verify_first(const Verify& a, int b, int* s_first) {
    const int T = a.B * (a.k + 1), nd = drafts_of(a, b);
    if (threadIdx.x == 0) *s_first = nd;
    __syncthreads();
    for (int i = threadIdx.x; i < nd; i += blockDim.x) {
        const int tr = b * (a.k + 1) + i, dr = b * a.k + i;
        const int64_t t = a.tokens[dr];
        bool ok = t >= 0 && t < a.V;
        if (ok) {
            const RowStat p = a.stat[tr];
            uint64_t qt = 1, Q = 1;
            if (a.draft) {
                const RowStat q = a.stat[T + dr];
                qt = weight(a, q.m, a.draft[(size_t)dr * a.ldd + t]);
                Q = q.s;
            }
            ok = __umul64hi(a.randoms[tr], qt * p.s) < weight(a, p.m, a.target[(size_t)tr * a.ldt + t]) * Q;
        }
        if (!ok) atomicMin(s_first, i);
    }
    __syncthreads();
    return *s_first;
}

__device__ inline Ending verify_ending(const Verify& a, int b, int first) {
    const int T = a.B * (a.k + 1), nd = drafts_of(a, b);
    Ending e{};
    e.n = first;
    const int tr = b * (a.k + 1) + e.n, dr = b * a.k + e.n;
    const RowStat p = a.stat[tr];
    e.prow = a.target + (size_t)tr * a.ldt;
    e.pm = p.m;
    e.P = p.s;
    e.Q = 1;
    e.not_j = -1;
    if (e.n < nd) {
        if (a.draft) {
            const RowStat q = a.stat[T + dr];
            e.qrow = a.draft + (size_t)dr * a.ldd;
            e.qm = q.m;
            e.Q = q.s;
        } else {
            e.not_j = a.tokens[dr];
        }
    }
    return e;
}

__device__ inline uint64_t ending_weight(const Verify& a, const Ending& e, int j, int32_t z) {
    const uint64_t p = weight(a, e.pm, z);
    if (p == 0 || j == e.not_j) return 0;
    const uint64_t x = p * e.Q;
    const uint64_t y = e.qrow ? weight(a, e.qm, e.qrow[j]) * e.P : 0;
    return x > y ? x - y : 0;
}

// The next token's weights, summed over every 256 values (a wave's quads).  Grid (chunks,
// sequences).  Both rows' quads are loaded together and the table waits in LDS: a lookup
// and a load of q per value that has a weight, one after another, took longer (24 sequences:
// 15.9 us, now 9.4), as did 256 threads, which come to eight wave sums each (12.7).
__global__ __launch_bounds__(kWeightThreads) void verify_weight_kernel(Verify a) {
    extern __shared__ uint16_t wt[];
    __shared__ int s_first;
    const int c = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    BinWeights<kWeightThreads> bw;
    bw.load(a);
    const int first = verify_first(a, b, &s_first);
    const Ending e = verify_ending(a, b, first);
    RowQuad v[kGroups<kWeightThreads>], u[kGroups<kWeightThreads>];
    int n[kGroups<kWeightThreads>];
    load_chunk<kWeightThreads>(e.prow, a.V, c * kVerifyChunk, v, n);
    if (e.qrow) load_chunk<kWeightThreads>(e.qrow, a.V, c * kVerifyChunk, u, n);
    bw.store(a, wt);
    __syncthreads();
    if (c == 0 && tid == 0) a.first[b] = first;
    uint64_t* out = a.sums + ((size_t)b * a.chunks + c) * (kVerifyChunk / 256);
    auto at = [&](int32_t m, int32_t z) -> uint64_t {
        const uint32_t below = (uint32_t)m - (uint32_t)z;
        return below < a.bins ? wt[below] : 0u;
    };
#pragma unroll
    for (int q = 0; q < kGroups<kWeightThreads>; ++q) {
        uint64_t s = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint64_t p = at(e.pm, v[q][k]);
            if (k >= n[q] || c * kVerifyChunk + q * 4 * kWeightThreads + 4 * tid + k == e.not_j) p = 0;
            const uint64_t x = p * e.Q, y = e.qrow ? at(e.qm, u[q][k]) * e.P : 0;
            s += x > y ? x - y : 0;
        }
        s = wave_sum_u64(s);
        if ((tid & 63) == 0) out[q * (kWeightThreads / 64) + (tid >> 6)] = s;
    }
}

__device__ inline uint64_t shfl_up_u64(uint64_t v, int d) {
    const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)v, d, 64);
    const uint32_t hi = (uint32_t)__shfl_up((int)(uint32_t)(v >> 32), d, 64);
    return ((uint64_t)hi << 32) | lo;
}
__device__ inline uint64_t wave_scan_u64(uint64_t v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = shfl_up_u64(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

__device__ inline void verify_write(const Verify& a, int b, int n, int64_t pick) {
    if (threadIdx.x == 0) a.accepted[b] = n;
    for (int i = threadIdx.x; i <= a.k; i += blockDim.x)
        a.out[(size_t)b * (a.k + 1) + i] = i < n ? a.tokens[(size_t)b * a.k + i] : (i == n ? pick : -1);
}

// floor(r W / 2^64)
__device__ inline myl_u128 threshold(uint64_t r, myl_u128 W) { return (myl_u128)r * (uint64_t)(W >> 64) + __umul64hi(r, (uint64_t)W); }

// The first j whose running sum of ending_weight passes the threshold of their total, by the
// whole block over the whole row; -1: the total is 0.  For endings whose sums are not at hand.
__device__ inline int64_t pick_by_row(const Verify& a, const Ending& e, uint64_t r, myl_u128* red, int* s_pick) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    myl_u128 part = 0;
    for (int j = tid; j < a.V; j += kBlk) part += ending_weight(a, e, j, e.prow[j]);
    const myl_u128 W = (myl_u128)block_sum_i128((myl_i128)part, (myl_i128*)red);
    if (W == 0) return -1;
    const myl_u128 thr = threshold(r, W);
    myl_u128 base = 0;
    for (int j0 = 0; j0 < a.V; j0 += kBlk) {
        const int j = j0 + tid;
        const uint64_t inc = wave_scan_u64(j < a.V ? ending_weight(a, e, j, e.prow[j]) : 0, lane);
        __syncthreads();
        if (tid == 0) *s_pick = a.V;
        if (lane == 63) red[w] = inc;
        __syncthreads();
        myl_u128 before = base;
        for (int k = 0; k < w; ++k) before += red[k];
        for (int k = 0; k < kBlk / 64; ++k) base += red[k];
        if (thr < base) {  // uniform
            if (j < a.V && thr < before + inc) atomicMin(s_pick, j);
            __syncthreads();
            return *s_pick;
        }
    }
    return a.V - 1;
}

// The first maximum of a row, by the whole block.
__device__ inline int64_t first_max(const int32_t* z, int V, uint64_t* red) {
    uint64_t key = 0;
    for (int i = threadIdx.x; i < V; i += kBlk) {
        const uint64_t o = max_key(z[i], (uint32_t)i);
        key = o > key ? o : key;
    }
    key = wave_max_u64(key);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = key;
    __syncthreads();
    for (int w = 0; w < kBlk / 64; ++w) key = red[w] > key ? red[w] : key;
    return (int64_t)(0xFFFFFFFFu - (uint32_t)key);
}

__global__ __launch_bounds__(kBlk) void verify_pick_kernel(Verify a) {
    __shared__ int s_pick;
    __shared__ myl_u128 red[kBlk];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    // each thread: `per` of the sequence's sums, in order (at most 2^20 / 256 / kBlk = 16)
    const int groups = a.chunks * (kVerifyChunk / 256), per = (groups + kBlk - 1) / kBlk;
    const uint64_t* sums = a.sums + (size_t)b * groups;
    const uint64_t r = a.randoms[(size_t)b * (a.k + 1) + a.k];
    myl_u128 own = 0;
    for (int i = 0; i < per; ++i) own += tid * per + i < groups ? sums[tid * per + i] : 0;
    Ending e = verify_ending(a, b, a.first[b]);
    red[tid] = own;
    __syncthreads();
    // running totals of the 256 shares: 64 lanes of each wave, four shares each
    myl_u128 four[4], before = 0, W = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) four[k] = red[4 * lane + k];
    {
        const myl_u128 t = four[0] + four[1] + four[2] + four[3];
        // 128-bit scan as two words, the low 56 bits (64 of them stay below 2^62) and the rest
        const uint64_t mask = (1ull << 56) - 1;
        const uint64_t lo = wave_scan_u64((uint64_t)t & mask, lane), hi = wave_scan_u64((uint64_t)(t >> 56), lane);
        const myl_u128 inc = ((myl_u128)hi << 56) + lo;
        before = inc - t;
        W = ((myl_u128)readlane_u64(hi, 63) << 56) + readlane_u64(lo, 63);
    }
    if (W == 0) {  // nothing is left: the target's own weights, or without any its maximum
        e.qrow = nullptr;
        e.not_j = -1;
        e.Q = 1;
        int64_t pick = pick_by_row(a, e, r, red, &s_pick);
        if (pick < 0) pick = first_max(e.prow, a.V, reinterpret_cast<uint64_t*>(red));
        verify_write(a, b, e.n, pick);
        return;
    }
    // wave 0 finds the share, then the 256 values, then the value
    if (w == 0) {
        const myl_u128 thr = threshold(r, W);
        const int l = (int)__builtin_ctzll(__ballot(thr < before + four[0] + four[1] + four[2] + four[3]));
        int share = 4 * lane;
        myl_u128 base = before;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const bool past = thr < base + four[k];
            if (past) break;
            base += four[k];
            ++share;
        }
        const uint64_t blo = readlane_u64((uint64_t)base, l), bhi = readlane_u64((uint64_t)(base >> 64), l);
        base = ((myl_u128)bhi << 64) | blo;
        share = readlane_i32(share, l);
        int g = share * per;
        {
            const uint64_t own_g = lane < per && g + lane < groups ? sums[g + lane] : 0;  // per <= 16 sums below 2^58
            const uint64_t inc = wave_scan_u64(own_g, lane);
            const int at = (int)__builtin_ctzll(__ballot(thr < base + inc));
            base += readlane_u64(inc - own_g, at);
            g += at;
        }
        uint64_t wv[4], t = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int j = g * 256 + 4 * lane + k;
            wv[k] = j < a.V ? ending_weight(a, e, j, e.prow[j]) : 0;
            t += wv[k];
        }
        const uint64_t inc = wave_scan_u64(t, lane);
        const int at = (int)__builtin_ctzll(__ballot(thr < base + inc));
        myl_u128 run = base + inc - t;
        int j = g * 256 + 4 * lane;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            run += wv[k];
            if (thr < run) break;
            ++j;
        }
        j = readlane_i32(j, at);
        if (lane == 0) s_pick = j;
    }
    __syncthreads();
    verify_write(a, b, e.n, s_pick);
}

// ---- without a table: the first maxima --------------------------------------------

__global__ __launch_bounds__(kBlk) void verify_max_kernel(Verify a) {
    __shared__ uint64_t red[kBlk / 64];
    const int c = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
    const int32_t* z = row_of(a, r);
    if (!z) return;
    RowQuad v[kGroups<kBlk>];
    int n[kGroups<kBlk>];
    load_chunk<kBlk>(z, a.V, c * kVerifyChunk, v, n);
    int32_t best = INT32_MIN;
    int at = -1;
#pragma unroll
    for (int q = 0; q < kGroups<kBlk>; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool up = (e < n[q]) & ((v[q][e] > best) | (at < 0));
            best = up ? v[q][e] : best;
            at = up ? c * kVerifyChunk + q * 1024 + 4 * tid + e : at;
        }
    const uint64_t key = wave_max_u64(at < 0 ? 0 : max_key(best, (uint32_t)at));
    if ((tid & 63) == 0) red[tid >> 6] = key;
    __syncthreads();
    if (tid == 0) {
        uint64_t k = red[0];
        for (int w = 1; w < kBlk / 64; ++w) k = red[w] > k ? red[w] : k;
        a.keys[(size_t)r * a.chunks + c] = k;
    }
}

// A wave per row of the sequence.
__global__ __launch_bounds__(kBlk) void verify_greedy_kernel(Verify a) {
    __shared__ int s_first;
    __shared__ int32_t s_at;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, nd = drafts_of(a, b);
    if (tid == 0) s_first = nd;
    __syncthreads();
    auto choice = [&](int i) {
        const uint64_t* keys = a.keys + ((size_t)b * (a.k + 1) + i) * a.chunks;
        uint64_t key = 0;
        for (int c = lane; c < a.chunks; c += 64) key = keys[c] > key ? keys[c] : key;
        return (int64_t)(0xFFFFFFFFu - (uint32_t)wave_max_u64(key));
    };
    for (int i = tid >> 6; i < nd; i += kBlk / 64)
        if (choice(i) != a.tokens[(size_t)b * a.k + i]) {
            if (lane == 0) atomicMin(&s_first, i);
            break;
        }
    __syncthreads();
    const int n = s_first;
    if (tid < 64) {
        const int64_t pick = choice(n);
        if (lane == 0) s_at = (int32_t)pick;
    }
    __syncthreads();
    verify_write(a, b, n, s_at);
}

}  // namespace
}  // namespace myl

using namespace myl;

extern "C" {

size_t myl_verify_drafts_workspace(const myl_ctx* ctx, size_t n_seqs, size_t k, size_t vocab, size_t lut_len) {
    const VerifyShape s{n_seqs, k, vocab, lut_len};
    return !ctx || verify_refuse(s) ? 0 : verify_plan(s).bytes;
}

int myl_verify_drafts_dev(myl_ctx* ctx, const int32_t* target, size_t ldt, const int32_t* draft, size_t ldd, size_t n_seqs,
                          size_t k, size_t vocab, const int64_t* tokens, const int32_t* n_draft, const uint64_t* randoms,
                          const int16_t* exp_lut, size_t lut_len, int32_t* accepted, int64_t* out, void* workspace,
                          size_t workspace_bytes) {
    if (!ctx) return MYL_E_INVALID;
    const char* what = "verify_drafts_dev";
    auto bad = [&](const char* why) { return ctx->fail(MYL_E_INVALID, std::string(what) + ": " + why); };
    if (!exp_lut) {
        lut_len = 0;
        draft = nullptr;
    }
    const VerifyShape s{n_seqs, k, vocab, lut_len};
    if (const char* why = verify_refuse(s)) return bad(why);
    if (exp_lut && lut_len == 0) return bad("the exp table must hold 1 to 32768 entries");
    if (ldt < vocab || (draft && ldd < vocab)) return bad("leading dimension too small");
    if (n_seqs == 0) return MYL_OK;
    if (!target || !accepted || !out || (k && !tokens) || (exp_lut && !randoms)) return bad("null operand");
    const VerifyPlan pl = verify_plan(s);
    if (!workspace || workspace_bytes < pl.bytes) return bad("workspace too small (myl_verify_drafts_workspace)");
    if ((uintptr_t)workspace & 15) return bad("workspace must be 16-byte aligned");
    const DeviceGuard guard(ctx->device);
    const hipStream_t st = ctx->stream;
    char* ws = static_cast<char*>(workspace);
    Verify a{};
    a.target = target; a.draft = draft; a.tokens = tokens; a.n_draft = n_draft; a.randoms = randoms;
    a.lut = exp_lut; a.accepted = accepted; a.out = out; a.ldt = ldt; a.ldd = ldd;
    a.B = (int)n_seqs; a.k = (int)k; a.V = (int)vocab;
    a.k1 = SmallDiv::of(k + 1); a.kd = SmallDiv::of(k ? k : 1);
    a.chunks = pl.chunks; a.bins = pl.bins; a.words = pl.words;
    a.stat = reinterpret_cast<RowStat*>(ws + pl.off_stat);
    a.cmax = reinterpret_cast<int32_t*>(ws + pl.off_max);
    a.counts = reinterpret_cast<uint32_t*>(ws + pl.off_counts);
    a.sums = reinterpret_cast<uint64_t*>(ws + pl.off_sums);
    a.keys = reinterpret_cast<uint64_t*>(ws + pl.off_sums);
    a.first = reinterpret_cast<int32_t*>(ws + pl.off_first);
    const unsigned T = (unsigned)(a.B * (a.k + 1)), rows = T + (draft ? (unsigned)(a.B * a.k) : 0u), chunks = (unsigned)pl.chunks;
    if (!exp_lut) {
        verify_max_kernel<<<dim3(chunks, T), kBlk, 0, st>>>(a);
        verify_greedy_kernel<<<a.B, kBlk, 0, st>>>(a);
        return ctx->hip(hipGetLastError(), what);
    }
    verify_count_kernel<<<dim3(chunks, rows), kBlk, (size_t)pl.words * 8, st>>>(a);
    verify_sum_kernel<<<rows, kSumThreads, (size_t)pl.bins * 2, st>>>(a);
    verify_weight_kernel<<<dim3(chunks, (unsigned)a.B), kWeightThreads, (size_t)pl.bins * 2, st>>>(a);
    verify_pick_kernel<<<a.B, kBlk, 0, st>>>(a);
    return ctx->hip(hipGetLastError(), what);
}

}  // extern "C"
