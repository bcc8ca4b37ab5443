// logprobs.hip -- log probabilities of given tokens, the entropy and the most likely
// alternatives of rows of logits: myl_logprobs_dev.
//
// A row z has the weights of the integer log-softmax (fixed.h): e_j =
// exp_lut[(m - z_j) << 2] with m = max z, 0 past the table; S = sum e_j.  In Q16
//   ln p_j = (z_j - m) 2^10 - ln_q16(S)
//   -sum p_j ln p_j = ln_q16(S) + RNE(2^10 sum e_j (m - z_j) / S)
// so both need, of a row, how many of its values lie k below the maximum, for
// the k that the table covers.  A block counts a chunk of a row below the chunk's own
// maximum (logp_count_kernel), and one per row adds the chunks' counts up, each shifted by how
// far its maximum is below the row's (logp_row_kernel).  The row is read once.
// The n most likely tokens lie in the n tiles of 256 values whose maxima are the
// largest (of equal ones the first): n others each hold a value before any in
// another tile.  So the count keeps every tile's maximum, and n tiles are read again.
// Many rows are bound by the bytes: 2003 rows of 152064 values take 241 us (5.05 TB/s, a large
// copy's rate), the count 212 of them.  Few rows are bound by two launches and the
// second one's chain of loads: 24 rows with 20 alternatives 17.3 us (5.4 and 11.5), one row of
// 32001 values 11.6 (4.7 and 6.9).
#include "abi_internal.h"
#include "ops.h"
#include "paged_plan.h"
#include "wave.h"

#include <string>

namespace myl {
namespace {

struct Logp {
    const int32_t* z;
    const int64_t* tokens;
    const int16_t* lut;
    int64_t *logprobs, *entropy, *top_tokens, *top_logprobs;  // entropy may be null
    size_t ldz;
    int V, T, n, chunks, tiles;
    uint32_t bins, words;
    // the workspace
    int32_t* cmax;     // [rows][chunks]
    int32_t* tmax;     // [rows][tiles]
    uint32_t* counts;  // [rows][chunks][words]
};

constexpr int kBlk = 256;
constexpr int kQuads = kLogpChunk / (4 * kBlk);

typedef int32_t RowQuad __attribute__((ext_vector_type(4), aligned(4)));

constexpr uint32_t kPerLogit = 1u << (MYL_TV_EXP_INPUT_FRAC - MYL_TV_LOGIT_FRAC_BITS);  // table entries per logit step
__device__ inline uint32_t weight_below(const Logp& a, uint32_t below) {
    return below < a.bins ? (uint32_t)max(0, (int32_t)a.lut[below * kPerLogit]) : 0u;
}
// By value, then by the smaller index; neither 0 nor ~0.
__device__ inline uint64_t max_key(int32_t v, uint32_t idx) {
    return ((uint64_t)((uint32_t)v ^ 0x80000000u) << 32) | (uint64_t)(0x7FFFFFFFu - idx);
}
__device__ inline int32_t key_value(uint64_t k) { return (int32_t)((uint32_t)(k >> 32) ^ 0x80000000u); }
__device__ inline uint32_t key_index(uint64_t k) { return 0x7FFFFFFFu - (uint32_t)k; }

__global__ __launch_bounds__(kBlk) void logp_count_kernel(Logp a) {
    extern __shared__ uint32_t cnt[];
    __shared__ int32_t red[kBlk / 64];
    const int c = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
    const int32_t* z = a.z + (size_t)r * a.ldz;
    RowQuad v[kQuads];
    int n[kQuads];
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
        const int i = c * kLogpChunk + q * 4 * kBlk + 4 * tid;
        n[q] = min(max(a.V - i, 0), 4);
        if (n[q] == 4) v[q] = __builtin_nontemporal_load(reinterpret_cast<const RowQuad*>(z + i));
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) v[q][e] = e < n[q] ? z[i + e] : INT32_MIN;
    }
    for (uint32_t i = tid; i < a.words * 2; i += kBlk) cnt[i] = 0;
    int32_t mx = INT32_MIN;
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
        const int32_t own = max(max(v[q][0], v[q][1]), max(v[q][2], v[q][3]));
        mx = max(mx, own);
        if (a.n) {
            const int32_t top = wave_max_i32(own);
            const int tile = (c * kLogpChunk + q * 4 * kBlk) / kLogpTile + (tid >> 6);
            if ((tid & 63) == 0 && tile < a.tiles) a.tmax[(size_t)r * a.tiles + tile] = top;
        }
    }
    mx = block_max_i32_dpp(mx, red);  // its barrier also publishes the cleared counters
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
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
    // counts are at most kLogpChunk: 16 bits each
    uint32_t* out = a.counts + ((size_t)r * a.chunks + c) * a.words;
    for (uint32_t i = tid; i < a.words; i += kBlk) out[i] = cnt[2 * i] | (cnt[2 * i + 1] << 16);
    if (tid == 0) a.cmax[(size_t)r * a.chunks + c] = mx;
}

// RNE(num / den) for num < 2^59, den >= 1 and num / den < 2^24, bit by bit.
__device__ inline int64_t div_round(uint64_t num, uint64_t den) {
    uint64_t q = 0;
    for (int b = 23; b >= 0; --b)
        if (num >> b >= den) {
            num -= den << b;
            q |= 1ull << b;
        }
    const uint64_t twice = 2 * num;
    return (int64_t)(q + (twice > den || (twice == den && (q & 1)) ? 1 : 0));
}

// The counts' table in LDS.  Its first entries are on their way while the block loads the maxima.
template <int THREADS>
struct BinWeights {
    static constexpr int kEach = 1024 / THREADS;
    uint32_t w[kEach];
    __device__ inline void load(const Logp& a) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) w[i] = weight_below(a, threadIdx.x + i * THREADS);
    }
    __device__ inline void store(const Logp& a, uint16_t* wt) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (threadIdx.x + i * THREADS < a.bins) wt[threadIdx.x + i * THREADS] = (uint16_t)w[i];
        for (uint32_t i = threadIdx.x + 1024; i < a.bins; i += THREADS) wt[i] = (uint16_t)weight_below(a, i);
    }
};

constexpr size_t kLogpFewRows = 512;  // two blocks of 16 waves per CU

// Where the alternatives are looked for.
constexpr int kLogpCandidates = 512, kLogpTiles = 128;
struct TopLds {
    uint64_t cand[kLogpCandidates], red[16], last;
    int tile[kLogpTiles];
    int tiles, count;
    int32_t edge;
};

// A value that n tiles at least reach, by one wave: one that n of the maxima over every 64th tile
// reach, or the least value where there are fewer tiles.  (Ranking the 64 maxima among one
// another took 1 us more than this search.)
__device__ inline int32_t logp_edge(const Logp& a, const int32_t* tm) {
    const int lane = threadIdx.x & 63;
    int32_t own = INT32_MIN;
    for (int i0 = lane; i0 < a.tiles; i0 += 64 * 8) {
        int32_t x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = i0 + 64 * k < a.tiles ? tm[i0 + 64 * k] : INT32_MIN;
#pragma unroll
        for (int k = 0; k < 8; ++k) own = max(own, x[k]);
    }
    if (a.n > a.tiles) return INT32_MIN;
    // the largest number that n of the 64 reach, bit by bit from the first in which they differ; its low
    // bits need not be known once no more than n do
    const uint32_t u = (uint32_t)own ^ 0x80000000u;
    const uint32_t high = (uint32_t)__builtin_amdgcn_readfirstlane(wave_max_i32(own)) ^ 0x80000000u;
    const uint32_t low = (uint32_t)__builtin_amdgcn_readfirstlane(~wave_max_i32(~own)) ^ 0x80000000u;
    const int bits = 32 - __builtin_clz((high ^ low) | 1u);
    uint32_t reached = bits == 32 ? 0u : high >> bits << bits;
    for (int b = bits - 1; b >= 0; --b) {
        const uint32_t t = reached | (1u << b);
        const int c = __builtin_popcountll(__ballot(u >= t));
        if (c < a.n) continue;
        reached = t;
        if (c == a.n) break;
    }
    return (int32_t)(reached ^ 0x80000000u);
}

// The n largest values one after another, by the whole block: of the n tiles with the largest
// maxima (of equal ones the first), found by the first wave.  For rows with many equal values.
template <int THREADS, class Answer>
__device__ inline void logp_top_in_turn(const Logp& a, const int32_t* z, const int32_t* tm, TopLds& t, const Answer& answer) {
    constexpr int kWaves = THREADS / 64, kEach = (int)kLogpMaxTop / kWaves;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), n = min(a.n, a.tiles);
    if (w == 0) {
        auto best_below = [&](uint64_t last) {
            uint64_t key = 0;
            for (int i0 = lane; i0 < a.tiles; i0 += 64 * 4) {
                int32_t x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = i0 + 64 * k < a.tiles ? tm[i0 + 64 * k] : 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint64_t o = max_key(x[k], (uint32_t)(i0 + 64 * k));
                    if (i0 + 64 * k < a.tiles && o < last && o > key) key = o;
                }
            }
            return key;
        };
        uint64_t own = best_below(~0ull);
        for (int k = 0; k < n; ++k) {
            const uint64_t top = wave_max_u64(own);
            if (lane == 0) t.tile[k] = (int)key_index(top);
            if (own == top) own = best_below(top);
        }
    }
    __syncthreads();
    uint64_t key[kEach][4];
#pragma unroll
    for (int k = 0; k < kEach; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = w + k * kWaves < n ? t.tile[w + k * kWaves] * kLogpTile + 4 * lane + e : a.V;
            key[k][e] = i < a.V ? max_key(z[i], (uint32_t)i) : 0;
        }
    uint64_t last = ~0ull;
    for (int k = 0; k < a.n; ++k) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (key[i][e] < last && key[i][e] > best) best = key[i][e];
        best = wave_max_u64(best);
        if (lane == 0) t.red[w] = best;
        __syncthreads();
        if (w == 0) {
            best = wave_max_u64(lane < kWaves ? t.red[lane] : 0);
            if (lane == 0) {
                t.last = best;
                answer(k, best);
            }
        }
        __syncthreads();
        last = t.last;
    }
}

// A block per row adds the chunks' counts up, a wave per chunk, and finds the alternatives: every
// tile that reaches the edge is read, every value of it that does is a candidate, and a
// candidate's place is how many are before it.  Few are, unless many values are
// equal; past the room for them, logp_top_in_turn.  16 waves where few rows wait for it, four
// where rows fill the chip.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void logp_row_kernel(Logp a) {
    constexpr int kWaves = THREADS / 64;
    extern __shared__ uint16_t wt[];
    __shared__ TopLds top;
    __shared__ uint64_t red[2][kWaves];
    __shared__ int64_t s_ln;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int32_t* z = a.z + (size_t)r * a.ldz;
    const int32_t* cm = a.cmax + (size_t)r * a.chunks;
    const int32_t* tm = a.tmax + (size_t)r * a.tiles;
    BinWeights<THREADS> bw;
    bw.load(a);
    int32_t m = INT32_MIN;
    for (int c = lane; c < a.chunks; c += 64) m = max(m, cm[c]);
    bw.store(a, wt);
    if (tid == 0) top.count = top.tiles = 0;
    m = wave_max_i32(m);
    __syncthreads();
    if (w == kWaves - 1 && a.n) {
        const int32_t edge = logp_edge(a, tm);
        if (lane == 0) top.edge = edge;
    }
    uint64_t s = 0, moment = 0;  // below 2^35 and 2^48
    for (int c = w; c < a.chunks; c += kWaves) {
        const uint32_t d = (uint32_t)m - (uint32_t)cm[c];
        if (d >= a.bins) continue;
        const uint32_t* n = a.counts + ((size_t)r * a.chunks + c) * a.words;
        for (uint32_t i0 = lane; i0 < a.words; i0 += 8 * 64) {
            uint32_t two[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) two[k] = i0 + 64 * k < a.words ? n[i0 + 64 * k] : 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t at = d + 2 * (i0 + 64 * k);
                const uint64_t e0 = (uint64_t)(two[k] & 0xFFFFu) * (at < a.bins ? wt[at] : 0u);
                const uint64_t e1 = (uint64_t)(two[k] >> 16) * (at + 1 < a.bins ? wt[at + 1] : 0u);
                s += e0 + e1;
                moment += e0 * at + e1 * (at + 1);
            }
        }
    }
    s = wave_sum_u64(s);
    moment = wave_sum_u64(moment);
    if (lane == 0) {
        red[0][w] = s;
        red[1][w] = moment;
    }
    __syncthreads();
    if (w == 0) {
        s = wave_sum_u64(lane < kWaves ? red[0][lane] : 0);
        moment = wave_sum_u64(lane < kWaves ? red[1][lane] : 0);
        const int64_t ln = ln_q16_of_sum(s < 1 ? 1u : s);
        if (lane == 0) {
            s_ln = ln;
            if (a.entropy) a.entropy[r] = s ? ln + div_round(moment << 10, s) : 0;
        }
    }
    if (a.n) {
        const int32_t edge = top.edge;
        for (int i = tid; i < a.tiles; i += THREADS)
            if (tm[i] >= edge) {
                const int at = atomicAdd(&top.tiles, 1);
                if (at < kLogpTiles) top.tile[at] = i;
            }
        __syncthreads();
        const int n = min(top.tiles, kLogpTiles);
        for (int k = w; k < n; k += kWaves) {
            const int i = top.tile[k] * kLogpTile + 4 * lane;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int32_t x = i + e < a.V ? z[i + e] : INT32_MIN;
                if (i + e >= a.V || x < edge) continue;
                const int at = atomicAdd(&top.count, 1);
                if (at < kLogpCandidates) top.cand[at] = max_key(x, (uint32_t)(i + e));
            }
        }
    }
    __syncthreads();
    const int64_t ln = s_ln;
    for (int i = tid; i < a.T; i += THREADS) {
        const int64_t t = a.tokens[(size_t)r * a.T + i];
        a.logprobs[(size_t)r * a.T + i] = t < 0 || t >= a.V ? 0 : ((int64_t)z[t] - (int64_t)m) * 1024 - ln;
    }
    if (!a.n) return;
    auto answer = [&](int k, uint64_t o) {
        a.top_tokens[(size_t)r * a.n + k] = key_index(o);
        a.top_logprobs[(size_t)r * a.n + k] = ((int64_t)key_value(o) - (int64_t)m) * 1024 - ln;
    };
    const int count = top.count;  // at least n
    if (top.tiles > kLogpTiles || count > kLogpCandidates) {
        logp_top_in_turn<THREADS>(a, z, tm, top, answer);
        return;
    }
    for (int i = tid; i < count; i += THREADS) {
        const uint64_t own = top.cand[i];
        int before = 0;
        for (int j = 0; j < count; ++j) before += top.cand[j] > own ? 1 : 0;
        if (before < a.n) answer(before, own);
    }
}

}  // namespace
}  // namespace myl

using namespace myl;

extern "C" {

size_t myl_logprobs_workspace(const myl_ctx* ctx, size_t rows, size_t vocab, size_t top_n, size_t lut_len) {
    const LogpShape s{rows, vocab, 0, top_n, lut_len};
    return !ctx || logp_refuse(s) ? 0 : logp_plan(s).bytes;
}

int myl_logprobs_dev(myl_ctx* ctx, const int32_t* logits, size_t rows, size_t vocab, size_t ldz, const int16_t* exp_lut,
                     size_t lut_len, const int64_t* tokens, size_t n_tokens, size_t top_n, int64_t* logprobs, int64_t* entropy,
                     int64_t* top_tokens, int64_t* top_logprobs, void* workspace, size_t workspace_bytes) {
    if (!ctx) return MYL_E_INVALID;
    const char* what = "logprobs_dev";
    auto bad = [&](const char* why) { return ctx->fail(MYL_E_INVALID, std::string(what) + ": " + why); };
    const LogpShape s{rows, vocab, n_tokens, top_n, lut_len};
    if (const char* why = logp_refuse(s)) return bad(why);
    if (ldz < vocab) return bad("leading dimension too small");
    if (rows == 0) return MYL_OK;
    if (!logits || !exp_lut || (n_tokens && (!tokens || !logprobs)) || (top_n && (!top_tokens || !top_logprobs))) return bad("null operand");
    const LogpPlan pl = logp_plan(s);
    if (!workspace || workspace_bytes < pl.bytes) return bad("workspace too small (myl_logprobs_workspace)");
    if ((uintptr_t)workspace & 15) return bad("workspace must be 16-byte aligned");
    const DeviceGuard guard(ctx->device);
    char* ws = static_cast<char*>(workspace);
    Logp a{};
    a.z = logits; a.tokens = tokens; a.lut = exp_lut;
    a.logprobs = logprobs; a.entropy = entropy; a.top_tokens = top_tokens; a.top_logprobs = top_logprobs;
    a.ldz = ldz; a.V = (int)vocab; a.T = (int)n_tokens; a.n = (int)top_n;
    a.chunks = pl.chunks; a.tiles = pl.tiles; a.bins = pl.bins; a.words = pl.words;
    a.cmax = reinterpret_cast<int32_t*>(ws + pl.off_max);
    a.tmax = reinterpret_cast<int32_t*>(ws + pl.off_tiles);
    a.counts = reinterpret_cast<uint32_t*>(ws + pl.off_counts);
    logp_count_kernel<<<dim3((unsigned)pl.chunks, (unsigned)rows), kBlk, (size_t)pl.words * 8, ctx->stream>>>(a);
    if (rows <= kLogpFewRows) logp_row_kernel<1024><<<(unsigned)rows, 1024, (size_t)pl.bins * 2, ctx->stream>>>(a);
    else logp_row_kernel<256><<<(unsigned)rows, 256, (size_t)pl.bins * 2, ctx->stream>>>(a);
    return ctx->hip(hipGetLastError(), what);
}

}  // extern "C"
