// paged_attn.hip -- integer attention (attention.rs:42-90 with softmax.rs:12-64) of each
// sequence's newest rows over a paged cache, split over the length and joined:
// myl_attention_paged_dev.
//
// A probability p_j = RNE(e_j 2^f / S) needs the exact maximum and exp sum of its whole
// row before it is rounded, so a row is not joined from finished pieces; four launches
// follow one another, each with a block per tile of vectors (query heads of a
// sequence's rows that read one KV head) and range of keys:
//   paged_qk_kernel    the scores z_j, kept, and each range's maximum
//   paged_sum_kernel   e_j = exp_lut[(max - z_j) >> lut_shift] as 16 bits, the ranges' sums
//   paged_pv_kernel    p_j from e_j and S, sum p_j v_j over each range
//   paged_out_kernel   the sums over the ranges, rounded and clamped
// Keys and values are read once each, the scores and exp values (6 bytes a key and head) written
// and read beside them.  us by traced kernel in that order (apart from the calls, not adding up to them),
// heads of 128, seven to a KV head of four: 64 rows of up to 12000 keys 120 + 24 + 122 + 6 (284 a call;
// 4.1 TB/s of keys and values), one row of 100000 23 + 8.5 + 22 + 4.8 (58), 24 rows of up to 2500
// 13 + 7 + 14 + 4 (36), of which starting and draining four launches is most; 3 x 500 rows of prompts
// before 2000 keys 111 + 79 + 344 + 49 (581: made for a sequence's newest few rows).  Joining the
// ranges in the tile's last block instead of a fourth launch took longer (24 x 2500: 38.7 us with
// write-through stores and loads, 107 with device fences).  Few keys take one launch
// (paged_short_kernel).
#include "abi_internal.h"
#include "attn_fixed.h"
#include "gemm_mfma.h"
#include "ops.h"
#include "paged_plan.h"
#include "wave.h"

#include <algorithm>
#include <string>

namespace myl {
namespace {

struct PagedAttn {
    const int16_t *q, *kp, *vp;
    const int32_t *tables, *lens;
    const int16_t* lut;
    int16_t* out;
    // the workspace, for each tile: scores [keys / 4][width][4], exp values the same, maxima and
    // sums [ranges][width], whether a range holds keys on no page [ranges], sums of p v
    // [ranges][width][hd]
    int32_t* z;
    uint16_t* e;
    int32_t *pmax, *pout, *holes;
    uint32_t* psum;
    size_t ldq, ldo, ldt, page_stride, head_stride, pos_stride;
    int64_t mult;
    ScoreScale scale;
    SmallDiv n, G, page, kvh, tiles, ranges_d, width_d, heads_d, range_d;
    int heads, max_len, n_pages, keys, range, ranges, width, vectors, places, entries;  // entries: of a block's page table
    uint32_t lut_len;
    uint8_t shift, lut_shift, prob_frac;
};

// A block's part of the work.
struct Part {
    int seq, g, v0, nv;  // KV head; first vector, vectors of the tile
    int tile;            // among all
    int range, j0, j1;   // keys [j0, j1) of the sequence, j1 up to the longest row's end
    int lmin;            // the shortest row's end
    int row0;
};

// The row and head of a tile's vector v (places past the last repeat it).
__device__ inline int vector_of(const PagedAttn& a, const Part& p, int v, int& head) {
    int h;
    const int row = p.row0 + divmod(a.G, p.v0 + min(v, p.nv - 1), h);
    head = p.g * (int)a.G.d + h;
    return row;
}
// The keys of a row, counted from position 0.
__device__ inline int keys_of(const PagedAttn& a, int row) { return min(max(a.lens[row], 0), a.max_len); }

// The block's tile and range; false: none.  Blocks of the tiles that read one range follow one
// another on one XCD (block b runs on XCD b % 8).
__device__ inline bool place_of_block(const PagedAttn& a, Part& p) {
    int tile, rest;
    const int q = divmod(a.tiles, (int)(blockIdx.x >> 3), tile), i = 8 * q + (int)(blockIdx.x & 7);
    p.tile = -1;
    if (i >= a.places) return false;
    rest = divmod(a.ranges_d, i, p.range);
    p.seq = divmod(a.kvh, rest, p.g);
    p.tile = rest * (int)a.tiles.d + tile;
    p.v0 = tile * a.width;
    p.nv = min(a.width, a.vectors - p.v0);
    p.row0 = p.seq * (int)a.n.d;
    p.j0 = p.range * a.range;
    return true;
}
// The range's end; false: it has no key.  Returns the keys of the thread's vector, v % 16, in lim.
__device__ inline bool ends_of(const PagedAttn& a, Part& p, int v, int& lim) {
    int head;
    lim = keys_of(a, vector_of(a, p, v & 15, head));
    p.j1 = min(p.j0 + a.range, __builtin_amdgcn_readfirstlane(wave_max_i32(lim)));
    p.lmin = __builtin_amdgcn_readfirstlane(~wave_max_i32(~lim));
    return p.j0 < p.j1;
}
__device__ inline bool ends_of(const PagedAttn& a, Part& p, int v) {
    int lim;
    return ends_of(a, p, v, lim);
}
// Both; lim of vector lane % 16.  p.tile < 0: the block has no tile.
__device__ inline bool part_of(const PagedAttn& a, Part& p, int& lim) {
    return place_of_block(a, p) && ends_of(a, p, threadIdx.x, lim);
}

// The element offsets of a range's pages in LDS, kNoPage where a table names none.  The table
// names pages up to max_len at least, so its loads need not wait for the rows' lengths.
constexpr uint64_t kNoPage = ~0ull;
__device__ inline int pages_of_range(const PagedAttn& a, const Part& p, uint64_t* tab, int* bad) {
    int rem;
    const int p0 = divmod(a.page, p.j0, rem);
    const int most = divmod(a.page, min(p.j0 + a.range, a.max_len) - 1, rem) - p0 + 1, n = divmod(a.page, p.j1 - 1, rem) - p0 + 1;
    const int32_t* t = a.tables + (size_t)p.seq * a.ldt + p0;
    bool none = false;
    for (int i = threadIdx.x; i < most; i += blockDim.x) {
        const int id = t[i];
        const bool ok = id >= 0 && id < a.n_pages;
        none |= !ok && i < n;
        tab[i] = ok ? (uint64_t)id * a.page_stride + (uint64_t)p.g * a.head_stride : kNoPage;
    }
    const bool any = __any(none);
    if ((threadIdx.x & 63) == 0) bad[threadIdx.x >> 6] = any ? 1 : 0;
    return p0;
}
// Where position j lies (one on no page: some place of the pages).
__device__ inline size_t place_of(const PagedAttn& a, const uint64_t* tab, int p0, int j) {
    int off;
    const int at = divmod(a.page, j, off) - p0;
    const uint64_t base = tab[at];
    return (base == kNoPage ? 0 : base) + (size_t)off * a.pos_stride;
}
__device__ inline bool on_page(const PagedAttn& a, const uint64_t* tab, int p0, int j) {
    int off;
    return tab[divmod(a.page, j, off) - p0] != kNoPage;
}

// A barrier that leaves loads in flight.
__device__ inline void block_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ inline int32_t dot_pairs(uint32_t w, uint32_t x, int32_t acc) {
    typedef short __attribute__((ext_vector_type(2))) s2;
    return __builtin_amdgcn_sdot2(__builtin_bit_cast(s2, w), __builtin_bit_cast(s2, x), acc, false);
}
__device__ inline void planes8(const uint4& x, uint32_t* h, uint32_t* l) {
    h[0] = __builtin_amdgcn_perm(x.y, x.x, 0x07050301u);
    h[1] = __builtin_amdgcn_perm(x.w, x.z, 0x07050301u);
    l[0] = __builtin_amdgcn_perm(x.y, x.x, 0x06040200u) ^ 0x80808080u;
    l[1] = __builtin_amdgcn_perm(x.w, x.z, 0x06040200u) ^ 0x80808080u;
}
// 16 dimensions (two 16-byte loads) as matrix operands: byte planes x = 256 hi + lo' + 128.
__device__ inline void planes16(const uint4 (&x)[2], v4i32_t& h, v4i32_t& l) {
    uint32_t hw[4], lw[4];
    planes8(x[0], hw, lw);
    planes8(x[1], hw + 2, lw + 2);
    h = v4i32_t{(int)hw[0], (int)hw[1], (int)hw[2], (int)hw[3]};
    l = v4i32_t{(int)lw[0], (int)lw[1], (int)lw[2], (int)lw[3]};
}

// A wave's 16-key tiles of keys, tile after tile straight into a ring of NB (two) places in
// its own LDS: key r of a tile is row r, its 16-byte chunk x at place x ^ (r mod chunks).
// Loads retire in order, so a tile has landed when only younger ones' are outstanding.
// Where pages hold whole tiles (ALIGNED: a multiple of 16 positions), a tile is one address for
// the wave and 32-bit offsets of the lanes; elsewhere each lane and load divides (64 rows of 12000 keys by
// pages of 100 310 us, of 64 281; 12 x 4 of 3001 by 24 46.1, by 16 41.3).  What one block alone reads is loaded past the caches'
// usual order (64 rows of 12000 keys: 284 us a call, 306 without; two tiles that share their
// keys: 55.9 against 52.2, so there not).
typedef __attribute__((address_space(1))) const void global_void;
typedef __attribute__((address_space(3))) void lds_void;
constexpr int kOnce = 2;  // nontemporal
template <int HD, int NB, bool ALIGNED>
struct Tiles {
    static constexpr int CH = HD / 8, ROWS = 64 / CH, NI = 16 / ROWS, kBytes = 32 * HD;
    const char* pages;
    int8_t* ring;
    uint32_t lane[NI];  // ALIGNED: the lane's bytes from the tile's first
    int row, chunk;
    __device__ inline void begin(const PagedAttn& a, const int16_t* p, int8_t* lds) {
        pages = reinterpret_cast<const char*>(p);
        ring = lds;
        const int l = threadIdx.x & 63;
        row = l / CH;
        chunk = l % CH;
#pragma unroll
        for (int i = 0; i < NI; ++i) lane[i] = 2u * ((uint32_t)(i * ROWS + row) * (uint32_t)a.pos_stride + 8u * (uint32_t)at(i * ROWS + row, chunk));
    }
    __device__ static inline int at(int r, int x) { return x ^ (r & (CH - 1)); }
    // Keys j .. j + 15 into place `slot`; those from j1 on hold anything.
    __device__ inline void issue(const PagedAttn& a, const uint64_t* tab, int p0, int j, int j1, int slot) const {
        int8_t* to = ring + slot * kBytes;
        if (ALIGNED) {
            const char* base = pages + 2 * uniform_u64(place_of(a, tab, p0, j));
            if (a.tiles.d == 1)
#pragma unroll
                for (int i = 0; i < NI; ++i)
                    __builtin_amdgcn_global_load_lds((global_void*)(uintptr_t)(base + lane[i]), (lds_void*)(to + i * 1024), 16, 0, kOnce);
            else
#pragma unroll
                for (int i = 0; i < NI; ++i)
                    __builtin_amdgcn_global_load_lds((global_void*)(uintptr_t)(base + lane[i]), (lds_void*)(to + i * 1024), 16, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const uint64_t from = place_of(a, tab, p0, min(j + i * ROWS + row, j1 - 1)) + (uint64_t)(8 * at(i * ROWS + row, chunk));
                __builtin_amdgcn_global_load_lds((global_void*)(uintptr_t)(pages + 2 * from), (lds_void*)(to + i * 1024), 16, 0, 0);
            }
        }
    }
    // The oldest tile has landed when `left` younger ones and OTHER accesses behind them remain.
    template <int OTHER>
    __device__ static inline void wait(int left) {
        static_assert(NB == 2, "the cases below");
        if (left >= 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NI + OTHER) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(OTHER) : "memory");
    }
};

// How many of a range's tiles fall to a wave, every NW-th.
template <int NW>
__device__ inline int tiles_of_wave(const Part& p, int wave) {
    static_assert((NW & (NW - 1)) == 0, "a shift");
    return max(((p.j1 - p.j0 + 15) >> 4) - wave + NW - 1, 0) / NW;
}

// Scores on v_mfma_i32_16x16x64_i8: K positions are rows, vectors columns, so lane l holds
// vector l % 16 and positions 4 (l / 16) .. + 3 of a 16-position tile.  The byte planes of the
// keys are k = 256 kh + kl + 128 with kl = (k & 255) - 128; those of the queries q = 256 qh +
// ql with ql the low byte as a signed one, which exist for q < 32640:
//   q.k = 65536 qh kh + 256 (qh kl + ql kh) + ql kl + 128 sum q
// with no sum over k.  A tile with a larger q takes q = 256 qh + ql + 128 too (BALANCED
// false), for which 256 128 sum kh + 128 sum kl come from the matrix cores as well (a B operand
// of 64s, added twice).  As 256 u + r the score takes 32-bit steps (ScoreScale);
// other scales take the 64-bit form (FAST false).
// 64 rows of up to 12000 keys: 119 us, bound by bytes; short calls by the loads' latency: two
// tiles a wave are on their way.
constexpr int kQkRing = 2;
// NW: waves of the block, a tile in turn each.  STORED: the scores go to memory, not LDS.
template <int HD, bool FAST, bool ALIGNED, bool BALANCED, int NW, bool STORED>
__device__ inline void paged_scores(const PagedAttn& a, const Part& p, int lim, const uint64_t* tab, int p0, bool holes, int8_t* ring,
                                    const uint4 (&qx)[HD / 64][2], int32_t* z0, int32_t* red) {
    using T = Tiles<HD, kQkRing, ALIGNED>;
    constexpr int NS = HD / 64, NB = kQkRing;
    const int lane = threadIdx.x & 63, c = lane & 15, kb = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    T tiles;
    tiles.begin(a, a.kp, ring);
    const int n = tiles_of_wave<NW>(p, wave), jw = p.j0 + 16 * wave;
#pragma unroll
    for (int t = 0; t < NB; ++t)
        if (t < n) tiles.issue(a, tab, p0, jw + 16 * NW * t, p.j1, t);
    v4i32_t qh[NS], ql[NS];
    int32_t qsum = 0;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const uint32_t w[8] = {qx[s][0].x, qx[s][0].y, qx[s][0].z, qx[s][0].w, qx[s][1].x, qx[s][1].y, qx[s][1].z, qx[s][1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) qsum = dot_pairs(w[i], 0x00010001u, qsum);
        if (BALANCED) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // 128 carries into the high byte; into the upper half's too, where it is taken back
                auto carried = [](uint32_t x) { return ((x & 0xFFFFu) + 0x80u) | (((x >> 16) + 0x80u) << 16); };
                qh[s][i] = (int)__builtin_amdgcn_perm(carried(w[2 * i + 1]), carried(w[2 * i]), 0x07050301u);
                ql[s][i] = (int)__builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x06040200u);
            }
        } else {
            planes16(qx[s], qh[s], ql[s]);
        }
    }
    qsum += __shfl_xor(qsum, 16, 64);
    qsum = 128 * (qsum + __shfl_xor(qsum, 32, 64));
    const v4i32_t sixty4 = {0x40404040, 0x40404040, 0x40404040, 0x40404040}, zero = {0, 0, 0, 0}, qs4 = {qsum, qsum, qsum, qsum};
    int32_t* const zt = z0 + 4 * (kb * a.width + c);
    int32_t best = INT32_MIN;
    int slot = 0;
    for (int t = 0; t < n; ++t) {
        const int j = jw + 16 * NW * t;
        // one score store at least for each of the last NB - 1 tiles lies between
        if (STORED && t >= NB) T::template wait<NB - 1>(n - 1 - t);
        else T::template wait<0>(n - 1 - t);
        const int8_t* k8 = ring + slot * T::kBytes + c * 2 * HD;
        v4i32_t raw[NS][2];
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) raw[s][i] = *reinterpret_cast<const v4i32_t*>(k8 + (T::at(c, 8 * s + 2 * kb + i) << 4));
        // in registers before the tile's place is loaded again
        if (NS == 2) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(raw[0][0]), "+v"(raw[0][1]), "+v"(raw[NS - 1][0]), "+v"(raw[NS - 1][1])::"memory");
        else asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(raw[0][0]), "+v"(raw[0][1])::"memory");
        if (t + NB < n) tiles.issue(a, tab, p0, j + 16 * NW * NB, p.j1, slot);
        slot = slot + 1 == NB ? 0 : slot + 1;
        v4i32_t kh[NS], kl[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            uint4 x[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) x[i] = make_uint4((uint32_t)raw[s][i][0], (uint32_t)raw[s][i][1], (uint32_t)raw[s][i][2], (uint32_t)raw[s][i][3]);
            planes16(x, kh[s], kl[s]);
        }
        v4i32_t hh = zero, mid = zero, ll = qs4;
        if (!BALANCED)
#pragma unroll
            for (int s = 0; s < 2 * NS; ++s) {
                mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(kh[s / 2], sixty4, mid, 0, 0, 0);
                ll = __builtin_amdgcn_mfma_i32_16x16x64_i8(kl[s / 2], sixty4, ll, 0, 0, 0);
            }
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(kh[s], ql[s], mid, 0, 0, 0);
            ll = __builtin_amdgcn_mfma_i32_16x16x64_i8(kl[s], ql[s], ll, 0, 0, 0);
            hh = __builtin_amdgcn_mfma_i32_16x16x64_i8(kh[s], qh[s], hh, 0, 0, 0);
            mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(kl[s], qh[s], mid, 0, 0, 0);
        }
        int32_t z[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int32_t u = 256 * hh[i] + mid[i] + (ll[i] >> 8);
            const uint32_t r = (uint32_t)ll[i] & 255u;
            z[i] = FAST ? a.scale(u, r) : (int32_t)rshift_round64(wmul64(256 * (int64_t)u + (int64_t)r, a.mult), a.shift);
        }
        if (c < a.width) *reinterpret_cast<int4*>(zt + (size_t)j * a.width) = make_int4(z[0], z[1], z[2], z[3]);
        if (!holes && j + 16 <= p.lmin) {
            best = max(best, max(max(z[0], z[1]), max(z[2], z[3])));
        } else {
            for (int i = 0; i < 4; ++i) {
                const int key = j + 4 * kb + i;
                const bool ok = key < min(lim, p.j1) && (!holes || on_page(a, tab, p0, min(key, p.j1 - 1)));
                best = ok ? max(best, z[i]) : best;
            }
        }
    }
    best = max(best, __shfl_xor(best, 16, 64));
    best = max(best, __shfl_xor(best, 32, 64));
    if (kb == 0) red[16 * wave + c] = best;
}

// A tile's vectors in whole lines to LDS; whether one is too large for the signed low byte, by wave.
template <int HD>
__device__ inline void stage_queries(const PagedAttn& a, const Part& p, int8_t* qlds, int* large) {
    constexpr int CH = HD / 8;
    const int tid = threadIdx.x, v = tid / CH;
    bool over = false;
    if (v < 16) {
        int head;
        const int row = vector_of(a, p, v, head);
        const uint4 x = *reinterpret_cast<const uint4*>(a.q + (size_t)row * a.ldq + (size_t)head * HD + 8 * (tid % CH));
        *reinterpret_cast<uint4*>(qlds + v * 2 * HD + (((tid % CH) ^ (v & (CH - 1))) << 4)) = x;
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) over |= (int16_t)(w[i] & 0xFFFFu) >= 32640 || (int32_t)w[i] >> 16 >= 32640;
    }
    over = __any(over);
    if ((tid & 63) == 0) large[tid >> 6] = over ? 1 : 0;
}
template <int N>
__device__ inline bool any_of(const int (&x)[N]) {
    int s = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) s |= x[i];
    return __builtin_amdgcn_readfirstlane(s) != 0;
}

template <int HD, bool FAST, bool ALIGNED, int NW, bool STORED>
__device__ inline void scores_of_range(const PagedAttn& a, const Part& p, int lim, const uint64_t* tab, int p0, bool holes, int8_t* rings,
                                       const int8_t* qlds, bool large, int32_t* z0, int32_t* red) {
    constexpr int NS = HD / 64, CH = HD / 8;
    const int lane = threadIdx.x & 63, c = lane & 15, kb = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint4 qx[NS][2];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            qx[s][i] = *reinterpret_cast<const uint4*>(qlds + c * 2 * HD + (((8 * s + 2 * kb + i) ^ (c & (CH - 1))) << 4));
    int8_t* const ring = rings + wave * kQkRing * 32 * HD;
    if (large) paged_scores<HD, FAST, ALIGNED, false, NW, STORED>(a, p, lim, tab, p0, holes, ring, qx, z0, red);
    else paged_scores<HD, FAST, ALIGNED, true, NW, STORED>(a, p, lim, tab, p0, holes, ring, qx, z0, red);
}

template <int HD, bool FAST, bool ALIGNED>
__global__ __launch_bounds__(256, 4) void paged_qk_kernel(PagedAttn a) {
    extern __shared__ __align__(16) int8_t lds[];  // the waves' rings, the range's pages
    __shared__ __align__(16) int8_t qlds[16 * 2 * HD];
    __shared__ int32_t red[64];
    __shared__ int bad[4], large[4];
    static_assert(sizeof qlds + sizeof red + sizeof bad + sizeof large <= kPagedOwnLds, "paged_ranges");
    uint64_t* const tab = reinterpret_cast<uint64_t*>(lds + 4 * kQkRing * 32 * HD);
    Part p;
    int lim;
    if (!part_of(a, p, lim)) return;
    const int tid = threadIdx.x;
    stage_queries<HD>(a, p, qlds, large);
    const int p0 = pages_of_range(a, p, tab, bad);
    __syncthreads();
    const bool holes = any_of(bad);
    scores_of_range<HD, FAST, ALIGNED, 4, true>(a, p, lim, tab, p0, holes, lds, qlds, any_of(large), a.z + (size_t)p.tile * a.width * a.keys, red);
    __syncthreads();
    const size_t at = (size_t)p.tile * a.ranges + p.range;
    if (tid < a.width) a.pmax[at * a.width + tid] = max(max(red[tid], red[16 + tid]), max(red[32 + tid], red[48 + tid]));
    if (tid == 0) a.holes[at] = holes ? 1 : 0;
}

// The lane's vector and groups of four keys: c = tid % width, the groups tid / width and on.
struct Lanes {
    int c, k, step;  // step 0: the thread has none
    __device__ static inline Lanes of(const PagedAttn& a) {
        Lanes l;
        int rem;
        l.step = divmod(a.width_d, (int)blockDim.x, rem);
        l.k = divmod(a.width_d, (int)threadIdx.x, l.c);
        if (l.k >= l.step) l.step = 0;
        return l;
    }
};

__device__ inline int lim_of(const PagedAttn& a, const Part& p, int v) {
    int head;
    return keys_of(a, vector_of(a, p, v, head));
}

// e_j and their sums.  Bound by latency (a launch that loads, computes and stores once), so every
// load that needs no other's result is issued first: the rows' lengths, the ranges' maxima, the
// table's start and the thread's first scores.
constexpr uint32_t kSumLut = kPagedLdsLut;  // entries in LDS
constexpr int kSumAhead = 4, kFoldAhead = 4;
// Eight table entries, negative ones as 0, and 0 from entry n on.
__device__ inline uint4 table8(const int16_t* lut, uint32_t i, uint32_t n) {
    uint32_t w[4] = {0, 0, 0, 0};
    if (i + 8 <= n) {
        const uint4 x = *reinterpret_cast<const uint4*>(lut + i);
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    } else {
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k)
            if (i + k < n) w[k / 2] |= (uint32_t)(uint16_t)lut[i + k] << (16 * (k & 1));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] &= ((w[k] & 0x8000u) ? 0u : 0xFFFFu) | ((w[k] >> 31) ? 0u : 0xFFFF0000u);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// The copy's first entries, before what they wait behind; the rest, and the copy's `have` entries and a 0.
template <int THREADS>
struct TableCopy {
    static constexpr int kEach = 512 / THREADS;
    uint4 x[kEach];
    __device__ inline void load(const PagedAttn& a, uint32_t have) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) x[i] = table8(a.lut, 8u * (threadIdx.x + (uint32_t)THREADS * i), have);
    }
    __device__ inline void store(const PagedAttn& a, uint32_t have, uint16_t* lut) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t at = 8u * (threadIdx.x + (uint32_t)THREADS * i);
            if (at <= have) *reinterpret_cast<uint4*>(lut + at) = x[i];
        }
        for (uint32_t i = 8u * (threadIdx.x + 512u); i <= have; i += 8u * THREADS) *reinterpret_cast<uint4*>(lut + i) = table8(a.lut, i, have);
    }
};
// e of four keys of a vector with the maximum m, and their sum.
__device__ inline uint32_t exps_of(const PagedAttn& a, const Part& p, const uint16_t* lut, uint32_t have, int32_t m, const int4& v, int key, int lim,
                                   bool holes, const uint64_t* tab, int p0, uint32_t (&e)[4]) {
    const int32_t z[4] = {v.x, v.y, v.z, v.w};
    uint32_t s = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // sat_sub and the lookup of softmax.rs:12-38
        const uint32_t below = min((uint32_t)m - (uint32_t)z[i], 0x7FFFFFFFu) >> (a.lut_shift & 31u);
        uint32_t x = lut[min(below, have)];
        if (a.lut_len > kSumLut && below >= have && below < a.lut_len) x = (uint32_t)max((int32_t)a.lut[below], 0);
        bool ok = key + i < lim;
        if (holes) ok = ok && on_page(a, tab, p0, min(key + i, p.j1 - 1));
        e[i] = ok ? x : 0u;
        s += e[i];
    }
    return s;
}

__global__ __launch_bounds__(256) void paged_sum_kernel(PagedAttn a) {
    extern __shared__ __align__(16) uint64_t tab[];
    __shared__ __align__(16) uint16_t lut[kSumLut + 8];
    __shared__ int32_t s_max[16];
    __shared__ uint32_t s_sum[16];
    __shared__ int bad[4];
    Part p;
    if (!place_of_block(a, p)) return;
    const int tid = threadIdx.x;
    const Lanes l = Lanes::of(a);
    const size_t at = (size_t)p.tile * a.ranges, base = (size_t)p.tile * a.width * a.keys;
    const uint32_t have = min(a.lut_len, kSumLut);
    // within the workspace whatever the lengths: groups of four keys below a.keys
    auto group = [&](int i) { return (p.j0 >> 2) + l.k + i * l.step; };
    int4 z4[kSumAhead];
#pragma unroll
    for (int i = 0; i < kSumAhead; ++i) z4[i] = *reinterpret_cast<const int4*>(a.z + base + ((size_t)min(group(i), a.keys / 4 - 1) * a.width + l.c) * 4);
    int32_t m4[kFoldAhead];
#pragma unroll
    for (int i = 0; i < kFoldAhead; ++i) m4[i] = a.pmax[(at + min(l.k + i * l.step, a.ranges - 1)) * a.width + l.c];
    const int any_holes = a.holes[at + p.range];
    TableCopy<256> table;
    table.load(a, have);
    const int lim = lim_of(a, p, l.c);
    if (!ends_of(a, p, tid)) return;
    const bool holes = __builtin_amdgcn_readfirstlane(any_holes) != 0;
    int p0 = 0;
    if (holes) p0 = pages_of_range(a, p, tab, bad);
    if (tid < 16) {
        s_max[tid] = INT32_MIN;
        s_sum[tid] = 0;
    }
    table.store(a, have, lut);
    __syncthreads();
    int32_t m = INT32_MIN;
#pragma unroll
    for (int i = 0; i < kFoldAhead; ++i)
        if (l.k + i * l.step < a.ranges && (l.k + i * l.step) * a.range < lim) m = max(m, m4[i]);
    if (l.step) {
        for (int r = l.k + kFoldAhead * l.step; r < a.ranges && r * a.range < lim; r += l.step) m = max(m, a.pmax[(at + r) * a.width + l.c]);
        atomicMax(&s_max[l.c], m);
    }
    __syncthreads();
    m = s_max[l.c];
    uint32_t s = 0;
    auto one = [&](int k, const int4& v) {
        uint32_t e[4];
        s += exps_of(a, p, lut, have, m, v, 4 * k, lim, holes, tab, p0, e);
        *reinterpret_cast<uint2*>(a.e + base + ((size_t)k * a.width + l.c) * 4) = make_uint2(e[0] | (e[1] << 16), e[2] | (e[3] << 16));
    };
    if (l.step) {
#pragma unroll
        for (int i = 0; i < kSumAhead; ++i)
            if (4 * group(i) < p.j1) one(group(i), z4[i]);
        for (int k = group(kSumAhead); 4 * k < p.j1; k += l.step) one(k, *reinterpret_cast<const int4*>(a.z + base + ((size_t)k * a.width + l.c) * 4));
        atomicAdd(&s_sum[l.c], s);
    }
    __syncthreads();
    if (tid < a.width) a.psum[(at + p.range) * a.width + tid] = s_sum[tid];
}

// S = 0: every key that is there has the same share (softmax.rs:42-48), the first ones a unit
// more.  base and extra of a row of lim keys; before: its keys in front of the range.
struct Uniform {
    uint32_t base, extra, before;
};
__device__ inline Uniform uniform_of(const PagedAttn& a, const Part& p, int lim) {
    const int32_t* t = a.tables + (size_t)p.seq * a.ldt;
    uint32_t n = 0, before = 0;
    for (int i = 0; i * (int)a.page.d < lim; ++i) {
        if (t[i] < 0 || t[i] >= a.n_pages) continue;
        const int first = i * (int)a.page.d;
        n += (uint32_t)min((int)a.page.d, lim - first);
        before += (uint32_t)min(max(p.j0 - first, 0), (int)a.page.d);
    }
    Uniform u{0, 0, before};
    if (n) udivmod32(1u << a.prob_frac, n, recip32(n), &u.base, &u.extra);
    return u;
}

// Groups of four keys a thread has on their way from the start.  us of a call with 4 / 6 / 8: 12 x 4 rows of
// 3001 keys 41.7 / 40.0 / 40.3, one row of 100000 58.9 / 57.9 / 57.9, 24 rows of 2500 36.3 / 36.3 / 36.6.
constexpr int kPvAhead = 6;

// p of the four keys from `key` on, from their e, as two pairs.
struct Probs {
    ProbDiv div;
    Uniform uni;
    uint32_t s;
    int lim;
    __device__ inline static Probs of(const PagedAttn& a, const Part& p, uint32_t s, int lim) {
        Probs r{ProbDiv::of(s ? s : 1u, a.prob_frac), Uniform{0, 0, 0}, s, lim};
        if (s == 0) r.uni = uniform_of(a, p, lim);
        return r;
    }
    __device__ inline uint2 operator()(const PagedAttn& a, const Part& p, int key, const uint2& e, bool holes, const uint64_t* tab, int p0) const {
        if (key >= p.j1) return make_uint2(0, 0);
        if (s) return make_uint2(div(e.x & 0xFFFFu) | (div(e.x >> 16) << 16), div(e.y & 0xFFFFu) | (div(e.y >> 16) << 16));
        uint32_t u[4];
        for (int i = 0; i < 4; ++i) {
            uint32_t rank = uni.before;
            bool ok = key + i < lim;
            if (holes) {
                ok = ok && on_page(a, tab, p0, min(key + i, p.j1 - 1));
                for (int b = p.j0; ok && b < key + i; ++b) rank += on_page(a, tab, p0, b) ? 1u : 0u;
            } else {
                rank += (uint32_t)(key + i - p.j0);
            }
            u[i] = ok ? uni.base + (rank < uni.extra ? 1u : 0u) : 0u;
        }
        return make_uint2(u[0] | (u[1] << 16), u[2] | (u[3] << 16));
    }
};

// The byte planes of a range's p, p = 256 ph + pl with pl the low byte as a signed one (p <= 2^14),
// in LDS: [16 keys][W vectors][16], first ph of the whole range, then pl.
template <int W>
__device__ inline void store_planes(int8_t* ph, int8_t* pl, int k, int c, const uint2& two) {
    const int at = (k >> 2) * 16 * W + 16 * c + 4 * (k & 3);
    *reinterpret_cast<uint32_t*>(pl + at) = __builtin_amdgcn_perm(two.y, two.x, 0x06040200u);
    // 128 carries into the high byte
    *reinterpret_cast<uint32_t*>(ph + at) = __builtin_amdgcn_perm(two.y + 0x00800080u, two.x + 0x00800080u, 0x07050301u);
}

// Units of 64 values in a ring of NB places in the block's LDS, each wave loading 64 / NW of them:
// key r of a unit is row r, its 16-byte chunk x at place x ^ turn(r), so that the transposing reads
// of 8 keys and the 16 bytes of one chunk meet different banks.
template <int HD, int NB, bool ALIGNED, int NW>
struct Units {
    static constexpr int CH = HD / 8, ROWS = 64 / CH, RW = 64 / NW, NI = RW / ROWS, kBytes = 64 * 2 * HD;
    const char* pages;
    int8_t* ring;
    uint32_t lane[NI];  // ALIGNED: the lane's bytes from the wave's first key
    int first, row, chunk;
    __device__ static inline int turn(int r) { return HD == 128 ? (r & 7) | (((r >> 4) & 1) << 3) : (r & 7) ^ ((r >> 4) & 1); }
    __device__ inline void begin(const PagedAttn& a, int8_t* lds) {
        pages = reinterpret_cast<const char*>(a.vp);
        ring = lds;
        const int l = threadIdx.x & 63;
        first = RW * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        row = l / CH;
        chunk = l % CH;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = i * ROWS + row;
            lane[i] = 2u * ((uint32_t)r * (uint32_t)a.pos_stride + 8u * (uint32_t)(chunk ^ turn(first + r)));
        }
    }
    // How many units of the keys [j0, j1) the wave has a part of.
    __device__ inline int count(const Part& p) const { return max(p.j1 - p.j0 - first + 63, 0) >> 6; }
    // The wave's part of unit u to place `slot`; keys from j1 on hold anything.
    __device__ inline void issue(const PagedAttn& a, const Part& p, const uint64_t* tab, int p0, int u, int slot) const {
        const int j = p.j0 + 64 * u + first;
        int8_t* to = ring + slot * kBytes + first * 2 * HD;
        if (ALIGNED) {
            const char* base = pages + 2 * uniform_u64(place_of(a, tab, p0, j));
            if (a.tiles.d == 1)
#pragma unroll
                for (int i = 0; i < NI; ++i)
                    __builtin_amdgcn_global_load_lds((global_void*)(uintptr_t)(base + lane[i]), (lds_void*)(to + i * 1024), 16, 0, kOnce);
            else
#pragma unroll
                for (int i = 0; i < NI; ++i)
                    __builtin_amdgcn_global_load_lds((global_void*)(uintptr_t)(base + lane[i]), (lds_void*)(to + i * 1024), 16, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = i * ROWS + row;
                const uint64_t from = place_of(a, tab, p0, min(j + r, p.j1 - 1)) + (uint64_t)(8 * (chunk ^ turn(first + r)));
                __builtin_amdgcn_global_load_lds((global_void*)(uintptr_t)(pages + 2 * from), (lds_void*)(to + i * 1024), 16, 0, 0);
            }
        }
    }
    // The oldest unit's part has landed when `left` (at most NB - 2) younger ones remain.
    __device__ static inline void wait(int left) {
        static_assert(NB >= 2 && NB <= 4, "the cases below");
        if (NB > 3 && left >= 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NI) : "memory");
        else if (NB > 2 && left >= 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NI) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
};

typedef int v2i32_t __attribute__((ext_vector_type(2)));
__device__ inline uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(lds_void*)p; }

// A unit's operands from LDS, there when it returns: the p planes (16 bytes each) and, for each of
// G chunks, 8 keys of a byte by two transposing reads, the second 8 rows further on.  In one
// statement with its wait: for reads of its own the compiler waits for every load to LDS in flight.
template <int HD, int G>
__device__ inline void read_unit(uint32_t ph, uint32_t pl, const uint32_t (&at)[G], v4i32_t& bh, v4i32_t& bl, v2i32_t (&v)[G][2]) {
    constexpr int kNext = 8 * 2 * HD;
    if constexpr (G == 1)
        asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b64_tr_b8 %2, %6\n\tds_read_b64_tr_b8 %3, %6 offset:%7\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(bh), "=&v"(bl), "=&v"(v[0][0]), "=&v"(v[0][1])
                     : "v"(ph), "v"(pl), "v"(at[0]), "n"(kNext)
                     : "memory");
    else if constexpr (G == 2)
        asm volatile("ds_read_b128 %0, %6\n\tds_read_b128 %1, %7\n\tds_read_b64_tr_b8 %2, %8\n\tds_read_b64_tr_b8 %3, %8 offset:%10\n\t"
                     "ds_read_b64_tr_b8 %4, %9\n\tds_read_b64_tr_b8 %5, %9 offset:%10\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(bh), "=&v"(bl), "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1])
                     : "v"(ph), "v"(pl), "v"(at[0]), "v"(at[1]), "n"(kNext)
                     : "memory");
    else {
        static_assert(G == 4, "chunks of a wave");
        asm volatile("ds_read_b128 %0, %10\n\tds_read_b128 %1, %11\n\tds_read_b64_tr_b8 %2, %12\n\tds_read_b64_tr_b8 %3, %12 offset:%16\n\t"
                     "ds_read_b64_tr_b8 %4, %13\n\tds_read_b64_tr_b8 %5, %13 offset:%16\n\tds_read_b64_tr_b8 %6, %14\n\t"
                     "ds_read_b64_tr_b8 %7, %14 offset:%16\n\tds_read_b64_tr_b8 %8, %15\n\tds_read_b64_tr_b8 %9, %15 offset:%16\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(bh), "=&v"(bl), "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1]), "=&v"(v[2][0]), "=&v"(v[2][1]), "=&v"(v[3][0]),
                       "=&v"(v[3][1])
                     : "v"(ph), "v"(pl), "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(kNext)
                     : "memory");
    }
}

// sum p_j v_j over a range, whose first NB - 1 units are on their way.  A wave takes 2 HD / NW bytes
// of every vector (whole chunks of 8 dimensions: its low and high bytes in turn) as rows of
// v_mfma_i32_16x16x64_i8, the p planes as columns, so with v = 256 vh + vl + 128
//   sum p v = 65536 (ph vh) + 256 (ph vl + pl vh) + pl vl + 128 sum p
// modulo 2^32, which holds the whole sum, from rows 2 d and 2 d + 1 that one lane has.  The transposing
// read gives a lane 8 keys of one byte of a chunk: no vector instruction goes on the layout but the
// low bytes' sign.  emit(vector, dimension, two sums), dimension even.
template <int HD, int W, int NB, bool ALIGNED, int NW, class Emit>
__device__ inline void paged_values(const PagedAttn& a, const Part& p, const uint64_t* tab, int p0, const Units<HD, NB, ALIGNED, NW>& units,
                                    const int8_t* ph, const int8_t* pl, const uint32_t* p_sum, const Emit& emit) {
    using U = Units<HD, NB, ALIGNED, NW>;
    constexpr int GROUPS = HD / 8 / NW;  // chunks of a wave
    const int lane = threadIdx.x & 63, c = lane & 15, kb = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v4i32_t ah[GROUPS], al[GROUPS];
    uint32_t at[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        ah[g] = al[g] = v4i32_t{0, 0, 0, 0};
        // in a group of 16 lanes lane 2 k + h gives bytes 8 h .. + 7 of key k (U::turn is key + 8's too)
        const int key = 16 * kb + (c >> 1), x = wave * GROUPS + g;
        at[g] = lds_addr(units.ring) + (uint32_t)(key * 2 * HD + ((x ^ U::turn(key)) << 4) + 8 * (c & 1));
    }
    const uint32_t p_at = (uint32_t)((kb * W + (c & (W - 1))) * 16), ph0 = lds_addr(ph) + p_at, pl0 = lds_addr(pl) + p_at;
    const int sign = c & 1 ? 0 : (int)0x80808080;  // low bytes are the even rows
    const int own = units.count(p), n = (p.j1 - p.j0 + 63) >> 6;
    int slot = 0;
    for (int u = 0; u < n; ++u) {
        if (u < own) U::wait(min(own - 1 - u, NB - 2));
        block_barrier();  // the unit is there; the one before it is done with
        if (u + NB - 1 < own) units.issue(a, p, tab, p0, u + NB - 1, slot == 0 ? NB - 1 : slot - 1);
        v4i32_t bh, bl;
        v2i32_t v[GROUPS][2];
        uint32_t now[GROUPS];
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) now[g] = at[g] + (uint32_t)(slot * U::kBytes);
        slot = slot + 1 == NB ? 0 : slot + 1;
        read_unit<HD, GROUPS>(ph0 + (uint32_t)(u * 64 * W), pl0 + (uint32_t)(u * 64 * W), now, bh, bl, v);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const v4i32_t x = {v[g][0][0] ^ sign, v[g][0][1] ^ sign, v[g][1][0] ^ sign, v[g][1][1] ^ sign};
            ah[g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, bh, ah[g], 0, 0, 0);
            al[g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, bl, al[g], 0, 0, 0);
        }
    }
    if (c >= a.width) return;
    const uint32_t add = 128u * p_sum[c];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        uint32_t y[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            y[i] = ((uint32_t)ah[g][2 * i + 1] << 16) + (((uint32_t)ah[g][2 * i] + (uint32_t)al[g][2 * i + 1]) << 8) + (uint32_t)al[g][2 * i] + add;
        emit(c, 8 * (wave * GROUPS + g) + 2 * kb, (int32_t)y[0], (int32_t)y[1]);
    }
}

// Two dimensions of a tile's vector v, rounded and clamped.
template <int HD>
__device__ inline void write_two(const PagedAttn& a, const Part& p, int v, int d, int32_t x, int32_t y) {
    if (v >= p.nv) return;
    int head;
    const int row = vector_of(a, p, v, head);
    const uint32_t lo = (uint32_t)(uint16_t)clamp_i16(rshift_round32(x, a.prob_frac)), hi = (uint32_t)(uint16_t)clamp_i16(rshift_round32(y, a.prob_frac));
    *reinterpret_cast<uint32_t*>(a.out + (size_t)row * a.ldo + (size_t)head * HD + d) = lo | (hi << 16);
}

constexpr int kPvRing = 3;
template <int HD, int W, bool ALIGNED>
__global__ __launch_bounds__(256, 4) void paged_pv_kernel(PagedAttn a) {
    using U = Units<HD, kPvRing, ALIGNED, 4>;
    constexpr int NB = kPvRing;
    extern __shared__ __align__(16) int8_t lds[];  // the ring, the range's p planes, its pages
    __shared__ uint32_t s_sum[16], p_sum[16];
    __shared__ int bad[4];
    static_assert(sizeof s_sum + sizeof p_sum + sizeof bad <= kPagedOwnLds, "allow_lds");
    int8_t* const ph = lds + NB * U::kBytes;
    int8_t* const pl = ph + a.range * W;
    uint64_t* const tab = reinterpret_cast<uint64_t*>(pl + a.range * W);
    Part p;
    if (!place_of_block(a, p)) return;
    // what needs no other load's result first: sums of ranges, exp values (within the workspace
    // whatever the lengths)
    const Lanes l = Lanes::of(a);
    const size_t at = (size_t)p.tile * a.ranges;
    const uint16_t* et = a.e + (size_t)p.tile * a.keys * a.width + 4 * l.c;
    auto exps = [&](int k) { return reinterpret_cast<const uint2*>(et + (size_t)min(p.j0 + 4 * k, a.keys - 4) * a.width); };
    uint2 e4[kPvAhead];
    uint32_t s4[kFoldAhead];
#pragma unroll
    for (int i = 0; i < kFoldAhead; ++i) s4[i] = a.psum[(at + min(l.k + i * l.step, a.ranges - 1)) * a.width + l.c];
#pragma unroll
    for (int i = 0; i < kPvAhead; ++i) e4[i] = *exps(l.k + i * l.step);
    const bool some = ends_of(a, p, threadIdx.x);
    if (!some) {
        if (a.ranges == 1)  // no key at all
            for (int i = threadIdx.x; i < p.nv * (HD / 2); i += 256) write_two<HD>(a, p, i / (HD / 2), 2 * (i % (HD / 2)), 0, 0);
        return;
    }
    const int tid = threadIdx.x;
    const int lim = lim_of(a, p, l.c);
    if (tid < 16) s_sum[tid] = p_sum[tid] = 0;
    const int p0 = pages_of_range(a, p, tab, bad);
    __syncthreads();
    U units;
    units.begin(a, lds);
#pragma unroll
    for (int u = 0; u < NB - 1; ++u)
        if (u < units.count(p)) units.issue(a, p, tab, p0, u, u);
    const bool holes = any_of(bad);
    uint32_t s = 0;
#pragma unroll
    for (int i = 0; i < kFoldAhead; ++i)
        if (l.k + i * l.step < a.ranges && (l.k + i * l.step) * a.range < lim) s += s4[i];
    if (l.step) {
        for (int r = l.k + kFoldAhead * l.step; r < a.ranges && r * a.range < lim; r += l.step) s += a.psum[(at + r) * a.width + l.c];
        if (s) atomicAdd(&s_sum[l.c], s);
    }
    block_barrier();
    if (l.step) {
        const Probs probs = Probs::of(a, p, s_sum[l.c], lim);
        const int groups = (p.j1 - p.j0 + 63) / 64 * 16;
        uint32_t sum = 0;
        auto one = [&](int k, const uint2& x) {
            const uint2 two = probs(a, p, p.j0 + 4 * k, x, holes, tab, p0);
            sum = (uint32_t)dot_pairs(two.x, 0x00010001u, dot_pairs(two.y, 0x00010001u, (int32_t)sum));
            store_planes<W>(ph, pl, k, l.c, two);
        };
#pragma unroll
        for (int i = 0; i < kPvAhead; ++i)
            if (l.k + i * l.step < groups) one(l.k + i * l.step, e4[i]);
        for (int k = l.k + kPvAhead * l.step; k < groups; k += l.step) one(k, *exps(k));
        atomicAdd(&p_sum[l.c], sum);
    }
    // the loop's first barrier stands between the planes and their use, p_sum's too
    int32_t* o = a.pout + (at + p.range) * a.width * HD;
    paged_values<HD, W, NB, ALIGNED, 4>(a, p, tab, p0, units, ph, pl, p_sum, [&](int v, int d, int32_t x, int32_t y) {
        if (a.ranges > 1) *reinterpret_cast<int2*>(o + v * HD + d) = make_int2(x, y);
        else write_two<HD>(a, p, v, d, x, y);
    });
}

// Few keys: a block per tile does all of it in one launch, the scores in LDS.
constexpr int kShortWaves = 8, kShortRing = 4;
template <int HD, int W, bool FAST, bool ALIGNED>
__global__ __launch_bounds__(64 * kShortWaves, 4) void paged_short_kernel(PagedAttn a) {
    constexpr int NB = kShortRing, NW = kShortWaves, kThreads = 64 * NW;
    using U = Units<HD, NB, ALIGNED, NW>;
    static_assert(NB * U::kBytes == NW * kQkRing * 32 * HD, "the values' ring lies where the keys' rings were");
    extern __shared__ __align__(16) int8_t lds[];  // the rings, scores, p planes, pages, the exp table
    __shared__ __align__(16) int8_t qlds[16 * 2 * HD];
    __shared__ int32_t red[16 * NW];
    __shared__ uint32_t s_sum[16], p_sum[16];
    __shared__ int bad[NW], large[NW];
    static_assert(sizeof qlds + sizeof red + sizeof s_sum + sizeof p_sum + sizeof bad + sizeof large <= kPagedOwnLds, "allow_lds");
    int32_t* const z = reinterpret_cast<int32_t*>(lds + NB * U::kBytes);  // [keys / 4][width][4]
    int8_t* const ph = reinterpret_cast<int8_t*>(z + (size_t)a.keys * a.width);
    int8_t* const pl = ph + a.keys * W;
    uint64_t* const tab = reinterpret_cast<uint64_t*>(pl + a.keys * W);
    uint16_t* const lut = reinterpret_cast<uint16_t*>(tab + a.entries);
    Part p;
    int lane_lim;
    if (!place_of_block(a, p)) return;
    const int tid = threadIdx.x;
    const uint32_t have = min(a.lut_len, kSumLut);
    TableCopy<kThreads> table;
    table.load(a, have);
    if (!ends_of(a, p, tid, lane_lim)) {
        for (int i = tid; i < p.nv * (HD / 2); i += kThreads) write_two<HD>(a, p, i / (HD / 2), 2 * (i % (HD / 2)), 0, 0);
        return;
    }
    const Lanes l = Lanes::of(a);
    const int lim = lim_of(a, p, l.c);
    stage_queries<HD>(a, p, qlds, large);
    const int p0 = pages_of_range(a, p, tab, bad);
    if (tid < 16) s_sum[tid] = p_sum[tid] = 0;
    table.store(a, have, lut);
    __syncthreads();
    const bool holes = any_of(bad);
    scores_of_range<HD, FAST, ALIGNED, NW, false>(a, p, lane_lim, tab, p0, holes, lds, qlds, any_of(large), z, red);
    block_barrier();  // the scores are there, the keys' rings free
    U units;
    units.begin(a, lds);
#pragma unroll
    for (int u = 0; u < NB - 1; ++u)  // on their way while the softmax runs
        if (u < units.count(p)) units.issue(a, p, tab, p0, u, u);
    int32_t m = red[l.c];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = max(m, red[16 * w + l.c]);
    const int groups = (p.j1 + 63) / 64 * 16;
    if (l.step) {
        uint32_t s = 0;
        for (int k = l.k; 4 * k < p.j1; k += l.step) {
            int4* const at = reinterpret_cast<int4*>(z + (size_t)(k * a.width + l.c) * 4);
            uint32_t e[4];
            s += exps_of(a, p, lut, have, m, *at, 4 * k, lim, holes, tab, p0, e);
            *reinterpret_cast<uint2*>(at) = make_uint2(e[0] | (e[1] << 16), e[2] | (e[3] << 16));
        }
        atomicAdd(&s_sum[l.c], s);
    }
    block_barrier();
    if (l.step) {
        const Probs probs = Probs::of(a, p, s_sum[l.c], lim);
        uint32_t sum = 0;
        for (int k = l.k; k < groups; k += l.step) {
            const uint2 two = probs(a, p, 4 * k, *reinterpret_cast<const uint2*>(z + (size_t)(k * a.width + l.c) * 4), holes, tab, p0);
            sum = (uint32_t)dot_pairs(two.x, 0x00010001u, dot_pairs(two.y, 0x00010001u, (int32_t)sum));
            store_planes<W>(ph, pl, k, l.c, two);
        }
        atomicAdd(&p_sum[l.c], sum);
    }
    // the loop's first barrier stands between the planes and their use, p_sum's too
    paged_values<HD, W, NB, ALIGNED, NW>(a, p, tab, p0, units, ph, pl, p_sum, [&](int v, int d, int32_t x, int32_t y) { write_two<HD>(a, p, v, d, x, y); });
}

// The ranges' sums, one rounding (attention.rs:84-86).  A block per row and head: four
// dimensions and every so-many-th range per thread.
template <int HD, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_out_kernel(PagedAttn a) {
    constexpr int Q = HD / 4, SHARES = THREADS / Q;
    __shared__ int64_t part[SHARES][HD];
    int head, h, in_seq, v;
    const int row = divmod(a.heads_d, (int)blockIdx.x, head), q = threadIdx.x % Q, share = threadIdx.x / Q;
    const int seq = divmod(a.n, row, in_seq), g = divmod(a.G, head, h);
    const int tile = divmod(a.width_d, in_seq * (int)a.G.d + h, v), lim = keys_of(a, row);
    const size_t at = (((size_t)seq * a.kvh.d + g) * a.tiles.d + tile) * a.ranges;
    int64_t s[4] = {0, 0, 0, 0};
    int rem;
    const int last = min(a.ranges, divmod(a.range_d, lim + a.range - 1, rem));
    for (int r0 = share; r0 < last; r0 += 8 * SHARES) {
        int4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            x[k] = r0 + k * SHARES < last ? *reinterpret_cast<const int4*>(a.pout + ((at + r0 + k * SHARES) * a.width + v) * HD + 4 * q) : make_int4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            s[0] += x[k].x;
            s[1] += x[k].y;
            s[2] += x[k].z;
            s[3] += x[k].w;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) part[share][4 * q + k] = s[k];
    __syncthreads();
    if (threadIdx.x < HD) {
        int64_t y = 0;
#pragma unroll
        for (int k = 0; k < SHARES; ++k) y += part[k][threadIdx.x];
        a.out[(size_t)row * a.ldo + (size_t)head * HD + threadIdx.x] = clamp_i16_i64(rshift_round64(y, a.prob_frac));
    }
}

constexpr size_t kAlignedStride = (size_t)1 << 26;  // 15 of them and a vector are 32 bits of bytes

// A launch with more LDS than the 64 KiB it has by default, the kernel's own included.  The attribute
// is the process's, so every call sets the same: another thread's launch may lie behind this one.
template <class K>
hipError_t allow_lds(K kernel, size_t bytes) {
    return bytes + kPagedOwnLds <= 65536 ? hipSuccess
                                         : hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)(kPagedLds - kPagedOwnLds));
}

template <int HD, bool ALIGNED, int W>
hipError_t paged_in_one(const PagedAttn& a, const PagedPlan& pl, hipStream_t st) {
    const size_t bytes = paged_short_lds(pl, HD, (int)a.page.d, a.lut_len);
    auto kernel = a.scale.fast ? paged_short_kernel<HD, W, true, ALIGNED> : paged_short_kernel<HD, W, false, ALIGNED>;
    const hipError_t e = allow_lds(kernel, bytes);
    if (e != hipSuccess) return e;
    kernel<<<(unsigned)pl.blocks, 64 * kShortWaves, bytes, st>>>(a);
    return hipGetLastError();
}

template <int HD, bool ALIGNED>
hipError_t paged_ranges(const PagedAttn& a, const PagedPlan& pl, hipStream_t st) {
    const int W = a.width <= 8 ? 8 : 16;
    if (pl.in_one) return W == 8 ? paged_in_one<HD, ALIGNED, 8>(a, pl, st) : paged_in_one<HD, ALIGNED, 16>(a, pl, st);
    const unsigned grid = (unsigned)pl.blocks;
    const size_t tab = (size_t)a.entries * 8;
    const size_t qk = 4 * kQkRing * 32 * HD + tab;
    static_assert(4 * kQkRing * 32 * HD + paged_table_entries(kPagedMaxRange, 1) * 8 + kPagedOwnLds <= 65536, "rings, pages and its own");
    auto scores = a.scale.fast ? paged_qk_kernel<HD, true, ALIGNED> : paged_qk_kernel<HD, false, ALIGNED>;
    scores<<<grid, 256, qk, st>>>(a);
    paged_sum_kernel<<<grid, 256, tab, st>>>(a);
    const size_t pv = kPvRing * 64 * 2 * HD + (size_t)a.range * W * 2 + tab;
    auto values = W == 8 ? paged_pv_kernel<HD, 8, ALIGNED> : paged_pv_kernel<HD, 16, ALIGNED>;
    const hipError_t e = allow_lds(values, pv);
    if (e != hipSuccess) return e;
    values<<<grid, 256, pv, st>>>(a);
    return hipGetLastError();
}

template <int HD>
hipError_t paged_launch(const PagedAttn& a, const PagedPlan& pl, int rows, hipStream_t st) {
    if (pl.ranges) {
        const hipError_t e = a.page.d % 16 == 0 && a.pos_stride <= kAlignedStride ? paged_ranges<HD, true>(a, pl, st) : paged_ranges<HD, false>(a, pl, st);
        if (e != hipSuccess) return e;
    }
    if (pl.ranges > 32) paged_out_kernel<HD, 1024><<<(unsigned)(rows * a.heads), 1024, 0, st>>>(a);
    else if (pl.ranges != 1) paged_out_kernel<HD, 256><<<(unsigned)(rows * a.heads), 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace
}  // namespace myl

using namespace myl;

extern "C" {

size_t myl_attention_paged_workspace(const myl_ctx* ctx, size_t n_seqs, size_t rows_per_seq, size_t heads, size_t kv_heads,
                                     size_t head_dim, size_t max_len) {
    const PagedShape s{n_seqs, rows_per_seq, heads, kv_heads, head_dim, max_len};
    if (!ctx || paged_refuse(s) || (head_dim != 64 && head_dim != 128)) return 0;
    return paged_plan(s, ctx->prop.multiProcessorCount).bytes;
}

int myl_attention_paged_dev(myl_ctx* ctx, const int16_t* q, size_t n_seqs, size_t rows_per_seq, size_t ldq, size_t heads,
                            size_t kv_heads, size_t head_dim, const int16_t* k_pages, const int16_t* v_pages, size_t n_pages,
                            size_t page_size, size_t page_stride, size_t head_stride, size_t pos_stride, const int32_t* tables,
                            size_t table_len, size_t table_stride, const int32_t* lens, size_t max_len, int64_t score_mult,
                            uint8_t score_shift, const int16_t* exp_lut, size_t lut_len, uint8_t lut_shift, uint8_t prob_frac,
                            int16_t* out, size_t ldo, void* workspace, size_t workspace_bytes) {
    if (!ctx) return MYL_E_INVALID;
    const char* what = "attention_paged_dev";
    auto bad = [&](const char* why) { return ctx->fail(MYL_E_INVALID, std::string(what) + ": " + why); };
    if (head_dim != 64 && head_dim != 128) return ctx->fail(MYL_E_UNSUPPORTED, std::string(what) + ": head_dim 64 or 128");
    const PagedShape s{n_seqs, rows_per_seq, heads, kv_heads, head_dim, max_len};
    if (const char* why = paged_refuse(s)) return bad(why);
    if (const char* why = pages_refuse({n_pages, page_size, page_stride, head_stride, pos_stride, n_seqs, table_len, table_stride, kv_heads, head_dim}))
        return bad(why);
    if (max_len > table_len * page_size) return bad("max_len is at most table_len pages");
    if (ldq < heads * head_dim || ldo < heads * head_dim) return bad("leading dimension too small");
    if (lut_len == 0 || lut_len > kPagedMaxLut) return bad("the exp table must hold 1 to 32768 entries");
    if (prob_frac > 14) return bad("prob_frac is at most 14");
    if (n_seqs == 0 || rows_per_seq == 0) return MYL_OK;
    if (!q || !out || !exp_lut || !lens || !k_pages || !v_pages || (max_len && !tables)) return bad("null operand");
    const uintptr_t ptrs = (uintptr_t)q | (uintptr_t)out | (uintptr_t)exp_lut | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)workspace;
    if ((ptrs & 15) || ((ldq | ldo | page_stride | head_stride | pos_stride) & 7))
        return bad("operands must be 16-byte aligned, strides multiples of 8");
    const PagedPlan pl = paged_plan(s, ctx->prop.multiProcessorCount);
    if (!workspace || workspace_bytes < pl.bytes) return bad("workspace too small (myl_attention_paged_workspace)");
    const DeviceGuard guard(ctx->device);
    char* ws = static_cast<char*>(workspace);
    PagedAttn a{};
    a.q = q; a.kp = k_pages; a.vp = v_pages; a.tables = tables; a.lens = lens; a.lut = exp_lut; a.out = out;
    a.z = reinterpret_cast<int32_t*>(ws + pl.off_z);
    a.e = reinterpret_cast<uint16_t*>(ws + pl.off_e);
    a.pmax = reinterpret_cast<int32_t*>(ws + pl.off_max);
    a.psum = reinterpret_cast<uint32_t*>(ws + pl.off_sum);
    a.holes = reinterpret_cast<int32_t*>(ws + pl.off_holes);
    a.pout = reinterpret_cast<int32_t*>(ws + pl.off_out);
    a.ldq = ldq; a.ldo = ldo; a.ldt = table_stride; a.page_stride = page_stride; a.head_stride = head_stride; a.pos_stride = pos_stride;
    a.mult = score_mult;
    a.scale = ScoreScale::of(score_mult, score_shift, (int)head_dim);
    auto div = [](size_t d) { return SmallDiv::of(std::max<size_t>(d, 1)); };
    a.n = div(rows_per_seq); a.G = div(heads / kv_heads); a.page = div(page_size); a.kvh = div(kv_heads);
    a.tiles = div((size_t)pl.tiles); a.ranges_d = div((size_t)pl.ranges); a.width_d = div((size_t)pl.width); a.heads_d = div(heads);
    a.range_d = div((size_t)pl.range); a.entries = pl.ranges ? paged_table_entries(pl.range, (int)page_size) : 0;
    a.heads = (int)heads; a.max_len = (int)max_len; a.n_pages = (int)n_pages; a.keys = pl.keys;
    a.range = pl.range; a.ranges = pl.ranges; a.width = pl.width; a.vectors = (int)(rows_per_seq * (heads / kv_heads));
    a.places = (int)(n_seqs * kv_heads * (size_t)pl.ranges);
    a.lut_len = (uint32_t)lut_len; a.shift = score_shift; a.lut_shift = lut_shift; a.prob_frac = prob_frac;
    const int rows = (int)(n_seqs * rows_per_seq);
    return ctx->hip(head_dim == 128 ? paged_launch<128>(a, pl, rows, ctx->stream) : paged_launch<64>(a, pl, rows, ctx->stream), what);
}

}  // extern "C"
