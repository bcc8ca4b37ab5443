// prefix_attn.hip -- integer attention (attention.rs:42-90 with
// softmax.rs:12-64) of a batch whose sequences share a prefix of K/V rows and
// continue with their own tails: myl_attention_prefix_dev.
//
// A probability p_j = RNE(e_j 2^f / S) needs the exact maximum and exp sum of
// its whole row before it is rounded, so a row cannot be finished in one pass
// with a running maximum; four launches follow one another:
//   prefix_qk_kernel<MAX>  the maximum score of each vector (query head of a
//                          row) over each range of keys
//   prefix_qk_kernel<EXP>  the scores once more, e_j = exp_lut[(max - z_j) >> lut_shift]
//                          as 16 bits, and the ranges' sums of them
//   prefix_pv_kernel       p_j from e_j and S, sum p_j v_j over each range
//   prefix_out_kernel      the sums over the ranges, rounded and clamped
// With few keys one launch does it all (prefix_short_kernel).
// The prefix is read once for 64 vectors of any rows: their tiles and the
// tails' tiles (vectors of one sequence) run side by side in every launch.
#include "abi_internal.h"
#include "attn_fixed.h"
#include "bufload.h"
#include "gemm_mfma.h"
#include "ops.h"
#include "qk_planes.h"
#include "serve_plan.h"
#include "wave.h"

#include <algorithm>
#include <string>
#include <type_traits>

namespace myl {
namespace {

constexpr int kShortThreads = 512;
constexpr int kQkTile = kPrefixQkTile, kPvTile = kPrefixPvTile;  // vectors of a block

// The call, as every kernel sees it.  Row r = seq * rows_per_seq + i attends
// keys 0 .. P-1 of the prefix, then the first lens[r] of its sequence's tail.
struct PrefixAttn {
    const int16_t *q, *kp, *vp, *kt, *vt;
    const int32_t *slots, *lens;
    const int16_t* lut;
    int16_t* out;
    int32_t *pmax, *psum, *pout;  // [range][pair], [range][pair], [range][pair][hd]; pair = row * heads + head
    uint16_t *pexp, *texp;        // exp values of the prefix's and the tails' keys (exp_tile)
    size_t ldq, ldo, ph, ts, th;  // strides in elements: q/out rows, prefix heads, tail slots, tail heads
    int64_t mult;
    ScoreScale scale;
    SmallDiv n, G, np, nt, kvh;
    struct Cut {
        SmallDiv tp, tt;  // tiles of the prefix's and of a sequence's vectors
        int blocks_p;
    } qk, pv;
    int short_cap;                // keys that a block of prefix_short_kernel has room for
    int R, heads, P, max_tail, n_slots, vp_count, vt_count, np_count, nt_count, rp, rt, vp16, vt16, pgroups, tgroups;
    uint32_t pairs, lut_len;
    uint8_t shift, lut_shift, prob_frac;
};

// The slot of sequence s, or -1; tail positions of row r (-1: left out).
__device__ inline int slot_of(const PrefixAttn& a, int s) {
    const int slot = a.slots ? a.slots[s] : s;
    return slot < 0 || slot >= a.n_slots ? -1 : slot;
}
__device__ inline int tail_of(const PrefixAttn& a, int r, int slot) {
    const int len = a.lens[r];
    return len < 0 ? -1 : (slot < 0 ? 0 : min(len, a.max_tail));
}

// A block's part of the work.
struct Part {
    bool tail;
    int g, v0, nv;         // KV head; first vector, vectors
    int row0;              // row of vector 0 (of the batch or the sequence)
    int range, j0, j1;     // range index among all, keys [j0, j1) of the prefix or the tail
    int seq, slot;
    int subs;              // 16-vector tiles with a vector
};
// False: nothing to do.  Prefix blocks of one range follow one another on one XCD
// (block b runs on XCD b % 8), so its L2 serves the range's K and V to all tiles.
template <int TILE>
__device__ inline bool part_of(const PrefixAttn& a, const PrefixAttn::Cut& cut, Part& p) {
    const int b = blockIdx.x;
    p.tail = b >= cut.blocks_p;
    if (!p.tail) {
        const int t = (b & 7) * (cut.blocks_p >> 3) + (b >> 3);
        int tile, rng;
        const int q = divmod(cut.tp, t, tile);
        p.g = divmod(a.np, q, rng);
        if (p.g >= (int)a.kvh.d) return false;
        p.range = rng;
        p.j0 = rng * a.rp;
        p.j1 = min(a.P, p.j0 + a.rp);
        p.v0 = tile * TILE;
        p.nv = min(TILE, a.vp_count - p.v0);
        p.row0 = 0;
        p.seq = p.slot = 0;
    } else {
        int tile, rng;
        int q = divmod(cut.tt, b - cut.blocks_p, tile);
        q = divmod(a.nt, q, rng);
        const int s = divmod(a.kvh, q, p.g);
        p.range = a.np_count + rng;
        p.j0 = rng * a.rt;
        p.j1 = min(a.max_tail, p.j0 + a.rt);
        p.v0 = tile * TILE;
        p.nv = min(TILE, a.vt_count - p.v0);
        p.seq = s;
        p.row0 = s * (int)a.n.d;
        p.slot = __builtin_amdgcn_readfirstlane(slot_of(a, s));
        if (p.slot < 0) return false;
    }
    p.subs = (p.nv + 15) >> 4;
    return true;
}

// The exp values lie as the matrix instructions leave them, so that a wave stores (and
// 16 lanes load) whole lines: [16 vectors][16 keys] blocks of four keys of a vector per
// lane, entry 64 (key / 4) + 4 vector + key % 4, a vector tile's key groups in a row.
__device__ inline uint16_t* exp_tile(const PrefixAttn& a, const Part& p, int t) {
    const size_t tile = (size_t)(p.v0 >> 4) + (size_t)t;
    if (!p.tail) return a.pexp + ((size_t)p.g * (size_t)a.vp16 + tile) * (size_t)a.pgroups * 256;
    return a.texp + (((size_t)p.seq * a.kvh.d + (size_t)p.g) * (size_t)a.vt16 + tile) * (size_t)a.tgroups * 256;
}

// The vectors of a tile, worked out once per block: places past the last vector repeat it.
template <int TILE>
struct Vectors {
    size_t q[TILE];      // element offset of the query vector
    uint32_t pair[TILE];
    int32_t lim[TILE];   // keys of this part (the prefix, or the sequence's tail) that it attends
    int32_t tail[TILE];  // TAILS: tail positions of its row, -1: left out
};
template <int TILE, bool TAILS>
__device__ inline void vectors_of(const PrefixAttn& a, const Part& p, int hd, Vectors<TILE>& vs) {
    const int v = threadIdx.x;
    if (v < TILE) {
        int h, rem;
        const int row = p.row0 + divmod(a.G, p.v0 + min(v, p.nv - 1), h), head = p.g * (int)a.G.d + h;
        vs.q[v] = (size_t)row * a.ldq + (size_t)(head * hd);
        vs.pair[v] = (uint32_t)row * (uint32_t)a.heads + (uint32_t)head;
        int tail = 0;
        if (p.tail) tail = tail_of(a, row, p.slot);
        else if (TAILS && a.nt_count) tail = tail_of(a, row, slot_of(a, divmod(a.n, row, rem)));
        vs.lim[v] = p.tail ? max(tail, 0) : a.P;
        vs.tail[v] = tail;
    }
}

__device__ inline const int16_t* keys_of(const PrefixAttn& a, const Part& p, const int16_t* prefix, const int16_t* tail) {
    return uniform_ptr(p.tail ? tail + (size_t)p.slot * a.ts + (size_t)p.g * a.th : prefix + (size_t)p.g * a.ph);
}

__device__ inline int32_t dot_pairs(uint32_t w, uint32_t x, int32_t acc) {
    typedef short __attribute__((ext_vector_type(2))) s2;
    return __builtin_amdgcn_sdot2(__builtin_bit_cast(s2, w), __builtin_bit_cast(s2, x), acc, false);
}
__device__ inline int32_t sum_pairs(uint32_t w, int32_t acc) { return dot_pairs(w, 0x00010001u, acc); }
// 8 int16 as their byte planes x = 256 hi + lo' + 128.
__device__ inline void planes8(const uint4& x, uint32_t* h, uint32_t* l) {
    h[0] = __builtin_amdgcn_perm(x.y, x.x, 0x07050301u);
    h[1] = __builtin_amdgcn_perm(x.w, x.z, 0x07050301u);
    l[0] = __builtin_amdgcn_perm(x.y, x.x, 0x06040200u) ^ 0x80808080u;
    l[1] = __builtin_amdgcn_perm(x.w, x.z, 0x06040200u) ^ 0x80808080u;
}
// 16 dimensions (two 16-byte loads) as matrix operands.
__device__ inline void planes16(const uint4 (&x)[2], v4i32_t& h, v4i32_t& l) {
    uint32_t hw[4], lw[4];
    planes8(x[0], hw, lw);
    planes8(x[1], hw + 2, lw + 2);
    h = v4i32_t{(int)hw[0], (int)hw[1], (int)hw[2], (int)hw[3]};
    l = v4i32_t{(int)lw[0], (int)lw[1], (int)lw[2], (int)lw[3]};
}

__device__ inline void block_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Over the four 16-lane rows of a wave.
__device__ inline int32_t quarters_sum(int32_t v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
__device__ inline int32_t quarters_max(int32_t v) {
    v = max(v, __shfl_xor(v, 16, 64));
    return max(v, __shfl_xor(v, 32, 64));
}

// A thread's share of a vector's partials over its ranges (all of the prefix's, its
// tail's up to `tail` positions, which follow them), SHARES threads per vector: eight
// loads in flight.
template <int SHARES, class Fold>
__device__ inline void fold_ranges(const PrefixAttn& a, const int32_t* __restrict__ part, uint32_t pair, int tail, int share,
                                   const Fold& fold) {
    const int all = a.np_count + a.nt_count;
    for (int i0 = share; i0 < all; i0 += 8 * SHARES) {
        int32_t x[8];
        bool ok[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = i0 + k * SHARES;
            ok[k] = i < all && (i < a.np_count || (i - a.np_count) * a.rt < tail);
            x[k] = ok[k] ? part[(size_t)i * a.pairs + pair] : 0;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (ok[k]) fold(x[k]);
    }
}

enum Pass { kMaxPass, kExpPass };

// The exp table's copy in LDS, eight entries per load: entries past the table are 0 (one at
// least follows it), negative ones count as 0.  An odd last entry is loaded by itself: the
// words' loads return 0 from it on.
struct TablePiece {
    uint4 x[4];
    uint32_t last;
    __device__ inline void load(const PrefixAttn& a, uint32_t i0) {
        const __amdgpu_buffer_rsrc_t rl = weight_rsrc(a.lut, prefix_table_bytes(a.lut_len));
        last = (uint16_t)a.lut[a.lut_len - 1u];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = cload16(rl, 2u * (i0 + 2048u * k));
    }
    __device__ inline void store(const PrefixAttn& a, uint32_t i0, uint16_t* tab) const {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t i = i0 + 2048u * k;
            if (i > a.lut_len) break;
            uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                if (i + 2 * b + 1 == a.lut_len) w[b] = last;
                const uint32_t lo = i + 2 * b < a.lut_len && !(w[b] & 0x8000u) ? w[b] & 0xFFFFu : 0u;
                const uint32_t hi = i + 2 * b + 1 < a.lut_len && !(w[b] >> 31) ? w[b] & 0xFFFF0000u : 0u;
                w[b] = lo | hi;
            }
            *reinterpret_cast<uint4*>(tab + i) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
};

// Scores of a tile's vectors with a range's keys on v_mfma_i32_16x16x64_i8: K
// positions are rows, vectors columns, so lane l holds vector l % 16 of each 16-vector
// tile and positions 4 (l / 16) .. + 3 of a 16-position group.  With byte
// planes x = 256 hi + lo' + 128 of both operands
//   q.k = 65536 hh + 256 (hl + lh + 128 sum k_hi) + ll + 128 sum k_lo' + 128 sum q
// where the sums over k come from the matrix cores too (a B operand of 64s, doubled)
// and start the accumulators, and sum q is one value per lane.  As 256 u + r the score
// takes 32-bit steps (ScoreScale); other scales take the 64-bit form (FAST false).
// A wave holds the vectors' planes in registers and streams its groups of K rows, the
// next step's loads in flight; no barrier in the loop.  Bound by issue (each instruction takes
// about four cycles beside the matrix instructions): 64 rows of 28 heads by 30000 keys of
// 128 take 45 us for the maxima (1.2 POP/s) and 73 for the exp values, whose table lookup and
// store come on top.  Tiles of 32 vectors took 1.5 times as long, two steps of K in flight or
// operands read a step ahead as long or longer (236 registers; spills).
// SUBS 16-vector tiles, GU 16-position groups per wave and step.
constexpr int qk_groups(int subs) { return subs == 1 ? 2 : 1; }
template <int HD, bool FAST, Pass PASS, int SUBS>
__device__ inline void prefix_qk_part(const PrefixAttn& a, const Part& p, Vectors<kQkTile>& vs, uint16_t* tab, int8_t* klds,
                                      int32_t (*red)[kQkTile], int32_t* s_max) {
    constexpr int NS = HD / 64, GU = qk_groups(SUBS), CH = HD / 8, NI = CH / 4;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, kb = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int16_t* kg = keys_of(a, p, a.kp, a.kt);
    const __amdgpu_buffer_rsrc_t rk = weight_rsrc(kg, (uint32_t)(p.tail ? a.max_tail : a.P) * HD * 2u);
    // K rows come in whole lines (CH lanes of 16 bytes a row) and reach the operands' lanes
    // through the wave's own LDS, chunk x of row r at x ^ (r % CH): in order within a
    // wave, so without a barrier.  (Loaded straight to the operands, 16 rows per
    // instruction, they cost a cache access per lane: 1.6 times as long.)
    const int krow = lane / CH, kch = lane % CH;
    const uint32_t klane = (uint32_t)krow * HD + 8u * kch;
    int8_t* const kl_w = klds + wave * GU * 32 * HD;
    uint4 kx[GU][NI];
    auto load = [&](int j) {
#pragma unroll
        for (int g = 0; g < GU; ++g)
#pragma unroll
            for (int i = 0; i < NI; ++i) kx[g][i] = cload16(rk, ((uint32_t)(j + 64 * g + i * (64 / CH)) * HD + klane) * 2u);
    };
    int j = p.j0 + 16 * wave;
    load(j);
    TablePiece piece;
    if (PASS == kExpPass) piece.load(a, 8 * tid);
    vectors_of<kQkTile, PASS == kExpPass>(a, p, HD, vs);
    block_barrier();
    uint16_t* eo[SUBS];
    int lim[SUBS];  // keys of this range that the vector attends end here
    int lmax = 0, lmin = 0x7FFFFFFF;
    // the vectors once per block, in whole lines, into the K rows' place
    constexpr int QI = (16 * SUBS * CH + 255) / 256;
    uint4 qs[QI];
#pragma unroll
    for (int i = 0; i < QI; ++i) {
        const int v = (tid + 256 * i) / CH;
        qs[i] = *reinterpret_cast<const uint4*>(a.q + vs.q[min(v, kQkTile - 1)] + 8 * (tid % CH));
    }
#pragma unroll
    for (int t = 0; t < SUBS; ++t) {
        // tiles past the last one repeat it: the same values to the same addresses
        const int tile = min(t, p.subs - 1), v = 16 * tile + c;
        lim[t] = vs.lim[v];
        lmax = max(lmax, lim[t]);
        lmin = min(lmin, lim[t]);
        eo[t] = exp_tile(a, p, tile) + 4 * lane;
    }
    lmax = wave_max_i32(lmax);
    lmin = min(p.j1, ~wave_max_i32(~lmin));
    const int j1 = min(p.j1, lmax);  // uniform over the block: every wave holds every vector
    if (p.j0 >= j1) return;
    int32_t mx = INT32_MIN;
    if (PASS == kExpPass) {
        // the maxima over all ranges
        const int v = tid & (kQkTile - 1), share = tid / kQkTile;
        fold_ranges<256 / kQkTile>(a, a.pmax, vs.pair[v], vs.tail[v], share, [&](int32_t x) { mx = max(mx, x); });
        red[share][v] = mx;
        piece.store(a, 8 * tid, tab);
        for (uint32_t i0 = 8 * tid + 8192; i0 <= a.lut_len; i0 += 8192) {
            piece.load(a, i0);
            piece.store(a, i0, tab);
        }
    }
#pragma unroll
    for (int i = 0; i < QI; ++i) {
        const int v = (tid + 256 * i) / CH;
        if (v < 16 * SUBS) *reinterpret_cast<uint4*>(klds + v * 2 * HD + (((tid % CH) ^ (v & (CH - 1))) << 4)) = qs[i];
    }
    block_barrier();
    v4i32_t qh[SUBS][NS], ql[SUBS][NS];
    int32_t qsum[SUBS], m[SUBS];
#pragma unroll
    for (int t = 0; t < SUBS; ++t) {
        qsum[t] = 0;
        const int v = 16 * min(t, p.subs - 1) + c;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            uint4 x[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                x[i] = *reinterpret_cast<const uint4*>(klds + v * 2 * HD + (((8 * s + 2 * kb + i) ^ (c & (CH - 1))) << 4));
            planes16(x, qh[t][s], ql[t][s]);
            const uint32_t w[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
#pragma unroll
            for (int i = 0; i < 8; ++i) qsum[t] = sum_pairs(w[i], qsum[t]);
        }
        qsum[t] = 128 * quarters_sum(qsum[t]);
    }
    if (PASS == kExpPass) {
        if (tid < kQkTile) {
            int32_t v = red[0][tid];
#pragma unroll
            for (int i = 1; i < 256 / kQkTile; ++i) v = max(v, red[i][tid]);
            s_max[tid] = v;
        }
    }
    block_barrier();  // the vectors are read, the table is complete
    if (PASS == kExpPass) {
#pragma unroll
        for (int t = 0; t < SUBS; ++t) m[t] = s_max[16 * min(t, p.subs - 1) + c];
    }
    // kMaxPass: the largest dot as u * 2^32 + r (FAST), or the largest score; kExpPass: the sum
    int64_t top[SUBS];
    int32_t best[SUBS];
#pragma unroll
    for (int t = 0; t < SUBS; ++t) {
        top[t] = INT64_MIN;
        best[t] = PASS == kMaxPass ? INT32_MIN : 0;
    }
    const v4i32_t sixty4 = {0x40404040, 0x40404040, 0x40404040, 0x40404040}, zero = {0, 0, 0, 0};
    // MASK: the step holds keys past some vector's (or the range's) end
    auto step = [&](auto mask) {
        constexpr bool MASK = decltype(mask)::value;
        v4i32_t kh[GU][NS], kl[GU][NS];
#pragma unroll
        for (int g = 0; g < GU; ++g)
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int row = i * (64 / CH) + krow;
                *reinterpret_cast<uint4*>(kl_w + g * 32 * HD + row * 2 * HD + ((kch ^ (row & (CH - 1))) << 4)) = kx[g][i];
            }
        load(j + 64 * GU);
#pragma unroll
        for (int g = 0; g < GU; ++g)
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                uint4 x[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    x[i] = *reinterpret_cast<const uint4*>(kl_w + g * 32 * HD + c * 2 * HD + (((8 * s + 2 * kb + i) ^ (c & (CH - 1))) << 4));
                planes16(x, kh[g][s], kl[g][s]);
            }
#pragma unroll
        for (int g = 0; g < GU; ++g) {
            const int jg = j + 64 * g;
            v4i32_t mid0 = zero, ll0 = zero;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                mid0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kh[g][s], sixty4, mid0, 0, 0, 0);
                ll0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kl[g][s], sixty4, ll0, 0, 0, 0);
            }
            mid0 += mid0;
            ll0 += ll0;
#pragma unroll
            for (int t = 0; t < SUBS; ++t) {
                v4i32_t hh = zero, mid = mid0, ll = ll0;
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    hh = __builtin_amdgcn_mfma_i32_16x16x64_i8(kh[g][s], qh[t][s], hh, 0, 0, 0);
                    mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(kh[g][s], ql[t][s], mid, 0, 0, 0);
                    mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(kl[g][s], qh[t][s], mid, 0, 0, 0);
                    ll = __builtin_amdgcn_mfma_i32_16x16x64_i8(kl[g][s], ql[t][s], ll, 0, 0, 0);
                }
                uint32_t ev[4];
                int64_t key[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int32_t lo = ll[i] + qsum[t];
                    const int32_t u = 256 * hh[i] + mid[i] + (lo >> 8);
                    const uint32_t r = (uint32_t)lo & 255u;
                    const bool ok = !MASK || jg + 4 * kb + i < min(lim[t], j1);
                    if (PASS == kMaxPass) {
                        if (FAST) {
                            key[i] = (int64_t)(((uint64_t)(uint32_t)(ok ? u : INT32_MIN) << 32) | r);
                        } else {
                            const int64_t dot = 256 * (int64_t)u + (int64_t)r;
                            const int32_t z = (int32_t)rshift_round64(wmul64(dot, a.mult), a.shift);
                            best[t] = ok ? max(best[t], z) : best[t];
                        }
                    } else {
                        // sat_sub and the lookup of softmax.rs:12-38; the table ends with a 0.
                        // FAST: a saturated difference is past the table as it is.
                        const int32_t z = FAST ? a.scale(u, r)
                                               : (int32_t)rshift_round64(wmul64(256 * (int64_t)u + (int64_t)r, a.mult), a.shift);
                        const uint32_t diff = (uint32_t)m[t] - (uint32_t)z;
                        const uint32_t below = FAST ? diff : min(diff, 0x7FFFFFFFu);
                        const uint32_t e = tab[min(below >> (a.lut_shift & 31u), a.lut_len)];
                        ev[i] = ok ? e : 0u;
                        best[t] += (int32_t)ev[i];
                    }
                }
                if (PASS == kMaxPass && FAST) top[t] = max(top[t], max(max(key[0], key[1]), max(key[2], key[3])));
                if (PASS == kExpPass && (!MASK || jg < j1))
                    *reinterpret_cast<uint2*>(eo[t] + 16 * jg) = make_uint2(ev[0] | (ev[1] << 16), ev[2] | (ev[3] << 16));
            }
        }
    };
    for (; j + 64 * (GU - 1) + 16 <= lmin; j += 64 * GU) step(std::false_type{});
    for (; j < j1; j += 64 * GU) step(std::true_type{});
    // the block's value per vector
    block_barrier();
#pragma unroll
    for (int t = 0; t < SUBS; ++t) {
        int32_t v = best[t];
        if (PASS == kMaxPass) {
            if (FAST) v = (int32_t)(top[t] >> 32) == INT32_MIN ? INT32_MIN : a.scale((int32_t)(top[t] >> 32), (uint32_t)top[t]);
            v = quarters_max(v);
        } else {
            v = quarters_sum(v);
        }
        if (kb == 0) red[wave][16 * t + c] = v;
    }
    block_barrier();
    if (tid < p.nv) {
        const size_t o = (size_t)p.range * a.pairs + vs.pair[tid];
        const int32_t r0 = red[0][tid], r1 = red[1][tid], r2 = red[2][tid], r3 = red[3][tid];
        if (PASS == kMaxPass) a.pmax[o] = max(max(r0, r1), max(r2, r3));
        else a.psum[o] = r0 + r1 + r2 + r3;
    }
}

template <int HD, bool FAST, Pass PASS>
__global__ __launch_bounds__(256, 3) void prefix_qk_kernel(PrefixAttn a) {
    extern __shared__ __align__(16) uint16_t tab[];  // kExpPass: the table and a 0
    __shared__ __align__(16) int8_t klds[4 * qk_groups(1) * 32 * HD];
    __shared__ Vectors<kQkTile> vs;
    __shared__ int32_t red[256 / kQkTile][kQkTile], s_max[kQkTile];
    Part p;
    if (!part_of<kQkTile>(a, a.qk, p)) return;
    if (p.subs == 1) prefix_qk_part<HD, FAST, PASS, 1>(a, p, vs, tab, klds, red, s_max);
    else if (p.subs == 2) prefix_qk_part<HD, FAST, PASS, 2>(a, p, vs, tab, klds, red, s_max);
    else prefix_qk_part<HD, FAST, PASS, 4>(a, p, vs, tab, klds, red, s_max);
}

// What a vector's probabilities need.
struct ProbRow {
    ProbDiv div;
    uint32_t base, extra;  // S = 0: the uniform split (softmax.rs:42-48), 1 more for keys below `extra`
    int32_t uniform, pad;
};

// sum p_j v_j of a tile's vectors over a range, HD dimensions: the dimensions are the
// rows of v_mfma_i32_16x16x64_i8, the vectors its columns.  A step covers KU x 64 keys per
// key wave.  p <= 2^14 splits into two signed bytes exactly (p = 256 ph + pl), v into
// v = 256 vh + vl' + 128, so
//   sum p v = 65536 hh + 256 (hl + lh) + ll + 128 sum p
// modulo 2^32, and the whole sum fits 32 bits (serve_plan.h).  V is turned in registers:
// lane l loads dimensions 2 (l % 16), + 1 of the 16 keys of its block l / 16 and
// gathers each dimension's bytes of four keys with v_perm, which is the A operand.
// The p planes pass through LDS, two steps' places in turn, one barrier a step.  Bound by
// issue like the scores: 65 us at 64 rows of 28 heads by 30000 keys of 128.
template <int HD>
struct PvShape {
    static constexpr int DW = HD / 32;  // waves side by side over the dimensions
    static constexpr int KW = 4 / DW;   // over the keys
};

template <int HD, int SUB, int KU>
struct PvLds {
    static constexpr int kKeys = 64 * PvShape<HD>::KW * KU;  // keys of a step
    static constexpr int kChunks = kKeys / 16;
    static constexpr int kRow = 16 * SUB * 16;               // bytes of a 16-key chunk of all vectors
    static constexpr int kPlane = kChunks * kRow;
    static constexpr int kBytes = 4 * kPlane;                // two planes, two steps
};

template <int HD, int SUB, int KU>
__device__ inline void prefix_pv_part(const PrefixAttn& a, const Part& p, const Vectors<kPvTile>& vs, int8_t* lds, ProbRow* rows,
                                      int32_t* p_sum, int32_t (*red)[kPvTile]) {
    using L = PvLds<HD, SUB, KU>;
    constexpr int DW = PvShape<HD>::DW, KW = PvShape<HD>::KW, CH = L::kChunks;
    constexpr int V = 16 * SUB, ITEMS = (V * CH + 255) / 256;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, kb = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), dw = wave % DW, kw = wave / DW;
    const int16_t* vg = keys_of(a, p, a.vp, a.vt);
    const __amdgpu_buffer_rsrc_t rv = weight_rsrc(vg, (uint32_t)(p.tail ? a.max_tail : a.P) * HD * 2u);
    const uint32_t vlane = (uint32_t)(64 * kw + 16 * kb) * HD + 32u * dw + 2u * c;
    uint32_t vx[KU][16];
    auto load_v = [&](int j) {
#pragma unroll
        for (int k = 0; k < KU; ++k) {
            const uint32_t at = ((uint32_t)(j + 64 * k * KW) * HD + vlane) * 2u;
#pragma unroll
            for (int i = 0; i < 16; ++i) vx[k][i] = cload4(rv, at + 2u * HD * i);
        }
    };
    load_v(p.j0);
    // the vectors' exp sums over all ranges, and what follows from them
    const int v0 = tid & (kPvTile - 1), share = tid / kPvTile;
    const int j1 = min(p.j1, wave_max_i32(vs.lim[v0]));
    if (p.j0 >= j1) return;  // uniform: every wave's lanes hold all vectors
    {
        uint32_t s = 0;
        fold_ranges<256 / kPvTile>(a, a.psum, vs.pair[v0], vs.tail[v0], share, [&](int32_t x) { s += (uint32_t)x; });
        red[share][v0] = (int32_t)s;
        block_barrier();
        if (tid < kPvTile) {
            const uint32_t S = (uint32_t)(red[0][tid] + red[1][tid] + red[2][tid] + red[3][tid]);
            ProbRow r{};
            r.div = ProbDiv::of(S ? S : 1u, a.prob_frac);
            r.uniform = S == 0 ? 1 : 0;
            const uint32_t keys = (uint32_t)(a.P + max(vs.tail[tid], 0)), one = 1u << a.prob_frac;
            if (S == 0 && keys) udivmod32(one, keys, recip32(keys), &r.base, &r.extra);
            rows[tid] = r;
            p_sum[tid] = 0;
        }
        block_barrier();
    }
    v4i32_t hh[SUB][2], mid[SUB][2], ll[SUB][2];
#pragma unroll
    for (int t = 0; t < SUB; ++t)
#pragma unroll
        for (int d = 0; d < 2; ++d) hh[t][d] = mid[t][d] = ll[t][d] = v4i32_t{0, 0, 0, 0};
    // the thread's vectors and its 16-key chunk of a step
    int32_t psum[ITEMS], lim[ITEMS];
    ProbDiv div[ITEMS];
    const uint16_t* erow[ITEMS];
    uint2 ex[ITEMS][4];
    const int kfirst = p.tail ? a.P : 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int it = tid + 256 * i, v = it % V, ch = it / V;
        psum[i] = 0;
        lim[i] = ch < CH ? min(vs.lim[v], j1) - 16 * ch : 0;
        div[i] = rows[v].div;
        erow[i] = exp_tile(a, p, min(v >> 4, p.subs - 1)) + 256 * ch + 4 * (v & 15);  // tiles past the last repeat it
    }
    auto load_e = [&](int j) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) ex[i][k] = make_uint2(0, 0);
            if (j < lim[i])
#pragma unroll
                for (int k = 0; k < 4; ++k) ex[i][k] = *reinterpret_cast<const uint2*>(erow[i] + 16 * j + 64 * k);
        }
    };
    load_e(p.j0);
    int buf = 0;
    for (int j = p.j0; j < j1; j += L::kKeys, buf ^= 1) {
        int8_t* ph = lds + buf * 2 * L::kPlane;
        int8_t* pl = ph + L::kPlane;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int it = tid + 256 * i, v = it % V, ch = it / V;
            if (it >= V * CH) break;
            const uint32_t w[8] = {ex[i][0].x, ex[i][0].y, ex[i][1].x, ex[i][1].y, ex[i][2].x, ex[i][2].y, ex[i][3].x, ex[i][3].y};
            uint32_t pw[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) pw[k] = div[i](w[k] & 0xFFFFu) | (div[i](w[k] >> 16) << 16);
            if (rows[v].uniform) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    uint32_t two = 0;
#pragma unroll
                    for (int b = 0; b < 2; ++b)
                        if (j + 2 * k + b < lim[i])
                            two |= (rows[v].base + ((uint32_t)(kfirst + j + 16 * ch + 2 * k + b) < rows[v].extra ? 1u : 0u)) << (16 * b);
                    pw[k] = two;
                }
            }
            uint32_t hw[4], lw[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                psum[i] = sum_pairs(pw[2 * k], psum[i]);
                psum[i] = sum_pairs(pw[2 * k + 1], psum[i]);
                // pl = p as a signed byte, ph = (p - pl) / 256: 128 carries into the high byte
                lw[k] = __builtin_amdgcn_perm(pw[2 * k + 1], pw[2 * k], 0x06040200u);
                hw[k] = __builtin_amdgcn_perm(pw[2 * k + 1] + 0x00800080u, pw[2 * k] + 0x00800080u, 0x07050301u);
            }
            *reinterpret_cast<uint4*>(ph + ch * L::kRow + v * 16) = make_uint4(hw[0], hw[1], hw[2], hw[3]);
            *reinterpret_cast<uint4*>(pl + ch * L::kRow + v * 16) = make_uint4(lw[0], lw[1], lw[2], lw[3]);
        }
        v4i32_t vh[KU][2], vl[KU][2];
#pragma unroll
        for (int k = 0; k < KU; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t* x = vx[k] + 4 * i;
                // bytes of two dimensions at four keys: low, high of the first, low, high of the second
                const uint32_t a0 = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), a1 = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
                const uint32_t b0 = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u), b1 = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
                vl[k][0][i] = (int)(__builtin_amdgcn_perm(a1, a0, 0x05040100u) ^ 0x80808080u);
                vh[k][0][i] = (int)__builtin_amdgcn_perm(a1, a0, 0x07060302u);
                vl[k][1][i] = (int)(__builtin_amdgcn_perm(b1, b0, 0x05040100u) ^ 0x80808080u);
                vh[k][1][i] = (int)__builtin_amdgcn_perm(b1, b0, 0x07060302u);
            }
        load_e(j + L::kKeys);
        load_v(j + L::kKeys);
        block_barrier();
#pragma unroll
        for (int k = 0; k < KU; ++k)
#pragma unroll
            for (int t = 0; t < SUB; ++t) {
                const int off = (4 * (k * KW + kw) + kb) * L::kRow + (16 * t + c) * 16;
                const v4i32_t bh = *reinterpret_cast<const v4i32_t*>(ph + off), bl = *reinterpret_cast<const v4i32_t*>(pl + off);
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    hh[t][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vh[k][d], bh, hh[t][d], 0, 0, 0);
                    mid[t][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vh[k][d], bl, mid[t][d], 0, 0, 0);
                    mid[t][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vl[k][d], bh, mid[t][d], 0, 0, 0);
                    ll[t][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vl[k][d], bl, ll[t][d], 0, 0, 0);
                }
            }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int it = tid + 256 * i;
        if (it < V * CH) atomicAdd(&p_sum[it % V], psum[i]);
    }
    block_barrier();
    // the key waves' sums meet in LDS (in place of the P planes)
    int32_t* sums = reinterpret_cast<int32_t*>(lds);  // [vector][HD + 4]
    constexpr int SROW = HD + 4;
    static_assert(KW == 1 || 16 * SUB * SROW * 4 <= L::kBytes, "the sums fit the planes' place");
    uint32_t o[SUB][8];
#pragma unroll
    for (int t = 0; t < SUB; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < 2; ++d)
                o[t][2 * i + d] = ((uint32_t)hh[t][d][i] << 16) + ((uint32_t)mid[t][d][i] << 8) + (uint32_t)ll[t][d][i];
    const int d0 = 32 * dw + 8 * kb;
    if (KW == 2) {
        if (kw == 1)
#pragma unroll
            for (int t = 0; t < SUB; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<uint4*>(sums + (16 * t + c) * SROW + d0 + 4 * h) =
                        make_uint4(o[t][4 * h], o[t][4 * h + 1], o[t][4 * h + 2], o[t][4 * h + 3]);
        block_barrier();
        if (kw == 1) return;
#pragma unroll
        for (int t = 0; t < SUB; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i) o[t][i] += (uint32_t)sums[(16 * t + c) * SROW + d0 + i];
    }
#pragma unroll
    for (int t = 0; t < SUB; ++t) {
        const int v = 16 * t + c;
        if (v >= p.nv) continue;
        const uint32_t add = 128u * (uint32_t)p_sum[v];
        int32_t* dst = a.pout + ((size_t)p.range * a.pairs + vs.pair[v]) * HD + d0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            *reinterpret_cast<uint4*>(dst + 4 * h) = make_uint4(o[t][4 * h] + add, o[t][4 * h + 1] + add, o[t][4 * h + 2] + add, o[t][4 * h + 3] + add);
    }
}

template <int HD>
__global__ __launch_bounds__(256, 3) void prefix_pv_kernel(PrefixAttn a) {
    constexpr int kLds = std::max({PvLds<HD, 4, 1>::kBytes, PvLds<HD, 2, 1>::kBytes, PvLds<HD, 1, 2>::kBytes});
    __shared__ __align__(16) int8_t lds[kLds];
    __shared__ __align__(16) ProbRow rows[kPvTile];
    __shared__ Vectors<kPvTile> vs;
    __shared__ int32_t red[4][kPvTile], p_sum[kPvTile];
    Part p;
    if (!part_of<kPvTile>(a, a.pv, p)) return;
    vectors_of<kPvTile, true>(a, p, HD, vs);
    block_barrier();
    if (p.subs == 1) prefix_pv_part<HD, 1, 2>(a, p, vs, lds, rows, p_sum, red);
    else if (p.subs == 2) prefix_pv_part<HD, 2, 1>(a, p, vs, lds, rows, p_sum, red);
    else prefix_pv_part<HD, 4, 1>(a, p, vs, lds, rows, p_sum, red);
}

// The ranges' sums, one rounding (attention.rs:84-86); four dimensions per thread.
template <int HD>
__global__ __launch_bounds__(256) void prefix_out_kernel(PrefixAttn a) {
    const int row = blockIdx.y, i = 4 * (blockIdx.x * 256 + (int)threadIdx.x);
    if (i >= a.heads * HD) return;
    int rem;
    const int seq = divmod(a.n, row, rem), tail = tail_of(a, row, slot_of(a, seq));
    uint32_t s[4] = {0, 0, 0, 0};
    // the ranges with a key of the row, eight loads in flight
    const int all = a.np_count + a.nt_count;
    for (int r0 = 0; tail >= 0 && r0 < all; r0 += 8) {
        uint4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int r = r0 + k;
            x[k] = make_uint4(0, 0, 0, 0);
            if (r < all && (r < a.np_count || (r - a.np_count) * a.rt < tail))
                x[k] = *reinterpret_cast<const uint4*>(a.pout + ((size_t)r * a.pairs + (size_t)row * a.heads) * HD + i);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            s[0] += x[k].x;
            s[1] += x[k].y;
            s[2] += x[k].z;
            s[3] += x[k].w;
        }
    }
    uint32_t y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = (uint32_t)(uint16_t)clamp_i16(rshift_round32((int32_t)s[k], a.prob_frac));
    *reinterpret_cast<uint2*>(a.out + (size_t)row * a.ldo + i) = make_uint2(y[0] | (y[1] << 16), y[2] | (y[3] << 16));
}

// ---- few keys: one launch ---------------------------------------------------------

// A block per row and KV head does all of it: scores of the row's query heads (at most 8, of
// the 15 of qk_planes_wave) with all keys into LDS, a wave per head for the softmax,
// P.V with a pair of dimensions and every so-many-th eight keys per thread.  The keys are
// read for every row instead of every 64 vectors, but nothing waits for another launch: 9.1 us
// for 2 rows of 14 heads by 131 keys of 64, where four launches took 19.  Bound by the chain
// of loads, softmax and sums in a block; the adds into acc are of integers, in any order.
template <int HD>
__global__ __launch_bounds__(kShortThreads) void prefix_short_kernel(PrefixAttn a) {
    constexpr int PAIRS = HD / 2, STREAMS = kShortThreads / PAIRS, WAVES = kShortThreads / 64;
    static_assert(WAVES >= (int)kPrefixShortHeads);
    extern __shared__ __align__(16) int32_t z[];  // [G][cap] scores, [G][cap] probabilities, [G][HD] sums
    const int G = (int)a.G.d, cap = a.short_cap;
    uint16_t* ps = reinterpret_cast<uint16_t*>(z + G * cap);
    int32_t* acc = reinterpret_cast<int32_t*>(ps + G * cap);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int g, rem;
    const int row = divmod(a.kvh, (int)blockIdx.x, g), slot = slot_of(a, divmod(a.n, row, rem));
    const int tail = __builtin_amdgcn_readfirstlane(tail_of(a, row, slot)), L = tail < 0 ? 0 : a.P + tail;
    int16_t* out = a.out + (size_t)row * a.ldo + (size_t)(g * G * HD);
    for (int i = tid; i < G * HD; i += kShortThreads) acc[i] = 0;
    const size_t toff = (size_t)max(slot, 0) * a.ts + (size_t)g * a.th, poff = (size_t)g * a.ph;
    const int16_t* q = a.q + (size_t)row * a.ldq + (size_t)(g * G * HD);
    const int gp = tail < 0 ? 0 : (a.P + 15) >> 4, groups = gp + (max(tail, 0) + 15) / 16;
    for (int i = wave; i < groups; i += WAVES) {
        if (i < gp) qk_planes_wave<HD>(a.P, 16 * i, a.kp + poff, q, G, a.mult, a.shift, z, (size_t)cap);
        else qk_planes_wave<HD>(tail, 16 * (i - gp), a.kt + toff, q, G, a.mult, a.shift, z + a.P, (size_t)cap);
    }
    __syncthreads();
    if (const int h = wave; h < G && L > 0) {
        int32_t* zh = z + h * cap;
        int32_t m = INT32_MIN;
        for (int j = lane; j < L; j += 64) m = max(m, zh[j]);
        m = wave_max_i32(m);
        uint32_t s = 0;
        for (int j = lane; j < L; j += 64) {  // sat_sub and the lookup of softmax.rs:12-38
            const uint32_t i = min((uint32_t)m - (uint32_t)zh[j], 0x7FFFFFFFu) >> (a.lut_shift & 31u);
            const int32_t e = i < a.lut_len ? max((int32_t)a.lut[i], 0) : 0;
            zh[j] = e;
            s += (uint32_t)e;
        }
        s = (uint32_t)wave_sum_i32((int32_t)s);
        const ProbDiv div = ProbDiv::of(s ? s : 1u, a.prob_frac);
        uint32_t base = 0, extra = 0;
        if (s == 0) udivmod32(1u << a.prob_frac, (uint32_t)L, recip32((uint32_t)L), &base, &extra);
        for (int j = lane; j < ((L + 7) & ~7); j += 64) {
            const uint32_t p = j >= L ? 0u : s ? div((uint32_t)zh[j]) : base + ((uint32_t)j < extra ? 1u : 0u);
            ps[h * cap + j] = (uint16_t)p;
        }
    }
    __syncthreads();
    // dimensions 2 dp, + 1; the probabilities are at most 2^14, so pairs of keys fit v_dot2
    const int dp = tid % PAIRS, stream = tid / PAIRS;
    const int16_t *vp = a.vp + poff + 2 * dp, *vt = a.vt + toff + 2 * dp;
    if (L > 0) {
        int32_t s0[kPrefixShortHeads], s1[kPrefixShortHeads];
#pragma unroll
        for (int h = 0; h < (int)kPrefixShortHeads; ++h) s0[h] = s1[h] = 0;
        for (int j0 = 8 * stream; j0 < L; j0 += 8 * STREAMS) {
            uint32_t v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int j = min(j0 + k, L - 1);
                v[k] = *reinterpret_cast<const uint32_t*>((j < a.P ? vp : vt) + (size_t)(j < a.P ? j : j - a.P) * HD);
            }
            uint32_t w0[4], w1[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                w0[k] = __builtin_amdgcn_perm(v[2 * k + 1], v[2 * k], 0x05040100u);
                w1[k] = __builtin_amdgcn_perm(v[2 * k + 1], v[2 * k], 0x07060302u);
            }
#pragma unroll
            for (int h = 0; h < (int)kPrefixShortHeads; ++h) {
                if (h >= G) break;
                const uint4 p4 = *reinterpret_cast<const uint4*>(ps + h * cap + j0);
                const uint32_t p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    s0[h] = dot_pairs(w0[k], p[k], s0[h]);
                    s1[h] = dot_pairs(w1[k], p[k], s1[h]);
                }
            }
        }
#pragma unroll
        for (int h = 0; h < (int)kPrefixShortHeads; ++h) {
            if (h >= G) break;
            atomicAdd(&acc[h * HD + 2 * dp], s0[h]);
            atomicAdd(&acc[h * HD + 2 * dp + 1], s1[h]);
        }
    }
    __syncthreads();
    for (int i = tid; i < G * HD; i += kShortThreads) out[i] = clamp_i16(rshift_round32(acc[i], a.prob_frac));
}

template <int HD, bool FAST>
hipError_t prefix_scores(const PrefixAttn& a, unsigned grid, hipStream_t st) {
    prefix_qk_kernel<HD, FAST, kMaxPass><<<grid, 256, 0, st>>>(a);
    const size_t tab = ((size_t)a.lut_len / 8 + 1) * 16;
    if (tab > 24 * 1024) {  // with the K rows' place more than the 64 KiB a launch has by default
        const hipError_t e = hipFuncSetAttribute((const void*)prefix_qk_kernel<HD, FAST, kExpPass>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)((kPrefixMaxLut / 8 + 1) * 16));
        if (e != hipSuccess) return e;
    }
    prefix_qk_kernel<HD, FAST, kExpPass><<<grid, 256, tab, st>>>(a);
    return hipGetLastError();
}

template <int HD>
hipError_t prefix_launch(const PrefixAttn& a, const PrefixPlan& pl, hipStream_t st) {
    if (pl.short_cap) {
        prefix_short_kernel<HD><<<(unsigned)(a.R * (int)a.kvh.d), kShortThreads, prefix_short_lds(pl.G, pl.short_cap, HD), st>>>(a);
        return hipGetLastError();
    }
    const unsigned grid = (unsigned)(pl.qk.blocks_p + pl.qk.blocks_t);
    if (grid) {
        // 2^31 >> lut_shift is past every table
        const bool fast = a.scale.fast && (a.lut_shift & 31) <= 15;
        const hipError_t e = fast ? prefix_scores<HD, true>(a, grid, st) : prefix_scores<HD, false>(a, grid, st);
        if (e != hipSuccess) return e;
        prefix_pv_kernel<HD><<<(unsigned)(pl.pv.blocks_p + pl.pv.blocks_t), 256, 0, st>>>(a);
    }
    prefix_out_kernel<HD><<<dim3((unsigned)((a.heads * HD + 1023) / 1024), (unsigned)a.R), 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace
}  // namespace myl

using namespace myl;

extern "C" {

size_t myl_attention_prefix_workspace(const myl_ctx* ctx, size_t n_seqs, size_t rows_per_seq, size_t heads, size_t kv_heads,
                                      size_t head_dim, size_t prefix_len, size_t max_tail) {
    const PrefixShape s{n_seqs, rows_per_seq, heads, kv_heads, head_dim, prefix_len, max_tail};
    if (!ctx || prefix_refuse(s) || (head_dim != 64 && head_dim != 128)) return 0;
    return prefix_plan(s, ctx->prop.multiProcessorCount).bytes;
}

int myl_attention_prefix_dev(myl_ctx* ctx, const int16_t* q, size_t n_seqs, size_t rows_per_seq, size_t ldq, size_t heads,
                             size_t kv_heads, size_t head_dim, const int16_t* k_prefix, const int16_t* v_prefix,
                             size_t prefix_len, size_t prefix_head_stride, const int16_t* k_tail, const int16_t* v_tail,
                             size_t n_slots, size_t tail_slot_stride, size_t tail_head_stride, size_t max_tail,
                             const int32_t* slots, const int32_t* lens, int64_t score_mult, uint8_t score_shift,
                             const int16_t* exp_lut, size_t lut_len, uint8_t lut_shift, uint8_t prob_frac, int16_t* out,
                             size_t ldo, void* workspace, size_t workspace_bytes) {
    if (!ctx) return MYL_E_INVALID;
    const char* what = "attention_prefix_dev";
    auto bad = [&](const char* why) { return ctx->fail(MYL_E_INVALID, std::string(what) + ": " + why); };
    if (head_dim != 64 && head_dim != 128) return ctx->fail(MYL_E_UNSUPPORTED, std::string(what) + ": head_dim 64 or 128");
    const PrefixShape s{n_seqs, rows_per_seq, heads, kv_heads, head_dim, prefix_len, max_tail};
    if (const char* why = prefix_refuse(s)) return bad(why);
    if (ldq < heads * head_dim || ldo < heads * head_dim) return bad("leading dimension too small");
    if (kv_heads > 1 && (prefix_head_stride < prefix_len * head_dim || tail_head_stride < max_tail * head_dim))
        return bad("head stride too small");
    if (n_slots > kInt) return bad("too many slots");
    if (lut_len == 0 || lut_len > kPrefixMaxLut) return bad("the exp table must hold 1 to 32768 entries");
    if (prob_frac > 14) return bad("prob_frac is at most 14");
    if (n_seqs == 0 || rows_per_seq == 0) return MYL_OK;
    if (!q || !out || !exp_lut || !lens) return bad("null operand");
    if (prefix_len && (!k_prefix || !v_prefix)) return bad("null prefix");
    if (max_tail && n_slots && (!k_tail || !v_tail)) return bad("null tail");
    const uintptr_t ptrs = (uintptr_t)q | (uintptr_t)out | (uintptr_t)exp_lut | (uintptr_t)k_prefix | (uintptr_t)v_prefix | (uintptr_t)k_tail |
                           (uintptr_t)v_tail | (uintptr_t)workspace;
    if ((ptrs & 15) || ((ldq | ldo | prefix_head_stride | tail_slot_stride | tail_head_stride) & 7))
        return bad("operands must be 16-byte aligned, strides multiples of 8");
    const PrefixPlan pl = prefix_plan(s, ctx->prop.multiProcessorCount);
    if (!workspace || workspace_bytes < pl.bytes) return bad("workspace too small (myl_attention_prefix_workspace)");
    const DeviceGuard guard(ctx->device);
    char* ws = static_cast<char*>(workspace);
    PrefixAttn a{};
    a.q = q; a.kp = k_prefix; a.vp = v_prefix; a.kt = k_tail; a.vt = v_tail;
    a.slots = slots; a.lens = lens; a.lut = exp_lut; a.out = out;
    a.pmax = reinterpret_cast<int32_t*>(ws + pl.off_max);
    a.psum = reinterpret_cast<int32_t*>(ws + pl.off_sum);
    a.pexp = reinterpret_cast<uint16_t*>(ws + pl.off_pexp);
    a.texp = reinterpret_cast<uint16_t*>(ws + pl.off_texp);
    a.pout = reinterpret_cast<int32_t*>(ws + pl.off_out);
    a.ldq = ldq; a.ldo = ldo; a.ph = prefix_head_stride; a.ts = tail_slot_stride; a.th = tail_head_stride;
    a.mult = score_mult;
    a.scale = ScoreScale::of(score_mult, score_shift, (int)head_dim);
    auto div = [](size_t d) { return SmallDiv::of(std::max<size_t>(d, 1)); };
    a.n = div(rows_per_seq); a.G = div((size_t)pl.G); a.kvh = div(kv_heads);
    a.np = div((size_t)pl.np); a.nt = div((size_t)pl.nt);
    auto cut = [&](const PrefixPlan::Cut& c) { return PrefixAttn::Cut{div((size_t)c.tp), div((size_t)c.tt), (int)c.blocks_p}; };
    a.qk = cut(pl.qk); a.pv = cut(pl.pv);
    a.short_cap = pl.short_cap;
    a.R = (int)(n_seqs * rows_per_seq); a.heads = (int)heads; a.P = (int)prefix_len; a.max_tail = (int)max_tail;
    a.n_slots = (int)n_slots; a.vp_count = pl.vp; a.vt_count = pl.vt; a.np_count = pl.np; a.nt_count = pl.nt;
    a.rp = pl.rp; a.rt = pl.rt; a.vp16 = (pl.vp + 15) / 16; a.vt16 = (pl.vt + 15) / 16; a.pgroups = pl.pgroups; a.tgroups = pl.tgroups;
    a.pairs = (uint32_t)pl.pairs; a.lut_len = (uint32_t)lut_len;
    a.shift = score_shift; a.lut_shift = lut_shift; a.prob_frac = prob_frac;
    return ctx->hip(head_dim == 128 ? prefix_launch<128>(a, pl, ctx->stream) : prefix_launch<64>(a, pl, ctx->stream), what);
}

}  // extern "C"
