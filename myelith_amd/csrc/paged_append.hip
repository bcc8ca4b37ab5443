// paged_append.hip -- new rows of a paged cache: biases (linear.rs:132-145), norms of
// each head (rmsnorm.rs:61-161), the rotation of the row's position (rope.rs:17-59),
// keys and values into their pages: myl_kv_append_paged_dev.
//
// A thread takes dimensions 8 c .. + 7 of a head and the 8 they rotate with, half a head
// further on: two 16-byte loads and two 16-byte stores a row.  A norm's sum of squares goes over
// the head's hd / 16 neighbouring threads.  Bound by the bytes for many rows, so long as
// few instructions go on each value (with the general shifts and a bias worked out for every row
// 16384 rows took 89 us): a thread keeps its dimensions over several rows, four of them in flight,
// and the biases are brought to their scale once for all of them; the rounding shifts take
// 32-bit steps where their shifts allow it.  16384 rows of 36 heads of 128 take 69 us (4.4 TB/s;
// loads past the caches 68, but 13.6 against 12.8 for 1503 rows with norms, so not taken).  With
// norms registers bound it too (96 for 16 values and their channels; held to 80 or 64, 1503 rows took 16
// and 23 us instead of 12.8; 16384 rows, four of them in flight at 150, 94).  Few rows: the launch and two loads that
// follow one another, 5 us.
#include "abi_internal.h"
#include "ops.h"
#include "paged_plan.h"
#include "wave.h"

#include <string>

namespace myl {
namespace {

struct Append {
    const int16_t *q, *k, *v;
    int16_t *kp, *vp, *qo;
    const int16_t* bias;
    const uint8_t* bias_shifts;
    const int16_t *cos, *sin;
    const int32_t *pos, *seqs, *tables;
    const int8_t *q_gamma, *k_gamma;
    const uint8_t *q_gamma_shifts, *k_gamma_shifts;
    RmsParams rms;
    size_t ldq, ldk, ldv, ldo, page_stride, head_stride, pos_stride, ldt;
    SmallDiv per_row, n_pos, page;
    int items, rows, group;  // threads; rows of a thread
    int heads, kv_heads, n_seqs, table_len, n_pages;
    uint8_t q_frac, k_frac, v_frac, q_norm_frac, k_norm_frac, rope_frac;
};

__device__ inline void unpack8(const uint4 x, int32_t (&v)[8]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = (int32_t)(int16_t)(w[i] & 0xFFFFu);
        v[2 * i + 1] = (int32_t)w[i] >> 16;
    }
}
__device__ inline uint4 pack8(const int32_t (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = ((uint32_t)v[2 * i] & 0xFFFFu) | ((uint32_t)v[2 * i + 1] << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ inline uint4 load8(const int16_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ inline int32_t sat16(int32_t x) { return min(max(x, -32768), 32767); }

// The biases of 8 dimensions at the rows' scale (linear.rs:132-145).
__device__ inline void bias8(const Append& a, size_t at, uint8_t frac, int32_t (&b)[8]) {
    unpack8(load8(a.bias + at), b);
    const uint2 s = *reinterpret_cast<const uint2*>(a.bias_shifts + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int32_t r = rescale32(b[i], (uint8_t)((i < 4 ? s.x : s.y) >> (8 * (i & 3))), frac);
        b[i] = min(max(r, -65536), 65536);  // added to 16 bits and clamped to them: the same
    }
}

// clamp_i16(rshift_round32(v, s)) for shifts of 1 .. 16: half a unit less a bit, and the bit that
// makes a tie even, carry into the result; where that passes 2^31 the result is past 16 bits.
struct TurnRound {
    uint32_t s;
    int32_t half;
    bool fast;
    __device__ inline static TurnRound of(uint8_t frac) {
        const bool ok = frac >= 1 && frac <= 16;
        return TurnRound{ok ? frac : 1u, ok ? (1 << (frac - 1)) - 1 : 0, ok};
    }
    __device__ inline int32_t operator()(int32_t v) const {
        return sat16(__builtin_elementwise_add_sat(v, half + (int32_t)(((uint32_t)v >> s) & 1u)) >> s);
    }
};

// A thread's 8 channels of a norm, as they are in memory: unpacked where they are used.
struct Gamma8 {
    uint2 g, s;
    uint32_t least, most;
    __device__ static inline uint32_t byte(const uint2& w, int i) { return ((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 255u; }
    __device__ inline void load(const int8_t* gamma, const uint8_t* shifts) {
        g = *reinterpret_cast<const uint2*>(gamma);
        s = *reinterpret_cast<const uint2*>(shifts);
        least = 255;
        most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            least = min(least, byte(s, i));
            most = max(most, byte(s, i));
        }
    }
    // rms_out of 8 values.  |x gamma lut| < 2^37, so right shifts by 6 .. 31 leave 32 bits.
    __device__ inline void apply(const RmsFactor& f, uint8_t frac, int32_t (&x)[8]) const {
        const int32_t base = (int32_t)f.norm_frac - (int32_t)frac;
        if (!f.zero && base + (int32_t)least >= 6 && base + (int32_t)most <= 31) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t sh = (uint32_t)base + byte(s, i);
                const int64_t p = (int64_t)(x[i] * (int32_t)(int8_t)byte(g, i)) * (int64_t)(int32_t)f.lut_val;
                const uint32_t lo = (uint32_t)p, hi = (uint32_t)((uint64_t)p >> 32);
                const uint32_t q = __builtin_amdgcn_alignbit(hi, lo, sh);
                const uint32_t rest = lo & ((1u << sh) - 1u);
                x[i] = sat16((int32_t)(q + ((rest + ((1u << (sh - 1)) - 1u) + (q & 1u)) >> sh)));
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = rms_out((int16_t)x[i], 0, (int8_t)byte(g, i), (uint8_t)byte(s, i), f, frac);
    }
};

// The sum of 8 squares in pairs: 2^31 at most each, unsigned.
__device__ inline uint64_t squares8(const uint4 x) {
    typedef short __attribute__((ext_vector_type(2))) s2;
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint64_t s = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) s += (uint32_t)__builtin_amdgcn_sdot2(__builtin_bit_cast(s2, w[i]), __builtin_bit_cast(s2, w[i]), 0, false);
    return s;
}

// rms_factor_of a head's sum of squares, at most 2^37: (sum inv_n) >> 20 with inv_n <= 2^20 in 64 bits.
__device__ inline RmsFactor head_factor(uint64_t sum, const RmsParams& p) {
    RmsIdx r{sum == 0, 0, 0};
    if (!r.zero) {
        const uint64_t m = (sum * (uint64_t)(uint32_t)p.inv_n_q20) >> 20;
        const uint32_t most = (uint32_t)p.lut_len - 1u;
        const uint32_t bm = 64u - (uint32_t)__builtin_clzll(m | 1u), bi = 32u - (uint32_t)__builtin_clz(most);
        r.q = bm > bi ? (bm - bi) & ~1u : 0u;
        if (m >> r.q > most) r.q += 2;
        r.idx = (int)min((uint32_t)rne_shift64_small((int64_t)m, r.q), most);
    }
    return rms_factor_at(r, 0, p, r.zero ? 0 : (int64_t)p.lut[r.idx]);
}

// R rows at a time, `group` of them to a thread.
template <int HD, bool BIAS, bool NORM, int R>
__global__ __launch_bounds__(256) void append_kernel(Append a) {
    constexpr int CH = HD / 16, HALF = HD / 2;
    const int t = (int)(blockIdx.x * 256u + threadIdx.x);
    if (t >= a.items) return;
    int rem;
    const int first = divmod(a.per_row, t, rem) * a.group, hh = rem / CH, d = 8 * (rem % CH);
    const int kind = hh < a.heads ? 0 : hh < a.heads + a.kv_heads ? 1 : 2;  // q, k, v
    const int h = hh - (kind == 0 ? 0 : kind == 1 ? a.heads : a.heads + a.kv_heads);
    const size_t ld = kind == 0 ? a.ldq : kind == 1 ? a.ldk : a.ldv;
    const int16_t* src = (kind == 0 ? a.q : kind == 1 ? a.k : a.v) + (size_t)h * HD + d;
    const TurnRound turn_round = TurnRound::of(a.rope_frac);
    int32_t b0[8], b1[8];
    if (BIAS) {
        const uint8_t frac = kind == 0 ? a.q_frac : kind == 1 ? a.k_frac : a.v_frac;
        bias8(a, (size_t)hh * HD + d, frac, b0);
        bias8(a, (size_t)hh * HD + d + HALF, frac, b1);
    }
    Gamma8 g0, g1;
    const int8_t* gamma = kind == 0 ? a.q_gamma : kind == 1 ? a.k_gamma : nullptr;
    const uint8_t norm_frac = kind == 0 ? a.q_norm_frac : a.k_norm_frac;
    if (NORM && gamma) {
        const uint8_t* shifts = kind == 0 ? a.q_gamma_shifts : a.k_gamma_shifts;
        g0.load(gamma + d, shifts + d);
        g1.load(gamma + d + HALF, shifts + d + HALF);
    }
    for (int row0 = first; row0 < min(first + a.group, a.rows); row0 += R) {
        int pos[R], seq[R], id[R], off[R];
        uint4 raw[R][2], cs[R][2];
        bool in[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = min(row0 + r, a.rows - 1);
            raw[r][0] = load8(src + (size_t)row * ld);
            raw[r][1] = load8(src + (size_t)row * ld + HALF);
            pos[r] = a.pos[row];
            seq[r] = a.seqs ? a.seqs[row] : row;
            in[r] = row0 + r < a.rows;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            in[r] = in[r] && pos[r] >= 0 && seq[r] >= 0 && seq[r] < a.n_seqs;
            if (!in[r]) pos[r] = 0;
            if (kind < 2) {
                int turn;
                divmod(a.n_pos, pos[r], turn);
                cs[r][0] = load8(a.cos + (size_t)turn * HALF + d);
                cs[r][1] = load8(a.sin + (size_t)turn * HALF + d);
            }
            id[r] = -1;
            if (kind > 0) {
                const int at = divmod(a.page, pos[r], off[r]);
                if (in[r] && at < a.table_len) id[r] = a.tables[(size_t)seq[r] * a.ldt + at];
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            int32_t x0[8], x1[8];
            unpack8(raw[r][0], x0);
            unpack8(raw[r][1], x1);
            if (BIAS)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x0[i] = sat16(x0[i] + b0[i]);
                    x1[i] = sat16(x1[i] + b1[i]);
                }
            if (NORM) {
                uint64_t s = BIAS ? squares8(pack8(x0)) + squares8(pack8(x1)) : squares8(raw[r][0]) + squares8(raw[r][1]);  // at most 128 2^30
                s = dpp_add64<dpp::kXor1>(s);
                s = dpp_add64<dpp::kXor2>(s);
                if (CH == 8) s = dpp_add64<dpp::kHalfMirror>(s);
                if (gamma) {
                    const RmsFactor f = head_factor(s, a.rms);
                    g0.apply(f, norm_frac, x0);
                    g1.apply(f, norm_frac, x1);
                }
            }
            if (kind < 2) {
                int32_t c[8], s[8];
                unpack8(cs[r][0], c);
                unpack8(cs[r][1], s);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int32_t u = x0[i], w = x1[i];
                    const int32_t y0 = wsub32(wmul32(u, c[i]), wmul32(w, s[i])), y1 = wadd32(wmul32(w, c[i]), wmul32(u, s[i]));
                    x0[i] = turn_round.fast ? turn_round(y0) : clamp_i16(rshift_round32(y0, a.rope_frac));
                    x1[i] = turn_round.fast ? turn_round(y1) : clamp_i16(rshift_round32(y1, a.rope_frac));
                }
            }
            if (!in[r]) continue;
            int16_t* dst;
            if (kind == 0) {
                dst = a.qo + (size_t)(row0 + r) * a.ldo + (size_t)h * HD + d;
            } else {
                if (id[r] < 0 || id[r] >= a.n_pages) continue;
                dst = (kind == 1 ? a.kp : a.vp) + (size_t)id[r] * a.page_stride + (size_t)h * a.head_stride + (size_t)off[r] * a.pos_stride + d;
            }
            *reinterpret_cast<uint4*>(dst) = pack8(x0);
            *reinterpret_cast<uint4*>(dst + HALF) = pack8(x1);
        }
    }
}

template <int HD, bool BIAS, bool NORM>
void append_rows(const Append& a, hipStream_t st) {
    const unsigned grid = (unsigned)((a.items + 255) / 256);
    if (a.group == 1) append_kernel<HD, BIAS, NORM, 1><<<grid, 256, 0, st>>>(a);
    else append_kernel<HD, BIAS, NORM, 4><<<grid, 256, 0, st>>>(a);
}
template <int HD>
void append_launch(const Append& a, bool norm, hipStream_t st) {
    if (a.bias && norm) append_rows<HD, true, true>(a, st);
    else if (a.bias) append_rows<HD, true, false>(a, st);
    else if (norm) append_rows<HD, false, true>(a, st);
    else append_rows<HD, false, false>(a, st);
}

}  // namespace
}  // namespace myl

using namespace myl;

extern "C" {

int myl_kv_append_paged_dev(myl_ctx* ctx, const int16_t* q, size_t ldq, const int16_t* k, size_t ldk, const int16_t* v,
                            size_t ldv, size_t rows, size_t heads, size_t kv_heads, size_t head_dim, const int16_t* bias,
                            const uint8_t* bias_shifts, uint8_t q_frac, uint8_t k_frac, uint8_t v_frac,
                            const myl_head_norm* norm, const int16_t* cos_lut, const int16_t* sin_lut, size_t lut_len,
                            uint8_t rope_frac, const int32_t* positions, const int32_t* seqs, const int32_t* tables,
                            size_t n_seqs, size_t table_len, size_t table_stride, int16_t* k_pages, int16_t* v_pages,
                            size_t n_pages, size_t page_size, size_t page_stride, size_t head_stride, size_t pos_stride,
                            int16_t* q_out, size_t ldo) {
    if (!ctx) return MYL_E_INVALID;
    const char* what = "kv_append_paged_dev";
    auto bad = [&](const char* why) { return ctx->fail(MYL_E_INVALID, std::string(what) + ": " + why); };
    if (head_dim != 64 && head_dim != 128) return ctx->fail(MYL_E_UNSUPPORTED, std::string(what) + ": head_dim 64 or 128");
    if (const char* why = append_refuse(rows, heads, kv_heads, head_dim)) return bad(why);
    if (const char* why = pages_refuse({n_pages, page_size, page_stride, head_stride, pos_stride, n_seqs, table_len, table_stride, kv_heads, head_dim}))
        return bad(why);
    if ((heads && (ldq < heads * head_dim || ldo < heads * head_dim)) || ldk < kv_heads * head_dim || ldv < kv_heads * head_dim)
        return bad("leading dimension too small");
    const size_t half = head_dim / 2;
    if (lut_len < half || lut_len / half > kInt) return bad("the rotation's tables hold 1 to 2^31 - 1 positions of head_dim / 2");
    if (norm) {
        if ((!norm->q_gamma != !norm->q_gamma_shifts) || (!norm->k_gamma != !norm->k_gamma_shifts)) return bad("a norm has gamma and its shifts");
        if (norm->lut_input_shift % 2) return bad("lut_input_shift must be even (rmsnorm.rs:76)");
        if (norm->rsqrt_len < 2 || norm->rsqrt_len > kInt) return bad("the rsqrt table must hold 2 to 2^31 - 1 entries");
        if (norm->inv_n_q20 < 0 || norm->inv_n_q20 > (1 << 20)) return bad("inv_n_q20 must be 0 to 2^20");
        if (!norm->rsqrt_lut) return bad("null rsqrt table");
    }
    if (rows == 0) return MYL_OK;
    if ((heads && (!q || !q_out)) || !k || !v || !cos_lut || !sin_lut || !positions || !k_pages || !v_pages || (n_seqs && table_len && !tables) ||
        (!bias != !bias_shifts))
        return bad("null operand");
    uintptr_t ptrs = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)bias | (uintptr_t)bias_shifts |
                     (uintptr_t)cos_lut | (uintptr_t)sin_lut | (uintptr_t)k_pages | (uintptr_t)v_pages;
    if (norm)
        ptrs |= (uintptr_t)norm->q_gamma | (uintptr_t)norm->q_gamma_shifts | (uintptr_t)norm->k_gamma | (uintptr_t)norm->k_gamma_shifts;
    if ((ptrs & 15) || ((ldq | ldk | ldv | ldo | page_stride | head_stride | pos_stride) & 7))
        return bad("operands must be 16-byte aligned, strides multiples of 8");
    const DeviceGuard guard(ctx->device);
    Append a{};
    a.q = q; a.k = k; a.v = v; a.kp = k_pages; a.vp = v_pages; a.qo = q_out;
    a.bias = bias; a.bias_shifts = bias_shifts; a.cos = cos_lut; a.sin = sin_lut;
    a.pos = positions; a.seqs = seqs; a.tables = tables;
    a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldo = ldo;
    a.page_stride = page_stride; a.head_stride = head_stride; a.pos_stride = pos_stride; a.ldt = table_stride;
    const size_t per_row = (heads + 2 * kv_heads) * (head_dim / 16);
    a.per_row = SmallDiv::of(per_row); a.n_pos = SmallDiv::of(lut_len / half); a.page = SmallDiv::of(page_size);
    a.rows = (int)rows; a.group = append_group(rows, per_row, ctx->prop.multiProcessorCount);
    a.items = (int)((rows + (size_t)a.group - 1) / (size_t)a.group * per_row); a.heads = (int)heads; a.kv_heads = (int)kv_heads;
    a.n_seqs = (int)n_seqs; a.table_len = (int)table_len; a.n_pages = (int)n_pages;
    a.q_frac = q_frac; a.k_frac = k_frac; a.v_frac = v_frac; a.rope_frac = rope_frac;
    const bool normed = norm && (norm->q_gamma || norm->k_gamma);
    if (normed) {
        a.q_gamma = norm->q_gamma; a.k_gamma = norm->k_gamma;
        a.q_gamma_shifts = norm->q_gamma_shifts; a.k_gamma_shifts = norm->k_gamma_shifts;
        a.rms.lut = norm->rsqrt_lut; a.rms.lut_len = (int)norm->rsqrt_len;
        a.rms.lut_input_shift = norm->lut_input_shift; a.rms.lut_output_frac = norm->lut_output_frac;
        a.rms.inv_n_q20 = norm->inv_n_q20;
        a.q_norm_frac = norm->q_out_frac; a.k_norm_frac = norm->k_out_frac;
    }
    if (head_dim == 128) append_launch<128>(a, normed, ctx->stream);
    else append_launch<64>(a, normed, ctx->stream);
    return ctx->hip(hipGetLastError(), what);
}

}  // extern "C"
