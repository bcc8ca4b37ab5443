// paged_append.hip -- new rows of a paged cache: biases (linear.rs:132-145), norms of
// each head (rmsnorm.rs:61-161), the rotation of the row's position (rope.rs:17-59),
// keys and values into their pages: myl_kv_append_paged_dev.
//
// A thread takes dimensions 8 c .. + 7 of a head and the 8 they rotate with, half a head
// further on: two 16-byte loads and two 16-byte stores.  A norm's sum of squares goes over
// the head's hd / 16 neighbouring threads.
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
    int items, heads, kv_heads, n_seqs, table_len, n_pages;
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

__device__ inline void add_bias8(const Append& a, size_t at, uint8_t frac, int32_t (&x)[8]) {
    int32_t b[8];
    unpack8(load8(a.bias + at), b);
    const uint2 s = *reinterpret_cast<const uint2*>(a.bias_shifts + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint8_t sh = (uint8_t)((i < 4 ? s.x : s.y) >> (8 * (i & 3)));
        x[i] = clamp_i16_i64((int64_t)x[i] + (int64_t)rescale32(b[i], sh, frac));
    }
}

template <int HD, bool BIAS, bool NORM>
__global__ __launch_bounds__(256) void append_kernel(Append a) {
    constexpr int CH = HD / 16, HALF = HD / 2;
    const int t = (int)(blockIdx.x * 256u + threadIdx.x);
    if (t >= a.items) return;
    int rem;
    const int row = divmod(a.per_row, t, rem), hh = rem / CH, d = 8 * (rem % CH);
    const int pos = a.pos[row], seq = a.seqs ? a.seqs[row] : row;
    if (pos < 0 || seq < 0 || seq >= a.n_seqs) return;
    const int kind = hh < a.heads ? 0 : hh < a.heads + a.kv_heads ? 1 : 2;  // q, k, v
    const int h = hh - (kind == 0 ? 0 : kind == 1 ? a.heads : a.heads + a.kv_heads);
    const int16_t* src = (kind == 0 ? a.q + (size_t)row * a.ldq : kind == 1 ? a.k + (size_t)row * a.ldk : a.v + (size_t)row * a.ldv) +
                         (size_t)h * HD + d;
    int32_t x0[8], x1[8];
    unpack8(load8(src), x0);
    unpack8(load8(src + HALF), x1);
    if (BIAS) {
        const uint8_t frac = kind == 0 ? a.q_frac : kind == 1 ? a.k_frac : a.v_frac;
        add_bias8(a, (size_t)hh * HD + d, frac, x0);
        add_bias8(a, (size_t)hh * HD + d + HALF, frac, x1);
    }
    if (NORM) {
        const int8_t* gamma = kind == 0 ? a.q_gamma : kind == 1 ? a.k_gamma : nullptr;
        const uint8_t* shifts = kind == 0 ? a.q_gamma_shifts : a.k_gamma_shifts;
        uint64_t s = 0;  // at most 128 2^30
#pragma unroll
        for (int i = 0; i < 8; ++i) s += (uint64_t)((int64_t)x0[i] * x0[i]) + (uint64_t)((int64_t)x1[i] * x1[i]);
        s = dpp_add64<dpp::kXor1>(s);
        s = dpp_add64<dpp::kXor2>(s);
        if (CH == 8) s = dpp_add64<dpp::kHalfMirror>(s);
        if (gamma) {
            const RmsFactor f = rms_factor_of((myl_i128)s, 0, a.rms);
            const uint8_t frac = kind == 0 ? a.q_norm_frac : a.k_norm_frac;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x0[i] = rms_out((int16_t)x0[i], 0, gamma[d + i], shifts[d + i], f, frac);
                x1[i] = rms_out((int16_t)x1[i], 0, gamma[d + HALF + i], shifts[d + HALF + i], f, frac);
            }
        }
    }
    if (kind < 2) {
        int turn;
        divmod(a.n_pos, pos, turn);
        int32_t c[8], s[8];
        unpack8(load8(a.cos + (size_t)turn * HALF + d), c);
        unpack8(load8(a.sin + (size_t)turn * HALF + d), s);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int32_t u = x0[i], w = x1[i];
            x0[i] = clamp_i16(rshift_round32(wsub32(wmul32(u, c[i]), wmul32(w, s[i])), a.rope_frac));
            x1[i] = clamp_i16(rshift_round32(wadd32(wmul32(w, c[i]), wmul32(u, s[i])), a.rope_frac));
        }
    }
    int16_t* dst;
    if (kind == 0) {
        dst = a.qo + (size_t)row * a.ldo + (size_t)h * HD + d;
    } else {
        int off;
        const int at = divmod(a.page, pos, off);
        const int id = at < a.table_len ? a.tables[(size_t)seq * a.ldt + at] : -1;
        if (id < 0 || id >= a.n_pages) return;
        dst = (kind == 1 ? a.kp : a.vp) + (size_t)id * a.page_stride + (size_t)h * a.head_stride + (size_t)off * a.pos_stride + d;
    }
    *reinterpret_cast<uint4*>(dst) = pack8(x0);
    *reinterpret_cast<uint4*>(dst + HALF) = pack8(x1);
}

template <int HD>
void append_launch(const Append& a, bool norm, hipStream_t st) {
    const unsigned grid = (unsigned)((a.items + 255) / 256);
    if (a.bias && norm) append_kernel<HD, true, true><<<grid, 256, 0, st>>>(a);
    else if (a.bias) append_kernel<HD, true, false><<<grid, 256, 0, st>>>(a);
    else if (norm) append_kernel<HD, false, true><<<grid, 256, 0, st>>>(a);
    else append_kernel<HD, false, false><<<grid, 256, 0, st>>>(a);
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
    a.items = (int)(rows * per_row); a.heads = (int)heads; a.kv_heads = (int)kv_heads;
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
