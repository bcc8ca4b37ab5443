// prefix_attn.hip -- integer attention (attention.rs:42-90 with
// softmax.rs:12-64) of a batch whose sequences share a prefix of K/V rows and
// continue with their own tails: myl_attention_prefix_dev.
#include "abi_internal.h"
#include "gemm_mfma.h"
#include "ops.h"

#include <string>

namespace myl {
namespace {

// The call, as every kernel sees it.  Row r = seq * rows_per_seq + i attends
// keys 0 .. P-1 of the prefix, then the first lens[r] of its sequence's tail.
struct PrefixAttn {
    const int16_t *q, *kp, *vp, *kt, *vt;
    const int32_t *slots, *lens;
    const int16_t* lut;
    int16_t* out;
    size_t ldq, ldo, ph, ts, th;  // strides in elements: q/out rows, prefix heads, tail slots, tail heads
    int64_t mult;
    Divider n, G;  // rows per sequence, query heads per KV head
    int R, heads, P, max_tail, n_slots, lcap;
    uint32_t lut_len;
    uint8_t shift, lut_shift, prob_frac;
};

// Tail positions of row r: -1 leaves the row out; a slot outside the cache has none.
__device__ inline int quotient(const Divider& d, int n) {
    uint32_t q, r;
    d.divmod((uint32_t)n, q, r);
    return (int)q;
}
__device__ inline int slot_of(const PrefixAttn& a, int r) {
    const int s = quotient(a.n, r);
    return a.slots ? a.slots[s] : s;
}
__device__ inline int tail_len(const PrefixAttn& a, int r) {
    const int len = a.lens[r], slot = slot_of(a, r);
    if (len < 0) return -1;
    return slot < 0 || slot >= a.n_slots ? 0 : min(len, a.max_tail);
}
__device__ inline size_t tail_off(const PrefixAttn& a, int r, int g) {
    return (size_t)slot_of(a, r) * a.ts + (size_t)g * a.th;
}

template <int HD>
__global__ __launch_bounds__(256) void scores_kernel(PrefixAttn a, int32_t* __restrict__ z) {
    const int j = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y, r = blockIdx.z, g = quotient(a.G, h);
    const int t = tail_len(a, r);
    if (t < 0 || j >= a.P + t) return;
    const int16_t* k = j < a.P ? a.kp + g * a.ph + (size_t)j * HD : a.kt + tail_off(a, r, g) + (size_t)(j - a.P) * HD;
    const int16_t* q = a.q + (size_t)r * a.ldq + (size_t)h * HD;
    int64_t dot = 0;
    for (int d = 0; d < HD; ++d) dot += (int32_t)q[d] * (int32_t)k[d];
    z[((size_t)r * a.heads + h) * a.lcap + j] = (int32_t)rshift_round64(wmul64(dot, a.mult), a.shift);
}

__device__ inline int32_t table(const PrefixAttn& a, int32_t below) {
    return max(0, exp_lookup(below, a.lut, a.lut_len, a.lut_shift, (int32_t)a.lut[0]));
}

__global__ __launch_bounds__(256) void probs_kernel(PrefixAttn a, const int32_t* __restrict__ zs, int16_t* __restrict__ ps) {
    __shared__ int32_t redm[4];
    __shared__ uint32_t reds[4];
    const int r = blockIdx.x, h = blockIdx.y, t = tail_len(a, r), L = a.P + t;
    if (t < 0 || L == 0) return;
    const int32_t* z = zs + ((size_t)r * a.heads + h) * a.lcap;
    int16_t* p = ps + ((size_t)r * a.heads + h) * a.lcap;
    int32_t mx = INT32_MIN;
    for (int j = threadIdx.x; j < L; j += 256) mx = max(mx, z[j]);
    mx = block_max_i32_dpp(mx, redm);
    uint32_t s = 0;
    for (int j = threadIdx.x; j < L; j += 256) s += (uint32_t)table(a, sat_sub32(mx, z[j]));
    const int32_t S = (int32_t)block_sum_u32_dpp(s, reds);
    const int32_t one = 1 << a.prob_frac;
    if (S == 0) {  // the uniform split (softmax.rs:42-48)
        uint32_t q, rem;
        udivmod32((uint32_t)one, (uint32_t)L, recip32((uint32_t)L), &q, &rem);
        for (int j = threadIdx.x; j < L; j += 256) p[j] = (int16_t)(q + ((uint32_t)j < rem ? 1 : 0));
        return;
    }
    const uint32_t m = recip32_u32((uint32_t)S);
    for (int j = threadIdx.x; j < L; j += 256) p[j] = (int16_t)softmax_div_round_pos(table(a, sat_sub32(mx, z[j])) << a.prob_frac, S, m);
}

template <int HD>
__global__ __launch_bounds__(HD) void pv_kernel(PrefixAttn a, const int16_t* __restrict__ ps) {
    const int r = blockIdx.x, h = blockIdx.y, g = quotient(a.G, h), d = threadIdx.x, t = tail_len(a, r);
    int64_t s = 0;
    if (t >= 0) {
        const int16_t* p = ps + ((size_t)r * a.heads + h) * a.lcap;
        for (int j = 0; j < a.P; ++j) s += (int32_t)p[j] * (int32_t)a.vp[g * a.ph + (size_t)j * HD + d];
        if (t > 0) {
            const int16_t* v = a.vt + tail_off(a, r, g);
            for (int j = 0; j < t; ++j) s += (int32_t)p[a.P + j] * (int32_t)v[(size_t)j * HD + d];
        }
    }
    a.out[(size_t)r * a.ldo + (size_t)h * HD + d] = clamp_i16_i64(rshift_round64(s, a.prob_frac));
}

// At most 65536 keys per row: with non-negative table entries the exp sums stay
// below 2^31.
constexpr size_t kMaxKeys = 65536;

struct Space {
    int32_t* z;
    int16_t* p;
    size_t bytes;
    static Space of(void* base, size_t R, size_t heads, size_t keys) {
        Carve c{(char*)base};
        Space s;
        s.z = c.take<int32_t>(R * heads * keys);
        s.p = c.take<int16_t>(R * heads * keys);
        s.bytes = c.used ? c.used : 256;  // 0 stands for sizes that a call refuses
        return s;
    }
};

}  // namespace
}  // namespace myl

using namespace myl;

extern "C" {

size_t myl_attention_prefix_workspace(const myl_ctx* ctx, size_t n_seqs, size_t rows_per_seq, size_t heads, size_t kv_heads,
                                      size_t head_dim, size_t prefix_len, size_t max_tail) {
    if (!ctx || !fits_int(n_seqs) || !fits_int(rows_per_seq) || !fits_int(n_seqs * rows_per_seq) ||
        (head_dim != 64 && head_dim != 128) || kv_heads == 0 || heads % kv_heads || heads > 65535 ||
        prefix_len > kMaxKeys || max_tail > kMaxKeys - prefix_len)
        return 0;
    return Space::of(nullptr, n_seqs * rows_per_seq, heads, prefix_len + max_tail).bytes;
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
    if (kv_heads == 0 || heads == 0 || heads % kv_heads) return bad("heads must be a multiple of kv_heads");
    if (heads > 65535 || !fits_int(n_seqs) || !fits_int(rows_per_seq) || n_seqs * rows_per_seq > 65535)
        return bad("too many rows or heads (65535 each)");
    if (prefix_len > kMaxKeys || max_tail > kMaxKeys - prefix_len) return bad("more than 65536 keys per row");
    if (ldq < heads * head_dim || ldo < heads * head_dim) return bad("leading dimension too small");
    if (prefix_len && prefix_head_stride < prefix_len * head_dim && kv_heads > 1) return bad("prefix head stride too small");
    if (max_tail && (tail_head_stride < max_tail * head_dim && kv_heads > 1)) return bad("tail head stride too small");
    if (!fits_int(n_slots)) return bad("too many slots");
    if (lut_len == 0 || !fits_int(lut_len)) return bad("the exp table must hold 1 to 2^31 - 1 entries");
    if (prob_frac > 14) return bad("prob_frac is at most 14");
    if (n_seqs == 0 || rows_per_seq == 0) return MYL_OK;
    if (!q || !out || !exp_lut || !lens) return bad("null operand");
    if (prefix_len && (!k_prefix || !v_prefix)) return bad("null prefix");
    if (max_tail && (!k_tail || !v_tail)) return bad("null tail");
    const uintptr_t ptrs = (uintptr_t)q | (uintptr_t)out | (uintptr_t)k_prefix | (uintptr_t)v_prefix | (uintptr_t)k_tail |
                           (uintptr_t)v_tail | (uintptr_t)workspace;
    if ((ptrs & 15) || ((ldq | ldo | prefix_head_stride | tail_slot_stride | tail_head_stride) & 7))
        return bad("operands must be 16-byte aligned, strides multiples of 8");
    const size_t R = n_seqs * rows_per_seq;
    const Space s = Space::of(workspace, R, heads, prefix_len + max_tail);
    if (!workspace || workspace_bytes < s.bytes) return bad("workspace too small (myl_attention_prefix_workspace)");
    const DeviceGuard guard(ctx->device);
    const hipStream_t st = ctx->stream;
    PrefixAttn a{};
    a.q = q; a.kp = k_prefix; a.vp = v_prefix; a.kt = k_tail; a.vt = v_tail;
    a.slots = slots; a.lens = lens; a.lut = exp_lut; a.out = out;
    a.ldq = ldq; a.ldo = ldo; a.ph = prefix_head_stride; a.ts = tail_slot_stride; a.th = tail_head_stride;
    a.mult = score_mult; a.R = (int)R; a.n = Divider::of((uint32_t)rows_per_seq); a.heads = (int)heads;
    a.G = Divider::of((uint32_t)(heads / kv_heads));
    a.P = (int)prefix_len; a.max_tail = (int)max_tail; a.n_slots = (int)n_slots; a.lcap = (int)(prefix_len + max_tail);
    a.lut_len = (uint32_t)lut_len; a.shift = score_shift; a.lut_shift = lut_shift; a.prob_frac = prob_frac;
    if (a.lcap > 0) {
        const dim3 sg((unsigned)((a.lcap + 255) / 256), (unsigned)heads, (unsigned)R);
        if (head_dim == 128) scores_kernel<128><<<sg, 256, 0, st>>>(a, s.z);
        else scores_kernel<64><<<sg, 256, 0, st>>>(a, s.z);
        probs_kernel<<<dim3((unsigned)R, (unsigned)heads), 256, 0, st>>>(a, s.z, s.p);
    }
    if (head_dim == 128) pv_kernel<128><<<dim3((unsigned)R, (unsigned)heads), 128, 0, st>>>(a, s.p);
    else pv_kernel<64><<<dim3((unsigned)R, (unsigned)heads), 64, 0, st>>>(a, s.p);
    return ctx->hip(hipGetLastError(), what);
}

}  // extern "C"
