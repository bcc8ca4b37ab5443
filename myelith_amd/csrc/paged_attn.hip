// paged_attn.hip -- integer attention (attention.rs:42-90 with softmax.rs:12-64) of each
// sequence's newest rows over a paged cache: myl_attention_paged_dev.
#include "abi_internal.h"
#include "attn_fixed.h"
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
    int32_t* z;  // [pair][keys]; pair = row * heads + head
    size_t ldq, ldo, ldt, page_stride, head_stride, pos_stride;
    int64_t mult;
    SmallDiv n, G, page;
    int heads, max_len, n_pages, keys;
    uint32_t lut_len;
    uint8_t shift, lut_shift, prob_frac;
};

// The keys of row r, counted from position 0: at most max_len and what the table names.
__device__ inline int keys_of(const PagedAttn& a, int r) { return min(max(a.lens[r], 0), a.max_len); }

// The element offset of a position's vector in the pages, or -1: no such page.
__device__ inline int64_t place_of(const PagedAttn& a, int seq, int pos) {
    int off;
    const int at = divmod(a.page, pos, off), id = a.tables[(size_t)seq * a.ldt + at];
    return id < 0 || id >= a.n_pages ? -1 : (int64_t)((size_t)id * a.page_stride + (size_t)off * a.pos_stride);
}

// A block per (row, head).
template <int HD>
__global__ __launch_bounds__(256) void paged_simple_kernel(PagedAttn a) {
    __shared__ int32_t red[4];
    __shared__ uint32_t s_extra[2];
    __shared__ int16_t qs[HD];
    int rem;
    const int row = blockIdx.y, head = blockIdx.x, tid = threadIdx.x;
    const int seq = divmod(a.n, row, rem), g = divmod(a.G, head, rem);
    const int L = keys_of(a, row);
    int32_t* z = a.z + ((size_t)row * a.heads + head) * a.keys;
    if (tid < HD) qs[tid] = a.q[(size_t)row * a.ldq + (size_t)head * HD + tid];
    __syncthreads();
    int32_t mx = INT32_MIN, count = 0;
    for (int j = tid; j < L; j += 256) {
        const int64_t at = place_of(a, seq, j);
        if (at < 0) continue;
        const int16_t* k = a.kp + at + (size_t)g * a.head_stride;
        uint64_t acc = 0;
        for (int d = 0; d < HD; ++d) acc += (uint64_t)((int64_t)qs[d] * (int64_t)k[d]);
        z[j] = (int32_t)rshift_round64(wmul64((int64_t)acc, a.mult), a.shift);
        mx = max(mx, z[j]);
        ++count;
    }
    mx = block_max_i32(mx, red);
    const uint32_t n = block_sum_u32((uint32_t)count, (uint32_t*)red);
    uint32_t s = 0;
    for (int j = tid; j < L; j += 256) {
        uint32_t e = 0;
        if (place_of(a, seq, j) >= 0) {
            const uint32_t i = min((uint32_t)mx - (uint32_t)z[j], 0x7FFFFFFFu) >> (a.lut_shift & 31u);
            e = i < a.lut_len ? (uint32_t)max((int32_t)a.lut[i], 0) : 0u;
        }
        z[j] = (int32_t)e;
        s += e;
    }
    s = block_sum_u32(s, (uint32_t*)red);
    if (tid == 0 && n) udivmod32(1u << a.prob_frac, n, recip32(n), &s_extra[0], &s_extra[1]);
    __syncthreads();
    if (tid >= HD) return;
    const ProbDiv div = ProbDiv::of(s ? s : 1u, a.prob_frac);
    int64_t acc = 0;
    uint32_t seen = 0;
    for (int j = 0; j < L; ++j) {
        const int64_t at = place_of(a, seq, j);
        if (at < 0) continue;
        const uint32_t p = s ? div((uint32_t)z[j]) : s_extra[0] + (seen < s_extra[1] ? 1u : 0u);
        ++seen;
        acc += (int64_t)p * a.vp[at + (size_t)g * a.head_stride + tid];
    }
    a.out[(size_t)row * a.ldo + (size_t)head * HD + tid] = clamp_i16_i64(rshift_round64(acc, a.prob_frac));
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
    a.ldq = ldq; a.ldo = ldo; a.ldt = table_stride; a.page_stride = page_stride; a.head_stride = head_stride; a.pos_stride = pos_stride;
    a.mult = score_mult;
    a.n = SmallDiv::of(rows_per_seq); a.G = SmallDiv::of(heads / kv_heads); a.page = SmallDiv::of(page_size);
    a.heads = (int)heads; a.max_len = (int)max_len; a.n_pages = (int)n_pages; a.keys = pl.keys;
    a.lut_len = (uint32_t)lut_len; a.shift = score_shift; a.lut_shift = lut_shift; a.prob_frac = prob_frac;
    const dim3 grid((unsigned)heads, (unsigned)(n_seqs * rows_per_seq));
    if (head_dim == 128) paged_simple_kernel<128><<<grid, 256, 0, ctx->stream>>>(a);
    else paged_simple_kernel<64><<<grid, 256, 0, ctx->stream>>>(a);
    return ctx->hip(hipGetLastError(), what);
}

}  // extern "C"
