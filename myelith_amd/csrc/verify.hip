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
#include "abi_internal.h"
#include "ops.h"
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
    int B, k, V;
    uint32_t lut_len;
};

struct RowStat {
    int32_t m, at;  // the maximum, its first index
    uint64_t s;     // the sum of the weights
};

__device__ inline uint32_t weight(const Verify& a, int32_t m, int32_t z) {
    const uint64_t i = (uint64_t)((int64_t)m - (int64_t)z) << (MYL_TV_EXP_INPUT_FRAC - MYL_TV_LOGIT_FRAC_BITS);
    return i < a.lut_len ? (uint32_t)max(0, (int32_t)a.lut[i]) : 0u;
}

__device__ inline uint64_t max_key(int32_t v, uint32_t idx) {  // by value, then by the smaller index
    return ((uint64_t)((uint32_t)v ^ 0x80000000u) << 32) | (uint64_t)(0xFFFFFFFFu - idx);
}

// Row blockIdx.x: the target's B (k + 1) rows, then the draft's B k.
__global__ __launch_bounds__(1024) void verify_rows_kernel(Verify a, RowStat* __restrict__ stat) {
    __shared__ uint64_t red[16];
    __shared__ uint64_t reds[16];
    const int T = a.B * (a.k + 1), r = blockIdx.x, tid = threadIdx.x;
    const int32_t* z = r < T ? a.target + (size_t)r * a.ldt : a.draft + (size_t)(r - T) * a.ldd;
    uint64_t key = 0;
    for (int i = tid; i < a.V; i += 1024) {
        const uint64_t o = max_key(z[i], (uint32_t)i);
        key = o > key ? o : key;
    }
    key = wave_max_u64(key);
    if ((tid & 63) == 0) red[tid >> 6] = key;
    __syncthreads();
    key = wave_max_u64((tid & 63) < 16 ? red[tid & 63] : 0);
    const int32_t m = (int32_t)((uint32_t)(key >> 32) ^ 0x80000000u);
    uint64_t s = 0;
    if (a.lut)
        for (int i = tid; i < a.V; i += 1024) s += weight(a, m, z[i]);
    s = wave_sum_u64(s);
    if ((tid & 63) == 0) reds[tid >> 6] = s;
    __syncthreads();
    s = wave_sum_u64((tid & 63) < 16 ? reds[tid & 63] : 0);
    if (tid == 0) stat[r] = RowStat{m, (int32_t)(0xFFFFFFFFu - (uint32_t)key), s};
}

// How a sequence's drafts end: the accepted ones, and the weights of the next
// token, w_j = max(0, p_j Q - q_j P) (q_j = 0 where qrow is null, but 1 at `not_j`).
struct Ending {
    int n;
    const int32_t *prow, *qrow;
    int32_t pm, qm, at;
    uint64_t P, Q;
    int64_t not_j;
};

__device__ inline Ending verify_ending(const Verify& a, const RowStat* __restrict__ stat, int b) {
    const int T = a.B * (a.k + 1);
    const int nd = a.n_draft ? min(max(a.n_draft[b], 0), a.k) : a.k;
    Ending e{};
    e.not_j = -1;
    for (;; ++e.n) {
        const int tr = b * (a.k + 1) + e.n, dr = b * a.k + e.n;
        const RowStat p = stat[tr];
        e.prow = a.target + (size_t)tr * a.ldt;
        e.pm = p.m;
        e.at = p.at;
        e.P = p.s;
        e.Q = 1;
        if (e.n == nd) break;
        const int64_t t = a.tokens[dr];
        const bool in = t >= 0 && t < a.V;
        if (!a.lut) {
            if (t == (int64_t)p.at) continue;
            break;
        }
        uint64_t qt = in ? 1 : 0;
        const int32_t* qrow = nullptr;
        RowStat q{};
        if (a.draft) {
            q = stat[T + dr];
            qrow = a.draft + (size_t)dr * a.ldd;
            qt = in ? weight(a, q.m, qrow[t]) : 0;
            e.Q = q.s;
        }
        if (in && __umul64hi(a.randoms[(size_t)b * (a.k + 1) + e.n], qt * p.s) < weight(a, p.m, e.prow[t]) * e.Q) continue;
        e.qrow = qrow;
        e.qm = q.m;
        if (!a.draft) e.not_j = in ? t : -1;
        break;
    }
    return e;
}

__device__ inline uint64_t ending_weight(const Verify& a, const Ending& e, int j) {
    const uint64_t p = weight(a, e.pm, e.prow[j]);
    if (p == 0 || j == e.not_j) return 0;
    const uint64_t x = p * e.Q;
    const uint64_t y = e.qrow ? weight(a, e.qm, e.qrow[j]) * e.P : 0;
    return x > y ? x - y : 0;
}

__device__ inline uint64_t shfl_up_u64(uint64_t v, int d) {
    const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)v, d, 64);
    const uint32_t hi = (uint32_t)__shfl_up((int)(uint32_t)(v >> 32), d, 64);
    return ((uint64_t)hi << 32) | lo;
}

__global__ __launch_bounds__(1024) void verify_pick_kernel(Verify a, const RowStat* __restrict__ stat) {
    __shared__ uint64_t wt[2][16];
    __shared__ myl_u128 red[1024];
    __shared__ int s_pick;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    Ending e = verify_ending(a, stat, b);
    int64_t pick = a.lut ? -1 : e.at;
    for (int again = 0; a.lut && again < 2; ++again) {
        myl_u128 part = 0;
        for (int j = tid; j < a.V; j += 1024) part += ending_weight(a, e, j);
        const myl_u128 W = (myl_u128)block_sum_i128((myl_i128)part, (myl_i128*)red);
        if (W == 0) {  // the residual leaves nothing: the target's own weights
            if (again == 1 || e.P == 0) {
                pick = e.at;
                break;
            }
            e.qrow = nullptr;
            e.not_j = -1;
            e.Q = 1;
            __syncthreads();
            continue;
        }
        const uint64_t r = a.randoms[(size_t)b * (a.k + 1) + a.k];
        const myl_u128 thr = (myl_u128)r * (uint64_t)(W >> 64) + __umul64hi(r, (uint64_t)W);
        myl_u128 base = 0;
        if (tid == 0) s_pick = a.V;
        for (int j0 = 0; j0 < a.V; j0 += 1024) {
            const int j = j0 + tid;
            const uint64_t own = j < a.V ? ending_weight(a, e, j) : 0;
            uint64_t inc = own;
            for (int d = 1; d < 64; d <<= 1) {
                const uint64_t o = shfl_up_u64(inc, d);
                if (lane >= d) inc += o;
            }
            if (lane == 63) wt[(j0 >> 10) & 1][w] = inc;
            __syncthreads();
            uint64_t before = 0, all = 0;
            for (int k = 0; k < 16; ++k) {
                const uint64_t t = wt[(j0 >> 10) & 1][k];
                before += k < w ? t : 0;
                all += t;
            }
            if (thr < base + all) {
                if (j < a.V && thr < base + before + inc) atomicMin(&s_pick, j);
                __syncthreads();
                break;
            }
            base += all;
        }
        pick = s_pick;
        break;
    }
    if (tid == 0) a.accepted[b] = e.n;
    for (int i = tid; i <= a.k; i += 1024)
        a.out[(size_t)b * (a.k + 1) + i] = i < e.n ? a.tokens[(size_t)b * a.k + i] : (i == e.n ? pick : -1);
}

constexpr size_t kMaxVocab = (size_t)1 << 20;

struct Space {
    RowStat* stat;
    size_t bytes;
    static Space of(void* base, size_t B, size_t k) {
        Carve c{(char*)base};
        Space s;
        s.stat = c.take<RowStat>(B * (2 * k + 1));
        s.bytes = c.used ? c.used : 256;  // 0 stands for sizes that a call refuses
        return s;
    }
};

}  // namespace
}  // namespace myl

using namespace myl;

extern "C" {

size_t myl_verify_drafts_workspace(const myl_ctx* ctx, size_t n_seqs, size_t k, size_t vocab, size_t lut_len) {
    if (!ctx || !fits_int(n_seqs) || k > 1024 || !fits_int(n_seqs * (2 * k + 1)) || vocab > kMaxVocab) return 0;
    (void)lut_len;
    return Space::of(nullptr, n_seqs, k).bytes;
}

int myl_verify_drafts_dev(myl_ctx* ctx, const int32_t* target, size_t ldt, const int32_t* draft, size_t ldd, size_t n_seqs,
                          size_t k, size_t vocab, const int64_t* tokens, const int32_t* n_draft, const uint64_t* randoms,
                          const int16_t* exp_lut, size_t lut_len, int32_t* accepted, int64_t* out, void* workspace,
                          size_t workspace_bytes) {
    if (!ctx) return MYL_E_INVALID;
    const char* what = "verify_drafts_dev";
    auto bad = [&](const char* why) { return ctx->fail(MYL_E_INVALID, std::string(what) + ": " + why); };
    if (vocab == 0 || vocab > kMaxVocab) return bad("the vocabulary must hold 1 to 2^20 tokens");
    if (ldt < vocab || (draft && ldd < vocab)) return bad("leading dimension too small");
    if (k > 1024 || !fits_int(n_seqs) || !fits_int(n_seqs * (2 * k + 1)) || !fits_int(ldt) || !fits_int(ldd))
        return bad("too many drafts, sequences or logits");
    if (exp_lut && (lut_len == 0 || lut_len > 32768)) return bad("the exp table must hold 1 to 32768 entries");
    if (n_seqs == 0) return MYL_OK;
    if (!target || !accepted || !out || (k && !tokens) || (exp_lut && !randoms)) return bad("null operand");
    const Space s = Space::of(workspace, n_seqs, k);
    if (!workspace || workspace_bytes < s.bytes) return bad("workspace too small (myl_verify_drafts_workspace)");
    if ((uintptr_t)workspace & 15) return bad("workspace must be 16-byte aligned");
    const DeviceGuard guard(ctx->device);
    Verify a{};
    a.target = target; a.draft = exp_lut ? draft : nullptr; a.tokens = tokens; a.n_draft = n_draft; a.randoms = randoms;
    a.lut = exp_lut; a.accepted = accepted; a.out = out; a.ldt = ldt; a.ldd = ldd;
    a.B = (int)n_seqs; a.k = (int)k; a.V = (int)vocab; a.lut_len = (uint32_t)lut_len;
    const int rows = a.B * (a.k + 1) + (a.draft ? a.B * a.k : 0);
    verify_rows_kernel<<<rows, 1024, 0, ctx->stream>>>(a, s.stat);
    verify_pick_kernel<<<a.B, 1024, 0, ctx->stream>>>(a, s.stat);
    return ctx->hip(hipGetLastError(), what);
}

}  // extern "C"
