// attn_fixed.h -- the two fixed-point steps that attention applies to every
// (query, key) pair, in as few 32-bit operations as their ranges allow: the
// score's rounding shift (attention.rs:66-67) and the probability's rounded
// division (softmax.rs:50-63).
#pragma once

#include "fixed.h"

// z = (i32)RNE(dot mult / 2^shift) of dot = 256 u + r (0 <= r < 256).  With
// t = shift - 8 and v = floor(dot mult / 256): w = v + 2^(t-1) shifted by t
// rounds halves up, and a half (the t bits of w and the byte below v all zero)
// goes back to the even value.  fast: |mult| < 2^23 (r mult is 32-bit), t in 1 .. 31,
// and mult >= 0 with |dot| <= 2^30 hd keeps z in 32 bits, so that z rises with dot
// and the maximum score is the score of the maximum dot.
struct ScoreScale {
    int32_t mult;
    uint32_t t, mask, fast;
    int32_t half;
    MYL_FN ScoreScale of(int64_t mult, uint8_t shift, int hd) {
        bool ok = mult >= 0 && mult < (1 << 23) && shift >= 9 && shift <= 39;
        ok = ok && ((((uint64_t)hd << 30) * (uint64_t)mult >> shift) < (1ull << 31) - 1);
        const uint32_t t = ok ? (uint32_t)shift - 8u : 1u;
        return ScoreScale{ok ? (int32_t)mult : 0, t, (1u << t) - 1u, ok ? 1u : 0u, (int32_t)(1u << (t - 1))};
    }
    MYL_MEM int32_t operator()(int32_t u, uint32_t r) const {
#if defined(__HIP_DEVICE_COMPILE__)
        const int32_t rm = __mul24((int32_t)r, mult);
#else
        const int32_t rm = (int32_t)r * mult;
#endif
        const int64_t w = (int64_t)u * mult + (int64_t)(uint64_t)(((uint32_t)rm >> 8) + (uint32_t)half);
        const uint32_t lo = (uint32_t)w, hi = (uint32_t)((uint64_t)w >> 32);
#if defined(__HIP_DEVICE_COMPILE__)
        const uint32_t z = __builtin_amdgcn_alignbit(hi, lo, t);
#else
        const uint32_t z = (uint32_t)((((uint64_t)hi << 32) | lo) >> t);
#endif
        return (int32_t)(((lo & mask) | ((uint32_t)rm & 255u)) == 0 ? z & ~1u : z);
    }
};

// RNE(e 2^f / S) for 0 <= e < 2^15, f <= 14 and 1 <= S < 2^31.  With l =
// ceil(log2 S), K = 16 + l and m = ceil(2^(K+f) / S),
//   e m / 2^K = e 2^f / S + d,  0 <= d < e / 2^K < 2^-(1+l) <= 1 / (2 S),
// and e 2^f / S + 1/2 is a whole number or at least 1 / (2 S) below the next, so
// P = e m + 2^(K-1) has the quotient rounded half up above bit K.  Below it, the
// remainder is less than 2^15 at a tie and at least 2^K / (2 S) >= 2^15
// elsewhere; a tie goes back to the even value.  One 32 x 32 + 64-bit multiply-add
// and no division or correction step.  S > 2^30: e 2^f < S / 2, the result is 0 (m = 0).
struct ProbDiv {
    uint32_t m, half_hi, half_lo, up;  // 2^(K-1); up = l + 1 = K - 15
    MYL_FN ProbDiv of(uint32_t s, uint32_t f) {
        uint32_t l = s <= 1 ? 0u : 32u - (uint32_t)__builtin_clz(s - 1u), m = 0;
        if (l < 31) {
            uint32_t q = 1, r = (1u << l) - s;  // 2^(l-1) < s <= 2^l
            for (uint32_t i = 0; i < 16u + f; ++i) {
                r <<= 1;
                const bool take = r >= s;
                r -= take ? s : 0u;
                q = (q << 1) | (take ? 1u : 0u);
            }
            m = q + (r ? 1u : 0u);
        } else {
            l = 30;
        }
        const uint64_t half = 1ull << (15 + l);
        return ProbDiv{m, (uint32_t)(half >> 32), (uint32_t)half, l + 1u};
    }
    MYL_MEM uint32_t operator()(uint32_t e) const {
        const uint64_t p = (uint64_t)e * m + (((uint64_t)half_hi << 32) | half_lo);
#if defined(__HIP_DEVICE_COMPILE__)
        const uint32_t x = __builtin_amdgcn_alignbit((uint32_t)(p >> 32), (uint32_t)p, 15);
#else
        const uint32_t x = (uint32_t)(p >> 15);
#endif
        const uint32_t q = x >> up;
        return (x & ((1u << up) - 1u)) == 0 ? q & ~1u : q;
    }
};
