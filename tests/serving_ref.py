"""Plain 64-bit forms of the serving operators (adapters beside a projection,
attention over a shared prefix, draft verification) on the CPU, written from
the definitions in include/myl_hip.h with numpy and Python's whole numbers.
Every output is a whole number that the definitions fix, so a comparison with
them is exact."""
from __future__ import annotations

import numpy as np

I32 = 1 << 32


def wrap32(v):
    v = np.asarray(v, np.int64) & (I32 - 1)
    return np.where(v >= I32 // 2, v - I32, v)


def rne_shift(v, s):
    """fixed_point.rs:57-71 in int64, s a scalar or an array of 0 .. 62."""
    v, s = np.broadcast_arrays(np.asarray(v, np.int64), np.asarray(s, np.int64))
    q = v >> s
    r = v - (q << s)
    half = np.where(s > 0, np.int64(1) << np.maximum(s - 1, 0), np.int64(1))
    return q + ((s > 0) & ((r > half) | ((r == half) & ((q & 1) == 1))))


def rescale(v, frac_in, frac_out):
    """fixed_point.rs:181-191: the difference as int8; a negative one shifts left."""
    d = (np.asarray(frac_in, np.int64) - np.asarray(frac_out, np.int64) + 128) % 256 - 128
    with np.errstate(over="ignore"):
        left = np.asarray(v, np.int64) << np.clip(-d, 0, 63)
    return np.where(d >= 0, rne_shift(v, np.maximum(d, 0)), left)


def clamp16(v):
    return np.clip(v, -32768, 32767)


def dots(x, w):
    """x [M x K] times w [N x K]: sums below 2^53 in any order."""
    return (x.astype(np.float64) @ w.astype(np.float64).T).astype(np.int64)


def linear(x, W, shifts, act_frac, out_frac):
    return clamp16(rescale(dots(x, W), shifts.astype(np.int64) + act_frac, out_frac))


def adapters(x, W, w_shifts, act_frac, ids, A, a_shifts, mid_frac, B, b_shifts, out_frac):
    out = linear(x, W, w_shifts, act_frac, out_frac)
    for m, a in enumerate(ids):
        if 0 <= a < A.shape[0]:
            u = linear(x[m:m + 1], A[a], a_shifts[a], act_frac, mid_frac)
            out[m] += linear(u, B[a], b_shifts[a], mid_frac, out_frac)[0]
    return clamp16(out).astype(np.int16)


def softmax_probs(z, lut, lut_shift, prob_frac):
    """softmax.rs:12-64 of one row; negative table entries count as 0."""
    L = z.size
    below = np.clip(z.max() - z, 0, 2**31 - 1)
    at = below >> lut_shift
    e = np.where(at < lut.size, np.maximum(lut.astype(np.int64), 0)[np.minimum(at, lut.size - 1)], 0)
    e = np.where(below == 0, max(0, int(lut[0])), e)
    S, one = int(e.sum()), 1 << prob_frac
    if S == 0:
        return np.full(L, one // L) + (np.arange(L) < one % L)
    p, r = (e * one) // S, (e * one) % S
    return p + ((2 * r > S) | ((2 * r == S) & (p % 2 == 1)))


def attention(q, kp, vp, kt, vt, lens, mult, shift, lut, lut_shift, prob_frac, rows_per_seq=1, slots=None, max_tail=None):
    R, H, hd = q.shape
    KH, T = kp.shape[0], kt.shape[2]
    max_tail = T if max_tail is None else max_tail
    out = np.zeros((R, H, hd), np.int16)
    for r in range(R):
        slot = r // rows_per_seq if slots is None else int(slots[r // rows_per_seq])
        n = int(lens[r])
        if n < 0:
            continue
        n = min(n, max_tail) if 0 <= slot < kt.shape[0] else 0
        for h in range(H):
            g = h // (H // KH)
            k, v = kp[g], vp[g]
            if n:
                k, v = np.concatenate([k, kt[slot, g, :n]]), np.concatenate([v, vt[slot, g, :n]])
            if not len(k):
                continue
            d = dots(q[r, h][None], k)[0]
            with np.errstate(over="ignore"):
                z = wrap32(rne_shift(d * np.int64(mult), shift & 63))
            p = softmax_probs(z, lut, lut_shift, prob_frac)
            out[r, h] = clamp16(rne_shift(dots(p[None], v.T)[0], prob_frac))
    return out


def row_weights(z, lut):
    below = (int(z.max()) - z.astype(np.int64)) << 2
    return np.where(below < lut.size, np.maximum(lut.astype(np.int64), 0)[np.minimum(below, lut.size - 1)], 0)


def verify(target, tokens, randoms, lut=None, draft=None, n_draft=None):
    B, k1, V = target.shape
    k = k1 - 1
    accepted, out = np.zeros(B, np.int32), np.full((B, k1), -1, np.int64)
    for b in range(B):
        nd = k if n_draft is None else min(max(int(n_draft[b]), 0), k)
        for i in range(nd + 1):
            row = target[b, i]
            first = int(row.argmax())
            t = int(tokens[b, i]) if i < nd else -1
            if lut is None:
                if i < nd and t == first:
                    continue
                new = first
                break
            p = row_weights(row, lut)
            w = p.astype(object)
            if i < nd:
                q = np.zeros(V, np.int64)
                if draft is not None:
                    q = row_weights(draft[b, i], lut)
                elif 0 <= t < V:
                    q[t] = 1
                P, Q = int(p.sum()), int(q.sum()) if draft is not None else 1
                if 0 <= t < V and int(randoms[b, i]) * int(q[t]) * P < int(p[t]) * Q << 64:
                    continue
                rest = np.maximum(w * Q - q.astype(object) * P, 0)
                if rest.sum() > 0:
                    w = rest
            total = int(w.sum())
            new = first
            if total:
                thr = (int(randoms[b, k]) * total) >> 64
                new = int(np.nonzero(np.cumsum(w) > thr)[0][0])
            break
        accepted[b] = i
        out[b, :i] = tokens[b, :i]
        out[b, i] = new
    return accepted, out
