"""Plain 64-bit forms of the operators over a paged cache (appending, attention) and of
the log probabilities on the CPU, written from the definitions in include/myl_hip.h
with numpy and Python's whole numbers.  Every output is a whole number that the
definitions fix, so a comparison with them is exact."""
from __future__ import annotations

import numpy as np

import serving_ref as ref

LN2_Q30 = 744261118


def place(tables, seq, pos, page, n_pages):
    """(page id, place in it) of a sequence's position, or None."""
    if pos // page >= tables.shape[1]:
        return None
    i = int(tables[seq, pos // page])
    return (i, pos % page) if 0 <= i < n_pages else None


# ---- appending ------------------------------------------------------------------

def bias_of(b, shift, frac):
    """rescale of an int16 bias (fixed_point.rs:173-191) for differences of -31 .. 31."""
    d = shift.astype(np.int64) - frac
    return np.where(d >= 0, ref.rne_shift(b, np.maximum(d, 0)), ref.wrap32(b.astype(np.int64) << np.maximum(-d, 0)))


def wrap128(v):
    v &= (1 << 128) - 1
    return v - (1 << 128) if v >> 127 else v


def rne_shift128(v, s):
    """fixed_point.rs:155-169: shift amounts count modulo 128."""
    if s == 0:
        return v
    mask, half = wrap128(1 << (s & 127)) - 1, wrap128(1 << ((s - 1) & 127))
    q, r = v >> (s & 127), v & mask
    return q + (r > half or (r == half and q & 1))


def head_norm(x, gamma, shifts, n):
    """rmsnorm (rmsnorm.rs:61-161) of one head with equal input scales."""
    total = int((x.astype(np.int64) ** 2).sum())
    if total == 0:
        return np.zeros_like(x)
    most, mean, q = n["rsqrt"].size - 1, total * n["inv_n_q20"] >> 20, 0
    while mean >> q > most:
        q += 2
    at = min(int(ref.rne_shift(mean, q)), most)
    down = n["lut_output_frac"] + n["lut_input_shift"] // 2 + q // 2 + shifts.astype(np.int64) - n["out_frac"]
    p = x.astype(np.int64) * gamma * int(n["rsqrt"][at])
    return ref.clamp16(np.array([max(min(rne_shift128(a, d) if d >= 0 else wrap128(a << (-d & 127)), 2**31), -2**31)
                                 for a, d in zip(p.tolist(), down.tolist())]))


def rotate(x, c, s, frac):
    """rope (rope.rs:17-59) of one head."""
    half = x.size // 2
    a, b = x[:half].astype(np.int64), x[half:].astype(np.int64)
    c, s = c.astype(np.int64), s.astype(np.int64)
    turn = lambda v: ref.clamp16(ref.rne_shift(ref.wrap32(v), frac))
    return np.concatenate([turn(a * c - b * s), turn(b * c + a * s)])


def append(q, k, v, positions, kp, vp, tables, cos, sin, rope_frac, q_out, seqs=None, bias=None, bias_shifts=None, fracs=(10, 10, 10),
           norm=None, page_at=2):
    """q_out and the pages ([pages][heads][positions], position axis page_at) after the call."""
    R, H, hd = q.shape
    KH, page = k.shape[1], kp.shape[page_at]
    q_out, kp, vp = q_out.copy(), kp.copy(), vp.copy()
    for r in range(R):
        pos, seq = int(positions[r]), r if seqs is None else int(seqs[r])
        if pos < 0 or not 0 <= seq < tables.shape[0]:
            continue
        to = place(tables, seq, pos, page, kp.shape[0])
        turn = pos % cos.shape[0]
        for part, x, at in ((0, q, 0), (1, k, H), (2, v, H + KH)):
            for h in range(x.shape[1]):
                y = x[r, h].astype(np.int64)
                if bias is not None:
                    w = slice((at + h) * hd, (at + h + 1) * hd)
                    y = ref.clamp16(y + bias_of(bias[w], bias_shifts[w], fracs[part]))
                if norm is not None and part < 2 and norm["gamma"][part] is not None:
                    y = head_norm(y, norm["gamma"][part].astype(np.int64), norm["shifts"][part], dict(norm, out_frac=norm["out_fracs"][part]))
                if part < 2:
                    y = rotate(y, cos[turn], sin[turn], rope_frac)
                if part == 0:
                    q_out[r, h] = y
                elif to is not None:
                    pages = kp if part == 1 else vp
                    pages[(to[0], h, to[1]) if page_at == 2 else (to[0], to[1], h)] = y
    return q_out, kp, vp


# ---- attention ------------------------------------------------------------------

def attention(q, kp, vp, tables, lens, mult, shift, lut, lut_shift, prob_frac, rows_per_seq=1, max_len=None):
    """Pages [pages][heads][positions][dims]."""
    R, H, hd = q.shape
    n_pages, KH, page = kp.shape[:3]
    max_len = tables.shape[1] * page if max_len is None else max_len
    out = np.zeros((R, H, hd), np.int16)
    for r in range(R):
        L = min(max(int(lens[r]), 0), max_len)
        j = np.arange(L)
        ids = tables[r // rows_per_seq, j // page].astype(np.int64)
        j, ids = j[(ids >= 0) & (ids < n_pages)], ids[(ids >= 0) & (ids < n_pages)]
        if not j.size:
            continue
        for g in range(KH):
            k, v = kp[ids, g, j % page], vp[ids, g, j % page]
            heads = slice(g * (H // KH), (g + 1) * (H // KH))
            for h, d in zip(range(heads.start, heads.stop), ref.dots(q[r, heads], k)):
                with np.errstate(over="ignore"):
                    z = ref.wrap32(ref.rne_shift(d * np.int64(mult), shift & 63))
                p = ref.softmax_probs(z, lut, lut_shift & 31, prob_frac)  # shift amounts count modulo 32
                out[r, h] = ref.clamp16(ref.rne_shift(ref.dots(p[None], v.T)[0], prob_frac))
    return out


# ---- log probabilities ------------------------------------------------------------

def ln_q16(S):
    """ln(S / 2^14) in Q16 (csrc/fixed.h)."""
    e = S.bit_length() - 1
    x, f = S << (62 - e), 0
    for _ in range(16):
        x = x * x >> 62
        f *= 2
        if x >= 1 << 63:
            x >>= 1
            f += 1
    return half_even(((e - 14) * 65536 + f) * LN2_Q30, 1 << 30)


def half_even(num, den):
    q, r = divmod(num, den)
    return q + (2 * r > den or (2 * r == den and q % 2 == 1))


def logprobs(z, tokens, lut, top_n):
    R, V = z.shape
    many = tokens.reshape(R, -1)
    logp, entropy = np.zeros(many.shape, np.int64), np.zeros(R, np.int64)
    tops, toplp = np.zeros((R, top_n), np.int64), np.zeros((R, top_n), np.int64)
    for r in range(R):
        m, row = int(z[r].max()), z[r].astype(np.int64)
        w = ref.row_weights(z[r], lut)
        S = int(w.sum())
        moment = int((w * np.where(w > 0, m - row, 0)).sum())
        ln = ln_q16(max(S, 1))
        entropy[r] = ln + half_even(moment << 10, S) if S else 0
        for i, t in enumerate(many[r].tolist()):
            logp[r, i] = (int(row[t]) - m) * 1024 - ln if 0 <= t < V else 0
        order = np.lexsort((np.arange(V), -row))[:top_n]
        tops[r], toplp[r] = order, (row[order] - m) * 1024 - ln
    return logp.reshape(tokens.shape), entropy, tops, toplp
