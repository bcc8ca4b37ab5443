"""What is measured of the operators of a serving step: many requests that share
a system prompt, carry their own adapters and check drafted tokens.

  adapters   `linear_w8a16_adapters_dev`: a W8A16 projection of M rows with the
             low-rank adapter of each row's request added to it
  attention  `attention_prefix_dev`: integer attention of a batch whose sequences
             attend one shared prefix and then their own tails
  verify     `verify_drafts_dev`: drafted tokens checked against the target's
             probabilities with given random numbers

Every output is a whole number that the fixed-point definitions fix bit for bit.
`own` false computes them with elementary torch operations: whole numbers below
2^53 in float64 products, everything else in int64.
"""
from __future__ import annotations

import math

import torch

own = False

# (N, K) of the projections of the Qwen2.5-0.5B and -7B layouts: q/k/v, o_proj, gate (or up), down.
PROJECTIONS = [(1152, 896), (896, 896), (4864, 896), (896, 4864),
               (4608, 3584), (3584, 3584), (18944, 3584), (3584, 18944)]
HEADS = {"7b": (28, 4, 128), "0.5b": (14, 2, 64)}  # query heads, KV heads, head size
V7, V05 = 152064, 151936

# the fixed-point formats of the layers: Q10 activations, Q14 scores and probabilities
ACT_FRAC, OUT_FRAC, MID_FRAC = 10, 10, 10
Q_FRAC, K_FRAC, SCORE_FRAC, PROB_FRAC = 10, 10, 14, 14
SCORE_SHIFT = Q_FRAC + K_FRAC + 15 - SCORE_FRAC
LUT_SHIFT = SCORE_FRAC - 8


def listed():
    return [
        # one request alone through the smallest projection: launches and latency count
        dict(name="adapters_m1_small", kind="adapters", M=1, N=896, K=896, rank=8, n=3, order="mixed"),
        # a decode batch of 24 requests with an adapter each through q/k/v
        dict(name="adapters_m24_qkv", kind="adapters", M=24, N=4608, K=3584, rank=16, n=24, order="mixed"),
        # a larger batch with wide adapters through the long down projection, odd row count
        dict(name="adapters_m61_down", kind="adapters", M=61, N=3584, K=18944, rank=64, n=32, order="mixed"),
        # the prompts of five requests in one chunk through a gate projection
        dict(name="adapters_m2003_gate", kind="adapters", M=2003, N=18944, K=3584, rank=16, n=5, order="runs"),
        # two chats shortly after a short system prompt: latency
        dict(name="attention_2x131", kind="attention", arch="0.5b", seqs=2, rows=1, prefix=131, tail=20),
        # a decode batch behind a system prompt, every chat some hundred tokens in
        dict(name="attention_24x2000", kind="attention", arch="7b", seqs=24, rows=1, prefix=2000, tail=500),
        # five drafted rows per request behind a long document
        dict(name="attention_16x5x8001", kind="attention", arch="7b", seqs=16, rows=5, prefix=8001, tail=777),
        # a large batch behind a very long shared context
        dict(name="attention_64x30000", kind="attention", arch="7b", seqs=64, rows=1, prefix=30000, tail=2000),
        # one request, four drafted tokens, a small vocabulary: latency
        dict(name="verify_1x4_small", kind="verify", B=1, k=4, V=32001, mode="draft", ragged=False),
        # a serving batch with a draft model, some requests with fewer drafts than others
        dict(name="verify_24x5", kind="verify", B=24, k=5, V=V7, mode="draft", ragged=True),
        # drafts looked up in the prompt: no draft probabilities
        dict(name="verify_16x8_lookup", kind="verify", B=16, k=8, V=V05, mode="lookup", ragged=True),
        # greedy decoding with drafts
        dict(name="verify_32x4_greedy", kind="verify", B=32, k=4, V=V7, mode="greedy", ragged=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["adapters", "attention", "verify"])
    if kind == "adapters":
        N, K = rng.choice(PROJECTIONS)
        if rng.random() < 0.3:
            N -= rng.randrange(1, 64)  # a shard or a pruned projection: any row count
        M = _log(rng, 1, 2000)
        return dict(kind=kind, M=M, N=N, K=K, rank=rng.choice([4, 8, 16, 16, 24, 32, 64]), n=_log(rng, 1, 64),
                    order="runs" if M > 100 and rng.random() < 0.8 else "mixed")
    if kind == "attention":
        arch = rng.choice(list(HEADS))
        seqs, rows = _log(rng, 1, 64), rng.choice([1, 1, 1, rng.randrange(2, 9)])
        most = min(30000, 64 * 30000 // (seqs * rows))
        return dict(kind=kind, arch=arch, seqs=seqs, rows=rows, prefix=_log(rng, 16, most), tail=_log(rng, 1, 2000))
    B, V = _log(rng, 1, 64), rng.choice([V7, V05, 32001])
    k = rng.randrange(1, 9)
    while B * (2 * k + 1) > 288:
        k -= 1
    return dict(kind=kind, B=B, k=k, V=V, mode=rng.choice(["draft", "draft", "lookup", "greedy"]), ragged=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _gauss16(shape, g, sigma):
    x = torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).mul_(sigma)
    return x.round_().clamp_(-32767, 32767).to(torch.int16)


def _int8(shape, g):
    return torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=g)


def _shifts(shape, lo, g):
    return torch.randint(lo, lo + 2, shape, dtype=torch.uint8, device="cuda", generator=g)


def exp_table():
    """round(exp(-i / 2^8) 2^14) up to its last entry that is not zero."""
    t = [round(math.exp(-i / 256.0) * 16384) for i in range(16385)]
    while not t[-1]:
        t.pop()
    return torch.tensor(t, dtype=torch.int16, device="cuda")


def _growth(k):
    """log2 of the sums' deviation over the inputs', k products with uniform int8."""
    return int(math.log2(73.0 * math.sqrt(k)))


def _adapters(case, seed):
    """Gaussian activations of deviation 2000, uniform int8 weights and scales
    that keep activations of that size; an adapter adds about a quarter of it.
    Every ninth row on average belongs to a request without an adapter."""
    g = _gen(seed)
    M, N, K, r, n = (case[c] for c in ("M", "N", "K", "rank", "n"))
    s = dict(x=_gauss16((M, K), g, 2000), W=_int8((N, K), g), w_shifts=_shifts((N,), _growth(K), g),
             A=_int8((n, r, K), g), a_shifts=_shifts((n, r), _growth(K), g),
             B=_int8((n, N, r), g), b_shifts=_shifts((n, N), _growth(r) + 2, g))
    ids = torch.randint(0, n, (M,), dtype=torch.int32, device="cuda", generator=g)
    if case["order"] == "runs":  # the rows of a request follow one another
        ids = ids.sort().values
    elif M > 1:
        ids = torch.where(torch.rand(M, device="cuda", generator=g) < 1 / 9, torch.full_like(ids, -1), ids)
    s["ids"] = ids
    return s


def _attention(case, seed):
    """Post-RoPE q and k of deviation 2 and 1 (scores of deviation 2), tails of
    any length; row i of a request attends up to its own drafted position.  In
    a batch of more than four the last request's rows are padding."""
    g = _gen(seed)
    H, KH, hd = HEADS[case["arch"]]
    S, n, P, T = case["seqs"], case["rows"], case["prefix"], case["tail"] + case["rows"]
    s = dict(q=_gauss16((S * n, H, hd), g, 2048), kp=_gauss16((KH, P, hd), g, 1024), vp=_gauss16((KH, P, hd), g, 2000),
             kt=_gauss16((S, KH, T, hd), g, 1024), vt=_gauss16((S, KH, T, hd), g, 2000), lut=exp_table(),
             mult=round(2 ** 15 / math.sqrt(hd)))
    base = torch.randint(0, case["tail"] + 1, (S, 1), dtype=torch.int32, device="cuda", generator=g)
    lens = base + 1 + torch.arange(n, dtype=torch.int32, device="cuda")
    if S > 4:
        lens[-1] = -1
    s["lens"] = lens.reshape(-1)
    s["slots"] = torch.randperm(S, device="cuda", generator=g).to(torch.int32)
    return s


def _verify(case, seed):
    """Q6 logits: Gaussian of deviation 2.5 with some likely tokens a row; the
    draft model's differ a little from the target's, drafted tokens follow it."""
    g = _gen(seed)
    B, k, V = case["B"], case["k"], case["V"]
    z = torch.randn((B, k + 1, V), device="cuda", generator=g).mul_(160)
    top = torch.randint(0, V, (B, k + 1, 8), device="cuda", generator=g)
    z.scatter_(2, top, torch.randint(700, 1400, top.shape, device="cuda", generator=g).float())
    z = z.round_().to(torch.int32)
    d = z[:, :k].clone()
    near = d.gather(2, top[:, :k])
    d.scatter_(2, top[:, :k], near + torch.randint(-60, 61, near.shape, dtype=torch.int32, device="cuda", generator=g))
    u = torch.rand((B, k, 8), device="cuda", generator=g).clamp_min_(1e-6)
    pick = (d.gather(2, top[:, :k]).float() / 64 - torch.log(-torch.log(u))).argmax(2, keepdim=True)
    tokens = top[:, :k].gather(2, pick).squeeze(2)
    if case["mode"] == "greedy":  # drafts that are mostly the target's choice
        right = torch.rand((B, k), device="cuda", generator=g) < 0.8
        tokens = torch.where(right, z[:, :k].argmax(2), tokens)
    s = dict(target=z, draft=d.contiguous() if case["mode"] == "draft" else None, tokens=tokens.contiguous(),
             randoms=torch.randint(-2 ** 63, 2 ** 63 - 1, (B, k + 1), dtype=torch.int64, device="cuda", generator=g),
             lut=None if case["mode"] == "greedy" else exp_table(), n_draft=None)
    if case["ragged"]:
        s["n_draft"] = torch.randint(0, k + 1, (B,), dtype=torch.int32, device="cuda", generator=g)
    return s


_INPUTS = {"adapters": _adapters, "attention": _attention, "verify": _verify}
_BACKEND = None


def backend():
    """One context per process on torch's stream, as a serving program keeps it."""
    global _BACKEND
    if _BACKEND is None:
        from myelith_amd.backend import RocmBackend
        _BACKEND = RocmBackend(0)
        _BACKEND.use_torch_stream()
    return _BACKEND


def prepare(case, seed):
    s = dict(case, **_INPUTS[case["kind"]](case, seed))
    if own:  # the outputs and the workspace that a serving program keeps from step to step
        be = s["be"] = backend()
        if case["kind"] == "adapters":
            s["out"] = torch.empty((case["M"], case["N"]), dtype=torch.int16, device="cuda")
            s["ws"] = be.linear_w8a16_adapters_workspace(s["x"], s["W"], s["A"])
        elif case["kind"] == "attention":
            s["out"] = torch.empty_like(s["q"])
            s["ws"] = be.attention_prefix_workspace(s["q"], s["kp"], s["kt"], rows_per_seq=case["rows"])
        else:
            s["out"] = torch.empty((case["B"], case["k"] + 1), dtype=torch.int64, device="cuda")
            s["accepted"] = torch.empty(case["B"], dtype=torch.int32, device="cuda")
            s["ws"] = be.verify_drafts_workspace(s["target"], s["lut"], s["draft"])
    torch.cuda.synchronize()
    return s


def run(s):
    if not own:
        return _PLAIN[s["kind"]](s)
    be = s["be"]
    if s["kind"] == "adapters":
        return be.linear_w8a16_adapters_dev(s["x"], s["W"], s["w_shifts"], ACT_FRAC, s["ids"], s["A"], s["a_shifts"],
                                            MID_FRAC, s["B"], s["b_shifts"], OUT_FRAC, out=s["out"], workspace=s["ws"])
    if s["kind"] == "attention":
        return be.attention_prefix_dev(s["q"], s["kp"], s["vp"], s["kt"], s["vt"], s["lens"], s["mult"], SCORE_SHIFT,
                                       s["lut"], LUT_SHIFT, PROB_FRAC, rows_per_seq=s["rows"], slots=s["slots"],
                                       out=s["out"], workspace=s["ws"])
    return be.verify_drafts_dev(s["target"], s["tokens"], s["randoms"], exp_lut=s["lut"], draft=s["draft"],
                                n_draft=s["n_draft"], accepted=s["accepted"], out=s["out"], workspace=s["ws"])


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _rne(v, shift):
    """v / 2^shift of int64 tensors, rounded half to even; shift > 0."""
    q = v >> shift
    r, half = v - (q << shift), torch.ones_like(v) << (shift - 1)
    return q + ((r > half) | ((r == half) & ((q & 1) == 1))).to(torch.int64)


def _product(x, w):
    """x [.., M, K] times w [.., N, K] transposed: whole numbers below 2^53."""
    return (x.double() @ w.double().transpose(-1, -2).contiguous()).to(torch.int64)


def _clamp16(v):
    return torch.clamp(v, -32768, 32767)


def _plain_adapters(s):
    M, N, r, n = s["M"], s["N"], s["rank"], s["n"]
    base = _clamp16(_rne(_product(s["x"], s["W"]), s["w_shifts"].long() + (ACT_FRAC - OUT_FRAC)))
    ids = s["ids"].long()
    some = ids >= 0
    at = ids.clamp(min=0)
    # every row times every adapter, then each row's own
    u = _product(s["x"], s["A"].reshape(n * r, -1)).view(M, n, r)
    u = u.gather(1, at.view(M, 1, 1).expand(M, 1, r)).squeeze(1)
    u = _clamp16(_rne(u, s["a_shifts"][at].long() + (ACT_FRAC - MID_FRAC)))
    wide = torch.zeros((M, n, r), dtype=torch.int64, device=u.device)
    wide.scatter_(1, at.view(M, 1, 1).expand(M, 1, r), u.view(M, 1, r))
    d = _product(wide.view(M, n * r), s["B"].permute(1, 0, 2).reshape(N, n * r))
    d = _clamp16(_rne(d, s["b_shifts"][at].long() + (MID_FRAC - OUT_FRAC)))
    return _clamp16(base + torch.where(some.view(M, 1), d, torch.zeros_like(d))).to(torch.int16)


def _plain_attention(s):
    S, n, P = s["seqs"], s["rows"], s["prefix"]
    R, H, hd = s["q"].shape
    KH, T = s["kt"].shape[1], s["kt"].shape[2]
    G = H // KH
    q = s["q"].view(S, n, KH, G, hd).permute(2, 0, 1, 3, 4)                     # KV head, sequence, row, head
    slots = s["slots"].long()
    kt, vt = s["kt"][slots].transpose(0, 1), s["vt"][slots].transpose(0, 1)     # KV head, sequence, position
    zp = _product(q.reshape(KH, S * n * G, hd), s["kp"]).view(KH, S, n, G, P)
    zt = _product(q.reshape(KH, S, n * G, hd), kt).view(KH, S, n, G, T)
    z = _rne(torch.cat([zp, zt], -1) * s["mult"], SCORE_SHIFT)
    lens = s["lens"].long().view(1, S, n, 1, 1)
    j = torch.arange(P + T, device=z.device)
    seen = (lens >= 0) & (j < P + lens)
    m = torch.where(seen, z, torch.full_like(z, -2 ** 62)).amax(-1, keepdim=True)
    at = ((m - z) >> LUT_SHIFT).clamp(min=0)
    lut = torch.cat([s["lut"].long(), torch.zeros(1, dtype=torch.int64, device=z.device)])
    e = torch.where(seen, lut[at.clamp(max=lut.numel() - 1)], torch.zeros_like(z))
    total = e.sum(-1, keepdim=True).clamp(min=1)
    num = e << PROB_FRAC
    p = num // total
    twice = 2 * (num - p * total)
    p = p + ((twice > total) | ((twice == total) & ((p & 1) == 1))).long()
    pp, pt = p[..., :P].reshape(KH, S * n * G, P).double(), p[..., P:].reshape(KH, S, n * G, T).double()
    o = (pp @ s["vp"].double()).view(KH, S, n, G, hd) + (pt @ vt.double().contiguous()).view(KH, S, n, G, hd)
    o = _clamp16(_rne(o.to(torch.int64), PROB_FRAC))
    return o.permute(1, 2, 0, 3, 4).reshape(R, H, hd).to(torch.int16)


def _weights(z, lut):
    """Table weights of int32 logit rows (Q6) under their maximum."""
    below = (z.amax(-1, keepdim=True) - z).long() << 2
    ext = torch.cat([lut.long(), torch.zeros(1, dtype=torch.int64, device=z.device)])
    return ext[below.clamp(max=lut.numel())]


def _mulhi(a, b):
    """floor(a b / 2^64) of the bits a as an unsigned 64-bit number and 0 <= b < 2^63."""
    m32 = 0xFFFFFFFF
    ah, al, bh, bl = (a >> 32) & m32, a & m32, b >> 32, b & m32

    def top(x, y, add):  # floor((x y + add) / 2^32) and the low word, x, y, add < 2^32
        xh, xl = x >> 16, x & 0xFFFF
        low = xl * y + add
        mid = xh * y + (low >> 16)
        return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)

    c, _ = top(al, bl, torch.zeros_like(b))
    h1, l1 = top(ah, bl, c)
    h2, l2 = top(al, bh, l1)
    h3, l3 = top(ah, bh, h1)
    return (h3 << 32) + l3 + h2


def _plain_verify(s):
    z, tokens, B, k = s["target"], s["tokens"], s["B"], s["k"]
    dev = z.device
    n = torch.full((B,), k, device=dev) if s["n_draft"] is None else s["n_draft"].long()
    i = torch.arange(k, device=dev)
    seq = torch.arange(B, device=dev)
    if s["lut"] is None:
        best = z.amax(-1, keepdim=True)
        choice = torch.where(z == best, torch.arange(s["V"], device=dev), s["V"]).amin(-1)
        ok = choice[:, :k] == tokens
    else:
        p = _weights(z, s["lut"])
        P = p.sum(-1)
        pt = p[:, :k].gather(2, tokens.unsqueeze(2)).squeeze(2)
        if s["draft"] is None:
            Q, qt = torch.ones_like(pt), torch.ones_like(pt)
        else:
            q = _weights(s["draft"], s["lut"])
            Q = q.sum(-1)
            qt = q.gather(2, tokens.unsqueeze(2)).squeeze(2)
        ok = _mulhi(s["randoms"][:, :k], qt * P[:, :k]) < pt * Q
    run_of = (ok & (i < n.view(B, 1))).long().cumprod(1)
    acc = run_of.sum(1)
    if s["lut"] is None:
        new = choice[seq, acc]
    else:
        row = p[seq, acc]                       # the target's weights where the drafts end
        last = acc == n                         # every draft accepted: the target's own distribution
        at = acc.clamp(max=k - 1)
        if s["draft"] is None:
            left = row.scatter(1, tokens[seq, at].view(B, 1), 0)
        else:
            left = (row * Q[seq, at].view(B, 1) - q[seq, at] * P[seq, acc].view(B, 1)).clamp(min=0)
        w = torch.where(last.view(B, 1), row, left)
        w = torch.where(w.sum(1, keepdim=True) > 0, w, row)
        run = w.cumsum(1)
        thr = _mulhi(s["randoms"][:, k], run[:, -1])
        new = (run <= thr.view(B, 1)).sum(1)
    pos = torch.arange(k + 1, device=dev).view(1, k + 1)
    out = torch.cat([tokens, torch.zeros_like(tokens[:, :1])], 1)
    out = torch.where(pos < acc.view(B, 1), out, torch.full_like(out, -1))
    out = torch.where(pos == acc.view(B, 1), new.view(B, 1), out)
    return acc.to(torch.int32), out


_PLAIN = {"adapters": _plain_adapters, "attention": _plain_attention, "verify": _plain_verify}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["kind"] == "adapters":
        M, N, K, r, n = (case[c] for c in ("M", "N", "K", "rank", "n"))
        used = n * (1 - (1 - 1 / n) ** M)  # adapters with a row
        return {"bytes": int(N * K + 2 * M * K + 2 * M * N + N + 4 * M + used * (r * (K + N) + r + N)),
                "flops": 2 * M * N * K + 2 * M * r * (K + N)}
    if case["kind"] == "attention":
        H, KH, hd = HEADS[case["arch"]]
        S, n, P = case["seqs"], case["rows"], case["prefix"]
        used = S - 1 if S > 4 else S
        tail = case["tail"] / 2 + n
        return {"bytes": int(4 * KH * hd * (P + used * tail) + 4 * S * n * H * hd),
                "flops": int(4 * H * hd * used * n * (P + tail))}
    B, k, V = case["B"], case["k"], case["V"]
    kk = k / 2 if case["ragged"] else k
    rows = B * ((kk + 1) + (kk if case["mode"] == "draft" else 0))
    return {"bytes": int(4 * V * rows), "flops": int(2 * V * rows)}


# ---------------------------------------------------------------------------
# the definitions once more, one request at a time
# ---------------------------------------------------------------------------

def _half_even(num, den):
    """num / den of whole numbers, den > 0, to the nearest, ties to even."""
    fl = torch.div(num, den, rounding_mode="floor")
    twice = (num - fl * den) * 2 - den
    return fl + ((twice > 0) | ((twice == 0) & (fl.remainder(2) == 1))).to(fl.dtype)


def _exact_adapters(case, seed):
    s = _adapters(case, seed)
    two = torch.tensor(2, dtype=torch.int64, device="cuda")

    def layer(x, w, shifts, up, down):
        out = torch.empty((x.shape[0], w.shape[0]), dtype=torch.int64, device="cuda")
        for n0 in range(0, w.shape[0], 4096):
            c = slice(n0, n0 + 4096)
            acc = torch.mm(w[c].double(), x.double().T).T.to(torch.int64)
            out[:, c] = _half_even(acc, two ** (shifts[c].to(torch.int64) + up - down))
        return out.clamp(-32768, 32767)

    out = layer(s["x"], s["W"], s["w_shifts"], ACT_FRAC, OUT_FRAC)
    for a in range(case["n"]):
        rows = torch.nonzero(s["ids"] == a).flatten()
        if rows.numel():
            u = layer(s["x"][rows], s["A"][a], s["a_shifts"][a], ACT_FRAC, MID_FRAC)
            out[rows] += layer(u, s["B"][a], s["b_shifts"][a], MID_FRAC, OUT_FRAC)
    return out.clamp(-32768, 32767).to(torch.int16)


def _exact_attention(case, seed):
    s = _attention(case, seed)
    R, H, hd = s["q"].shape
    KH, n = s["kt"].shape[1], case["rows"]
    lens = s["lens"].tolist()
    out = torch.zeros((R, H, hd), dtype=torch.int16, device="cuda")
    table = s["lut"].to(torch.int64)
    kp, vp = s["kp"].double(), s["vp"].double()
    for r in range(R):
        if lens[r] < 0:
            continue
        slot = int(s["slots"][r // n])
        k = torch.cat([kp, s["kt"][slot, :, :lens[r]].double()], 1)     # KV head, position, dim
        v = torch.cat([vp, s["vt"][slot, :, :lens[r]].double()], 1)
        q = s["q"][r].view(KH, H // KH, hd).double()
        dots = torch.bmm(q, k.transpose(1, 2).contiguous()).to(torch.int64)
        z = _half_even(dots * s["mult"], torch.tensor(2 ** SCORE_SHIFT, device="cuda"))
        below = torch.div(z.amax(2, keepdim=True) - z, 2 ** LUT_SHIFT, rounding_mode="floor")
        e = torch.where(below < table.numel(), table[below.clamp(max=table.numel() - 1)], 0)
        p = _half_even(e * 2 ** PROB_FRAC, e.sum(2, keepdim=True))
        o = torch.bmm(p.double(), v).to(torch.int64)
        out[r] = _half_even(o, torch.tensor(2 ** PROB_FRAC, device="cuda")).clamp(-32768, 32767).view(H, hd).to(torch.int16)
    return out


def _exact_verify(case, seed):
    """One request at a time; Python's whole numbers for the comparisons."""
    s = _verify(case, seed)
    B, k, V = case["B"], case["k"], case["V"]
    accepted, out = [], []

    def weights(row):
        below = 4 * (int(row.max()) - row.to(torch.int64))
        w = torch.zeros(V, dtype=torch.int64, device="cuda")
        near = torch.nonzero(below < s["lut"].numel()).flatten()
        w[near] = s["lut"].to(torch.int64)[below[near]]
        return w

    for b in range(B):
        drafts = s["tokens"][b].tolist()[:k if s["n_draft"] is None else int(s["n_draft"][b])]
        rnd = [x % 2 ** 64 for x in s["randoms"][b].tolist()]
        taken, new = [], None
        for i, t in enumerate(drafts + [None]):
            row = s["target"][b, i]
            if s["lut"] is None:
                choice = int(torch.nonzero(row == row.max())[0])
                if t == choice:
                    taken.append(t)
                    continue
                new = choice
                break
            w = weights(row)
            total = int(w.sum())
            if t is not None:
                if s["draft"] is None:
                    q = torch.zeros_like(w)
                    q[t] = 1
                else:
                    q = weights(s["draft"][b, i])
                qsum = int(q.sum())
                if rnd[i] * int(q[t]) * total < int(w[t]) * qsum * 2 ** 64:
                    taken.append(t)
                    continue
                rest = (w * qsum - q * total).clamp(min=0)
                w = rest if int(rest.sum()) > 0 else w
            run = w.cumsum(0)
            threshold = rnd[k] * int(run[-1]) // 2 ** 64
            new = int(torch.nonzero(run > threshold)[0])
            break
        accepted.append(len(taken))
        out.append(taken + [new] + [-1] * (k - len(taken)))
    return (torch.tensor(accepted, dtype=torch.int32, device="cuda"), torch.tensor(out, dtype=torch.int64, device="cuda"))


def exact(case, seed):
    return {"adapters": _exact_adapters, "attention": _exact_attention, "verify": _exact_verify}[case["kind"]](case, seed)
