"""What is measured of a serving step over a paged cache: the new token's keys
and values go into pages, its query attends them through a table, and its
logits answer with log probabilities.

  append     `kv_append_paged_dev`: rows of queries, keys and values take their
             biases, norms of each head (where a layer has them) and the rotation of
             their position; keys and values are stored in the pages of a cache
  attention  `attention_paged_dev`: integer attention of each sequence's newest
             rows over its pages, split over the length and joined
  logprobs   `logprobs_dev`: the log probabilities of given tokens, the entropy
             and the most likely alternatives of rows of logits

Every output is a whole number that the fixed-point definitions fix bit for bit.
`own` false computes them with elementary torch operations: whole numbers below
2^53 in float64 products, everything else in int64.
"""
from __future__ import annotations

import math

import torch

own = False

HEADS = {"7b": (28, 4, 128), "0.5b": (14, 2, 64)}  # query heads, KV heads, head size
V7, V05 = 152064, 151936

# the fixed-point formats of the layers: Q10 activations and normed heads, Q14 scores and
# probabilities; the rotation's tables hold 2048 positions in Q8, the rsqrt table Q8 of Q8
Q_FRAC, K_FRAC, V_FRAC, NORM_FRAC, ROPE_FRAC = 10, 10, 10, 10, 8
SCORE_FRAC, PROB_FRAC = 14, 14
SCORE_SHIFT = Q_FRAC + K_FRAC + 15 - SCORE_FRAC
LUT_SHIFT = SCORE_FRAC - 8
ROPE_ROWS, ROPE_THETA = 2048, 1000000.0
RSQRT_SHIFT, RSQRT_FRAC, RSQRT_LEN = 8, 8, 32768


def listed():
    return [
        # one request's new token in the smallest layout: launches and latency count
        dict(name="append_1_small", kind="append", arch="0.5b", seqs=1, rows=1, context=300, page=16, bias=True, norm=False),
        # a decode batch, one new token each at any position
        dict(name="append_24", kind="append", arch="7b", seqs=24, rows=1, context=2500, page=64, bias=True, norm=False),
        # the prompts of three requests in one chunk of a model with norms of its heads, ragged
        dict(name="append_3x501_norm", kind="append", arch="7b", seqs=3, rows=501, context=1300, page=16, bias=False, norm=True),
        # the largest chunk of prompts
        dict(name="append_8x2048", kind="append", arch="7b", seqs=8, rows=2048, context=4096, page=128, bias=True, norm=False),
        # one short chat: latency
        dict(name="attention_1x130", kind="attention", arch="0.5b", seqs=1, rows=1, length=130, page=16),
        # a decode batch, every chat some thousand tokens in
        dict(name="attention_24x2500", kind="attention", arch="7b", seqs=24, rows=1, length=2500, page=64),
        # four drafted rows of each request, pages of 16
        dict(name="attention_12x4x3001", kind="attention", arch="7b", seqs=12, rows=4, length=3001, page=16),
        # one very long document: few rows, so the length is what is split
        dict(name="attention_1x100000", kind="attention", arch="7b", seqs=1, rows=1, length=100000, page=128),
        # a large batch of long chats
        dict(name="attention_64x12000", kind="attention", arch="7b", seqs=64, rows=1, length=12000, page=64),
        # one request with a small vocabulary and five alternatives: latency
        dict(name="logprobs_1_small", kind="logprobs", R=1, V=32001, tokens=1, top=5),
        # a decode batch with as many alternatives as an interface offers
        dict(name="logprobs_24_top20", kind="logprobs", R=24, V=V7, tokens=1, top=20),
        # a whole prompt's log probabilities
        dict(name="logprobs_2003_top1", kind="logprobs", R=2003, V=V7, tokens=1, top=1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


PAGES = [8, 16, 16, 24, 32, 64, 64, 100, 128, 256]


def draw(rng):
    kind = rng.choice(["append", "attention", "logprobs"])
    if kind == "append":
        seqs = _log(rng, 1, 64)
        rows = 1 if rng.random() < 0.4 else _log(rng, 2, 16384 // seqs)
        return dict(kind=kind, arch=rng.choice(list(HEADS)), seqs=seqs, rows=rows, context=rows + _log(rng, 1, 2000),
                    page=rng.choice(PAGES), bias=rng.random() < 0.5, norm=rng.random() < 0.5)
    if kind == "attention":
        seqs, rows = _log(rng, 1, 64), rng.choice([1, 1, 1, rng.randrange(2, 9)])
        return dict(kind=kind, arch=rng.choice(list(HEADS)), seqs=seqs, rows=rows, page=rng.choice(PAGES),
                    length=_log(rng, 16, min(100000, 64 * 12000 // (seqs * rows))))
    return dict(kind=kind, R=_log(rng, 1, 2000), V=rng.choice([V7, V05, 32001]), tokens=rng.choice([1, 1, 1, 2, 4]),
                top=rng.choice([0, 1, 5, 8, 20]))


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


def _ints(lo, hi, shape, dtype, g):
    return torch.randint(lo, hi, shape, dtype=dtype, device="cuda", generator=g)


def exp_table():
    """round(exp(-i / 2^8) 2^14) up to its last entry that is not zero."""
    t = [round(math.exp(-i / 256.0) * 16384) for i in range(16385)]
    while not t[-1]:
        t.pop()
    return torch.tensor(t, dtype=torch.int16, device="cuda")


def rsqrt_table():
    """round(2^8 / sqrt(x / 2^8)), the entry of 0 that of 1.0."""
    x = torch.arange(RSQRT_LEN, dtype=torch.float64, device="cuda")
    t = torch.round(2.0 ** RSQRT_FRAC / torch.sqrt(x / 2.0 ** RSQRT_SHIFT))
    t[0] = 2.0 ** RSQRT_FRAC
    return t.to(torch.int16)


def rotation_tables(hd):
    """round(2^8 cos) and round(2^8 sin) of position times theta^-(j / half)."""
    j = torch.arange(hd // 2, dtype=torch.float64, device="cuda")
    angle = torch.arange(ROPE_ROWS, dtype=torch.float64, device="cuda").view(-1, 1) * ROPE_THETA ** (-j / (hd // 2))
    return [torch.round(f(angle) * 2.0 ** ROPE_FRAC).to(torch.int16).contiguous() for f in (torch.cos, torch.sin)]


def _pages(lens, longest, page, KH, hd, g, filled):
    """Pages in any order for sequences of given lengths; table entries past a
    sequence's last page name none."""
    S, T = lens.numel(), -(-longest // page)
    n = S * T + 3
    tables = torch.randperm(n, device="cuda", generator=g)[:S * T].to(torch.int32).view(S, T)
    past = torch.arange(T, device="cuda") * page >= lens.view(S, 1)
    tables = torch.where(past, torch.full_like(tables, -1), tables).contiguous()
    shape = (n, KH, page, hd)
    if not filled:
        return tables, torch.zeros(shape, dtype=torch.int16, device="cuda"), torch.zeros(shape, dtype=torch.int16, device="cuda")
    return tables, _gauss16(shape, g, 1024), _gauss16(shape, g, 2000)


def _append(case, seed):
    """Projections of deviation 2000 with biases of the same size; `rows` new tokens of each
    sequence at any place of its context.  In a batch of more than four the last
    sequence's rows are padding."""
    g = _gen(seed)
    H, KH, hd = HEADS[case["arch"]]
    S, n, ctx = case["seqs"], case["rows"], case["context"]
    qkv = _gauss16((S * n, (H + 2 * KH) * hd), g, 2000)  # one product's rows: queries, keys, values
    first = _ints(0, ctx - n + 1, (S, 1), torch.int32, g)
    positions = first + torch.arange(n, dtype=torch.int32, device="cuda")
    if S > 4:
        positions[-1] = -1
    s = dict(qkv=qkv, positions=positions.reshape(-1).contiguous(),
             seqs=torch.arange(S, dtype=torch.int32, device="cuda").repeat_interleave(n))
    s["tables"], s["kpages"], s["vpages"] = _pages((first + n).view(-1), ctx, case["page"], KH, hd, g, False)
    s["cos"], s["sin"] = rotation_tables(hd)
    s["bias"] = s["bias_shifts"] = None
    if case["bias"]:
        s["bias"] = _gauss16(((H + 2 * KH) * hd,), g, 8000)
        s["bias_shifts"] = _ints(11, 14, ((H + 2 * KH) * hd,), torch.uint8, g)
    if case["norm"]:
        s.update(q_gamma=_ints(40, 128, (hd,), torch.int8, g), k_gamma=_ints(40, 128, (hd,), torch.int8, g),
                 q_gamma_shifts=_ints(6, 8, (hd,), torch.uint8, g), k_gamma_shifts=_ints(6, 8, (hd,), torch.uint8, g),
                 rsqrt=rsqrt_table(), inv_n_q20=(1 << 20) // hd)
    return s


def _attention(case, seed):
    """Post-RoPE q and k of deviation 2 and 1 (scores of deviation 2); sequences between
    half of the length and all of it, row i of a sequence up to its own position.
    In a batch of more than four the last sequence's rows are padding."""
    g = _gen(seed)
    H, KH, hd = HEADS[case["arch"]]
    S, n, L = case["seqs"], case["rows"], case["length"] + case["rows"] - 1
    base = _ints((case["length"] + 1) // 2, case["length"] + 1, (S, 1), torch.int32, g)
    if S == 1:
        base.fill_(case["length"])
    lens = base + torch.arange(n, dtype=torch.int32, device="cuda")
    s = dict(q=_gauss16((S * n, H, hd), g, 2048), lut=exp_table(), mult=round(2 ** 15 / math.sqrt(hd)))
    s["tables"], s["kpages"], s["vpages"] = _pages((base + n - 1).view(-1), L, case["page"], KH, hd, g, True)
    if S > 4:
        lens[-1] = -1
    s["lens"] = lens.reshape(-1).contiguous()
    return s


def _logprobs(case, seed):
    """Q6 logits: Gaussian of deviation 2.5 with some likely tokens a row; the given tokens
    are among those."""
    g = _gen(seed)
    R, V = case["R"], case["V"]
    z = torch.empty((R, V), dtype=torch.int32, device="cuda")
    for r0 in range(0, R, 256):
        z[r0:r0 + 256] = torch.randn((min(256, R - r0), V), device="cuda", generator=g).mul_(160).round_().to(torch.int32)
    likely = _ints(0, V, (R, 8), torch.int64, g)
    z.scatter_(1, likely, _ints(700, 1400, (R, 8), torch.int32, g))
    return dict(logits=z, tokens=likely[:, :case["tokens"]].contiguous(), lut=exp_table())


_INPUTS = {"append": _append, "attention": _attention, "logprobs": _logprobs}
_BACKEND = None


def backend():
    """One context per process on torch's stream, as a serving program keeps it."""
    global _BACKEND
    if _BACKEND is None:
        from myelith_amd.backend import RocmBackend
        _BACKEND = RocmBackend(0)
        _BACKEND.use_torch_stream()
    return _BACKEND


def _views(s):
    """The queries, keys and values of a product's rows."""
    H, KH, hd = HEADS[s["arch"]]
    x = s["qkv"].view(-1, H + 2 * KH, hd)
    return x[:, :H], x[:, H:H + KH], x[:, H + KH:]


def prepare(case, seed):
    s = dict(case, **_INPUTS[case["kind"]](case, seed))
    if case["kind"] == "append":
        H, _, hd = HEADS[case["arch"]]
        s["q_out"] = torch.zeros((s["qkv"].shape[0], H, hd), dtype=torch.int16, device="cuda")
    if own:  # the outputs and the workspace that a serving program keeps from step to step
        be = s["be"] = backend()
        if case["kind"] == "append":
            s["q"], s["k"], s["v"] = _views(s)
            s["norm"] = None
            if case["norm"]:
                from myelith_amd.backend import HeadNorm
                s["norm"] = HeadNorm(s["q_gamma"], s["q_gamma_shifts"], s["k_gamma"], s["k_gamma_shifts"], s["rsqrt"],
                                     RSQRT_SHIFT, RSQRT_FRAC, s["inv_n_q20"], NORM_FRAC, NORM_FRAC)
        elif case["kind"] == "attention":
            s["out"] = torch.empty_like(s["q"])
            s["max_len"] = case["length"] + case["rows"] - 1
            s["ws"] = be.attention_paged_workspace(s["q"], s["kpages"], s["max_len"], rows_per_seq=case["rows"])
        else:
            R, T, n = case["R"], case["tokens"], case["top"]
            s["logprobs"] = torch.empty((R, T), dtype=torch.int64, device="cuda")
            s["entropy"] = torch.empty(R, dtype=torch.int64, device="cuda")
            s["top_tokens"] = torch.empty((R, n), dtype=torch.int64, device="cuda")
            s["top_logprobs"] = torch.empty((R, n), dtype=torch.int64, device="cuda")
            s["ws"] = be.logprobs_workspace(s["logits"], s["lut"], n)
    torch.cuda.synchronize()
    return s


def run(s):
    if not own:
        return _PLAIN[s["kind"]](s)
    be = s["be"]
    if s["kind"] == "append":
        be.kv_append_paged_dev(s["q"], s["k"], s["v"], s["positions"], s["kpages"], s["vpages"], s["tables"], s["cos"], s["sin"],
                               ROPE_FRAC, seqs=s["seqs"], bias=s["bias"], bias_shifts=s["bias_shifts"], q_frac=Q_FRAC,
                               k_frac=K_FRAC, v_frac=V_FRAC, norm=s["norm"], q_out=s["q_out"])
        return s["q_out"], s["kpages"], s["vpages"]
    if s["kind"] == "attention":
        return be.attention_paged_dev(s["q"], s["kpages"], s["vpages"], s["tables"], s["lens"], s["mult"], SCORE_SHIFT, s["lut"],
                                      LUT_SHIFT, PROB_FRAC, rows_per_seq=s["rows"], max_len=s["max_len"], out=s["out"],
                                      workspace=s["ws"])
    return be.logprobs_dev(s["logits"], s["tokens"], s["lut"], s["top"], logprobs=s["logprobs"], entropy=s["entropy"],
                           top_tokens=s["top_tokens"], top_logprobs=s["top_logprobs"], workspace=s["ws"])


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _rne(v, shift):
    """v / 2^shift of int64 tensors, rounded half to even; a negative shift goes left."""
    if not torch.is_tensor(shift):
        shift = torch.tensor(shift, dtype=torch.int64, device=v.device)
    down = shift.clamp(min=0)
    q = v >> down
    r = v - (q << down)
    half = torch.where(down > 0, torch.ones_like(down) << (down - 1).clamp(min=0), torch.ones_like(down))
    q = q + ((down > 0) & ((r > half) | ((r == half) & ((q & 1) == 1)))).long()
    return q << (-shift).clamp(min=0)


def _product(x, w):
    """x [.., M, K] times w [.., N, K] transposed: whole numbers below 2^53."""
    return (x.double() @ w.double().transpose(-1, -2).contiguous()).to(torch.int64)


def _clamp16(v):
    return torch.clamp(v, -32768, 32767)


def _biased(x, s, at, frac):
    x = x.long()
    if s["bias"] is None:
        return x
    b, sh = s["bias"][at].long(), s["bias_shifts"][at].long()
    return _clamp16(x + _rne(b, sh - frac).view(x.shape[1:]))


def _normed(x, s, gamma, shifts):
    """The norm of each head: x over its root mean square, times gamma."""
    m = (x.square().sum(-1) * s["inv_n_q20"]) >> 20
    q = torch.zeros_like(m)
    for _ in range(20):
        q = torch.where((m >> q) > RSQRT_LEN - 1, q + 2, q)
    root = s["rsqrt"].long()[_rne(m, q).clamp(max=RSQRT_LEN - 1)]
    down = (RSQRT_FRAC + RSQRT_SHIFT // 2 - NORM_FRAC) + (q // 2).unsqueeze(-1) + shifts.long()
    y = _clamp16(_rne(x * root.unsqueeze(-1) * gamma.long(), down))
    return torch.where((x == 0).all(-1, keepdim=True), torch.zeros_like(y), y)


def _rotated(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([_clamp16(_rne(a * cos - b * sin, ROPE_FRAC)), _clamp16(_rne(b * cos + a * sin, ROPE_FRAC))], -1)


def _plain_append(s):
    H, KH, hd = HEADS[s["arch"]]
    nq, nkv = H * hd, KH * hd
    q, k, v = _views(s)
    q = _biased(q, s, slice(0, nq), Q_FRAC)
    k = _biased(k, s, slice(nq, nq + nkv), K_FRAC)
    v = _biased(v, s, slice(nq + nkv, nq + 2 * nkv), V_FRAC)
    if s["norm"]:
        q = _normed(q, s, s["q_gamma"], s["q_gamma_shifts"])
        k = _normed(k, s, s["k_gamma"], s["k_gamma_shifts"])
    pos = s["positions"].long()
    some = pos >= 0
    at = pos.clamp(min=0)
    cos, sin = (t.long()[at % ROPE_ROWS].unsqueeze(1) for t in (s["cos"], s["sin"]))
    q, k = _rotated(q, cos, sin), _rotated(k, cos, sin)
    page = s["tables"][s["seqs"].long(), at // s["page"]].long()
    to = (page[some], slice(None), (at % s["page"])[some])
    for pages, x in ((s["kpages"], k), (s["vpages"], v)):
        pages[to] = x[some].to(torch.int16)
    return torch.where(some.view(-1, 1, 1), q, torch.zeros_like(q)).to(torch.int16), s["kpages"], s["vpages"]


def _gathered(pages, tables, L, page):
    """[KV head, sequence, position, dim] of the first L positions of every table."""
    j = torch.arange(L, device=pages.device)
    ids = tables[:, j // page].long().clamp(min=0)
    return pages.permute(1, 0, 2, 3)[:, ids, (j % page).view(1, L)]


def _plain_attention(s):
    S, n, page = s["seqs"], s["rows"], s["page"]
    R, H, hd = s["q"].shape
    KH, L = s["kpages"].shape[1], s["length"] + n - 1
    G = H // KH
    q = s["q"].view(S, n, KH, G, hd).permute(2, 0, 1, 3, 4).reshape(KH, S, n * G, hd)
    z = _product(q, _gathered(s["kpages"], s["tables"], L, page)).view(KH, S, n, G, L)
    z = _rne(z * s["mult"], SCORE_SHIFT)
    seen = torch.arange(L, device=z.device) < s["lens"].long().view(1, S, n, 1, 1)
    m = torch.where(seen, z, torch.full_like(z, -2 ** 62)).amax(-1, keepdim=True)
    at = ((m - z) >> LUT_SHIFT).clamp(min=0)
    lut = torch.cat([s["lut"].long(), torch.zeros(1, dtype=torch.int64, device=z.device)])
    e = torch.where(seen, lut[at.clamp(max=lut.numel() - 1)], torch.zeros_like(z))
    total = e.sum(-1, keepdim=True).clamp(min=1)
    num = e << PROB_FRAC
    p = num // total
    twice = 2 * (num - p * total)
    p = p + ((twice > total) | ((twice == total) & ((p & 1) == 1))).long()
    v = _gathered(s["vpages"], s["tables"], L, page).double()
    o = (p.view(KH, S, n * G, L).double() @ v).to(torch.int64)
    o = _clamp16(_rne(o, PROB_FRAC)).view(KH, S, n, G, hd)
    return o.permute(1, 2, 0, 3, 4).reshape(R, H, hd).to(torch.int16)


LN2_Q30 = 744261118


def _ln_q16(S):
    """ln(S / 2^14) in Q16 of int64 1 <= S < 2^62: the first 16 fraction bits of log2 by
    squaring, times ln 2 in Q30."""
    e = torch.zeros_like(S)
    for b in (32, 16, 8, 4, 2, 1):
        big = (S >> (e + b)) > 0
        e = torch.where(big, e + b, e)
    x = S << (62 - e)
    f = torch.zeros_like(S)
    for _ in range(16):
        h, l = x >> 32, x & 0xFFFFFFFF
        a = h * l
        # floor(x x / 2^62) below 2^64: the top bit is the sign
        x = ((h * h) << 2) + (a >> 29) + (((a & 0x1FFFFFFF) + (((l * l) >> 33) & 0x7FFFFFFF)) >> 29)
        over = x < 0
        f = 2 * f + over.long()
        x = torch.where(over, (x >> 1) & 0x7FFFFFFFFFFFFFFF, x)
    return _rne(((e - 14) * 65536 + f) * LN2_Q30, 30)


def _plain_logprobs(s):
    z, R, V, top = s["logits"], s["R"], s["V"], s["top"]
    lut = torch.cat([s["lut"].long(), torch.zeros(1, dtype=torch.int64, device=z.device)])
    logp, entropy = torch.empty_like(s["tokens"]), torch.empty(R, dtype=torch.int64, device=z.device)
    tops, toplp = (torch.empty((R, top), dtype=torch.int64, device=z.device) for _ in range(2))
    low = V - 1 - torch.arange(V, device=z.device)
    for r0 in range(0, R, 512):
        r = slice(r0, r0 + 512)
        x = z[r].long()
        m = x.amax(1, keepdim=True)
        below = m - x
        w = lut[(below << 2).clamp(max=lut.numel() - 1)]
        total = w.sum(1)
        ln = _ln_q16(total.clamp(min=1))
        logp[r] = (x.gather(1, s["tokens"][r]) - m) * 1024 - ln.view(-1, 1)
        num, den = (w * below).sum(1) * 1024, total.clamp(min=1)
        part = num // den
        twice = 2 * (num - part * den)
        entropy[r] = ln + part + ((twice > den) | ((twice == den) & ((part & 1) == 1))).long()
        if top:
            key = (x << 20) + low  # by the logit, then by the lower index
            best = key.topk(top, dim=1).values
            tops[r] = V - 1 - (best & (2 ** 20 - 1))
            toplp[r] = ((best >> 20) - m) * 1024 - ln.view(-1, 1)
    return logp, entropy, tops, toplp


_PLAIN = {"append": _plain_append, "attention": _plain_attention, "logprobs": _plain_logprobs}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["kind"] == "append":
        H, KH, hd = HEADS[case["arch"]]
        S, n = case["seqs"], case["rows"]
        rows = (S - 1 if S > 4 else S) * n
        once = 2 * hd * min(rows, ROPE_ROWS) + 8 * rows + (3 * (H + 2 * KH) * hd if case["bias"] else 0)
        return {"bytes": int(4 * rows * (H + 2 * KH) * hd + once), "flops": int(rows * (H + KH) * hd * (3 + 4 * case["norm"]))}
    if case["kind"] == "attention":
        H, KH, hd = HEADS[case["arch"]]
        S, n, L = case["seqs"], case["rows"], case["length"]
        used = S - 1 if S > 4 else S
        keys = (L if S == 1 else 0.75 * L) + n - 1
        return {"bytes": int(4 * KH * hd * used * keys + 4 * S * n * H * hd), "flops": int(4 * H * hd * used * n * keys)}
    R, V = case["R"], case["V"]
    return {"bytes": int(4 * V * R + 8 * R * (2 * case["tokens"] + 1 + 2 * case["top"])), "flops": int(2 * V * R)}


# ---------------------------------------------------------------------------
# the definitions once more, one sequence or row at a time
# ---------------------------------------------------------------------------

def _half_even(num, den):
    """num / den of whole numbers, den > 0, to the nearest, ties to even."""
    fl = torch.div(num, den, rounding_mode="floor")
    twice = (num - fl * den) * 2 - den
    return fl + ((twice > 0) | ((twice == 0) & (fl.remainder(2) == 1))).to(fl.dtype)


def _scaled(v, down):
    """v / 2^down, half to even; v 2^-down where down is negative (int64 tensors)."""
    two = torch.tensor(2, dtype=torch.int64, device=v.device)
    return _half_even(v * two ** (-down).clamp(min=0), two ** down.clamp(min=0))


def _sat(v):
    return v.clamp(-32768, 32767)


def _exact_append(case, seed):
    s = dict(case, **_append(case, seed))
    H, KH, hd = HEADS[case["arch"]]
    half, page = hd // 2, case["page"]
    x = s["qkv"].to(torch.int64)
    if case["bias"]:
        x = _sat(x + _scaled(s["bias"].to(torch.int64), s["bias_shifts"].to(torch.int64) - Q_FRAC))
    x = x.view(-1, H + 2 * KH, hd)
    q, k, v = x[:, :H].clone(), x[:, H:H + KH].clone(), x[:, H + KH:].clone()
    if case["norm"]:
        table = s["rsqrt"].tolist()
        for y, gamma, shifts in ((q, s["q_gamma"], s["q_gamma_shifts"]), (k, s["k_gamma"], s["k_gamma_shifts"])):
            squares = (y * y).sum(2).flatten().tolist()
            value, frac = [], []
            for total in squares:
                mean, e = total * s["inv_n_q20"] // 2 ** 20, 0
                while mean // 2 ** e > RSQRT_LEN - 1:
                    e += 2
                fl, rest = divmod(mean, 2 ** e)
                fl += 2 * rest > 2 ** e or (2 * rest == 2 ** e and e > 0 and fl % 2 == 1)
                value.append(table[min(fl, RSQRT_LEN - 1)] if total else 0)
                frac.append(RSQRT_FRAC + RSQRT_SHIFT // 2 + e // 2)
            value, frac = (torch.tensor(t, dtype=torch.int64, device="cuda").view(*y.shape[:2], 1) for t in (value, frac))
            y.copy_(_sat(_scaled(y * value * gamma.to(torch.int64), frac + shifts.to(torch.int64) - NORM_FRAC)))
    pos = s["positions"].tolist()
    turn = torch.tensor([max(p, 0) % ROPE_ROWS for p in pos], device="cuda")
    c, sn = s["cos"].to(torch.int64)[turn][:, None], s["sin"].to(torch.int64)[turn][:, None]
    one = torch.tensor(2 ** ROPE_FRAC, dtype=torch.int64, device="cuda")
    for y in (q, k):
        lo, hi = y[:, :, :half].clone(), y[:, :, half:].clone()
        y[:, :, :half] = _sat(_half_even(lo * c - hi * sn, one))
        y[:, :, half:] = _sat(_half_even(hi * c + lo * sn, one))
    q_out = torch.zeros((len(pos), H, hd), dtype=torch.int16, device="cuda")
    tables, seqs = s["tables"].tolist(), s["seqs"].tolist()
    rows = [r for r, p in enumerate(pos) if p >= 0]
    to = torch.tensor([tables[seqs[r]][pos[r] // page] * page + pos[r] % page for r in rows], device="cuda")
    rows = torch.tensor(rows, device="cuda")
    q_out[rows] = q[rows].to(torch.int16)
    for pages, y in ((s["kpages"], k), (s["vpages"], v)):
        flat = pages.transpose(1, 2).reshape(-1, KH, hd)
        flat.index_copy_(0, to, y[rows].to(torch.int16))
        pages.copy_(flat.view(-1, page, KH, hd).transpose(1, 2))
    return q_out, s["kpages"], s["vpages"]


def _exact_attention(case, seed):
    s = _attention(case, seed)
    R, H, hd = s["q"].shape
    KH, page, n = s["kpages"].shape[1], case["page"], case["rows"]
    lens = s["lens"].tolist()
    out = torch.zeros((R, H, hd), dtype=torch.int16, device="cuda")
    table = s["lut"].to(torch.int64)
    for b in range(R // n):
        most = max(lens[b * n:b * n + n])
        if most < 1:
            continue
        ids = s["tables"][b, :-(-most // page)].to(torch.int64)
        k, v = (t[ids].transpose(0, 1).reshape(KH, -1, hd).double() for t in (s["kpages"], s["vpages"]))
        for r in range(b * n, b * n + n):
            kr, vr = k[:, :lens[r]], v[:, :lens[r]].contiguous()
            dots = torch.bmm(s["q"][r].view(KH, H // KH, hd).double(), kr.transpose(1, 2).contiguous()).to(torch.int64)
            z = _half_even(dots * s["mult"], torch.tensor(2 ** SCORE_SHIFT, device="cuda"))
            below = torch.div(z.amax(2, keepdim=True) - z, 2 ** LUT_SHIFT, rounding_mode="floor")
            e = torch.where(below < table.numel(), table[below.clamp(max=table.numel() - 1)], 0)
            p = _half_even(e * 2 ** PROB_FRAC, e.sum(2, keepdim=True))
            o = torch.bmm(p.double(), vr).to(torch.int64)
            out[r] = _sat(_half_even(o, torch.tensor(2 ** PROB_FRAC, device="cuda"))).view(H, hd).to(torch.int16)
    return out


def _whole_ln_q16(total):
    """ln(total / 2^14) in Q16 with Python's whole numbers."""
    e = total.bit_length() - 1
    x, f = total << (62 - e), 0
    for _ in range(16):
        x = x * x >> 62
        f *= 2
        if x >= 2 ** 63:
            x //= 2
            f += 1
    fl, rest = divmod(((e - 14) * 65536 + f) * LN2_Q30, 2 ** 30)
    return fl + (2 * rest > 2 ** 30 or (2 * rest == 2 ** 30 and fl % 2 == 1))


def _exact_logprobs(case, seed):
    s = _logprobs(case, seed)
    R, V, top = case["R"], case["V"], case["top"]
    table = s["lut"].to(torch.int64)
    logp, entropy, tops, toplp = [], [], [], []
    for r in range(R):
        row = s["logits"][r]
        best = int(row.max())
        near = torch.nonzero(row > best - table.numel()).flatten()
        below = best - row[near].to(torch.int64)
        w = torch.where(4 * below < table.numel(), table[(4 * below).clamp(max=table.numel() - 1)], 0)
        total, moment = torch.stack([w.sum(), (w * below).sum()]).tolist()
        ln = _whole_ln_q16(total)
        fl, rest = divmod(moment * 1024, total)
        entropy.append(ln + fl + (2 * rest > total or (2 * rest == total and fl % 2 == 1)))
        logp.append([(z - best) * 1024 - ln for z in row[s["tokens"][r]].tolist()])
        if top:
            # values past the top-th largest, and of that one the lowest indices
            edge = torch.sort(row, descending=True).values[top - 1]
            at = torch.nonzero(row >= edge).flatten().tolist()
            order = sorted(zip((-row[row >= edge].to(torch.int64)).tolist(), at))[:top]
            tops.append([i for _, i in order])
            toplp.append([(-z - best) * 1024 - ln for z, _ in order])
    t = lambda v, *shape: torch.tensor(v, dtype=torch.int64, device="cuda").view(shape)
    return t(logp, R, case["tokens"]), t(entropy, R), t(tops, R, top), t(toplp, R, top)


def exact(case, seed):
    return {"append": _exact_append, "attention": _exact_attention, "logprobs": _exact_logprobs}[case["kind"]](case, seed)
