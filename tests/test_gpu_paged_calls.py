"""Calls over a paged cache that their documentation allows and that differ from an ordinary
step's: steps that run them together, captured and replayed, on several streams, in a kept
workspace, at the largest sizes; every comparison is for equality."""
from __future__ import annotations

import numpy as np
import pytest

import paged_ref as ref
import serving_ref
from conftest import case
from test_gpu_paged import (FRACS, append_inputs, attention_inputs, check_append, check_attention, check_logprobs, gpu_norm, head_norm, logits, on_gpu,
                            random_tables, rotation, run_append)
from test_gpu_serving import dirty, exp_lut, gauss16, gpu, rng, same  # noqa: F401

pytestmark = pytest.mark.gpu


class Step:
    """Sequences that decode: the q/k/v product of their newest rows, appending, attention, the
    head's logits, log probabilities; and the same with the plain forms."""

    def __init__(self, b, lut, seqs=5, H=6, KH=2, hd=64, hidden=96, V=1500, page=8, start=20, steps=4, seed=1, rows=1):
        r = rng(seed)
        self.b, self.lut, self.rows, self.page = b, lut, rows, page
        self.H, self.KH, self.hd, self.V = H, KH, hd, V
        R, self.N = seqs * rows, (H + 2 * KH) * hd
        T = -(-(start + rows * (steps + 1)) // page)
        self.norm = head_norm(r, hd, out_fracs=(10, 10))
        self.s = dict(x=gauss16(r, (R, hidden), 2000), W=r.integers(-127, 128, (self.N, hidden)).astype(np.int8),
                      w_shifts=r.integers(8, 11, self.N).astype(np.uint8), bias=gauss16(r, self.N, 3000), bias_shifts=r.integers(9, 13, self.N).astype(np.uint8),
                      head=r.integers(-127, 128, (V, H * hd)).astype(np.int8), head_shifts=r.integers(10, 12, V).astype(np.uint8),
                      kp=gauss16(r, (seqs * T + 2, KH, page, hd), 900), vp=gauss16(r, (seqs * T + 2, KH, page, hd), 900),
                      tables=random_tables(r, seqs, T, seqs * T + 2), tokens=r.integers(0, V, R))
        self.s["cos"], self.s["sin"] = rotation(r, 16, hd)
        self.first = (r.integers(0, start, (seqs, 1)) + np.arange(rows)).reshape(-1).astype(np.int32)
        if seqs > 2:
            self.first[-rows:] = -(2**30)  # padding
        self.seqs = np.repeat(np.arange(seqs), rows).astype(np.int32)
        self.mult, self.len = int(2**15 / np.sqrt(hd)), T * page
        import torch
        self.d = on_gpu(self.s)
        self.d.update(seqs=gpu(self.seqs), positions=gpu(self.first), lens=gpu(self.first + 1), lut=gpu(lut), norm=gpu_norm(self.norm))
        empty = lambda dtype, *shape: torch.full(shape, -7, dtype=dtype, device="cuda")
        self.o = dict(qkv=empty(torch.int16, R, self.N), q=torch.zeros((R, H, hd), dtype=torch.int16, device="cuda"), att=empty(torch.int16, R, H, hd),
                      z=empty(torch.int32, R, V), lp=empty(torch.int64, R), ent=empty(torch.int64, R), top=empty(torch.int64, R, 4), toplp=empty(torch.int64, R, 4))
        self.ws = [dirty(b.attention_paged_workspace(self.o["q"], self.d["kp"], self.len, rows)), dirty(b.logprobs_workspace(self.o["z"], self.d["lut"], 4))]

    def product(self):
        """The library's own product may allocate: outside of captures."""
        self.b.linear_w8a16_dev(self.d["x"], self.d["W"], self.d["w_shifts"], 10, 10, out=self.o["qkv"])

    def append_and_attend(self):
        b, d, o = self.b, self.d, self.o
        q = o["qkv"].view(-1, self.H + 2 * self.KH, self.hd)
        b.kv_append_paged_dev(q[:, :self.H], q[:, self.H:self.H + self.KH], q[:, self.H + self.KH:], d["positions"], d["kp"], d["vp"], d["tables"], d["cos"],
                              d["sin"], 8, seqs=d["seqs"], bias=d["bias"], bias_shifts=d["bias_shifts"], q_frac=10, k_frac=10, v_frac=10, norm=d["norm"], q_out=o["q"])
        b.attention_paged_dev(o["q"], d["kp"], d["vp"], d["tables"], d["lens"], self.mult, 21, d["lut"], 6, 14, rows_per_seq=self.rows, max_len=self.len, out=o["att"],
                              workspace=self.ws[0])

    def to_logits(self):
        self.b.logits_dev(self.o["att"].view(-1, self.H * self.hd), self.d["head"], self.d["head_shifts"], 10, 6, out=self.o["z"])

    def answer(self):
        self.b.logprobs_dev(self.o["z"], self.d["tokens"], self.d["lut"], 4, logprobs=self.o["lp"], entropy=self.o["ent"], top_tokens=self.o["top"],
                            top_logprobs=self.o["toplp"], workspace=self.ws[1])

    def advance(self):
        self.d["positions"] += self.rows
        self.d["lens"] += self.rows

    def check(self, turn, what):
        """The plain forms' step number `turn` on the plain forms' cache."""
        s, pos = self.s, self.first + self.rows * turn
        qkv = serving_ref.linear(s["x"], s["W"], s["w_shifts"], 10, 10).astype(np.int16).reshape(-1, self.H + 2 * self.KH, self.hd)
        q0 = np.zeros((len(pos), self.H, self.hd), np.int16)
        q, s["kp"], s["vp"] = ref.append(qkv[:, :self.H], qkv[:, self.H:self.H + self.KH], qkv[:, self.H + self.KH:], pos, s["kp"], s["vp"], s["tables"], s["cos"],
                                         s["sin"], 8, q0, self.seqs, s["bias"], s["bias_shifts"], FRACS, self.norm)
        att = ref.attention(q, s["kp"], s["vp"], s["tables"], pos + 1, self.mult, 21, self.lut, 6, 14, self.rows)
        for name, want in (("q", q), ("att", att)):
            same(self.o[name], want, f"{what}: {name}")
        same(self.d["kp"], s["kp"], f"{what}: keys")
        same(self.d["vp"], s["vp"], f"{what}: values")
        z = np.clip(serving_ref.rescale(serving_ref.dots(att.reshape(len(pos), -1), s["head"]), s["head_shifts"].astype(np.int64) + 10, 6), -2**31, 2**31 - 1)
        same(self.o["z"], z.astype(np.int32), f"{what}: logits")
        for name, want in zip(("lp", "ent", "top", "toplp"), ref.logprobs(z.astype(np.int32), s["tokens"], self.lut, 4)):
            same(self.o[name], want, f"{what}: {name}")


@pytest.mark.parametrize("seqs,rows,H,KH,hd,page,start", [(5, 1, 6, 2, 64, 8, 20), (3, 1, 28, 4, 128, 16, 700), (2, 3, 14, 2, 64, 40, 1400), (1, 2, 17, 1, 128, 64, 100)])
def test_steps_together(backend, exp_lut, seqs, rows, H, KH, hd, page, start):
    case(f"steps of {seqs} x {rows} rows, {H} heads, from {start}")
    s = Step(backend, exp_lut, seqs=seqs, rows=rows, H=H, KH=KH, hd=hd, page=page, start=start, seed=start)
    for turn in range(3):
        s.product()
        s.append_and_attend()
        s.to_logits()
        s.answer()
        s.check(turn, f"step {turn}")
        s.advance()


@pytest.mark.parametrize("start,hd,seqs", [(30, 64, 4), (2200, 64, 4), (500, 128, 4), (12000, 128, 9)])
def test_captured_steps(backend, exp_lut, start, hd, seqs):
    """The three calls captured and replayed, each replay a step further, with the program's own eager
    work and synchronizations between."""
    import torch
    case(f"captured steps of {seqs} sequences from {start}, heads of {hd}")
    s = Step(backend, exp_lut, seqs=seqs, H=14, KH=2, hd=hd, start=start, steps=6, seed=2)
    stream = torch.cuda.Stream()
    try:
        s.product()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            backend.use_torch_stream()
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for g, part in zip(graphs, (s.append_and_attend, s.answer)):
            with torch.cuda.graph(g, stream=stream):
                part()
        torch.cuda.synchronize()
        for turn in range(5):
            for name in ("att", "lp", "ent", "top", "toplp"):
                s.o[name].fill_(-7)
            for w in s.ws:
                dirty(w)
            s.o["q"].zero_()
            torch.cuda.synchronize()
            graphs[0].replay()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                s.to_logits()
            torch.cuda.synchronize()
            graphs[1].replay()
            torch.cuda.synchronize()
            s.check(turn, f"replay {turn}")
            s.advance()
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()


def test_two_graphs_of_one_workspace_in_turn(backend, exp_lut):
    """Two captured calls that share a workspace, replayed one after the other in any order."""
    import torch
    case("two graphs, one workspace")
    a, b = (attention_inputs(40 + i, 3, 1, 14, 2, 64, n, 16) for i, n in enumerate((1500, 200)))
    das, outs, graphs = [on_gpu(s) for s in (a, b)], [], []
    ws = dirty(backend.attention_paged_workspace(das[0]["q"], das[0]["kp"], 1500))
    lut, stream = gpu(exp_lut), torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(stream):
            backend.use_torch_stream()
        for s, d in zip((a, b), das):
            outs.append(torch.empty_like(d["q"]))
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                backend.attention_paged_dev(d["q"], d["kp"], d["vp"], d["tables"], d["lens"], s["mult"], 21, lut, 6, 14, max_len=s["max_len"], out=outs[-1], workspace=ws)
        want = [ref.attention(**s, lut=exp_lut) for s in (a, b)]
        for i in (0, 1, 1, 0, 0, 1):
            outs[i].fill_(-7)
            torch.cuda.synchronize()
            graphs[i].replay()
            torch.cuda.synchronize()
            same(outs[i], want[i], f"graph {i}")
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()


def test_two_streams_at_once(backend, exp_lut):
    """Steps of two contexts on two streams, each with its own cache and workspaces."""
    import torch
    from myelith_amd.backend import RocmBackend
    case("two streams")
    other = RocmBackend(0)
    try:
        steps = [Step(backend, exp_lut, seed=3, start=900, H=14, KH=2), Step(other, exp_lut, seed=4, seqs=3, rows=2, start=100)]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                s.b.use_torch_stream()
        for turn in range(3):
            for part in ("product", "append_and_attend", "to_logits", "answer"):
                for s, stream in zip(steps, streams):
                    with torch.cuda.stream(stream):
                        getattr(s, part)()
            torch.cuda.synchronize()
            for i, s in enumerate(steps):
                s.check(turn, f"stream {i}")
                s.advance()
            torch.cuda.synchronize()
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()
        other.close()


def test_left_out_outputs_and_workspaces(backend, exp_lut):
    """The calls allocate what they are not given, on the context's own stream beside torch's."""
    import torch
    case("outputs left out")
    s = attention_inputs(50, 4, 1, 6, 2, 64, 900, 16)
    a, z = append_inputs(51, 6, 4, 2, 64, 16), logits(52, 3, 5000)
    tokens = np.array([1, -1, 4999])
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            backend.use_torch_stream()
        for _ in range(3):
            d = on_gpu(s)
            same(backend.attention_paged_dev(d["q"], d["kp"], d["vp"], d["tables"], d["lens"], s["mult"], 21, gpu(exp_lut), 6, 14), ref.attention(**s, lut=exp_lut), "attention")
            d = dict(on_gpu(a), norm=None)
            got = run_append(backend, d, None)
            backend.synchronize()
            want = ref.append(a["q"], a["k"], a["v"], a["positions"], a["kp"], a["vp"], a["tables"], a["cos"], a["sin"], 8, a["q"], a["seqs"], a["bias"], a["bias_shifts"], FRACS)
            same(got, want[0], "queries")
            same(d["vp"], want[2], "values")
            got = backend.logprobs_dev(gpu(z), gpu(tokens), gpu(exp_lut), 3)
            backend.synchronize()
            for g, w in zip(got, ref.logprobs(z, tokens, exp_lut, 3)):
                same(g, w, "logprobs")
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()


@pytest.mark.parametrize("seqs,rows,length", [(6, 2, 2000), (6, 1, 2000), (1, 1, 2000), (1, 2, 500), (3, 2, 100), (2, 1, 1990)])
def test_attention_in_the_workspace_of_more(backend, exp_lut, seqs, rows, length):
    case(f"attention workspace kept, {seqs} x {rows} rows of {length}")
    most = attention_inputs(60, 6, 2, 14, 2, 64, 2000, 16)
    d = on_gpu(most)
    ws = dirty(backend.attention_paged_workspace(d["q"], d["kp"], 2000, 2))
    s = attention_inputs(61 + seqs, seqs, rows, 14, 2, 64, length, 16)
    d = on_gpu(s)
    got = backend.attention_paged_dev(d["q"], d["kp"], d["vp"], d["tables"], d["lens"], s["mult"], 21, gpu(exp_lut), 6, 14, rows_per_seq=rows, max_len=length, workspace=ws)
    same(got, ref.attention(**s, lut=exp_lut), "kept workspace")


# ---- the largest sizes ------------------------------------------------------------------------------

@pytest.mark.parametrize("page", [16, 100])
def test_attention_of_131072_keys(backend, exp_lut, page):
    case(f"attention of 131072 keys, pages of {page}")
    s = attention_inputs(70, 1, 2, 2, 1, 64, 131072, page, lens=[131071, 131072])
    check_attention(backend, s, exp_lut)
    s.update(mult=0)
    flat = np.full(32768, 32767, np.int16)  # an exp sum just below 2^32
    check_attention(backend, s, flat, "large entries")
    s["lens"][:] = [65535, 16384]
    check_attention(backend, s, flat, "fewer keys")
    check_attention(backend, s, np.zeros(9, np.int16), "uniform")


@pytest.mark.parametrize("hd,page", [(128, 16), (64, 16), (64, 40), (128, 40)])
def test_pages_past_4_gib(backend, exp_lut, hd, page):
    """Pages whose elements lie more than 2^32 into the pools, appended to and attended."""
    import torch
    case(f"pages past 4 GiB hd={hd}")
    KH, H, n = 2, 6, (1 << 32) // (2 * page * hd) + 50
    kp, vp = (torch.empty((n, KH, page, hd), dtype=torch.int16, device="cuda") for _ in range(2))
    r = rng(71)
    L, T = 700, -(-700 // page)
    tables = np.stack([n - 1 - np.arange(T), np.arange(T) * (n // T), (n // 2 + np.arange(T) * 7) % n]).astype(np.int32)
    rows = 3 * L
    seqs, pos = np.repeat(np.arange(3), L).astype(np.int32), np.tile(np.arange(L), 3).astype(np.int32)
    q, k, v = gauss16(r, (rows, H, hd), 2000), gauss16(r, (rows, KH, hd), 1000), gauss16(r, (rows, KH, hd), 2000)
    cos, sin = rotation(r, 50, hd)
    got = backend.kv_append_paged_dev(gpu(q), gpu(k), gpu(v), gpu(pos), kp, vp, gpu(tables), gpu(cos), gpu(sin), 8, seqs=gpu(seqs))
    rot = lambda x: np.stack([[ref.rotate(x[i, h], cos[pos[i] % 50], sin[pos[i] % 50], 8) for h in range(x.shape[1])] for i in range(rows)]).astype(np.int16)
    kr, qr = rot(k), rot(q)
    same(got, qr, "queries")
    at = torch.from_numpy(np.stack([tables[s, p // page] for s, p in zip(seqs, pos)]).astype(np.int64)).cuda()
    off = torch.from_numpy((pos % page).astype(np.int64)).cuda()
    same(kp[at, :, off], kr, "keys")
    same(vp[at, :, off], v, "values")
    newest = np.arange(3) * L + L - 1
    out = backend.attention_paged_dev(gpu(qr[newest]), kp, vp, gpu(tables), gpu(np.full(3, L, np.int32)), 2896, 21, gpu(exp_lut), 6, 14, max_len=L)
    for s in range(3):
        one = slice(s * L, s * L + L)
        want = ref.attention(qr[newest[s]][None], kr[one].transpose(1, 0, 2)[None], v[one].transpose(1, 0, 2)[None], np.zeros((1, 1), np.int32), [L], 2896, 21, exp_lut, 6, 14)
        same(out[s:s + 1], want, f"sequence {s}")


def test_append_many_rows(backend):
    """More rows than a thread keeps, of every group's remainder; positions far past the tables of the rotation."""
    import torch
    case("append many rows")
    for rows, H, KH, hd in ((16385, 28, 4, 128), (70001, 1, 1, 64), (33333, 14, 2, 64)):
        g = torch.Generator(device="cuda").manual_seed(rows)
        qkv = torch.randint(-3000, 3001, (rows, H + 2 * KH, hd), dtype=torch.int16, device="cuda", generator=g)
        page, T = 64, -(-rows // 64)
        kp, vp = (torch.zeros((T, KH, page, hd), dtype=torch.int16, device="cuda") for _ in range(2))
        pos = torch.arange(rows, dtype=torch.int32, device="cuda")
        tables = torch.randperm(T, device="cuda", generator=g).to(torch.int32).view(1, T)
        cos, sin = (torch.randint(-256, 257, (33, hd // 2), dtype=torch.int16, device="cuda", generator=g) for _ in range(2))
        bias = torch.randint(-2000, 2001, ((H + 2 * KH) * hd,), dtype=torch.int16, device="cuda", generator=g)
        shifts = torch.full_like(bias, 11, dtype=torch.uint8)
        got = backend.kv_append_paged_dev(qkv[:, :H], qkv[:, H:H + KH], qkv[:, H + KH:], pos, kp, vp, tables, cos, sin, 8, seqs=torch.zeros_like(pos), bias=bias,
                                          bias_shifts=shifts, q_frac=10, k_frac=10, v_frac=10)
        b = bias.long()
        b = (b >> 1) + ((b & 3) == 3).long()  # half of it, to even
        x = (qkv.long() + b.view(H + 2 * KH, hd)).clamp(-32768, 32767)
        c, s = (t[pos.long() % 33].long().unsqueeze(1) for t in (cos, sin))
        lo, hi = x[:, :H + KH, :hd // 2], x[:, :H + KH, hd // 2:]
        turned = torch.cat([lo * c - hi * s, hi * c + lo * s], 2)
        down, rest = turned >> 8, turned & 255
        turned = (down + ((rest > 128) | ((rest == 128) & ((down & 1) == 1))).long()).clamp(-32768, 32767).to(torch.int16)
        assert (got == turned[:, :H]).all()
        at = tables[0].long()[pos.long() // page]
        assert (kp[at, :, pos.long() % page] == turned[:, H:]).all() and (vp[at, :, pos.long() % page] == x[:, H + KH:].to(torch.int16)).all()


def test_append_positions_at_the_end_of_their_type(backend):
    case("append far positions")
    s = append_inputs(72, 4, 2, 1, 64, 16, n_pos=2047)
    s["positions"][:] = [2**31 - 1, 2**31 - 2, 3, 2**30]
    check_append(backend, s)


@pytest.mark.parametrize("R,V,top", [(1, 1 << 20, 32), (65535, 3, 3), (2000, 300, 7), (513, 8193, 1)])
def test_logprobs_at_the_largest_sizes(backend, exp_lut, R, V, top):
    case(f"logprobs R={R} V={V} top={top}")
    r = rng(73)
    z = r.integers(-900, 900, (R, V)).astype(np.int32)
    check_logprobs(backend, z, r.integers(0, V, (R, 1)), exp_lut, top)


@pytest.mark.parametrize("R", [3, 600])
def test_logprobs_more_equal_values_than_candidates(backend, exp_lut, R):
    """Rows of zeros, of two values, with one tile of 300 large values or many tiles that reach the edge."""
    case(f"logprobs equal values R={R}")
    V = 30000
    z = np.zeros((R, V), np.int32)
    z[1, ::3] = 7
    z[2, 1000:1300] = 50
    for r in range(3, R):
        z[r, (r * 37) % V::(r % 700) + 1] = r
    check_logprobs(backend, z, np.arange(R), exp_lut, 32)
    check_logprobs(backend, z, np.arange(R), exp_lut, 1)


@pytest.mark.parametrize("rows", [6, 3000])
def test_append_rows_left_out_of_allocated_queries(backend, rows):
    """Without q_out, rows that are left out answer with zeros, whatever the memory held before."""
    import torch
    case(f"append rows left out of an allocated output, {rows} rows")
    s = append_inputs(80 + rows, rows, 4, 2, 64, 16, seqs=6, context=600)
    s["positions"][::3] = -1
    s["seqs"][1::6] = 6
    want = ref.append(s["q"], s["k"], s["v"], s["positions"], s["kp"], s["vp"], s["tables"], s["cos"], s["sin"], 8, np.zeros_like(s["q"]), s["seqs"],
                      s["bias"], s["bias_shifts"], FRACS)
    try:
        for stream in (None, torch.cuda.Stream()):  # torch's stream, and the context's own beside it
            if stream is not None:
                torch.cuda.synchronize()
                with torch.cuda.stream(stream):
                    backend.use_torch_stream()
            d = dict(on_gpu(s), norm=None)
            used = [torch.full((rows, 4, 64), 77, dtype=torch.int16, device="cuda") for _ in range(4)]
            torch.cuda.synchronize()
            del used
            got = run_append(backend, d, None)
            torch.cuda.synchronize()
            for what, g, w in zip(("queries", "keys", "values"), (got, d["kp"], d["vp"]), want):
                same(g, w, what)
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()


def test_attention_of_drafts_in_the_workspace_of_a_decode_batch(backend, exp_lut):
    """64 requests of one row each keep a workspace; 21 of them then take three drafted rows."""
    case("attention of 21 x 3 rows in the workspace of 64 x 1")
    s = attention_inputs(81, 21, 3, 28, 4, 64, 1300, 16)
    d = on_gpu(s)
    one = d["q"].new_empty((64, 28, 64))
    ws = dirty(backend.attention_paged_workspace(one, d["kp"], 1300))
    got = backend.attention_paged_dev(d["q"], d["kp"], d["vp"], d["tables"], d["lens"], s["mult"], 21, gpu(exp_lut), 6, 14, rows_per_seq=3, max_len=1300, workspace=ws)
    same(got, ref.attention(**s, lut=exp_lut), "kept workspace")


@pytest.mark.parametrize("keys", [513, 560, 576])
def test_attention_of_launches_just_past_64_kib(backend, exp_lut, keys):
    """One launch whose rings, scores, pages and table pass 64 KiB only with what the kernel declares."""
    case(f"attention of {keys} keys, 14 heads on 2 of 64")
    check_attention(backend, attention_inputs(82, 3, 1, 14, 2, 64, keys, 16), exp_lut)


def test_attention_of_ranges_just_past_64_kib(backend, exp_lut):
    """Ranges of 960 keys by pages of 8: the same for P.V over ranges."""
    case("attention of 48 rows of 10000 keys, pages of 8")
    r = rng(83)
    s = attention_inputs(83, 1, 1, 1, 1, 128, 2400, 8)
    s.update(q=gauss16(r, (48, 1, 128), 2048), tables=r.integers(0, s["kp"].shape[0], (48, 1250)).astype(np.int32), max_len=10000,
             lens=r.integers(1, 10001, 48).astype(np.int32))
    s["lens"][0] = 10000
    check_attention(backend, s, exp_lut)


def test_append_captured_with_its_allocated_queries(backend):
    """A captured call that allocates its queries clears them on every replay."""
    import torch
    case("append captured with allocated queries")
    s = append_inputs(84, 40, 4, 2, 64, 16, seqs=6, context=60)
    s["positions"][::4] = -5
    want = ref.append(s["q"], s["k"], s["v"], s["positions"], s["kp"], s["vp"], s["tables"], s["cos"], s["sin"], 8, np.zeros_like(s["q"]), s["seqs"],
                      s["bias"], s["bias_shifts"], FRACS)
    d, stream, graph = dict(on_gpu(s), norm=None), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(stream):
            backend.use_torch_stream()
        with torch.cuda.graph(graph, stream=stream):
            got = run_append(backend, d, None)
        for turn in range(4):
            got.fill_(77)
            d["kp"].copy_(gpu(s["kp"]))
            d["vp"].copy_(gpu(s["vp"]))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for what, g, w in zip(("queries", "keys", "values"), (got, d["kp"], d["vp"]), want):
                same(g, w, f"replay {turn}: {what}")
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()
