"""The operators over a paged cache and the log probabilities on the GPU against plain
64-bit forms (tests/paged_ref.py), bit for bit, and a step that runs them together.
All outputs are whole numbers, so every comparison is for equality."""
from __future__ import annotations

import numpy as np
import pytest

import paged_ref as ref
from conftest import case
from test_gpu_serving import dirty, exp_lut, gauss16, gpu, rng, same  # noqa: F401

pytestmark = pytest.mark.gpu

FRACS = (10, 10, 10)


def on_gpu(s):
    return {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in s.items()}


def rotation(r, n, hd):
    """Tables of any values up to 1.0 in Q8."""
    return [r.integers(-256, 257, (n, hd // 2)).astype(np.int16) for _ in range(2)]


def random_tables(r, seqs, length, n_pages):
    """No page twice."""
    return r.permutation(n_pages)[:seqs * length].reshape(seqs, length).astype(np.int32)


# ---- appending ------------------------------------------------------------------

def head_norm(r, hd, parts=(True, True), **over):
    gamma = [r.integers(-128, 128, hd).astype(np.int8) if p else None for p in parts]
    shifts = [r.integers(4, 10, hd).astype(np.uint8) if p else None for p in parts]
    x = np.arange(32768) / 256
    with np.errstate(divide="ignore"):
        t = np.rint(256 / np.sqrt(x))
    t[0] = 256
    return dict(dict(gamma=gamma, shifts=shifts, rsqrt=t.astype(np.int16), lut_input_shift=8, lut_output_frac=8, inv_n_q20=(1 << 20) // hd,
                     out_fracs=(10, 11)), **over)


def append_inputs(seed, rows, H, KH, hd, page, seqs=None, context=100, bias=True, norm=None, n_pos=64, spare=5):
    r = rng(seed)
    seqs = rows if seqs is None else seqs
    T = -(-context // page)
    n_pages = seqs * T + spare
    s = dict(q=gauss16(r, (rows, H, hd), 2000), k=gauss16(r, (rows, KH, hd), 2000), v=gauss16(r, (rows, KH, hd), 2000),
             kp=gauss16(r, (n_pages, KH, page, hd), 900), vp=gauss16(r, (n_pages, KH, page, hd), 900),
             tables=random_tables(r, seqs, T, n_pages), seqs=r.integers(0, seqs, rows).astype(np.int32))
    # places of their own: a random order of all of them
    every = [(a, b) for a in range(seqs) for b in range(context)]
    pick = [every[i] for i in r.permutation(len(every))[:rows]]
    s["seqs"] = np.array([a for a, _ in pick], np.int32)
    s["positions"] = np.array([b for _, b in pick], np.int32)
    s["cos"], s["sin"] = rotation(r, n_pos, hd)
    s["bias"] = gauss16(r, (H + 2 * KH) * hd, 9000) if bias else None
    s["bias_shifts"] = r.integers(5, 16, (H + 2 * KH) * hd).astype(np.uint8) if bias else None
    s["norm"] = norm
    return s


def gpu_norm(n):
    from myelith_amd.backend import HeadNorm
    if n is None:
        return None
    return HeadNorm(gpu(n["gamma"][0]), gpu(n["shifts"][0]), gpu(n["gamma"][1]), gpu(n["shifts"][1]), gpu(n["rsqrt"]), n["lut_input_shift"],
                    n["lut_output_frac"], n["inv_n_q20"], *n["out_fracs"])


def run_append(backend, d, q_out, rope_frac=8, fracs=FRACS):
    return backend.kv_append_paged_dev(d["q"], d["k"], d["v"], d["positions"], d["kp"], d["vp"], d["tables"], d["cos"], d["sin"], rope_frac,
                                       seqs=d["seqs"], bias=d["bias"], bias_shifts=d["bias_shifts"], q_frac=fracs[0], k_frac=fracs[1],
                                       v_frac=fracs[2], norm=d["norm"], q_out=q_out)


def check_append(backend, s, rope_frac=8, fracs=FRACS):
    """Everything that the call must write, and nothing else, is written."""
    import torch
    d = dict(on_gpu(s), norm=gpu_norm(s["norm"]))
    out = np.full(s["q"].shape, -7, np.int16)
    got = run_append(backend, d, gpu(out), rope_frac, fracs)
    torch.cuda.synchronize()
    want = ref.append(s["q"], s["k"], s["v"], s["positions"], s["kp"], s["vp"], s["tables"], s["cos"], s["sin"], rope_frac, out, s["seqs"],
                      s["bias"], s["bias_shifts"], fracs, s["norm"])
    for what, g, w in zip(("queries", "keys", "values"), (got, d["kp"], d["vp"]), want):
        same(g, w, what)


@pytest.mark.parametrize("rows,H,KH,hd,page", [(1, 1, 1, 64, 16), (1, 28, 4, 128, 64), (3, 14, 2, 64, 16), (24, 28, 4, 128, 16), (7, 3, 3, 128, 1),
                                               (33, 16, 1, 64, 24), (5, 0, 2, 128, 7), (70, 5, 5, 64, 100), (129, 8, 2, 128, 128)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("norm", [None, (True, True), (True, False), (False, True)])
def test_append(backend, rows, H, KH, hd, page, bias, norm):
    case(f"append rows={rows} H={H} KH={KH} hd={hd} page={page} bias={bias} norm={norm}")
    r = rng(7 * rows + hd)
    check_append(backend, append_inputs(rows + page, rows, H, KH, hd, page, bias=bias, norm=None if norm is None else head_norm(r, hd, norm)))


def test_append_rows_left_out(backend):
    """Negative positions and sequences outside the tables leave everything as it was; positions
    past the table or on no page keep their query only."""
    case("append rows left out")
    s = append_inputs(1, 12, 4, 2, 64, 16, seqs=4)
    s["positions"][[0, 5]] = [-1, -2**31]
    s["seqs"][[1, 6, 7]] = [-1, 4, 2**31 - 1]
    s["positions"][[2, 8]] = [s["tables"].shape[1] * 16, 2**31 - 1]
    s["seqs"][3], s["positions"][3] = 0, 17
    s["tables"][0, 1] = -1
    s["seqs"][9], s["positions"][9] = 1, 33
    s["tables"][1, 2] = s["kp"].shape[0]
    s["seqs"][10], s["positions"][10] = 2, 5
    s["tables"][2, 0] = 2**31 - 1
    check_append(backend, s)


@pytest.mark.parametrize("norm", [False, True])
def test_append_extremes(backend, norm):
    """Full-range values, biases that saturate, zero heads, all scales; tables of one position."""
    case(f"append extremes norm={norm}")
    r = rng(2)
    for hd, n_pos, frac, fracs in ((64, 1, 8, (0, 20, 15)), (128, 3, 14, (15, 0, 31)), (64, 2048, 0, (10, 10, 10))):
        n = None
        if norm:
            n = head_norm(r, hd, out_fracs=(0, 20))
            n["shifts"][0][:8] = [0, 1, 30, 40, 60, 100, 200, 255]
        s = append_inputs(hd + frac, 9, 5, 2, hd, 8, n_pos=n_pos, norm=n)
        s["q"][0], s["q"][1], s["k"][0], s["v"][0] = -32768, 32767, -32768, 32767
        s["q"][2], s["k"][2], s["q"][3] = 0, 0, 1
        s["cos"][:], s["sin"][0] = r.integers(-32768, 32768, s["cos"].shape), 32767
        s["bias"][:hd], s["bias"][hd:2 * hd] = -32768, 0
        s["bias_shifts"][:] = r.integers(0, 32, s["bias_shifts"].shape)
        check_append(backend, s, frac, fracs)


@pytest.mark.parametrize("rsqrt,inv", [(2, 1 << 20), (3, 1), (32768, 0), (1000, 8192)])
def test_append_norm_tables(backend, rsqrt, inv):
    """Short tables, means of 0 and of the whole sum, entries of any sign."""
    case(f"append norm table of {rsqrt}, 1/n {inv}")
    r = rng(rsqrt)
    n = head_norm(r, 128, rsqrt=r.integers(-32768, 32768, rsqrt).astype(np.int16), inv_n_q20=inv, lut_input_shift=4, lut_output_frac=11)
    s = append_inputs(3, 11, 3, 1, 128, 16, norm=n)
    s["q"][0], s["q"][1] = -32768, 0
    s["q"][2] = 0
    s["q"][2, :, 5] = 1
    check_append(backend, s)


@pytest.mark.parametrize("hd", [64, 128])
def test_append_is_the_framework_s_own_steps(backend, hd):
    """add_bias_i16, rmsnorm and rope of the host slices in turn."""
    case(f"append against the host calls hd={hd}")
    r = rng(4)
    n = head_norm(r, hd)
    s = append_inputs(5, 6, 3, 2, hd, 16, norm=n)
    d = dict(on_gpu(s), norm=gpu_norm(n))
    got = run_append(backend, d, None).cpu().numpy()
    kp, vp = d["kp"].cpu().numpy(), d["vp"].cpu().numpy()
    H = s["q"].shape[1]
    for row in range(6):
        for part, x, at in ((0, s["q"], 0), (1, s["k"], H), (2, s["v"], H + 2)):
            for h in range(x.shape[1]):
                w = slice((at + h) * hd, (at + h + 1) * hd)
                y = backend.add_bias_i16(x[row, h], s["bias"][w], s["bias_shifts"][w], 10)
                if part < 2:
                    y = backend.rmsnorm(y, np.full(hd, 10, np.uint8), n["gamma"][part], n["shifts"][part], n["rsqrt"], 8, 8, (1 << 20) // hd,
                                        n["out_fracs"][part])
                    y = backend.rope(y[None], y[None], s["cos"].ravel(), s["sin"].ravel(), s["positions"][row:row + 1], 8)[0][0]
                to = ref.place(s["tables"], s["seqs"][row], int(s["positions"][row]), 16, kp.shape[0])
                is_ = got[row, h] if part == 0 else (kp if part == 1 else vp)[to[0], h, to[1]]
                assert (is_ == y).all(), (row, part, h)


@pytest.mark.parametrize("layout", ["position first", "beside each other", "wide"])
def test_append_strides(backend, layout):
    """Pages as [page][position][head], keys beside values, room between; queries, keys and
    values as parts of one product's rows; rotated in place."""
    import torch
    case(f"append strides {layout}")
    s = append_inputs(6, 10, 6, 2, 64, 16)
    d = on_gpu(s)
    n, KH, page, hd = s["kp"].shape
    if layout == "position first":
        kp, vp = (torch.empty((n, page, KH, hd), dtype=torch.int16, device="cuda").transpose(1, 2) for _ in range(2))
    elif layout == "beside each other":
        both = torch.empty((n, 2, KH, page, hd), dtype=torch.int16, device="cuda")
        kp, vp = both[:, 0], both[:, 1]
    else:
        kp, vp = (torch.empty((n, KH + 1, page + 3, hd + 8), dtype=torch.int16, device="cuda")[:, :KH, :page, :hd] for _ in range(2))
    kp.copy_(d["kp"]), vp.copy_(d["vp"])
    qkv = torch.empty((10, 6 + 2 * 2 + 1, hd), dtype=torch.int16, device="cuda")
    q, k, v = qkv[:, :6], qkv[:, 6:8], qkv[:, 8:10]
    q.copy_(d["q"]), k.copy_(d["k"]), v.copy_(d["v"])
    tables = torch.full((10, d["tables"].shape[1] + 4), -5, dtype=torch.int32, device="cuda")[:, :d["tables"].shape[1]]
    tables.copy_(d["tables"])
    got = run_append(backend, dict(d, q=q, k=k, v=v, kp=kp, vp=vp, tables=tables, norm=None), q)
    assert got is q
    want = ref.append(s["q"], s["k"], s["v"], s["positions"], s["kp"], s["vp"], s["tables"], s["cos"], s["sin"], 8, s["q"], s["seqs"], s["bias"],
                      s["bias_shifts"], FRACS)
    for what, g, w in zip(("queries", "keys", "values"), (q, kp, vp), want):
        same(g.contiguous(), w, what)
    same(k.contiguous(), s["k"], "the keys' rows")


# ---- attention ------------------------------------------------------------------

def attention_inputs(seed, seqs, rows, H, KH, hd, length, page, lens=None, spare=3):
    r = rng(seed)
    T = max(-(-length // page), 1)
    n_pages = seqs * T + spare
    R = seqs * rows
    s = dict(q=gauss16(r, (R, H, hd), 2048), kp=gauss16(r, (n_pages, KH, page, hd), 1024), vp=gauss16(r, (n_pages, KH, page, hd), 2000),
             tables=random_tables(r, seqs, T, n_pages), mult=int(round(2**15 / np.sqrt(hd))), shift=21, lut_shift=6, prob_frac=14,
             rows_per_seq=rows, max_len=length)
    if lens is None:
        base = r.integers(1, max(length - rows + 1, 1) + 1, (seqs, 1))
        base[0] = max(length - rows + 1, 1)
        lens = (base + np.arange(rows)).reshape(-1)
    s["lens"] = np.broadcast_to(np.asarray(lens), (R,)).astype(np.int32).copy()
    return s


def run_attention(backend, s, lut, **over):
    d = dict(on_gpu(s), **over)
    ws = dirty(backend.attention_paged_workspace(d["q"], d["kp"], d["max_len"], d["rows_per_seq"]))
    return backend.attention_paged_dev(d["q"], d["kp"], d["vp"], d["tables"], d["lens"], d["mult"], d["shift"], gpu(lut), d["lut_shift"],
                                       d["prob_frac"], rows_per_seq=d["rows_per_seq"], max_len=d["max_len"], workspace=ws)


def check_attention(backend, s, lut, what="attention"):
    same(run_attention(backend, s, lut), ref.attention(**s, lut=lut), what)


@pytest.mark.parametrize("seqs,rows,H,KH,hd,length,page", [
    (1, 1, 1, 1, 64, 1, 1), (1, 1, 14, 2, 64, 130, 16), (2, 1, 28, 4, 128, 64, 64), (3, 1, 7, 1, 128, 65, 16), (5, 1, 28, 4, 128, 333, 24),
    (2, 1, 8, 8, 64, 700, 100), (4, 3, 14, 2, 64, 515, 16), (1, 1, 28, 4, 128, 4100, 128), (2, 5, 28, 4, 128, 1500, 32), (1, 8, 12, 2, 64, 2049, 1),
    (3, 1, 16, 1, 128, 900, 7), (2, 1, 17, 1, 64, 640, 16), (1, 2, 40, 1, 128, 390, 48), (33, 1, 4, 2, 64, 257, 8), (9, 1, 3, 3, 128, 2000, 256),
    (1, 33, 6, 2, 64, 100, 16), (2, 16, 14, 2, 64, 1300, 64)])
def test_attention(backend, exp_lut, seqs, rows, H, KH, hd, length, page):
    case(f"attention seqs={seqs} rows={rows} H={H} KH={KH} hd={hd} length={length} page={page}")
    check_attention(backend, attention_inputs(seqs + length, seqs, rows, H, KH, hd, length, page), exp_lut)


@pytest.mark.parametrize("length", [40, 1000])
def test_attention_lens(backend, exp_lut, length):
    """No key, one, the ends of pages and tiles, all, more than there are."""
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, length - 1, length, length + 1, -1, -2**31, 2**31 - 1, 24]
    case(f"attention lens up to {length}")
    s = attention_inputs(11, len(lens), 1, 14, 2, 64, length, 24, lens=lens)
    check_attention(backend, s, exp_lut)
    s["max_len"] = length - 7
    check_attention(backend, s, exp_lut, "a smaller max_len")
    s["lens"][:] = 0
    check_attention(backend, s, exp_lut, "no key at all")
    s.update(max_len=0)
    check_attention(backend, s, exp_lut, "max_len 0")


@pytest.mark.parametrize("length,page", [(200, 16), (1500, 24), (1500, 1), (3000, 128)])
def test_attention_missing_pages(backend, exp_lut, length, page):
    """Positions on no page count as not there: single pages, the first, the last, all but
    one, all; and the uniform split of a table without weights counts those that are."""
    case(f"attention missing pages {length} by {page}")
    s = attention_inputs(12, 6, 1, 14, 2, 64, length, page, lens=[length, length - 1, length, length, length, 70])
    T = s["tables"].shape[1]
    s["tables"][0, ::3] = -1
    s["tables"][1, 0] = s["kp"].shape[0]
    s["tables"][2, T - 1] = 2**31 - 1
    s["tables"][3, np.arange(T) != T // 2] = -2**31
    s["tables"][4] = -1
    check_attention(backend, s, exp_lut)
    check_attention(backend, s, np.zeros(5, np.int16), "uniform")
    s["prob_frac"] = 3
    check_attention(backend, s, np.zeros(1, np.int16), "uniform, fewer units than keys")


@pytest.mark.parametrize("length", [100, 1200])
@pytest.mark.parametrize("mult,shift,lut_shift", [(2896, 21, 6), (2**40, 50, 6), (-2896, 21, 6), (1, 0, 0), (2896, 3, 0), (2**62, 63, 31), (0, 9, 6),
                                                  (4096, 38, 40), (8388607, 33, 15), (2896, 21, 18)])
def test_attention_scales(backend, exp_lut, length, mult, shift, lut_shift):
    """Multipliers and shifts of every form, scores that wrap among them; full-range operands."""
    case(f"attention scales {mult} {shift} {lut_shift} length {length}")
    s = attention_inputs(13, 3, 1, 14, 2, 64, length, 16)
    s["q"][0], s["kp"][s["tables"][0, 0], :, :8] = -32768, -32768
    s["vp"][s["tables"][0]] = -32768
    s["vp"][s["tables"][1]] = 32767
    s.update(mult=mult, shift=shift, lut_shift=lut_shift)
    check_attention(backend, s, exp_lut)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("top", [32639, 32640, 32767])
def test_attention_large_queries(backend, exp_lut, hd, top):
    """Queries about the largest whose low byte is taken as a signed one, in one vector of a tile."""
    case(f"attention queries up to {top} hd={hd}")
    s = attention_inputs(16, 3, 1, 6, 2, hd, 700, 16)
    s["q"] = rng(17).integers(-32768, top + 1, s["q"].shape).astype(np.int16)
    s["q"][:2] = np.minimum(s["q"][:2], 32000)
    s["q"][2, 4, hd - 1] = top
    s["kp"] = rng(18).integers(-32768, 32768, s["kp"].shape).astype(np.int16)
    s["shift"] = 33
    check_attention(backend, s, exp_lut)


@pytest.mark.parametrize("length", [90, 900])
def test_attention_tables(backend, length):
    """Exp tables: one entry, negative entries, the largest ones, all of 32768; every prob_frac."""
    case(f"attention exp tables length {length}")
    r = rng(14)
    luts = [np.array([16384], np.int16), np.array([-5, -1, 7, -32768, 9], np.int16), np.full(32768, 32767, np.int16),
            r.integers(-3000, 32768, 4099).astype(np.int16), np.array([0, 0, 3], np.int16)]
    for i, lut in enumerate(luts):
        for f in (14, 13, 7, 0):
            s = attention_inputs(15 + i, 2, 1, 6, 2, 128, length, 16)
            s["prob_frac"] = f
            check_attention(backend, s, lut, f"table {i} prob_frac {f}")


@pytest.mark.parametrize("layout", ["position first", "beside each other", "wide"])
@pytest.mark.parametrize("length", [100, 1100])
def test_attention_strides(backend, exp_lut, layout, length):
    import torch
    case(f"attention strides {layout} {length}")
    s = attention_inputs(21, 4, 2, 12, 4, 128, length, 16)
    d = on_gpu(s)
    n, KH, page, hd = s["kp"].shape
    if layout == "position first":
        kp, vp = (torch.empty((n, page, KH, hd), dtype=torch.int16, device="cuda").transpose(1, 2) for _ in range(2))
    elif layout == "beside each other":
        both = torch.empty((n, 2, KH, page, hd), dtype=torch.int16, device="cuda")
        kp, vp = both[:, 0], both[:, 1]
    else:
        kp, vp = (torch.empty((n, KH + 1, page + 3, hd + 8), dtype=torch.int16, device="cuda")[:, :KH, :page, :hd] for _ in range(2))
    kp.copy_(d["kp"]), vp.copy_(d["vp"])
    q = torch.empty((8, 15, hd), dtype=torch.int16, device="cuda")[:, 1:13]
    q.copy_(d["q"])
    tables = torch.full((4, d["tables"].shape[1] + 3), 2**30, dtype=torch.int32, device="cuda")[:, :d["tables"].shape[1]]
    tables.copy_(d["tables"])
    out = torch.full((8, 14, hd), -7, dtype=torch.int16, device="cuda")
    backend.attention_paged_dev(q, kp, vp, tables, d["lens"], s["mult"], s["shift"], gpu(exp_lut), 6, 14, rows_per_seq=2, max_len=length,
                                out=out[:, :12])
    same(out[:, :12].contiguous(), ref.attention(**s, lut=exp_lut), "attention")
    assert (out[:, 12:] == -7).all()


def test_attention_shared_pages(backend, exp_lut):
    """Sequences that share their first pages, and one that names a page twice."""
    case("attention shared pages")
    s = attention_inputs(22, 5, 1, 14, 2, 64, 800, 32)
    s["tables"][:, :10] = s["tables"][0, :10]
    s["tables"][2, 12:] = s["tables"][2, 11]
    check_attention(backend, s, exp_lut)


# ---- log probabilities --------------------------------------------------------------

def logits(seed, R, V, spread=160):
    r = rng(seed)
    z = np.rint(r.normal(0, spread, (R, V))).astype(np.int32)
    for row in z:
        row[r.integers(0, V, 6)] = r.integers(600, 1400, 6)
    return z


def check_logprobs(backend, z, tokens, lut, top_n, what="log probabilities"):
    d = gpu(z)
    ws = dirty(backend.logprobs_workspace(d, gpu(lut), top_n))
    got = backend.logprobs_dev(d, gpu(tokens), gpu(lut), top_n, workspace=ws)
    for name, g, w in zip(("logprobs", "entropy", "tokens", "their logprobs"), got, ref.logprobs(z, tokens, lut, top_n)):
        same(g, w, f"{what}: {name}")


@pytest.mark.parametrize("R,V,T,top", [(1, 1, 1, 1), (1, 2, 1, 2), (3, 255, 2, 5), (2, 256, 0, 32), (5, 257, 1, 32), (7, 1024, 1, 20), (1, 32001, 4, 20),
                                       (24, 8192, 1, 8), (24, 8193, 1, 0), (3, 100003, 3, 32), (300, 4099, 1, 5), (2, 1 << 20, 1, 32),
                                       (70, 33, 70, 32), (11, 151936, 1, 1)])
def test_logprobs(backend, exp_lut, R, V, T, top):
    case(f"logprobs R={R} V={V} T={T} top={top}")
    tokens = rng(R + V).integers(-2, V + 2, (R, T))
    check_logprobs(backend, logits(R * V, R, V), tokens, exp_lut, top)


def test_logprobs_of_rows(backend, exp_lut):
    """Rows that are constant, rise, fall, hold only a few values or the type's ends; masked ones."""
    case("logprobs rows")
    V = 20011
    r = rng(31)
    low = np.iinfo(np.int32).min
    z = np.zeros((14, V), np.int32)
    z[1], z[2], z[3] = np.arange(V), -np.arange(V), r.integers(0, 3, V)
    z[4], z[5] = low, np.iinfo(np.int32).max
    z[6] = low
    z[6, 7777] = -5
    z[7] = low
    z[7, [3, 300, 19999]] = [np.iinfo(np.int32).max, 0, 1]
    z[8] = np.where(np.arange(V) % 2 == 0, low, 100)
    z[9, 15000:] = 1
    z[10] = r.integers(-2**31, 2**31, V)
    z[11, 512:768] = np.arange(256)[::-1] + 5  # all alternatives in one tile
    z[12] = np.repeat(np.arange(V // 256 + 1), 256)[:V]
    z[13] = (np.arange(V) % 256 == 255) * 50
    tokens = np.stack([np.arange(14), np.full(14, V - 1)], 1)
    for top in (0, 1, 7, 32):
        check_logprobs(backend, z, tokens, exp_lut, top, f"top {top}")


@pytest.mark.parametrize("lut", ["one", "negative", "none", "long", "odd"])
def test_logprobs_tables(backend, lut):
    case(f"logprobs table {lut}")
    r = rng(32)
    table = dict(one=np.array([16384]), negative=np.array([-1, 0, 0, 0, 9, 0, 0, 0, -32768]), none=np.zeros(40), long=np.full(32768, 32767),
                 odd=r.integers(-100, 32768, 4099))[lut].astype(np.int16)
    z = logits(33, 6, 9000, 60)
    z[5] = r.integers(-9000, 1, 9000)
    check_logprobs(backend, z, r.integers(0, 9000, 6), table, 5)


def test_logprobs_strides_and_the_log_softmax(backend, exp_lut):
    """Rows at any 4-byte address with room between them; the same as logsoftmax_dev."""
    import torch
    case("logprobs strides")
    z = logits(34, 5, 30011)
    wide = torch.zeros((5, 30011 + 6), dtype=torch.int32, device="cuda")
    view = wide[:, 3:3 + 30011]
    view.copy_(gpu(z))
    tokens = rng(35).integers(0, 30011, 5)
    got = backend.logprobs_dev(view, gpu(tokens), gpu(exp_lut), 9)
    for name, g, w in zip(("logprobs", "entropy", "tokens", "their logprobs"), got, ref.logprobs(z, tokens, exp_lut, 9)):
        same(g, w, name)
    same(backend.logsoftmax_dev(gpu(z), gpu(exp_lut), gpu(tokens)), got[0].cpu().numpy(), "logsoftmax_dev")
    assert (got[2][:, 0].cpu().numpy() == z.argmax(1)).all()
