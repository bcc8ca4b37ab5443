"""The operators of a serving step on the GPU against plain 64-bit forms
(tests/serving_ref.py), bit for bit: adapters beside a projection, attention
over a shared prefix, draft verification, and a step that runs them together.
All outputs are whole numbers, so every comparison is for equality."""
from __future__ import annotations

import numpy as np
import pytest

import serving_ref as ref
from conftest import case

pytestmark = pytest.mark.gpu


def rng(seed):
    return np.random.default_rng(seed)


def gauss16(r, shape, sigma):
    return np.clip(np.rint(r.normal(0, sigma, shape)), -32767, 32767).astype(np.int16)


def gpu(a):
    import torch
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def same(got, want, what):
    got = got.cpu().numpy()
    assert got.shape == want.shape and got.dtype == want.dtype, what
    bad = np.argwhere(got != want)
    assert not bad.size, f"{what}: {len(bad)} of {want.size} differ, first at {bad[0]}: {got[tuple(bad[0])]} != {want[tuple(bad[0])]}"


def dirty(ws):
    """A workspace's contents before a call mean nothing."""
    ws.fill_(0xA5)
    return ws


@pytest.fixture(scope="module")
def exp_lut():
    from myelith_amd.luts import exp_lut
    t = exp_lut()
    return t[:np.flatnonzero(t)[-1] + 1].copy()


# ---- adapters ------------------------------------------------------------------

def adapter_inputs(seed, M, N, K, rank, n, ids=None):
    r = rng(seed)
    g, gr = int(np.log2(73 * np.sqrt(K))), int(np.log2(73 * np.sqrt(rank)))
    return dict(x=gauss16(r, (M, K), 2000), W=r.integers(-128, 128, (N, K)).astype(np.int8),
                w_shifts=r.integers(g, g + 3, N).astype(np.uint8), act_frac=10,
                ids=(r.integers(-1, n + 1, M) if ids is None else np.asarray(ids)).astype(np.int32),
                A=r.integers(-128, 128, (n, rank, K)).astype(np.int8),
                a_shifts=r.integers(g, g + 3, (n, rank)).astype(np.uint8), mid_frac=10,
                B=r.integers(-128, 128, (n, N, rank)).astype(np.int8),
                b_shifts=r.integers(gr, gr + 3, (n, N)).astype(np.uint8))


def run_adapters(backend, s, out_frac=10, pc=None, **kw):
    import torch
    d = {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in s.items()}
    ws = dirty(backend.linear_w8a16_adapters_workspace(d["x"], d["W"], d["A"]))
    got = backend.linear_w8a16_adapters_dev(d["x"], d["W"], d["w_shifts"], d["act_frac"], d["ids"], d["A"], d["a_shifts"],
                                            d["mid_frac"], d["B"], d["b_shifts"], out_frac,
                                            out_frac_pc=gpu(pc), workspace=ws, **kw)
    torch.cuda.synchronize()
    return got


def want_adapters(s, out_frac=10, pc=None):
    return ref.adapters(**s, out_frac=out_frac if pc is None else pc.astype(np.int64))


@pytest.mark.parametrize("M,N,K,rank,n", [
    (1, 1, 1, 1, 1), (1, 37, 16, 3, 2), (1, 896, 896, 8, 3), (2, 64, 64, 16, 2), (3, 65, 130, 17, 4), (5, 130, 48, 1, 9),
    (15, 200, 896, 16, 40), (16, 256, 1024, 16, 16), (17, 129, 512, 24, 5), (33, 896, 4864, 8, 33), (7, 300, 18944, 64, 3),
    (40, 96, 3584, 256, 2), (70, 515, 320, 33, 7), (130, 1152, 896, 16, 3), (129, 72, 72, 100, 11), (600, 130, 256, 4, 1)])
def test_adapters(backend, M, N, K, rank, n):
    case(f"adapters M={M} N={N} K={K} rank={rank} n={n}")
    s = adapter_inputs(M + 7 * N + K, M, N, K, rank, n)
    same(run_adapters(backend, s), want_adapters(s), "scalar output scale")
    pc = rng(1).integers(7, 13, N).astype(np.uint8)
    same(run_adapters(backend, s, pc=pc), want_adapters(s, pc=pc), "per-channel output scale")


@pytest.mark.parametrize("ids", [[-1] * 20, [2] * 20, list(range(20)), [0] * 7 + [19] * 13, [3, 3, 1, 1, 3, 0] * 3 + [20, 2**31 - 1],
                                 [-2**31] * 19 + [4]])
def test_adapters_ids(backend, ids):
    """Rows without adapters, one for all, one each, runs, repeats and ids outside the range."""
    case(f"adapters ids {ids[:3]}..{ids[-2:]}")
    s = adapter_inputs(11, 20, 100, 192, 12, 20, ids)
    same(run_adapters(backend, s), want_adapters(s), "ids")


def test_adapters_runs_of_rows(backend):
    """The rows of a request follow one another and end inside any tile."""
    case("adapters runs")
    ids = np.repeat([4, -1, 0, 3, 2, 1], [37, 5, 64, 1, 90, 16])
    s = adapter_inputs(12, ids.size, 200, 448, 16, 5, ids)
    same(run_adapters(backend, s), want_adapters(s), "runs")


@pytest.mark.parametrize("act,mid,out", [(0, 0, 0), (10, 0, 20), (2, 14, 14), (0, 30, 0), (20, 4, 8)])
def test_adapters_scales_and_extremes(backend, act, mid, out):
    """Full-range operands; shifts to the left, of nothing and of everything."""
    case(f"adapters scales {act} {mid} {out}")
    s = adapter_inputs(13, 18, 70, 128, 20, 3)
    s["x"][:9] = -32768
    s["x"][9] = 32767
    s["A"][0] = -128
    s["B"][0] = -128
    s["B"][1] = 127
    s["a_shifts"] = rng(2).integers(0, 24, s["a_shifts"].shape).astype(np.uint8)
    s["b_shifts"] = rng(3).integers(0, 24, s["b_shifts"].shape).astype(np.uint8)
    s.update(act_frac=act, mid_frac=mid)
    same(run_adapters(backend, s, out), want_adapters(s, out), "scales")


def test_adapters_strided_rows_and_no_adapters(backend):
    import torch
    case("adapters strided")
    s = adapter_inputs(14, 21, 90, 96, 8, 4)
    wide = torch.zeros((21, 96 + 33), dtype=torch.int16, device="cuda")
    wide[:, 1:97] = gpu(s["x"])
    out = torch.full((21, 101), 77, dtype=torch.int16, device="cuda")
    want = want_adapters(s)
    d = dict(s, x=wide[:, 1:97])
    got = run_adapters(backend, d, out=out[:, 3:93])
    same(got, want, "strided")
    assert (out[:, :3] == 77).all() and (out[:, 93:] == 77).all()
    none = dict(s, A=s["A"][:0], a_shifts=s["a_shifts"][:0], B=s["B"][:0], b_shifts=s["b_shifts"][:0])
    same(run_adapters(backend, none), ref.linear(s["x"], s["W"], s["w_shifts"], 10, 10).astype(np.int16), "no adapters")
    empty = adapter_inputs(14, 0, 90, 96, 8, 4)
    assert run_adapters(backend, empty).shape == (0, 90)


# ---- attention over a shared prefix -----------------------------------------------

def attention_inputs(seed, seqs, rows, prefix, tail, H, KH, hd, slots=None, kscale=1024):
    r = rng(seed)
    S = seqs + 1
    return dict(q=gauss16(r, (seqs * rows, H, hd), 2048), kp=gauss16(r, (KH, prefix, hd), kscale),
                vp=gauss16(r, (KH, prefix, hd), 2000), kt=gauss16(r, (S, KH, tail, hd), kscale),
                vt=gauss16(r, (S, KH, tail, hd), 2000), lens=r.integers(0, tail + 1, seqs * rows).astype(np.int32),
                mult=round(2**15 / np.sqrt(hd)), shift=21, lut_shift=6, prob_frac=14, rows_per_seq=rows,
                slots=r.permutation(S)[:seqs].astype(np.int32) if slots is None else np.asarray(slots, np.int32))


def run_attention(backend, s, lut, **kw):
    import torch
    d = {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in s.items()}
    n = d["rows_per_seq"]
    ws = dirty(backend.attention_prefix_workspace(d["q"], d["kp"], d["kt"], n))
    got = backend.attention_prefix_dev(d["q"], d["kp"], d["vp"], d["kt"], d["vt"], d["lens"], d["mult"], d["shift"], gpu(lut),
                                       d["lut_shift"], d["prob_frac"], rows_per_seq=n, slots=d["slots"],
                                       max_tail=d.get("max_tail"), workspace=ws, **kw)
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("seqs,rows,prefix,tail,H,KH,hd", [
    (1, 1, 1, 0, 1, 1, 64), (1, 1, 0, 1, 2, 1, 64), (1, 1, 1, 1, 2, 2, 128), (2, 1, 15, 3, 14, 2, 64), (2, 1, 16, 16, 28, 4, 128),
    (3, 1, 17, 33, 8, 8, 64), (5, 2, 63, 65, 14, 2, 64), (4, 1, 64, 64, 28, 4, 128), (9, 1, 65, 5, 32, 4, 128),
    (1, 8, 127, 129, 28, 4, 128), (3, 5, 255, 30, 16, 1, 64), (2, 3, 256, 256, 33, 3, 128), (17, 1, 300, 40, 14, 2, 64),
    (6, 4, 513, 70, 28, 4, 128), (1, 1, 1025, 1, 40, 1, 128), (33, 1, 700, 20, 28, 4, 128), (2, 20, 130, 300, 12, 2, 64)])
def test_attention(backend, exp_lut, seqs, rows, prefix, tail, H, KH, hd):
    case(f"attention {seqs}x{rows} prefix={prefix} tail={tail} heads={H}/{KH} hd={hd}")
    s = attention_inputs(prefix + tail, seqs, rows, prefix, tail, H, KH, hd)
    same(run_attention(backend, s, exp_lut), ref.attention(**s, lut=exp_lut), "attention")


@pytest.mark.parametrize("prefix,tail,seqs,rows", [(9000, 300, 2, 1), (4097, 1, 20, 1), (40, 5000, 1, 3), (0, 3000, 3, 2)])
def test_attention_long(backend, exp_lut, prefix, tail, seqs, rows):
    case(f"attention long prefix={prefix} tail={tail}")
    s = attention_inputs(3, seqs, rows, prefix, tail, 14, 2, 64)
    same(run_attention(backend, s, exp_lut), ref.attention(**s, lut=exp_lut), "long")


@pytest.mark.parametrize("prefix,tail", [(50, 20), (0, 20), (50, 0), (0, 0), (1000, 400)])
def test_attention_rows_left_out_and_bad_slots(backend, exp_lut, prefix, tail):
    """Negative lengths, empty tails, lengths past the tails, the same slot twice, slots outside the cache."""
    case(f"attention left out prefix={prefix} tail={tail}")
    s = attention_inputs(21, 7, 2, prefix, tail, 14, 2, 64, slots=[3, 3, -1, 8, 0, 2**31 - 1, -2**31])
    s["lens"] = np.array([0, tail, -1, 2, 1, tail + 5, 2**31 - 1, -2**31, tail, -7, 3, 0, 1, -1], np.int32)
    want = ref.attention(**s, lut=exp_lut)
    same(run_attention(backend, s, exp_lut), want, "left out")
    assert not want[2].any() and not want[7].any()
    s["max_tail"] = tail // 2
    same(run_attention(backend, s, exp_lut), ref.attention(**s, lut=exp_lut), "max_tail")


@pytest.mark.parametrize("mult,shift,lut_shift,prob_frac", [(2896, 21, 6, 14), (2896, 30, 0, 8), (1, 9, 3, 0), (-4096, 22, 6, 14),
                                                           (2896, 5, 6, 14), (1 << 30, 40, 6, 14), (2896, 62, 6, 14), (0, 21, 6, 14),
                                                           (3, 0, 31, 13), (2896, 63, 6, 14)])
def test_attention_scales(backend, exp_lut, mult, shift, lut_shift, prob_frac):
    """Score scales on and off the 32-bit form's range (scores that wrap among them)."""
    case(f"attention scales {mult} {shift} {lut_shift} {prob_frac}")
    s = attention_inputs(22, 3, 2, 70, 30, 14, 2, 64)
    s.update(mult=mult, shift=shift, lut_shift=lut_shift, prob_frac=prob_frac)
    same(run_attention(backend, s, exp_lut), ref.attention(**s, lut=exp_lut), "scales")


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_extremes(backend, exp_lut, hd):
    """Operands at the ends of int16; keys all alike; one key that takes every weight."""
    case(f"attention extremes hd={hd}")
    s = attention_inputs(23, 4, 2, 150, 40, 8, 2, hd)
    s["q"][0], s["q"][1], s["q"][2] = -32768, 32767, 0
    s["kp"][0, ::2], s["kp"][0, 1::2] = -32768, 32767
    s["vp"][0, ::3], s["vp"][1] = -32768, 32767
    s["kt"][:, 0], s["vt"][:, 1] = -32768, -32768
    s["kp"][1, 77] = 20000
    for shift in (21, 36):
        s["shift"] = shift
        same(run_attention(backend, s, exp_lut), ref.attention(**s, lut=exp_lut), f"extremes shift {shift}")


@pytest.mark.parametrize("name", ["one", "zero", "negative", "short", "whole", "flat", "large"])
def test_attention_tables(backend, exp_lut, name):
    """Tables that leave nothing (the uniform split), of one entry, with negative and large entries."""
    from myelith_amd.luts import exp_lut as whole
    case(f"attention table {name}")
    lut = {"one": exp_lut[:1], "zero": np.zeros(5, np.int16), "short": exp_lut[:300], "whole": whole(),
           "negative": np.where(np.arange(exp_lut.size) % 3 == 1, -5, exp_lut).astype(np.int16),
           "flat": np.full(30000, 16384, np.int16), "large": np.full(9000, 32767, np.int16)}[name]
    for prefix, tail in ((90, 30), (700, 100)):
        s = attention_inputs(24, 3, 2, prefix, tail, 14, 2, 64)
        same(run_attention(backend, s, lut), ref.attention(**s, lut=lut), name)


def test_attention_strided_cache(backend, exp_lut):
    """Views of larger caches (a layer of [slot][layer][head][position], a prefix
    shorter than its buffer), q rows inside q/k/v rows, no slot table."""
    import torch
    case("attention strided")
    s = attention_inputs(25, 5, 1, 75, 33, 14, 2, 64)
    s["slots"] = np.arange(5, dtype=np.int32)
    want = ref.attention(**s, lut=exp_lut)
    d = {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in s.items()}
    S = d["kt"].shape[0]
    caches = []
    for t in (d["kt"], d["vt"]):
        c = torch.full((S, 3, 2, 50, 64), 31000, dtype=torch.int16, device="cuda")
        c[:, 1, :, :33] = t
        caches.append(c[:, 1, :, :33])
    pre = []
    for t in (d["kp"], d["vp"]):
        c = torch.full((2, 200, 64), -31000, dtype=torch.int16, device="cuda")
        c[:, 100:175] = t
        pre.append(c[:, 100:175])
    qkv = torch.full((5, 18, 64), 9, dtype=torch.int16, device="cuda")
    qkv[:, 2:16] = d["q"]
    out = torch.full((5, 18, 64), 9, dtype=torch.int16, device="cuda")
    backend.attention_prefix_dev(qkv[:, 2:16], pre[0], pre[1], caches[0], caches[1], d["lens"], d["mult"], d["shift"],
                                 gpu(exp_lut), 6, 14, out=out[:, 2:16])
    same(out[:, 2:16].contiguous(), want, "strided")
    assert (out[:, :2] == 9).all() and (out[:, 16:] == 9).all()


# ---- verification ----------------------------------------------------------------------

def verify_inputs(seed, B, k, V, spread=160, near=True):
    r = rng(seed)
    z = np.rint(r.normal(0, spread, (B, k + 1, V))).astype(np.int32)
    hot = r.integers(0, V, (B, k + 1, 4))
    np.put_along_axis(z, hot, r.integers(700, 1000, hot.shape).astype(np.int32), 2)
    d = (z[:, :k] + r.integers(-40, 41, (B, k, V))).astype(np.int32)
    t = hot[:, :k, 0] if near else r.integers(0, V, (B, k))
    return dict(target=z, draft=d, tokens=t.astype(np.int64),
                randoms=r.integers(0, 2**64, (B, k + 1), dtype=np.uint64))


def run_verify(backend, s, lut):
    import torch
    d = {k: gpu(v.view(np.int64) if v.dtype == np.uint64 else v) for k, v in s.items() if v is not None}
    table = gpu(lut)
    ws = dirty(backend.verify_drafts_workspace(d["target"], table, d.get("draft")))
    got = backend.verify_drafts_dev(d["target"], d["tokens"], d.get("randoms"), exp_lut=table, draft=d.get("draft"),
                                    n_draft=d.get("n_draft"), workspace=ws)
    torch.cuda.synchronize()
    return got


def check_verify(backend, s, lut, what):
    got, want = run_verify(backend, s, lut), ref.verify(lut=lut, **s)
    same(got[0], want[0], what + ": accepted")
    same(got[1], want[1], what + ": tokens")
    return want


@pytest.mark.parametrize("B,k,V", [(1, 0, 1), (1, 1, 1), (2, 0, 1000), (1, 4, 2), (3, 2, 63), (5, 3, 64), (2, 8, 1023), (4, 5, 1025),
                                   (20, 1, 4097), (9, 3, 8192), (2, 4, 16385), (3, 2, 32001), (1, 2, 152064)])
def test_verify(backend, exp_lut, B, k, V):
    case(f"verify B={B} k={k} V={V}")
    s = verify_inputs(B + k + V, B, k, V)
    check_verify(backend, s, exp_lut, "draft model")
    check_verify(backend, dict(s, draft=None), exp_lut, "lookup")
    check_verify(backend, s, None, "greedy")
    s["n_draft"] = rng(V).integers(-1, k + 2, B).astype(np.int32)
    for draft, lut, what in ((s["draft"], exp_lut, "draft model"), (None, exp_lut, "lookup"), (None, None, "greedy")):
        check_verify(backend, dict(s, draft=draft), lut, what + ", ragged")


def test_verify_greedy_follows_the_first_maximum(backend):
    case("verify greedy")
    s = verify_inputs(31, 40, 5, 700, spread=2)
    s["target"] = np.minimum(s["target"], 3)  # many ties
    s["tokens"] = s["target"][:, :5].argmax(2).astype(np.int64)
    s["tokens"][::3, 3] += 1
    want = check_verify(backend, s, None, "greedy")
    assert set(want[0]) == {3, 5}


@pytest.mark.parametrize("draft", [True, False])
def test_verify_random_numbers_at_their_ends(backend, exp_lut, draft):
    """0 accepts any token with weight, 2^64 - 1 the hardest; the last draws the first and the last weight."""
    case(f"verify random ends draft={draft}")
    for ends in ([0, 0], [2**64 - 1, 2**64 - 1], [2**64 - 1, 0], [2**63, 2**63 - 1]):
        s = verify_inputs(32, 6, 3, 3000, near=False)
        s["tokens"][:3] = s["target"][:3, :3].argmax(2)
        s["randoms"][:, :3], s["randoms"][:, 3] = ends
        check_verify(backend, s if draft else dict(s, draft=None), exp_lut, str(ends))


def test_verify_the_same_distribution_accepts_everything(backend, exp_lut):
    case("verify same distribution")
    s = verify_inputs(33, 12, 4, 2000)
    s["draft"] = s["target"][:, :4].copy()
    s["randoms"][:, :4] = 2**64 - 1
    assert (check_verify(backend, s, exp_lut, "same")[0] == 4).all()


def test_verify_nothing_left_and_bad_tokens(backend, exp_lut):
    """A rejected token without weight whose residual is empty, tokens outside the
    vocabulary, masked rows, tables of zeros and with negative entries."""
    case("verify nothing left")
    s = verify_inputs(34, 8, 2, 500)
    s["draft"] = s["target"][:, :2].copy()
    s["tokens"][0] = s["target"][0, :2].argmin(1)
    s["tokens"][1], s["tokens"][2], s["tokens"][3] = -1, 500, 2**62
    s["tokens"][4] = -2**63
    s["target"][5] = -2**31                                # nothing but the mask
    s["target"][6, :, 1:], s["target"][6, :, 0] = -2**31, 2**31 - 1
    s["draft"][7] = -2**31
    for lut in (exp_lut, np.zeros(4, np.int16), np.where(np.arange(900) % 8 == 4, -3, exp_lut[:900]).astype(np.int16),
                np.full(32768, 32767, np.int16), exp_lut[:1]):
        check_verify(backend, s, lut, f"draft model, table of {lut.size}")
        check_verify(backend, dict(s, draft=None), lut, f"lookup, table of {lut.size}")
    check_verify(backend, s, None, "greedy")


def test_verify_flat_rows(backend, exp_lut):
    """Every logit the same, or of two values: the sums at their largest."""
    case("verify flat")
    for V in (1000, 20000):
        s = verify_inputs(35, 3, 2, V)
        s["target"][:] = 7
        s["draft"][:, :, V // 2:] = -5
        s["draft"][:, :, :V // 2] = 60
        check_verify(backend, s, exp_lut, "flat")
        check_verify(backend, s, np.full(2000, 32767, np.int16), "flat, large entries")


def test_verify_strided_rows(backend, exp_lut):
    import torch
    case("verify strided")
    s = verify_inputs(36, 4, 3, 777)
    want = ref.verify(lut=exp_lut, **s)
    rows = torch.full((16, 801), 2**30, dtype=torch.int32, device="cuda")
    rows[:, 5:782] = gpu(s["target"]).reshape(16, 777)
    drafts = torch.full((12, 778), 2**30, dtype=torch.int32, device="cuda")
    drafts[:, 1:] = gpu(s["draft"]).reshape(12, 777)
    got = backend.verify_drafts_dev(rows.view(4, 4, 801)[:, :, 5:782], gpu(s["tokens"]), gpu(s["randoms"].view(np.int64)),
                                    exp_lut=gpu(exp_lut), draft=drafts.view(4, 3, 778)[:, :, 1:])
    same(got[0], want[0], "accepted")
    same(got[1], want[1], "tokens")


# ---- refusals ---------------------------------------------------------------------------

def test_refusals(backend, exp_lut):
    import torch
    case("serving refusals")
    s = adapter_inputs(41, 3, 40, 64, 8, 2)
    small = torch.empty(8, dtype=torch.uint8, device="cuda")
    d = {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in s.items()}
    args = (d["x"], d["W"], d["w_shifts"], 10, d["ids"], d["A"], d["a_shifts"], 10, d["B"], d["b_shifts"], 10)
    with pytest.raises(ValueError, match="workspace"):
        backend.linear_w8a16_adapters_dev(*args, workspace=small)
    t = {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in attention_inputs(42, 2, 1, 20, 8, 4, 2, 64).items()}

    def att(**over):
        a = dict(t, **over)
        return backend.attention_prefix_dev(a["q"], a["kp"], a["vp"], a["kt"], a["vt"], a["lens"], 1, 20, gpu(exp_lut), 6,
                                            a.get("prob_frac", 14), slots=a["slots"], workspace=a.get("workspace"))
    with pytest.raises(ValueError, match="workspace"):
        att(workspace=small)
    with pytest.raises(ValueError, match="prob_frac"):
        att(prob_frac=15)
    from myelith_amd.backend import MylError
    with pytest.raises(MylError, match="head_dim"):
        att(**{k: t[k][..., :32].contiguous() for k in ("q", "kp", "vp", "kt", "vt")})
    long = torch.zeros((2, 65530, 64), dtype=torch.int16, device="cuda")
    with pytest.raises(ValueError, match="65536"):
        att(kp=long, vp=long)
    odd = torch.zeros(2 * 4 * 64 + 1, dtype=torch.int16, device="cuda")[1:].view(2, 4, 64)
    with pytest.raises(ValueError, match="aligned"):
        att(q=odd)
    v = verify_inputs(43, 2, 2, 100)
    z, tok, rnd = gpu(v["target"]), gpu(v["tokens"]), gpu(v["randoms"].view(np.int64))
    with pytest.raises(ValueError, match="workspace"):
        backend.verify_drafts_dev(z, tok, rnd, exp_lut=gpu(exp_lut), workspace=small)
    with pytest.raises(ValueError, match="table"):
        backend.verify_drafts_dev(z, tok, rnd, exp_lut=torch.zeros(32769, dtype=torch.int16, device="cuda"))
    assert att().shape == (2, 4, 64)  # the context is as good as before


# ---- the form that shares the keys between rows, at the sizes that one launch takes with fewer heads ----

@pytest.mark.parametrize("seqs,rows,prefix,tail,H,KH,hd", [
    (1, 1, 1, 0, 9, 1, 64), (1, 1, 0, 1, 10, 1, 64), (1, 1, 1, 1, 18, 2, 128), (2, 1, 15, 3, 18, 2, 64), (2, 1, 16, 16, 36, 4, 128),
    (3, 1, 17, 33, 9, 1, 64), (5, 2, 63, 65, 20, 2, 64), (4, 1, 64, 64, 18, 2, 128), (9, 1, 65, 5, 36, 4, 128), (1, 8, 127, 129, 9, 1, 128),
    (700, 1, 40, 9, 14, 2, 64)])
def test_attention_many_heads_or_rows(backend, exp_lut, seqs, rows, prefix, tail, H, KH, hd):
    case(f"attention {seqs}x{rows} prefix={prefix} tail={tail} heads={H}/{KH} hd={hd}")
    s = attention_inputs(prefix + tail, seqs, rows, prefix, tail, H, KH, hd)
    same(run_attention(backend, s, exp_lut), ref.attention(**s, lut=exp_lut), "attention")


@pytest.mark.parametrize("prefix,tail", [(50, 20), (0, 20), (50, 0), (0, 0)])
def test_attention_many_heads_left_out_and_bad_slots(backend, exp_lut, prefix, tail):
    case(f"attention many heads left out prefix={prefix} tail={tail}")
    s = attention_inputs(24, 7, 2, prefix, tail, 18, 2, 64, slots=[3, 3, -1, 8, 0, 2**31 - 1, -2**31])
    s["lens"] = np.array([0, tail, -1, 2, 1, tail + 5, 2**31 - 1, -2**31, tail, -7, 3, 0, 1, -1], np.int32)
    same(run_attention(backend, s, exp_lut), ref.attention(**s, lut=exp_lut), "left out")


@pytest.mark.parametrize("H", [8, 18])
@pytest.mark.parametrize("mult,shift,lut_shift,prob_frac", [(2896, 30, 0, 8), (1, 9, 3, 0), (-4096, 22, 6, 14), (1 << 30, 40, 6, 14),
                                                           (0, 21, 6, 14), (3, 0, 31, 13), (2896, 63, 6, 14)])
def test_attention_scales_of_both_forms(backend, exp_lut, H, mult, shift, lut_shift, prob_frac):
    case(f"attention scales H={H} {mult} {shift} {lut_shift} {prob_frac}")
    s = attention_inputs(25, 3, 2, 70, 30, H, 2, 128)
    s.update(mult=mult, shift=shift, lut_shift=lut_shift, prob_frac=prob_frac)
    same(run_attention(backend, s, exp_lut), ref.attention(**s, lut=exp_lut), "scales")


@pytest.mark.parametrize("H", [8, 18])
@pytest.mark.parametrize("table", ["one", "negative", "zero", "long"])
def test_attention_tables_of_both_forms(backend, H, table):
    """Tables of one entry, with negative entries, without weight (a uniform split), and of 32768."""
    case(f"attention table {table} H={H}")
    lut = {"one": np.array([5], np.int16), "negative": rng(7).integers(-300, 300, 500).astype(np.int16), "zero": np.zeros(3, np.int16),
           "long": rng(8).integers(0, 32768, 32768).astype(np.int16)}[table]
    s = attention_inputs(26, 3, 2, 70, 30, H, 2, 64)
    s.update(lut_shift=0 if table == "long" else 3)
    same(run_attention(backend, s, lut), ref.attention(**s, lut=lut), table)


# ---- many rows, long offsets --------------------------------------------------------------

@pytest.mark.parametrize("M,N,K,rank,n", [(1500, 520, 64, 8, 300), (257, 70, 130, 12, 2), (1030, 33, 96, 70, 17)])
def test_adapters_many_rows(backend, M, N, K, rank, n):
    """Several windows of rows, adapters with rows in each, more columns than a block takes at once."""
    case(f"adapters many rows M={M} N={N} K={K} rank={rank} n={n}")
    s = adapter_inputs(M, M, N, K, rank, n)
    same(run_adapters(backend, s), want_adapters(s), "many rows")
    s["ids"] = np.repeat(rng(5).integers(-1, n, M // 50 + 1), 50)[:M].astype(np.int32)
    same(run_adapters(backend, s), want_adapters(s), "runs")


def test_adapters_past_4_gib(backend):
    """Adapters whose rows lie more than 2^32 bytes into A."""
    import torch
    case("adapters past 4 GiB")
    n, rank, K = 270, 256, 65472
    ids = [269, 0, 260]
    s = adapter_inputs(51, 3, 8, K, 1, n, ids)
    A = torch.empty((n, rank, K), dtype=torch.int8, device="cuda")
    for i in ids:
        A[i].random_(-128, 128)
    s.update(A=A, a_shifts=np.full((n, rank), 14, np.uint8), B=rng(6).integers(-128, 128, (n, 8, rank)).astype(np.int8),
             b_shifts=np.full((n, 8), 10, np.uint8))
    got = run_adapters(backend, s)
    keep = dict(s, A=np.stack([A[i].cpu().numpy() for i in ids]), ids=np.arange(3))
    for name in ("a_shifts", "B", "b_shifts"):
        keep[name] = s[name][ids]
    same(got, want_adapters(keep), "past 4 GiB")


def test_attention_past_4_gib(backend, exp_lut):
    """Prefix heads, tail slots and rows of queries and outputs more than 2^32 bytes apart."""
    import torch
    case("attention past 4 GiB")
    P, T, far = 70, 40, 1 << 30
    kv = torch.empty(2 * far + (1 << 21), dtype=torch.int16, device="cuda")
    rows = torch.zeros(2 * far + (1 << 21), dtype=torch.int16, device="cuda")
    s = attention_inputs(52, 3, 1, P, T, 4, 2, 64, slots=[2, 0, 1])
    s["kt"], s["vp"] = s["kt"][:3], s["kp"]
    s["vt"] = s["kt"]
    prefix = kv.as_strided((2, P, 64), (2 * far, 64, 1))
    tails = kv.as_strided((3, 2, T, 64), (far, T * 64, 64, 1), 1 << 20)
    q, out = (rows.as_strided((3, 4, 64), (far, 64, 1), at) for at in (0, 1 << 20))
    for t, v in ((prefix, s["kp"]), (tails, s["kt"]), (q, s["q"])):
        t.copy_(gpu(v))
    got = backend.attention_prefix_dev(q, prefix, prefix, tails, tails, gpu(s["lens"]), s["mult"], s["shift"], gpu(exp_lut), 6, 14,
                                       slots=gpu(s["slots"]), out=out)
    torch.cuda.synchronize()
    same(got, ref.attention(**s, lut=exp_lut), "past 4 GiB")
    assert int(torch.count_nonzero(rows)) == int(torch.count_nonzero(q)) + int(torch.count_nonzero(out))


def test_verify_past_4_gib(backend, exp_lut):
    import torch
    case("drafts past 4 GiB")
    s = verify_inputs(53, 2, 1, 9000)
    far = 1 << 29
    buf = torch.empty(3 * far + (1 << 20), dtype=torch.int32, device="cuda")
    target = buf.as_strided((2, 2, 9000), (2 * far, far, 1))
    draft = buf.as_strided((2, 1, 9000), (3 * far, 3 * far, 1), 1 << 16)
    target.copy_(gpu(s["target"]))
    draft.copy_(gpu(s["draft"]))
    got = backend.verify_drafts_dev(target, gpu(s["tokens"]), gpu(s["randoms"].view(np.int64)), exp_lut=gpu(exp_lut), draft=draft)
    torch.cuda.synchronize()
    want = ref.verify(**s, lut=exp_lut)
    same(got[0], want[0], "accepted")
    same(got[1], want[1], "tokens")


# ---- a serving step: the operators together -----------------------------------------------

class Step:
    """A projection with adapters, attention behind the shared prefix, logits and the check of
    the drafts, for seqs sequences of k drafts; one workspace serves all calls in turn."""

    def __init__(self, backend, exp_lut, seqs=5, k=3, seed=61, prefix=150):
        import torch
        self.b, self.lut, self.k, self.seqs = backend, exp_lut, k, seqs
        H, hd, V, rows = 14, 64, 1500, seqs * (k + 1)
        r = rng(seed)
        self.ad = adapter_inputs(seed, rows, H * hd, 448, 16, 4, np.repeat(r.integers(-1, 4, seqs), k + 1))
        self.at = attention_inputs(seed + 1, seqs, k + 1, prefix, 33, H, 2, hd)
        self.Wv = r.integers(-128, 128, (V, H * hd)).astype(np.int8)
        self.v_shifts = np.full(V, 9, np.uint8)
        self.d = {n: gpu(v) for n, v in [*self.ad.items(), *self.at.items(), ("Wv", self.Wv), ("v_shifts", self.v_shifts)]
                  if isinstance(v, np.ndarray)}
        self.table = gpu(exp_lut)
        self.proj = torch.empty((rows, H * hd), dtype=torch.int16, device="cuda")
        self.mix = torch.empty((rows, H, hd), dtype=torch.int16, device="cuda")
        self.logits = torch.empty((rows, V), dtype=torch.int32, device="cuda")
        self.accepted = torch.empty(seqs, dtype=torch.int32, device="cuda")
        self.tokens = torch.empty((seqs, k + 1), dtype=torch.int64, device="cuda")
        self.target = self.logits.view(seqs, k + 1, V)
        d = self.d
        spaces = [backend.linear_w8a16_adapters_workspace(d["x"], d["W"], d["A"]),
                  backend.attention_prefix_workspace(self.mix, d["kp"], d["kt"], k + 1),
                  backend.verify_drafts_workspace(self.target, self.table)]
        self.ws = dirty(max(spaces, key=lambda t: t.numel()))
        self.new_inputs(seed)

    def new_inputs(self, seed):
        import torch
        r = rng(seed)
        self.ad["x"] = gauss16(r, self.ad["x"].shape, 2000)
        self.at["lens"] = (r.integers(0, 30, (self.seqs, 1)) + np.arange(self.k + 1)).reshape(-1).astype(np.int32)
        drafts = r.integers(0, 1500, (self.seqs, self.k)).astype(np.int64)
        self.randoms = r.integers(0, 2**64, (self.seqs, self.k + 1), dtype=np.uint64)
        for name, v in (("x", self.ad["x"]), ("lens", self.at["lens"]), ("drafts", drafts), ("randoms", self.randoms.view(np.int64))):
            if name in self.d:
                self.d[name].copy_(gpu(v))
            else:
                self.d[name] = gpu(v)
        torch.cuda.synchronize()

    def project_and_attend(self):
        d, b = self.d, self.b
        b.linear_w8a16_adapters_dev(d["x"], d["W"], d["w_shifts"], 10, d["ids"], d["A"], d["a_shifts"], 10, d["B"], d["b_shifts"], 10,
                                    out=self.proj, workspace=self.ws)
        b.attention_prefix_dev(self.proj.view(self.mix.shape), d["kp"], d["vp"], d["kt"], d["vt"], d["lens"], self.at["mult"],
                               self.at["shift"], self.table, 6, 14, rows_per_seq=self.k + 1, slots=d["slots"], out=self.mix, workspace=self.ws)

    def to_logits(self):
        """And a first draft that the target is fond of."""
        self.b.logits_dev(self.mix.view(self.proj.shape), self.d["Wv"], self.d["v_shifts"], 10, 6, out=self.logits)
        self.d["drafts"][:, 0] = self.target[:, 0].argmax(-1)

    def check_drafts(self):
        self.b.verify_drafts_dev(self.target, self.d["drafts"], self.d["randoms"], exp_lut=self.table, accepted=self.accepted,
                                 out=self.tokens, workspace=self.ws)

    def check(self, what):
        """Every stage against its plain form (the logits, which other tests check, as they are)."""
        import torch
        torch.cuda.synchronize()
        proj = want_adapters(self.ad)
        same(self.proj, proj, f"{what}: projection")
        same(self.mix, ref.attention(**dict(self.at, q=proj.reshape(self.mix.shape)), lut=self.lut), f"{what}: attention")
        z = self.target.cpu().numpy()
        want = ref.verify(z, self.d["drafts"].cpu().numpy(), self.randoms, lut=self.lut)
        same(self.accepted, want[0], f"{what}: accepted")
        same(self.tokens, want[1], f"{what}: tokens")
        return want


@pytest.mark.parametrize("prefix", [150, 900])
def test_serving_step(backend, exp_lut, prefix):
    case("serving step")
    step = Step(backend, exp_lut, prefix=prefix)
    for turn in range(3):
        case(f"serving step, turn {turn}")
        step.project_and_attend()
        step.to_logits()
        step.check_drafts()
        accepted, tokens = step.check(f"turn {turn}")
        assert ((tokens >= 0).sum(1) == accepted + 1).all()
        step.new_inputs(70 + turn)


@pytest.mark.parametrize("prefix", [150, 900])
def test_serving_step_captured(backend, exp_lut, prefix):
    """Two captured graphs on one workspace, replayed several times with eager work, new inputs
    and synchronisations between."""
    import torch
    case("serving step captured")
    step = Step(backend, exp_lut, seed=62, prefix=prefix)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    try:
        with torch.cuda.stream(stream):
            backend.use_torch_stream()
            step.project_and_attend()
            step.to_logits()
            step.check_drafts()
        torch.cuda.synchronize()
        graphs = []
        for part in (step.project_and_attend, step.check_drafts):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                part()
            graphs.append(g)
        torch.cuda.synchronize()
        for turn in range(4):
            case(f"replay {turn}")
            step.new_inputs(80 + turn)
            step.ws.fill_(turn + 1)
            for t in (step.proj, step.mix, step.logits, step.accepted, step.tokens):
                t.fill_(-7)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                backend.use_torch_stream()
                graphs[0].replay()
                step.to_logits()
                graphs[1].replay()
                torch.cuda.synchronize()
            step.check(f"replay {turn}")
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()


def test_two_steps_at_once(backend, exp_lut):
    """Two contexts on two streams of their own, each with its workspace, side by side."""
    import torch
    from myelith_amd.backend import RocmBackend
    case("two steps at once")
    other = RocmBackend(0)
    try:
        steps = [Step(backend, exp_lut, seed=63), Step(other, exp_lut, seqs=9, k=1, seed=64, prefix=1200)]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                s.b.use_torch_stream()
        for _ in range(10):
            for s, stream in zip(steps, streams):
                with torch.cuda.stream(stream):
                    s.project_and_attend()
                    s.to_logits()
                    s.check_drafts()
        for i, s in enumerate(steps):
            s.check(f"step {i}")
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()
        other.close()


def test_calls_without_workspace_or_outputs(backend, exp_lut):
    """The calls' own workspaces and outputs, on the context's stream and on another than torch's."""
    import torch
    case("own workspaces")
    s, t, v = adapter_inputs(65, 9, 70, 96, 8, 3), attention_inputs(66, 3, 2, 90, 20, 4, 2, 64), verify_inputs(67, 3, 2, 700)
    da, dt = ({k: gpu(x) if isinstance(x, np.ndarray) else x for k, x in y.items()} for y in (s, t))
    z, tok, rnd, table = gpu(v["target"]), gpu(v["tokens"]), gpu(v["randoms"].view(np.int64)), gpu(exp_lut)
    draft = gpu(v["draft"])
    side = torch.cuda.Stream()
    try:
        for where in ("torch's stream", "another stream"):
            torch.cuda.synchronize()
            if where == "another stream":
                with torch.cuda.stream(side):
                    backend.use_torch_stream()
            for _ in range(3):  # the memory of a call that has ended may be handed to the next
                a = backend.linear_w8a16_adapters_dev(da["x"], da["W"], da["w_shifts"], 10, da["ids"], da["A"], da["a_shifts"], 10,
                                                      da["B"], da["b_shifts"], 10)
                b = backend.attention_prefix_dev(dt["q"], dt["kp"], dt["vp"], dt["kt"], dt["vt"], dt["lens"], dt["mult"], dt["shift"],
                                                 table, 6, 14, rows_per_seq=2, slots=dt["slots"])
                c = backend.verify_drafts_dev(z, tok, rnd, exp_lut=table, draft=draft)
            torch.cuda.synchronize()
            same(a, want_adapters(s), where)
            same(b, ref.attention(**t, lut=exp_lut), where)
            want = ref.verify(**v, lut=exp_lut)
            same(c[0], want[0], where)
            same(c[1], want[1], where)
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()


def test_adapters_odd_addresses(backend):
    """Adapters, shifts and rows that start anywhere; an odd K and rank."""
    import torch
    case("adapters odd addresses")
    s = adapter_inputs(71, 37, 333, 1031, 5, 6)

    def shifted(a):
        t = torch.zeros(a.size + 3, dtype=torch.from_numpy(a[:0].copy()).dtype, device="cuda")
        t[1:1 + a.size] = gpu(a).reshape(-1)
        return t[1:1 + a.size].view(a.shape)

    d = dict(s, **{k: shifted(s[k]) for k in ("x", "A", "a_shifts", "B", "b_shifts")})
    pc = rng(9).integers(7, 13, 333).astype(np.uint8)
    same(run_adapters(backend, d), want_adapters(s), "odd addresses")
    same(run_adapters(backend, d, pc=pc), want_adapters(s, pc=pc), "odd addresses, per-channel output scale")


def test_one_context_on_two_streams(backend, exp_lut):
    """Calls of one context on two streams, side by side, each step with its workspace."""
    import torch
    case("one context on two streams")
    steps = [Step(backend, exp_lut, seed=72), Step(backend, exp_lut, seqs=3, k=2, seed=73, prefix=800)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    try:
        for s in steps:
            s.project_and_attend()
            s.to_logits()
        torch.cuda.synchronize()
        for _ in range(10):
            for s, stream in zip(steps, streams):
                with torch.cuda.stream(stream):
                    backend.use_torch_stream()
                    s.project_and_attend()
                    s.check_drafts()
        for i, s in enumerate(steps):
            s.check(f"step {i}")
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()
