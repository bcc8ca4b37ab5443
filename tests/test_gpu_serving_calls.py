"""Calls of a serving step's operators on the GPU that their documentation
allows and that differ from an ordinary step's in how the operands lie, how
large they are or which stream they come from; every comparison is for equality."""
from __future__ import annotations

import numpy as np
import pytest

import serving_ref as ref
from conftest import case
from test_gpu_serving import (Step, adapter_inputs, attention_inputs, dirty, exp_lut, gauss16, gpu, rng, run_adapters, run_attention, run_verify,  # noqa: F401
                              same, verify_inputs, want_adapters)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prefix", [70, 700])
def test_tails_that_all_slots_share(backend, exp_lut, prefix):
    """A slot stride of 0: every sequence continues with the same tail."""
    case(f"attention shared tail prefix={prefix}")
    s = attention_inputs(81, 6, 2, prefix, 30, 14, 2, 64)
    s["kt"][:], s["vt"][:] = s["kt"][:1], s["vt"][:1]
    d = dict(s, kt=gpu(s["kt"][:1]).expand(s["kt"].shape), vt=gpu(s["vt"][:1]).expand(s["vt"].shape))
    same(run_attention(backend, d, exp_lut), ref.attention(**s, lut=exp_lut), "shared tail")


@pytest.mark.parametrize("torchs", ["null", "side"])
@pytest.mark.parametrize("context", ["own", "side"])
def test_allocated_memory_still_in_use_on_torchs_stream(backend, torchs, context):
    """A temporary that torch's queued kernels still read is freed just before a call on
    another stream, which takes its memory for the output."""
    import torch
    case(f"memory in use on torch's {torchs} stream, the context on its {context} one")
    M, N = 64, 16384
    s = adapter_inputs(82, M, N, 64, 8, 3)
    d = {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in s.items()}
    args = (d["x"], d["W"], d["w_shifts"], 10, d["ids"], d["A"], d["a_shifts"], 10, d["B"], d["b_shifts"], 10)
    ws = backend.linear_w8a16_adapters_workspace(d["x"], d["W"], d["A"])
    a = torch.ones((8192, 8192), dtype=torch.float32, device="cuda")
    product = torch.empty_like(a)
    current = torch.cuda.default_stream() if torchs == "null" else torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(torch.cuda.default_stream() if context == "own" else torch.cuda.Stream()):
            backend.use_torch_stream()  # the null stream leaves a context its own
        for turn in range(3):
            with torch.cuda.stream(current):
                torch.cuda.empty_cache()
                seen = torch.empty((M, N), dtype=torch.int16, device="cuda")
                temporary = torch.full((M, N), 1000 + turn, dtype=torch.int16, device="cuda")
                torch.cuda.synchronize()
                for _ in range(4):  # some ten milliseconds each
                    torch.mm(a, a, out=product)
                seen.copy_(temporary)
                place = temporary.data_ptr()
                del temporary
                out = backend.linear_w8a16_adapters_dev(*args, workspace=ws)
                torch.cuda.synchronize()
                assert out.data_ptr() == place  # the memory is the temporary's
                assert (seen == 1000 + turn).all()
                same(out, want_adapters(s), f"turn {turn}")
                del out, seen
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()


def test_allocating_in_a_capture_of_both_streams(backend):
    """The context's stream forked off the captured one: memory and launch are the graph's."""
    import torch
    case("capture of two streams")
    s = adapter_inputs(83, 20, 90, 128, 8, 4)
    d = {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in s.items()}
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(side):
            backend.use_torch_stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=main):
            side.wait_stream(main)
            out = backend.linear_w8a16_adapters_dev(d["x"], d["W"], d["w_shifts"], 10, d["ids"], d["A"], d["a_shifts"], 10, d["B"],
                                                    d["b_shifts"], 10)
            main.wait_stream(side)
        for turn in range(4):
            s["x"] = gauss16(rng(84 + turn), s["x"].shape, 2000)
            d["x"].copy_(gpu(s["x"]))
            out.fill_(-7)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            same(out, want_adapters(s), f"replay {turn}")
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()


# ---- more rows than a grid's second dimension holds -----------------------------------------

def want_adapters_by_id(s, out_frac=10):
    """want_adapters, the rows of an adapter together."""
    out = ref.linear(s["x"], s["W"], s["w_shifts"], 10, out_frac)
    for a in range(s["A"].shape[0]):
        rows = np.flatnonzero(s["ids"] == a)
        u = ref.linear(s["x"][rows], s["A"][a], s["a_shifts"][a], 10, 10)
        out[rows] += ref.linear(u, s["B"][a], s["b_shifts"][a], 10, out_frac)
    return ref.clamp16(out).astype(np.int16)


@pytest.mark.parametrize("M,N,K", [(65600, 5, 64), (65600, 3, 33), (65535, 2, 16), (65536, 7, 192), (131200, 2, 17)])
def test_adapters_past_65535_rows(backend, M, N, K):
    """Rows of byte planes (K a multiple of 64), of the plain sums (K 33, 17) and of the tiles between."""
    case(f"adapters M={M} N={N} K={K}")
    s = adapter_inputs(M + K, M, N, K, 4, 6)
    same(run_adapters(backend, s), want_adapters_by_id(s), "many rows")


@pytest.mark.parametrize("K", [64, 33])
def test_products_past_65535_rows(backend, K):
    """The projection itself and the sums it is made of."""
    case(f"products past 65535 rows K={K}")
    r = rng(K)
    x, W = gauss16(r, (65700, K), 2000), r.integers(-128, 128, (3, K)).astype(np.int8)
    shifts = np.array([8, 9, 10], np.uint8)
    same(backend.linear_w8a16_dev(gpu(x), gpu(W), gpu(shifts), 10, 10), ref.linear(x, W, shifts, 10, 10).astype(np.int16), "projection")
    same(backend.dot_i8_i16_dev(gpu(x), gpu(W)), ref.dots(x, W), "sums")


def test_adapters_planes_past_4_gib(backend):
    """Rows whose byte planes lie more than 2^32 bytes into the workspace."""
    import torch
    case("adapters planes past 4 GiB")
    M, N, K = 131400, 6, 16448
    assert 2 * M * K > 2**32
    few = adapter_inputs(85, 40, N, K, 4, 3)
    x = torch.empty((M, K), dtype=torch.int16, device="cuda")
    x.random_(-3000, 3001)
    ids = rng(86).integers(-1, 4, M)
    got = run_adapters(backend, dict(few, x=x, ids=ids.astype(np.int32))).cpu().numpy()
    at = np.unique(np.concatenate([rng(87).integers(0, M, 300), [0, 65534, 65535, 65536, 131069, 131070, 131071, M - 1]]))
    keep = dict(few, x=x[torch.from_numpy(at).cuda()].cpu().numpy(), ids=ids[at])
    bad = np.flatnonzero((got[at] != want_adapters_by_id(keep)).any(1))
    assert not bad.size, at[bad]


# ---- a workspace kept from the largest step ----------------------------------------------------

@pytest.mark.parametrize("rows", [114, 113, 100, 57, 16, 3, 1])
def test_adapters_in_the_workspace_of_more_rows(backend, rows):
    case(f"adapters workspace kept, {rows} rows")
    s = adapter_inputs(88, 120, 4608, 3584, 16, 24)
    d = {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in s.items()}
    ws = dirty(backend.linear_w8a16_adapters_workspace(d["x"], d["W"], d["A"]))
    got = backend.linear_w8a16_adapters_dev(d["x"][:rows], d["W"], d["w_shifts"], 10, d["ids"][:rows], d["A"], d["a_shifts"], 10, d["B"],
                                            d["b_shifts"], 10, workspace=ws)
    same(got, want_adapters(dict(s, x=s["x"][:rows], ids=s["ids"][:rows])), "fewer rows")


@pytest.mark.parametrize("seqs,tail", [(1, 1856), (1, 1792), (2, 1792), (2, 450), (1, 448), (2, 0)])
def test_attention_in_the_workspace_of_longer_tails(backend, exp_lut, seqs, tail):
    """The workspace of two sequences at the tails' capacity, for fewer and for shorter tails."""
    case(f"attention workspace kept, {seqs} sequences, tails of {tail}")
    s = attention_inputs(89, 2, 1, 1000, 1856, 28, 4, 128)
    d = {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in s.items()}
    ws = dirty(backend.attention_prefix_workspace(d["q"], d["kp"], d["kt"]))
    s.update(q=s["q"][:seqs], lens=np.minimum(s["lens"][:seqs], tail), slots=s["slots"][:seqs], max_tail=tail)
    got = backend.attention_prefix_dev(d["q"][:seqs], d["kp"], d["vp"], d["kt"], d["vt"], gpu(s["lens"]), s["mult"], s["shift"], gpu(exp_lut), 6, 14,
                                       slots=gpu(s["slots"]), max_tail=tail, workspace=ws)
    same(got, ref.attention(**s, lut=exp_lut), "shorter tails")
    own = backend.attention_prefix_workspace(d["q"][:seqs], d["kp"], d["kt"], max_tail=tail)
    assert own.numel() <= ws.numel()
    same(backend.attention_prefix_dev(d["q"][:seqs], d["kp"], d["vp"], d["kt"], d["vt"], gpu(s["lens"]), s["mult"], s["shift"], gpu(exp_lut), 6, 14,
                                      slots=gpu(s["slots"]), max_tail=tail, workspace=dirty(own)), ref.attention(**s, lut=exp_lut), "own workspace")


@pytest.mark.parametrize("entries", [1, 2, 3, 7, 8, 9, 15, 17, 2047, 2049, 2661, 8191, 8193, 16385, 32767])
def test_tables_that_end_inside_a_load(backend, entries):
    """The last entry counts and what lies behind it does not, wherever the table ends."""
    case(f"attention table of {entries}")
    import torch
    lut = rng(entries).integers(1, 32768, entries).astype(np.int16)
    behind = torch.full((entries + 64,), 32767, dtype=torch.int16, device="cuda")
    behind[:entries] = gpu(lut)
    s = attention_inputs(90, 3, 1, 500, 40, 18, 2, 64)
    s["lut_shift"] = 0
    # a scale at which some score lies at the table's last entry and others behind it
    spread = np.abs(ref.dots(s["q"].reshape(-1, 64), s["kp"].reshape(-1, 64))).max()
    s["mult"] = max(1, int(entries * 2.0**s["shift"] / spread))
    without = np.append(lut[:-1], 0).astype(np.int16)
    while ((want := ref.attention(**s, lut=lut)) == ref.attention(**s, lut=without)).all():
        s["mult"] += 1
    d = {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in s.items()}
    got = backend.attention_prefix_dev(d["q"], d["kp"], d["vp"], d["kt"], d["vt"], d["lens"], s["mult"], s["shift"], behind[:entries],
                                       s["lut_shift"], 14, slots=d["slots"])
    same(got, want, f"{entries} entries")


# ---- steps side by side ---------------------------------------------------------------------------

def junk(step):
    """Nothing that a step wrote before is left."""
    for t in (step.proj, step.mix, step.accepted, step.tokens):
        t.fill_(-7)
    dirty(step.ws)


@pytest.mark.parametrize("contexts", [1, 2])
def test_each_of_two_streams_writes_all_of_its_outputs(backend, exp_lut, contexts):
    """Two steps on two streams, of one context or of one each: the last turn starts from
    outputs and workspaces that hold nothing of the turns before."""
    import torch
    from myelith_amd.backend import RocmBackend
    case(f"two streams, {contexts} contexts")
    other = backend if contexts == 1 else RocmBackend(0)
    try:
        steps = [Step(backend, exp_lut, seed=91), Step(other, exp_lut, seqs=4, k=2, seed=92, prefix=900)]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for s in steps:
            s.project_and_attend()
            s.to_logits()
        torch.cuda.synchronize()
        for turn in range(6):
            case(f"turn {turn}")
            if turn in (0, 5):
                torch.cuda.synchronize()
                for s in steps:
                    junk(s)
                torch.cuda.synchronize()
            for s, stream in zip(steps, streams):
                with torch.cuda.stream(stream):
                    if contexts == 1 or turn == 0:
                        s.b.use_torch_stream()
                    s.project_and_attend()
                    s.check_drafts()
        for i, s in enumerate(steps):
            s.check(f"step {i}")
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()
        if other is not backend:
            other.close()


# ---- a request's prompt behind the prefix ----------------------------------------------------------

@pytest.mark.parametrize("seqs,rows,prefix,H,KH,hd", [(1, 300, 500, 14, 2, 64), (2, 150, 130, 8, 2, 128), (3, 257, 0, 3, 1, 64)])
def test_attention_prompts(backend, exp_lut, seqs, rows, prefix, H, KH, hd):
    """Hundreds of rows of a sequence, each attending its own position and all before it."""
    case(f"attention prompts {seqs}x{rows} behind {prefix}")
    s = attention_inputs(93, seqs, rows, prefix, rows + 20, H, KH, hd)
    s["lens"] = (np.array([[0], [20], [7]][:seqs]) + 1 + np.arange(rows)).reshape(-1).astype(np.int32)
    same(run_attention(backend, s, exp_lut), ref.attention(**s, lut=exp_lut), "prompts")


# ---- the tokens' distribution ---------------------------------------------------------------------

@pytest.mark.parametrize("drafted", ["sampled", "argmax"])
def test_tokens_follow_the_target(backend, exp_lut, drafted):
    """Drafts that the call itself draws from the draft's logits (no drafts: a token per row), or
    the draft's argmax handed over without probabilities; then their check.  Counts of n
    independent tokens lie within 6 deviations sqrt(n p (1 - p)) of n p."""
    import torch
    case(f"tokens follow the target, {drafted} drafts")
    B, V = 20000, 11
    r = rng(94)
    zt = r.integers(-150, 150, V).astype(np.int32)
    zd = (zt + r.integers(-60, 61, V)).astype(np.int32)
    table = gpu(exp_lut)
    target = gpu(zt).expand(B, 2, V).contiguous()
    draft = gpu(zd).expand(B, 1, V).contiguous()
    rnd = gpu(r.integers(0, 2**64, (B, 3), dtype=np.uint64).view(np.int64))
    none = torch.zeros((B, 0), dtype=torch.int64, device="cuda")
    if drafted == "sampled":
        accepted, tokens = backend.verify_drafts_dev(draft, none, rnd[:, :1].contiguous(), exp_lut=table)
        assert not accepted.any()
    else:
        tokens = backend.argmax_dev(draft.view(B, V)).view(B, 1)
    accepted, out = backend.verify_drafts_dev(target, tokens, rnd[:, 1:].contiguous(), exp_lut=table,
                                              draft=draft if drafted == "sampled" else None)
    p = ref.row_weights(zt, exp_lut) / ref.row_weights(zt, exp_lut).sum()
    accepted, out = accepted.cpu().numpy(), out.cpu().numpy()
    assert 0.1 < accepted.mean() < 0.95
    for what, got in (("first tokens", out[:, 0]), ("tokens behind an accepted draft", out[accepted == 1, 1])):
        n = got.size
        count = np.bincount(got, minlength=V)
        assert (np.abs(count - n * p) <= 6 * np.sqrt(n * p * (1 - p))).all(), (what, count / n, p)


# ---- the largest sizes ------------------------------------------------------------------------------

@pytest.mark.parametrize("prefix,tail", [(65536, 0), (0, 65536), (65000, 536), (1, 65535)])
def test_attention_of_65536_keys(backend, exp_lut, prefix, tail):
    case(f"attention of {prefix} + {tail} keys")
    s = attention_inputs(95, 1, 2, prefix, tail, 2, 1, 64)
    s["lens"] = np.array([tail, max(tail - 1, 0)], np.int32)
    same(run_attention(backend, s, exp_lut), ref.attention(**s, lut=exp_lut), "65536 keys")
    flat = np.full(32768, 32767, np.int16)  # the exp sums at their largest
    s.update(mult=0)
    same(run_attention(backend, s, flat), ref.attention(**s, lut=flat), "65536 keys, large entries")


@pytest.mark.parametrize("B,k,V", [(1, 1, 1 << 20), (31, 1024, 5), (65535, 0, 2), (21845, 1, 3)])
def test_verify_at_the_largest_sizes(backend, exp_lut, B, k, V):
    case(f"verify B={B} k={k} V={V}")
    s = verify_inputs(96, B, k, V)
    for draft, lut in ((s["draft"], exp_lut), (None, exp_lut), (None, None)):
        got, want = run_verify(backend, dict(s, draft=draft), lut), ref.verify(lut=lut, **dict(s, draft=draft))
        same(got[0], want[0], "accepted")
        same(got[1], want[1], "tokens")


def test_verify_accepts_1024_drafts(backend, exp_lut):
    case("verify 1024 drafts accepted")
    s = verify_inputs(97, 3, 1024, 6)
    s["draft"] = s["target"][:, :1024].copy()
    s["randoms"][:, :1024] = 2**64 - 1
    s["tokens"] = s["target"][:, :1024].argmax(2).astype(np.int64)
    s["tokens"][1, 1023] = -1
    s["n_draft"] = np.array([1024, 1024, 1000], np.int32)
    got, want = run_verify(backend, s, exp_lut), ref.verify(lut=exp_lut, **s)
    assert want[0].tolist() == [1024, 1023, 1000]
    same(got[0], want[0], "accepted")
    same(got[1], want[1], "tokens")


@pytest.mark.parametrize("M,N,K,rank,n", [(3, 1100003, 16, 3, 2), (2, 70, 262144 + 48, 5, 2), (1, 40, 131072, 256, 3)])
def test_adapters_wide_and_deep(backend, M, N, K, rank, n):
    case(f"adapters M={M} N={N} K={K} rank={rank}")
    s = adapter_inputs(98, M, N, K, rank, n)
    same(run_adapters(backend, s), want_adapters(s), "wide or deep")


@pytest.mark.parametrize("H", [8, 18])
def test_attention_captured_with_the_whole_table(backend, H):
    """The table as luts.exp_lut() makes it takes more LDS than a launch has by default."""
    import torch
    from myelith_amd.luts import exp_lut as whole
    case(f"attention captured, whole table, {H} heads")
    s = attention_inputs(99, 3, 1, 400, 30, H, 1, 64)
    d = {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in s.items()}
    lut = whole()
    table, out = gpu(lut), torch.empty_like(d["q"])
    ws = backend.attention_prefix_workspace(d["q"], d["kp"], d["kt"])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(stream):
            backend.use_torch_stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            backend.attention_prefix_dev(d["q"], d["kp"], d["vp"], d["kt"], d["vt"], d["lens"], s["mult"], s["shift"], table, 6, 14,
                                         slots=d["slots"], out=out, workspace=ws)
        for turn in range(4):
            s["q"] = gauss16(rng(100 + turn), s["q"].shape, 2048)
            d["q"].copy_(gpu(s["q"]))
            out.fill_(-7)
            dirty(ws)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            same(out, ref.attention(**s, lut=lut), f"replay {turn}")
    finally:
        torch.cuda.synchronize()
        backend.use_torch_stream()
