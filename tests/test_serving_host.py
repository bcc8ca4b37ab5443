"""The operators of a serving step without a GPU: what the host decides for a
call (csrc/serve_plan.h, under AddressSanitizer and
UndefinedBehaviorSanitizer), the 32-bit forms of the attention's divisions
(csrc/attn_fixed.h) against the general ones, and refused calls."""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "myelith_amd" / "csrc"

PLANS = r"""
#include "serve_plan.h"
#include <cstdio>
#include <map>
#include <utility>
#include <vector>
using namespace myl;
static long checked = 0, bad = 0;
#define CHECK(ok, ...) (++checked, (ok) ? 0 : (bad++ < 20 ? std::printf(__VA_ARGS__), std::printf("\n") : 0))
static uint64_t sm = 7;
static uint64_t next() {
    uint64_t z = (sm += 0x9E3779B97F4A7C15ull);
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}
static size_t upto(size_t most) { return 1 + (size_t)(next() % ((size_t)1 << (next() % 64 % (64 - __builtin_clzll(most))))) % most; }

// pieces of a workspace: in order, apart, within its bytes
static void pieces(const char* what, std::vector<std::pair<size_t, size_t>> p, size_t bytes) {
    size_t end = 0;
    for (auto& x : p) {
        CHECK(x.first % 256 == 0 && x.first >= end, "%s: a piece at %zu starts before %zu", what, x.first, end);
        end = x.first + x.second;
    }
    CHECK(end <= bytes && bytes >= 256, "%s: %zu of %zu bytes", what, end, bytes);
}

static void adapters(AdapterShape s, int cus) {
    if (adapter_refuse(s)) return;
    const AdapterPlan p = adapter_plan(s, cus);
    if (s.n == 0 || s.M == 0 || s.N == 0) return;
    const int64_t units = ((int64_t)s.K + kAdapterUnit - 1) / kAdapterUnit, block = 4 * (int64_t)p.per_wave;
    CHECK(p.splits >= 1 && p.splits <= 65535 && block * p.splits >= units && block * (p.splits - 1) < units, "splits %d of %zu", p.splits, s.K);
    CHECK((int64_t)p.per_wave * kAdapterUnit <= (1 << 16), "a wave sums %d units", p.per_wave);  // 2^16 2^14 < 2^31
    CHECK(16 * p.rank_tiles * p.rank_groups >= (int)s.rank && 16 * p.rank_tiles * p.rank_groups <= std::max(16, 2 * (int)s.rank + 63), "rank %zu", s.rank);
    CHECK(p.rank_pad >= (int)s.rank && (p.rank_pad & (p.rank_pad - 1)) == 0 && p.rank_pad >= 16 && p.rank_pad <= 256, "pad %zu", s.rank);
    CHECK((int64_t)p.n_chunk * p.n_chunks >= (int64_t)s.N && (int64_t)p.n_chunk * (p.n_chunks - 1) < (int64_t)s.N && p.n_chunk % 256 == 0, "chunks of %zu", s.N);
    CHECK((int64_t)p.windows * kAdapterWindow >= (int64_t)s.M && p.down_tiles >= p.up_tiles && p.up_tiles >= 1, "windows of %zu", s.M);
    CHECK((uint64_t)p.windows * p.down_tiles * 256 < (1ull << 32) && (uint64_t)p.n_chunks * 256 < (1ull << 32) &&
          (uint64_t)p.windows * p.up_tiles <= 32768ull * 65535, "grids of %zu", s.M);
    pieces("adapters", {{p.off_planes, s.M >= 2 ? 2 * s.M * s.K : 0}, {p.off_acc, 8 * p.acc_elems},
                        {p.off_part, (size_t)p.splits * s.M * p.rank_pad * 8},
                        {p.off_tiles, (size_t)p.windows * p.up_tiles * kAdapterTileBytes}}, p.bytes);
    // tiles of random groupings of a window
    const int w = (int)std::min<size_t>(s.M, 256);
    for (int t = 0; t < 4; ++t) {
        std::map<uint64_t, int> rows;
        const uint64_t kinds = t == 0 ? s.n : 1 + next() % s.n;
        for (int i = 0; i < w; ++i) rows[t == 0 ? i % kinds : next() % kinds]++;
        int down = 0, up = 0;
        for (auto& g : rows) down += (g.second + 15) / 16, up += (g.second + 63) / 64;
        CHECK(down <= p.down_tiles && up <= p.up_tiles, "%d and %d tiles, room for %d and %d", down, up, p.down_tiles, p.up_tiles);
    }
}

static void prefix(PrefixShape s, int cus) {
    if (prefix_refuse(s)) return;
    const PrefixPlan p = prefix_plan(s, cus);
    if (p.short_cap) {
        const size_t keys = s.prefix_len + s.max_tail;
        CHECK(keys > 0 && (size_t)p.short_cap >= keys && p.short_cap % 64 == 0 && p.G <= 8 && p.bytes == 256 &&
              prefix_short_lds(p.G, p.short_cap, s.head_dim) <= 65536 && s.n_seqs * s.rows_per_seq * s.kv_heads <= 4 * (size_t)cus, "short: %zu keys", keys);
        return;
    }
    const int64_t P = (int64_t)s.prefix_len, T = (int64_t)s.max_tail, R = (int64_t)(s.n_seqs * s.rows_per_seq);
    auto ranges = [&](int64_t keys, int n, int len, bool any) {
        if (keys == 0 || !any) return CHECK(n == 0, "ranges without keys"), void();
        CHECK(len % 64 == 0 && (int64_t)n * len >= keys && (int64_t)(n - 1) * len < keys, "%d ranges of %d for %lld keys", n, len, (long long)keys);
    };
    ranges(P, p.np, p.rp, R > 0);
    ranges(T, p.nt, p.rt, R > 0);
    for (auto& c : {std::make_pair(p.qk, kPrefixQkTile), std::make_pair(p.pv, kPrefixPvTile)}) {
        CHECK((int64_t)c.first.tp * c.second >= p.vp && (int64_t)c.first.tt * c.second >= p.vt, "tiles of %d", c.second);
        CHECK(c.first.blocks_p % 8 == 0 && (c.first.blocks_p + c.first.blocks_t) * 256 < (1ll << 32), "%lld blocks",
              (long long)(c.first.blocks_p + c.first.blocks_t));
        CHECK(c.first.blocks_p >= (int64_t)s.kv_heads * c.first.tp * p.np, "prefix blocks");
    }
    const size_t parts = (size_t)R * s.heads * (size_t)(p.np + p.nt);
    pieces("attention", {{p.off_max, parts * 4}, {p.off_sum, parts * 4},
                         {p.off_pexp, s.kv_heads * ((p.vp + 15) / 16) * (size_t)p.pgroups * 512},
                         {p.off_texp, s.kv_heads * s.n_seqs * ((p.vt + 15) / 16) * (size_t)p.tgroups * 512},
                         {p.off_out, parts * s.head_dim * 4}}, p.bytes);
}

static void verify(VerifyShape s) {
    if (verify_refuse(s)) return;
    const VerifyPlan p = verify_plan(s);
    const size_t rows = s.n_seqs * (2 * s.k + 1), c = (size_t)p.chunks;
    CHECK((size_t)p.chunks * kVerifyChunk >= s.vocab && (size_t)(p.chunks - 1) * kVerifyChunk < s.vocab, "chunks of %zu", s.vocab);
    CHECK(4 * (size_t)p.bins >= s.lut_len && 2 * p.words >= p.bins && (size_t)p.words * 8 <= 65536, "bins of %zu", s.lut_len);
    pieces("drafts", {{p.off_stat, rows * 16}, {p.off_max, rows * c * 4}, {p.off_counts, rows * c * p.words * 4},
                      {p.off_sums, rows * c * 8}, {p.off_first, s.n_seqs * 4}}, p.bytes);
}

int main() {
    for (int i = 0; i < 30000; ++i) {
        const int cus = i % 3 ? 256 : (int)upto(512);
        adapters({upto(4096), upto(20000), upto(20000), upto(256), upto(300)}, cus);
        adapters({upto((size_t)1 << 23), upto((size_t)1 << 30), upto((size_t)1 << 30), upto(256), upto((size_t)1 << 31)}, cus);
        const size_t kvh = upto(64), hd = i & 1 ? 64 : 128;
        prefix({upto(64), upto(9), kvh * upto(16), kvh, hd, upto(65537) - 1, upto(3000) - 1}, cus);
        prefix({upto(65535), upto(65535), kvh * upto(64), kvh, hd, upto(65537) - 1, upto(65537) - 1}, cus);
        verify({upto(300), upto(9) - 1, upto((size_t)1 << 20), upto(32769) - 1});
        verify({upto(65535), upto(1025) - 1, upto((size_t)1 << 20), upto(32769) - 1});
    }
    const size_t big = (size_t)1 << 31;
    CHECK(adapter_refuse({1, 1, 0, 1, 1}) && adapter_refuse({1, 1, 1, 0, 1}) && adapter_refuse({1, 1, 1, 257, 1}), "adapters: K, rank");
    CHECK(adapter_refuse({((size_t)1 << 23) + 1, 1, 1, 1, 1}) && adapter_refuse({1, big, 1, 1, 1}) && adapter_refuse({1, 1, big, 1, 1}) &&
          adapter_refuse({1, 1, 1, 1, big}) && adapter_refuse({1, (size_t)1 << 30, 1, 256, big - 1}) && adapter_refuse({1, 1, (size_t)1 << 30, 256, big - 1}),
          "adapters: sizes");
    CHECK(!adapter_refuse({0, 0, 1, 0, 0}) && !adapter_refuse({(size_t)1 << 23, 1, 1, 256, 1}), "adapters: allowed sizes");
    CHECK(adapter_plan({0, 5, 7, 3, 2}, 256).bytes == 256 && adapter_plan({1, 0, 7, 3, 2}, 256).bytes == 256, "adapters: nothing to do");
    CHECK(prefix_refuse({1, 1, 3, 2, 64, 1, 1}) && prefix_refuse({1, 1, 0, 0, 64, 1, 1}) && prefix_refuse({1, 1, 0, 1, 64, 1, 1}), "attention: heads");
    CHECK(prefix_refuse({1, 1, 1, 1, 64, 65537, 0}) && prefix_refuse({1, 1, 1, 1, 64, 0, 65537}) && prefix_refuse({1, 1, 1, 1, 64, 1, 65536}) &&
          prefix_refuse({1, 1, 1, 1, 64, ~(size_t)0, 1}) && prefix_refuse({1, 1, 1, 1, 64, 1, ~(size_t)0}), "attention: keys");
    CHECK(prefix_refuse({65536, 1, 1, 1, 64, 1, 1}) && prefix_refuse({256, 256, 1, 1, 64, 1, 1}) && prefix_refuse({~(size_t)0, 2, 1, 1, 64, 1, 1}) &&
          prefix_refuse({65535, 1, 128, 1, 64, 1, 1}), "attention: rows");
    CHECK(!prefix_refuse({65535, 1, 64, 1, 64, 65535, 1}) && !prefix_refuse({0, 0, 1, 1, 64, 0, 0}), "attention: allowed sizes");
    CHECK(verify_refuse({1, 0, 0, 1}) && verify_refuse({1, 0, ((size_t)1 << 20) + 1, 1}) && verify_refuse({1, 1025, 1, 1}) &&
          verify_refuse({65536, 0, 1, 1}) && verify_refuse({32, 1024, 1, 1}) && verify_refuse({1, 1, 1, 32769}) && verify_refuse({~(size_t)0, 1, 1, 1}),
          "drafts: sizes");
    CHECK(!verify_refuse({65535, 0, (size_t)1 << 20, 32768}) && !verify_refuse({31, 1024, 1, 0}), "drafts: allowed sizes");
    std::printf("checked %ld bad %ld\n", checked, bad);
    return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ absent")
def test_plans_and_refusals_under_asan_and_ubsan(tmp_path):
    src, exe = tmp_path / "plans.cpp", tmp_path / "plans"
    src.write_text(PLANS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I", str(CSRC),
                    str(src), "-o", str(exe)], check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, (r.stdout[-3000:], r.stderr[-3000:])
    assert int(re.match(r"checked (\d+) bad 0", r.stdout.strip().splitlines()[-1]).group(1)) > 500000


DIVISIONS = r"""
#include <hip/hip_runtime.h>
#include <cstdio>
#include "attn_fixed.h"
static uint64_t sm = 1;
static uint64_t next() {
    uint64_t z = (sm += 0x9E3779B97F4A7C15ull);
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}
static long bad = 0, n = 0;
static void prob(uint32_t e, uint32_t f, uint32_t s) {
    const ProbDiv d = ProbDiv::of(s, f);
    const uint64_t num = (uint64_t)e << f, r = num % s;
    uint64_t q = num / s;
    if (2 * r > s || (2 * r == s && (q & 1))) q++;
    ++n;
    if (d(e) != q && bad++ < 10) printf("e=%u f=%u s=%u: %u, not %llu\n", e, f, s, d(e), (unsigned long long)q);
}
static void score(int64_t dot, int64_t mult, uint8_t shift, int hd) {
    const ScoreScale s = ScoreScale::of(mult, shift, hd);
    if (!s.fast) return;
    const int64_t want = rshift_round64(dot * mult, shift);
    const int32_t z = s((int32_t)(dot >> 8), (uint32_t)(dot & 255));
    ++n;
    if (z != want && bad++ < 10) printf("dot=%lld mult=%lld shift=%d: %d, not %lld\n", (long long)dot, (long long)mult, shift, z, (long long)want);
}
int main() {
    for (uint32_t s : {1u, 2u, 3u, 4u, 5u, 7u, 8u, 16384u, 32767u, 32768u, 65535u, (1u << 30) - 1, 1u << 30, (1u << 30) + 1, 2147483647u})
        for (uint32_t f = 0; f <= 14; ++f)
            for (uint32_t e : {0u, 1u, 2u, 3u, 16383u, 16384u, 16385u, 32766u, 32767u}) prob(e, f, s);
    for (int i = 0; i < 1500000; ++i) {
        const uint32_t f = (uint32_t)(next() % 15);
        uint32_t s = 1 + (uint32_t)(next() >> 33) % (i & 1 ? 2147483646u : 1u << (1 + next() % 30)), e = (uint32_t)(next() % 32768);
        if (i % 5 == 0 && e > s) e %= s;
        if (i % 17 == 0) s = 2 * (1 + (uint32_t)(next() % 4000)), e = s / 2 * (1 + 2 * (uint32_t)(next() % 8)), e = e > 32767 ? 32767 : e;  // ties
        prob(e, f, s);
    }
    for (int i = 0; i < 1500000; ++i) {
        const int hd = i & 1 ? 64 : 128;
        const uint8_t shift = (uint8_t)(9 + next() % 31);
        const int64_t mult = (int64_t)(next() % (1u << next() % 24)), most = (int64_t)hd << 30;
        int64_t dot = (int64_t)(next() % (2 * (uint64_t)most + 1)) - most;
        if (i % 3 == 0) dot >>= next() % 36;
        if (i % 7 == 0 && mult) {  // about a tie
            dot = ((int64_t)(next() % 100000) * 2 + 1) << (shift - 1 > 30 ? 30 : shift - 1);
            dot = dot / mult > most ? most : dot / mult;
            if (next() & 1) dot = -dot;
        }
        score(dot, mult, shift, hd);
        if (i < 64) score(i & 2 ? most : -most, mult, shift, hd);
    }
    for (int i = 0; i < 500000; ++i) {
        const uint32_t d = 1 + (uint32_t)(next() >> 33) % (1u << (1 + next() % 30));
        const int v = i % 4 ? (int)(next() >> 33) : 2147483647 - i;
        int rem;
        const int q = divmod(SmallDiv::of(d), v, rem);
        ++n;
        if ((q != v / (int)d || rem != v % (int)d) && bad++ < 10) printf("%d / %u: %d rest %d\n", v, d, q, rem);
    }
    printf("checked %ld, mismatches %ld\n", n, bad);
    return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("hipcc") is None and not Path("/opt/rocm/bin/hipcc").exists(), reason="hipcc absent")
def test_division_forms_match_the_general_ones(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    src, exe = tmp_path / "t.hip", tmp_path / "t"
    src.write_text(DIVISIONS)
    subprocess.run([hipcc, "-O2", "-std=c++17", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-I", str(CSRC), str(src), "-o", str(exe)], check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "mismatches 0" in r.stdout, r.stdout


# ---- refused calls -----------------------------------------------------------------

@pytest.fixture(scope="module")
def bare():
    """The backend's checks of arguments, without a context: nothing reaches a device."""
    from myelith_amd.backend import RocmBackend
    b = RocmBackend.__new__(RocmBackend)
    b._h, b._device_id = None, 0
    return b


def adapter_args(**over):
    import torch
    a = dict(x=torch.zeros((3, 32), dtype=torch.int16), W=torch.zeros((5, 32), dtype=torch.int8),
             w_shifts=torch.zeros(5, dtype=torch.uint8), act_frac=10, ids=torch.zeros(3, dtype=torch.int32),
             A=torch.zeros((2, 4, 32), dtype=torch.int8), a_shifts=torch.zeros((2, 4), dtype=torch.uint8), mid_frac=10,
             B=torch.zeros((2, 5, 4), dtype=torch.int8), b_shifts=torch.zeros((2, 5), dtype=torch.uint8), out_frac=10)
    a.update(over)
    return a


def attention_args(**over):
    import torch
    z = lambda *s: torch.zeros(s, dtype=torch.int16)
    a = dict(q=z(4, 4, 64), k_prefix=z(2, 9, 64), v_prefix=z(2, 9, 64), k_tail=z(2, 2, 5, 64), v_tail=z(2, 2, 5, 64),
             lens=torch.zeros(4, dtype=torch.int32), score_mult=1, score_shift=20, exp_lut=z(100), lut_shift=6, prob_frac=14,
             rows_per_seq=2)
    a.update(over)
    return a


def verify_args(**over):
    import torch
    a = dict(target=torch.zeros((2, 4, 50), dtype=torch.int32), tokens=torch.zeros((2, 3), dtype=torch.int64),
             randoms=torch.zeros((2, 4), dtype=torch.int64), exp_lut=torch.zeros(100, dtype=torch.int16),
             draft=torch.zeros((2, 3, 50), dtype=torch.int32))
    a.update(over)
    return a


def test_refused_arguments(bare):
    import torch
    i16, i32, i8 = torch.int16, torch.int32, torch.int8
    calls = [
        (bare.linear_w8a16_adapters_dev, adapter_args, [
            ("W must be", dict(W=torch.zeros((5, 32), dtype=i16))), ("W must be", dict(W=torch.zeros((5, 31), dtype=i8))),
            ("ids must be", dict(ids=torch.zeros(2, dtype=i32))), ("ids must be", dict(ids=torch.zeros(3, dtype=torch.int64))),
            ("a_shifts must be", dict(a_shifts=torch.zeros((2, 3), dtype=torch.uint8))),
            ("B must be", dict(B=torch.zeros((2, 4, 5), dtype=i8))), ("B must be", dict(B=torch.zeros((2, 4, 5), dtype=i8).transpose(1, 2))),
            ("out_frac_pc must be", dict(out_frac_pc=torch.zeros(4, dtype=torch.uint8))),
            ("follow one another", dict(x=torch.zeros((32, 3), dtype=i16).t())),
            ("out must be", dict(out=torch.zeros((3, 6), dtype=i16))), ("out must be", dict(out=torch.zeros((3, 5), dtype=i32))),
            ("out must be", dict(out=torch.zeros((5, 3), dtype=i16).t())), ("on device 0", {})]),
        (bare.attention_prefix_dev, attention_args, [
            ("multiple of rows_per_seq", dict(rows_per_seq=3)), ("multiple of rows_per_seq", dict(rows_per_seq=0)),
            ("prefix", dict(v_prefix=torch.zeros((2, 8, 64), dtype=i16))), ("tails", dict(v_tail=torch.zeros((2, 2, 6, 64), dtype=i16))),
            ("max_tail", dict(max_tail=6)), ("max_tail", dict(max_tail=-1)), ("lens must be", dict(lens=torch.zeros(3, dtype=i32))),
            ("slots must be", dict(slots=torch.zeros(4, dtype=i32))), ("fewer tails", dict(rows_per_seq=1)),
            ("exp_lut must be", dict(exp_lut=torch.zeros(100, dtype=i32))), ("out must", dict(out=torch.zeros((4, 4, 32), dtype=i16))),
            ("heads of a row", dict(q=torch.zeros((4, 64, 4), dtype=i16).transpose(1, 2))),
            ("positions of a KV head", dict(k_prefix=torch.zeros((9, 2, 64), dtype=i16).transpose(0, 1))),
            ("same strides", dict(k_prefix=torch.zeros((2, 10, 64), dtype=i16)[:, :9])), ("on device 0", {})]),
        (bare.verify_drafts_dev, verify_args, [
            ("target must be", dict(target=torch.zeros((2, 4, 50), dtype=i16))), ("tokens must be", dict(tokens=torch.zeros((2, 3), dtype=i32))),
            ("tokens must be", dict(tokens=torch.zeros((2, 4), dtype=torch.int64))), ("target must be", dict(target=torch.zeros((2, 0, 50), dtype=i32))),
            ("random numbers", dict(randoms=None)), ("randoms must be", dict(randoms=torch.zeros((2, 3), dtype=torch.int64))),
            ("draft must be", dict(draft=torch.zeros((2, 4, 50), dtype=i32))), ("n_draft must be", dict(n_draft=torch.zeros(3, dtype=i32))),
            ("evenly spaced", dict(target=torch.zeros((2, 5, 50), dtype=i32)[:, :4])), ("out must be", dict(out=torch.zeros((2, 3), dtype=torch.int64))),
            ("evenly spaced", dict(target=torch.zeros((2, 50, 4), dtype=i32).transpose(1, 2))), ("on device 0", {})]),
    ]
    for call, args, cases in calls:
        for match, over in cases:
            with pytest.raises(ValueError, match=match):
                call(**args(**over))


def test_calls_without_a_context():
    """The C entries refuse a null context before they look at anything else."""
    from myelith_amd._lib import SIGNATURES as sig, lib
    for name in ("linear_w8a16_adapters", "attention_prefix", "verify_drafts"):
        w, d = f"myl_{name}_workspace", f"myl_{name}_dev"
        assert getattr(lib(), w)(None, *[1] * (len(sig[w][1]) - 1)) == 0
        assert getattr(lib(), d)(None, *[0] * (len(sig[d][1]) - 1)) != 0
