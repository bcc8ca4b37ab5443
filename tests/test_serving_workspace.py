"""Workspaces that a program makes once, for its largest step: every call none of
whose sizes is larger fits in them (csrc/serve_plan.h, under AddressSanitizer and
UndefinedBehaviorSanitizer)."""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "myelith_amd" / "csrc"

PROGRAM = r"""
#include "serve_plan.h"
#include <cstdio>
using namespace myl;
static long checked = 0, bad = 0;
static uint64_t sm = 11;
static uint64_t next() {
    uint64_t z = (sm += 0x9E3779B97F4A7C15ull);
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}
static size_t upto(size_t most) { return 1 + (size_t)(next() % ((size_t)1 << (next() % 64 % (64 - __builtin_clzll(most))))) % most; }
// A size of the smaller call: often the same, one less, a half, or any.
static size_t below(size_t n, size_t least) {
    const uint64_t r = next() % 6;
    const size_t v = r < 2 ? n : r == 2 ? n - 1 : r == 3 ? n / 2 : r == 4 ? n - n / 8 : (size_t)(next() % (n + 1));
    return v < least || v > n ? least : v;
}
static void hold(const char* what, size_t small, size_t large, const size_t (&s)[7], const size_t (&l)[7]) {
    ++checked;
    if (small <= large || bad++ >= 20) return;
    std::printf("%s: %zu bytes, %zu for no smaller sizes:", what, small, large);
    for (int i = 0; i < 7; ++i) std::printf(" %zu/%zu", s[i], l[i]);
    std::printf("\n");
}
static void adapters(AdapterShape l, int cus) {
    const AdapterShape s{below(l.M, 0), below(l.N, 0), below(l.K, 1), below(l.rank, 1), below(l.n, 0)};
    if (!adapter_refuse(l) && !adapter_refuse(s))
        hold("adapters", adapter_plan(s, cus).bytes, adapter_plan(l, cus).bytes, {s.M, s.N, s.K, s.rank, s.n}, {l.M, l.N, l.K, l.rank, l.n});
}
static void prefix(PrefixShape l, int cus) {
    PrefixShape s = l;
    s.n_seqs = below(l.n_seqs, 0);
    s.rows_per_seq = below(l.rows_per_seq, 0);
    s.prefix_len = below(l.prefix_len, 0);
    s.max_tail = below(l.max_tail, 0);
    if (!prefix_refuse(l) && !prefix_refuse(s))
        hold("attention", prefix_plan(s, cus).bytes, prefix_plan(l, cus).bytes, {s.n_seqs, s.rows_per_seq, s.heads, s.kv_heads, s.head_dim, s.prefix_len, s.max_tail},
             {l.n_seqs, l.rows_per_seq, l.heads, l.kv_heads, l.head_dim, l.prefix_len, l.max_tail});
}
static void verify(VerifyShape l) {
    const VerifyShape s{below(l.n_seqs, 0), below(l.k, 0), below(l.vocab, 1), below(l.lut_len, 0)};
    if (!verify_refuse(l) && !verify_refuse(s))
        hold("drafts", verify_plan(s).bytes, verify_plan(l).bytes, {s.n_seqs, s.k, s.vocab, s.lut_len}, {l.n_seqs, l.k, l.vocab, l.lut_len});
}
int main() {
    for (int i = 0; i < 60000; ++i) {
        const int cus = i % 3 ? 256 : (int)upto(512);
        adapters({upto(4096), upto(20000), upto(20000), upto(256), upto(300)}, cus);
        adapters({upto(600), 4608, 3584, 16, 24}, cus);
        adapters({upto((size_t)1 << 23), upto((size_t)1 << 30), upto((size_t)1 << 30), upto(256), upto((size_t)1 << 31)}, cus);
        const size_t kvh = upto(64), hd = i & 1 ? 64 : 128;
        prefix({upto(64), upto(9), kvh * upto(16), kvh, hd, upto(65537) - 1, upto(3000) - 1}, cus);
        prefix({upto(8), upto(3), 28, 4, 128, 1000, upto(8000)}, cus);
        prefix({upto(65535), upto(65535), kvh * upto(64), kvh, hd, upto(65537) - 1, upto(65537) - 1}, cus);
        verify({upto(300), upto(9) - 1, upto((size_t)1 << 20), upto(32769) - 1});
        verify({upto(65535), upto(1025) - 1, upto((size_t)1 << 20), upto(32769) - 1});
    }
    // every step of one size alone
    for (size_t T = 1; T < 9000; ++T)
        hold("tails", prefix_plan({1, 1, 28, 4, 128, 1000, T - 1}, 256).bytes, prefix_plan({1, 1, 28, 4, 128, 1000, T}, 256).bytes, {T - 1}, {T});
    for (size_t P = 1; P <= 65536; P += 64)
        hold("prefix", prefix_plan({3, 2, 28, 4, 128, P - 1, 0}, 256).bytes, prefix_plan({3, 2, 28, 4, 128, P, 0}, 256).bytes, {P - 1}, {P});
    for (size_t n = 1; n < 600; ++n)
        hold("sequences", prefix_plan({n - 1, 2, 28, 4, 128, 8000, 700}, 256).bytes, prefix_plan({n, 2, 28, 4, 128, 8000, 700}, 256).bytes, {n - 1}, {n});
    for (size_t M = 1; M < 3000; ++M)
        hold("rows", adapter_plan({M - 1, 4608, 3584, 16, 24}, 256).bytes, adapter_plan({M, 4608, 3584, 16, 24}, 256).bytes, {M - 1}, {M});
    std::printf("checked %ld bad %ld\n", checked, bad);
    return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ absent")
def test_a_workspace_serves_every_smaller_call(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I", str(CSRC),
                    str(src), "-o", str(exe)], check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, (r.stdout[-3000:], r.stderr[-3000:])
    assert int(re.match(r"checked (\d+) bad 0", r.stdout.strip().splitlines()[-1]).group(1)) > 300000


TABLE = r"""
#include "serve_plan.h"
#include <cstdio>
int main() {
    for (uint32_t n = 1; n <= myl::kPrefixMaxLut; ++n) {
        const uint32_t b = myl::prefix_table_bytes(n);
        if (b % 4 || b > 2 * n || b + 2 < 2 * n) return std::printf("%u entries: %u bytes\n", n, b), 1;
    }
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ absent")
def test_wide_loads_of_a_table_end_inside_it(tmp_path):
    """The exp table is read by whole words, which cover all but an odd last entry."""
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(TABLE)
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), str(src), "-o", str(exe)], check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
