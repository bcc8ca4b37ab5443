"""The operators over a paged cache and the log probabilities without a GPU: what the host
decides for a call (csrc/paged_plan.h, under AddressSanitizer and
UndefinedBehaviorSanitizer), the probabilities' division at the largest sums, launches
at the largest sizes, refused calls, and what the calls hand to the library."""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from test_launch_limits import HIPCC, PROGRAM
from test_serving_calls import FakeStream, OnGpu, on_gpu, one, recorded, streams  # noqa: F401
from test_serving_host import PLANS, bare  # noqa: F401

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "myelith_amd" / "csrc"

# the checker, random numbers and pieces() of the serving plans, then these plans
MORE_PLANS = PLANS[:PLANS.index("static void adapters(")].replace('#include "serve_plan.h"', '#include "paged_plan.h"') + r"""
constexpr size_t kLds = 160 * 1024;
static void attention(PagedShape s, int cus, int page, uint32_t lut) {
    if (paged_refuse(s)) return;
    const PagedPlan p = paged_plan(s, cus);
    const size_t vectors = s.rows_per_seq * (s.heads / s.kv_heads);
    CHECK((size_t)p.width * p.tiles >= vectors && p.width <= 16 && (vectors == 0 || (size_t)p.width * (p.tiles - 1) < vectors), "tiles of %zu", vectors);
    CHECK(p.keys % 64 == 0 && (size_t)p.keys >= s.max_len && (size_t)p.keys < s.max_len + 64, "keys of %zu", s.max_len);
    if (p.parts == 0 || p.keys == 0) return CHECK(p.ranges == 0 && p.blocks == 0, "nothing to do"), void();
    CHECK(p.range % 64 == 0 && p.range >= 64 && p.range <= 1024 && (int64_t)p.range * p.ranges >= p.keys && (int64_t)p.range * (p.ranges - 1) < p.keys,
          "%d ranges of %d for %d", p.ranges, p.range, p.keys);
    CHECK(p.blocks % 8 == 0 && p.blocks >= (int64_t)p.parts * p.ranges && p.blocks < (int64_t)p.parts * p.ranges + 8 * p.tiles && p.blocks * (p.in_one ? 512 : 256) < (1ll << 32),
          "%lld blocks", (long long)p.blocks);
    CHECK(!p.in_one || (p.ranges == 1 && s.max_len <= 1024), "one launch for %zu keys", s.max_len);
    const size_t vecs = p.parts * (size_t)p.width, pieces_of = vecs * (size_t)p.ranges;
    pieces("attention", {{p.off_z, vecs * p.keys * 4}, {p.off_e, vecs * p.keys * 2}, {p.off_max, pieces_of * 4}, {p.off_sum, pieces_of * 4},
                         {p.off_holes, p.parts * p.ranges * 4}, {p.off_out, pieces_of * s.head_dim * 4}}, p.bytes);
    // the LDS of every kernel, with the most that they declare themselves
    const size_t tab = (size_t)paged_table_entries(p.range, page) * 8, W = p.width <= 8 ? 8 : 16;
    int first = 0;
    for (int j0 = 0; j0 < p.keys && first < 50; j0 += p.range, ++first)
        CHECK((std::min(j0 + p.range, p.keys) - 1) / page - j0 / page + 1 <= paged_table_entries(p.range, page), "pages of %d keys from %d by %d", p.range, j0, page);
    CHECK(tab % 16 == 0, "entries");
    if (p.in_one) CHECK(paged_short_lds(p, s.head_dim, page, lut) + 4800 <= kLds, "%zu bytes in one", paged_short_lds(p, s.head_dim, page, lut));
    CHECK(4 * 2 * 32 * s.head_dim + tab + 4400 <= kLds && 3 * 64 * 2 * s.head_dim + p.range * W * 2 + tab + 200 <= kLds && tab + 16600 <= kLds, "LDS of %d keys", p.range);
    // a smaller call's pieces lie within this one's workspace: the same heads, fewer rows and keys
    PagedShape t = s;
    t.n_seqs = upto(s.n_seqs);
    t.rows_per_seq = upto(s.rows_per_seq);
    t.max_len = s.max_len ? upto(s.max_len) : 0;
    CHECK(paged_plan(t, cus).bytes <= p.bytes, "%zu x %zu rows of %zu in the workspace of %zu x %zu of %zu", t.n_seqs, t.rows_per_seq, t.max_len, s.n_seqs,
          s.rows_per_seq, s.max_len);
}

static void logprobs(LogpShape s) {
    if (logp_refuse(s)) return;
    const LogpPlan p = logp_plan(s);
    CHECK((size_t)p.chunks * kLogpChunk >= s.vocab && (size_t)(p.chunks - 1) * kLogpChunk < s.vocab, "chunks of %zu", s.vocab);
    CHECK((size_t)p.tiles * kLogpTile >= s.vocab && (size_t)(p.tiles - 1) * kLogpTile < s.vocab, "tiles of %zu", s.vocab);
    CHECK(4 * (size_t)p.bins >= s.lut_len && 2 * p.words >= p.bins && (size_t)p.words * 8 <= 65536 && (size_t)p.bins * 2 + 8192 <= 65536, "bins of %zu", s.lut_len);
    pieces("logprobs", {{p.off_max, s.rows * p.chunks * 4}, {p.off_tiles, s.top_n ? s.rows * p.tiles * 4 : 0}, {p.off_counts, s.rows * p.chunks * p.words * 4}}, p.bytes);
    const LogpShape t{upto(s.rows), upto(s.vocab), s.n_tokens, s.top_n ? std::min(upto(s.top_n), upto(s.vocab)) : 0, upto(s.lut_len)};
    if (!logp_refuse(t)) CHECK(logp_plan(t).bytes <= p.bytes, "fewer rows of fewer values");
}

int main() {
    for (int i = 0; i < 30000; ++i) {
        const int cus = i % 3 ? 256 : (int)upto(512);
        const size_t kvh = upto(64), hd = i & 1 ? 64 : 128;
        attention({upto(64), upto(9), kvh * upto(16), kvh, hd, upto(131073) - 1}, cus, (int)upto(300), (uint32_t)upto(32768));
        attention({upto(65535), upto(65535), kvh * upto(64), kvh, hd, upto(131073) - 1}, cus, (int)upto(65536), (uint32_t)upto(32768));
        attention({upto(300), upto(5), kvh * upto(16), kvh, hd, upto(1100)}, cus, (int)upto(64), (uint32_t)upto(32768));
        logprobs({upto(65535), upto((size_t)1 << 20), upto(65537) - 1, upto(33) - 1, upto(32768)});
        const size_t rows = upto((size_t)1 << 31), heads = upto(1 << 16), kv = upto(1 << 12);
        if (!append_refuse(rows, heads, kv, hd)) {
            const size_t per_row = (heads + 2 * kv) * (hd / 16), g = (size_t)append_group(rows, per_row, cus);
            CHECK((g == 1 || g % 4 == 0) && g <= 16 && (rows + g - 1) / g * per_row <= kInt - 255, "groups of %zu rows", g);
        }
    }
    const size_t big = (size_t)1 << 31;
    CHECK(paged_refuse({1, 1, 3, 2, 64, 1}) && paged_refuse({1, 1, 0, 0, 64, 1}) && paged_refuse({1, 1, 0, 1, 64, 1}), "heads");
    CHECK(paged_refuse({1, 1, 1, 1, 64, 131073}) && paged_refuse({1, 1, 1, 1, 64, ~(size_t)0}) && paged_refuse({65535, 1, 64, 2, 64, 131072}), "keys");
    CHECK(paged_refuse({65536, 1, 1, 1, 64, 1}) && paged_refuse({256, 256, 1, 1, 64, 1}) && paged_refuse({~(size_t)0, 2, 1, 1, 64, 1}) && paged_refuse({65535, 1, 128, 1, 64, 1}), "rows");
    CHECK(!paged_refuse({65535, 1, 64, 4, 64, 32768}) && !paged_refuse({1, 1, 1, 1, 64, 131072}) && !paged_refuse({0, 0, 1, 1, 64, 0}), "allowed sizes");
    CHECK(pages_refuse({1, 0, 64, 64, 64, 1, 1, 1, 1, 64}) && pages_refuse({1, 65537, 64, 64, 64, 1, 1, 1, 1, 64}), "page size");
    CHECK(pages_refuse({0, 16, 64, 64, 64, 1, 1, 1, 1, 64}) && pages_refuse({big, 16, 64, 64, 64, 1, 1, 1, 1, 64}) && pages_refuse({1, 16, 64, 64, 64, big, 1, 1, 1, 64}) &&
          pages_refuse({1, 16, 64, 64, 64, 1, big, big, 1, 64}), "pages and tables");
    CHECK(pages_refuse({1, 2, 64, 64, 63, 1, 1, 1, 1, 64}) && pages_refuse({1, 1, 64, 63, 64, 1, 1, 1, 2, 64}) && pages_refuse({2, 1, 0, 64, 64, 1, 1, 1, 1, 64}) &&
          pages_refuse({1, 1, 64, 64, ((size_t)1 << 40) + 1, 1, 1, 1, 1, 64}) && pages_refuse({1, 1, 64, 64, 64, 2, 5, 4, 1, 64}), "strides");
    CHECK(!pages_refuse({1, 1, 0, 0, 0, 1, 7, 0, 1, 64}) && !pages_refuse({big - 1, 65536, (size_t)1 << 40, 64, 64, big - 1, 1, 1, 1, 64}), "allowed pages");
    CHECK(append_refuse(1, 1, 0, 64) && append_refuse(big, 1, 1, 64) && append_refuse(1, big, 1, 64) && append_refuse(1, 1, ~(size_t)0, 64) && append_refuse(1 << 27, 2, 1, 64), "rows to append");
    CHECK(!append_refuse(0, 0, 1, 64) && !append_refuse((1 << 27) - 64, 2, 1, 64), "allowed rows");
    CHECK(logp_refuse({1, 0, 1, 0, 1}) && logp_refuse({1, ((size_t)1 << 20) + 1, 1, 0, 1}) && logp_refuse({65536, 1, 1, 0, 1}) && logp_refuse({1, 1, 65537, 0, 1}) &&
          logp_refuse({1, 100, 1, 33, 1}) && logp_refuse({1, 4, 1, 5, 1}) && logp_refuse({1, 1, 1, 0, 0}) && logp_refuse({1, 1, 1, 0, 32769}), "logprobs: sizes");
    CHECK(!logp_refuse({65535, (size_t)1 << 20, 65536, 32, 32768}) && !logp_refuse({0, 32, 0, 32, 1}), "logprobs: allowed sizes");
    std::printf("checked %ld bad %ld\n", checked, bad);
    return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ absent")
def test_plans_and_refusals_under_asan_and_ubsan(tmp_path):
    src, exe = tmp_path / "plans.cpp", tmp_path / "plans"
    src.write_text(MORE_PLANS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I", str(CSRC),
                    str(src), "-o", str(exe)], check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, (r.stdout[-3000:], r.stderr[-3000:])
    assert int(re.match(r"checked (\d+) bad 0", r.stdout.strip().splitlines()[-1]).group(1)) > 500000


LARGE_SUMS = r"""
#include <hip/hip_runtime.h>
#include <cstdio>
#include "attn_fixed.h"
int main() {
    long n = 0, bad = 0;
    uint64_t sm = 1;
    for (int i = 0; i < 400000; ++i) {
        sm = sm * 6364136223846793005ull + 1442695040888963407ull;
        const uint32_t s = i < 8 ? 0xFFFFFFFFu - (uint32_t)i : i < 16 ? 0x80000000u + (uint32_t)(i - 12) : 0x40000000u + (uint32_t)(sm >> 33) % 0xBFFFFFFFu;
        const uint32_t f = (uint32_t)(sm & 15) % 15, e = i & 1 ? 32767u : (uint32_t)(sm >> 20) & 32767u;
        const uint64_t num = (uint64_t)e << f, r = num % s;
        uint64_t q = num / s;
        if (2 * r > s || (2 * r == s && (q & 1))) q++;
        ++n;
        bad += ProbDiv::of(s, f)(e) != q;
    }
    printf("checked %ld, mismatches %ld\n", n, bad);
    return bad != 0;
}
"""


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc absent")
def test_probabilities_of_the_largest_sums(tmp_path):
    """131072 keys bring an exp sum close to 2^32."""
    src, exe = tmp_path / "t.hip", tmp_path / "t"
    src.write_text(LARGE_SUMS)
    subprocess.run([HIPCC, "-O2", "-std=c++17", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-I", str(CSRC), str(src),
                    "-o", str(exe)], check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "mismatches 0" in r.stdout, r.stdout


# ---- launches at the largest sizes ---------------------------------------------------

LAUNCHES = PROGRAM[:PROGRAM.index("int main() {")] + r"""
int main() {
    myl_ctx* c = nullptr;
    if (myl_init(0, &c) != MYL_OK) return 2;
    launches.clear();
    const int16_t* x = at<int16_t>(1 << 20);
    int16_t* out = at<int16_t>(1 << 22);
    void* ws = at<void>(1 << 23);
    const int32_t* ids = at<int32_t>(64);
    struct { size_t seqs, rows, heads, kvh, keys, page; } shapes[] = {
        {65535, 1, 64, 4, 32768, 1}, {65535, 1, 64, 64, 2048, 65536}, {1, 65535, 64, 8, 100, 16}, {1, 65535, 64, 8, 32000, 7}, {255, 257, 64, 64, 4000, 24},
        {1, 1, 65535, 65535, 131072, 16}, {1, 1, 65535, 1, 1000, 16}, {64, 1, 28, 4, 12000, 64}, {1, 1, 1, 1, 1, 1}, {1024, 1, 8, 1, 320, 1}, {3, 1, 8, 8, 0, 16},
        {1, 2, 16, 1, 512, 1}, {300, 2, 16, 2, 1024, 1}};
    for (auto& s : shapes)
        for (size_t hd : {(size_t)64, (size_t)128})
            for (int64_t mult : {(int64_t)2896, (int64_t)1 << 40})
                for (size_t lut : {(size_t)1, (size_t)2662, (size_t)32768}) {
                    const size_t bytes = myl_attention_paged_workspace(c, s.seqs, s.rows, s.heads, s.kvh, hd, s.keys), ld = s.heads * hd, len = (s.keys + s.page - 1) / s.page;
                    check("attention " + std::to_string(s.seqs) + " x " + std::to_string(s.rows) + " x " + std::to_string(s.heads) + ", " + std::to_string(s.keys),
                          myl_attention_paged_dev(c, x, s.seqs, s.rows, ld, s.heads, s.kvh, hd, x, x, 1000, s.page, s.kvh * s.page * hd, s.page * hd, hd, ids, len, len, ids,
                                                  s.keys, mult, 21, x, lut, 6, 14, out, ld, ws, bytes));
                }
    myl_head_norm norm = {at<int8_t>(64), at<uint8_t>(64), nullptr, nullptr, x, 32768, 8192, 8, 8, 10, 10};
    struct { size_t rows, heads, kvh; } appends[] = {{1, 0, 1}, {1, 28, 4}, {16384, 28, 4}, {(1 << 27) - 64, 2, 1}, {1000000, 64, 8}, {1, 65535, 65535}, {5, 1, 1}};
    for (auto& s : appends)
        for (size_t hd : {(size_t)64, (size_t)128}) {
            if (hd == 128 && s.rows > (1 << 26)) continue;
            for (const myl_head_norm* n : {(const myl_head_norm*)nullptr, (const myl_head_norm*)&norm})
                for (size_t bias : {(size_t)0, (size_t)1 << 16})
                    check("append " + std::to_string(s.rows) + " x " + std::to_string(s.heads),
                          myl_kv_append_paged_dev(c, x, s.heads * hd, x, s.kvh * hd, x, s.kvh * hd, s.rows, s.heads, s.kvh, hd, at<int16_t>(bias), at<uint8_t>(bias), 10, 10,
                                                  10, n, x, x, hd * 1024, 8, ids, ids, ids, 4, 100, 100, out, out, 7, 16, s.kvh * 16 * hd, 16 * hd, hd, out, s.heads * hd));
        }
    struct { size_t rows, vocab, tokens, top, lut; } logits[] = {{65535, (size_t)1 << 20, 65536, 32, 32768}, {1, 1, 0, 0, 1}, {512, 152064, 1, 20, 2662}, {513, 32001, 4, 1, 16385}};
    for (auto& s : logits)
        check("logprobs " + std::to_string(s.rows) + " x " + std::to_string(s.vocab),
              myl_logprobs_dev(c, ids, s.rows, s.vocab, s.vocab, x, s.lut, at<int64_t>(64), s.tokens, s.top, at<int64_t>(64), at<int64_t>(64), at<int64_t>(64), at<int64_t>(64), ws,
                               myl_logprobs_workspace(c, s.rows, s.vocab, s.top, s.lut)));
    // refused before any launch
    auto attend = [&](size_t hd, size_t n_pages, size_t page, size_t pos, size_t len, size_t keys, const void* q, const void* t, const void* w, size_t bytes, uint8_t f, size_t lut) {
        return myl_attention_paged_dev(c, (const int16_t*)q, 2, 1, 4 * hd, 4, 2, hd, x, x, n_pages, page, 4096, 2048, pos, (const int32_t*)t, len, len, ids, keys, 2896, 21, x, lut, 6, f,
                                       out, 4 * hd, (void*)w, bytes);
    };
    const size_t need = myl_attention_paged_workspace(c, 2, 1, 4, 2, 64, 160);
    check("attention", attend(64, 9, 16, 64, 10, 160, x, ids, ws, need, 14, 100));
    check("head size", attend(96, 9, 16, 96, 10, 160, x, ids, ws, need, 14, 100), false);
    check("no pages", attend(64, 0, 16, 64, 10, 160, x, ids, ws, need, 14, 100), false);
    check("page size", attend(64, 9, 0, 64, 10, 160, x, ids, ws, need, 14, 100), false);
    check("odd stride", attend(64, 9, 16, 68, 10, 160, x, ids, ws, need, 14, 100), false);
    check("beyond the table", attend(64, 9, 16, 64, 10, 161, x, ids, ws, need, 14, 100), false);
    check("null q", attend(64, 9, 16, 64, 10, 160, nullptr, ids, ws, need, 14, 100), false);
    check("odd q", attend(64, 9, 16, 64, 10, 160, at<int16_t>(1 << 20 | 2), ids, ws, need, 14, 100), false);
    check("null tables", attend(64, 9, 16, 64, 10, 160, x, nullptr, ws, need, 14, 100), false);
    check("null workspace", attend(64, 9, 16, 64, 10, 160, x, ids, nullptr, need, 14, 100), false);
    check("small workspace", attend(64, 9, 16, 64, 10, 160, x, ids, ws, need - 1, 14, 100), false);
    check("prob_frac", attend(64, 9, 16, 64, 10, 160, x, ids, ws, need, 15, 100), false);
    check("empty table", attend(64, 9, 16, 64, 10, 160, x, ids, ws, need, 14, 0), false);
    auto append = [&](const myl_head_norm* n, const void* bias, size_t lut_len, const void* pos, size_t ldk, const void* pages) {
        return myl_kv_append_paged_dev(c, x, 256, x, ldk, x, 128, 3, 4, 2, 64, (const int16_t*)bias, at<uint8_t>(1 << 12), 10, 10, 10, n, x, x, lut_len, 8, (const int32_t*)pos, nullptr,
                                       ids, 3, 5, 5, (int16_t*)pages, out, 9, 16, 2048, 1024, 64, out, 256);
    };
    check("append", append(&norm, x, 64, ids, 128, out));
    check("half a bias", append(nullptr, nullptr, 64, ids, 128, out), false);
    check("empty rotation", append(nullptr, x, 31, ids, 128, out), false);
    check("null positions", append(nullptr, x, 64, nullptr, 128, out), false);
    check("narrow keys", append(nullptr, x, 64, ids, 120, out), false);
    check("null pages", append(nullptr, x, 64, ids, 128, nullptr), false);
    myl_head_norm bad_norm = norm;
    bad_norm.q_gamma_shifts = nullptr;
    check("half a norm", append(&bad_norm, x, 64, ids, 128, out), false);
    bad_norm = norm, bad_norm.lut_input_shift = 7;
    check("odd norm shift", append(&bad_norm, x, 64, ids, 128, out), false);
    bad_norm = norm, bad_norm.inv_n_q20 = -1;
    check("negative 1/n", append(&bad_norm, x, 64, ids, 128, out), false);
    bad_norm = norm, bad_norm.rsqrt_len = 1;
    check("short rsqrt table", append(&bad_norm, x, 64, ids, 128, out), false);
    bad_norm = norm, bad_norm.q_gamma = at<int8_t>(65);
    check("odd gamma", append(&bad_norm, x, 64, ids, 128, out), false);
    std::printf("calls %ld bad %ld\n", calls, bad);
    return bad != 0;
}
"""


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc absent")
def test_launches_at_the_largest_sizes_and_refusals(tmp_path):
    """Grids, blocks and LDS within their limits; what is refused launches nothing."""
    from myelith_amd._lib import lib
    lib()
    so = ROOT / "myelith_amd" / "libmyl_hip.so"
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(LAUNCHES)
    subprocess.run([HIPCC, "-O1", "-std=c++17", "-I", str(ROOT / "include"), str(src), f"-L{so.parent}", f"-l:{so.name}", f"-Wl,-rpath,{so.parent}", "-Wl,--export-dynamic",
                    "-o", str(exe)], check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.stdout[-3000:], r.stderr[-1000:])
    assert int(re.match(r"calls (\d+) bad 0", r.stdout.strip().splitlines()[-1]).group(1)) > 200


# ---- what the calls check and pass on -----------------------------------------------------

i16 = lambda *s: torch.zeros(s, dtype=torch.int16)
i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
i64 = lambda *s: torch.zeros(s, dtype=torch.int64)
u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
i8 = lambda *s: torch.zeros(s, dtype=torch.int8)


def append_args(**over):
    return dict(dict(q=i16(3, 4, 64), k=i16(3, 2, 64), v=i16(3, 2, 64), positions=i32(3), k_pages=i16(7, 2, 16, 64), v_pages=i16(7, 2, 16, 64), tables=i32(3, 5),
                     cos_lut=i16(9, 32), sin_lut=i16(9, 32), rope_frac=8, seqs=i32(3), bias=i16(8 * 64), bias_shifts=u8(8 * 64)), **over)


def paged_args(**over):
    return dict(dict(q=i16(6, 4, 64), k_pages=i16(7, 2, 16, 64), v_pages=i16(7, 2, 16, 64), tables=i32(3, 5), lens=i32(6), score_mult=1, score_shift=20, exp_lut=i16(100),
                     lut_shift=6, prob_frac=14, rows_per_seq=2), **over)


def logprobs_args(**over):
    return dict(dict(logits=i32(3, 50), tokens=i64(3, 2), exp_lut=i16(100), top_n=5), **over)


def test_refused_arguments(bare):  # noqa: F811
    from myelith_amd.backend import HeadNorm
    norm = lambda n=64, **o: HeadNorm(**dict(dict(q_gamma=i8(n), q_gamma_shifts=u8(n), k_gamma=i8(n), k_gamma_shifts=u8(n), rsqrt_lut=i16(9), lut_input_shift=8,
                                                  lut_output_frac=8, inv_n_q20=16384, q_out_frac=10, k_out_frac=10), **o))
    calls = [
        (bare.kv_append_paged_dev, append_args, [
            ("k and v", dict(k=i16(3, 3, 64))), ("k and v", dict(v=i16(2, 2, 64))), ("k and v", dict(k_pages=i16(7, 2, 16, 128), v_pages=i16(7, 2, 16, 128))),
            ("k must be", dict(k=i32(3, 2, 64))), ("positions must be", dict(positions=i64(3))), ("positions must be", dict(positions=i32(4))),
            ("v_pages", dict(v_pages=i16(7, 2, 8, 64))), ("k_pages must be", dict(k_pages=i32(7, 2, 16, 64))), ("same strides", dict(v_pages=i16(7, 2, 17, 64)[:, :, :16])),
            ("elements of a position", dict(k_pages=i16(7, 2, 64, 16).transpose(2, 3), v_pages=i16(7, 2, 64, 16).transpose(2, 3))),
            ("tables must be", dict(tables=i32(3))), ("tables must be", dict(tables=i64(3, 5))), ("entries of a sequence", dict(tables=i32(5, 3).t())),
            ("cos_lut must be", dict(cos_lut=i16(9, 31))), ("sin_lut must be", dict(sin_lut=i16(8, 32))), ("cos_lut must be", dict(cos_lut=i16(9 * 32))),
            ("seqs must be", dict(seqs=i32(2))), ("go together", dict(bias=None)), ("bias must be", dict(bias=i16(7 * 64))), ("bias_shifts must be", dict(bias_shifts=i8(8 * 64))),
            ("norm must be", dict(norm=norm(128))), ("q_out must", dict(q_out=i16(3, 4, 32))), ("q_out must be", dict(q_out=i32(3, 4, 64))),
            ("heads of a row", dict(q=i16(3, 64, 4).transpose(1, 2))), ("on device 0", {})]),
        (bare.attention_paged_dev, paged_args, [
            ("rows_per_seq", dict(rows_per_seq=3)), ("rows_per_seq", dict(rows_per_seq=0)), ("head_dim", dict(q=i16(6, 4, 128))), ("lens must be", dict(lens=i32(3))),
            ("lens must be", dict(lens=i64(6))), ("max_len", dict(max_len=81)), ("max_len", dict(max_len=-1)), ("tables must be", dict(tables=i16(3, 5))),
            ("v_pages", dict(v_pages=i16(6, 2, 16, 64))), ("v_pages must be", dict(v_pages=u8(7, 2, 16, 64))), ("exp_lut must be", dict(exp_lut=i32(100))),
            ("exp_lut must be", dict(exp_lut=i16(10, 10))), ("out must", dict(out=i16(6, 4, 32))), ("out must be", dict(out=i32(6, 4, 64))),
            ("heads of a row", dict(out=i16(6, 64, 4).transpose(1, 2))), ("on device 0", {})]),
        (bare.logprobs_dev, logprobs_args, [
            ("logits must be", dict(logits=i64(3, 50))), ("tokens must be", dict(tokens=i32(3, 2))), ("tokens must be", dict(tokens=i64(2, 2))), ("tokens must be", dict(tokens=i64(3, 2, 1))),
            ("exp_lut must be", dict(exp_lut=i32(100))), ("top_n", dict(top_n=-1)), ("logits of a row", dict(logits=i32(50, 3).t())), ("logprobs must be", dict(logprobs=i64(3))),
            ("entropy must be", dict(entropy=i64(2))), ("top_tokens must be", dict(top_tokens=i64(3, 4))), ("top_logprobs must be", dict(top_logprobs=i32(3, 5))),
            ("on device 0", {})]),
    ]
    for call, args, cases in calls:
        for match, over in cases:
            with pytest.raises(ValueError, match=match):
                call(**args(**over))
    for match, over in [("inv_n_q20", dict(inv_n_q20=-1)), ("inv_n_q20", dict(inv_n_q20=2**20 + 1)), ("q_out_frac", dict(q_out_frac=256)), ("gamma and its shifts", dict(q_gamma=None)),
                        ("gamma and its shifts", dict(q_gamma=None, q_gamma_shifts=None, k_gamma=None, k_gamma_shifts=None)), ("k_gamma must be", dict(k_gamma=i8(63))),
                        ("q_gamma must be", dict(q_gamma=u8(64))), ("rsqrt_lut must be", dict(rsqrt_lut=i32(9)))]:
        with pytest.raises(ValueError, match=match):
            norm(**over)


def test_calls_without_a_context():
    from myelith_amd._lib import SIGNATURES as sig, lib
    for name in ("myl_kv_append_paged_dev", "myl_attention_paged_dev", "myl_logprobs_dev"):
        assert getattr(lib(), name)(None, *[0] * (len(sig[name][1]) - 1)) != 0
    for name in ("myl_attention_paged_workspace", "myl_logprobs_workspace"):
        assert getattr(lib(), name)(None, *[1] * (len(sig[name][1]) - 1)) == 0


def test_expanded_operands_are_refused(recorded):  # noqa: F811
    """An expanded tensor owns fewer elements than its shape says."""
    b, log = recorded
    ap, at, lp = append_args(q_out=i16(3, 4, 64)), paged_args(out=i16(6, 4, 64)), logprobs_args()
    cases = [(b.kv_append_paged_dev, ap, n, (0, 1, 2)) for n in ("q", "k", "v", "q_out")]
    cases += [(b.kv_append_paged_dev, ap, ("k_pages", "v_pages"), (0, 1, 2, 3)), (b.kv_append_paged_dev, ap, "tables", (0, 1))]
    cases += [(b.attention_paged_dev, at, n, (0, 1, 2)) for n in ("q", "out")]
    cases += [(b.attention_paged_dev, at, ("k_pages", "v_pages"), (0, 1, 2, 3)), (b.attention_paged_dev, at, "tables", (0, 1)), (b.logprobs_dev, lp, "logits", (0, 1))]
    for call, args, names, dims in cases:
        names = (names,) if isinstance(names, str) else names
        for dim in dims:
            with pytest.raises(ValueError):
                call(**dict(args, **{n: one(args[n], dim) for n in names}))
                pytest.fail(f"{names} expanded in dimension {dim}: {log[-1]}")


def test_strides_and_sizes_passed_on(recorded):  # noqa: F811
    b, log = recorded
    qkv = i16(3, 9, 64)
    both = i16(7, 2, 16, 2, 64)
    kp, vp = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    b.kv_append_paged_dev(**append_args(q=qkv[:, :4], k=qkv[:, 4:6], v=qkv[:, 6:8], k_pages=kp, v_pages=vp, tables=i32(3, 8)[:, :5], q_out=qkv[:, :4]))
    args = log[-1][1]
    assert args[2] == args[4] == args[6] == 9 * 64 and args[7:11] == (3, 4, 2, 64)
    assert args[24:27] == (3, 5, 8) and args[29:34] == (7, 16, 4096, 64, 128)
    b.attention_paged_dev(**paged_args(k_pages=kp, v_pages=vp, max_len=33))
    args = log[-1][1]
    assert args[10:15] == (7, 16, 4096, 64, 128) and args[16:18] == (5, 5) and args[19] == 33
    b.logprobs_dev(**logprobs_args(logits=i32(3, 60)[:, 4:54], tokens=i64(3)))
    args = log[-1][1]
    assert args[2:5] == (3, 50, 60) and args[8:10] == (1, 5)
    # one row, one page, one sequence: strides that say nothing
    odd = lambda dtype, shape, strides: torch.zeros(4096, dtype=dtype).as_strided(shape, strides)
    b.attention_paged_dev(**paged_args(q=odd(torch.int16, (1, 4, 64), (3, 64, 1)), k_pages=odd(torch.int16, (1, 1, 16, 64), (5, 0, 64, 1)),
                                       v_pages=odd(torch.int16, (1, 1, 16, 64), (7, 1, 64, 1)), tables=odd(torch.int32, (1, 2), (0, 1)), lens=i32(1), rows_per_seq=1))
    args = log[-1][1]
    assert args[4] == 256 and args[12:15] == (1024, 1024, 64) and args[17] == 2


def calls_of(b):
    space = dict(workspace=u8(256))
    return [(b.kv_append_paged_dev, on_gpu(append_args()), on_gpu(dict(q_out=i16(3, 4, 64)))),
            (b.attention_paged_dev, on_gpu(paged_args()), on_gpu(dict(space, out=i16(6, 4, 64)))),
            (b.logprobs_dev, on_gpu(logprobs_args()),
             on_gpu(dict(space, logprobs=i64(3, 2), entropy=i64(3), top_tokens=i64(3, 5), top_logprobs=i64(3, 5))))]


def test_allocated_memory_is_written_after_its_last_use(streams, monkeypatch):  # noqa: F811
    """A context on another stream than torch's waits behind the call's allocations."""
    b, log = streams
    monkeypatch.setattr(FakeStream, "torchs", 7)
    b._own_stream = 3
    for call, args, given in calls_of(b):
        for left_out in [given, *([k] for k in given)]:
            log.clear()
            OnGpu.recorded.clear()
            call(**args, **{k: v for k, v in given.items() if k not in left_out})
            kinds = [e[0] if e[0] in ("empty", "wait") else "launch" for e in log if not e[0].endswith("_workspace")]
            assert kinds == ["empty"] * len(left_out) + ["wait", "launch"], (call.__name__, list(left_out), kinds)
            assert [s for _, s in OnGpu.recorded] == [9] * len(left_out)
        log.clear()
        call(**args, **given)
        assert len(log) == 1, log
    monkeypatch.setattr(FakeStream, "captured", (7,))
    for call, args, given in calls_of(b):
        with pytest.raises(ValueError, match="captured"):
            call(**args)


def test_scalars_outside_their_type_are_refused(recorded):  # noqa: F811
    b, log = recorded
    for call, args, names in [(b.kv_append_paged_dev, append_args, ("rope_frac", "q_frac", "k_frac", "v_frac")),
                              (b.attention_paged_dev, paged_args, ("score_shift", "lut_shift", "prob_frac"))]:
        for name in names:
            for v in (-1, 256, 270):
                with pytest.raises(ValueError, match=name):
                    call(**args(**{name: v}))
    for v in (-2**63 - 1, 2**63):
        with pytest.raises(ValueError, match="score_mult"):
            b.attention_paged_dev(**paged_args(score_mult=v))
    assert not log


def test_allocated_queries_of_left_out_rows_are_zero(streams, monkeypatch):  # noqa: F811
    """The kernel writes nothing for a row that is left out: memory that the call allocates is
    cleared before it on the context's stream, a caller's q_out is not touched."""
    b, log = streams
    empty, zero = torch.empty, OnGpu.zero_
    monkeypatch.setattr(torch, "empty", lambda *a, **k: empty(*a, **k).fill_(77))
    monkeypatch.setattr(OnGpu, "zero_", lambda t: (log.append(("zero", torch.cuda.current_stream().cuda_stream)), zero(t))[1])
    args = on_gpu(append_args(positions=torch.tensor([0, -1, 5], dtype=torch.int32)))
    for torchs, own, kinds in ((7, 3, ["empty", "wait", "zero", "launch"]), (9, 3, ["empty", "zero", "launch"]), (0, 9, ["empty", "zero", "launch"])):
        monkeypatch.setattr(FakeStream, "torchs", torchs)
        b._own_stream = own
        log.clear()
        got = b.kv_append_paged_dev(**args)
        assert [e[0] if e[0] in ("empty", "wait", "zero") else "launch" for e in log] == kinds and ("zero", 9) in log
        assert log[-1][0] == "myl_kv_append_paged_dev" and log[-1][1][34] == got.data_ptr() and not got.any()
    log.clear()
    given = torch.full((3, 4, 64), -7, dtype=torch.int16).as_subclass(OnGpu)
    assert b.kv_append_paged_dev(**dict(args, q_out=given)) is given and (given == -7).all() and len(log) == 1


KEPT = PLANS[:PLANS.index("// pieces of a workspace")].replace('#include "serve_plan.h"', '#include "paged_plan.h"') + r"""
// A size of the smaller call: often the same, one less, a half, or any.
static size_t below(size_t n) {
    const uint64_t r = next() % 6;
    return r < 2 ? n : r == 2 ? n - 1 : r == 3 ? n / 2 : r == 4 ? n - n / 8 : (size_t)(next() % (n + 1));
}
static void hold(PagedShape l, PagedShape s, int cus) {
    if (paged_refuse(l) || paged_refuse(s)) return;
    const size_t large = paged_plan(l, cus).bytes, small = paged_plan(s, cus).bytes;
    CHECK(small <= large, "%zu bytes for %zu x %zu rows of %zu keys, %zu for %zu x %zu of %zu, heads %zu / %zu", small, s.n_seqs, s.rows_per_seq, s.max_len, large,
          l.n_seqs, l.rows_per_seq, l.max_len, l.heads, l.kv_heads);
}
int main() {
    hold({64, 1, 28, 4, 128, 2500}, {21, 3, 28, 4, 128, 2500}, 256);
    hold({241, 1, 1, 1, 64, 2500}, {1, 241, 1, 1, 64, 2500}, 256);
    for (int i = 0; i < 300000; ++i) {
        const size_t kvh = upto(16), hd = i & 1 ? 64 : 128;
        const PagedShape l{upto(i & 2 ? 80 : 3000), upto(i & 4 ? 9 : 3000), kvh * upto(20), kvh, hd, upto(131073) - 1};
        PagedShape s = l;
        s.rows_per_seq = i & 8 ? upto(40) : upto(l.n_seqs * l.rows_per_seq);
        s.n_seqs = below(l.n_seqs * l.rows_per_seq / s.rows_per_seq);
        s.max_len = below(l.max_len);
        hold(l, s, i % 3 ? 256 : (int)upto(512));
    }
    std::printf("checked %ld bad %ld\n", checked, bad);
    return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ absent")
def test_an_attention_workspace_serves_as_many_rows_of_any_sequences(tmp_path):
    """Rows may change from one per sequence to several (drafts of fewer requests): no more rows in
    all, of the same heads, and no more keys, fit where the former did."""
    src, exe = tmp_path / "kept.cpp", tmp_path / "kept"
    src.write_text(KEPT)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I", str(CSRC),
                    str(src), "-o", str(exe)], check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, (r.stdout[-3000:], r.stderr[-3000:])
    assert int(re.match(r"checked (\d+) bad 0", r.stdout.strip().splitlines()[-1]).group(1)) > 100000


# the launches with what each kernel was allowed before: dynamic LDS by function
LDS = PROGRAM[:PROGRAM.index("static long calls")].replace("#include <vector>", "#include <vector>\n#include <map>\n#include <set>\n#include \"paged_plan.h\"").replace(
    "struct Launch { dim3 grid, block; size_t lds; };", "struct Launch { dim3 grid, block; size_t lds, allowed; };\nstatic std::map<const void*, std::vector<int>> attributes;").replace(
    "hipLaunchKernel(const void*, dim3", "hipLaunchKernel(const void* f, dim3").replace(
    "launches.push_back({grid, block, lds});", "launches.push_back({grid, block, lds, attributes[f].empty() ? 0 : (size_t)attributes[f].back()});").replace(
    "hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return", "hipError_t hipFuncSetAttribute(const void* f, hipFuncAttribute, int v) { return attributes[f].push_back(v),") + r"""
template <class T>
static T* at(size_t n) { return reinterpret_cast<T*>(n); }  // never read on the host
static myl_ctx* c = nullptr;
static int attend(size_t seqs, size_t heads, size_t kvh, size_t hd, size_t keys, size_t page, size_t lut) {
    const size_t bytes = myl_attention_paged_workspace(c, seqs, 1, heads, kvh, hd, keys), ld = heads * hd, len = (keys + page - 1) / page;
    const int16_t* x = at<int16_t>(1 << 20);
    return myl_attention_paged_dev(c, x, seqs, 1, ld, heads, kvh, hd, x, x, 1000, page, kvh * page * hd, page * hd, hd, at<int32_t>(64), len, len, at<int32_t>(64), keys, 2896, 21, x,
                                   lut, 6, 14, at<int16_t>(1 << 22), ld, at<void>(1 << 23), bytes);
}
int main() {
    if (myl_init(0, &c) != MYL_OK) return 2;
    long n = 0, large = 0, bad = 0;
    for (size_t hd : {(size_t)64, (size_t)128})
        for (size_t lut : {(size_t)1, (size_t)2662, (size_t)32768})
            for (size_t page : {(size_t)1, (size_t)8, (size_t)16, (size_t)64})
                for (size_t g : {(size_t)1, (size_t)7, (size_t)8, (size_t)9, (size_t)16})
                    for (size_t seqs : {(size_t)1, (size_t)24, (size_t)64})
                        for (size_t keys = 64; keys <= 40000; keys += keys < 1024 ? 64 : keys / 3) {
                            attributes.clear();  // the first call of a process
                            launches.clear();
                            if (attend(seqs, 2 * g, 2, hd, keys, page, lut) != MYL_OK) return 3;
                            for (const Launch& l : launches) {
                                ++n;
                                // 64 KiB of both without the attribute; paged_sum_kernel's table is its own
                                const bool more = l.lds + 4800 > 65536;
                                large += more;
                                if ((more && l.allowed < l.lds) || l.lds + 4800 > 160 * 1024) {
                                    if (bad++ < 10) std::printf("%zu x %zu heads of %zu, %zu keys, pages of %zu: %zu bytes, %zu allowed\n", seqs, 2 * g, hd, keys, page, l.lds, l.allowed);
                                }
                            }
                        }
    std::printf("launches %ld large %ld bad %ld\n", n, large, bad);
    return bad != 0;
}
"""


def run_program(tmp_path, text):
    """A program that has its own functions in place of HIP's."""
    from myelith_amd._lib import lib
    lib()
    so = ROOT / "myelith_amd" / "libmyl_hip.so"
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(text)
    subprocess.run([HIPCC, "-O1", "-std=c++17", "-I", str(ROOT / "include"), "-I", str(CSRC), str(src), f"-L{so.parent}", f"-l:{so.name}", f"-Wl,-rpath,{so.parent}",
                    "-Wl,--export-dynamic", "-o", str(exe)], check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.stdout[-3000:], r.stderr[-1000:])
    return r.stdout


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc absent")
def test_launches_past_64_kib_of_both_kinds_of_lds_ask_for_it(tmp_path):
    """What a kernel declares counts beside what a launch gives it."""
    n = re.match(r"launches (\d+) large (\d+) bad 0", run_program(tmp_path, LDS).strip().splitlines()[-1])
    assert int(n.group(1)) > 5000 and int(n.group(2)) > 500


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc absent")
def test_a_kernel_asks_for_the_same_lds_in_every_call(tmp_path):
    """The attribute belongs to the process: what one call asks for must not lower another's, made at
    once from another host thread."""
    text = LDS[:LDS.index("int main() {")] + r"""
int main() {
    if (myl_init(0, &c) != MYL_OK) return 2;
    for (size_t hd : {(size_t)64, (size_t)128})
        for (size_t page : {(size_t)8, (size_t)16})
            for (size_t g : {(size_t)7, (size_t)16})
                for (size_t seqs : {(size_t)24, (size_t)64})
                    for (size_t keys = 64; keys <= 40000; keys += keys < 1024 ? 64 : keys / 3)
                        if (attend(seqs, 2 * g, 2, hd, keys, page, 2662) != MYL_OK) return 3;
    long several = 0, kernels = 0, least = 1 << 30;
    for (const auto& f : attributes) {
        if (f.second.empty()) continue;  // looked up by a launch
        const std::set<int> values(f.second.begin(), f.second.end());
        ++kernels;
        several += values.size() > 1;
        least = std::min(least, (long)*values.begin());
    }
    std::printf("kernels %ld several %ld least %ld\n", kernels, several, least);
    return 0;
}
"""
    n = re.match(r"kernels (\d+) several (\d+) least (\d+)", run_program(tmp_path, text).strip().splitlines()[-1])
    assert int(n.group(1)) >= 8 and int(n.group(2)) == 0 and int(n.group(3)) <= 160 * 1024 - 4800, n.group(0)
