// serve_plan.h -- what the host decides for the operators of a serving step:
// which calls are refused, how the work is cut, how the workspace is laid out.
// Plain C++ with no HIP dependency: the entry points call these functions, and a
// host build of them runs under AddressSanitizer and
// UndefinedBehaviorSanitizer in the CPU tests.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace myl {

constexpr size_t kInt = 0x7FFFFFFF;

// Pieces of a workspace in 256-byte steps.  A piece has room for every call none of whose
// sizes is larger, so that a program keeps the workspace of its largest step: where fewer
// rows or keys are cut into more parts, the room is a bound that grows with the sizes.
struct Layout {
    size_t used = 0;
    size_t take(size_t n, size_t each) {
        const size_t off = used;
        used += (n * each + 255) & ~(size_t)255;
        return off;
    }
};

// ---- adapters beside a projection ---------------------------------------------

constexpr size_t kAdapterMaxRank = 256;               // |sum B u| <= 2^7 2^15 2^8 = 2^30
constexpr size_t kAdapterMaxRows = (size_t)1 << 23;   // a block per slot, 256 threads each, below 2^32
constexpr size_t kAdapterMaxSide = (size_t)1 << 30;
constexpr size_t kAdapterAccElems = (size_t)512 << 10;  // products with more outputs do not split K
constexpr int kAdapterWindow = 256, kAdapterUnit = 128;

struct AdapterShape {
    size_t M, N, K, rank, n;
};

inline const char* adapter_refuse(const AdapterShape& s) {
    if (s.K == 0) return "K must be > 0";
    if (s.M > kAdapterMaxRows || s.N > kAdapterMaxSide || s.K > kAdapterMaxSide || s.n > kInt)
        return "shape too large (2^23 rows, 2^30 columns, 2^31 - 1 adapters)";
    if (s.n == 0) return nullptr;
    if (s.rank == 0 || s.rank > kAdapterMaxRank) return "rank must be 1 to 256";
    const size_t most = (size_t)1 << 47;  // bytes of A and B
    if (s.n > most / (s.K * s.rank) || (s.N > 0 && s.n > most / (s.N * s.rank))) return "adapters larger than the address space";
    return nullptr;
}

// The rows of one adapter within a window of 256 rows, 16 at a time, are a tile of x A: at
// most down_tiles in a window.  A block takes a tile, 16 rank_tiles rows of A and 4 per_wave
// units of 128 of K (a quarter each wave).  64 at a time they are a tile of u B: at most
// up_tiles in a window; a block takes one and n_chunk columns.
struct AdapterPlan {
    int windows, down_tiles, up_tiles, rank_tiles, rank_groups, splits, per_wave, n_chunk, n_chunks, rank_pad;
    size_t planes_bytes, acc_elems, off_planes, off_acc, off_part, off_tiles, bytes;
};
constexpr int64_t kAdapterMaxChunk = (int64_t)1 << 20;
constexpr size_t kAdapterTileBytes = 72;  // adapter, rows, and their 64 places in the window

// M x splits of any smaller call, which adapter_plan bounds by max(min(up(2 CUs, blocks),
// units / 4), units / 2048): M up(2 CUs, blocks) <= M + 2 CUs M / blocks, and blocks is at
// least 1 and at least M / 16 (a tile for 16 rows).
inline size_t adapter_most_parts(const AdapterShape& s, int cus) {
    const size_t units = (s.K + kAdapterUnit - 1) / kAdapterUnit;
    return std::max(std::min(s.M + 2 * (size_t)cus * std::min<size_t>(s.M, 16), s.M * ((units + 3) / 4)), s.M * ((units + 4 * 512 - 1) / (4 * 512)));
}

inline AdapterPlan adapter_plan(const AdapterShape& s, int cus) {
    AdapterPlan p{};
    Layout l;
    if (s.M >= 2) {
        p.planes_bytes = 2 * s.M * s.K;
        p.acc_elems = s.M * s.N <= kAdapterAccElems ? s.M * s.N : 0;
        p.off_planes = l.take(p.planes_bytes, 1);
        p.off_acc = l.take(std::max<size_t>(std::min(s.M * s.N, kAdapterAccElems), 1), 8);
    }
    if (s.M && s.N && s.n) {
        const int w = (int)std::min<size_t>(s.M, kAdapterWindow), d = (int)std::min<size_t>(s.n, (size_t)w);
        p.windows = (int)((s.M + kAdapterWindow - 1) / kAdapterWindow);
        p.down_tiles = d + (w - d) / 16;
        p.up_tiles = d + (w - d) / 64;
        const int tiles = (int)(s.rank + 15) / 16;
        p.rank_tiles = tiles <= 2 ? tiles : 4;
        p.rank_groups = (tiles + p.rank_tiles - 1) / p.rank_tiles;
        p.rank_pad = 16;
        while (p.rank_pad < (int)s.rank) p.rank_pad *= 2;
        auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
        // Two blocks per CU (61 rows, rank 64, K 18944: 14.7 us; four: 16.6), a unit per wave at
        // least and 512 at most: its i32 sums hold 2^16 products of up to 2^14.
        const int64_t units = up((int64_t)s.K, kAdapterUnit), blocks = (int64_t)p.windows * p.down_tiles * p.rank_groups;
        const int64_t want = std::max(std::min(up(2 * (int64_t)cus, blocks), up(units, 4)), up(units, 4 * 512));
        p.per_wave = (int)up(units, 4 * want);
        p.splits = (int)up(units, 4 * (int64_t)p.per_wave);
        // Four blocks per CU (2003 rows: 55 us; eight: 62), 256 columns at least.
        const int64_t cols = up((int64_t)s.N, up(4 * (int64_t)cus, (int64_t)p.windows * p.up_tiles));
        p.n_chunk = (int)std::min<int64_t>(up(cols, 256) * 256, kAdapterMaxChunk);
        p.n_chunks = (int)up((int64_t)s.N, p.n_chunk);
        p.off_part = l.take(adapter_most_parts(s, cus) * (size_t)p.rank_pad, 8);
        p.off_tiles = l.take((size_t)p.windows * (size_t)p.up_tiles, kAdapterTileBytes);
    }
    p.bytes = std::max<size_t>(l.used, 256);  // 0 stands for sizes that a call refuses
    return p;
}

// ---- attention over a shared prefix ------------------------------------------

// At most 65536 keys per row: with non-negative table entries below 2^15 the exp sums
// stay below 2^31, and sum p |v| <= (2^14 + keys / 2) 2^15 < 2^31.
constexpr size_t kPrefixMaxKeys = 65536;
constexpr size_t kPrefixMaxRows = 65535;
constexpr size_t kPrefixMaxPairs = (size_t)1 << 22;  // rows x heads
constexpr size_t kPrefixMaxLut = 32768;

struct PrefixShape {
    size_t n_seqs, rows_per_seq, heads, kv_heads, head_dim, prefix_len, max_tail;
};

// The reason why a shape is refused, or null.
inline const char* prefix_refuse(const PrefixShape& s) {
    if (s.kv_heads == 0 || s.heads == 0 || s.heads % s.kv_heads) return "heads must be a multiple of kv_heads";
    if (s.heads > kPrefixMaxRows || s.n_seqs > kPrefixMaxRows || s.rows_per_seq > kPrefixMaxRows ||
        s.n_seqs * s.rows_per_seq > kPrefixMaxRows || s.n_seqs * s.rows_per_seq * s.heads > kPrefixMaxPairs)
        return "too many rows or heads (65535 each, 2^22 together)";
    if (s.prefix_len > kPrefixMaxKeys || s.max_tail > kPrefixMaxKeys - s.prefix_len) return "more than 65536 keys per row";
    return nullptr;
}

// The work of a call.  The vectors (query heads of rows) that read one KV head are cut
// into tiles, the keys of the prefix and of the tails into ranges of a multiple of 64; a
// block takes one tile and one range.  Prefix tiles hold vectors of every row, tail
// tiles those of one sequence.
constexpr int kPrefixQkTile = 64, kPrefixPvTile = 64;

constexpr size_t kPrefixShortHeads = 8, kPrefixShortWork = 320 * 128;  // heads of a KV head; keys x head_dim
// LDS of a block that does a row's heads by itself: scores, probabilities, sums.
inline size_t prefix_short_lds(int G, int cap, size_t hd) { return (size_t)G * ((size_t)cap * 6 + hd * 4); }

// The whole words of an exp table, which wide loads may touch: not an odd last entry.
constexpr uint32_t prefix_table_bytes(uint32_t lut_len) { return lut_len / 2 * 4; }

struct PrefixPlan {
    int short_cap;         // > 0: one launch, blocks with room for so many keys; nothing below is used
    int G, vp, vt;       // query heads per KV head; vectors per KV head: of all rows, of one sequence
    struct Cut {
        int tp, tt;      // tiles of each
        int64_t blocks_p, blocks_t;
    } qk, pv;
    int np, rp, nt, rt;  // ranges of prefix and tail keys, keys per range
    int pgroups, tgroups;  // 16-key groups of the prefix and of a tail, rounded up to 64 keys
    size_t pairs;        // rows x heads
    size_t off_max, off_sum, off_pexp, off_texp, off_out, bytes;
};

// One launch with a block per row and KV head, which reads its keys for itself, or four
// launches that share the keys between rows.  Measured with seven heads per KV head, one /
// four launches: 320 keys of 128 18.1 / 22.4 us for one row, 18.6 / 24.3 for 16, 46.1 / 47.4
// for 256 rows of four KV heads; 512 keys 25.3 / 22.9, 25.7 / 25.0, 69.2 / 46.5; 512 keys of 64
// 18.1 / 21.9, 18.5 / 22.8, and 24.8 / 30.7 for 256 rows of two KV heads.  A wave does one head.
inline bool prefix_short(const PrefixShape& s, int cus) {
    const size_t blocks = s.n_seqs * s.rows_per_seq * s.kv_heads, keys = s.prefix_len + s.max_tail;
    return keys > 0 && s.heads / s.kv_heads <= kPrefixShortHeads && blocks <= 4 * (size_t)cus && keys * s.head_dim <= kPrefixShortWork;
}

// How many steps of 64 keys a range takes at least.
inline int prefix_least_steps(int steps) {
    int least = 2;
    while (7 * least * least < steps) ++least;
    return least;
}

// Vectors x ranges of any smaller call, `vectors` (of one KV head, or of one sequence and KV head)
// in each of `groups`: at most as many ranges as the steps allow (the most with the least
// steps of a range, or one less, which stop at 7 (least - 1)^2 steps), and at most
// 2 CUs / (groups ceil(vectors / 64)) of them, or one.
inline size_t prefix_most_parts(size_t vectors, size_t groups, size_t keys, int cus) {
    const int steps = (int)((keys + 63) / 64), least = prefix_least_steps(steps);
    const size_t ranges = (size_t)std::max((steps + least - 1) / least, least > 2 ? 7 * (least - 1) : 0);
    return std::min(vectors * groups * ranges, std::max(vectors * groups, std::min<size_t>(vectors, kPrefixPvTile) * 2 * (size_t)cus));
}

inline PrefixPlan prefix_plan(const PrefixShape& s, int cus) {
    PrefixPlan p{};
    const int64_t R = (int64_t)(s.n_seqs * s.rows_per_seq), kvh = (int64_t)s.kv_heads;
    p.G = (int)(s.heads / s.kv_heads);
    p.vp = (int)(R * p.G);
    p.vt = (int)(s.rows_per_seq * p.G);
    const int P = (int)s.prefix_len, T = (int)s.max_tail;
    if (prefix_short(s, cus)) {
        p.short_cap = (P + T + 63) / 64 * 64;
        p.bytes = 256;
        return p;
    }
    auto tiles = [](int v, int tile) { return (v + tile - 1) / tile; };
    // Two blocks of the P.V tiles per CU (the prefix's and the tails' each), but at least two
    // steps of 64 keys a range, and e of them where there are 7 (e - 1)^2 or more: each range costs
    // every later launch a partial result per vector, each step costs its block.  us a call at
    // ranges of at least 1 / 2 / 4 / 8 steps: 64 rows, 1000 keys 53 / 40 / 41; one row, 16000
    // keys - / 45 / 35 / 32; four rows, 30000 keys 56 / 55 / 52 / 47; 24 rows, 4000 keys 43 / 42 / 38
    // / 46 (3: 36).
    auto cut = [&](int keys, int64_t per_range, int& n, int& len) {
        n = len = 0;
        if (keys == 0 || per_range == 0) return;
        const int steps = (keys + 63) / 64;
        const int64_t want = std::max<int64_t>(1, 2 * cus / per_range);
        int each = (int)((steps + std::min<int64_t>(want, steps) - 1) / std::min<int64_t>(want, steps));
        each = std::max(each, prefix_least_steps(steps));
        len = 64 * each;
        n = (steps + each - 1) / each;
    };
    cut(P, kvh * tiles(p.vp, kPrefixPvTile), p.np, p.rp);
    cut(T, kvh * (int64_t)s.n_seqs * tiles(p.vt, kPrefixPvTile), p.nt, p.rt);
    auto blocks = [&](int tile, PrefixPlan::Cut& c) {
        c.tp = tiles(p.vp, tile);
        c.tt = tiles(p.vt, tile);
        c.blocks_p = (kvh * c.tp * p.np + 7) / 8 * 8;
        c.blocks_t = kvh * (int64_t)s.n_seqs * c.tt * p.nt;
    };
    blocks(kPrefixQkTile, p.qk);
    blocks(kPrefixPvTile, p.pv);
    p.pgroups = (P + 63) / 64 * 4;
    p.tgroups = (T + 63) / 64 * 4;
    p.pairs = (size_t)R * s.heads;
    Layout l;
    const size_t parts = prefix_most_parts((size_t)p.vp, s.kv_heads, s.prefix_len, cus) +
                         prefix_most_parts((size_t)p.vt, s.kv_heads * s.n_seqs, s.max_tail, cus);
    p.off_max = l.take(parts, 4);
    p.off_sum = l.take(parts, 4);
    p.off_pexp = l.take((size_t)kvh * (size_t)tiles(p.vp, 16) * (size_t)p.pgroups * 256, 2);
    p.off_texp = l.take((size_t)(kvh * (int64_t)s.n_seqs) * (size_t)tiles(p.vt, 16) * (size_t)p.tgroups * 256, 2);
    p.off_out = l.take(parts * s.head_dim, 4);
    p.bytes = std::max<size_t>(l.used, 256);  // 0 stands for sizes that a call refuses
    return p;
}

// ---- draft verification -------------------------------------------------------

constexpr size_t kVerifyMaxVocab = (size_t)1 << 20, kVerifyMaxDrafts = 1024, kVerifyMaxLut = 32768;
constexpr size_t kVerifyMaxRows = 65535;
constexpr int kVerifyChunk = 8192;  // values of a row per block

struct VerifyShape {
    size_t n_seqs, k, vocab, lut_len;
};

inline const char* verify_refuse(const VerifyShape& s) {
    if (s.vocab == 0 || s.vocab > kVerifyMaxVocab) return "the vocabulary must hold 1 to 2^20 tokens";
    if (s.k > kVerifyMaxDrafts || s.n_seqs > kVerifyMaxRows || s.n_seqs * (2 * s.k + 1) > kVerifyMaxRows)
        return "too many drafts (1024 a sequence) or rows (65535)";
    if (s.lut_len > kVerifyMaxLut) return "the exp table must hold 1 to 32768 entries";
    return nullptr;
}

// bins: how far below its maximum a logit can lie and have a weight, at four table entries a
// step; words: pairs of 16-bit counters for them.
struct VerifyPlan {
    int chunks;
    uint32_t bins, words;
    size_t off_stat, off_max, off_counts, off_sums, off_first, bytes;
};

inline VerifyPlan verify_plan(const VerifyShape& s) {
    VerifyPlan p{};
    p.chunks = (int)((s.vocab + kVerifyChunk - 1) / kVerifyChunk);
    p.bins = (uint32_t)((s.lut_len + 3) / 4);
    p.words = (p.bins + 1) / 2;
    const size_t rows = s.n_seqs * (2 * s.k + 1), c = (size_t)p.chunks;
    Layout l;
    p.off_stat = l.take(rows, 16);
    p.off_max = l.take(rows * c, 4);
    p.off_counts = l.take(rows * c * p.words, 4);
    p.off_sums = l.take(std::max(s.n_seqs * c * (kVerifyChunk / 256), rows * c), 8);
    p.off_first = l.take(s.n_seqs, 4);
    p.bytes = std::max<size_t>(l.used, 256);
    return p;
}

}  // namespace myl
