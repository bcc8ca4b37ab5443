// paged_plan.h -- what the host decides for the operators over a paged cache and
// for log probabilities: which calls are refused, how the work is cut, how the
// workspace is laid out (Layout, serve_plan.h).  Plain C++ with no HIP dependency:
// a host build of it runs under AddressSanitizer and UndefinedBehaviorSanitizer
// in the CPU tests.
#pragma once

#include "serve_plan.h"

namespace myl {

// ---- the pages of a cache -------------------------------------------------------

// Elements of strides and addresses: pages x page stride is formed in 64 bits.
constexpr size_t kPagedMaxStride = (size_t)1 << 40, kPagedMaxPage = 65536;
// int32 ids; a table's places are counted in 32 bits
constexpr size_t kPagedMaxIds = kInt;

struct PagesShape {
    size_t n_pages, page_size, page_stride, head_stride, pos_stride, n_seqs, table_len, table_stride, kv_heads, head_dim;
};

// Strides below a head vector's length are refused where they could be told from
// others: positions, heads and pages of one would lie in one another.
inline const char* pages_refuse(const PagesShape& s) {
    if (s.page_size == 0 || s.page_size > kPagedMaxPage) return "pages hold 1 to 65536 positions";
    if (s.n_pages == 0 || s.n_pages > kPagedMaxIds || s.table_len > kPagedMaxIds || s.n_seqs > kPagedMaxIds)
        return "1 to 2^31 - 1 pages, at most 2^31 - 1 sequences and table entries";
    if ((s.page_size > 1 && s.pos_stride < s.head_dim) || (s.kv_heads > 1 && s.head_stride < s.head_dim) ||
        (s.n_pages > 1 && s.page_stride < s.head_dim))
        return "page strides too small";
    if (s.page_stride > kPagedMaxStride || s.head_stride > kPagedMaxStride || s.pos_stride > kPagedMaxStride)
        return "page strides too large (2^40)";
    if (s.n_seqs > 1 && s.table_stride < s.table_len) return "table stride too small";
    if (s.table_stride > kPagedMaxStride) return "table stride too large (2^40)";
    return nullptr;
}

// ---- appending ------------------------------------------------------------------

// A thread takes 8 dimensions and the 8 they rotate with: threads of a call stay below 2^31.
inline const char* append_refuse(size_t rows, size_t heads, size_t kv_heads, size_t head_dim) {
    if (heads > kInt || kv_heads > kInt || kv_heads == 0) return "kv_heads must be > 0, heads and kv_heads below 2^31";
    const size_t per_row = (heads + 2 * kv_heads) * (head_dim / 16);
    if (per_row > kInt || rows > (kInt - 255) / per_row) return "too many rows or heads (2^31 pieces of 16 dimensions)";
    return nullptr;
}

// Rows of a thread: as many as leave a CU eight blocks of 256 threads, in fours (or one).  us with 1 / 4 / 8 / 16
// rows a thread, 28 + 2 x 4 heads of 128: with biases 1503 rows 13.9 / 13.3 / 16.1 / 25.0, 8000 49.0 / 40.5 /
// 40.8 / 42.1, 16384 92.4 / 70.6 / 69.9 / 75.3; with norms (three to five blocks fit a CU at once)
// 1503 14.0 / 16.9 / 21.3 / 36.5, 4000 27.5 / 32.3 / 36.2 / 48.8, 8000 52.6 / 52.5 / 56.9 / 64.6, 16384
// 96.8 / 92.1 / 94.1 / 107; with both 16384 160 / 114 / 106 / 114.
inline int append_group(size_t rows, size_t per_row, int cus) {
    const size_t each = rows * per_row / ((size_t)cus * 8 * 256);
    return each < 4 ? 1 : (int)std::min<size_t>(each / 4 * 4, 16);
}

// ---- attention ------------------------------------------------------------------

// At most 131072 keys per row: with non-negative table entries below 2^15 the exp sums
// stay below 2^32.
constexpr size_t kPagedMaxKeys = 131072;
constexpr size_t kPagedMaxRows = 65535;
constexpr size_t kPagedMaxPairs = (size_t)1 << 22;  // rows x heads
constexpr size_t kPagedMaxLut = 32768;
constexpr size_t kPagedMaxWork = (size_t)1 << 33;  // keys of all tiles: blocks of 256 threads below 2^32 of them
constexpr int kPagedTile = 16;                     // query vectors of a tile

struct PagedShape {
    size_t n_seqs, rows_per_seq, heads, kv_heads, head_dim, max_len;
};

inline const char* paged_refuse(const PagedShape& s) {
    if (s.kv_heads == 0 || s.heads == 0 || s.heads % s.kv_heads) return "heads must be a multiple of kv_heads";
    if (s.heads > kPagedMaxRows || s.n_seqs > kPagedMaxRows || s.rows_per_seq > kPagedMaxRows ||
        s.n_seqs * s.rows_per_seq > kPagedMaxRows || s.n_seqs * s.rows_per_seq * s.heads > kPagedMaxPairs)
        return "too many rows or heads (65535 each, 2^22 together)";
    if (s.max_len > kPagedMaxKeys) return "more than 131072 keys per row";
    const size_t tiles = (s.rows_per_seq * (s.heads / s.kv_heads) + kPagedTile - 1) / kPagedTile;
    if (s.n_seqs * s.kv_heads * tiles * s.max_len > kPagedMaxWork) return "too many keys in all (2^33 for each 16 query heads that share a KV head)";
    return nullptr;
}

// The query vectors (heads of rows) that read one sequence's KV head are cut into tiles of at
// most 16, the keys into ranges of a multiple of 64; a block takes one tile and one range.
// Within a range of at most 1024 keys sum p |v| <= (2^14 + 2^9) 2^15 < 2^30.
constexpr int kPagedMaxRange = 1024, kPagedMidRange = 512, kPagedLeastRange = 128;
constexpr int kPagedLdsLut = 8192;  // exp table entries that a block copies
constexpr size_t kPagedLds = 160 * 1024;  // of a block, all told
constexpr size_t kPagedOwnLds = 4800;  // the most LDS that a kernel declares beside what a launch may have to ask for

// The pages that a range of keys can touch.
constexpr int paged_table_entries(int range, int page) { return (range / page + 3) / 2 * 2; }  // an even number: what follows is 16-byte aligned

struct PagedPlan {
    int width, tiles;   // vectors of a tile; tiles of a sequence's KV head
    int keys;           // max_len rounded up to 64
    int ranges, range;  // ranges of keys, keys of a range
    bool in_one;        // one launch, a block per tile
    size_t parts;       // sequences x KV heads x tiles
    int64_t blocks;     // parts x ranges, the last eight filled up
    size_t off_z, off_e, off_max, off_sum, off_holes, off_out, bytes;
};

// LDS of a block that does all of a tile by itself: rings of eight waves, scores, p, pages, table.
constexpr size_t kPagedShortKeys = 1024, kPagedShortScores = 8192;
inline size_t paged_short_lds(const PagedPlan& p, size_t hd, int page, uint32_t lut_len) {
    const size_t w = p.width <= 8 ? 8 : 16, keys = (size_t)p.keys;
    const size_t lut = (std::min<size_t>(lut_len, kPagedLdsLut) + 8) / 8 * 16;
    return 8 * 2 * 32 * hd + keys * ((size_t)p.width * 4 + w * 2) + (size_t)paged_table_entries(p.range, page) * 8 + lut;
}

// One launch with a block per tile, or four that split the keys: up to 640 keys of 128, or 1024 keys
// (as far as their scores fit) where an eighth of the CUs has a block.  us of a call's launches, in
// one / split, heads of 128, seven to a KV head of four: one row of 130 keys 8.8 / 16.4, 600 15.1 / 17.0,
// 1000 21.9 / 17.6; eight rows of 1000 21.4 / 21.0; 64 of 300 13.0 / 22.4, of 1000 25.6 / 39.8; 256 of
// 1000 88 / 100.
inline bool paged_in_one(const PagedShape& s, const PagedPlan& p, int cus) {
    return s.max_len <= kPagedShortKeys && s.max_len * (size_t)p.width <= kPagedShortScores &&
           (s.max_len * s.head_dim <= 640 * 128 || p.parts * 8 >= (size_t)cus);
}

inline PagedPlan paged_plan(const PagedShape& s, int cus) {
    PagedPlan p{};
    const size_t vectors = s.rows_per_seq * (s.heads / s.kv_heads);
    p.tiles = (int)((vectors + kPagedTile - 1) / kPagedTile);
    p.width = p.tiles ? (int)((vectors + p.tiles - 1) / p.tiles) : 0;
    p.parts = s.n_seqs * s.kv_heads * (size_t)p.tiles;
    p.keys = (int)((s.max_len + 63) / 64 * 64);
    if (p.parts && p.keys) {
        if (paged_in_one(s, p, cus)) {
            p.in_one = true;
            p.range = p.keys;
        } else {
            // A block per CU where ranges of 128 to 512 keys make it, then two where up to 1024 keys
            // do.  us of a call's launches at 128 / 256 / 512 keys, heads of 128: one row of 5000 keys
            // 21.1 / 21.0 / 24.9, 10000 25.6 / 23.9 / 26.3, 30000 40.5 / 31.1 / 31.2; eight of 2000
            // 25.1 / 24.0 / 26.3; 64 of 300 27.7 / 28.4 / 22.2 (one range); 24 of 2500 48.7 / 41.9 / 37.1.
            const size_t each = (p.parts * (size_t)p.keys + (size_t)cus - 1) / (size_t)cus;
            const size_t want = each <= kPagedMidRange ? std::max<size_t>(each, kPagedLeastRange) : std::max<size_t>(each / 2, kPagedMidRange);
            p.range = (int)std::min<size_t>((want + 63) / 64 * 64, kPagedMaxRange);
        }
        p.ranges = (p.keys + p.range - 1) / p.range;
    }
    p.blocks = ((int64_t)s.n_seqs * (int64_t)s.kv_heads * p.ranges + 7) / 8 * 8 * p.tiles;
    // Room for any call of no more rows in all, however they lie in sequences, and no more keys.  A
    // sequence's v vectors take tiles x width <= v + tiles - 1 <= v + (v - 1) / 16 places; and its ranges,
    // ceil(keys / range), are at most as many as the least range makes, as many as the middle one
    // makes, or those of which a CU has about one.
    const size_t pairs = s.n_seqs * s.rows_per_seq * s.heads, vecs = pairs + pairs / kPagedTile, keys = (size_t)p.keys;
    const size_t pieces = std::min(vecs * ((keys + kPagedLeastRange - 1) / kPagedLeastRange),
                                   vecs * (1 + (keys + kPagedMidRange - 1) / kPagedMidRange) + (size_t)kPagedTile * (size_t)cus);
    Layout l;
    p.off_z = l.take(vecs * keys, 4);
    p.off_e = l.take(vecs * keys, 2);
    p.off_max = l.take(pieces, 4);
    p.off_sum = l.take(pieces, 4);
    p.off_holes = l.take(pieces, 4);
    p.off_out = l.take(pieces * s.head_dim, 4);
    p.bytes = std::max<size_t>(l.used, 256);  // 0 stands for sizes that a call refuses
    return p;
}

// ---- log probabilities ------------------------------------------------------------

constexpr size_t kLogpMaxVocab = (size_t)1 << 20, kLogpMaxRows = 65535, kLogpMaxTokens = 65536, kLogpMaxTop = 32, kLogpMaxLut = 32768;
constexpr int kLogpChunk = 8192, kLogpTile = 256;  // values of a row per block; per maximum that is kept

struct LogpShape {
    size_t rows, vocab, n_tokens, top_n, lut_len;
};

inline const char* logp_refuse(const LogpShape& s) {
    if (s.vocab == 0 || s.vocab > kLogpMaxVocab) return "the vocabulary must hold 1 to 2^20 tokens";
    if (s.rows > kLogpMaxRows || s.n_tokens > kLogpMaxTokens) return "too many rows (65535) or tokens of a row (65536)";
    if (s.top_n > kLogpMaxTop || s.top_n > s.vocab) return "at most 32 alternatives, and as many as the vocabulary holds";
    if (s.lut_len == 0 || s.lut_len > kLogpMaxLut) return "the exp table must hold 1 to 32768 entries";
    return nullptr;
}

// bins: how far below its maximum a logit can lie and have a weight, at four table entries a
// step; words: pairs of 16-bit counters for them.
struct LogpPlan {
    int chunks, tiles;
    uint32_t bins, words;
    size_t off_max, off_tiles, off_counts, bytes;
};

inline LogpPlan logp_plan(const LogpShape& s) {
    LogpPlan p{};
    Layout l;
    p.chunks = (int)((s.vocab + kLogpChunk - 1) / kLogpChunk);
    p.tiles = (int)((s.vocab + kLogpTile - 1) / kLogpTile);
    p.bins = (uint32_t)((s.lut_len + 3) / 4);
    p.words = (p.bins + 1) / 2;
    p.off_max = l.take(s.rows * (size_t)p.chunks, 4);
    p.off_tiles = l.take(s.top_n ? s.rows * (size_t)p.tiles : 0, 4);
    p.off_counts = l.take(s.rows * (size_t)p.chunks * p.words, 4);
    p.bytes = std::max<size_t>(l.used, 256);
    return p;
}

}  // namespace myl
