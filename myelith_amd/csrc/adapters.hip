// adapters.hip -- low-rank adapters of many requests beside a shared W8A16
// projection: myl_linear_w8a16_adapters_dev.  Each step is a reference
// primitive (linear.rs:43-119):
//   u[m] = linear_w8a16(x[m], A[id], a_shifts[id], act_frac, mid_frac)   [rank]
//   d[m] = linear_w8a16(u[m], B[id], b_shifts[id], mid_frac, out_frac)   [N]
//   out[m] = clamp_i16(linear_w8a16(x[m], W, w_shifts, act_frac, out_frac) + d[m])
// with id = ids[m]; a row whose id is outside [0, n_adapters) has d = 0.
//
//   adapters_down_kernel  rows of one adapter together, x A over slices of K: exact i64 sums
//   linear_w8a16          the shared product into out
//   adapters_up_kernel    u from the slices' sums, u B, added to out
//
// Both run on the int8 matrix cores over the byte planes x = 256 hi + lo' + 128
// (gemm_mfma.h), the sums of the weights from a third product with a vector of ones.
// The shared product takes most of the time: 61 rows, N 3584, K 18944, rank 64, 32 adapters:
// x A 13.8 us, W x 36, u B 7.8; 2003 rows, N 18944, K 3584, rank 16: 14, 321, 54.
#include "abi_internal.h"
#include "gemm_dispatch.h"
#include "qk_planes.h"
#include "serve_plan.h"

#include <algorithm>
#include <string>

namespace myl {
namespace {

// The rows of one adapter among a window's: up to 64 of them for the kernel that adds u B.
struct TileRows {
    int32_t id, rows;  // rows 0: nothing to do
    uint8_t at[64];    // places in the window
};
static_assert(sizeof(TileRows) == kAdapterTileBytes);

struct Adapters {
    const int16_t* x;
    const int32_t* ids;
    const int8_t *A, *B;
    const uint8_t *a_shifts, *b_shifts, *out_frac_pc;
    int16_t* out;
    int64_t* part;    // [split][M][rank_pad]
    TileRows* tiles;  // [window][up_tiles]
    uint64_t* acc;    // cleared for the shared product
    size_t acc_elems, ldx, ldo, b_bytes;
    int M, N, K, rank, rank_pad, n, splits, per_wave, units, n_chunk, tile_count;
    SmallDiv down_tiles, up_tiles;
    uint8_t act_frac, mid_frac, out_frac;
};

// Rows of A, B and x start anywhere.
typedef uint32_t Bytes16 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t Halves8 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t Halves2 __attribute__((aligned(2)));

__device__ inline v4i32_t operand(const Bytes16& v) { return v4i32_t{(int)v[0], (int)v[1], (int)v[2], (int)v[3]}; }
// 16 int16 as their byte planes.
__device__ inline void planes16(const Halves8 (&x)[2], v4i32_t& h, v4i32_t& l) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = x[i >> 1][2 * (i & 1)], b = x[i >> 1][2 * (i & 1) + 1];
        h[i] = (int)__builtin_amdgcn_perm(b, a, 0x07050301u);
        l[i] = (int)(__builtin_amdgcn_perm(b, a, 0x06040200u) ^ 0x80808080u);
    }
}
__device__ inline v4i32_t mfma(const v4i32_t& a, const v4i32_t& b, const v4i32_t& c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// ---- tiles of rows ---------------------------------------------------------------

struct Grouping {
    alignas(16) int32_t id[kAdapterWindow];
    uint64_t leads[4], leads64[4];
    int32_t tile_id, first, up, rows[4];
    uint8_t at[16];
};

// Tile t of window w: a row's number among its adapter's rows in the window is a count of
// equal ids before it, every 16th of them leads a tile, and tiles are numbered in the order
// of the rows that lead them.  Each block works its tile out: a launch to sort the rows
// first would take longer than the at most 256 compares of a thread.  Returns the tile's
// rows (0: no such tile), their places in s.at and its adapter in s.tile_id; `up`, if not
// null, are the window's tiles of 64 rows, to be written: each by the block whose tile's first
// row leads it, those that stay empty by the blocks of their number.
__device__ inline int group_rows(const Adapters& a, int w, int t, Grouping& s, TileRows* up) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rows = min(kAdapterWindow, a.M - w * kAdapterWindow);
    int id = tid < rows ? a.ids[(size_t)w * kAdapterWindow + tid] : -1;
    if ((uint32_t)id >= (uint32_t)a.n) id = -1;
    s.id[tid] = id;
    if (tid == 0) s.tile_id = -1;
    __syncthreads();
    int c = 0;
    if (64 * wave < rows) {
#pragma unroll 8
        for (int i = 0; i < 64 * wave; i += 4) {
            const int4 q = *reinterpret_cast<const int4*>(&s.id[i]);
            c += (q.x == id) + (q.y == id) + (q.z == id) + (q.w == id);
        }
        for (int i0 = 0; i0 < min(64, rows - 64 * wave); i0 += 16)
#pragma unroll
            for (int i = 0; i < 16; ++i) c += __builtin_amdgcn_readlane(id, i0 + i) == id && i0 + i < lane;
    }
    const bool lead = id >= 0 && (c & 15) == 0;
    const uint64_t b = __ballot(lead), b64 = __ballot(lead && (c & 63) == 0), below = (1ull << lane) - 1ull;
    if (lane == 0) {
        s.leads[wave] = b;
        s.leads64[wave] = b64;
    }
    __syncthreads();
    int mine = __popcll(b & below), mine64 = __popcll(b64 & below);
    for (int v = 0; v < wave; ++v) {
        mine += __popcll(s.leads[v]);
        mine64 += __popcll(s.leads64[v]);
    }
    if (lead && mine == t) {
        s.tile_id = id;
        s.first = c;
        s.up = (c & 63) == 0 ? mine64 : -1;
    }
    if (up && tid == 0 && t < (int)a.up_tiles.d &&
        t >= __popcll(s.leads64[0]) + __popcll(s.leads64[1]) + __popcll(s.leads64[2]) + __popcll(s.leads64[3]))
        up[t].rows = 0;
    __syncthreads();
    const int tile_id = s.tile_id, first = s.first;
    if (tile_id < 0) return 0;
    TileRows* full = up && s.up >= 0 ? up + s.up : nullptr;
    const bool member = id == tile_id && c >= first;
    if (member && c < first + 16) s.at[c - first] = (uint8_t)tid;
    if (full && member && c < first + 64) full->at[c - first] = (uint8_t)tid;
    const uint64_t m = __ballot(member);
    if (lane == 0) s.rows[wave] = __popcll(m);
    __syncthreads();
    const int all = s.rows[0] + s.rows[1] + s.rows[2] + s.rows[3];
    if (full && tid == 0) {
        full->id = tile_id;
        full->rows = min(all, 64);
    }
    return min(all, 16);
}

// ---- x A --------------------------------------------------------------------------

// Grid (windows x down_tiles, rank groups, splits of K); 256 threads.  Lane l holds row l % 16 of
// A and of x at 16 (l / 16) of each 64 of K: two matrix steps use up a line of A.  A wave
// loads the next unit while it multiplies one.  Bound by reading A: 38.8 MB in 13.8 us (61 rows,
// rank 64, 32 adapters, K 18944; 2.8 TB/s with the latency of ids, grouping and first loads).
// A wave per (row, rank) read A once per row: 91 us.
template <int RT>
__global__ __launch_bounds__(256, 2) void adapters_down_kernel(Adapters a) {
    __shared__ Grouping s;
    __shared__ int64_t red[4][RT][4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const size_t block = ((size_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
    for (size_t i = block * 256 + tid; i < a.acc_elems; i += (size_t)gridDim.x * gridDim.y * gridDim.z * 256) a.acc[i] = 0;
    int t;
    const int w = divmod(a.down_tiles, (int)blockIdx.x, t);
    const int rows = group_rows(a, w, t, s, blockIdx.y == 0 && blockIdx.z == 0 ? a.tiles + (size_t)w * a.up_tiles.d : nullptr);
    if (rows == 0) return;
    const int col = lane & 15, kq = lane >> 4;
    const size_t row = (size_t)w * kAdapterWindow + s.at[min(col, rows - 1)];
    const int16_t* x = a.x + row * a.ldx + 16 * kq;
    const int8_t* A[RT];
    const int j0 = 16 * RT * (int)blockIdx.y;
#pragma unroll
    for (int r = 0; r < RT; ++r)
        A[r] = a.A + ((size_t)s.tile_id * (size_t)a.rank + (size_t)min(j0 + 16 * r + col, a.rank - 1)) * (size_t)a.K + 16 * kq;

    struct Unit {
        Halves8 x[2][2];
        Bytes16 a[2][RT];
    };
    const v4i32_t one = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
    v4i32_t hi[RT], lo[RT], ones[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) hi[r] = lo[r] = ones[r] = v4i32_t{0, 0, 0, 0};
    auto load = [&](Unit& v, int u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const size_t k = (size_t)u * kAdapterUnit + 64 * h;
#pragma unroll
            for (int r = 0; r < RT; ++r) v.a[h][r] = *reinterpret_cast<const Bytes16*>(A[r] + k);
            v.x[h][0] = *reinterpret_cast<const Halves8*>(x + k);
            v.x[h][1] = *reinterpret_cast<const Halves8*>(x + k + 8);
        }
    };
    auto multiply = [&](const Unit& v) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v4i32_t xh, xl;
            planes16(v.x[h], xh, xl);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const v4i32_t w8 = operand(v.a[h][r]);
                hi[r] = mfma(w8, xh, hi[r]);
                lo[r] = mfma(w8, xl, lo[r]);
                ones[r] = mfma(w8, one, ones[r]);
            }
        }
    };
    const int64_t first = ((int64_t)blockIdx.z * 4 + wave) * a.per_wave;
    const int u0 = (int)min(first, (int64_t)a.units), u1 = (int)min(first + a.per_wave, (int64_t)a.units);
    const int whole = min(u1, a.K / kAdapterUnit);
    if (u0 < whole) {
        Unit v, next;
        load(v, u0);
        int u = u0;
        for (; u + 2 <= whole; u += 2) {
            load(next, u + 1);
            multiply(v);
            load(v, min(u + 2, whole - 1));
            multiply(next);
        }
        if (u < whole) multiply(v);
    }
    if (u0 < u1 && whole < u1) {  // the end of K: zero weights past it
        Unit v;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = whole * kAdapterUnit + 64 * h, left = a.K - k - 16 * kq;
#pragma unroll
            for (int r = 0; r < RT; ++r) v.a[h][r] = Bytes16{0, 0, 0, 0};
            v.x[h][0] = v.x[h][1] = Halves8{0, 0, 0, 0};
            if (left >= 16) {
#pragma unroll
                for (int r = 0; r < RT; ++r) v.a[h][r] = *reinterpret_cast<const Bytes16*>(A[r] + k);
                v.x[h][0] = *reinterpret_cast<const Halves8*>(x + k);
                v.x[h][1] = *reinterpret_cast<const Halves8*>(x + k + 8);
            } else {
#pragma unroll
                for (int e = 0; e < 15; ++e)
                    if (e < left) {
#pragma unroll
                        for (int r = 0; r < RT; ++r) v.a[h][r][e >> 2] |= (uint32_t)(uint8_t)A[r][k + e] << (8 * (e & 3));
                        v.x[h][e >> 3][(e & 7) >> 1] |= (uint32_t)(uint16_t)x[k + e] << (16 * (e & 1));
                    }
            }
        }
        multiply(v);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[wave][r][e][lane] = (int64_t)hi[r][e] * 256 + (int64_t)lo[r][e] + (int64_t)ones[r][e] * 128;
    __syncthreads();
    // lane l: row l % 16 of the tile, rank rows 4 (l / 16) .. + 3
    for (int r = wave; r < RT; r += 4) {
        const int j = j0 + 16 * r + 4 * kq;
        if (col >= rows || j >= a.rank_pad) continue;
        int64_t* p = a.part + ((size_t)blockIdx.z * (size_t)a.M + row) * (size_t)a.rank_pad + j;
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = red[0][r][e][lane] + red[1][r][e][lane] + red[2][r][e][lane] + red[3][r][e][lane];
    }
}

// ---- u B --------------------------------------------------------------------------

// The 16 bytes from p on, those at `end` and behind it zero.
__device__ inline v4i32_t bytes_until(const int8_t* p, const int8_t* end) {
    uint64_t v[2] = {0, 0};
#pragma nounroll
    for (int e = 0; e < 8; ++e) {
        if (p + e < end) v[0] |= (uint64_t)(uint8_t)p[e] << (8 * e);
        if (p + e + 8 < end) v[1] |= (uint64_t)(uint8_t)p[e + 8] << (8 * e);
    }
    return v4i32_t{(int)v[0], (int)(v[0] >> 32), (int)v[1], (int)(v[1] >> 32)};
}

// 64 columns of B as the rows of four matrix operands, and the shifts of the two columns
// (n0 + 2 (l % 32) and the next) whose outputs the lane adds to.
template <int KB>
struct Columns {
    v4i32_t w8[4][KB];
    uint8_t frac[2], to[2];
};

constexpr uint32_t kUpGrid = 32768;  // tiles in the second dimension of the grid
typedef short Short2 __attribute__((ext_vector_type(2)));

// Grid (chunks of columns, tiles, 32768s of tiles); 256 threads, KB steps of 64 of the rank.
// Chunks are the first dimension: tiles that stay empty do not leave an XCD idle.  The
// rows' u lie in LDS as byte planes, zero from the rank on.  A wave works on 16 rows and 64
// columns at a time: the products go through LDS, so that a load or store of out takes two
// whole lines and a lane has two columns' shifts.  It loads the next columns and the next
// rows' outputs before it multiplies.  Bound by reading and writing out: 152 MB in 55 us (2003
// rows by 18944, rank 16; 2.8 TB/s).  Outputs straight from the products' registers (16 rows
// of 64 bytes a load) took 62 us, a thread per output 612.
template <int KB>
__global__ __launch_bounds__(256, KB == 1 ? 3 : KB == 2 ? 2 : 1) void adapters_up_kernel(Adapters a) {
    constexpr int stride = 64 * KB + 16;
    __shared__ __align__(16) int8_t plane[2][64 * stride];
    __shared__ __align__(16) int32_t product[4][16 * 68];
    __shared__ size_t place[64];
    const int tile_index = (int)(blockIdx.z * kUpGrid + blockIdx.y);
    if (tile_index >= a.tile_count) return;
    const TileRows* tile = a.tiles + tile_index;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, kq = lane >> 4;
    const int pair = 2 * (lane & 31), odd = lane >> 5;  // its columns; its rows are odd, odd + 2, ..
    const int at0 = tile->at[lane];
    const int rows = __builtin_amdgcn_readfirstlane(tile->rows), id = __builtin_amdgcn_readfirstlane(tile->id);
    if (rows == 0) return;
    const int begin = (int)blockIdx.x * a.n_chunk, end = min(a.N, begin + a.n_chunk), subs = (rows + 15) >> 4;
    const int8_t *B = a.B + (size_t)id * (size_t)a.N * (size_t)a.rank, *b_end = a.B + a.b_bytes;
    const uint8_t* bs = a.b_shifts + (size_t)id * (size_t)a.N;
    int t;
    const size_t base = (size_t)divmod(a.up_tiles, tile_index, t) * kAdapterWindow;

    auto fetch = [&](Columns<KB>& c, int n0) {
        const int8_t* b = B + (size_t)n0 * (size_t)a.rank;
        if (n0 + 64 <= a.N && b + 63 * a.rank + 64 * KB <= b_end) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int k = 0; k < KB; ++k)
                    c.w8[q][k] = operand(*reinterpret_cast<const Bytes16*>(b + (uint32_t)((16 * q + col) * a.rank + 16 * kq) + 64 * k));
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int k = 0; k < KB; ++k) c.w8[q][k] = bytes_until(b + min(16 * q + col, a.N - 1 - n0) * a.rank + 16 * kq + 64 * k, b_end);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int n = min(n0 + pair + i, a.N - 1);
            c.frac[i] = bs[n];
            c.to[i] = a.out_frac_pc ? a.out_frac_pc[n] : a.out_frac;
        }
    };
    Columns<KB> cur, next;
    uint32_t old[8] = {}, ahead[8] = {};  // out at the lane's rows and columns, of these 16 rows and the next
    auto outputs = [&](uint32_t (&o)[8], auto&& place_of, int n0) {
        if (n0 + 64 <= a.N)
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = *reinterpret_cast<const Halves2*>(a.out + place_of(2 * i + odd) + n0 + pair);
    };
    int n0 = begin + 64 * wave;
    if (n0 < end) {
        fetch(cur, n0);
        outputs(old, [&](int r) { return (base + (size_t)__shfl(at0, min(r, rows - 1), 64)) * a.ldo; }, n0);
    }

    const int place0 = __shfl(at0, min(lane, rows - 1), 64);
    if (tid < 64) place[tid] = (base + (size_t)place0) * a.ldo;
    const int quads = __builtin_ctz((unsigned)a.rank_pad) - 2;  // a row's fours of the rank, as a shift
    for (int i = tid; i < rows << quads; i += 256) {
        const int r = i >> quads, j = 4 * (i & ((1 << quads) - 1));
        const int64_t* p = a.part + (base + (size_t)tile->at[r]) * (size_t)a.rank_pad + j;
        int64_t sum[4] = {0, 0, 0, 0};
#pragma unroll 4
        for (int k = 0; k < a.splits; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += p[(size_t)k * (size_t)a.M * (size_t)a.rank_pad + e];
        uint32_t h = 0, l = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (j + e < a.rank) {
                const uint8_t frac = (uint8_t)(a.a_shifts[(size_t)id * (size_t)a.rank + j + e] + a.act_frac);
                const uint32_t u = (uint16_t)clamp_i16_i64(rescale64(sum[e], frac, a.mid_frac));
                h |= (u >> 8) << (8 * e);
                l |= ((u & 255u) ^ 128u) << (8 * e);
            }
        *reinterpret_cast<uint32_t*>(&plane[0][r * stride + j]) = h;
        *reinterpret_cast<uint32_t*>(&plane[1][r * stride + j]) = l;
    }
    for (int r = tid >> 2, j = a.rank_pad + 16 * (tid & 3); j < 64 * KB; j += 64)
        *reinterpret_cast<v4i32_t*>(&plane[0][r * stride + j]) = *reinterpret_cast<v4i32_t*>(&plane[1][r * stride + j]) = v4i32_t{0, 0, 0, 0};
    __syncthreads();
    v4i32_t one[KB];  // ones below the rank
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int left = min(max(a.rank - 64 * b - 16 * kq - 4 * e, 0), 4);
            one[b][e] = left == 0 ? 0 : 0x01010101 >> (8 * (4 - left));
        }
    while (n0 < end) {
        const int n2 = n0 + 256;
        if (n2 < end) fetch(next, n2);
        uint32_t sh[2], half[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            sh[i] = (uint32_t)(uint8_t)(cur.frac[i] + a.mid_frac - cur.to[i]);
            half[i] = (1u << ((sh[i] - 1u) & 31u)) - 1u;
        }
        // 32-bit steps where the rounding shifts are 1 to 30
        const bool fast = n0 + 64 <= a.N && __all(sh[0] - 1u < 30u && sh[1] - 1u < 30u);
        v4i32_t sums[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            sums[q] = v4i32_t{0, 0, 0, 0};
#pragma unroll
            for (int b = 0; b < KB; ++b) sums[q] = mfma(cur.w8[q][b], one[b], sums[q]);
            sums[q] <<= 7;
        }
#pragma nounroll
        for (int u = 0; u < subs; ++u) {
            const size_t* places = place + 16 * u;
            if (u + 1 < subs) outputs(ahead, [&](int r) { return places[16 + r]; }, n0);
            else if (n2 < end) outputs(ahead, [&](int r) { return place[r]; }, n2);
            v4i32_t hi[4], lo[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                hi[q] = v4i32_t{0, 0, 0, 0};
                lo[q] = sums[q];
            }
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const int i = (16 * u + col) * stride + 64 * b + 16 * kq;
                const v4i32_t uh = *reinterpret_cast<const v4i32_t*>(&plane[0][i]), ul = *reinterpret_cast<const v4i32_t*>(&plane[1][i]);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    hi[q] = mfma(cur.w8[q][b], uh, hi[q]);
                    lo[q] = mfma(cur.w8[q][b], ul, lo[q]);
                }
            }
            int32_t* v = product[wave];  // [16 rows][64 columns], the wave's own
#pragma unroll
            for (int q = 0; q < 4; ++q) *reinterpret_cast<v4i32_t*>(&v[col * 68 + 16 * q + 4 * kq]) = (hi[q] << 8) + lo[q];
            asm volatile("" ::: "memory");
            if (fast) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = 2 * i + odd;
                    const int2 w = *reinterpret_cast<const int2*>(&v[r * 68 + pair]);
                    const int32_t d0 = (int32_t)((uint32_t)w.x + half[0] + (((uint32_t)w.x >> sh[0]) & 1u)) >> sh[0];
                    const int32_t d1 = (int32_t)((uint32_t)w.y + half[1] + (((uint32_t)w.y >> sh[1]) & 1u)) >> sh[1];
                    const Short2 sum = __builtin_elementwise_add_sat(Short2(__builtin_amdgcn_cvt_pk_i16(d0, d1)), __builtin_bit_cast(Short2, old[i]));
                    if (16 * u + r < rows) *reinterpret_cast<Halves2*>(a.out + places[r] + n0 + pair) = __builtin_bit_cast(uint32_t, sum);
                }
            } else {
#pragma nounroll
                for (int r = odd; r < min(16, rows - 16 * u); r += 2)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (n0 + pair + i < a.N) {
                            int16_t* o = a.out + places[r] + n0 + pair + i;
                            *o = clamp_i16((int32_t)*o + (int32_t)clamp_i16_i64(rescale64(v[r * 68 + pair + i], (uint8_t)sh[i], 0)));
                        }
            }
            asm volatile("" ::: "memory");
#pragma unroll
            for (int i = 0; i < 8; ++i) old[i] = ahead[i];
        }
        cur = next;
        n0 = n2;
    }
}

__global__ __launch_bounds__(256) void adapters_clear_kernel(uint64_t* __restrict__ p, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) p[i] = 0;
}

}  // namespace
}  // namespace myl

using namespace myl;

extern "C" {

size_t myl_linear_w8a16_adapters_workspace(const myl_ctx* ctx, size_t M, size_t N, size_t K, size_t rank, size_t n_adapters) {
    const AdapterShape s{M, N, K, rank, n_adapters};
    if (!ctx || adapter_refuse(s)) return 0;
    return adapter_plan(s, ctx->prop.multiProcessorCount).bytes;
}

int myl_linear_w8a16_adapters_dev(myl_ctx* ctx, const int16_t* x, size_t M, size_t ldx, const int8_t* W, size_t N,
                                  size_t K, const uint8_t* w_shifts, uint8_t act_frac, uint8_t out_frac,
                                  const uint8_t* out_frac_pc, const int32_t* ids, const int8_t* A,
                                  const uint8_t* a_shifts, uint8_t mid_frac, const int8_t* B, const uint8_t* b_shifts,
                                  size_t n_adapters, size_t rank, int16_t* out, size_t ldo, void* workspace,
                                  size_t workspace_bytes) {
    if (!ctx) return MYL_E_INVALID;
    const char* what = "linear_w8a16_adapters_dev";
    auto bad = [&](const char* why) { return ctx->fail(MYL_E_INVALID, std::string(what) + ": " + why); };
    const AdapterShape s{M, N, K, rank, n_adapters};
    if (const char* why = adapter_refuse(s)) return bad(why);
    if (ldx < K || ldo < N) return bad("leading dimension too small");
    if (!fits_int(ldx) || !fits_int(ldo)) return bad("leading dimension too large");
    if (M == 0 || N == 0) return MYL_OK;
    if (!x || !W || !w_shifts || !out) return bad("null operand");
    if (n_adapters > 0 && (!ids || !A || !a_shifts || !B || !b_shifts)) return bad("null adapter operand");
    const AdapterPlan p = adapter_plan(s, ctx->prop.multiProcessorCount);
    if (!workspace || workspace_bytes < p.bytes) return bad("workspace too small (myl_linear_w8a16_adapters_workspace)");
    if ((uintptr_t)workspace & 15) return bad("workspace must be 16-byte aligned");
    const DeviceGuard guard(ctx->device);
    const hipStream_t st = ctx->stream;
    char* ws = static_cast<char*>(workspace);
    MmCtx mm;
    mm.cus = std::max(ctx->prop.multiProcessorCount, 1);
    if (M >= 2) {
        mm.planes = reinterpret_cast<int8_t*>(ws + p.off_planes);
        mm.planes_bytes = p.planes_bytes;
        mm.acc = reinterpret_cast<unsigned long long*>(ws + p.off_acc);
        mm.acc_elems = p.acc_elems;
    }
    Adapters a{};
    a.acc = reinterpret_cast<uint64_t*>(mm.acc);
    a.acc_elems = p.acc_elems;
    if (n_adapters > 0) {
        a.x = x; a.ids = ids; a.A = A; a.B = B; a.a_shifts = a_shifts; a.b_shifts = b_shifts; a.out_frac_pc = out_frac_pc;
        a.out = out;
        a.part = reinterpret_cast<int64_t*>(ws + p.off_part);
        a.tiles = reinterpret_cast<TileRows*>(ws + p.off_tiles);
        a.ldx = ldx; a.ldo = ldo; a.b_bytes = n_adapters * N * rank;
        a.M = (int)M; a.N = (int)N; a.K = (int)K; a.rank = (int)rank; a.rank_pad = p.rank_pad; a.n = (int)n_adapters;
        a.splits = p.splits; a.per_wave = p.per_wave; a.units = (int)((K + kAdapterUnit - 1) / kAdapterUnit); a.n_chunk = p.n_chunk;
        a.down_tiles = SmallDiv::of((size_t)p.down_tiles);
        a.up_tiles = SmallDiv::of((size_t)p.up_tiles);
        a.tile_count = p.windows * p.up_tiles;
        a.act_frac = act_frac; a.mid_frac = mid_frac; a.out_frac = out_frac;
        const dim3 grid((unsigned)(p.windows * p.down_tiles), (unsigned)p.rank_groups, (unsigned)p.splits);
        if (p.rank_tiles == 1) adapters_down_kernel<1><<<grid, 256, 0, st>>>(a);
        else if (p.rank_tiles == 2) adapters_down_kernel<2><<<grid, 256, 0, st>>>(a);
        else adapters_down_kernel<4><<<grid, 256, 0, st>>>(a);
    } else if (p.acc_elems) {
        adapters_clear_kernel<<<(unsigned)std::min<size_t>((p.acc_elems + 255) / 256, 1024), 256, 0, st>>>(a.acc, a.acc_elems);
    }
    if (int rc = ctx->hip(hipGetLastError(), what)) return rc;
    int rc = ctx->hip(linear_w8a16(x, (int)M, (int)ldx, W, (int)N, (int)K, w_shifts, act_frac, out_frac, out_frac_pc, out,
                                   (int)ldo, st, &mm), what);
    if (rc || n_adapters == 0) return rc;
    const unsigned tiles = (unsigned)a.tile_count;
    const dim3 grid((unsigned)p.n_chunks, std::min(tiles, kUpGrid), (tiles + kUpGrid - 1) / kUpGrid);
    if (p.rank_pad <= 64) adapters_up_kernel<1><<<grid, 256, 0, st>>>(a);
    else if (p.rank_pad == 128) adapters_up_kernel<2><<<grid, 256, 0, st>>>(a);
    else adapters_up_kernel<4><<<grid, 256, 0, st>>>(a);
    return ctx->hip(hipGetLastError(), what);
}

}  // extern "C"
