// adapters.hip -- low-rank adapters of many requests beside a shared projection:
// output[t] = base[t] + scale[a] * B[a] (A[a] x[t]), a = ids[t].
//
// 4 * rank operations for each number of x and output: memory's work (x, base and output once,
// A and B of the adapters that occur), and for few tokens the launches'.  A window of 64 tokens
// is sorted by adapter inside each block, so no list of tokens is made first, and a captured
// launch follows its ids.  Both products are matrix products of 16 tokens of one adapter; what
// of the 16 is not filled costs nothing that these kernels are bound by.
#include "common.hpp"
#include "paged.hpp"
#include "spbitnet_amd.h"

#include <type_traits>

namespace spb {
namespace {

constexpr int kMaxSections = SPB_MAX_SECTIONS;
constexpr int kMaxRank = 256;
constexpr int kMaxSize = 1 << 20;  // tokens, rows and columns: indices and grids in 32 bits
constexpr int kWindow = kWave;     // tokens of a block: a lane looks at each one's id
constexpr int kTile = 16;          // rows and columns of a matrix product
constexpr int kStep = 32;          // and its depth

struct Args {
    const uint16_t* a;
    const uint16_t* b;
    const float* scales;
    const int* ranks;
    const int* ids;
    const uint16_t* x;
    const uint16_t* base;
    uint16_t* out;
    float* h;  // [splits][tokens][sections * rank]
    long a_adapter, a_row, b_adapter, b_row, xs, bs, os;
    int num, rank, cols, sections, tokens, rows;
    int id_bits;     // ids are below 2^id_bits
    int split_bits;  // 2^split_bits blocks split the columns of the inner products
    int end[kMaxSections];  // first row behind each section
    bool wide;              // base and output by 16 bytes
};

using Acc = float __attribute__((ext_vector_type(4)));

// Products of 16 x 32 by 32 x 16: lane l holds 8 numbers of row (column) l % 16 from
// depth l / 16 * 8 on; of the result rows l / 16 * 4 + 0 ... 3 of column l % 16.
template <class T>
struct Matrix;
template <>
struct Matrix<F16> {
    using V = _Float16 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ Acc mac(uint4 a, uint4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, a),
                                                      __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
};
template <>
struct Matrix<BF16> {
    using V = __bf16 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ Acc mac(uint4 a, uint4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, a),
                                                       __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
};

__device__ __forceinline__ int rank_of(const Args& g, int a) {
    return g.ranks ? min(max(g.ranks[a], 0), g.rank) : g.rank;
}

// 16 bytes, or zeros: what must not count is not read, so that a NaN there stays out of the
// products.
__device__ __forceinline__ uint4 load8(const uint16_t* p, bool valid) {
    uint4 v = {0, 0, 0, 0};
    if (valid) v = *reinterpret_cast<const uint4*>(p);
    return v;
}

__device__ __forceinline__ uint4 zero_unless(bool in, uint4 v) {
    return {in ? v.x : 0u, in ? v.y : 0u, in ? v.z : 0u, in ? v.w : 0u};
}

// The first n of 8 numbers.
__device__ __forceinline__ uint4 first_of(uint4 v, int n) {
    auto part = [n](uint32_t w, int i) { return n > i + 1 ? w : n > i ? w & 0xffffu : 0u; };
    return {part(v.x, 0), part(v.y, 2), part(v.z, 4), part(v.w, 6)};
}

// Place of the n-th set bit (from 0; there are more than n).
__device__ __forceinline__ int nth_bit(uint64_t m, int n) {
    int at = 0;
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) {
        const int c = __popcll(m & ((uint64_t{1} << w) - 1));
        const bool up = n >= c;
        n -= up ? c : 0;
        at += up ? w : 0;
        m >>= up ? w : 0;
    }
    return at;
}

// An adapter's tokens in a window.
struct Group {
    int adapter, many;
    int listed;  // lane n: the n-th one's place in the window (lanes from `many` on: the first's)
    // The n-th one's token.
    __device__ __forceinline__ long token(int window, int n) const {
        return window * kWindow + __shfl(listed, n, kWave);
    }
};

// A window's adapters: f(group) for the z-th, (z + step)-th, ... of those that occur, in the
// order of their first tokens.  Returns the tokens that have none.  A lane finds the tokens
// of its own adapter bit by bit of the ids; going through the adapters one after the other
// took 5 us of the 20 that 24 adapters' inner products did.
template <class F>
__device__ __forceinline__ uint64_t each_adapter(const Args& g, int window, int z, int step, F f) {
    const int lane = threadIdx.x % kWave, t = window * kWindow + lane;
    const int id = t < g.tokens ? g.ids[t] : -1;
    const bool has = id >= 0 && id < g.num;
    const uint64_t valid = __ballot(has);
    uint64_t same = valid;
    for (int b = 0; b < g.id_bits; ++b) {
        const bool one = id >> b & 1;
        const uint64_t ones = __ballot(one);
        same &= one ? ones : ~ones;
    }
    const uint64_t before = same & ((uint64_t{1} << lane) - 1);
    const uint64_t firsts = __ballot(has && before == 0);
    const int groups = __popcll(firsts);
    for (int i = z; i < groups; i += step) {
        const int first = __builtin_amdgcn_readfirstlane(nth_bit(firsts, i));
        Group q;
        q.adapter = __builtin_amdgcn_readlane(id, first);
        const bool mine = has && id == q.adapter;
        q.many = __popcll(__ballot(mine));
        // each of its lanes to the lane of its place in the group, the others to the last
        const int place = mine ? __popcll(before) : kWave - 1;
        const int got = __builtin_amdgcn_ds_permute(place * 4, lane);
        q.listed = lane < q.many ? got : first;
        f(q);
    }
    return __ballot(t < g.tokens) & ~valid;
}

// output = base in rows [row, end) of the tokens that have no adapter, a wave each.
__device__ __forceinline__ void copy_idle(const Args& g, int window, uint64_t idle, int row, int end,
                                          int wave, int waves) {
    if (g.base == g.out) return;
    const int lane = threadIdx.x % kWave;
    for (int i = 0; idle; ++i, idle &= idle - 1) {
        if (i % waves != wave) continue;
        const long t = window * kWindow + __builtin_ctzll(idle);
        int rest = row;  // rows that do not go by 8
        if (g.wide) {
            rest = row + (end - row) / 8 * 8;
            for (int r = row + lane * 8; r < rest; r += kWave * 8)
                *reinterpret_cast<uint4*>(g.out + t * g.os + r) =
                    *reinterpret_cast<const uint4*>(g.base + t * g.bs + r);
        }
        for (int r = rest + lane; r < end; r += kWave) g.out[t * g.os + r] = g.base[t * g.bs + r];
    }
}

// Inner products of 8 depths of one token as 16-bit numbers, h = (the parts' sum) * unit.  bf16:
// three, each the first 8 bits of what those before it leave, so they are the float32 number; two
// were off by 2^-18, as much as shows where two of them nearly cancel, and took 0.1 us of 7.6
// less (one token) and 0.5 of 59.6 (2049).  fp16: two, which are within 2^-22 of h, or 2^-38 of
// the token's largest where that is more; its range is made up for by a power of two for the token.
template <class T>
struct Parts {
    static constexpr int kMany = std::is_same_v<T, BF16> ? 3 : 2;
    uint4 v[kMany];
    __device__ __forceinline__ void set(const float (&h)[8], float by) {
        uint16_t a[kMany][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (std::is_same_v<T, BF16>) {
                float rest = h[e];
#pragma unroll
                for (int n = 0; n < kMany; ++n) {
                    const uint32_t first = __builtin_bit_cast(uint32_t, rest) & 0xffff0000u;
                    a[n][e] = static_cast<uint16_t>(first >> 16);
                    rest = __builtin_isfinite(h[e]) ? rest - __builtin_bit_cast(float, first) : 0.0f;
                }
            } else {
                const float v = h[e] * by;
                a[0][e] = T::from_float(v);
                const float rest = v - T::to_float(a[0][e]);
                a[1][e] = T::from_float(__builtin_isfinite(v) ? rest : 0.0f);
            }
        }
        auto two = [](uint16_t x, uint16_t y) { return static_cast<uint32_t>(y) << 16 | x; };
#pragma unroll
        for (int n = 0; n < kMany; ++n)
            v[n] = {two(a[n][0], a[n][1]), two(a[n][2], a[n][3]), two(a[n][4], a[n][5]), two(a[n][6], a[n][7])};
    }
};

// The larger of `most` and a finite h: beside an infinite one the others must stay finite too.
__device__ __forceinline__ float larger(float most, float h) {
    const float size = __builtin_fabsf(h);
    return size < __builtin_inff() ? __builtin_fmaxf(most, size) : most;
}

// The power of two that brings a token's inner products, at most `most`, below 2^14.
template <class T>
__device__ __forceinline__ int shift_of(float most) {
    if constexpr (std::is_same_v<T, BF16>) return 0;
    if (!(most > 0.0f)) return 0;
    const int exponent = static_cast<int>(__builtin_bit_cast(uint32_t, most) >> 23 & 255) - 126;
    return min(14 - exponent, 100);
}

// -- few tokens: both products in one launch.  A block has 128 rows of the output and an
// -- adapter's tokens of a window, and makes the inner products that it needs by itself: its
// -- 8 waves split the columns and add up in LDS.  One token, rank 16 on q|k|v of 2560 columns:
// -- 6.9 us of the kernel, 7.6 a call, for 0.4 MB: bound by dependent steps (ids, A and x, B)
// -- and the fetch of the code.

constexpr int kFusedWaves = 8, kFusedRows = kFusedWaves * kTile;
constexpr int kFusedRank = 64;                 // most ranks
constexpr int kFusedPad = kFusedRank + 4;      // numbers of a token in LDS

template <class T>
__global__ __launch_bounds__(kFusedWaves* kWave, 4) void fused_kernel(Args g) {
    __shared__ float part[kFusedWaves][kTile][kFusedPad];
    __shared__ float total[kTile][kFusedPad];
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int col = lane % kTile, quad = lane / kTile;
    int sec = 0, tile = blockIdx.x, row0 = 0;
    for (;; ++sec) {  // tiles do not cross sections
        row0 = sec ? g.end[sec - 1] : 0;
        const int tiles = (g.end[sec] - row0 + kFusedRows - 1) / kFusedRows;
        if (tile < tiles) break;
        tile -= tiles;
    }
    const int end = g.end[sec];
    row0 += tile * kFusedRows;
    const int window = blockIdx.z, steps = (g.cols + kStep - 1) / kStep;
    const int step0 = steps * wave / kFusedWaves, step1 = steps * (wave + 1) / kFusedWaves;
    const int full1 = min(step1, g.cols / kStep);  // of them whole
    const int brow = row0 + wave * kTile + col;  // of the outer product's left side
    const uint64_t idle = each_adapter(g, window, blockIdx.y, gridDim.y, [&](const Group& q) {
        const int a = q.adapter, r = rank_of(g, a), many = q.many;
        const uint16_t* left = g.a + a * g.a_adapter + static_cast<long>(sec * g.rank) * g.a_row;
        const float scale = g.scales[a];
        const int last = max(r - 1, 0);
        uint4 up[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int depth = k * kStep + quad * 8;
            up[k] = load8(g.b + a * g.b_adapter + brow * g.b_row + depth, brow < end && depth < r);
            up[k] = first_of(up[k], r - depth);
        }
        for (int first = 0; first < many; first += kTile) {
            const bool live = first + col < many;
            const long t = q.token(window, live ? first + col : first);
            const uint16_t* x = g.x + t * g.xs + quad * 8;
            const int row = row0 + wave * kTile + quad * 4;
            uint16_t old[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                old[e] = live && row + e < end ? g.base[t * g.bs + row + e] : 0;
            Acc acc[kFusedRank / kTile] = {};
            // rows of A from the adapter's rank on give numbers that are not used
            auto inner = [&](auto tiles) {
                constexpr int kTiles = decltype(tiles)::value;
                const uint16_t* w[kTiles];
#pragma unroll
                for (int m = 0; m < kTiles; ++m)
                    w[m] = left + min(m * kTile + col, last) * g.a_row + quad * 8;
                auto steps = [&](auto many, int s) {  // their loads in flight together
                    constexpr int kMany = decltype(many)::value;
                    uint4 v[kMany], q[kMany][kTiles];
#pragma unroll
                    for (int i = 0; i < kMany; ++i) {
                        v[i] = *reinterpret_cast<const uint4*>(x + (s + i) * kStep);
#pragma unroll
                        for (int m = 0; m < kTiles; ++m)
                            q[i][m] = *reinterpret_cast<const uint4*>(w[m] + (s + i) * kStep);
                    }
#pragma unroll
                    for (int i = 0; i < kMany; ++i)
#pragma unroll
                        for (int m = 0; m < kTiles; ++m) acc[m] = Matrix<T>::mac(q[i][m], v[i], acc[m]);
                };
                constexpr int kAhead = kTiles == 1 ? 5 : 4;
                int s = step0;
                for (; s + kAhead <= full1; s += kAhead) steps(std::integral_constant<int, kAhead>(), s);
                for (; s + 2 <= full1; s += 2) steps(std::integral_constant<int, 2>(), s);
                if (s < full1) steps(std::integral_constant<int, 1>(), s);
                if (full1 < step1) {  // columns that end inside a step
                    const bool in = full1 * kStep + quad * 8 < g.cols;
                    const uint4 v = load8(x + full1 * kStep, in);
#pragma unroll
                    for (int m = 0; m < kTiles; ++m)
                        acc[m] = Matrix<T>::mac(load8(w[m] + full1 * kStep, in), v, acc[m]);
                }
            };
            if (r <= kTile)
                inner(std::integral_constant<int, 1>());
            else if (r <= 2 * kTile)
                inner(std::integral_constant<int, 2>());
            else
                inner(std::integral_constant<int, 4>());
            const int tiles = (r + kTile - 1) / kTile;
#pragma unroll
            for (int m = 0; m < kFusedRank / kTile; ++m)
                if (m < tiles)
                    *reinterpret_cast<Acc*>(&part[wave][col][m * kTile + quad * 4]) = acc[m];
            __syncthreads();
            for (int i = tid; i < kTile * tiles * kTile; i += kFusedWaves * kWave) {
                const int c = i / (tiles * kTile), j = i % (tiles * kTile);
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < kFusedWaves; ++w) s += part[w][c][j];
                total[c][j] = s;
            }
            __syncthreads();
            float h[2][8], most = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int j = k * kStep + quad * 8 + e;
                    h[k][e] = j < r ? total[col][j] : 0.0f;
                    most = larger(most, h[k][e]);
                }
            most = __builtin_fmaxf(most, __shfl_xor(most, 16, kWave));
            most = __builtin_fmaxf(most, __shfl_xor(most, 32, kWave));
            const int shift = shift_of<T>(most);
            const float by = __builtin_ldexpf(1.0f, shift);
            Acc sum = {};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (k * kStep >= r) break;
                Parts<T> p;
                p.set(h[k], by);
#pragma unroll
                for (int n = 0; n < Parts<T>::kMany; ++n) sum = Matrix<T>::mac(up[k], p.v[n], sum);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (live && row + e < end)
                    g.out[t * g.os + row + e] = T::from_float(
                        T::to_float(old[e]) + __builtin_ldexpf(scale * sum[e], -shift));
        }
    });
    if (blockIdx.y == 0)
        copy_idle(g, window, idle, row0, min(row0 + kFusedRows, end), wave, kFusedWaves);
}

// -- many tokens or ranks: the inner products first, into memory, then the outer ones.

constexpr int kWaves = 4;
constexpr int kPart = 64;           // ranks of a block of the first, of a pass of the second
constexpr int kPad = kPart + 4;     // float32 of a token in LDS
constexpr int kRows = kWaves * 64;  // rows of a block of the second

// h of 16 of an adapter's tokens of a window and 64 rows of A: g.split_bits blocks and their
// waves split the columns, the waves add up in LDS.  Most of a block's time is fetching its
// code, which a launch finds in no cache of its CU: one loop, two bodies.  kDeep products'
// loads are in flight together: 2 where windows are few, and the code's fetch counts (32
// tokens of up to 20 adapters, rank 16, q|k|v of 2560: 5.3 us, with 5 6.5), 5 else (2049 tokens,
// rank 32: 14.4 us, with 2 18.0, with x (10 MB) and A (1.6 MB) in the last cache; 16.7 without).
template <class T, int kDeep>
__global__ __launch_bounds__(kWaves* kWave) void shrink_kernel(Args g) {
    __shared__ float part[kWaves][kTile][kPad];
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int col = lane % kTile, quad = lane / kTile, all = g.sections * g.rank;
    const int window = blockIdx.x, split = blockIdx.z & ((1 << g.split_bits) - 1);
    const int first = (blockIdx.z >> g.split_bits & 3) * kTile;  // of the adapter's tokens
    const int j0 = (blockIdx.z >> g.split_bits >> 2) * kPart;
    each_adapter(g, window, blockIdx.y, gridDim.y, [&](const Group& q) {
        if (first >= q.many) return;
        const int r = rank_of(g, q.adapter);
        int of_section = j0 + lane;  // the row's number in its section
        while (of_section >= g.rank) of_section -= g.rank;
        const uint64_t live = __ballot(j0 + lane < all && of_section < r);
        const int ranks = live ? kWave - __builtin_clzll(live) : 0;
        const int steps = (g.cols + kStep - 1) / kStep, way = split * kWaves + wave;
        const int bits = g.split_bits + 2, step0 = steps * way >> bits, step1 = steps * (way + 1) >> bits;
        const uint16_t* x = g.x + q.token(window, first + col < q.many ? first + col : first) * g.xs;
        const uint16_t* a = g.a + q.adapter * g.a_adapter + j0 * g.a_row;
        Acc acc[4] = {};
        auto inner = [&](auto tiles) {
            constexpr int kM = decltype(tiles)::value, kAhead = kM == 1 ? 4 : kDeep;
            const uint16_t* row[kM];
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                // the others' rows are a live one's: what they give is not used
                const int n = m * kTile + col;
                row[m] = a + (live >> n & 1 ? n : __builtin_ctzll(live)) * g.a_row;
            }
            for (int s = step0; s < step1; s += kAhead) {  // kAhead steps' loads in flight together
                uint4 v[kAhead], w[kAhead][kM];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int depth = (s + i) * kStep + quad * 8;
                    const bool in = s + i < step1 && depth < g.cols;
                    v[i] = zero_unless(in, *reinterpret_cast<const uint4*>(x + (in ? depth : 0)));
#pragma unroll
                    for (int m = 0; m < kM; ++m)
                        w[i][m] = zero_unless(in, *reinterpret_cast<const uint4*>(row[m] + (in ? depth : 0)));
                }
#pragma unroll
                for (int i = 0; i < kAhead; ++i)
#pragma unroll
                    for (int m = 0; m < kM; ++m) acc[m] = Matrix<T>::mac(w[i][m], v[i], acc[m]);
            }
        };
        if (ranks > kTile)
            inner(std::integral_constant<int, 4>());
        else if (ranks > 0)
            inner(std::integral_constant<int, 1>());
        __syncthreads();  // the last group's sums are read
#pragma unroll
        for (int m = 0; m < 4; ++m) *reinterpret_cast<Acc*>(&part[wave][col][m * kTile + quad * 4]) = acc[m];
        __syncthreads();
        const int n = tid / 16, j = tid % 16 * 4;  // 4 ranks of a token
        Acc sum = {};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += *reinterpret_cast<const Acc*>(&part[w][n][j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = live >> (j + e) & 1 ? sum[e] : 0.0f;
        const long t = q.token(window, first + n);
        if (first + n < q.many && j0 + j < all)
            *reinterpret_cast<Acc*>(g.h + (static_cast<long>(split) * g.tokens + t) * all + j0 + j) = sum;
    });
}

// 256 rows of an adapter's tokens of a window, 64 rows a wave.  Left rows are dealt to the
// products so that a lane's results of two are 8 neighbours, and with its three neighbours'
// 64 bytes of a token's output.  The adapter's part of B stays in registers, up to 64 ranks;
// more go in passes for every 16 tokens.  2049 tokens, rank 32 on gate|up of 6912 rows each:
// 44.5 us for 113 MB of base and output and the 4 parts of the inner products, 2.5 TB/s, or 35.0
// with all of it in the last cache; up to 20 adapters over 32 tokens, rank 16 on q|k|v: 7.3 us,
// bound as the kernel above.
template <class T, bool kPasses>
__global__ __launch_bounds__(kWaves* kWave) void expand_kernel(Args g) {
    constexpr int kHeld = kPasses ? 32 : kWindow;  // tokens in LDS
    constexpr int kWidth = kPasses ? kMaxRank + 8 : kPart + 8;
    constexpr int kMany = Parts<T>::kMany;
    __shared__ uint16_t inner[kMany][kHeld][kWidth];
    __shared__ int shifts[kHeld];
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int col = lane % kTile, quad = lane / kTile, all = g.sections * g.rank;
    int sec = 0, tile = blockIdx.x, row0 = 0;
    for (;; ++sec) {
        row0 = sec ? g.end[sec - 1] : 0;
        const int tiles = (g.end[sec] - row0 + kRows - 1) / kRows;
        if (tile < tiles) break;
        tile -= tiles;
    }
    const int end = g.end[sec], window = blockIdx.z;
    row0 += tile * kRows;
    const int mine = row0 + wave * 64 + quad * 8;  // a lane's rows: 8 from here on, and 8 from 32 on
    const bool whole = g.wide && mine + 40 <= end;
    const uint64_t idle = each_adapter(g, window, blockIdx.y, gridDim.y, [&](const Group& q) {
        const int r = rank_of(g, q.adapter);
        const float scale = g.scales[q.adapter];
        uint4 up[2][4];
        auto load_up = [&](int first) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int depth = first + k * kStep + quad * 8;
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const int row = row0 + wave * 64 + m / 2 * 32 + col / 4 * 8 + m % 2 * 4 + col % 4;
                    const bool in = row < end && depth < r;
                    up[k][m] = *reinterpret_cast<const uint4*>(g.b + q.adapter * g.b_adapter +
                                                               (in ? row * g.b_row + depth : row0 * g.b_row));
                    up[k][m] = first_of(up[k][m], in ? r - depth : 0);
                }
            }
        };
        if (!kPasses) load_up(0);
        for (int held = 0; held < q.many; held += kHeld) {
            uint4 old[2];
            auto load_old = [&](int slot) {
                const long t = q.token(window, slot < q.many ? slot : held);
                if (!whole) return;
                old[0] = *reinterpret_cast<const uint4*>(g.base + t * g.bs + mine);
                old[1] = *reinterpret_cast<const uint4*>(g.base + t * g.bs + mine + 32);
            };
            load_old(held + col);
            // inner products, 8 threads a token in passes and 4 else, 16 ranks at a time
            constexpr int kThreads = kWaves * kWave / kHeld;
            const int slot = tid / kThreads;
            const bool has = held + slot < q.many;
            const float* from = g.h + q.token(window, has ? held + slot : held) * all + sec * g.rank;
            constexpr int kTurns = (kPasses ? kMaxRank : kPart) / (kThreads * 8);
            float h[kTurns][8], most = 0.0f;
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
                const int k = (i * kThreads + tid % kThreads) * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) h[i][e] = 0.0f;
                if (!has || k >= r) continue;  // ranks are stored by 8, zeros behind the adapter's
                for (int s = 0; s < 1 << g.split_bits; ++s) {
                    const float* p = from + static_cast<long>(s) * g.tokens * all + k;
                    const Acc u = *reinterpret_cast<const Acc*>(p), v = *reinterpret_cast<const Acc*>(p + 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        h[i][e] += u[e];
                        h[i][4 + e] += v[e];
                    }
                }
                if (std::is_same_v<T, F16>)
#pragma unroll
                    for (int e = 0; e < 8; ++e) most = larger(most, h[i][e]);
            }
            int shift = 0;
            if (std::is_same_v<T, F16>) {
#pragma unroll
                for (int d = 1; d < kThreads; d *= 2) most = __builtin_fmaxf(most, __shfl_xor(most, d, kWave));
                shift = shift_of<T>(most);
            }
            __syncthreads();  // the last tokens' numbers are read
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
                const int k = (i * kThreads + tid % kThreads) * 8;
                if (k >= (r + kStep - 1) / kStep * kStep) continue;
                Parts<T> p;
                p.set(h[i], __builtin_ldexpf(1.0f, shift));
#pragma unroll
                for (int n = 0; n < kMany; ++n) *reinterpret_cast<uint4*>(&inner[n][slot][k]) = p.v[n];
            }
            if (tid % kThreads == 0) shifts[slot] = shift;
            __syncthreads();
            const int count = min(q.many - held, kHeld);
#pragma unroll 1
            for (int n = 0; n < count; n += kTile) {
                Acc acc[4] = {};
                for (int first = 0; first < r; first += kPart) {
                    if (kPasses) load_up(first);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if (first + k * kStep >= r) break;
                        const int depth = first + k * kStep + quad * 8;
                        uint4 u[kMany];
#pragma unroll
                        for (int i = 0; i < kMany; ++i)
                            u[i] = *reinterpret_cast<const uint4*>(&inner[i][n + col][depth]);
#pragma unroll
                        for (int m = 0; m < 4; ++m)
#pragma unroll
                            for (int i = 0; i < kMany; ++i) acc[m] = Matrix<T>::mac(up[k][m], u[i], acc[m]);
                    }
                    if (!kPasses) break;
                }
                const uint4 was[2] = {old[0], old[1]};
                const long t = q.token(window, n + col < count ? held + n + col : held);
                load_old(held + n + kTile + col);
                if (n + col >= count) continue;
                const int back = -shifts[n + col];
                auto add = [&](uint32_t half, int i) {
                    float v = scale * acc[i / 4][i % 4];
                    if (std::is_same_v<T, F16>) v = __builtin_ldexpf(v, back);
                    return T::from_float(T::to_float(static_cast<uint16_t>(half)) + v);
                };
                uint16_t* out = g.out + t * g.os + mine;
                if (whole) {
#pragma unroll
                    for (int h2 = 0; h2 < 2; ++h2) {
                        uint32_t w[4] = {was[h2].x, was[h2].y, was[h2].z, was[h2].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint16_t low = add(w[e], h2 * 8 + 2 * e);
                            w[e] = static_cast<uint32_t>(add(w[e] >> 16, h2 * 8 + 2 * e + 1)) << 16 | low;
                        }
                        *reinterpret_cast<uint4*>(out + h2 * 32) = uint4{w[0], w[1], w[2], w[3]};
                    }
                } else {
                    const uint16_t* base = g.base + t * g.bs + mine;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int at = i / 8 * 32 + i % 8;
                        if (mine + at < end) out[at] = add(base[at], i);
                    }
                }
            }
        }
    });
    if (blockIdx.y == 0) copy_idle(g, window, idle, row0, min(row0 + kRows, end), wave, kWaves);
}

int check(const char* fn, const spb_adapters* d) {
    if (!d) return invalid("%s: null adapters", fn);
    if (d->num_adapters < 1) return invalid("%s: a pool needs an adapter", fn);
    if (d->rank < 8 || d->rank % 8 || d->rank > kMaxRank)
        return invalid("%s: rank %d must be a multiple of 8 in [8, %d]", fn, d->rank, kMaxRank);
    if (d->cols < 8 || d->cols % 8 || d->cols > kMaxSize)
        return invalid("%s: cols %d must be a multiple of 8 in [8, %d]", fn, d->cols, kMaxSize);
    if (d->num_sections < 1 || d->num_sections > kMaxSections)
        return invalid("%s: %d sections, 1 to %d are possible", fn, d->num_sections, kMaxSections);
    long rows = 0;
    for (int s = 0; s < d->num_sections; ++s) {
        if (d->section_rows[s] < 1) return invalid("%s: a section needs a row", fn);
        rows += d->section_rows[s];
    }
    if (rows > kMaxSize) return invalid("%s: %ld rows, at most %d are possible", fn, rows, kMaxSize);
    if (!d->a || !d->b || !d->scales) return invalid("%s: null weights or scales", fn);
    if (!aligned_to(d->a, 16) || !aligned_to(d->b, 16))
        return invalid("%s: weights must be 16-byte aligned", fn);
    if (!aligned_to(d->scales, 4) || !aligned_to(d->ranks, 4))
        return invalid("%s: scales and ranks must be 4-byte aligned", fn);
    const long st[] = {d->a_adapter_stride, d->a_row_stride, d->b_adapter_stride, d->b_row_stride};
    for (long s : st)
        if (s < 0 || s % 8) return invalid("%s: weight strides must be multiples of 8", fn);
    if (d->a_row_stride < d->cols || d->b_row_stride < d->rank)
        return invalid("%s: weight strides smaller than a row", fn);
    return 0;
}

int check_tokens(const char* fn, int tokens) {
    if (tokens < 0) return invalid("%s: negative number of tokens", fn);
    if (tokens > kMaxSize)
        return invalid("%s: %d tokens, at most %d are possible", fn, tokens, kMaxSize);
    return 0;
}

constexpr int kFewWindows = 16;

// 2^n blocks split the columns of the inner products of up to kSplitWindows[n] windows, the
// largest such n: 512 blocks and more, two a CU, while the outer products' reading of the parts
// does not cost more.  gate|up of 2560 columns, rank 32, the same inputs again and again (they
// fit the last cache; others take 59.6 of the first 46.9): 2049 tokens 46.9 us by 4, 50.9 by 2,
// 57.9 by 8; 4096 86.6 by 4, 79.4 by 2; 1100 34.2 by 4, 40.0 by 8.
constexpr int kSplitWindows[] = {kMaxSize / kWindow, 127, 63, kFewWindows};
constexpr int kMostSplitBits = 3;

int split_bits_of(int tokens) {
    const int windows = (tokens + kWindow - 1) / kWindow;
    int bits = kMostSplitBits;
    while (bits > 0 && windows > kSplitWindows[bits]) --bits;
    return bits;
}

// Of the most parts that up to `tokens` tokens have, for a workspace serves fewer too.
size_t workspace_size(const spb_adapters& d, int tokens) {
    size_t most = 0;
    for (int bits = 0; bits <= kMostSplitBits; ++bits) {
        const int end = kSplitWindows[bits] * kWindow;
        const size_t parts = static_cast<size_t>(tokens < end ? tokens : end) << bits;
        most = parts > most ? parts : most;
    }
    return sizeof(float) * d.num_sections * d.rank * most;
}

// One launch where every CU has a block at most, and A is small: each block reads its section's
// A.  Rank 16 on q|k|v of 2560 columns: 8 tokens of 8 adapters 7.7 us in one launch (240
// blocks), 11.3 in two; 32 tokens of 16 (480) 15.9 and 11.5.  One token, rank 32 on 2560
// columns 9.6 and 11.0, rank 16 on 6912 11.9 and 10.4.
bool fused(const Args& g, long blocks) {
    return blocks <= device_cu_count() && g.rank <= kFusedRank && g.rank * g.cols <= 96 * 1024;
}

template <class T>
int run(const char* fn, const spb_adapters* d, const int* ids, const uint16_t* x,
        const uint16_t* base, uint16_t* output, int tokens, long xs, long bs, long os,
        void* workspace, size_t size, void* stream) {
    clear_error();
    if (int e = check(fn, d)) return e;
    if (int e = check_tokens(fn, tokens)) return e;
    if (tokens == 0) return 0;
    if (!ids || !x || !base || !output) return invalid("%s: null tensor", fn);
    if (!aligned_to(ids, 4)) return invalid("%s: ids must be 4-byte aligned", fn);
    if (!aligned_to(x, 16) || !aligned_to(base, 2) || !aligned_to(output, 2))
        return invalid("%s: x must be 16-byte aligned, base and output 2-byte", fn);
    Args g{};
    g.a = d->a;
    g.b = d->b;
    g.scales = d->scales;
    g.ranks = d->ranks;
    g.ids = ids;
    g.x = x;
    g.base = base;
    g.out = output;
    g.h = static_cast<float*>(workspace);
    g.a_adapter = d->a_adapter_stride;
    g.a_row = d->a_row_stride;
    g.b_adapter = d->b_adapter_stride;
    g.b_row = d->b_row_stride;
    g.xs = xs;
    g.bs = bs;
    g.os = os;
    g.num = d->num_adapters;
    g.rank = d->rank;
    g.cols = d->cols;
    g.sections = d->num_sections;
    g.tokens = tokens;
    while (g.id_bits < 31 && d->num_adapters > 1 << g.id_bits) ++g.id_bits;
    for (int s = 0; s < kMaxSections; ++s) {
        if (s < d->num_sections) g.rows += d->section_rows[s];
        g.end[s] = g.rows;
    }
    if (xs % 8 || xs < 0 || bs < 0 || os < 0 ||
        (tokens > 1 && (xs < d->cols || bs < g.rows || os < g.rows)))
        return invalid("%s: a stride is smaller than a row, or x's no multiple of 8", fn);
    if (base == output && tokens > 1 && bs != os) return invalid("%s: in place with two strides", fn);
    if (!workspace || size < workspace_size(*d, tokens) || !aligned_to(workspace, 16))
        return invalid("%s: a 16-byte aligned workspace of %zu bytes is needed", fn,
                       workspace_size(*d, tokens));
    const hipStream_t st = as_stream(stream);
    g.wide = aligned_to(base, 16) && aligned_to(output, 16) && bs % 8 == 0 && os % 8 == 0;
    for (int s = 0; s + 1 < d->num_sections; ++s) g.wide = g.wide && g.end[s] % 8 == 0;
    const int windows = (tokens + kWindow - 1) / kWindow;
    const int distinct = tokens < kWindow ? tokens : kWindow;  // most adapters of a window
    const int most = distinct < g.num ? distinct : g.num;
    auto tiles = [&](int size) {
        int n = 0;
        for (int s = 0; s < d->num_sections; ++s) n += (d->section_rows[s] + size - 1) / size;
        return n;
    };
    if (fused(g, static_cast<long>(tiles(kFusedRows)) * most * windows)) {
        hipLaunchKernelGGL(fused_kernel<T>, dim3(tiles(kFusedRows), most, windows),
                           dim3(kFusedWaves * kWave), 0, st, g);
        return launch_status(fn);
    }
    // blocks for a window's adapters: as many as can occur, as long as the grid is small
    auto ways = [&](int blocks) { return blocks >= 4096 ? 1 : 4096 / blocks < most ? 4096 / blocks : most; };
    g.split_bits = split_bits_of(tokens);
    const int parts = (g.sections * g.rank + kPart - 1) / kPart;
    const int blocks = parts * (kWindow / kTile) << g.split_bits;
    const dim3 inner(windows, ways(windows * blocks), blocks);
    if (windows <= kFewWindows)
        hipLaunchKernelGGL((shrink_kernel<T, 2>), inner, dim3(kWaves * kWave), 0, st, g);
    else
        hipLaunchKernelGGL((shrink_kernel<T, 5>), inner, dim3(kWaves * kWave), 0, st, g);
    const dim3 grid(tiles(kRows), ways(windows * tiles(kRows)), windows);
    if (g.rank <= kPart)
        hipLaunchKernelGGL((expand_kernel<T, false>), grid, dim3(kWaves * kWave), 0, st, g);
    else
        hipLaunchKernelGGL((expand_kernel<T, true>), grid, dim3(kWaves * kWave), 0, st, g);
    return launch_status(fn);
}

}  // namespace
}  // namespace spb

extern "C" {

size_t spb_adapters_workspace_size(const spb_adapters* adapters, int num_tokens) {
    const char* fn = "spb_adapters_workspace_size";
    spb::clear_error();
    if (spb::check(fn, adapters) || spb::check_tokens(fn, num_tokens)) return 0;
    return spb::workspace_size(*adapters, num_tokens > 0 ? num_tokens : 1);
}

int spb_adapters_f16(const spb_adapters* adapters, const int* ids, const uint16_t* x,
                     const uint16_t* base, uint16_t* output, int num_tokens, long x_stride,
                     long base_stride, long output_stride, void* workspace, size_t workspace_size,
                     spb_stream_t stream) {
    return spb::run<spb::F16>("spb_adapters_f16", adapters, ids, x, base, output, num_tokens,
                              x_stride, base_stride, output_stride, workspace, workspace_size,
                              stream);
}

int spb_adapters_bf16(const spb_adapters* adapters, const int* ids, const uint16_t* x,
                      const uint16_t* base, uint16_t* output, int num_tokens, long x_stride,
                      long base_stride, long output_stride, void* workspace,
                      size_t workspace_size, spb_stream_t stream) {
    return spb::run<spb::BF16>("spb_adapters_bf16", adapters, ids, x, base, output, num_tokens,
                               x_stride, base_stride, output_stride, workspace, workspace_size,
                               stream);
}

}  // extern "C"
