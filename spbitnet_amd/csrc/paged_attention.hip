// paged_attention.hip -- attention of a batch of new tokens over a paged cache.
//
// The rows of a tile are (token, query head) pairs of one sequence and one kv
// head, so K and V are read once for all query heads of a kv head.  A wave holds
// W = 32 (or 16) rows and walks over the keys with the matrix instructions that
// take W x W results:
//   S^T = K Q^T   lane l has row l % W and, of each W keys, those
//                 4 (64 / W) (i / 4) + 4 (l / W) + i % 4
//   p = 2^(s c - m), c = scale log2(e), m a running reference of the row
//   O^T += V^T P^T
// The sum over keys of the second product may run in any order, so P goes from
// the first product's result registers straight into the second's operand (keys
// permuted), and V^T's operand is read from LDS in the same permuted order by
// the transposing LDS read (4 keys of one column per lane).
#include <algorithm>
#include <type_traits>

#include "paged.hpp"

namespace spb {
namespace {

constexpr int kJoinBlock = 256;
constexpr float kLog2e = 1.44269504088896340736f;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

// The reference m of a row lets the largest probability be 2^kBias to 2^(kBias +
// kSlack): it moves, and what is summed so far is scaled, only when a score
// passes it by kSlack, which after a row's first tiles is rare.  Powers of two
// cancel in the quotient.  fp16 sits 2^7 up, so that probabilities down to 2^-21
// of the largest stay normal numbers (at most 2^15 of 65504); bf16 has float32's
// range.
template <class T> struct Prob;
template <> struct Prob<F16> {
    static constexpr float kBias = 7.0f, kSlack = 8.0f;
    static constexpr uint32_t kExp = 0x7C00u;
    typedef h16x8 frag;
    static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(frag, a),
                                                      __builtin_bit_cast(frag, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(frag, a),
                                                      __builtin_bit_cast(frag, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, h2{static_cast<_Float16>(x), static_cast<_Float16>(y)});
    }
};
template <> struct Prob<BF16> {
    static constexpr float kBias = 0.0f, kSlack = 8.0f;
    static constexpr uint32_t kExp = 0x7F80u;
    typedef b16x8 frag;
    static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(frag, a),
                                                       __builtin_bit_cast(frag, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(frag, a),
                                                       __builtin_bit_cast(frag, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, b2{static_cast<__bf16>(x), static_cast<__bf16>(y)});
    }
};

// What a worker leaves to the join: the tile that begins in its part and goes on in
// others' (pieces of the tile; 0 if there is none).
struct Split {
    int pieces, first, count, len, qt, kvh;
};

struct AttnArgs {
    BatchArgs b;
    const uint16_t *q, *k, *v;
    uint16_t* out;
    long q_stride, out_stride, page_stride, head_stride, slot_stride;
    int kv_heads, head_dim;
    FastDiv group;  // query heads of a kv head
    float c;        // scale * log2(e)
    int causal, window;
    // keys that a tile with a window sees at most: the window and its tokens, (BM -
    // 1) / group + 1 of them and one more where it begins inside a token
    double reach;
    double per_worker;  // 1 / the least cost worth a worker
    uint32_t workers;   // at most, = blocks launched
    Split* splits;      // [workers]
    float* ws;          // partial results, 2 per worker
};

// A tile of BM = 16 or 128 rows.  Four waves of 32 rows walk over the same keys; the
// 16 of a decoding step (half the arithmetic and registers of 32) are two waves' that
// take turns at 32 keys and join their results at the end.  Tiles of 32 and 64 rows,
// of two waves, were no faster than those of 128 (us, 4 sequences of 8 and 16 tokens,
// 8 heads on 2, 2000 to 4000 positions: 64 wide 23.4 against 18.3 and 26.3 against
// 23.1, 128 wide 27.1 against 25.5 and 39.3 against 29.2, 256 wide 63.3 against 48.9
// and 77.6 against 52.9).
template <int BM>
struct Shape {
    static constexpr int W = BM < 32 ? BM : 32;
    static constexpr int RG = BM / W, KG = RG == 1 ? 2 : 1;  // waves by rows and by keys
    static constexpr int kKeys = RG == 1 ? 32 : 64;          // of a wave
    static constexpr int kWaves = RG * KG, kThreads = kWave * kWaves;
    static constexpr int BN = kKeys * KG;
    static_assert(BN == kWave, "a lane per key of a tile");
};

// A product's result in a wave: W x W, element i of lane l is column l % W and row
// 4 (64 / W) (i / 4) + 4 (l / W) + i % 4.
template <int W> struct Acc;
template <> struct Acc<32> { typedef f32x16 type; };
template <> struct Acc<16> { typedef f32x4 type; };

// How a batch's work is shared out.  Its tiles stand in one line, ordered by
// sequence, kv head and row tile, each as long as its cost (keys seen times the
// group / 16, and a block for what a tile costs besides); the line is cut into
// equal parts, one per worker, and every worker walks over its part.  So the work
// per worker is the same whatever the mix of lengths, and a tile is split only where
// a cut falls into it.  Every wave computes the cuts by itself from the batch's
// arrays, a lane per sequence.  Places are whole numbers in float64, exact below
// 2^53 (rows times keys times the group / 256: 2^48 for a million tokens of 64
// heads over a million keys); a 64-bit integer division took a microsecond of the
// 10 that a small call has.  A cost need not be exact: it decides only who does
// what.
struct Plan {
    double part, total;  // of the line
    uint32_t workers;    // those with work
    __device__ __forceinline__ double cut(uint32_t w) const {
        return w >= workers ? total : floor(part * w);
    }
    // The worker in whose part lies the last of the line before `end` > 0.
    __device__ __forceinline__ uint32_t last_before(double end) const {
        uint32_t w = min(static_cast<uint32_t>(end / part), workers - 1);
        while (w > 0 && cut(w) >= end) --w;
        while (w + 1 < workers && cut(w + 1) < end) ++w;
        return w;
    }
};

// A sequence in the line: tile j of each kv head costs c0 + c1 j.
struct SeqCost {
    double c0, c1, head;  // head: all tiles of one kv head
    int tiles;
};

// Cost of the tiles before tile j.
__device__ __forceinline__ double cost_before(double c0, double c1, int j) {
    const double n = j;
    return n * c0 + c1 * (n * (n - 1.0) * 0.5);
}

template <int BM, int BN>
__device__ __forceinline__ SeqCost seq_cost(const AttnArgs& a, const SeqSpan& q) {
    const int group = a.group.d;
    const uint32_t rows = static_cast<uint32_t>(q.count) * group;
    SeqCost r;
    r.tiles = static_cast<int>((rows + BM - 1) / BM);
    const bool grows = a.causal && (a.window == 0 || a.reach >= q.len);
    const double keys = grows ? max(q.len - q.count, 0) : (a.causal ? a.reach : q.len);
    r.c0 = floor((keys + BN) * group * (1.0 / 16)) + (grows ? BM / 16 : 0) + 1.0;
    r.c1 = grows ? BM / 16 : 0.0;
    r.head = cost_before(r.c0, r.c1, r.tiles);
    return r;
}

__device__ __forceinline__ int lane_int(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
__device__ __forceinline__ double lane_f64(double v, int l) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = lane_int(static_cast<int>(u), l), hi = lane_int(static_cast<int>(u >> 32), l);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// A value that all lanes have, in scalar registers.
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ double scalar(double v) { return lane_f64(v, 0); }

// Sums over the lanes up to each lane, by lane shifts inside rows of 16 and two
// broadcasts across them.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), kCtrl, kRowMask, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), kCtrl, kRowMask, 0xF, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double prefix_sum(double v) {
    v += dpp_f64<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
    v += dpp_f64<0x112, 0xF>(v);
    v += dpp_f64<0x114, 0xF>(v);
    v += dpp_f64<0x118, 0xF>(v);
    v += dpp_f64<0x142, 0xA>(v);  // lane 15 of each even row into the next
    v += dpp_f64<0x143, 0xC>(v);  // lane 31 into the upper half
    return v;
}

// 64 sequences, a lane each: what they cost, and the places where they end in the
// line if the first begins at 0.
struct Lanes {
    SeqSpan q;
    SeqCost c;
    double end;
};

template <int BM, int BN>
__device__ __forceinline__ Lanes look(const AttnArgs& a, int base) {
    Lanes r;
    const int s = base + (threadIdx.x & (kWave - 1));
    r.q = {0, 0, 0};
    if (s < a.b.seqs) r.q = seq_span(a.b, s);
    r.c = seq_cost<BM, BN>(a, r.q);
    r.end = prefix_sum(r.c.head * a.kv_heads);
    return r;
}

template <int BM, int BN>
__device__ __forceinline__ Plan make_plan(const AttnArgs& a, const Lanes& first) {
    Plan p;
    p.total = lane_f64(first.end, kWave - 1);
    for (int base = kWave; base < a.b.seqs; base += kWave)
        p.total += lane_f64(look<BM, BN>(a, base).end, kWave - 1);
    const double most = p.total * a.per_worker + 1.0;
    p.workers = p.total == 0.0 ? 0 : scalar(static_cast<int>(fmin(most, a.workers)));
    p.part = scalar(p.total / p.workers);
    return p;
}

// The tile at a place of the line.
struct Tile {
    double begin, end;  // in the line
    double c0, c1;      // of its sequence
    int tiles, seq, first, count, len;
    int qt, kvh;
};

template <int BM, int BN>
__device__ __forceinline__ Tile find_tile(const AttnArgs& a, Lanes x, double at) {
    double before = 0.0;
    Tile r = {};
    for (int base = 0; base < a.b.seqs; base += kWave) {
        if (base) x = look<BM, BN>(a, base);
        const uint64_t hit = __ballot(at < before + x.end);
        if (hit) {
            const int l = __ffsll(static_cast<unsigned long long>(hit)) - 1;
            r.seq = base + l;
            r.first = lane_int(x.q.first, l);
            r.count = lane_int(x.q.count, l);
            r.len = lane_int(x.q.len, l);
            r.c0 = lane_f64(x.c.c0, l);
            r.c1 = lane_f64(x.c.c1, l);
            r.tiles = lane_int(x.c.tiles, l);
            const double head = lane_f64(x.c.head, l);
            // the place in the sequence
            double in = at - (before + lane_f64(x.end, l) - head * a.kv_heads);
            r.kvh = scalar(static_cast<int>(in / head));
            if (r.kvh * head > in) --r.kvh;  // a quotient that was rounded up
            in -= r.kvh * head;
            r.qt = 0;
            if (r.tiles > 1) {  // cost_before(j) = in, solved in float32, then put right
                const float h = static_cast<float>(r.c0 - 0.5 * r.c1), y = static_cast<float>(in);
                const float c1 = static_cast<float>(r.c1);
                const float j = c1 == 0.0f ? y / h : (sqrtf(h * h + 2.0f * c1 * y) - h) / c1;
                r.qt = min(max(scalar(static_cast<int>(j)), 0), r.tiles - 1);
                while (r.qt > 0 && cost_before(r.c0, r.c1, r.qt) > in) --r.qt;
                while (r.qt + 1 < r.tiles && cost_before(r.c0, r.c1, r.qt + 1) <= in) ++r.qt;
            }
            r.begin = scalar(at - in + cost_before(r.c0, r.c1, r.qt));
            r.end = scalar(r.begin + (r.c0 + r.c1 * r.qt));
            return r;
        }
        before += lane_f64(x.end, kWave - 1);
    }
    return r;
}

template <int BM, int BN>
__device__ __forceinline__ void next_tile(const AttnArgs& a, Tile& t) {
    if (++t.qt == t.tiles) {
        t.qt = 0;
        if (++t.kvh == a.kv_heads) {
            t = find_tile<BM, BN>(a, look<BM, BN>(a, 0), t.end);
            return;
        }
    }
    t.begin = t.end;
    t.end = scalar(t.end + (t.c0 + t.c1 * t.qt));
}

// The first key that a query at a position sees, from 0 on.  A position may be negative
// (fewer cached positions than new tokens) and the window anything up to 2^31 - 1, so
// they are compared before one is taken from the other.
__device__ __forceinline__ int first_seen(const AttnArgs& a, int pos) {
    return a.window && pos >= a.window ? pos - a.window + 1 : 0;
}

// Keys that the tile's rows see: [lo, hi).
template <int BM>
__device__ __forceinline__ void tile_range(const AttnArgs& a, const Tile& t, int& lo, int& hi) {
    const int rows = t.count * static_cast<int>(a.group.d);
    const int i0 = a.group.div(t.qt * BM), i1 = a.group.div(min(t.qt * BM + BM, rows) - 1);
    const int p0 = t.len - t.count + i0, p1 = t.len - t.count + i1;
    hi = a.causal ? min(p1 + 1, t.len) : t.len;
    lo = first_seen(a, p0);
    if (hi < lo) hi = lo;
}

// The blocks of BN keys of a tile that lie before a place of the line: the share of
// the tile's cost, so neighbours that compute it for their common cut agree.
__device__ __forceinline__ int blocks_before(const Tile& t, double at, int blocks) {
    if (at <= t.begin) return 0;
    if (at >= t.end) return blocks;
    return scalar(static_cast<int>((at - t.begin) * blocks / (t.end - t.begin)));
}

// Bytes of an LDS row of K or V, and the swizzle of its 16-byte units: lanes
// that read K take one unit of 32 consecutive keys (spread over the units by the
// key), those that read V take 64 bytes of 4 consecutive keys or 32 of 8.
template <int HD>
struct Row {
    static constexpr int kPitch = HD <= 64 ? 128 : (HD <= 128 ? 256 : 512);
    static constexpr int kUnits = kPitch / 16;
    static constexpr int kMask = kUnits < 16 ? kUnits - 1 : 15;
    static __device__ __forceinline__ int k_unit(int key, int unit) { return unit ^ (key & kMask); }
    static __device__ __forceinline__ int v_unit(int key, int unit) {
        return unit ^ (kPitch >= 256 ? (key & 3) << 2 | (key & 4) >> 1 : (key & 2) << 1 | (key & 4) >> 1);
    }
    static __device__ __forceinline__ int k_at(int key, int unit) {
        return key * kPitch + (k_unit(key, unit) << 4);
    }
    static __device__ __forceinline__ int v_at(int key, int unit) {
        return key * kPitch + (v_unit(key, unit) << 4);
    }
};

// 16 bytes of each active lane from memory to LDS, at lds + 16 lane.
template <bool kStream>  // kStream: non-temporal
__device__ __forceinline__ void load_to_lds(const void* from, uint8_t* lds) {
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)from,
        (__attribute__((address_space(3))) void*)lds, 16, 0, kStream ? 2 : 0);
}
// All of this wave's loads have arrived.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// Whether token i of a sequence sees any position.
__device__ __forceinline__ bool row_sees(const AttnArgs& a, int count, int len, int i) {
    const int pos = len - count + i;
    const int hi = a.causal ? min(pos + 1, len) : len;
    return hi > first_seen(a, pos);
}

// Two exchanges of lanes l and l ^ 32, l and l ^ 16: both lanes' values in both.
__device__ __forceinline__ float2 across32(float x) {
    const uint32_t a = __builtin_bit_cast(uint32_t, x);
    const auto s = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    // copies: a bit cast of a vector's element itself reads element 0
    const uint32_t lower = s[0], upper = s[1];
    return make_float2(__builtin_bit_cast(float, lower), __builtin_bit_cast(float, upper));
}
__device__ __forceinline__ float2 across16(float x) {
    const uint32_t a = __builtin_bit_cast(uint32_t, x);
    const auto s = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    const uint32_t lower = s[0], upper = s[1];
    return make_float2(__builtin_bit_cast(float, lower), __builtin_bit_cast(float, upper));
}
// Over the lanes that hold a row.
template <int W>
__device__ __forceinline__ float row_max(float x) {
    float2 h = across32(x);
    x = fmaxf(h.x, h.y);
    if (W == 32) return x;
    h = across16(x);
    return fmaxf(h.x, h.y);
}
template <int W>
__device__ __forceinline__ float row_sum(float x) {
    float2 h = across32(x);
    x = h.x + h.y;
    if (W == 32) return x;
    h = across16(x);
    return h.x + h.y;
}

// A partial result: O [BM][HD] float32, then (m, l) [BM].
template <int HD, int BM>
__device__ __forceinline__ float* partial(const AttnArgs& a, int slot) {
    return a.ws + static_cast<long>(slot) * (BM * (HD + 2));
}

template <class T>
__device__ __forceinline__ void store4(uint16_t* p, float x, float y, float z, float w) {
    uint2 r;
    r.x = Prob<T>::pack(x, y);
    r.y = Prob<T>::pack(z, w);
    *reinterpret_cast<uint2*>(p) = r;
}

// Not 0 where a packed pair holds an inf or NaN: an exponent of all ones carries
// into the bit above it, and no field into another.
template <class T>
__device__ __forceinline__ uint32_t non_finite(uint32_t x) {
    constexpr uint32_t e = Prob<T>::kExp, one = e & (0u - e);
    return ((x & (e << 16 | e)) + (one << 16 | one)) & 0x80008000u;
}

// One tile's state in a wave: W rows, their sums and statistics.
template <class T, int HD, int BM>
struct RowState {
    static constexpr int W = Shape<BM>::W;
    u32x4 q[HD * W / 512];          // Q^T operand: row lane % W, elements 512 / W step + 8 (lane / W) ..
    typename Acc<W>::type o[HD / W];  // O^T
    float m, l;                     // reference and (these lanes' part of the) sum of the lane's row
    int see_lo, see_hi;             // keys that the lane's row sees, of this piece
    int all_lo, all_hi;             // ... that all rows of the wave see
    int any_lo, any_hi;             // ... that any sees
    // Column of O^T's element i of tile c, in this lane.
    static __device__ __forceinline__ int column(int c, int i) {
        const int lane = threadIdx.x & (kWave - 1);
        return W * c + 256 / W * (i / 4) + 4 * (lane / W) + i % 4;
    }
};

// One tile of keys t .. t + BN in LDS (K, then V) against the wave's rows.  `between`
// is called kBetween times among the matrix products, whose time hides what it issues.
constexpr int kBetween = 4;
template <class T, int HD, int BM, class F>
__device__ __forceinline__ void attend(const AttnArgs& a, RowState<T, HD, BM>& r,
                                       const uint8_t* buf, int t, int kg, uint64_t there,
                                       F between) {
    typedef Row<HD> R;
    typedef Prob<T> P;
    constexpr int W = Shape<BM>::W, kKeys = Shape<BM>::kKeys;
    constexpr int kDepth = 512 / W;                  // of a product
    constexpr int kSteps = HD / kDepth, kTiles = kKeys / W, kCols = HD / W, kEach = W * W / kWave;
    typedef typename Acc<W>::type acc;
    const int j0 = t + kKeys * kg;  // this wave's keys
    if (j0 >= r.any_hi || j0 + kKeys <= r.any_lo) {
        for (int i = 0; i < kBetween; ++i) between(i);
        return;
    }
    const uint8_t* const kw = buf + kKeys * kg * R::kPitch;
    const uint8_t* const vw = kw + Shape<BM>::BN * R::kPitch;
    const int lane = threadIdx.x & (kWave - 1), part = lane / W;
    // Reads of LDS go out two groups ahead of the products that use them: left to itself
    // the compiler puts each right before its use, whose wait then shows.
    acc s[kTiles];
    constexpr int kGroup = kSteps % 2 ? 1 : 2, kGroups = kSteps / kGroup;  // steps
    u32x4 k[2][kGroup][kTiles];
    auto load_k = [&](int g) {
#pragma unroll
        for (int st = 0; st < kGroup; ++st)
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
                k[g & 1][st][n] = *reinterpret_cast<const u32x4*>(
                    kw + R::k_at(W * n + lane % W, kDepth / 8 * (g * kGroup + st) + part));
    };
    load_k(0);
    if (kGroups > 1) load_k(1);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        if (g < kBetween) between(g);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 0; st < kGroup; ++st)
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
                s[n] = P::mfma(k[g & 1][st][n], r.q[g * kGroup + st],
                               g + st == 0 ? acc{} : s[n]);
        __builtin_amdgcn_sched_barrier(0);
        if (g + 2 < kGroups) load_k(g + 2);
    }
#pragma unroll
    for (int g = kGroups; g < kBetween; ++g) between(g);
    // V^T operands of kDepth keys; lane: column W c + lane % W, keys 4 part .. and
    // kDepth / 2 + 4 part ..
    const int l16 = lane & 15;
    auto load_v = [&](int g, u32x4 (&v)[kCols]) {
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
            const int key = kDepth * g + 4 * part + (l16 >> 2);
            const int unit = W / 8 * c + (W == 32 ? lane >> 3 & 2 : 0) + ((l16 & 3) >> 1);
            const int off = (l16 & 1) << 3;
            union {
                s16x4 h[2];
                u32x4 v;
            } x;
            x.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)(vw + R::v_at(key, unit) + off));
            x.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)(vw + R::v_at(key + kDepth / 2, unit) + off));
            v[c] = x.v;
        }
    };
    auto key_of = [&](int n, int i) { return W * n + 256 / W * (i / 4) + i % 4; };  // + 4 part
    u32x4 v[2][kCols];
    if (j0 < r.all_lo || j0 + kKeys > r.all_hi || there != ~uint64_t{0}) {  // not all rows see all
        const int lo = r.see_lo - j0 - 4 * part, hi = r.see_hi - j0 - 4 * part;
        const uint64_t mine = there >> (kKeys * kg + 4 * part);
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int j = key_of(n, i);
                if (j < lo || j >= hi || !(mine >> j & 1)) s[n][i] = -INFINITY;
            }
    }
    // the row's largest score, and its reference
    float top = s[0][0];
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int i = 0; i < kEach; ++i) top = fmaxf(top, s[n][i]);
    top = row_max<W>(top) * a.c - P::kBias;
    const bool move = top > r.m + P::kSlack;  // also from m = -inf
    if (__any(move)) {
        const float f = move ? __builtin_amdgcn_exp2f(r.m - top) : 1.0f;
        if (move) r.m = top;
        r.l *= f;
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int i = 0; i < kEach; ++i) r.o[c][i] *= f;
    }
    const float ref = r.m == -INFINITY ? 0.0f : r.m;  // a row that has seen nothing yet
    load_v(0, v[0]);
    if (kKeys > kDepth) load_v(1, v[1]);
    __builtin_amdgcn_sched_barrier(0);
    constexpr int kParts = kKeys / kDepth;  // 8 probabilities of a lane each
    u32x4 pf[kParts];
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < kTiles * kEach; e += 2) {
        const acc& y = s[e / kEach];
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[e % kEach], a.c, -ref));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[e % kEach + 1], a.c, -ref));
        sum[e % 4] += p0;
        sum[e % 4 + 1] += p1;
        pf[e / 8][e % 8 / 2] = P::pack(p0, p1);
    }
    r.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    // O^T += V^T P^T
#pragma unroll
    for (int g = 0; g < kParts; ++g) {
#pragma unroll
        for (int c = 0; c < kCols; ++c) r.o[c] = P::mfma(v[g & 1][c], pf[g], r.o[c]);
        __builtin_amdgcn_sched_barrier(0);
        if (g + 2 < kParts) load_v(g + 2, v[g & 1]);
    }
}

// Keys of a loaded block that some rows of a tile do not see must not have inf or NaN
// in V: the product of a probability of 0 with them would reach those rows.  So in the
// blocks where the tile's rows differ, and in the one in which a window begins, whose
// first keys no row may see.  Replaces them by 0 in LDS and says whether there were any
// (here or in an earlier tile).  All threads call it.
template <class T, int HD, int BM>
__device__ __forceinline__ bool take_out(uint8_t* buf, int* found) {
    typedef Shape<BM> S;
    constexpr int kEach = S::BN * Row<HD>::kUnits / S::kThreads;
    u32x4* const v = reinterpret_cast<u32x4*>(buf + S::BN * Row<HD>::kPitch) + threadIdx.x;
    u32x4 x[kEach];
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) x[i] = v[i * S::kThreads];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        any |= non_finite<T>(x[i][0]) | non_finite<T>(x[i][1]) | non_finite<T>(x[i][2]) |
               non_finite<T>(x[i][3]);
    if (any) {
#pragma unroll 1
        for (int i = 0; i < kEach; ++i) {
            u32x4 y = v[i * S::kThreads];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t bad = non_finite<T>(y[e]);
                y[e] &= (bad & 0x8000u ? 0u : 0x0000FFFFu) | (bad >> 31 ? 0u : 0xFFFF0000u);
            }
            v[i * S::kThreads] = y;
        }
        *found = 1;
    }
    __syncthreads();
    return *found != 0;
}

// Adds what take_out took out of the tile to the rows that see it, from memory.
template <class T, int HD, int BM>
__device__ __forceinline__ void put_back(const AttnArgs& a, RowState<T, HD, BM>& r, int t, int end,
                                         int kg, const int* table, const uint16_t* vbase) {
    constexpr int W = Shape<BM>::W, kKeys = Shape<BM>::kKeys, kEach = W * W / kWave;
    const int part = (threadIdx.x & (kWave - 1)) / W;
    for (int j = t + kKeys * kg; j < min(t + kKeys * (kg + 1), end); ++j) {
        const int p = a.b.page.div(j), id = table[p];
        if (static_cast<unsigned>(id) >= static_cast<unsigned>(a.b.pages)) continue;
        const uint16_t* const v = vbase + id * a.page_stride +
                                  (j - p * static_cast<int>(a.b.page.d)) * a.slot_stride + 4 * part;
        const bool mine = j >= r.see_lo && j < r.see_hi;
        int hd = a.head_dim - 4 * part;
        asm volatile("" : "+v"(hd));  // else the comparisons below are kept over all tiles
#pragma unroll
        for (int c = 0; c < HD / W; ++c)
#pragma unroll
            for (int i = 0; i < kEach; i += 4) {
                const int d = W * c + 256 / W * (i / 4);
                if (d >= hd) continue;
                const uint2 x = *reinterpret_cast<const uint2*>(v + d);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t y = (e < 2 ? x.x : x.y) >> (e % 2 * 16) & 0xFFFFu;
                    if (mine && (y & Prob<T>::kExp) == Prob<T>::kExp)
                        r.o[c][i + e] += T::to_float(static_cast<uint16_t>(y));
                }
            }
    }
}

// What lanes load for keys and columns that are not there.
__device__ __align__(16) const uint32_t kZeros[4] = {0, 0, 0, 0};

// Blocks of a CU that LDS and registers hold.
template <int HD, int BM>
constexpr int resident() { return HD > 128 ? 1 : (BM == 16 && HD <= 64 ? 4 : 2); }
template <int HD, int BM>
constexpr int waves_per_simd() { return Shape<BM>::kWaves * resident<HD, BM>() >= 8 ? 2 : 1; }

// Tiles of 16 rows are a sequence's only ones: no two read the same keys, which are
// loaded non-temporal (32 ragged sequences of one token 75.8 -> 68.5 us).  With 128 rows
// others may read them too (2048 tokens 250 -> 313 us), and one tile of 20 to 64 rows
// gains nothing either (9 sequences of 5 tokens 18.1 against 17.9).
//
// What bounds it.  Decoding: memory, K and V being read once.  One sequence of 131,072
// positions (336 MB) takes 65.7 us with the join, 5.1 TB/s, 32 ragged ones (363 MB)
// 68.2, 5.3 TB/s; a large copy reaches 4.9.  Heads whose padded row has columns to spare
// go by load_any, and wait: one sequence of 131,072 takes 62.7 us 80 wide, 3.4 TB/s, and
// 161.6 us 192 wide, 3.1, where 64, 128 and 256 reach 4.5, 5.2 and 5.5.
// Many rows: 2048 tokens behind 8192 (193 GFLOP) take 233 to 262 us with the join, 0.74
// to 0.83 PFLOP/s, where a large library product reaches 1.17 to 1.22.  The kernel's part
// is 510,000 cycles, whose clock moves between 1.95 and 2.3 GHz.  By counters the matrix
// units are busy 45 % of the time and the vector units 50 %, as each wave does scores,
// softmax and values one after the other and the two waves of a SIMD overlap little.  10
// of the 256 registers are spilled (36 bytes a lane).  256 wide, one wave a SIMD, it is
// 69 of 512 (264 bytes): 2048 tokens behind 2048, 8 heads, 127 us, 0.41 PFLOP/s; 192 wide
// 111 us, 0.35, without spills; 128 wide 61 us, 0.42.
// Small calls: a chain of dependent steps.  One token behind 2048 positions: 14.6 us a
// call, traces 11.8 of it here and 4.0 in the join.  By time stamps a block's first wave
// takes 13,500 cycles, 5.4 us (lengths and the cut 4800, pages and Q until the first
// keys' loads are out 3200, keys 3000, the end 2500), the slowest block 8.4 (two tiles),
// and first start to last end 8.5; the rest of the trace is the launch's start and end.
// Not kept: K and V staged in registers (spills, whose reloads wait in order behind
// the loads: 444 us for the same 2048 tokens); two sets of 32 rows in a wave with K
// and V read once for both (512 registers, 150 spilled: 609 us); raised priorities
// around the products or the softmax (250.6 and 246 against 250).
template <class T, int HD, int BM>
__global__ __launch_bounds__((Shape<BM>::kThreads), (waves_per_simd<HD, BM>()))
void paged_attention_kernel(const AttnArgs a) {
    typedef Shape<BM> S;
    typedef Row<HD> R;
    constexpr int W = S::W, RG = S::RG, KG = S::KG, BN = S::BN;
    constexpr int kDepth = 512 / W, kSteps = HD / kDepth, kCols = HD / W, kEach = W * W / kWave;
    constexpr int kRows = kWave / R::kUnits;          // rows of K that a wave's load fills
    constexpr int kLoads = BN / (kRows * S::kWaves);  // loads of a wave, K and V each
    // Two tiles of keys: one is filled while the other is read.  Two arrays, so that
    // the compiler sees that reads of one need not wait for loads into the other.
    __shared__ __align__(16) uint8_t buf0[2 * BN * R::kPitch];
    __shared__ __align__(16) uint8_t buf1[2 * BN * R::kPitch];
    __shared__ float ml_lds[KG][BM][2];
    __shared__ int found_lds;  // take_out's

    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = scalar(tid / kWave);
    const int rg = wave % RG, kg = wave / RG, part = lane / W;
    const int group = a.group.d;
    if (tid == 0) found_lds = 0;  // the next barrier is before the first tile's
    Split left_over = {0, 0, 0, 0, 0, 0};
    Plan plan = {};
    Tile w = {};
    double from = 0.0, to = 0.0;
    uint32_t worker = 0;

    for (bool first = true;; first = false) {
        if (first) {  // in the loop: what the compiler takes out of it comes before these loads' wait
            const Lanes lanes = look<BM, BN>(a, 0);
            plan = make_plan<BM, BN>(a, lanes);
            if (blockIdx.x >= plan.workers) {
                if (tid == 0) a.splits[blockIdx.x].pieces = 0;
                return;
            }
            // Blocks go to the 8 dies in turn, each with its own L2: a die gets a run of
            // the line, whose neighbouring tiles read the same keys (2048 tokens behind 8192
            // 243 us; dies interleaved every 1, 4, 8, 16 or 32 workers 255, 250, 259, 254, 248).
            const uint32_t die = blockIdx.x & 7, of_die = plan.workers >> 3, more = plan.workers & 7;
            worker = die * of_die + min(die, more) + (blockIdx.x >> 3);
            from = scalar(plan.cut(worker));
            to = scalar(plan.cut(worker + 1));
            w = find_tile<BM, BN>(a, lanes, from);
        } else {
            next_tile<BM, BN>(a, w);
        }
        const int rows = w.count * group;
        const bool whole = w.begin >= from && w.end <= to;
        int kb, ke;  // this worker's keys of the tile
        {
            int lo, hi;
            tile_range<BM>(a, w, lo, hi);
            const int b0 = lo / BN, blocks = hi > lo ? (hi + BN - 1) / BN - b0 : 0;
            const int k0 = blocks_before(w, from, blocks), k1 = blocks_before(w, to, blocks);
            kb = (b0 + k0) * BN;
            ke = k0 == k1 ? kb : (k1 == blocks ? hi : (b0 + k1) * BN);
        }
        // Loads go from memory straight to LDS, 16 bytes a lane and a wave's lanes side
        // by side; the swizzle is in which unit of its row a lane fetches.  Lane i of a
        // wave finds the place of key t + i, its page a tile ahead of its use; a load's
        // lanes get their rows' places from it.  Keys past the piece's end, those of bad
        // pages and columns past head_dim are zeros.
        const int* const table = a.b.table + static_cast<long>(w.seq) * a.b.width;
        int page = 0;
        auto fetch_page = [&](int t) {
            if (t < ke) page = table[a.b.page.div(min(t + lane, ke - 1))];
        };
        fetch_page(kb);
        const uint16_t* const kbase = a.k + w.kvh * a.head_stride;
        const uint16_t* const vbase = a.v + w.kvh * a.head_stride;
        const int units = a.head_dim / 8;

        const int row0 = w.qt * BM + W * rg, row = row0 + lane % W;
        const int tok = a.group.div(min(row, rows - 1));
        const int head = w.kvh * group + min(row, rows - 1) - tok * group;
        RowState<T, HD, BM> r;
        {
            const uint16_t* qp = a.q + static_cast<long>(w.first + tok) * a.q_stride +
                                 static_cast<long>(head) * a.head_dim + 8 * part;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                r.q[s] = u32x4{0, 0, 0, 0};
                if (row < rows && kDepth * s + 8 * part < a.head_dim)
                    r.q[s] = *reinterpret_cast<const u32x4*>(qp + kDepth * s);
            }
        }
        r.see_lo = r.see_hi = r.all_lo = r.all_hi = r.any_lo = r.any_hi = 0;
        bool none = true;
        if (row < rows) {
            const int pos = w.len - w.count + tok;
            r.see_hi = a.causal ? min(pos + 1, w.len) : w.len;
            r.see_lo = first_seen(a, pos);
            none = r.see_hi <= r.see_lo;
        }
        if (row0 < rows) {
            const int t0 = a.group.div(row0), t1 = a.group.div(min(row0 + W, rows) - 1);
            const int p0 = w.len - w.count + t0, p1 = w.len - w.count + t1;
            r.all_hi = a.causal ? min(p0 + 1, w.len) : w.len;
            r.any_hi = a.causal ? min(p1 + 1, w.len) : w.len;
            r.all_lo = first_seen(a, p1);
            r.any_lo = first_seen(a, p0);
        }
        r.see_lo = max(r.see_lo, kb);
        r.see_hi = min(r.see_hi, ke);
        r.all_lo = max(r.all_lo, kb);
        r.all_hi = min(r.all_hi, ke);
        r.any_lo = max(r.any_lo, kb);
        r.any_hi = min(r.any_hi, ke);
        // where the rows' keys begin and end: from lo0 (the tile's first row) to lo1 (its
        // last), the same for a single token, and hi0 to hi1.  Keys from hi1 on are zeros
        // (ke), those before lo0 are not: a tile's first block begins at a multiple of BN.
        int lo0, lo1, hi0, hi1;
        {
            const int t0 = a.group.div(w.qt * BM), t1 = a.group.div(min(w.qt * BM + BM, rows) - 1);
            const int p0 = w.len - w.count + t0, p1 = w.len - w.count + t1;
            hi0 = a.causal ? p0 + 1 : w.len;
            hi1 = a.causal ? p1 + 1 : w.len;
            lo0 = first_seen(a, p0);
            lo1 = first_seen(a, p1);
        }
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int i = 0; i < kEach; ++i) r.o[c][i] = 0.0f;
        r.m = -INFINITY;
        r.l = 0.0f;

        // Where a page's slots come in whole runs of a load's rows, all rows of a load
        // have one place: a scalar base and a lane offset that stays the same.
        const bool runs = a.b.page.d % kRows == 0 && units == R::kUnits &&
                          a.slot_stride < (1L << 24);  // the offset is 32 bits
        const uint32_t lane_row = (lane / R::kUnits) * static_cast<uint32_t>(a.slot_stride) * 2;
        uint64_t there = ~uint64_t{0}, next = ~uint64_t{0};
        long at = 0;
        bool easy = true;
        auto place_tile = [&](int t) {  // of the next tile's keys, and which are there
            const int j = min(t + lane, ke - 1);
            const int slot = j - static_cast<int>(a.b.page.div(j) * a.b.page.d);
            const bool in_pool = static_cast<unsigned>(page) < static_cast<unsigned>(a.b.pages);
            next = __ballot(in_pool);
            const bool here = in_pool && t + lane < ke;
            at = here ? page * a.page_stride + slot * a.slot_stride : -1;
            easy = runs && __ballot(here) == ~uint64_t{0};
        };
        auto load_part = [&](int i, uint8_t* buf) {  // load i of kLoads, easy
            const int row = (i * S::kWaves + wave) * kRows;  // of the wave's first lane
            const uint32_t lo = lane_int(static_cast<int>(at), row);
            const uint32_t hi = lane_int(static_cast<int>(at >> 32), row);
            const long off = static_cast<long>(static_cast<uint64_t>(hi) << 32 | lo);
            const int key = row + lane / R::kUnits;
            const uint32_t ku = lane_row + 16 * R::k_unit(key, lane % R::kUnits);
            const uint32_t vu = lane_row + 16 * R::v_unit(key, lane % R::kUnits);
            load_to_lds<BM == 16>(reinterpret_cast<const char*>(kbase + off) + ku, buf + row * R::kPitch);
            load_to_lds<BM == 16>(reinterpret_cast<const char*>(vbase + off) + vu,
                                  buf + (BN + row) * R::kPitch);
        };
        auto load_any = [&](uint8_t* buf) {  // the tile, any lengths, pages and head_dim
            int ln = lane;
            asm volatile("" : "+v"(ln));  // its numbers are not held in registers meanwhile
            const int at_lo = static_cast<int>(at), at_hi = static_cast<int>(at >> 32);
#pragma unroll 1
            for (int i = 0; i < kLoads; ++i) {
                const int row = (i * S::kWaves + wave) * kRows;
                const int key = row + ln / R::kUnits;
                const uint32_t lo = __shfl(at_lo, key, kWave), hi = __shfl(at_hi, key, kWave);
                const long off = static_cast<long>(static_cast<uint64_t>(hi) << 32 | lo);
                const int ku = R::k_unit(key, ln % R::kUnits), vu = R::v_unit(key, ln % R::kUnits);
                const uint16_t* const zeros = reinterpret_cast<const uint16_t*>(kZeros);
                load_to_lds<BM == 16>(off < 0 || ku >= units ? zeros : kbase + off + 8 * ku,
                                      buf + row * R::kPitch);
                load_to_lds<BM == 16>(off < 0 || vu >= units ? zeros : vbase + off + 8 * vu,
                                      buf + (BN + row) * R::kPitch);
            }
        };
        if (kb < ke) {
            place_tile(kb);
            there = next;
            if (easy) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) load_part(i, buf0);
            } else {
                load_any(buf0);
            }
        }
        fetch_page(kb + BN);

        auto step = [&](int t, uint8_t* buf, uint8_t* other) {
            wait_loads();
            __syncthreads();
            bool spread = false;
            if (t + BN < ke) {
                place_tile(t + BN);
                spread = easy;
                if (!easy) load_any(other);
            }
            bool taken = false;
            if ((t < hi1 && t + BN > hi0 && hi0 < hi1) || (t < lo1 && t + BN > lo0))
                taken = take_out<T, HD, BM>(buf, &found_lds);
            attend<T, HD, BM>(a, r, buf, t, kg, there, [&](int i) {
                if (spread)
#pragma unroll
                    for (int k = 0; k < kLoads; ++k)
                        if (k * kBetween / kLoads == i) load_part(k, other);
            });
            if (taken) put_back<T, HD, BM>(a, r, t, ke, kg, table, vbase);
            fetch_page(t + 2 * BN);
            there = next;
        };
        for (int t = kb; t < ke; t += 2 * BN) {
            step(t, buf0, buf1);
            if (t + BN >= ke) break;
            step(t + BN, buf1, buf0);
        }

        r.l = row_sum<W>(r.l);
        float* const piece = partial<HD, BM>(a, 2 * worker + (w.begin >= from ? 1 : 0));
        const int rt = W * rg + lane % W;  // the lane's row of the tile
        if (KG == 1) {
            if (row >= rows) {
            } else if (!whole) {
                if (part == 0) {
                    piece[BM * HD + 2 * rt] = r.m;
                    piece[BM * HD + 2 * rt + 1] = r.l;
                }
#pragma unroll
                for (int c = 0; c < kCols; ++c)
#pragma unroll
                    for (int i = 0; i < kEach; i += 4)
                        *reinterpret_cast<float4*>(piece + rt * HD + r.column(c, i)) =
                            make_float4(r.o[c][i], r.o[c][i + 1], r.o[c][i + 2], r.o[c][i + 3]);
            } else {
                const float inv = none ? 0.0f : 1.0f / r.l;
                uint16_t* const op = a.out + static_cast<long>(w.first + tok) * a.out_stride +
                                     static_cast<long>(head) * a.head_dim;
#pragma unroll
                for (int c = 0; c < kCols; ++c)
#pragma unroll
                    for (int i = 0; i < kEach; i += 4) {
                        const int d = r.column(c, i);
                        if (d < a.head_dim)
                            store4<T>(op + d, r.o[c][i] * inv, r.o[c][i + 1] * inv,
                                      r.o[c][i + 2] * inv, r.o[c][i + 3] * inv);
                    }
            }
        } else {
            // join the waves' keys: the references first, then the scaled sums through LDS
            if (part == 0) {
                ml_lds[kg][rt][0] = r.m;
                ml_lds[kg][rt][1] = r.l;
            }
            __syncthreads();  // also: every wave has read its last keys
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < KG; ++k) top = fmaxf(top, ml_lds[k][rt][0]);
            const float f = r.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(r.m - top);
            float* const obuf = reinterpret_cast<float*>(buf0);  // [KG][BM][HD]
            const int left = min(rows - w.qt * BM, BM);
            if (row < rows)
#pragma unroll
                for (int c = 0; c < kCols; ++c)
#pragma unroll
                    for (int i = 0; i < kEach; i += 4)
                        *reinterpret_cast<float4*>(obuf + (kg * BM + rt) * HD + r.column(c, i)) =
                            make_float4(r.o[c][i] * f, r.o[c][i + 1] * f, r.o[c][i + 2] * f,
                                        r.o[c][i + 3] * f);
            __syncthreads();
            for (int idx = tid; idx < left * (HD / 4); idx += S::kThreads) {
                const int y = idx / (HD / 4), d = 4 * (idx % (HD / 4));
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float tm = -INFINITY, tl = 0.0f;
#pragma unroll
                for (int k = 0; k < KG; ++k) tm = fmaxf(tm, ml_lds[k][y][0]);
#pragma unroll
                for (int k = 0; k < KG; ++k) {
                    const float4 z = *reinterpret_cast<const float4*>(obuf + (k * BM + y) * HD + d);
                    const float km = ml_lds[k][y][0], kl = ml_lds[k][y][1];
                    tl += km == -INFINITY ? kl : kl * __builtin_amdgcn_exp2f(km - tm);
                    x.x += z.x;
                    x.y += z.y;
                    x.z += z.z;
                    x.w += z.w;
                }
                if (!whole) {
                    *reinterpret_cast<float4*>(piece + y * HD + d) = x;
                    if (d == 0) {
                        piece[BM * HD + 2 * y] = tm;
                        piece[BM * HD + 2 * y + 1] = tl;
                    }
                } else if (d < a.head_dim) {
                    const int gr = w.qt * BM + y, tk = a.group.div(gr);
                    const float inv = row_sees(a, w.count, w.len, tk) ? 1.0f / tl : 0.0f;
                    store4<T>(a.out + static_cast<long>(w.first + tk) * a.out_stride +
                                  static_cast<long>(w.kvh * group + gr - tk * group) * a.head_dim + d,
                              x.x * inv, x.y * inv, x.z * inv, x.w * inv);
                }
            }
        }
        if (w.end >= to || w.end <= w.begin) {
            if (w.begin >= from && w.end > to)  // who else has a part of it
                left_over = {static_cast<int>(plan.last_before(w.end) - worker) + 1, w.first, w.count,
                             w.len, w.qt, w.kvh};
            break;
        }
        __syncthreads();  // the next tile's loads overwrite what this one's waves read
    }
    if (tid == 0) a.splits[worker] = left_over;
}

// Joins the pieces of split tiles: block (worker in which the tile begins, rows).
// HD / 4 threads take a row, 4 columns each; kSpread: they take every kGroups-th
// piece of the block's one row, else all pieces of a row of their own.
template <class T, int HD, int BM, bool kSpread>
__global__ __launch_bounds__(kJoinBlock) void paged_attention_join_kernel(const AttnArgs a) {
    constexpr int kLanes = HD / 4, kGroups = kJoinBlock / kLanes;
    __shared__ float acc[kSpread ? kGroups : 1][HD + 2];
    const Split w = a.splits[blockIdx.x];
    if (w.pieces == 0) return;
    const int tid = threadIdx.x, g = tid / kLanes, d = 4 * (tid % kLanes);
    const int group = a.group.d, rows = w.count * group;
    const int left = min(rows - w.qt * BM, BM);
    const int per_block = kSpread ? 1 : kGroups;
    // on by the grid's rows if the batch has more than the caller told
    for (int r0 = blockIdx.y * per_block; r0 < left; r0 += gridDim.y * per_block) {
        const int r = kSpread ? r0 : r0 + g;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float m = -INFINITY, l = 0.0f;
        if (g < kGroups && r < left) {
#pragma unroll 4
            for (int s = kSpread ? g : 0; s < w.pieces; s += kSpread ? kGroups : 1) {
                // the piece where the tile begins is its worker's second, the others' first
                const float* const p = partial<HD, BM>(a, 2 * (blockIdx.x + s) + (s == 0 ? 1 : 0));
                const float2 ml = *reinterpret_cast<const float2*>(p + BM * HD + 2 * r);
                const float4 y = *reinterpret_cast<const float4*>(p + r * HD + d);
                const float top = fmaxf(m, ml.x);
                const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
                const float h = ml.x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ml.x - top);
                x.x = __builtin_fmaf(x.x, f, y.x * h);
                x.y = __builtin_fmaf(x.y, f, y.y * h);
                x.z = __builtin_fmaf(x.z, f, y.z * h);
                x.w = __builtin_fmaf(x.w, f, y.w * h);
                l = __builtin_fmaf(l, f, ml.y * h);
                m = top;
            }
        }
        if (kSpread) {
            if (g < kGroups) {
                acc[g][d] = x.x;
                acc[g][d + 1] = x.y;
                acc[g][d + 2] = x.z;
                acc[g][d + 3] = x.w;
                if (d == 0) {
                    acc[g][HD] = m;
                    acc[g][HD + 1] = l;
                }
            }
            __syncthreads();
            if (g == 0) {
                float top = -INFINITY;
                for (int k = 0; k < kGroups; ++k) top = fmaxf(top, acc[k][HD]);
                x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                l = 0.0f;
                for (int k = 0; k < kGroups; ++k) {
                    const float h = acc[k][HD] == -INFINITY
                                        ? 1.0f : __builtin_amdgcn_exp2f(acc[k][HD] - top);
                    x.x = __builtin_fmaf(acc[k][d], h, x.x);
                    x.y = __builtin_fmaf(acc[k][d + 1], h, x.y);
                    x.z = __builtin_fmaf(acc[k][d + 2], h, x.z);
                    x.w = __builtin_fmaf(acc[k][d + 3], h, x.w);
                    l = __builtin_fmaf(acc[k][HD + 1], h, l);
                }
            }
            __syncthreads();  // before the next row's
        }
        if ((kSpread ? g == 0 : g < kGroups && r < left) && d < a.head_dim) {
            const int gr = w.qt * BM + r, tk = a.group.div(gr);
            const float inv = row_sees(a, w.count, w.len, tk) ? 1.0f / l : 0.0f;
            store4<T>(a.out + static_cast<long>(w.first + tk) * a.out_stride +
                          static_cast<long>(w.kvh * group + gr - tk * group) * a.head_dim + d,
                      x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        }
    }
}

// ---- host -------------------------------------------------------------------

int padded_dim(int hd) { return hd <= 64 ? 64 : (hd <= 96 ? 96 : (hd <= 128 ? 128 : (hd <= 192 ? 192 : 256))); }

size_t splits_bytes(int workers) { return (workers * sizeof(Split) + 255) / 256 * 256; }

// A worker per resident block.
template <int HD, int BM>
int worker_count() { return device_cu_count() * resident<HD, BM>(); }

// A worker has at most two tiles that it shares with others: its first and its last.
template <int HD, int BM>
size_t workspace_of() {
    const size_t workers = worker_count<HD, BM>();
    return splits_bytes(workers) + 2 * workers * BM * (HD + 2) * sizeof(float);
}

template <int HD>
size_t workspace_of_any() {
    return std::max(workspace_of<HD, 16>(), workspace_of<HD, 128>());
}

size_t workspace_bytes(int hd) {
    switch (padded_dim(hd)) {
    case 64: return workspace_of_any<64>();
    case 96: return workspace_of_any<96>();
    case 128: return workspace_of_any<128>();
    case 192: return workspace_of_any<192>();
    default: return workspace_of_any<256>();
    }
}

template <class T, int HD, int BM>
int launch_attention(const char* fn, AttnArgs a, void* ws, int max_rows, hipStream_t st) {
    typedef Shape<BM> S;
    // Fewest keys worth a worker of their own.  us with 32 / 64 / 128 / 256 for one token
    // behind 2048: 15.7 / 14.2 / 15.6 / 17.5.  For 128 rows with 64 / 128: 4 sequences of 8
    // tokens (8 heads on 2, 2000 to 4000 positions) 33.7 / 26.6 at 128 wide, 22.8 / 18.7 at
    // 64; 9 of 5 tokens in a window of 1000 16.2 / 18.2; with 128 / 256 / 512: 256 tokens
    // 24.4 / 29.1 / 43.6, 2048 behind 8192 242 / 239 / 241.
    constexpr int kMinKeys = BM == 16 ? 64 : 128;
    a.workers = worker_count<HD, BM>();
    a.reach = static_cast<double>(a.window) + ((BM - 1) / a.group.d + 2);
    a.per_worker = 16.0 / (static_cast<double>(kMinKeys) * a.group.d);
    a.splits = static_cast<Split*>(ws);
    a.ws = reinterpret_cast<float*>(static_cast<char*>(ws) + splits_bytes(a.workers));
    hipLaunchKernelGGL((paged_attention_kernel<T, HD, BM>), dim3(a.workers),
                       dim3(S::kThreads), 0, st, a);
    if (int e = launch_status(fn)) return e;
    // few rows may have many pieces: a row a block, its pieces side by side
    constexpr bool kSpread = BM == 16;
    constexpr int per = kSpread ? 1 : kJoinBlock / (HD / 4);
    const int most = std::min(max_rows, BM);
    hipLaunchKernelGGL((paged_attention_join_kernel<T, HD, BM, kSpread>),
                       dim3(a.workers, (most + per - 1) / per), dim3(kJoinBlock), 0, st, a);
    return launch_status(fn);
}

template <class T, int HD>
int pick_rows(const char* fn, const AttnArgs& a, void* ws, int max_rows, hipStream_t st) {
    if (max_rows <= 16) return launch_attention<T, HD, 16>(fn, a, ws, max_rows, st);
    return launch_attention<T, HD, 128>(fn, a, ws, max_rows, st);
}

int check_heads(const char* fn, int nh, int nkv, int hd) {
    if (nh < 1 || nkv < 1 || nh % nkv)
        return invalid("%s: num_heads %d must be a positive multiple of num_kv_heads %d", fn, nh, nkv);
    if (hd < 8 || hd % 8 || hd > 256)
        return invalid("%s: head_dim %d must be a multiple of 8 in [8, 256]", fn, hd);
    return 0;
}

template <class T>
int paged_attention(const char* fn, const spb_paged_cache* c, const spb_paged_batch* b,
                    const uint16_t* q, uint16_t* out, long qs, long os, int nh, float scale,
                    int causal, int window, void* ws, size_t ws_size, spb_stream_t stream) {
    clear_error();
    if (int e = check_paged_cache(fn, c)) return e;
    if (int e = check_paged_batch(fn, b)) return e;
    if (int e = check_heads(fn, nh, c->num_kv_heads, c->head_dim)) return e;
    if (!(scale > 0.0f) || !(scale < INFINITY)) return invalid("%s: scale must be positive", fn);
    if (window < 0) return invalid("%s: negative window", fn);
    if (b->num_tokens == 0 || b->num_seqs == 0) return 0;
    const long row = static_cast<long>(nh) * c->head_dim;
    if (static_cast<long>(b->num_tokens) * nh > 0x7FFFFFFFL - 256)
        return invalid("%s: more than 2^31 rows", fn);
    if (!q || !out) return invalid("%s: null pointer", fn);
    if (!aligned_to(q, 16) || !aligned_to(out, 16) || qs % 8 || os % 8)
        return invalid("%s: q and output must be 16-byte aligned, their strides multiples of 8", fn);
    if (qs < 0 || (b->num_tokens > 1 && os < row))
        return invalid("%s: strides smaller than a token's heads", fn);
    if (q == out && qs != os) return invalid("%s: in place with two strides", fn);
    if (!ws || !aligned_to(ws, 16) || ws_size < workspace_bytes(c->head_dim))
        return invalid("%s: workspace must be 16-byte aligned and hold %zu bytes", fn,
                       workspace_bytes(c->head_dim));
    AttnArgs a = {};
    a.b = batch_args(*c, *b);
    a.q = q;
    a.k = c->k;
    a.v = c->v;
    a.out = out;
    a.q_stride = qs;
    a.out_stride = os;
    a.page_stride = c->page_stride;
    a.head_stride = c->head_stride;
    a.slot_stride = c->slot_stride;
    a.kv_heads = c->num_kv_heads;
    a.head_dim = c->head_dim;
    a.group = FastDiv(static_cast<uint32_t>(nh / c->num_kv_heads));
    a.c = scale * kLog2e;
    a.causal = causal != 0;
    a.window = window;
    const int most_new = b->max_new ? std::min(b->max_new, b->num_tokens) : b->num_tokens;
    const int max_rows = static_cast<int>(std::min<long>(
        static_cast<long>(most_new) * a.group.d, 0x7FFFFFFFL));
    const hipStream_t st = as_stream(stream);
    switch (padded_dim(c->head_dim)) {
    case 64: return pick_rows<T, 64>(fn, a, ws, max_rows, st);
    case 96: return pick_rows<T, 96>(fn, a, ws, max_rows, st);
    case 128: return pick_rows<T, 128>(fn, a, ws, max_rows, st);
    case 192: return pick_rows<T, 192>(fn, a, ws, max_rows, st);
    default: return pick_rows<T, 256>(fn, a, ws, max_rows, st);
    }
}

}  // namespace
}  // namespace spb

using namespace spb;

extern "C" {

size_t spb_paged_attention_workspace_size(int num_heads, int num_kv_heads, int head_dim) {
    clear_error();
    if (check_heads("spb_paged_attention_workspace_size", num_heads, num_kv_heads, head_dim))
        return 0;
    return workspace_bytes(head_dim);
}

int spb_paged_attention_f16(const spb_paged_cache* cache, const spb_paged_batch* batch,
                            const uint16_t* q, uint16_t* output, long q_stride,
                            long output_stride, int num_heads, float scale, int causal,
                            int window, void* workspace, size_t workspace_size,
                            spb_stream_t stream) {
    return paged_attention<F16>("spb_paged_attention_f16", cache, batch, q, output, q_stride,
                                output_stride, num_heads, scale, causal, window, workspace,
                                workspace_size, stream);
}
int spb_paged_attention_bf16(const spb_paged_cache* cache, const spb_paged_batch* batch,
                             const uint16_t* q, uint16_t* output, long q_stride,
                             long output_stride, int num_heads, float scale, int causal,
                             int window, void* workspace, size_t workspace_size,
                             spb_stream_t stream) {
    return paged_attention<BF16>("spb_paged_attention_bf16", cache, batch, q, output, q_stride,
                                 output_stride, num_heads, scale, causal, window, workspace,
                                 workspace_size, stream);
}

}  // extern "C"
