// paged_attention.hip -- attention of a batch of new tokens over a paged cache.
//
// The rows of a tile are (token, query head) pairs of one sequence and one kv
// head, so K and V are read once for all query heads of a kv head.  A wave holds
// 32 rows and walks over keys 32 at a time on the 32x32x16 matrix instructions:
//   S^T = K Q^T   lane l has row l % 32 and keys 8 (i / 4) + 4 (l / 32) + i % 4
//   p = 2^(s c - m), c = scale log2(e), m a running reference of the row
//   O^T += V^T P^T
// The sum over keys of the second product may run in any order, so P goes from
// the first product's result registers straight into the second's operand (keys
// permuted), and V^T's operand is read from LDS in the same permuted order by
// the transposing LDS read (4 keys of one column per lane).
#include <algorithm>
#include <atomic>

#include "paged.hpp"

namespace spb {
namespace {

constexpr int kAttnBlock = 256;
constexpr float kLog2e = 1.44269504088896340736f;

typedef float f32x16 __attribute__((ext_vector_type(16)));
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
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, b2{static_cast<__bf16>(x), static_cast<__bf16>(y)});
    }
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
    int target;   // pieces of work to aim at
    int slots;    // partial results that the workspace holds
    float* ws;
};

// A tile's shape: RG groups of 32 rows times KG groups of NS * 32 keys over the
// four waves.  One group of rows (decoding): the waves take different keys and
// their results are joined at the end; four: all waves read the same keys.
template <int RG>
struct Shape {
    static constexpr int KG = 4 / RG, NS = RG == 1 ? 1 : 2;
    static constexpr int BM = 32 * RG, BN = 32 * KG * NS;
};

// One piece of work: keys [kb, ke) for the tile `qt` of a sequence and kv head.
struct Piece {
    int seq, first, count, len;
    int qt, kvh, lo, hi;  // keys that any row of the tile sees
    int kb, ke;
    int nsplit;  // pieces of this tile
    int slot;    // the tile's first partial result
    int split;
};

__device__ __forceinline__ int lane_int(int v, int l) { return __builtin_amdgcn_readlane(v, l); }

// Positions that the tile's rows see: [lo, hi).
template <int BM>
__device__ __forceinline__ void tile_range(const AttnArgs& a, int count, int len, int qt, int& lo,
                                           int& hi) {
    const int rows = count * static_cast<int>(a.group.d);
    const int i0 = a.group.div(qt * BM), i1 = a.group.div(min(qt * BM + BM, rows) - 1);
    const int p0 = len - count + i0, p1 = len - count + i1;
    hi = a.causal ? min(p1 + 1, len) : len;
    lo = a.window ? max(p0 - a.window + 1, 0) : 0;
    if (hi < lo) hi = lo;
}

// Work item -> piece.  Every wave finds its own, a lane per sequence and 64
// sequences at a time: the total work W (tiles times blocks of BN keys) gives
// the blocks per piece C = ceil(W / target), so long sequences are split and
// short ones are not, whatever the mix; then a prefix sum over the sequences'
// pieces finds the item's.  kTiles: items are (tile, kv head), without splits.
template <int BM, int BN, bool kTiles>
__device__ __forceinline__ bool find_piece(const AttnArgs& a, unsigned item, Piece& r) {
    const int lane = threadIdx.x & (kWave - 1);
    const int group = a.group.d;
    // tokens of a tile: (BM - 1) / group + 1, one more where it begins inside a token
    const int reach = a.window > 0 && a.causal && a.window < 0x3FFFFFFF
                          ? a.window + (BM - 1) / group + 2 : 0x7FFFFFFF;
    SeqSpan q0 = {0, 0, 0};
    if (lane < a.b.seqs) q0 = seq_span(a.b, lane);
    uint64_t work = 0;
    for (int base = 0; base < a.b.seqs; base += kWave) {
        SeqSpan q = q0;
        if (base) {
            q = {0, 0, 0};
            if (base + lane < a.b.seqs) q = seq_span(a.b, base + lane);
        }
        const uint32_t tiles = (static_cast<uint32_t>(q.count) * group + BM - 1) / BM;
        // a window's keys need not begin at a block's
        const uint32_t blocks = min((q.len + BN - 1) / BN, reach / BN + 2);
        uint64_t w = static_cast<uint64_t>(tiles) * blocks;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1)
            w += static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(w), off, kWave));
        work += w;
    }
    work *= a.kv_heads;
    const uint64_t per64 = (work + a.target - 1) / a.target;
    const int per = static_cast<int>(min(max(per64, uint64_t{1}), uint64_t{0x7FFFFFFF}));
    unsigned seen = 0;
    int slot = 0;
    for (int base = 0; base < a.b.seqs; base += kWave) {
        SeqSpan q = q0;
        if (base) {
            q = {0, 0, 0};
            if (base + lane < a.b.seqs) q = seq_span(a.b, base + lane);
        }
        const unsigned tiles = (static_cast<unsigned>(q.count) * group + BM - 1) / BM;
        const int blocks = min((q.len + BN - 1) / BN, reach / BN + 2);
        const int split = max(1, (blocks + per - 1) / per);
        const unsigned all = tiles * a.kv_heads * split;
        const unsigned mine = kTiles ? tiles * a.kv_heads : all;
        const unsigned kept = split > 1 ? all : 0;
        unsigned sum = mine, ksum = kept;
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
            const unsigned x = __shfl_up(sum, off, kWave), y = __shfl_up(ksum, off, kWave);
            if (lane >= off) {
                sum += x;
                ksum += y;
            }
        }
        const uint64_t hit = __ballot(item < seen + sum && mine > 0);
        if (hit) {
            const int l = __ffsll(static_cast<unsigned long long>(hit)) - 1;
            r.seq = base + l;
            r.first = lane_int(q.first, l);
            r.count = lane_int(q.count, l);
            r.len = lane_int(q.len, l);
            const int ns = lane_int(split, l);
            unsigned local = item - (seen + lane_int(static_cast<int>(sum - mine), l));
            const int seq_slot = slot + lane_int(static_cast<int>(ksum - kept), l);
            int sp = 0;
            if (!kTiles) {
                sp = local % ns;
                local /= ns;
            }
            const int unit = local;
            r.kvh = unit % a.kv_heads;
            const int ntiles = lane_int(static_cast<int>(tiles), l);
            r.qt = ntiles - 1 - unit / a.kv_heads;  // the tiles that see most first
            r.slot = seq_slot + unit * ns;
            tile_range<BM>(a, r.count, r.len, r.qt, r.lo, r.hi);
            const int b0 = r.lo / BN, nb = r.hi > r.lo ? (r.hi + BN - 1) / BN - b0 : 0;
            // even pieces of the tile's own blocks
            r.nsplit = min(ns, max(1, (nb + per - 1) / per));
            const int each = max(1, (nb + r.nsplit - 1) / r.nsplit);
            r.nsplit = max(1, (nb + each - 1) / each);
            r.split = sp;
            r.kb = (b0 + sp * each) * BN;
            r.ke = static_cast<int>(min(static_cast<long>(r.hi),
                                        static_cast<long>(b0 + sp * each + each) * BN));
            return kTiles || sp < r.nsplit;
        }
        seen += lane_int(static_cast<int>(sum), kWave - 1);
        slot += lane_int(static_cast<int>(ksum), kWave - 1);
    }
    return false;
}

// Bytes of an LDS row of K or V, and the swizzle of its 16-byte units: lanes
// that read K take one unit of 32 consecutive keys (spread over the units by the
// key), those that read V take 64 bytes of 4 consecutive keys.
template <int HD>
struct Row {
    static constexpr int kPitch = HD <= 64 ? 128 : (HD <= 128 ? 256 : 512);
    static constexpr int kUnits = kPitch / 16;
    static constexpr int kMask = kUnits < 16 ? kUnits - 1 : 15;
    static __device__ __forceinline__ int k_at(int key, int unit) {
        return key * kPitch + ((unit ^ (key & kMask)) << 4);
    }
    static __device__ __forceinline__ int v_at(int key, int unit) {
        const int x = kPitch >= 256 ? (key & 3) << 2 : (key & 2) << 1;
        return key * kPitch + ((unit ^ x) << 4);
    }
};

// x of the lower and of the upper half of the wave, in all lanes.
__device__ __forceinline__ float2 halves(float x) {
    const uint32_t a = __builtin_bit_cast(uint32_t, x);
    const auto s = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    // copies: a bit cast of a vector's element itself reads element 0
    const uint32_t lower = s[0], upper = s[1];
    return make_float2(__builtin_bit_cast(float, lower), __builtin_bit_cast(float, upper));
}
__device__ __forceinline__ float half_max(float x) {
    const float2 h = halves(x);
    return fmaxf(h.x, h.y);
}
__device__ __forceinline__ float half_sum(float x) {
    const float2 h = halves(x);
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

// Inf and NaN of a packed pair replaced by 0; `bad` notes that there was one.
template <class T>
__device__ __forceinline__ uint32_t finite_pair(uint32_t x, bool& bad) {
    constexpr uint32_t e = Prob<T>::kExp;
    const bool lo = (x & e) == e, hi = (x & (e << 16)) == (e << 16);
    bad = bad || lo || hi;
    return x & (lo ? 0xFFFF0000u : 0xFFFFFFFFu) & (hi ? 0x0000FFFFu : 0xFFFFFFFFu);
}

template <class T, int HD, int RG>
__global__ __launch_bounds__(kAttnBlock, HD <= 128 ? 2 : 1) void paged_attention_kernel(
    const AttnArgs a) {
    typedef Shape<RG> S;
    typedef Row<HD> R;
    typedef Prob<T> P;
    constexpr int KG = S::KG, NS = S::NS, BM = S::BM, BN = S::BN;
    constexpr int kSteps = HD / 16, kCols = HD / 32, kUnits = HD / 8;
    constexpr int kLoads = BN * kUnits / kAttnBlock;  // 16-byte units of a thread, K and V each
    extern __shared__ __align__(16) uint8_t attn_smem[];
    uint8_t* const k_lds = attn_smem;
    uint8_t* const v_lds = attn_smem + BN * R::kPitch;
    float* const ml_lds = reinterpret_cast<float*>(attn_smem + 2 * BN * R::kPitch);  // [KG][BM][2]
    int* const bad_lds = reinterpret_cast<int*>(ml_lds + KG * BM * 2);

    Piece w;
    if (!find_piece<BM, BN, false>(a, blockIdx.x, w)) return;

    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int rg = wave % RG, kg = wave / RG, half = lane >> 5;
    const int group = a.group.d, rows = w.count * group;
    const int row0 = w.qt * BM + 32 * rg, row = row0 + (lane & 31);
    const int tok = a.group.div(min(row, rows - 1)), head = w.kvh * group + min(row, rows - 1) - tok * group;
    const bool live = row0 < rows;  // the wave has a row

    // the keys that this lane's row sees, of this piece
    int see_lo = 0, see_hi = 0;
    bool none = true;
    if (row < rows) {
        const int pos = w.len - w.count + tok;
        see_hi = a.causal ? min(pos + 1, w.len) : w.len;
        see_lo = a.window ? max(pos - a.window + 1, 0) : 0;
        none = see_hi <= see_lo;
    }
    // ... and all rows of the wave: keys [all_lo, all_hi) need no mask
    int all_lo = 0, all_hi = 0, any_lo = 0, any_hi = 0;
    if (live) {
        const int t0 = a.group.div(row0), t1 = a.group.div(min(row0 + 31, rows - 1));
        const int p0 = w.len - w.count + t0, p1 = w.len - w.count + t1;
        all_hi = a.causal ? min(p0 + 1, w.len) : w.len;
        any_hi = a.causal ? min(p1 + 1, w.len) : w.len;
        all_lo = a.window ? max(p1 - a.window + 1, 0) : 0;
        any_lo = a.window ? max(p0 - a.window + 1, 0) : 0;
    }
    see_lo = max(see_lo, w.kb);
    see_hi = min(see_hi, w.ke);
    all_lo = max(all_lo, w.kb);
    all_hi = min(all_hi, w.ke);
    any_lo = max(any_lo, w.kb);
    any_hi = min(any_hi, w.ke);

    // Q^T operand: row lane % 32, elements 16 step + 8 half ..
    u32x4 qf[kSteps];
    {
        const uint16_t* qp = a.q + static_cast<long>(w.first + tok) * a.q_stride +
                             static_cast<long>(head) * a.head_dim + 8 * half;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            qf[s] = u32x4{0, 0, 0, 0};
            if (row < rows && 16 * s + 8 * half < a.head_dim)
                qf[s] = *reinterpret_cast<const u32x4*>(qp + 16 * s);
        }
    }

    // Loads of a tile of keys: thread unit i is row (tid + 256 i) / kUnits, unit
    // (tid + 256 i) % kUnits.  Page ids are fetched a tile ahead of their pages.
    const int* const table = a.b.table + static_cast<long>(w.seq) * a.b.width;
    const uint16_t* const kbase = a.k + w.kvh * a.head_stride;
    const uint16_t* const vbase = a.v + w.kvh * a.head_stride;
    u32x4 kreg[kLoads], vreg[kLoads];
    int page[kLoads];
    auto fetch_pages = [&](int t) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int j = t + (tid + kAttnBlock * i) / kUnits;
            page[i] = -1;
            if (j < w.ke) page[i] = table[a.b.page.div(j)];
        }
    };
    bool saw_bad = false;
    auto load_tile = [&](int t) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int idx = tid + kAttnBlock * i, j = t + idx / kUnits, u = idx % kUnits;
            kreg[i] = u32x4{0, 0, 0, 0};
            vreg[i] = u32x4{0, 0, 0, 0};
            const bool there = static_cast<unsigned>(page[i]) < static_cast<unsigned>(a.b.pages);
            saw_bad = saw_bad || (j < w.ke && !there);
            if (j < w.ke && there && 8 * u < a.head_dim) {
                const int slot = j - static_cast<int>(a.b.page.div(j) * a.b.page.d);
                const long at = page[i] * a.page_stride + slot * a.slot_stride + 8 * u;
                kreg[i] = *reinterpret_cast<const u32x4*>(kbase + at);
                vreg[i] = *reinterpret_cast<const u32x4*>(vbase + at);
            }
        }
    };
    auto store_tile = [&]() {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int idx = tid + kAttnBlock * i, r = idx / kUnits, u = idx % kUnits;
            *reinterpret_cast<u32x4*>(k_lds + R::k_at(r, u)) = kreg[i];
            *reinterpret_cast<u32x4*>(v_lds + R::v_at(r, u)) = vreg[i];
        }
        if (saw_bad) *bad_lds = 1;
    };

    f32x16 o[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[c][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    if (tid == 0) *bad_lds = 0;
    fetch_pages(w.kb);
    load_tile(w.kb);
    fetch_pages(w.kb + BN);
    for (int t = w.kb; t < w.ke; t += BN) {
        __syncthreads();
        store_tile();
        __syncthreads();
        if (t + BN < w.ke) {
            load_tile(t + BN);
            fetch_pages(t + 2 * BN);
        }
        const int j0 = t + 32 * NS * kg;  // this wave's keys
        if (!live || j0 >= any_hi || j0 + 32 * NS <= any_lo) continue;
        const uint8_t* const kw = k_lds + 32 * NS * kg * R::kPitch;
        f32x16 s[NS];
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = 0.0f;
#pragma unroll
        for (int st = 0; st < kSteps; ++st)
#pragma unroll
            for (int n = 0; n < NS; ++n)
                s[n] = P::mfma(*reinterpret_cast<const u32x4*>(
                                   kw + R::k_at(32 * n + (lane & 31), 2 * st + half)),
                               qf[st], s[n]);
        const bool bad_page = *bad_lds != 0;
        const bool masked = j0 < all_lo || j0 + 32 * NS > all_hi || bad_page;
        if (masked) {
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int j = j0 + 32 * n + 8 * (i / 4) + 4 * half + i % 4;
                    if (j < see_lo || j >= see_hi) s[n][i] = -INFINITY;
                }
            if (bad_page) {
#pragma unroll
                for (int n = 0; n < NS; ++n)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int j = j0 + 32 * n + 8 * (i / 4) + 4 * half + i % 4;
                        if (j >= see_lo && j < see_hi &&
                            static_cast<unsigned>(table[a.b.page.div(j)]) >=
                                static_cast<unsigned>(a.b.pages))
                            s[n][i] = -INFINITY;
                    }
            }
        }
        // the row's largest score, and its reference
        float top = s[0][0];
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[n][i]);
        top = half_max(top) * a.c - P::kBias;
        const bool move = top > m + P::kSlack;  // also from m = -inf
        if (__any(move)) {
            const float f = move ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
            if (move) m = top;
            l *= f;
#pragma unroll
            for (int c = 0; c < kCols; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[c][i] *= f;
        }
        const float ref = m == -INFINITY ? 0.0f : m;  // a row that has seen nothing yet
        u32x4 pf[NS][2];
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i], a.c, -ref));
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i + 1], a.c, -ref));
                l += x;
                l += y;
                pf[n][i / 8][(i % 8) / 2] = P::pack(x, y);
            }
        // O^T += V^T P^T; lane: column 32 c + lane % 32, keys 4 half .. and 8 + 4 half ..
        const int l16 = lane & 15;
        const uint8_t* const vw = v_lds + 32 * NS * kg * R::kPitch;
        bool bad = false;
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
                    const int key = 32 * n + 16 * g + 4 * half + (l16 >> 2);
                    const int unit = 4 * c + 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
                    const int off = (l16 & 1) << 3;
                    union {
                        s16x4 h[2];
                        u32x4 v;
                    } x;
                    x.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4*)(vw + R::v_at(key, unit) + off));
                    x.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4*)(vw + R::v_at(key + 8, unit) + off));
                    if (masked) {  // 0 * inf would reach rows that do not see the key
#pragma unroll
                        for (int e = 0; e < 4; ++e) x.v[e] = finite_pair<T>(x.v[e], bad);
                    }
                    o[c] = P::mfma(x.v, pf[n][g], o[c]);
                }
        if (__any(bad)) {  // add what was taken out to the rows that see it
            for (int j = 0; j < 32 * NS; ++j) {
                const bool seen = j0 + j >= see_lo && j0 + j < see_hi;
#pragma unroll
                for (int c = 0; c < kCols; ++c)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int d = 32 * c + 8 * (i / 4) + 4 * half + i % 4;
                        const uint16_t x = *reinterpret_cast<const uint16_t*>(
                            vw + R::v_at(j, d >> 3) + 2 * (d & 7));
                        if (seen && (x & P::kExp) == P::kExp) o[c][i] += T::to_float(x);
                    }
            }
        }
    }

    l = half_sum(l);
    float* const part = partial<HD, BM>(a, w.slot + w.split);
    if (KG == 1) {
        if (row >= rows) return;
        const int r = 32 * rg + (lane & 31);
        if (w.nsplit > 1) {
            if (half == 0) {
                part[BM * HD + 2 * r] = m;
                part[BM * HD + 2 * r + 1] = l;
            }
#pragma unroll
            for (int c = 0; c < kCols; ++c)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<float4*>(part + r * HD + 32 * c + 8 * (i / 4) + 4 * half) =
                        make_float4(o[c][i], o[c][i + 1], o[c][i + 2], o[c][i + 3]);
            return;
        }
        const float inv = none ? 0.0f : 1.0f / l;
        uint16_t* const op = a.out + static_cast<long>(w.first + tok) * a.out_stride +
                             static_cast<long>(head) * a.head_dim;
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = 32 * c + 8 * (i / 4) + 4 * half;
                if (d < a.head_dim)
                    store4<T>(op + d, o[c][i] * inv, o[c][i + 1] * inv, o[c][i + 2] * inv,
                              o[c][i + 3] * inv);
            }
        return;
    }
    // join the key groups: the references first, then the scaled sums through LDS
    const int r32 = 32 * rg + (lane & 31);
    if (half == 0) {
        ml_lds[(kg * BM + r32) * 2] = m;
        ml_lds[(kg * BM + r32) * 2 + 1] = l;
    }
    __syncthreads();  // also: every wave has read its last keys
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < KG; ++k) top = fmaxf(top, ml_lds[(k * BM + r32) * 2]);
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
    float* const obuf = reinterpret_cast<float*>(attn_smem);  // [KG][BM][HD]
    const int left = min(rows - w.qt * BM, BM);
    if (row < rows)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = 32 * c + 8 * (i / 4) + 4 * half;
                *reinterpret_cast<float4*>(obuf + (kg * BM + r32) * HD + d) = make_float4(
                    o[c][i] * f, o[c][i + 1] * f, o[c][i + 2] * f, o[c][i + 3] * f);
            }
    __syncthreads();
    for (int idx = tid; idx < left * (HD / 4); idx += kAttnBlock) {
        const int r = idx / (HD / 4), d = 4 * (idx % (HD / 4));
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float tm = -INFINITY, tl = 0.0f;
#pragma unroll
        for (int k = 0; k < KG; ++k) tm = fmaxf(tm, ml_lds[(k * BM + r) * 2]);
#pragma unroll
        for (int k = 0; k < KG; ++k) {
            const float4 y = *reinterpret_cast<const float4*>(obuf + (k * BM + r) * HD + d);
            const float km = ml_lds[(k * BM + r) * 2];
            tl += km == -INFINITY ? ml_lds[(k * BM + r) * 2 + 1]
                                  : ml_lds[(k * BM + r) * 2 + 1] * __builtin_amdgcn_exp2f(km - tm);
            x.x += y.x;
            x.y += y.y;
            x.z += y.z;
            x.w += y.w;
        }
        if (w.nsplit > 1) {
            *reinterpret_cast<float4*>(part + r * HD + d) = x;
            if (d == 0) {
                part[BM * HD + 2 * r] = tm;
                part[BM * HD + 2 * r + 1] = tl;
            }
        } else if (d < a.head_dim) {
            const int gr = w.qt * BM + r, tk = a.group.div(gr);
            const int pos = w.len - w.count + tk;
            const int hi = a.causal ? min(pos + 1, w.len) : w.len;
            const int lo = a.window ? max(pos - a.window + 1, 0) : 0;
            const float inv = hi <= lo ? 0.0f : 1.0f / tl;
            store4<T>(a.out + static_cast<long>(w.first + tk) * a.out_stride +
                          static_cast<long>(w.kvh * group + gr - tk * group) * a.head_dim + d,
                      x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        }
    }
}

// Joins the pieces of split tiles: block (tile and kv head, rows), a group of
// head_dim / 4 threads per piece.
template <class T, int HD, int RG>
__global__ __launch_bounds__(kAttnBlock) void paged_attention_join_kernel(const AttnArgs a,
                                                                          const int per_block) {
    constexpr int BM = Shape<RG>::BM, BN = Shape<RG>::BN;
    constexpr int kLanes = HD / 4, kGroups = kAttnBlock / kLanes;
    __shared__ float acc[kGroups][HD + 2];
    Piece w;
    if (!find_piece<BM, BN, true>(a, blockIdx.x, w) || w.nsplit <= 1) return;
    const int tid = threadIdx.x, g = tid / kLanes, d = 4 * (tid % kLanes);
    const int group = a.group.d, rows = w.count * group;
    const int left = min(rows - w.qt * BM, BM);
    for (int i = 0;; ++i) {  // per_block rows, and on by the grid's if the batch has more than told
        const int r = (i / per_block * gridDim.y + blockIdx.y) * per_block + i % per_block;
        if (r >= left) break;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float m = -INFINITY, l = 0.0f;
        if (g < kGroups)
            for (int s = g; s < w.nsplit; s += kGroups) {
                const float* const p = partial<HD, BM>(a, w.slot + s);
                const float sm = p[BM * HD + 2 * r], sl = p[BM * HD + 2 * r + 1];
                const float4 y = *reinterpret_cast<const float4*>(p + r * HD + d);
                const float top = fmaxf(m, sm);
                const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
                const float h = sm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(sm - top);
                x.x = __builtin_fmaf(x.x, f, y.x * h);
                x.y = __builtin_fmaf(x.y, f, y.y * h);
                x.z = __builtin_fmaf(x.z, f, y.z * h);
                x.w = __builtin_fmaf(x.w, f, y.w * h);
                l = __builtin_fmaf(l, f, sl * h);
                m = top;
            }
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
        if (tid < kLanes && 4 * tid < a.head_dim) {
            float top = -INFINITY, total = 0.0f;
            for (int k = 0; k < kGroups; ++k) top = fmaxf(top, acc[k][HD]);
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int k = 0; k < kGroups; ++k) {
                const float h = acc[k][HD] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(acc[k][HD] - top);
                y.x = __builtin_fmaf(acc[k][d], h, y.x);
                y.y = __builtin_fmaf(acc[k][d + 1], h, y.y);
                y.z = __builtin_fmaf(acc[k][d + 2], h, y.z);
                y.w = __builtin_fmaf(acc[k][d + 3], h, y.w);
                total = __builtin_fmaf(acc[k][HD + 1], h, total);
            }
            const int gr = w.qt * BM + r, tk = a.group.div(gr);
            const int pos = w.len - w.count + tk;
            const int hi = a.causal ? min(pos + 1, w.len) : w.len;
            const int lo = a.window ? max(pos - a.window + 1, 0) : 0;
            const float inv = hi <= lo ? 0.0f : 1.0f / total;
            store4<T>(a.out + static_cast<long>(w.first + tk) * a.out_stride +
                          static_cast<long>(w.kvh * group + gr - tk * group) * a.head_dim + d,
                      y.x * inv, y.y * inv, y.z * inv, y.w * inv);
        }
        __syncthreads();
    }
}

// ---- host -------------------------------------------------------------------

int padded_dim(int hd) { return hd <= 64 ? 64 : (hd <= 96 ? 96 : (hd <= 128 ? 128 : (hd <= 192 ? 192 : 256))); }

// Two blocks per CU are resident; pieces that fill them once.
int target_pieces() { return 2 * device_cu_count(); }

// Split tiles have at most 2 target pieces together: one of a sequence with
// more than C blocks is ceil(blocks / C) < 2 blocks / C pieces, and all tiles'
// blocks / C together are at most the target.
size_t workspace_bytes(int hd) {
    return static_cast<size_t>(2 * target_pieces()) * Shape<4>::BM * (padded_dim(hd) + 2) *
           sizeof(float);
}

constexpr int kMaxAttnDevices = 64;

// Raises a kernel's LDS limit on the current device, once.
template <class F>
int raise_lds(const char* fn, F* kernel, size_t bytes, std::atomic<bool>* done) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxAttnDevices) dev = -1;
    if (dev >= 0 && done[dev].load(std::memory_order_acquire)) return 0;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(bytes));
    if (e != hipSuccess) return failed(fn, e);
    if (dev >= 0) done[dev].store(true, std::memory_order_release);
    return 0;
}

template <class T, int HD, int RG>
int launch_attention(const char* fn, const AttnArgs& a, int max_rows, hipStream_t st) {
    typedef Shape<RG> S;
    constexpr size_t lds = 2 * S::BN * Row<HD>::kPitch + S::KG * S::BM * 2 * sizeof(float) + 16;
    static std::atomic<bool> done[kMaxAttnDevices];
    if (int e = raise_lds(fn, paged_attention_kernel<T, HD, RG>, lds, done)) return e;
    const long rows = static_cast<long>(a.b.tokens) * a.group.d;
    const long tiles = std::min(rows, a.b.seqs + rows / S::BM) * a.kv_heads;
    hipLaunchKernelGGL((paged_attention_kernel<T, HD, RG>), dim3(a.target + tiles),
                       dim3(kAttnBlock), lds, st, a);
    if (int e = launch_status(fn)) return e;
    // a row a block where the rows are few
    const int per = RG == 1 ? 1 : 16;
    const int most = std::min(max_rows, S::BM);
    hipLaunchKernelGGL((paged_attention_join_kernel<T, HD, RG>),
                       dim3(tiles, (most + per - 1) / per), dim3(kAttnBlock), 0, st, a, per);
    return launch_status(fn);
}

template <class T, int HD>
int pick_rows(const char* fn, const AttnArgs& a, int max_rows, hipStream_t st) {
    if (max_rows <= 32) return launch_attention<T, HD, 1>(fn, a, max_rows, st);
    if (max_rows <= 64) return launch_attention<T, HD, 2>(fn, a, max_rows, st);
    return launch_attention<T, HD, 4>(fn, a, max_rows, st);
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
    a.target = target_pieces();
    a.slots = 2 * a.target;
    a.ws = static_cast<float*>(ws);
    const int most_new = b->max_new ? std::min(b->max_new, b->num_tokens) : b->num_tokens;
    const int max_rows = static_cast<int>(std::min<long>(
        static_cast<long>(most_new) * a.group.d, 0x7FFFFFFFL));
    const hipStream_t st = as_stream(stream);
    switch (padded_dim(c->head_dim)) {
    case 64: return pick_rows<T, 64>(fn, a, max_rows, st);
    case 96: return pick_rows<T, 96>(fn, a, max_rows, st);
    case 128: return pick_rows<T, 128>(fn, a, max_rows, st);
    case 192: return pick_rows<T, 192>(fn, a, max_rows, st);
    default: return pick_rows<T, 256>(fn, a, max_rows, st);
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
