// sampling.hip -- what follows a batch's logits: the next token of each row under
// its request's temperature, top-k, top-p and min-p, from given random numbers, and
// the log-probabilities of tokens with the best alternatives of each row.
//
// The tokens of a row stand in the order of falling logits, equal ones by index, with
// weights w = exp((l - max) / temperature); NaN counts as minus infinity.  Each of the
// three filters keeps a first part of that order, so the kept tokens are the first n,
// and the token taken is the first whose weight with those before it passes u times
// their sum M.  All that is looked for is a place in one order where a sum of counts
// or weights passes a bound: a histogram of the logits says in which bins, and only
// those bins' tokens are sorted.
//
// Sums of weights decide between neighbours among up to 2^24 tokens, and must not depend
// on the order of adding: weights are computed in float64, to 2^-38 of their values, and
// added as 64-bit whole numbers.  A step relative to a row's largest weight, 1, would lose what
// many far tokens weigh together (2^24 of them at e^-27 have 3e-5 of a row, each is below half
// a step of 2^-38): each bin has a step of its own, 2^-38 (2^24 tokens) to 2^-49 of its weights.
#include "common.hpp"
#include "paged.hpp"
#include "spbitnet_amd.h"

#include <type_traits>

namespace spb {
namespace {

constexpr int kMaxVocab = 1 << 24;
constexpr int kMaxRows = 1 << 20;
constexpr int kMaxTop = 64;
constexpr int kRow = 512;  // threads on one row
constexpr int kWaves = kRow / kWave;

struct F32 {
    using Bits = float;
    static constexpr int kVec = 4;  // logits of a 16-byte load
    static __device__ __forceinline__ float load(const Bits* p) { return *p; }
    static __device__ __forceinline__ void unpack(const uint4& q, float* v) {
        v[0] = __builtin_bit_cast(float, q.x);
        v[1] = __builtin_bit_cast(float, q.y);
        v[2] = __builtin_bit_cast(float, q.z);
        v[3] = __builtin_bit_cast(float, q.w);
    }
};
template <class T>
struct Half {
    using Bits = uint16_t;
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float load(const Bits* p) { return T::to_float(*p); }
    static __device__ __forceinline__ void unpack(const uint4& q, float* v) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = T::to_float(static_cast<uint16_t>(w[i]));
            v[2 * i + 1] = T::to_float(static_cast<uint16_t>(w[i] >> 16));
        }
    }
};

// A logit with NaN as minus infinity: the maximum of a NaN and a number is the number.
__device__ __forceinline__ float clean(float v) { return __builtin_fmaxf(v, -__builtin_inff()); }

// Order of the logits as unsigned numbers, with one zero.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_key(uint32_t k) {
    return __builtin_bit_cast(float, k >> 31 ? k & 0x7fffffffu : ~k);
}

// ---- over a wave and over a block of kRow threads -------------------------------------
// Lane to lane moves (DPP) of 4- and 8-byte values: a step is an instruction or two, where
// a shuffle goes through LDS.

// The value of the lane that kCtrl names, or `none` where there is no such lane.
template <int kCtrl, int kRowMask, class V>
__device__ __forceinline__ V lane_move(V none, V v) {
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(
            V, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v),
                                           kCtrl, kRowMask, 0xf, false));
    } else {
        const auto n = __builtin_bit_cast(uint64_t, none), b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_update_dpp(static_cast<int>(n), static_cast<int>(b),
                                                        kCtrl, kRowMask, 0xf, false);
        const uint32_t hi =
            __builtin_amdgcn_update_dpp(static_cast<int>(n >> 32), static_cast<int>(b >> 32),
                                        kCtrl, kRowMask, 0xf, false);
        return __builtin_bit_cast(V, static_cast<uint64_t>(hi) << 32 | lo);
    }
}

// op over the lanes up to this one; none: op(none, v) = v.
template <class V, class Op>
__device__ __forceinline__ V wave_scan(V v, V none, Op op) {
    v = op(lane_move<0x111, 0xf>(none, v), v);  // 1, 2, 4, 8 lanes below, within 16
    v = op(lane_move<0x112, 0xf>(none, v), v);
    v = op(lane_move<0x114, 0xf>(none, v), v);
    v = op(lane_move<0x118, 0xf>(none, v), v);
    v = op(lane_move<0x142, 0xa>(none, v), v);  // lane 15 of the 16 below
    v = op(lane_move<0x143, 0xc>(none, v), v);  // lane 31
    return v;
}

struct Add {
    template <class V>
    __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Min {
    template <class V>
    __device__ __forceinline__ V operator()(V a, V b) const { return b < a ? b : a; }
};
struct Max {
    template <class V>
    __device__ __forceinline__ V operator()(V a, V b) const { return b > a ? b : a; }
};

// The value of lane `from`, the same for all.
template <class V>
__device__ __forceinline__ V from_lane(V v, int from) {
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), from));
    } else {
        const auto b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), from);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), from);
        return __builtin_bit_cast(V, static_cast<uint64_t>(hi) << 32 | lo);
    }
}

// op over the waves' results in part, by each wave (kWaves <= 16 lanes).
template <class V, class Op>
__device__ __forceinline__ V parts_scan(const V* part, V none, Op op) {
    const int lane = threadIdx.x % kWave;
    V v = lane < kWaves ? part[lane] : none;
    v = op(lane_move<0x111, 0xf>(none, v), v);
    v = op(lane_move<0x112, 0xf>(none, v), v);
    v = op(lane_move<0x114, 0xf>(none, v), v);
    if constexpr (kWaves > 8) v = op(lane_move<0x118, 0xf>(none, v), v);
    return v;
}

// Every thread gets the result.  part: kWaves values.
template <class V, class Op>
__device__ __forceinline__ V block_reduce(V v, V none, V* part, Op op) {
    v = wave_scan(v, none, op);
    __syncthreads();
    if (threadIdx.x % kWave == kWave - 1) part[threadIdx.x / kWave] = v;
    __syncthreads();
    return from_lane(parts_scan(part, none, op), kWaves - 1);
}

// The sum of v over the threads before this one, and of all.  before() and after() are on
// either side of a barrier.
template <class V>
struct BlockScan {
    V upto;
    __device__ __forceinline__ void before(V v, V* part) {
        upto = wave_scan(v, V{0}, Add());
        if (threadIdx.x % kWave == kWave - 1) part[threadIdx.x / kWave] = upto;
    }
    __device__ __forceinline__ V after(const V* part, V* total) {
        const V below = lane_move<0x138, 0xf>(V{0}, upto);  // of the lane below
        const V parts = parts_scan(part, V{0}, Add());
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
        *total = from_lane(parts, kWaves - 1);
        return wave ? from_lane(parts, wave - 1) + below : below;
    }
};

template <class V>
__device__ __forceinline__ V block_scan(V v, V* part, V* total) {
    BlockScan<V> s;
    __syncthreads();
    s.before(v, part);
    __syncthreads();
    return s.after(part, total);
}

// The value of lane ^ kLanes.
template <int kLanes>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    if constexpr (kLanes == 1) return __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, false);
    if constexpr (kLanes == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, false);
    if constexpr (kLanes == 4) {  // the 8 mirrored (^ 7), then each 4 (^ 3)
        const uint32_t m = __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false);
        return __builtin_amdgcn_update_dpp(0, m, 0x1b, 0xf, 0xf, false);
    }
    if constexpr (kLanes == 8) return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false);
    if constexpr (kLanes == 16) {
        const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? p[0] : p[1];
    }
    const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? p[0] : p[1];
}
__device__ __forceinline__ uint64_t lane_xor(uint64_t v, int lanes) {
    const uint32_t lo = static_cast<uint32_t>(v), hi = static_cast<uint32_t>(v >> 32);
    auto both = [](uint32_t h, uint32_t l) { return static_cast<uint64_t>(h) << 32 | l; };
    switch (lanes) {
        case 1: return both(lane_xor<1>(hi), lane_xor<1>(lo));
        case 2: return both(lane_xor<2>(hi), lane_xor<2>(lo));
        case 4: return both(lane_xor<4>(hi), lane_xor<4>(lo));
        case 8: return both(lane_xor<8>(hi), lane_xor<8>(lo));
        case 16: return both(lane_xor<16>(hi), lane_xor<16>(lo));
        default: return both(lane_xor<32>(hi), lane_xor<32>(lo));
    }
}

// ---- sampling -------------------------------------------------------------------

struct SampleArgs {
    const void* logits;
    long stride;
    const float* uniforms;
    int* tokens;
    float* logprobs;  // may be null
    int vocab;
    spb_sampling set;
};

constexpr double kPerUnit = 0x1.71547652b82fep+6;  // 64 / ln 2

// A row's settings, with what is off or out of range taken care of.
struct Settings {
    double t, u;
    double top_p, min_p;  // 1 and 0: off
    int k;                // vocab: off
    double per;           // 1/64 octaves of a weight per unit of a logit
    float bins;           // bins per unit of a logit
    uint32_t octaves;     // a bin's width in 2^-20 octaves of a weight, at most 2^20 / 64 / ln 2
    int bits;             // a bin's weights, as numbers of up to 1, are added as whole numbers
    double one;           // of 2^-bits; one = 2^(52 - bits)
};

__device__ __forceinline__ Settings settings_of(const SampleArgs& g, int row) {
    Settings s;
    float heat = g.set.temperatures ? g.set.temperatures[row] : g.set.temperature;
    int k = g.set.top_ks ? g.set.top_ks[row] : g.set.top_k;
    const float p = g.set.top_ps ? g.set.top_ps[row] : g.set.top_p;
    const float m = g.set.min_ps ? g.set.min_ps[row] : g.set.min_p;
    const float u = g.uniforms[row];
    if (k <= 0 || k > g.vocab) k = g.vocab;
    if (!(heat > 0.0f)) {  // greedy: the first token of the order
        heat = 1.0f;
        k = 1;
    }
    if (p <= 0.0f) k = 1;
    s.top_p = p < 1.0f && p > 0.0f ? p : 1.0;
    s.min_p = m > 0.0f ? (m < 1.0f ? m : 1.0) : 0.0;
    s.k = k;
    s.t = heat;
    s.per = kPerUnit / s.t;
    s.u = u > 0.0f ? (u < 1.0f ? u : 0x1.fffffep-1) : 0.0;
    s.bits = min(49, 31 + __clz(g.vocab));  // a row of ones stays below 2^63
    s.one = __builtin_ldexp(1.0, 52 - s.bits);
    return s;
}

// 2^(y / 64) for y in [-64, 0] times 64 / ln 2, times 2^(up / 2^20), up a multiple of 2^20: y is
// a whole number k and a rest; 2^(k / 64) from a table of 64 in LDS and the exponent, the rest's
// exponential by its series, of which float64 needs to hold the first term only: the others
// are below 2^-15 and in float32 off by 2^-38.7 of the result at most (20 million y compared with
// long double).  A float64 instruction takes twice a float32 one's time (8 cycles a wave, as
// measured): 11 of them here with y's own, where a series for a whole octave takes 19.
__device__ __forceinline__ void fill_powers(double* powers) {
    if (threadIdx.x < 64) powers[threadIdx.x] = exp2(threadIdx.x / 64.0);
}
__device__ __forceinline__ double power_of(double y, uint32_t up, const double* powers) {
    constexpr double kStep = 0x1.62e42fefa39efp-7;  // ln 2 / 64
    const double z = y + 0x1.8p52;                  // its low word is y rounded
    const int k = static_cast<int>(__builtin_bit_cast(uint64_t, z));
    const double r = y - (z - 0x1.8p52);
    const float f = static_cast<float>(r);
    constexpr float c2 = kStep * kStep / 2, c3 = kStep * kStep * kStep / 6,
                    c4 = kStep * kStep * kStep * kStep / 24;
    const float rest = f * f * __builtin_fmaf(f, __builtin_fmaf(f, c4, c3), c2);
    const double p = __builtin_fma(r, kStep, static_cast<double>(rest));
    const double t = powers[k & 63];
    const auto w = __builtin_bit_cast(uint64_t, __builtin_fma(t, p, t));
    const uint32_t hi = static_cast<uint32_t>(w >> 32) + (static_cast<uint32_t>(k) << 14 & 0xfff00000u) + up;
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | static_cast<uint32_t>(w));
}

// Weight of a logit (not minus infinity) at or below `top`.
__device__ __forceinline__ double weight_of(float l, float top, double per, const double* powers) {
    const double y = (static_cast<double>(l) - static_cast<double>(top)) * per;
    if (l == top) return 1.0;
    // 2^24 weights below e^-64 are nothing beside the first, 1
    return y > -64.0 * kPerUnit ? power_of(y, 0, powers) : 0.0;
}

// A weight as a whole number of 2^-52 * one: the sum's low bits (those of a power of two are 0).
__device__ __forceinline__ unsigned long long fixed(double w, double one) {
    const auto b = __builtin_bit_cast(unsigned long long, w + one);
    const uint32_t hi = static_cast<uint32_t>(b >> 32) -
                        static_cast<uint32_t>(__builtin_bit_cast(unsigned long long, one) >> 32);
    return static_cast<unsigned long long>(hi) << 32 | static_cast<uint32_t>(b);
}

// -- from the row itself, in up to 15 readings (its sums, four digits for each of the three
// -- places, twice for the token's index): for rows whose borders fall among thousands of
// -- nearly equal logits, and those that bins do not fit

// A sum of weights of all sizes up to 1: whole numbers of 2^-38, and what that leaves of each
// (2^-39 at most, of either sign) as whole numbers of 2^-76.  2^24 weights are off by 2^-53.
struct Mass {
    unsigned long long coarse, fine;

    static __device__ __forceinline__ Mass of(double w) {
        const double z = w + 0x1p14, rest = w - (z - 0x1p14);
        return {fixed(w, 0x1p14), __builtin_bit_cast(unsigned long long, rest + 0x1.8p-24) -
                                      __builtin_bit_cast(unsigned long long, 0x1.8p-24)};
    }
    __device__ __forceinline__ double value() const {
        return __builtin_fma(static_cast<double>(static_cast<long long>(fine)), 0x1p-76,
                             static_cast<double>(coarse) * 0x1p-38);
    }
};

// Four of each digit side by side, a lane adds to one of them: most lanes have the same digit.
struct Hist {
    static constexpr int kSides = 4;
    unsigned long long coarse[256][kSides], fine[256][kSides];
    int count[256][kSides];
    int digit;
    int before_count;
    Mass before_mass;
};

template <class T>
struct Row {
    const typename T::Bits* l;
    const double* powers;
    int vocab;
    float top;
    double per;

    __device__ __forceinline__ double weight(float v) const { return weight_of(v, top, per, powers); }

    // f(logit) of this thread's, minus infinities apart; the loads of the next four are in flight.
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        constexpr int kAhead = 4;
        float v[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
            const int i = threadIdx.x + n * kRow;
            v[n] = i < vocab ? T::load(l + i) : 0.0f;
        }
#pragma unroll 1
        for (int i = threadIdx.x; i < vocab; i += kRow) {
            const float now = clean(v[0]);
#pragma unroll
            for (int n = 1; n < kAhead; ++n) v[n - 1] = v[n];
            if (i + kAhead * kRow < vocab) v[kAhead - 1] = T::load(l + i + kAhead * kRow);
            if (now != -__builtin_inff()) f(now);
        }
    }
};

// A place in the order: the logit there, how many of that logit stand before it, and the
// weights before it.
struct Place {
    uint32_t key;
    int before_ties;
    double mass;
};

// By count, the token of rank `rank`; by mass, the first token whose weight with those
// before it is above bound (at the end of all of them the last with a weight).  Four
// digits of the key, each a histogram of the tokens that share the digits before it.
template <bool kMass, class T>
__device__ __forceinline__ Place select(const Row<T>& r, int rank, double bound, Hist& h) {
    uint32_t prefix = 0;
    int count = 0;
    Mass mass = {0, 0};
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256 * Hist::kSides; i += kRow) {
            (&h.coarse[0][0])[i] = 0;
            (&h.fine[0][0])[i] = 0;
            (&h.count[0][0])[i] = 0;
        }
        __syncthreads();
        r.each([&](float l) {
            const uint32_t key = key_of(l);
            if (shift < 24 && (key >> (shift + 8)) != (prefix >> (shift + 8))) return;
            const int d = key >> shift & 255;
            // equal logits are added by one lane: a row of 128256 times one value took 1000 us
            // with each lane adding its own, 440 so
            const bool led = key == __builtin_amdgcn_readfirstlane(key);
            const unsigned long long same = __ballot(led);
            const int times = led ? __popcll(same) : 1;
            if (led && threadIdx.x % kWave != __ffsll(same) - 1) return;
            const Mass m = Mass::of(r.weight(l));
            const int side = threadIdx.x % Hist::kSides;
            atomicAdd(&h.count[d][side], times);
            atomicAdd(&h.coarse[d][side], times * m.coarse);
            atomicAdd(&h.fine[d][side], times * m.fine);
        });
        __syncthreads();
        if (threadIdx.x < kWave) {  // a wave takes the digits from the highest on, 4 a lane
            const int lane = threadIdx.x;
            int c[4], sum_c = 0;
            Mass m[4], sum_m = {0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 255 - 4 * lane - i;
                c[i] = 0;
                m[i] = {0, 0};
#pragma unroll
                for (int side = 0; side < Hist::kSides; ++side) {
                    c[i] += h.count[d][side];
                    m[i].coarse += h.coarse[d][side];
                    m[i].fine += h.fine[d][side];
                }
                sum_c += c[i];
                sum_m.coarse += m[i].coarse;
                sum_m.fine += m[i].fine;
            }
            const int upto_c = wave_scan(sum_c, 0, Add());
            int bc = count + upto_c - sum_c, at_c = 0, first = -1, last = -1;
            Mass bm = {mass.coarse + wave_scan(sum_m.coarse, 0ull, Add()) - sum_m.coarse,
                       mass.fine + wave_scan(sum_m.fine, 0ull, Add()) - sum_m.fine},
                 at_m = {0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (first >= 0) continue;
                if (kMass ? (m[i].coarse | m[i].fine) != 0 : c[i] != 0) {
                    last = i;
                    at_c = bc;
                    at_m = bm;
                }
                bc += c[i];
                bm.coarse += m[i].coarse;
                bm.fine += m[i].fine;
                if (last == i && (kMass ? bm.value() > bound : bc > rank)) first = i;
            }
            // the first digit that passes, or the last that has tokens
            const unsigned long long passed = __ballot(first >= 0), some = __ballot(last >= 0);
            const int to = passed ? __ffsll(passed) - 1 : some ? 63 - __clzll(some) : -1;
            if (to < 0 ? lane == 0 : lane == to) {
                h.digit = to < 0 ? -1 : 255 - 4 * lane - last;
                h.before_count = at_c;
                h.before_mass = at_m;
            }
        }
        __syncthreads();
        if (h.digit < 0) break;
        prefix |= static_cast<uint32_t>(h.digit) << shift;
        count = h.before_count;
        mass = h.before_mass;
    }
    Place p;
    p.key = prefix;
    int ties = 0;
    for (int side = 0; side < Hist::kSides; ++side) ties += h.count[prefix & 255][side];
    const double w = r.weight(from_key(prefix));
    p.mass = mass.value();
    double in = kMass ? (bound - p.mass) / w : rank - count;
    in = in < ties - 1 ? in : ties - 1;
    p.before_ties = in > 0 ? static_cast<int>(in) : 0;
    p.mass += p.before_ties * w;
    return p;
}

template <class T>
__device__ __forceinline__ void sample_row(const SampleArgs& g, int row, const Settings& s, float top, const double* powers,
                           Hist& h) {
    __shared__ union {
        int i[kWaves];
        unsigned long long u[kWaves];
    } part;
    Row<T> r;
    r.l = static_cast<const typename T::Bits*>(g.logits) + row * g.stride;
    r.powers = powers;
    r.vocab = g.vocab;
    r.per = s.per;
    r.top = top;
    // the kept mass: the least of what each filter keeps
    Mass all = {0, 0}, high = {0, 0};
    int live = 0;
    r.each([&](float l) {
        ++live;
        const double w = r.weight(l);
        const Mass m = Mass::of(w);
        all.coarse += m.coarse;
        all.fine += m.fine;
        if (w >= s.min_p) {
            high.coarse += m.coarse;
            high.fine += m.fine;
        }
    });
    live = block_reduce(live, 0, part.i, Add());
    auto sum = [](const Mass& m) {
        return Mass{block_reduce(m.coarse, 0ull, part.u, Add()), block_reduce(m.fine, 0ull, part.u, Add())}
            .value();
    };
    double kept = sum(all);
    const double over = sum(high);
    if (s.k < live) kept = select<false>(r, s.k, 0.0, h).mass;
    if (s.top_p < 1.0) {
        // the token at the place passes the bound: it is the last that stays, unless the
        // mass before it is the bound already
        const double bound = s.top_p * kept;
        const Place p = select<true>(r, 0, bound, h);
        const double cut = p.mass < bound ? p.mass + r.weight(from_key(p.key)) : p.mass;
        kept = cut < kept ? cut : kept;
    }
    if (s.min_p > 0.0 && over < kept) kept = over;
    const Place p = select<true>(r, 0, s.u * kept, h);
    // the before_ties-th token of that logit, in the order of indices
    const int each = (g.vocab + kRow - 1) / kRow;
    const int first = min(static_cast<int>(threadIdx.x) * each, g.vocab);
    const int end = min(first + each, g.vocab);
    int here = 0;
    for (int i = first; i < end; ++i) here += key_of(clean(T::load(r.l + i))) == p.key;
    int ties;
    int left = p.before_ties - block_scan(here, part.i, &ties);
    if (left < 0 || left >= here) return;
    for (int i = first; i < end; ++i) {
        if (key_of(clean(T::load(r.l + i))) != p.key) continue;
        if (left-- > 0) continue;
        g.tokens[row] = i;
        if (g.logprobs)
            g.logprobs[row] = static_cast<float>(log(r.weight(from_key(p.key)) / kept));
        break;
    }
}

// -- with a histogram: of 2048 bins of the logits, from the row's largest down, the weights
// -- and, where top-k is on, the tokens.  Bins are 1/64 of the temperature wide, or where that
// -- reaches below the row's least logit, 1/2047 of the row's range: 256 rows of nearly equal
// -- logits (128256 within 0.2) took 1290 us with the fixed width, their bins' tokens being more
// -- than the list holds, and 112 so.  What is below the last bin is in the last.  A bin's weights
// -- are within a factor of 1.02 of each other and are added as multiples of a power of two of
// -- their own; those in the last bin go on down from 2^-46 (where bins go by the range, they end
// -- with it).  The sums say which bins hold a border of a filter or the place of u: their tokens
// -- (some hundreds, mostly) are taken from the row, sorted, and decide.  Between the bins nothing needs an order.  So a row is read three
// -- times: for its largest logit, for the bins, and for those tokens; parts whose largest
// -- logit is below the bins in question are left out the third time.
// --
// -- 512 rows of 128256 float32 logits, top-p 0.95, a block a row: 168 us.  Mean of the blocks: 42
// -- for the largest logits (memory, 6 TB/s), 63 for the bins (issue of the weights' float64), 3 for
// -- their sums and borders, 34 for the tokens in question (memory), 11 for sorting them and the end,
// -- 152 in all; the slowest one's bins take 80.  The two blocks of a CU go through them in step.
// --
// -- A bin of thousands of equal logits overflows the list and leaves the row to the selection
// -- above.  16-bit logits have such bins in flat rows: bfloat16 ones between 8 and 16 are 1/16
// -- apart.  512 flat bfloat16 rows of 128256 take 1.1 ms (float32 0.17, fp16 0.17), of 200000 at a
// -- temperature of 1.5 2.3 ms (float32 0.28).

constexpr int kBins = 2048;
constexpr int kOwn = kBins / kRow;  // bins of a thread
constexpr int kList = 4096;         // tokens of the bins in question
constexpr int kSplitBins = 64;      // most bins that are split again
constexpr int kPeaks = 1024;        // units of a row whose largest logit is kept in LDS
constexpr int kSplitBlock = 256;
constexpr float kMask = -4096.0f;   // no model's logit: below it a mask's finite stand-in

struct SampleWork {
    float* peaks;              // [rows][units]: the largest logit of each
    float* lows;               // [rows][units]: the least one (Lows)
    unsigned long long* mass;  // [rows][kBins]
    int* count;                // [rows][kBins], where top-k is on
    unsigned long long* list;  // [rows][kList]
    int* listed;               // [rows]: tokens in the list, and blocks that are done
    int* done;
    int units, parts;  // units of a row, blocks of a row in the last kernel
};

// A wave's part of a row: 16 logits a lane in loads of 16 bytes, from 16-byte boundaries
// on, so unit u begins up to 7 logits before u * kSize.
template <class T>
struct Unit {
    static constexpr int kLoads = 16 / T::kVec, kSize = 16 * kWave;
    uint4 bits[kLoads];

    static __device__ __forceinline__ int start(const typename T::Bits* row, int unit) {
        const int skew = (reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename T::Bits);
        return unit * kSize - skew + static_cast<int>(threadIdx.x % kWave) * T::kVec;
    }
    __device__ __forceinline__ void load(const typename T::Bits* row, int vocab, int unit) {
        const int first = start(row, unit);
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int i = first + n * kWave * T::kVec;
            if (i >= 0 && i + T::kVec <= vocab)
                bits[n] = *reinterpret_cast<const uint4*>(row + i);
        }
    }
    // f(logit as it is, index, number of it) of each loaded one; minus infinity outside the row.
    template <class F>
    __device__ __forceinline__ void each(const typename T::Bits* row, int vocab, int unit, F f) const {
        const int first = start(row, unit);
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int i = first + n * kWave * T::kVec;
            float v[T::kVec];
            if (i >= 0 && i + T::kVec <= vocab) {
                T::unpack(bits[n], v);
            } else {
#pragma unroll
                for (int e = 0; e < T::kVec; ++e)
                    v[e] = i + e >= 0 && i + e < vocab ? T::load(row + i + e) : -__builtin_inff();
            }
#pragma unroll
            for (int e = 0; e < T::kVec; ++e) f(v[e], i + e, n * T::kVec + e);
        }
    }
};

template <class T>
int units_of(int vocab) {
    const int most_skew = 16 / static_cast<int>(sizeof(typename T::Bits)) - 1;
    return (vocab + most_skew + Unit<T>::kSize - 1) / Unit<T>::kSize;
}

// Units `first`, first + step, ... of a row that `want` names, the next one's loads in flight.
template <class T, class Want, class F>
__device__ __forceinline__ void each_unit(const typename T::Bits* row, int vocab, int first, int step,
                                          int units, Want want, F f) {
    auto next = [&](int u) {
        while (u < units && !want(u)) u += step;
        return u;
    };
    Unit<T> now, ahead;
    int u = next(first);
    if (u < units) now.load(row, vocab, u);
    while (u < units) {
        const int v = next(u + step);
        if (v < units) ahead.load(row, vocab, v);
        f(now, u);
        now = ahead;
        u = v;
    }
}

// A logit's bin below `top`.
__device__ __forceinline__ int bin_of(float l, float top, float bins) {
    return static_cast<int>(__builtin_fminf((top - l) * bins, kBins - 1.0f));
}

// A row's least logits but minus infinity: of those from kMask on, and of the parts that have
// none of these.
struct Lows {
    float near = __builtin_inff(), deep = __builtin_inff();

    __device__ __forceinline__ void add(float low) {  // a part's
        near = __builtin_fminf(near, low < kMask ? __builtin_inff() : low);
        deep = __builtin_fminf(deep, low);
    }
    __device__ __forceinline__ float of(float top) const { return top < kMask ? deep : near; }
};

// The largest logit of a unit, the same for all, and to a lane's `low` the least of its own.
template <class T>
__device__ __forceinline__ float unit_peak(const Unit<T>& x, const typename T::Bits* row, int vocab, int u,
                                           Lows& low) {
    float peak = -__builtin_inff();
    x.each(row, vocab, u, [&](float l, int, int) {
        peak = __builtin_fmaxf(peak, l);
        low.near = __builtin_fminf(low.near, l < kMask ? __builtin_inff() : l);
    });
    peak = from_lane(wave_scan(peak, -__builtin_inff(), Max()), kWave - 1);
    if (peak < kMask)
        x.each(row, vocab, u, [&](float l, int, int) {
            low.deep = __builtin_fminf(low.deep, l == -__builtin_inff() ? __builtin_inff() : l);
        });
    return peak;
}

// The least logit whose weight is not below e^-64, and no infinite one.
__device__ __forceinline__ float cut_of(float top, double t) {
    return __builtin_fmaxf(static_cast<float>(top - 64.0 * t), -0x1.fffffep127f);
}

// The bins of a row whose largest logit is `top`; false if bins do not fit it.  What is below
// kMask has no part in the range, unless all of the row is: masks of -1e9 would leave bins as wide
// as they get.
__device__ __forceinline__ bool fit_bins(Settings& s, float top, float low) {
    // bins below an infinite logit have no width
    if (__builtin_isinf(top)) return false;
    // differences of logits that have weights must not overflow
    if (__builtin_isinf(top - cut_of(top, s.t))) return false;
    // nor the bins.  A logit of 2^-80 or more is 2^-104 and more from any other: below a
    // temperature of 2^-114 the others have no weight.
    if (s.t < 0x1p-114) {
        if (__builtin_fabsf(top) < 0x1p-80f) return false;
        s.t = 0x1p-114;
        s.per = 0x1p114 * kPerUnit;
    }
    const float per = static_cast<float>(s.per);
    s.bins = __builtin_fmaxf(per * 0x1.62e42ep-1f, 0x1p-110f);  // ln 2: 64 a temperature
    s.bins = __builtin_fmaxf(s.bins, __builtin_fminf((kBins - 1) / (top - low), 0x1p40f));
    s.octaves = static_cast<uint32_t>(per / s.bins * 0x1p14f);
    return true;
}

// The power of two that brings a bin's weights to [0.49, 1.0001].
__device__ __forceinline__ uint32_t octaves_of(int bin, const Settings& s) {
    return __umul24(static_cast<uint32_t>(bin), s.octaves);  // 2^-20 of one
}

// A bin's sum of whole numbers as a weight.
__device__ __forceinline__ double mass_of(unsigned long long sum, int bin, const Settings& s) {
    return __builtin_ldexp(static_cast<double>(sum), -s.bits - static_cast<int>(octaves_of(bin, s) >> 20));
}

// Adds a unit to a histogram in LDS; `cut`: below it (and for a NaN) a weight counts as 0.
template <class T, bool kCount>
__device__ __forceinline__ void add_unit(const Unit<T>& x, const typename T::Bits* row, int vocab, int u,
                                         const Settings& s, float top, float cut, const double* powers,
                                         unsigned long long* mass, int* count) {
    x.each(row, vocab, u, [&](float l, int, int) {
        const double y = (static_cast<double>(l) - static_cast<double>(top)) * s.per;
        const int b = bin_of(l, top, s.bins);
        const unsigned long long m = fixed(power_of(y, octaves_of(b, s) & 0xfff00000u, powers), s.one);
        if (l >= cut) atomicAdd(&mass[b], m);
        if (kCount && l > -__builtin_inff()) atomicAdd(&count[b], 1);
    });
}

// Few rows: units over blocks.  First their largest logits (1 row of 128256 2.0 us, 32 rows
// 4.2) ...
template <class T>
__global__ __launch_bounds__(kSplitBlock) void sample_peaks_kernel(SampleArgs g, SampleWork w) {
    const int row = blockIdx.y, tid = threadIdx.x;
    const int u = blockIdx.x * (kSplitBlock / kWave) + tid / kWave;
    const typename T::Bits* logits = static_cast<const typename T::Bits*>(g.logits) + row * g.stride;
    Unit<T> x;
    if (u < w.units) x.load(logits, g.vocab, u);
    for (int b = blockIdx.x * kSplitBlock + tid; b < kBins; b += gridDim.x * kSplitBlock) {
        w.mass[static_cast<long>(row) * kBins + b] = 0;
        w.count[static_cast<long>(row) * kBins + b] = 0;
    }
    if (blockIdx.x == 0 && tid == 0) {
        w.listed[row] = 0;
        w.done[row] = 0;
    }
    if (u >= w.units) return;
    Lows lows;
    const float peak = unit_peak<T>(x, logits, g.vocab, u, lows);
    const float low = from_lane(wave_scan(lows.of(peak), __builtin_inff(), Min()), kWave - 1);
    if (tid % kWave == 0) {
        w.peaks[static_cast<long>(row) * w.units + u] = peak;
        w.lows[static_cast<long>(row) * w.units + u] = low;
    }
}

// ... then the histogram, added up in LDS and from there in memory (5.9 and 14.5 us: clearing,
// the float64 weights, and additions in memory past L2) ...
template <class T>
__global__ __launch_bounds__(kSplitBlock) void sample_bins_kernel(SampleArgs g, SampleWork w) {
    __shared__ unsigned long long mass[kBins];
    __shared__ int count[kBins];
    __shared__ double powers[64];
    __shared__ float part[3][kSplitBlock / kWave];
    constexpr int kTogether = kSplitBlock / kWave;
    const int row = blockIdx.y, tid = threadIdx.x;
    const typename T::Bits* logits = static_cast<const typename T::Bits*>(g.logits) + row * g.stride;
    Settings s = settings_of(g, row);
    const bool by_count = s.k < g.vocab;
    fill_powers(powers);
    for (int b = tid; b < kBins; b += kSplitBlock) {
        mass[b] = 0;
        if (by_count) count[b] = 0;
    }
    float top = -__builtin_inff();
    Lows lows;
    for (int i = tid; i < w.units; i += kSplitBlock) {
        top = __builtin_fmaxf(top, w.peaks[static_cast<long>(row) * w.units + i]);
        lows.add(w.lows[static_cast<long>(row) * w.units + i]);
    }
    top = wave_scan(top, -__builtin_inff(), Max());
    lows.near = wave_scan(lows.near, __builtin_inff(), Min());
    lows.deep = wave_scan(lows.deep, __builtin_inff(), Min());
    if (tid % kWave == kWave - 1) {
        part[0][tid / kWave] = top;
        part[1][tid / kWave] = lows.near;
        part[2][tid / kWave] = lows.deep;
    }
    __syncthreads();
    top = part[0][0];
    lows = {part[1][0], part[2][0]};
    for (int i = 1; i < kTogether; ++i) {
        top = __builtin_fmaxf(top, part[0][i]);
        lows.near = __builtin_fminf(lows.near, part[1][i]);
        lows.deep = __builtin_fminf(lows.deep, part[2][i]);
    }
    const float low = lows.of(top);
    if (!fit_bins(s, top, low)) return;
    const float cut = cut_of(top, s.t);
    each_unit<T>(logits, g.vocab, blockIdx.x * kTogether + tid / kWave, gridDim.x * kTogether, w.units,
                 [](int) { return true; }, [&](const Unit<T>& x, int u) {
                     if (by_count)
                         add_unit<T, true>(x, logits, g.vocab, u, s, top, cut, powers, mass, count);
                     else
                         add_unit<T, false>(x, logits, g.vocab, u, s, top, cut, powers, mass, count);
                 });
    __syncthreads();
    for (int b = tid; b < kBins; b += kSplitBlock) {
        if (mass[b])
            __hip_atomic_fetch_add(&w.mass[static_cast<long>(row) * kBins + b], mass[b], __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
        if (by_count && count[b])
            __hip_atomic_fetch_add(&w.count[static_cast<long>(row) * kBins + b], count[b], __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
    }
}

// Sorts list[0, n) ascending, n <= kRow * kEach; a thread holds kEach neighbours.  Pairs at
// doubling distances: within a thread, within a wave by lane moves, and only pairs of
// different waves through LDS.
template <int kEach>
__device__ __forceinline__ void sort_list(unsigned long long* list, int n) {
    const int tid = threadIdx.x;
    int size = 2 * kEach;
    while (size < n) size *= 2;
    const bool active = tid / kWave * kWave * kEach < size;  // whole waves
    uint64_t v[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) v[e] = tid * kEach + e < n ? list[tid * kEach + e] : ~0ull;
    auto keep = [](uint64_t& a, uint64_t o, bool smaller) { a = (o < a) == smaller ? o : a; };
    for (int k = 2; k <= size; k *= 2) {
        for (int d = k / 2; d >= kEach; d /= 2) {
            const int lanes = d / kEach;
            const bool smaller = ((tid * kEach & d) == 0) == ((tid * kEach & k) == 0);
            if (lanes >= kWave) {
                __syncthreads();
                if (active)
#pragma unroll
                    for (int e = 0; e < kEach; ++e) list[tid * kEach + e] = v[e];
                __syncthreads();
                if (active)
#pragma unroll
                    for (int e = 0; e < kEach; ++e)
                        keep(v[e], list[(tid ^ lanes) * kEach + e], smaller);
            } else if (active) {
#pragma unroll
                for (int e = 0; e < kEach; ++e) keep(v[e], lane_xor(v[e], lanes), smaller);
            }
        }
        if constexpr (kEach > 1) {
#pragma unroll
            for (int d = kEach / 2; d > 0; d /= 2) {
                if (d >= k) continue;
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    if (e & d) continue;
                    const bool up = ((tid * kEach + e) & k) == 0;
                    const uint64_t a = v[e], b = v[e + d];
                    if ((b < a) == up) {
                        v[e] = b;
                        v[e + d] = a;
                    }
                }
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        if (tid * kEach + e < n) list[tid * kEach + e] = v[e];
    __syncthreads();
}

// ... and the token of a row (11.8 and 25.4 us: a chain of dependent steps, a barrier each, and
// the fetch of their code).  kWhole: all of it by this block; else from the histogram in memory,
// the tokens in question gathered by w.parts blocks.
template <class T, bool kWhole>
__global__ __launch_bounds__(kRow, 4) void sample_pick_kernel(SampleArgs g, SampleWork w) {
    __shared__ union {
        unsigned long long fixed[kBins];
        double before[kBins + 1];  // before each bin, and of all
    } masses;
    double* const mass = masses.before;
    __shared__ int count[kBins + 1];
    __shared__ union {
        unsigned long long list[kList];  // ~key, index: ascending in the order
        Hist hist;
    } u;
    __shared__ float own_peaks[kWhole ? kPeaks : 1];
    __shared__ double powers[64];
    __shared__ union {
        float f[kWaves];
        int i[kWaves];
        double d[kWaves];
    } part;
    __shared__ struct {
        double mass[kWaves];
        int count[kWaves];
    } sums;
    __shared__ uint32_t marked[kBins / 32], marked_parts[kBins / 32];
    __shared__ int slots[kBins / 32];  // marked bins before each word
    __shared__ int bin_at[kSplitBins + 1];  // and the bin of each
    __shared__ double gap_mass[2][kSplitBins + 1];  // between marked bins: from, to
    __shared__ int gap_count[2][kSplitBins + 1];
    __shared__ int listed, found[5], heaviest_bin, base;
    __shared__ double cut_mass;
    __shared__ float spans[4][2];
    const int row = kWhole ? blockIdx.x : blockIdx.y, q = kWhole ? 0 : blockIdx.x;
    const int tid = threadIdx.x;
    const int lane = tid % kWave, wave = tid / kWave, own = tid * kOwn;
    const typename T::Bits* logits = static_cast<const typename T::Bits*>(g.logits) + row * g.stride;
    const float* peaks = kWhole ? own_peaks : w.peaks + static_cast<long>(row) * w.units;
    Settings s = settings_of(g, row);
    const bool by_count = s.k < g.vocab;
    fill_powers(powers);
    if (tid < 5) found[tid] = kBins;
    if (tid == 5) listed = 0;
    if (tid == 6) heaviest_bin = 0;
    auto all_units = [](int) { return true; };
    float top = -__builtin_inff();
    Lows lows;
    if constexpr (kWhole) {
        each_unit<T>(logits, g.vocab, wave, kWaves, w.units, all_units, [&](const Unit<T>& x, int u) {
            const float peak = unit_peak<T>(x, logits, g.vocab, u, lows);
            if (lane == 0 && u < kPeaks) own_peaks[u] = peak;
            top = __builtin_fmaxf(top, peak);
        });
    } else {
        for (int i = tid; i < w.units; i += kRow) {
            top = __builtin_fmaxf(top, peaks[i]);
            lows.add(w.lows[static_cast<long>(row) * w.units + i]);
        }
    }
    top = block_reduce(top, -__builtin_inff(), part.f, Max());
    const float low = block_reduce(lows.of(top), __builtin_inff(), part.f, Min());
    if (top == -__builtin_inff()) {
        if (q == 0 && tid == 0) {
            g.tokens[row] = -1;
            if (g.logprobs) g.logprobs[row] = top;
        }
        return;
    }
    if (!fit_bins(s, top, low)) {
        if (q == 0) sample_row<T>(g, row, s, top, powers, u.hist);
        return;
    }
    // kOwn neighbouring bins a thread
    double mine[kOwn];
    int mine_count[kOwn] = {};
    if constexpr (kWhole) {
        for (int b = tid; b < kBins; b += kRow) {
            masses.fixed[b] = 0;
            if (by_count) count[b] = 0;
        }
        __syncthreads();
        const float cut = cut_of(top, s.t);
        each_unit<T>(logits, g.vocab, wave, kWaves, w.units, all_units, [&](const Unit<T>& x, int u) {
            if (by_count)
                add_unit<T, true>(x, logits, g.vocab, u, s, top, cut, powers, masses.fixed, count);
            else
                add_unit<T, false>(x, logits, g.vocab, u, s, top, cut, powers, masses.fixed, count);
        });
        __syncthreads();
    }
#pragma unroll
    for (int h = 0; h < kOwn; ++h) {
        const long at = static_cast<long>(row) * kBins + own + h;
        mine[h] = mass_of(kWhole ? masses.fixed[own + h] : w.mass[at], own + h, s);
        if (by_count) mine_count[h] = kWhole ? count[own + h] : w.count[at];
    }
    // A bin's place among the marked ones, once they are split.
    int parts_of_bin = 0;  // 0: bins are not split
    auto place_of = [&](float y) {  // y: bins below the largest logit
        const int b = static_cast<int>(__builtin_fminf(y, kBins - 1.0f));
        if (parts_of_bin == 0) return b;
        const uint32_t below = marked[b / 32] & ((1u << (b % 32)) - 1);
        const int slot = slots[b / 32] + __popc(below), first = slot * parts_of_bin;
        if (!(marked[b / 32] >> (b % 32) & 1)) return first;
        const int part = static_cast<int>(__builtin_fminf(y - b, 1.0f) * (parts_of_bin - 1));
        return first + 1 + min(part, parts_of_bin - 2);
    };
    double total;
    int total_count;
    auto add_up = [&]() {  // mine[], mine_count[] -> mass[], count[]
        double sum = 0.0;
        int sum_count = 0;
#pragma unroll
        for (int h = 0; h < kOwn; ++h) {
            sum += mine[h];
            sum_count += mine_count[h];
        }
        BlockScan<double> m;
        BlockScan<int> c;
        m.before(sum, sums.mass);
        c.before(sum_count, sums.count);
        __syncthreads();
        sum = m.after(sums.mass, &total);
        sum_count = c.after(sums.count, &total_count);
#pragma unroll
        for (int h = 0; h < kOwn; ++h) {
            mass[own + h] = sum;
            count[own + h] = sum_count;
            sum += mine[h];
            sum_count += mine_count[h];
        }
        if (tid == 0) {
            mass[kBins] = total;
            count[kBins] = total_count;
        }
        __syncthreads();
    };
    // The bins in question.  The bounds of a sum that a bin leaves open give a first and a
    // last bin, a little widened: sums over bins and over tokens round differently.
    double end[kOwn], k_mass = 0.0;
    int k_bin = 0, p_bin, marks, to;  // marks: spans of bins in question; to: the last one
    constexpr float kLowest = -0x1.fffffep127f;
    uint32_t my_marks;  // word tid of the marks
    auto decide = [&]() {
        const double less = 1.0 - 0x1p-36, more = 1.0 + 0x1p-36;
        int heavy = -1;
        auto find = [&](int which, auto holds) {  // the first bin of which it holds
            int first = kBins;
#pragma unroll
            for (int h = kOwn - 1; h >= 0; --h)
                if (holds(h)) first = own + h;
            const unsigned long long set = __ballot(first < kBins);
            if (set) {
                first = from_lane(first, __ffsll(set) - 1);
                if (lane == 0) atomicMin(&found[which], first);
            }
        };
#pragma unroll
        for (int h = 0; h < kOwn; ++h) {
            end[h] = mass[own + h + 1];
            if (mine[h] > 0.0) heavy = own + h;
        }
        const unsigned long long heavies = __ballot(heavy >= 0);
        if (heavies) {
            heavy = from_lane(heavy, 63 - __clzll(heavies));
            if (lane == 0) atomicMax(&heaviest_bin, heavy);
        }
        if (by_count) find(0, [&](int h) { return count[own + h + 1] >= s.k; });
        __syncthreads();
        // bins behind the last one with a weight need no order: whatever is kept of them
        const int heaviest = heaviest_bin;
        double low = total, upper = total;  // bounds of what top-k keeps
        if (parts_of_bin && k_bin == kBins) {
            // where top-k ends with a bin that is not marked, the parts do not show it
            low = upper = k_mass;
        } else if (k_bin = kBins; by_count && s.k < total_count && found[0] <= heaviest) {
            k_bin = found[0];
            low = upper = mass[k_bin + 1];
            if (count[k_bin + 1] == s.k)
                k_bin = kBins;  // ends with the bin
            else
                low = mass[k_bin];
        }
        k_mass = upper;  // of top-k, where no bin is in question
        marks = 0;
        to = -1;
        my_marks = 0;
        auto mark = [&](int a, int b) {
            a = max(a, 0);
            b = min(b, heaviest);
            if (a > b) return;
            // as bounds of the logits, a little widened; minus infinity is in none
            if (tid == 0) {
                spans[marks][0] = top - a / s.bins * 0.9999f;
                spans[marks][1] = b < kBins - 1 ? __builtin_fmaxf(top - (b + 1) / s.bins * 1.0001f, kLowest) : kLowest;
            }
            ++marks;
            to = max(to, b);
            if (tid >= a / 32 && tid <= b / 32) {
                uint32_t bits = ~0u;
                if (tid == a / 32) bits &= ~0u << (a % 32);
                if (tid == b / 32) bits &= ~0u >> (31 - b % 32);
                my_marks |= bits;
            }
        };
        if (k_bin < kBins) mark(k_bin, k_bin);
        if (s.top_p < 1.0) {
            find(1, [&](int h) { return end[h] >= s.top_p * low * less; });
            find(2, [&](int h) { return end[h] >= s.top_p * upper * more; });
            __syncthreads();
            const int a = min(found[1], heaviest), b = min(found[2], heaviest);
            mark(a, b);
            low = __builtin_fmin(low, s.top_p * low * less);
            upper = __builtin_fmin(upper, mass[b + 1]);
        }
        p_bin = kBins;  // the last bin that min-p may keep a part of
        if (s.min_p > 0.0) {
            const double x = -log(s.min_p) * s.t * s.bins;
            const double off = 1e-6 + 3e-7 * x;  // a logit's place among the bins is float32
            const int first = place_of(static_cast<float>(__builtin_fmax(x - off, 0.0)));
            p_bin = place_of(static_cast<float>(x + off));
            mark(first, p_bin);
            low = __builtin_fmin(low, mass[first]);
            upper = __builtin_fmin(upper, mass[p_bin + 1]);
        }
        low = __builtin_fmax(low, 1.0);  // the first token stays
        find(3, [&](int h) { return end[h] > s.u * low * less; });
        find(4, [&](int h) { return end[h] > s.u * upper * more; });
        __syncthreads();
        mark(min(found[3], heaviest), min(found[4], heaviest));
    };
    add_up();
    decide();
    if (tid < kBins / 32) marked[tid] = my_marks;
    __syncthreads();
    // their tokens: by bounds of the logits, then by their bins
    each_unit<T>(
        logits, g.vocab, q * kWaves + wave, w.parts * kWaves, w.units,
        [&](int u) { return (kWhole && u >= kPeaks) || bin_of(peaks[u], top, s.bins) <= to; },
        [&](const Unit<T>& x, int unit) {
            uint32_t near = 0;
            for (int m = 0; m < marks; ++m) {
                const float above = spans[m][0], below = spans[m][1];
                x.each(logits, g.vocab, unit, [&](float l, int, int e) {
                    near |= static_cast<uint32_t>(l >= below && l <= above) << e;
                });
            }
            const int start = Unit<T>::start(logits, unit);
            while (__any(near != 0)) {  // a logit of each lane that has one, read again
                const int e = __ffs(near) - 1, i = start + e / T::kVec * (kWave * T::kVec) + e % T::kVec;
                float l = 0.0f;
                bool hit = near != 0;
                if (hit) {
                    l = clean(T::load(logits + i));
                    const int b = bin_of(l, top, s.bins);
                    hit = marked[b / 32] >> (b % 32) & 1;
                }
                near &= near - 1;
                const unsigned long long hits = __ballot(hit);
                if (hits == 0) continue;
                int at = 0;
                if (lane == 0) at = atomicAdd(&listed, static_cast<int>(__popcll(hits)));
                at = from_lane(at, 0) + __popcll(hits & ((1ull << lane) - 1));
                if (hit && at < kList)
                    u.list[at] = static_cast<unsigned long long>(~key_of(l)) << 32 | static_cast<uint32_t>(i);
            }
        });
    __syncthreads();
    int n = __builtin_amdgcn_readfirstlane(listed);
    if (!kWhole && w.parts > 1) {  // the block that is done last has all of them, and goes on
        // Stores and loads past the per-XCD L2s (agent scope), each block's stores done
        // (s_waitcnt) before it counts itself; a fence would write a whole L2 back: 90 us of
        // 150 at 32 rows of 128256.
        if (tid == 0)
            base = __hip_atomic_fetch_add(&w.listed[row], n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        const int to = base;
        for (int i = tid; i < min(n, kList); i += kRow)
            if (to + i < kList)
                __hip_atomic_store(&w.list[static_cast<long>(row) * kList + to + i], u.list[i],
                                   __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (tid == 0)
            base = __hip_atomic_fetch_add(&w.done[row], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (base != w.parts - 1) return;
        n = __builtin_amdgcn_readfirstlane(
            __hip_atomic_load(&w.listed[row], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        for (int i = tid; i < min(n, kList); i += kRow)
            u.list[i] = __hip_atomic_load(&w.list[static_cast<long>(row) * kList + i],
                                          __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
    }
    if (n > kList) {
        sample_row<T>(g, row, s, top, powers, u.hist);
        return;
    }
    if (n > kRow) {
        // The marked bins again, each split into as many parts as there is room for; what is
        // between them is a part of its own.  It leaves a token or two of each in question:
        // sorting 1200 took a fifth of the time of 512 flat rows.
        const uint32_t word = marked[lane];
        const int own_bits = __popc(word), words = wave_scan(own_bits, 0, Add());
        const int many = from_lane(words, kWave - 1);
        if (many <= kSplitBins) {
            if (wave == 0) slots[lane] = words - own_bits;
            __syncthreads();
            auto slot_of = [&](int b) {
                return slots[b / 32] + __popc(marked[b / 32] & ((1u << (b % 32)) - 1));
            };
            if (tid == 0) {
                gap_mass[0][0] = 0.0;
                gap_count[0][0] = 0;
                gap_mass[1][many] = total;
                gap_count[1][many] = total_count;
            }
#pragma unroll
            for (int h = 0; h < kOwn; ++h) {
                const int b = own + h;
                if (!(marked[b / 32] >> (b % 32) & 1)) continue;
                const int slot = slot_of(b);
                bin_at[slot] = b;
                gap_mass[1][slot] = mass[b];
                gap_count[1][slot] = count[b];
                gap_mass[0][slot + 1] = mass[b + 1];
                gap_count[0][slot + 1] = count[b + 1];
            }
            parts_of_bin = (kBins - 1) / many;
            __syncthreads();
            for (int b = tid; b < kBins; b += kRow) {
                masses.fixed[b] = 0;
                count[b] = 0;
            }
            if (tid < 5) found[tid] = kBins;
            if (tid == 5) listed = 0;
            if (tid == 6) heaviest_bin = 0;
            __syncthreads();
            uint64_t keep[kList / kRow];
#pragma unroll
            for (int e = 0; e < kList / kRow; ++e) {
                const int i = tid + e * kRow;
                if (i >= n) continue;
                keep[e] = u.list[i];
                const float l = from_key(~static_cast<uint32_t>(keep[e] >> 32));
                const int b = place_of((top - l) * s.bins);
                const int up = octaves_of(bin_of(l, top, s.bins), s) >> 20;
                const double weight = __builtin_ldexp(weight_of(l, top, s.per, powers), up);
                atomicAdd(&masses.fixed[b], fixed(weight, s.one));
                atomicAdd(&count[b], 1);
            }
            __syncthreads();
#pragma unroll
            for (int h = 0; h < kOwn; ++h) {
                const int b = own + h, slot = b / parts_of_bin;
                mine[h] = slot < many ? mass_of(masses.fixed[b], bin_at[slot], s) : 0.0;
                mine_count[h] = count[b];
                if (slot * parts_of_bin == b && slot <= many) {
                    mine[h] += gap_mass[1][slot] - gap_mass[0][slot];
                    mine_count[h] += gap_count[1][slot] - gap_count[0][slot];
                }
            }
            add_up();
            decide();
            if (tid < kBins / 32) marked_parts[tid] = my_marks;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kList / kRow; ++e) {
                if (tid + e * kRow >= n) continue;
                const float l = from_key(~static_cast<uint32_t>(keep[e] >> 32));
                const int b = place_of((top - l) * s.bins);
                if (marked_parts[b / 32] >> (b % 32) & 1) u.list[atomicAdd(&listed, 1)] = keep[e];
            }
            __syncthreads();
            n = __builtin_amdgcn_readfirstlane(listed);
        }
    }
    if (n <= kRow)
        sort_list<1>(u.list, n);
    else
        sort_list<kList / kRow>(u.list, n);
    // A thread's neighbours in the list, one mostly: f(place, weight, bin, weights before it
    // in the list).
    const int each = (n + kRow - 1) / kRow, first = min(tid * each, n), behind = min(first + each, n);
    auto place_at = [&](int i) {
        return place_of((top - from_key(~static_cast<uint32_t>(u.list[i] >> 32))) * s.bins);
    };
    auto each_listed = [&](double before, auto f) {
        for (int i = first; i < behind; ++i) {
            const float l = from_key(~static_cast<uint32_t>(u.list[i] >> 32));
            const double weight = weight_of(l, top, s.per, powers);
            f(i, weight, place_of((top - l) * s.bins), before);
            before += weight;
        }
        return before;
    };
    double list_mass;
    const double sum = block_scan(each_listed(0.0, [](int, double, int, double) {}), part.d, &list_mass);
    each_listed(sum, [&](int i, double, int b, double before) {
        if (i > 0 && place_at(i - 1) == b) return;
        mass[b] -= before;  // weights before the bin, less those before it in the list
        count[b] -= i;
    });
    if (tid == 0) cut_mass = k_mass;
    __syncthreads();
    each_listed(sum, [&](int i, double, int b, double before) {
        if (b == k_bin && count[b] + i == s.k) cut_mass = before + mass[b];  // the first that top-k leaves out
    });
    __syncthreads();
    double kept = cut_mass;
    const double bound = s.top_p < 1.0 ? s.top_p * kept : __builtin_inf();
    double least = kept;
#pragma unroll
    for (int h = 0; h < kOwn; ++h)
        if (end[h] >= bound || own + h == p_bin) least = __builtin_fmin(least, end[h]);
    each_listed(sum, [&](int, double weight, int b, double before) {
        before += mass[b];
        if (before >= bound || weight < s.min_p) least = __builtin_fmin(least, before);
    });
    kept = block_reduce(least, __builtin_inf(), part.d, Min());
    const double target = s.u * kept;
    int chosen = kList, last = -1;
    each_listed(sum, [&](int i, double weight, int b, double before) {
        before += mass[b];
        if (weight > 0.0 && before <= target) last = i;
        if (before + weight > target) chosen = min(chosen, i);
    });
    chosen = block_reduce(chosen, kList, part.i, Min());
    if (chosen == kList) {  // past them by a rounding: the last
        last = block_reduce(last, -1, part.i, Max());
        chosen = max(last, 0);
    }
    if (chosen < first || chosen >= behind) return;
    const unsigned long long token = u.list[chosen];
    g.tokens[row] = static_cast<int>(static_cast<uint32_t>(token));
    if (g.logprobs)
        g.logprobs[row] = static_cast<float>(
            log(weight_of(from_key(~static_cast<uint32_t>(token >> 32)), top, s.per, powers) / kept));
}

// Most rows that are split: the workspace is bounded.
constexpr int kSplitRows = 192;

// One block a row where rows fill the GPU, or are a few units: one launch and no trip through
// memory, where the split takes three.  top-k 50 and top-p 0.95, one block a row / split: rows
// of 16500 23 / 24 us for 32, 24 / 28 for 64; 32003 31 / 26 for 32, 31 / 37 for 96; 64000
// 49 / 46 for 128, 52 / 59 for 192; 128256 62 / 21 for 1, 82 / 66 for 128, 85 / 85 for 192.
bool sample_whole(int rows, int units) { return units <= 16 || rows > 2 * units || rows > kSplitRows; }

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// The workspace's parts for a number of rows; its size.
size_t sample_layout(int rows, int units, char* base, SampleWork* w) {
    const size_t n = rows < 1 ? 1 : rows < kSplitRows ? rows : kSplitRows;
    size_t at = 0;
    SampleWork none;
    SampleWork& t = w ? *w : none;
    auto take = [&](auto*& p, size_t count) {
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(base + at);
        at += align256(count * sizeof(*p));
    };
    take(t.peaks, n * units);
    take(t.lows, n * units);
    take(t.mass, n * kBins);
    take(t.count, n * kBins);
    take(t.list, n * kList);
    take(t.listed, n);
    take(t.done, n);
    return at;
}

// Of any type: 16-bit rows may begin 7 logits before a boundary.
size_t sample_workspace(int rows, int vocab) {
    return sample_layout(rows, units_of<Half<F16>>(vocab), nullptr, nullptr);
}

int check_rows(const char* fn, int rows, int vocab) {
    if (rows < 0 || vocab < 0) return invalid("%s: negative size", fn);
    if (rows > kMaxRows) return invalid("%s: %d rows, at most %d are possible", fn, rows, kMaxRows);
    if (vocab > kMaxVocab)
        return invalid("%s: a vocabulary of %d, at most %d is possible", fn, vocab, kMaxVocab);
    return 0;
}

int check_logits(const char* fn, const void* logits, long stride, int rows, int vocab, int size) {
    if (vocab < 1) return invalid("%s: a row needs a token", fn);
    if (!logits) return invalid("%s: null logits", fn);
    if (!aligned_to(logits, size)) return invalid("%s: logits must be %d-byte aligned", fn, size);
    if (rows > 1 && stride < vocab) return invalid("%s: rows overlap", fn);
    return 0;
}

int check_workspace(const char* fn, const void* ws, size_t size, size_t need) {
    if (!ws || size < need || !aligned_to(ws, 16))
        return invalid("%s: a 16-byte aligned workspace of %zu bytes is needed", fn, need);
    return 0;
}

template <class T>
int sample(const char* fn, const void* logits, long stride, const float* uniforms, int* tokens,
           float* logprobs, int rows, int vocab, const spb_sampling* set, void* ws, size_t size,
           void* stream) {
    clear_error();
    if (int e = check_rows(fn, rows, vocab)) return e;
    if (!set) return invalid("%s: null sampling", fn);
    if (!set->temperatures && !(set->temperature >= 0.0f))
        return invalid("%s: temperature must not be negative", fn);
    if (!set->top_ks && set->top_k < 0) return invalid("%s: top_k must not be negative", fn);
    if (!set->top_ps && !(set->top_p >= 0.0f && set->top_p <= 1.0f))
        return invalid("%s: top_p must be in [0, 1]", fn);
    if (!set->min_ps && !(set->min_p >= 0.0f && set->min_p <= 1.0f))
        return invalid("%s: min_p must be in [0, 1]", fn);
    if (rows == 0) return 0;
    if (int e = check_logits(fn, logits, stride, rows, vocab, sizeof(typename T::Bits))) return e;
    if (!uniforms || !tokens) return invalid("%s: null pointer", fn);
    const void* four[] = {uniforms, tokens, logprobs, set->temperatures, set->top_ks, set->top_ps,
                          set->min_ps};
    for (const void* p : four)
        if (!aligned_to(p, 4)) return invalid("%s: a vector is not 4-byte aligned", fn);
    if (int e = check_workspace(fn, ws, size, sample_workspace(rows, vocab))) return e;
    SampleArgs g{logits, stride, uniforms, tokens, logprobs, vocab, *set};
    SampleWork w{};
    w.units = units_of<T>(vocab);
    sample_layout(rows, w.units, static_cast<char*>(ws), &w);
    const hipStream_t st = as_stream(stream);
    if (sample_whole(rows, w.units)) {
        w.parts = 1;
        hipLaunchKernelGGL((sample_pick_kernel<T, true>), dim3(rows), dim3(kRow), 0, st, g, w);
        return launch_status(fn);
    }
    const int blocks = (w.units + kSplitBlock / kWave - 1) / (kSplitBlock / kWave);
    const int most = (w.units + kWaves - 1) / kWaves, fill = (256 + rows - 1) / rows;
    w.parts = fill < most ? fill : most;
    if (w.parts > 16) w.parts = 16;
    hipLaunchKernelGGL(sample_peaks_kernel<T>, dim3(blocks, rows), dim3(kSplitBlock), 0, st, g, w);
    // Each block adds its bins to the row's: fewer blocks a row, fewer additions in memory.
    const int share = (512 + rows - 1) / rows;
    hipLaunchKernelGGL(sample_bins_kernel<T>, dim3(blocks < share ? blocks : share, rows),
                       dim3(kSplitBlock), 0, st, g, w);
    hipLaunchKernelGGL((sample_pick_kernel<T, false>), dim3(w.parts, rows), dim3(kRow), 0, st, g, w);
    return launch_status(fn);
}

// ---- log-probabilities --------------------------------------------------------------

struct LogprobArgs {
    const void* logits;
    long stride;
    const int* tokens;  // may be null
    float* logprobs;
    int* top_ids;
    float* top_logprobs;
    int vocab, top;
};

constexpr int kGroups = kRow;      // groups of a row's units whose largest logits are compared
constexpr int kCandidates = 4096;  // = kMaxTop lanes' largest logits

// A sum of exponentials: the largest logit, how many there are of it, and the exponentials of
// the others less it.  The largest are counted apart: beside a 1, weights of 1e-11 would lose
// digits, and a token with nearly all of the mass is told from them.
struct Sum {
    float top;
    int count;
    double rest;

    static __device__ __forceinline__ double less(float low, float high) {
        return __builtin_amdgcn_exp2f((low - high) * 0x1.715476p+0f);
    }
    // Before a unit with the largest logit `peak`.  In float64: a row that rises slowly comes here
    // for each unit, with the same difference each time, and 2048 float32 roundings to the same
    // side (2^24 tokens rising by 0.2) put a log-probability off by 6e-6.
    __device__ __forceinline__ void raise(float peak, int own) {
        if (!(peak > top)) return;
        if (top != -__builtin_inff()) rest = (rest + own) * exp(static_cast<double>(top) - peak);
        top = peak;
        count = 0;
    }
};

struct LogprobWork {
    Sum* sums;  // [rows][units]
    int units;
};

// Adds a unit to a wave's sum: top and count are the wave's, rest is each lane's.  Float32
// exponentials of float32 differences are off by (|difference| + 1) * 2^-23; 16 of them are
// added in float32, by pairs, and those in float64.
template <class T>
__device__ __forceinline__ float sum_unit(Sum& s, const Unit<T>& x, const typename T::Bits* row, int vocab,
                                          int u) {
    float peak = -__builtin_inff();
    x.each(row, vocab, u, [&](float l, int, int) { peak = __builtin_fmaxf(peak, l); });
    peak = from_lane(wave_scan(peak, -__builtin_inff(), Max()), kWave - 1);
    if (peak == -__builtin_inff()) return peak;
    s.raise(peak, threadIdx.x % kWave == 0 ? s.count : 0);
    const bool has = peak == s.top;
    float w[16];
    int equal = 0;
    x.each(row, vocab, u, [&](float l, int, int e) {
        l = clean(l);
        w[e] = __builtin_amdgcn_exp2f((l - s.top) * 0x1.715476p+0f);
        if (has) {
            w[e] = l == s.top ? 0.0f : w[e];
            equal += l == s.top;
        }
    });
#pragma unroll
    for (int d = 8; d > 0; d /= 2)
#pragma unroll
        for (int e = 0; e < d; ++e) w[e] += w[e + d];
    s.rest += w[0];
    if (has) s.count += from_lane(wave_scan(equal, 0, Add()), kWave - 1);
    return peak;
}

__device__ __forceinline__ unsigned long long rank_key(float l, int index) {
    return static_cast<unsigned long long>(~key_of(l)) << 32 | static_cast<uint32_t>(index);
}

// Few rows: a wave has a unit, and another kernel adds up.  1 row of 128256 2.2 us and 14.5 in
// the other (20 alternatives), 32 rows 3.8 and 10.6 (5).
template <class T>
__global__ __launch_bounds__(kSplitBlock) void logprob_units_kernel(LogprobArgs g, LogprobWork w) {
    const int row = blockIdx.y;
    const int u = blockIdx.x * (kSplitBlock / kWave) + static_cast<int>(threadIdx.x / kWave);
    if (u >= w.units) return;
    const typename T::Bits* logits = static_cast<const typename T::Bits*>(g.logits) + row * g.stride;
    Unit<T> x;
    x.load(logits, g.vocab, u);
    Sum s{-__builtin_inff(), 0, 0.0};
    sum_unit<T>(s, x, logits, g.vocab, u);
    s.rest = from_lane(wave_scan(s.rest, 0.0, Add()), kWave - 1);
    if (threadIdx.x % kWave == 0) w.sums[static_cast<long>(row) * w.units + u] = s;
}

// A row's log-probabilities, and its `top` likeliest tokens.  kWhole: all of it by this block;
// else from the units' sums.
//
// The likeliest are in the `top` groups of units with the largest logits (equal ones: the
// first), for any other group has `top` tokens before its own.  These groups are read again,
// and their tokens from the last of those logits on are sorted: a few more than `top`, mostly.
// Where they are many, the same is done with lanes for groups: at most 16 of each of `top` lanes
// are left.  They are many in a row in rising order, and wherever a row has fewer groups than
// alternatives are asked for (vocabularies up to 1024 (top - 1)), for then the groups say nothing:
// 20 of 16384 tokens take 67 us for 1 row, 70 for 256, of 20480 18 and 23; 64 of 32003 76 and 86.
//
// 2048 rows of 128256 float32 logits, 5 alternatives: 209 us for 1.05 GB, 5.0 TB/s, what a copy
// reaches; the row's few groups are read again from the caches.  1023 rows of 32003 bf16: 22.5 us,
// 2.9 TB/s: rows of 64 KB, whose start and end (launch, sums over the block) show.
template <class T, bool kWhole>
__global__ __launch_bounds__(kRow) void logprob_kernel(LogprobArgs g, LogprobWork w) {
    __shared__ uint32_t peaks[kGroups];
    __shared__ unsigned long long list[kCandidates];
    __shared__ union {
        float f[kWaves];
        int i[kWaves];
        double d[kWaves];
        unsigned long long u[kWaves];
    } part;
    __shared__ int chosen[kMaxTop], listed;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int token = g.tokens ? g.tokens[row] : 0;
    if (token < 0 || token >= g.vocab) return;
    const typename T::Bits* logits = static_cast<const typename T::Bits*>(g.logits) + row * g.stride;
    const float mine = clean(T::load(logits + token));
    const int size = (w.units + kGroups - 1) / kGroups, groups = (w.units + size - 1) / size;
    if (tid < groups) peaks[tid] = 0;
    if (tid == 0) listed = 0;
    __syncthreads();
    // a thread's part of the sum: in kWhole each wave's by its first lane, else some units'
    Sum s{-__builtin_inff(), 0, 0.0};
    auto peak_of = [&](int u, float peak) {
        if (!g.top) return;
        if (size == 1)
            peaks[u] = key_of(peak);
        else
            atomicMax(&peaks[u / size], key_of(peak));
    };
    if constexpr (kWhole) {
        each_unit<T>(logits, g.vocab, wave, kWaves, w.units, [](int) { return true; },
                     [&](const Unit<T>& x, int u) {
                         const float peak = sum_unit<T>(s, x, logits, g.vocab, u);
                         if (lane == 0) peak_of(u, peak);
                     });
        if (lane > 0) s.count = 0;
    } else {
        for (int u = tid; u < w.units; u += kRow) {
            const Sum o = w.sums[static_cast<long>(row) * w.units + u];
            peak_of(u, o.top);
            if (o.top == -__builtin_inff()) continue;
            s.raise(o.top, s.count);
            s.rest += o.top == s.top ? o.rest : (o.rest + o.count) * Sum::less(o.top, s.top);
            s.count += o.top == s.top ? o.count : 0;
        }
    }
    const float top = block_reduce(s.top, -__builtin_inff(), part.f, Max());
    double rest = 0.0;
    if (s.top != -__builtin_inff()) rest = s.top == top ? s.rest : (s.rest + s.count) * Sum::less(s.top, top);
    rest = block_reduce(rest, 0.0, part.d, Add());
    const int equal = block_reduce(s.top == top ? s.count : 0, 0, part.i, Add());
    auto logprob = [&](float l) {
        if (l == -__builtin_inff()) return l;
        return static_cast<float>((l == top ? 0.0 : static_cast<double>(l) - top) - log1p(rest + (equal - 1)));
    };
    if (tid == 0 && g.tokens) g.logprobs[row] = logprob(mine);
    if (g.top == 0) return;
    // the groups: a group's rank is the number of better ones
    const int many = min(g.top, groups);
    if (tid < groups) {
        const uint32_t key = peaks[tid];
        int rank = 0;
        for (int i = 0; i < groups; ++i) rank += peaks[i] > key || (peaks[i] == key && i < tid);
        if (rank < many) chosen[rank] = tid;
    }
    __syncthreads();
    const float bound = many < g.top ? -__builtin_inff() : from_key(peaks[chosen[many - 1]]);
    // f(unit's logits, index) for the units of the groups, a wave each
    auto each_chosen = [&](auto f) {
        for (int i = wave; i < many * size; i += kWaves) {
            const int u = chosen[i / size] * size + i % size;
            if (u >= w.units) continue;
            Unit<T> x;
            x.load(logits, g.vocab, u);
            f(x, u, i / size);
        }
    };
    auto gather = [&](float least, unsigned long long last) {
        each_chosen([&](const Unit<T>& x, int u, int) {
            uint32_t hits = 0;
            x.each(logits, g.vocab, u, [&](float l, int i, int e) {
                l = clean(l);
                const bool in = l >= least && i >= 0 && i < g.vocab && rank_key(l, i) <= last;
                hits |= static_cast<uint32_t>(in) << e;
            });
            const int own = __popc(hits), upto = wave_scan(own, 0, Add()), all = from_lane(upto, kWave - 1);
            if (all == 0) return;
            int at = 0;
            if (lane == 0) at = atomicAdd(&listed, all);
            at = from_lane(at, 0) + upto - own;
            x.each(logits, g.vocab, u, [&](float l, int i, int e) {
                if (!(hits >> e & 1)) return;
                if (at < kCandidates) list[at] = rank_key(clean(l), i);
                ++at;
            });
        });
        __syncthreads();
        return __builtin_amdgcn_readfirstlane(listed);
    };
    int n = gather(bound, ~0ull);
    if (n > kRow) {
        // the best of each of the groups' lanes, and of those the last that can be wanted
        __syncthreads();
        if (tid == 0) listed = 0;
        for (int i = tid; i < kMaxTop * kWave; i += kRow) list[i] = ~0ull;
        __syncthreads();
        each_chosen([&](const Unit<T>& x, int u, int c) {
            unsigned long long best = ~0ull;
            x.each(logits, g.vocab, u, [&](float l, int i, int) {
                if (i < 0 || i >= g.vocab) return;
                const unsigned long long k = rank_key(clean(l), i);
                best = k < best ? k : best;
            });
            atomicMin(&list[c * kWave + lane], best);
        });
        __syncthreads();
        sort_list<kCandidates / kRow>(list, many * kWave);
        const unsigned long long last = list[g.top - 1];
        __syncthreads();
        n = gather(-__builtin_inff(), last);
    }
    if (n > kCandidates) {
        // groups of many units (vocabularies of millions) in rising order: one after the other
        unsigned long long last = 0;
        for (int i = 0; i < g.top; ++i) {
            unsigned long long best = ~0ull;
            for (int j = tid; j < g.vocab; j += kRow) {
                const unsigned long long k = rank_key(clean(T::load(logits + j)), j);
                if ((i == 0 || k > last) && k < best) best = k;
            }
            last = block_reduce(best, ~0ull, part.u, Min());
            if (tid == 0) list[i] = last;
        }
        __syncthreads();
    } else if (n <= kRow) {
        sort_list<1>(list, n);
    } else {
        sort_list<kCandidates / kRow>(list, n);
    }
    if (tid < g.top) {
        const unsigned long long k = list[tid];
        g.top_ids[static_cast<long>(row) * g.top + tid] = static_cast<int>(static_cast<uint32_t>(k));
        g.top_logprobs[static_cast<long>(row) * g.top + tid] = logprob(from_key(~static_cast<uint32_t>(k >> 32)));
    }
}

size_t logprobs_layout(int rows, int units, char* base, LogprobWork* w) {
    const size_t n = rows < 1 ? 1 : rows < kSplitRows ? rows : kSplitRows;
    if (w) w->sums = reinterpret_cast<Sum*>(base);
    return align256(n * units * sizeof(Sum));
}

size_t logprobs_workspace(int rows, int vocab) {
    return logprobs_layout(rows, units_of<Half<F16>>(vocab), nullptr, nullptr);
}

// The same for log-probabilities: 32003 14.0 / 12.3 us for 96 rows, 14.3 / 14.5 for 192; 128256
// 30 / 14 for 1, 35 / 28 for 192.
bool logprobs_whole(int rows, int units) { return units <= 16 || rows > kSplitRows; }

int check_top(const char* fn, int top) {
    if (top < 0 || top > kMaxTop) return invalid("%s: top %d must be in [0, %d]", fn, top, kMaxTop);
    return 0;
}

template <class T>
int token_logprobs(const char* fn, const void* logits, long stride, const int* tokens,
                   float* logprobs, int* top_ids, float* top_logprobs, int rows, int vocab,
                   int top, void* ws, size_t size, void* stream) {
    clear_error();
    if (int e = check_rows(fn, rows, vocab)) return e;
    if (int e = check_top(fn, top)) return e;
    if (rows == 0) return 0;
    if (int e = check_logits(fn, logits, stride, rows, vocab, sizeof(typename T::Bits))) return e;
    if (top > vocab) return invalid("%s: top %d of a vocabulary of %d", fn, top, vocab);
    if ((tokens == nullptr) != (logprobs == nullptr))
        return invalid("%s: tokens and logprobs come together", fn);
    if (!tokens && !top) return invalid("%s: neither tokens nor alternatives", fn);
    if (top && (!top_ids || !top_logprobs)) return invalid("%s: null pointer", fn);
    const void* four[] = {tokens, logprobs, top_ids, top_logprobs};
    for (const void* p : four)
        if (!aligned_to(p, 4)) return invalid("%s: a vector is not 4-byte aligned", fn);
    if (int e = check_workspace(fn, ws, size, logprobs_workspace(rows, vocab))) return e;
    LogprobArgs g{logits, stride, tokens, logprobs, top_ids, top_logprobs, vocab, top};
    LogprobWork w{};
    w.units = units_of<T>(vocab);
    logprobs_layout(rows, w.units, static_cast<char*>(ws), &w);
    const hipStream_t st = as_stream(stream);
    if (logprobs_whole(rows, w.units)) {
        hipLaunchKernelGGL((logprob_kernel<T, true>), dim3(rows), dim3(kRow), 0, st, g, w);
        return launch_status(fn);
    }
    const int blocks = (w.units + kSplitBlock / kWave - 1) / (kSplitBlock / kWave);
    hipLaunchKernelGGL(logprob_units_kernel<T>, dim3(blocks, rows), dim3(kSplitBlock), 0, st, g, w);
    hipLaunchKernelGGL((logprob_kernel<T, false>), dim3(rows), dim3(kRow), 0, st, g, w);
    return launch_status(fn);
}

}  // namespace
}  // namespace spb

using namespace spb;

extern "C" {

size_t spb_sample_workspace_size(int rows, int vocab) {
    clear_error();
    return check_rows("spb_sample_workspace_size", rows, vocab) ? 0 : sample_workspace(rows, vocab);
}
int spb_sample_f32(const float* logits, long logits_stride, const float* uniforms, int* tokens,
                   float* logprobs, int rows, int vocab, const spb_sampling* sampling,
                   void* workspace, size_t workspace_size, spb_stream_t s) {
    return sample<F32>("spb_sample_f32", logits, logits_stride, uniforms, tokens, logprobs, rows,
                       vocab, sampling, workspace, workspace_size, s);
}
int spb_sample_f16(const uint16_t* logits, long logits_stride, const float* uniforms, int* tokens,
                   float* logprobs, int rows, int vocab, const spb_sampling* sampling,
                   void* workspace, size_t workspace_size, spb_stream_t s) {
    return sample<Half<F16>>("spb_sample_f16", logits, logits_stride, uniforms, tokens, logprobs,
                             rows, vocab, sampling, workspace, workspace_size, s);
}
int spb_sample_bf16(const uint16_t* logits, long logits_stride, const float* uniforms, int* tokens,
                    float* logprobs, int rows, int vocab, const spb_sampling* sampling,
                    void* workspace, size_t workspace_size, spb_stream_t s) {
    return sample<Half<BF16>>("spb_sample_bf16", logits, logits_stride, uniforms, tokens, logprobs,
                              rows, vocab, sampling, workspace, workspace_size, s);
}

size_t spb_token_logprobs_workspace_size(int rows, int vocab, int top) {
    clear_error();
    const char* fn = "spb_token_logprobs_workspace_size";
    return check_rows(fn, rows, vocab) || check_top(fn, top) ? 0 : logprobs_workspace(rows, vocab);
}
int spb_token_logprobs_f32(const float* logits, long logits_stride, const int* tokens,
                           float* logprobs, int* top_ids, float* top_logprobs, int rows,
                           int vocab, int top, void* workspace, size_t workspace_size,
                           spb_stream_t s) {
    return token_logprobs<F32>("spb_token_logprobs_f32", logits, logits_stride, tokens, logprobs,
                               top_ids, top_logprobs, rows, vocab, top, workspace, workspace_size,
                               s);
}
int spb_token_logprobs_f16(const uint16_t* logits, long logits_stride, const int* tokens,
                           float* logprobs, int* top_ids, float* top_logprobs, int rows,
                           int vocab, int top, void* workspace, size_t workspace_size,
                           spb_stream_t s) {
    return token_logprobs<Half<F16>>("spb_token_logprobs_f16", logits, logits_stride, tokens,
                                     logprobs, top_ids, top_logprobs, rows, vocab, top, workspace,
                                     workspace_size, s);
}
int spb_token_logprobs_bf16(const uint16_t* logits, long logits_stride, const int* tokens,
                            float* logprobs, int* top_ids, float* top_logprobs, int rows,
                            int vocab, int top, void* workspace, size_t workspace_size,
                            spb_stream_t s) {
    return token_logprobs<Half<BF16>>("spb_token_logprobs_bf16", logits, logits_stride, tokens,
                                      logprobs, top_ids, top_logprobs, rows, vocab, top, workspace,
                                      workspace_size, s);
}

}  // extern "C"
