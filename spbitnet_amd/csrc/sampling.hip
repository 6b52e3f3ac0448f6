// sampling.hip -- what follows a batch's logits: the next token of each row under
// its request's temperature, top-k, top-p and min-p, from given random numbers, and
// the log-probabilities of tokens with the best alternatives of each row.
//
// The tokens of a row stand in the order of falling logits, equal ones by index, with
// weights w = exp((l - max) / temperature); NaN counts as minus infinity.  Each of the
// three filters keeps a first part of that order, so the kept tokens are the first n,
// and the token taken is the first whose weight with those before it passes u times
// their sum M.  All that is looked for is a place in one order where a sum of counts
// or weights passes a bound: a selection by digits of the logits' bits, without a sort.
//
// Sums of weights decide between neighbours among up to 2^24 tokens, so they are held
// to ~2^-46 of the largest weight and do not depend on the order of adding: weights are
// computed in float64 and added as 64-bit whole numbers.
#include "common.hpp"
#include "paged.hpp"
#include "spbitnet_amd.h"

namespace spb {
namespace {

constexpr int kMaxVocab = 1 << 24;
constexpr int kMaxRows = 1 << 20;
constexpr int kMaxTop = 64;
constexpr int kRow = 1024;  // threads on one row
constexpr int kWaves = kRow / kWave;

struct F32 {
    using Bits = float;
    static __device__ __forceinline__ float load(const Bits* p) { return *p; }
};
template <class T>
struct Half {
    using Bits = uint16_t;
    static __device__ __forceinline__ float load(const Bits* p) { return T::to_float(*p); }
};

// A logit with NaN as minus infinity and one zero.
__device__ __forceinline__ float clean(float v) {
    return v != v ? -__builtin_inff() : v + 0.0f;
}

// Order of the logits as unsigned numbers.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_key(uint32_t k) {
    return __builtin_bit_cast(float, k >> 31 ? k & 0x7fffffffu : ~k);
}

// ---- reductions over a block of kRow threads; every thread gets the result ----

template <class V, class Op>
__device__ __forceinline__ V block_reduce(V v, V* part, Op op) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = op(v, __shfl_xor(v, off, kWave));
    __syncthreads();
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    V r = part[0];
    for (int w = 1; w < kWaves; ++w) r = op(r, part[w]);
    return r;
}

// ---- sampling -------------------------------------------------------------------

struct SampleArgs {
    const void* logits;
    long stride;
    const float* uniforms;
    int* tokens;
    float* logprobs;  // may be null
    int rows, vocab;
    spb_sampling set;
};

// A row's settings, with what is off or out of range taken care of.
struct Settings {
    double inv_t, u;
    double top_p, min_p;  // 1 and 0: off
    int k;                // vocab: off
};

__device__ __forceinline__ Settings settings_of(const SampleArgs& g, int row) {
    Settings s;
    float t = g.set.temperatures ? g.set.temperatures[row] : g.set.temperature;
    int k = g.set.top_ks ? g.set.top_ks[row] : g.set.top_k;
    float p = g.set.top_ps ? g.set.top_ps[row] : g.set.top_p;
    float m = g.set.min_ps ? g.set.min_ps[row] : g.set.min_p;
    if (k <= 0 || k > g.vocab) k = g.vocab;
    if (!(t > 0.0f)) {  // greedy: the first token of the order
        t = 1.0f;
        k = 1;
    }
    if (p <= 0.0f) k = 1;
    s.top_p = p < 1.0f && p > 0.0f ? p : 1.0;
    s.min_p = m > 0.0f ? (m < 1.0f ? m : 1.0) : 0.0;
    s.k = k;
    s.inv_t = 1.0 / static_cast<double>(t);
    const float u = g.uniforms[row];
    s.u = u > 0.0f ? (u < 1.0f ? u : 0x1.fffffep-1) : 0.0;
    return s;
}

// Weight of a logit (not minus infinity) below or at the maximum.
__device__ __forceinline__ double weight_of(float l, float top, double inv_t) {
    if (l == top) return 1.0;
    const double d = (static_cast<double>(l) - static_cast<double>(top)) * inv_t;
    return d > -64.0 ? exp(d) : 0.0;  // 2^24 weights below e^-64 are nothing beside the first, 1
}

// Where a sum of counts or weights along the order passes a bound: the logit there, how
// many of that logit stand before the place, and the sums before it.
struct Place {
    uint32_t key;
    int before_ties;    // tokens of that logit before the place
    long long count;    // tokens before the place
    double mass;        // weights before the place
};

struct Hist {
    unsigned long long mass[256];
    int count[256];
    int digit;
    long long before_count;
    unsigned long long before_mass;
};

template <class T>
struct Row {
    const typename T::Bits* l;
    int vocab;
    float top;
    double inv_t;
    double one;   // 2^52 / unit: added to a weight, leaves it as a multiple of 1 / unit
    double unit;  // weights are whole numbers of 1 / unit; a row of ones stays below 2^63
};

__device__ __forceinline__ unsigned long long fixed(double w, double one) {
    return __builtin_bit_cast(unsigned long long, w + one) -
           __builtin_bit_cast(unsigned long long, one);
}

// The first place of the order whose token ends past the bound: by count, the token of
// rank `rank` (so the sums before it are those of the first `rank` tokens); by mass, the
// first token whose weight with those before it is > bound.  Four digits of the key, each
// a histogram of counts and weights of the tokens that share the digits before it.
template <bool kMass, class T>
__device__ Place select(const Row<T>& r, long long rank, double bound, Hist& h) {
    uint32_t prefix = 0;
    long long count = 0;
    unsigned long long mass = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) {
            h.mass[threadIdx.x] = 0;
            h.count[threadIdx.x] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < r.vocab; i += kRow) {
            const float l = clean(T::load(r.l + i));
            if (l == -__builtin_inff()) continue;
            const uint32_t key = key_of(l);
            if (shift < 24 && (key >> (shift + 8)) != (prefix >> (shift + 8))) continue;
            const int d = key >> shift & 255;
            atomicAdd(&h.count[d], 1);
            atomicAdd(&h.mass[d], fixed(weight_of(l, r.top, r.inv_t), r.one));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int last = -1, d = 255;
            long long c = count, lc = 0;
            unsigned long long m = mass, lm = 0;
            for (; d >= 0; --d) {
                if (!h.count[d]) continue;
                if (!kMass || h.mass[d]) {  // past every weight: the last token that has one
                    last = d;
                    lc = c;
                    lm = m;
                }
                c += h.count[d];
                m += h.mass[d];
                if (kMass ? static_cast<double>(m) > bound * r.unit : c > rank) break;
            }
            h.digit = last;
            h.before_count = lc;
            h.before_mass = lm;
        }
        __syncthreads();
        if (h.digit < 0) break;
        prefix |= static_cast<uint32_t>(h.digit) << shift;
        count = h.before_count;
        mass = h.before_mass;
    }
    Place p;
    p.key = prefix;
    const int ties = h.count[prefix & 255];
    const double w = weight_of(from_key(prefix), r.top, r.inv_t);
    p.mass = static_cast<double>(mass) / r.unit;
    long long in = kMass ? static_cast<long long>((bound - p.mass) / w) : rank - count;
    in = in < 0 ? 0 : in >= ties ? ties - 1 : in;
    p.before_ties = static_cast<int>(in);
    p.count = count + in;
    p.mass += in * w;
    return p;
}

// One block a row, everything from the row itself: right for any row, at up to a dozen
// readings of it.
template <class T>
__global__ __launch_bounds__(kRow) void sample_row_kernel(SampleArgs g) {
    __shared__ Hist h;
    __shared__ union {
        float f[kWaves];
        int i[kWaves];
        unsigned long long u[kWaves];
    } part;
    const int row = blockIdx.x;
    const Settings s = settings_of(g, row);
    Row<T> r;
    r.l = static_cast<const typename T::Bits*>(g.logits) + row * g.stride;
    r.vocab = g.vocab;
    r.inv_t = s.inv_t;
    const int bits = 32 - __clz(g.vocab);  // vocab < 2^bits
    r.unit = __builtin_ldexp(1.0, min(49, 63 - bits));
    r.one = __builtin_ldexp(1.0, 52) / r.unit;
    float top = -__builtin_inff();
    int live = 0;
    for (int i = threadIdx.x; i < g.vocab; i += kRow) {
        const float l = clean(T::load(r.l + i));
        top = __builtin_fmaxf(top, l);
        live += l != -__builtin_inff();
    }
    r.top = top = block_reduce(top, part.f, [](float a, float b) { return __builtin_fmaxf(a, b); });
    live = block_reduce(live, part.i, [](int a, int b) { return a + b; });
    if (live == 0) {
        if (threadIdx.x == 0) {
            g.tokens[row] = -1;
            if (g.logprobs) g.logprobs[row] = -__builtin_inff();
        }
        return;
    }
    // the kept mass: the least of what each filter keeps
    unsigned long long all = 0, high = 0;
    for (int i = threadIdx.x; i < g.vocab; i += kRow) {
        const float l = clean(T::load(r.l + i));
        if (l == -__builtin_inff()) continue;
        const double w = weight_of(l, r.top, r.inv_t);
        all += fixed(w, r.one);
        if (w >= s.min_p) high += fixed(w, r.one);
    }
    auto add = [](unsigned long long a, unsigned long long b) { return a + b; };
    double kept = static_cast<double>(block_reduce(all, part.u, add)) / r.unit;
    const double over = static_cast<double>(block_reduce(high, part.u, add)) / r.unit;
    if (s.k < live) kept = select<false>(r, s.k, 0.0, h).mass;
    if (s.top_p < 1.0) {
        // tokens stay while the mass before them is below p * kept: the first one that
        // reaches it is the last
        const double bound = s.top_p * kept;
        Place p = select<true>(r, 0, bound, h);
        // the place's token passes the bound (mass with it > bound); it stays unless
        // the mass before it is the bound already
        const double with = p.mass + weight_of(from_key(p.key), r.top, r.inv_t);
        const double cut = p.mass < bound ? with : p.mass;
        kept = cut < kept ? cut : kept;
    }
    if (s.min_p > 0.0 && over < kept) kept = over;
    const Place p = select<true>(r, 0, s.u * kept, h);
    // the before_ties-th token of that logit, in the order of indices
    int here = 0;
    const int each = (g.vocab + kRow - 1) / kRow;
    const int first = min(static_cast<int>(threadIdx.x) * each, g.vocab);
    const int end = min(first + each, g.vocab);
    for (int i = first; i < end; ++i) here += key_of(clean(T::load(r.l + i))) == p.key;
    int upto = here;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const int o = __shfl_up(upto, off, kWave);
        if (lane >= off) upto += o;
    }
    __syncthreads();
    if (lane == kWave - 1) part.i[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; ++w) upto += part.i[w];
    int left = p.before_ties - (upto - here);
    if (left >= 0 && left < here) {
        for (int i = first; i < end; ++i) {
            if (key_of(clean(T::load(r.l + i))) != p.key) continue;
            if (left-- == 0) {
                g.tokens[row] = i;
                if (g.logprobs)
                    g.logprobs[row] = static_cast<float>(
                        log(weight_of(from_key(p.key), r.top, r.inv_t) / kept));
                break;
            }
        }
    }
}

size_t sample_workspace(int rows, int vocab) { return 256; }

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
    SampleArgs g{logits, stride, uniforms, tokens, logprobs, rows, vocab, *set};
    hipLaunchKernelGGL(sample_row_kernel<T>, dim3(rows), dim3(kRow), 0, as_stream(stream), g);
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
    int rows, vocab, top;
};

// One block a row.  log(sum of exp(l - max)) = log1p(the weights of all but one token of
// the largest logit), so that a token with nearly all of the mass keeps its digits.
template <class T>
__global__ __launch_bounds__(kRow) void logprob_row_kernel(LogprobArgs g) {
    __shared__ union {
        float f[kWaves];
        double d[kWaves];
        int i[kWaves];
        unsigned long long u[kWaves];
    } part;
    const int row = blockIdx.x;
    const int token = g.tokens ? g.tokens[row] : 0;
    if (token < 0 || token >= g.vocab) return;
    const typename T::Bits* l = static_cast<const typename T::Bits*>(g.logits) + row * g.stride;
    float top = -__builtin_inff();
    for (int i = threadIdx.x; i < g.vocab; i += kRow) top = __builtin_fmaxf(top, clean(T::load(l + i)));
    top = block_reduce(top, part.f, [](float a, float b) { return __builtin_fmaxf(a, b); });
    // the largest ones are counted apart: beside a 1, weights of 1e-11 would lose digits
    double rest = 0.0;
    int largest = 0;
    for (int i = threadIdx.x; i < g.vocab; i += kRow) {
        const float v = clean(T::load(l + i));
        if (v == top)
            ++largest;
        else if (v != -__builtin_inff())
            rest += expf(v - top);
    }
    rest = block_reduce(rest, part.d, [](double a, double b) { return a + b; });
    largest = block_reduce(largest, part.i, [](int a, int b) { return a + b; });
    const double norm = log1p(rest + (largest - 1));
    auto logprob = [&](float v) {
        return v == -__builtin_inff() ? v : static_cast<float>((v == top ? 0.0 : static_cast<double>(v) - top) - norm);
    };
    if (threadIdx.x == 0 && g.tokens) g.logprobs[row] = logprob(clean(T::load(l + token)));
    unsigned long long last = ~0ull;  // key, then the lowest index
    for (int n = 0; n < g.top; ++n) {
        unsigned long long best = 0;
        for (int i = threadIdx.x; i < g.vocab; i += kRow) {
            const unsigned long long c =
                static_cast<unsigned long long>(key_of(clean(T::load(l + i)))) << 32 |
                static_cast<uint32_t>(~i);
            if (c < last && c > best) best = c;
        }
        last = block_reduce(best, part.u, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
        if (threadIdx.x == 0) {
            g.top_ids[static_cast<long>(row) * g.top + n] = static_cast<int>(~static_cast<uint32_t>(last));
            g.top_logprobs[static_cast<long>(row) * g.top + n] = logprob(from_key(static_cast<uint32_t>(last >> 32)));
        }
    }
}

size_t logprobs_workspace(int rows, int vocab, int top) { return 256; }

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
    if (int e = check_workspace(fn, ws, size, logprobs_workspace(rows, vocab, top))) return e;
    LogprobArgs g{logits, stride, tokens, logprobs, top_ids, top_logprobs, rows, vocab, top};
    hipLaunchKernelGGL(logprob_row_kernel<T>, dim3(rows), dim3(kRow), 0, as_stream(stream), g);
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
    return check_rows(fn, rows, vocab) || check_top(fn, top) ? 0 : logprobs_workspace(rows, vocab, top);
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
