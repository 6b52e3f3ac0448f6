// rope_batch.hip -- rotary positions of a batch of tokens, norms of query and
// key heads with the rotation, and appending keys and values to a paged cache
// with the rotation on the way: one kernel over the heads of a token batch.
//
// Every element is read once and written once (4 bytes per element): the
// operators are bound by memory for long batches and by the launch for short
// ones.  The angle of pair i at position p is p * inv_freq[i] radians; in
// float32 its error grows with p (0.008 rad at p = 131072), so the product and
// its reduction to (-1/2, 1/2] turns are float64, and the hardware's sine and
// cosine, which take turns, see a small number (v_sin_f32 and v_cos_f32 on
// 65,536 turns of [-1/2, 1/2): at most 1.2e-7 off).  A token's sines and
// cosines are computed once per block into LDS and used by all of its heads.
#include <algorithm>
#include <cmath>

#include "paged.hpp"

namespace spb {
namespace {

constexpr int kHeadBlock = 256;
constexpr int kMaxTile = 2;      // tokens of a block
constexpr int kMaxHalf = 128;    // pairs of the widest head
constexpr int kMaxBlocks = 1 << 23;  // of a launch, which holds less than 2^32 lanes

// A run of heads of the batch's tokens: head h of token t at
// src + t * src_stride + h * head_dim.
struct HeadSpan {
    const uint16_t* src;
    uint16_t* dst;  // nullptr: into the cache
    long src_stride, dst_stride;
    const float* weight;  // RMSNorm before the rotation, or nullptr
    int heads;
    bool rotate;
};

struct HeadsArgs {
    HeadSpan span[3];  // q, k, v (a single span of any heads for spb_rope_tokens)
    int head_dim, tokens;
    int first;  // token of the launch's first block
    FastDiv all_heads;
    int units;      // lanes' shares of a head: head_dim / (2 V)
    int rot_units;  // those that are rotated: rotary / (2 V)
    int lanes_log;  // lanes of a head, 2^lanes_log >= units / kUnits
    int half;       // rotary / 2
    int interleaved;
    float scale, eps;
    const double* inv_freq;
    const int* positions;
    // the cache and its batch (kPaged)
    BatchArgs batch;
    uint16_t *k_pages, *v_pages;
    long page_stride, head_stride, slot_stride;
};

// A token's place: its position (negative: not there) and the element offset of
// its slot (negative: none).
struct Place {
    int pos;
    long slot;
};

// The place of token t; all lanes of the wave call it with the same t.  A lane
// takes a sequence (64 at a time), so the search is one round of loads for up
// to 64 sequences.
__device__ __forceinline__ Place find_place(const HeadsArgs& a, int t) {
    const int lane = threadIdx.x & (kWave - 1);
    Place r = {-1, -1};
    for (int base = 0; base < a.batch.seqs; base += kWave) {
        const int s = base + lane;
        SeqSpan q = {0, 0, 0};
        if (s < a.batch.seqs) q = seq_span(a.batch, s);
        const uint64_t hit = __ballot(t >= q.first && t - q.first < q.count);
        if (hit == 0) continue;
        const int l = __ffsll(static_cast<unsigned long long>(hit)) - 1;
        const int first = __shfl(q.first, l, kWave), count = __shfl(q.count, l, kWave);
        // The position comes from the length as it is given: one past the table has no slot.
        // A negative length is one of 0, whose tokens' positions are negative as well: near
        // -2^31 the difference would not fit in 32 bits.
        const int pos = max(a.batch.lens[base + l], 0) - count + (t - first);
        r.pos = pos;
        if (pos >= 0 && pos < a.batch.capacity) {
            const int p = a.batch.page.div(pos);
            const int id = a.batch.table[static_cast<long>(base + l) * a.batch.width + p];
            if (static_cast<unsigned>(id) < static_cast<unsigned>(a.batch.pages))
                r.slot = static_cast<long>(id) * a.page_stride +
                         static_cast<long>(pos - p * static_cast<int>(a.batch.page.d)) * a.slot_stride;
        }
        break;
    }
    return r;
}

template <int V>
struct Part {  // V 16-bit values that are loaded and stored at once
    uint16_t w[V];
};
template <int V>
__device__ __forceinline__ Part<V> load_part(const uint16_t* p) {
    Part<V> r;
    __builtin_memcpy(r.w, __builtin_assume_aligned(p, 2 * V), 2 * V);
    return r;
}
template <class T, int V, bool kStream>
__device__ __forceinline__ void store_part(uint16_t* p, const float (&f)[V]) {
    Part<V> r;
#pragma unroll
    for (int e = 0; e < V; ++e) r.w[e] = T::from_float(f[e]);
    if (V > 1 && kStream) {
        typedef uint32_t words __attribute__((ext_vector_type(V > 1 ? V / 2 : 2)));
        words x;
        __builtin_memcpy(&x, r.w, V > 1 ? 2 * V : 0);
        __builtin_nontemporal_store(x, reinterpret_cast<words*>(p));
    } else {
        __builtin_memcpy(__builtin_assume_aligned(p, 2 * V), r.w, 2 * V);
    }
}
// V floats of a lane in LDS: four at a time, lane after lane, so that neighbouring
// lanes read neighbouring 16 bytes.  Value i of `units` lanes' V values each:
template <int V>
__device__ __forceinline__ int lds_at(int i, int units) {
    if (V == 1) return i;
    return (i % V / 4 * units + i / V) * 4 + i % 4;
}
template <int V>
__device__ __forceinline__ void load_lds(const float* p, int u, int units, float (&f)[V]) {
    if (V == 1) {
        f[0] = p[u];
    } else {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const float4 x = reinterpret_cast<const float4*>(p)[j / 4 * units + u];
            f[j] = x.x;
            f[(j + 1) % V] = x.y;
            f[(j + 2) % V] = x.z;
            f[(j + 3) % V] = x.w;
        }
    }
}

// A block takes `tile` tokens.  2^lanes_log lanes take a head and each lane V
// pairs of it (unit u): elements [V u, V u + V) and the same past half in the
// half layout, [2 V u, 2 V u + 2 V) in the interleaved one and past the rotary
// part.  kUnits: units of a lane (2 only where a head has more than 64).  A head
// is loaded while the one before it is worked on, the first while the angles are.
// 8192 tokens of 25 heads of 128, half of each rotated: 20.2 us, 5.2 TB/s (a large
// copy reaches 4.9); 2049 tokens with norms 8.2 us with calls in a row, 3.2 TB/s (9.1 in
// a trace, which sets them apart); one token 2.8 us in a trace.
// kStream: non-temporal stores (a template's, as the compiler joins the two stores of
// a branch into a plain one).
template <class T, int V, int kUnits, bool kNorm, bool kPaged, bool kStream>
__global__ __launch_bounds__(kHeadBlock) void heads_kernel(const HeadsArgs a, const int tile) {
    __shared__ __align__(16) float cs[2][kMaxTile * kMaxHalf];
    __shared__ __align__(16) float wt[kNorm ? 2 : 1][kNorm ? 2 * kMaxHalf : 1];
    __shared__ Place place[kMaxTile];
    const int tid = threadIdx.x, t0 = a.first + blockIdx.x * tile;
    const int n = min(tile, a.tokens - t0);
    const int lanes = 1 << a.lanes_log, u0 = tid & (lanes - 1);
    const int heads = a.all_heads.d, items = n * heads, step = kHeadBlock >> a.lanes_log;

    int item = tid >> a.lanes_log;
    Part<V> raw[kUnits][2], ahead[kUnits][2];
    int at[kUnits][2];
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
        const int u = u0 + (k << a.lanes_log);
        const bool split = u < a.rot_units && !a.interleaved;
        at[k][0] = split ? V * u : 2 * V * u;
        at[k][1] = split ? V * u + a.half : 2 * V * u + V;
    }
    auto fetch = [&](int it, Part<V> (&to)[kUnits][2]) {
        const int tt = a.all_heads.div(it);
        int h = it - tt * heads;
        const int n0 = a.span[0].heads, n1 = n0 + a.span[1].heads;
        const uint16_t* src = h < n0 ? a.span[0].src : (h < n1 ? a.span[1].src : a.span[2].src);
        const long stride = h < n0 ? a.span[0].src_stride
                                   : (h < n1 ? a.span[1].src_stride : a.span[2].src_stride);
        h -= h < n0 ? 0 : (h < n1 ? n0 : n1);
        src += (t0 + tt) * stride + static_cast<long>(h) * a.head_dim;
#pragma unroll
        for (int k = 0; k < kUnits; ++k)
            if (u0 + (k << a.lanes_log) < a.units) {
                to[k][0] = load_part<V>(src + at[k][0]);
                to[k][1] = load_part<V>(src + at[k][1]);
            }
    };
    if (item < items) fetch(item, raw);

    if (kPaged) {
        for (int w = tid / kWave; w < n; w += kHeadBlock / kWave) {
            const Place p = find_place(a, t0 + w);
            if ((tid & (kWave - 1)) == 0) place[w] = p;
        }
        __syncthreads();
    }
    if (kNorm)
        for (int i = tid; i < 2 * a.head_dim; i += kHeadBlock) {
            const int which = i >= a.head_dim, d = i - which * a.head_dim;
            const float* const w = which ? a.span[1].weight : a.span[0].weight;
            if (w) wt[which][d] = w[d];
        }
    for (int i = tid; i < n * a.half; i += kHeadBlock) {
        const int tt = i / a.half, pair = i - tt * a.half;
        const int pos = kPaged ? place[tt].pos : a.positions[t0 + tt];
        double turns = static_cast<double>(pos) * (a.inv_freq[pair] * 0.15915494309189533577);
        turns -= rint(turns);
        const float x = static_cast<float>(turns);
        const int to = tt * a.half + lds_at<V>(pair, a.rot_units);
        cs[0][to] = __builtin_amdgcn_cosf(x) * a.scale;
        cs[1][to] = __builtin_amdgcn_sinf(x) * a.scale;
    }
    __syncthreads();
    for (; item < items; item += step) {
        if (item + step < items) fetch(item + step, ahead);
        const int tt = a.all_heads.div(item);
        int h = item - tt * heads, which = 0;
        if (h >= a.span[0].heads) {
            h -= a.span[0].heads;
            which = 1;
            if (h >= a.span[1].heads) {
                h -= a.span[1].heads;
                which = 2;
            }
        }
        // selects, not an index: indexed kernel arguments are copied to scratch memory
        const HeadSpan sp = which == 0 ? a.span[0] : (which == 1 ? a.span[1] : a.span[2]);
        const int pos = kPaged ? place[tt].pos : (a.positions ? a.positions[t0 + tt] : 0);
        const long t = t0 + tt;
        uint16_t* dst = nullptr;
        if (pos >= 0) {  // else padding; all lanes of a head agree
            if (!kPaged || sp.dst)
                dst = sp.dst + t * sp.dst_stride + static_cast<long>(h) * a.head_dim;
            else if (place[tt].slot >= 0)
                dst = (which == 1 ? a.k_pages : a.v_pages) + place[tt].slot + h * a.head_stride;
        }
        if (dst) {
            float x[kUnits][2][V];
#pragma unroll
            for (int k = 0; k < kUnits; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const bool have = u0 + (k << a.lanes_log) < a.units;
                    x[k][0][e] = have ? T::to_float(raw[k][0].w[e]) : 0.0f;
                    x[k][1][e] = have ? T::to_float(raw[k][1].w[e]) : 0.0f;
                }
            if (kNorm && sp.weight) {
                float ss = 0.0f;
#pragma unroll
                for (int k = 0; k < kUnits; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        ss = __builtin_fmaf(x[k][0][e], x[k][0][e], ss);
                        ss = __builtin_fmaf(x[k][1][e], x[k][1][e], ss);
                    }
                for (int off = lanes >> 1; off > 0; off >>= 1) ss += __shfl_xor(ss, off, kWave);
                const float inv = 1.0f / sqrtf(ss / static_cast<float>(a.head_dim) + a.eps);
#pragma unroll
                for (int k = 0; k < kUnits; ++k)
                    if (u0 + (k << a.lanes_log) < a.units)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float w[V];
                            __builtin_memcpy(w, __builtin_assume_aligned(
                                &wt[which][at[k][j]], V == 1 ? 4 : 16), 4 * V);
#pragma unroll
                            for (int e = 0; e < V; ++e) x[k][j][e] = (x[k][j][e] * inv) * w[e];
                        }
            }
#pragma unroll
            for (int k = 0; k < kUnits; ++k) {
                const int u = u0 + (k << a.lanes_log);
                if (u >= a.units) continue;
                if (sp.rotate && u < a.rot_units) {
                    float c[V], s[V], y[2 * V];
                    load_lds<V>(&cs[0][tt * a.half], u, a.rot_units, c);
                    load_lds<V>(&cs[1][tt * a.half], u, a.rot_units, s);
#pragma unroll
                    for (int e = 0; e < 2 * V; ++e) y[e] = x[k][e / V][e % V];
                    if (a.interleaved) {
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const float p = y[2 * e], q = y[2 * e + 1];
                            x[k][2 * e / V][2 * e % V] = __builtin_fmaf(p, c[e], -(q * s[e]));
                            x[k][(2 * e + 1) / V][(2 * e + 1) % V] = __builtin_fmaf(p, s[e], q * c[e]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const float p = y[e], q = y[V + e];
                            x[k][0][e] = __builtin_fmaf(p, c[e], -(q * s[e]));
                            x[k][1][e] = __builtin_fmaf(p, s[e], q * c[e]);
                        }
                    }
                }
                store_part<T, V, kStream>(dst + at[k][0], x[k][0]);
                store_part<T, V, kStream>(dst + at[k][1], x[k][1]);
            }
        }
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            raw[k][0] = ahead[k][0];
            raw[k][1] = ahead[k][1];
        }
    }
}

// ---- host -------------------------------------------------------------------

int check_rope(const char* fn, const spb_rope* r, int head_dim) {
    if (!r) return 0;
    if (!r->inv_freq) return invalid("%s: null inv_freq", fn);
    if (!aligned_to(r->inv_freq, 8)) return invalid("%s: inv_freq must be 8-byte aligned", fn);
    if (r->rotary_dim < 2 || r->rotary_dim % 2 || r->rotary_dim > head_dim)
        return invalid("%s: rotary_dim %d must be even and in [2, head_dim %d]", fn, r->rotary_dim,
                       head_dim);
    return 0;
}

int check_head_dim(const char* fn, int hd) {
    if (hd < 2 || hd % 2 || hd > 2 * kMaxHalf)
        return invalid("%s: head_dim %d must be even and in [2, %d]", fn, hd, 2 * kMaxHalf);
    return 0;
}

// Tokens must not overlap one another in an output.
int check_span(const char* fn, const char* what, const HeadSpan& s, int tokens, int hd) {
    if (s.heads < 0) return invalid("%s: negative number of heads", fn);
    if (!s.heads) return 0;
    const long row = static_cast<long>(s.heads) * hd;
    if (!s.src) return invalid("%s: null %s", fn, what);
    if (s.src_stride < 0 || (tokens > 1 && s.dst && s.dst_stride < row))
        return invalid("%s: %s stride smaller than a token's heads", fn, what);
    if (!aligned_to(s.src, 2) || !aligned_to(s.dst, 2))
        return invalid("%s: %s must be 2-byte aligned", fn, what);
    return 0;
}

template <class T, int V, int kUnits, bool kNorm, bool kPaged>
void launch_heads(HeadsArgs& a, int tile, bool past, hipStream_t st) {
    const dim3 block(kHeadBlock);
    const long most = static_cast<long>(kMaxBlocks) * tile;
    for (long first = 0; first < a.tokens; first += most) {
        const dim3 grid(static_cast<unsigned>((std::min(most, a.tokens - first) + tile - 1) / tile));
        a.first = static_cast<int>(first);
        if (past) hipLaunchKernelGGL((heads_kernel<T, V, kUnits, kNorm, kPaged, V != 1>), grid, block, 0, st, a, tile);
        else hipLaunchKernelGGL((heads_kernel<T, V, kUnits, kNorm, kPaged, false>), grid, block, 0, st, a, tile);
    }
}

template <class T, int V, int kUnits>
void pick_heads(HeadsArgs& a, int tile, bool norm, bool paged, bool past, hipStream_t st) {
    if (paged && norm) launch_heads<T, V, kUnits, true, true>(a, tile, past, st);
    else if (paged) launch_heads<T, V, kUnits, false, true>(a, tile, past, st);
    else if (norm) launch_heads<T, V, kUnits, true, false>(a, tile, past, st);
    else launch_heads<T, V, kUnits, false, false>(a, tile, past, st);
}

// Launches over the filled spans; the widest pair count whose parts all lie
// whole and aligned in a lane's loads.
template <class T>
int run_heads(const char* fn, HeadsArgs& a, const spb_rope* rope, bool paged, spb_stream_t stream) {
    const int rot = rope ? rope->rotary_dim : 0, hd = a.head_dim;
    a.half = rot / 2;
    a.interleaved = rope ? rope->interleaved != 0 : 1;
    a.scale = rope ? rope->scale : 1.0f;
    a.inv_freq = rope ? rope->inv_freq : nullptr;
    const long heads = static_cast<long>(a.span[0].heads) + a.span[1].heads + a.span[2].heads;
    bool norm = false;
    auto fits = [&](int v) {
        if (hd % (2 * v) || rot % (2 * v)) return false;
        for (const HeadSpan& s : a.span)
            if (s.heads && (!aligned_to(s.src, 2 * v) || !aligned_to(s.dst, 2 * v) ||
                            s.src_stride % v || s.dst_stride % v))
                return false;
        return true;  // the cache's strides are multiples of 8, its pages 16-byte aligned
    };
    for (const HeadSpan& s : a.span) norm = norm || (s.heads && s.weight);
    const int v = fits(8) ? 8 : (fits(4) ? 4 : 1);
    a.units = hd / (2 * v);
    a.rot_units = rot / (2 * v);
    a.lanes_log = 0;
    while ((1 << a.lanes_log) < a.units && a.lanes_log < 6) ++a.lanes_log;
    // Two tokens a block once one a block fills the chip.  us for 1 / 2 / 3 / 5 / 8:
    // 8192 tokens of 25 heads of 128 27.2 / 25.8 / 26.8 / 28.1 / 27.4, 2049 normed
    // tokens 10.4 / 10.4 / 11.1 / 12.3 / 15.6, 3540 tokens appended 20.7 / 19.9 /
    // 21.3 / 21.3 / 24.9 (in traces, with plain stores).
    const int tile = a.tokens >= 4 * device_cu_count() ? kMaxTile : 1;
    // a block counts its heads and one step further in 32 bits
    if (heads * tile > 0x7FFFFFFFL - kHeadBlock) return invalid("%s: more than 2^31 heads", fn);
    a.all_heads = FastDiv(static_cast<uint32_t>(heads));
    // What is larger than a die's L2 is written past it: 25.8 -> 20.1, 10.4 -> 9.6
    // and 19.9 -> 17.8 us in traces of the same three (non-temporal loads lose as much).
    const bool past = static_cast<long>(a.tokens) * heads * hd * 2 > (4L << 20);
    const hipStream_t st = as_stream(stream);
    if (v == 8) pick_heads<T, 8, 1>(a, tile, norm, paged, past, st);
    else if (v == 4) pick_heads<T, 4, 1>(a, tile, norm, paged, past, st);
    else pick_heads<T, 1, 2>(a, tile, norm, paged, past, st);
    return launch_status(fn);
}

template <class T>
int rope_tokens(const char* fn, const uint16_t* x, uint16_t* y, const int* pos,
                const spb_rope* rope, int n, int heads, int hd, long xs, long ys, spb_stream_t st) {
    clear_error();
    if (n < 0 || heads < 0) return invalid("%s: negative size", fn);
    if (!rope) return invalid("%s: null rope", fn);
    if (int e = check_head_dim(fn, hd)) return e;
    if (int e = check_rope(fn, rope, hd)) return e;
    if (n == 0 || heads == 0) return 0;
    HeadsArgs a = {};
    a.span[0] = {x, y, xs, ys, nullptr, heads, true};
    if (!y || !pos) return invalid("%s: null pointer", fn);
    if (int e = check_span(fn, "x or output", a.span[0], n, hd)) return e;
    if (x == y && xs != ys) return invalid("%s: in place with two strides", fn);
    a.head_dim = hd;
    a.tokens = n;
    a.positions = pos;
    return run_heads<T>(fn, a, rope, false, st);
}

template <class T>
int qk_norm_rope(const char* fn, const uint16_t* q, const uint16_t* k, uint16_t* qo, uint16_t* ko,
                 const float* qw, const float* kw, const int* pos, const spb_rope* rope, int n,
                 int nh, int nkv, int hd, long qs, long ks, long qos, long kos, float eps,
                 spb_stream_t st) {
    clear_error();
    if (n < 0 || nh < 0 || nkv < 0) return invalid("%s: negative size", fn);
    if (int e = check_head_dim(fn, hd)) return e;
    if (int e = check_rope(fn, rope, hd)) return e;
    if (!(eps >= 0.0f)) return invalid("%s: eps must not be negative", fn);
    if (n == 0 || nh + nkv == 0) return 0;
    HeadsArgs a = {};
    a.span[0] = {q, qo, qs, qos, qw, nh, rope != nullptr};
    a.span[1] = {k, ko, ks, kos, kw, nkv, rope != nullptr};
    if ((nh && (!qo || !qw)) || (nkv && (!ko || !kw)) || (rope && !pos))
        return invalid("%s: null pointer", fn);
    if (int e = check_span(fn, "q", a.span[0], n, hd)) return e;
    if (int e = check_span(fn, "k", a.span[1], n, hd)) return e;
    if ((nh && q == qo && qs != qos) || (nkv && k == ko && ks != kos))
        return invalid("%s: in place with two strides", fn);
    a.head_dim = hd;
    a.tokens = n;
    a.positions = rope ? pos : nullptr;
    a.eps = eps;
    return run_heads<T>(fn, a, rope, false, st);
}

template <class T>
int paged_append(const char* fn, const spb_paged_cache* c, const spb_paged_batch* b,
                 const uint16_t* k, const uint16_t* v, const uint16_t* q, uint16_t* qo, long ks,
                 long vs, long qs, long qos, int nh, const float* qw, const float* kw, float eps,
                 const spb_rope* rope, spb_stream_t st) {
    clear_error();
    if (int e = check_paged_cache(fn, c)) return e;
    if (int e = check_paged_batch(fn, b)) return e;
    if (int e = check_rope(fn, rope, c->head_dim)) return e;
    if (nh < 0) return invalid("%s: negative number of heads", fn);
    if (!(eps >= 0.0f)) return invalid("%s: eps must not be negative", fn);
    // before the pointers: those of empty tensors are null
    if (b->num_tokens == 0 || b->num_seqs == 0) return 0;
    if ((k == nullptr) != (v == nullptr)) return invalid("%s: k and v come together", fn);
    if ((q == nullptr) != (qo == nullptr)) return invalid("%s: q and q_output come together", fn);
    if (!k && !q) return invalid("%s: neither keys nor queries", fn);
    if (q && nh < 1) return invalid("%s: queries need num_heads >= 1", fn);
    if ((qw && !q) || (kw && !k)) return invalid("%s: a weight without its heads", fn);
    HeadsArgs a = {};
    const int nkv = c->num_kv_heads, hd = c->head_dim;
    if (q) a.span[0] = {q, qo, qs, qos, qw, nh, rope != nullptr};
    if (k) {
        a.span[1] = {k, nullptr, ks, 0, kw, nkv, rope != nullptr};
        a.span[2] = {v, nullptr, vs, 0, nullptr, nkv, false};
    }
    if (int e = check_span(fn, "q", a.span[0], b->num_tokens, hd)) return e;
    if (int e = check_span(fn, "k", a.span[1], b->num_tokens, hd)) return e;
    if (int e = check_span(fn, "v", a.span[2], b->num_tokens, hd)) return e;
    if (q && q == qo && qs != qos) return invalid("%s: in place with two strides", fn);
    a.head_dim = hd;
    a.tokens = b->num_tokens;
    a.eps = eps;
    a.batch = batch_args(*c, *b);
    a.k_pages = c->k;
    a.v_pages = c->v;
    a.page_stride = c->page_stride;
    a.head_stride = c->head_stride;
    a.slot_stride = c->slot_stride;
    return run_heads<T>(fn, a, rope, true, st);
}

}  // namespace

int check_paged_cache(const char* fn, const spb_paged_cache* c) {
    if (!c) return invalid("%s: null cache", fn);
    if (!c->k || !c->v) return invalid("%s: null pages", fn);
    if (c->num_pages < 1 || c->page_size < 1 || c->num_kv_heads < 1)
        return invalid("%s: a cache needs a page, a slot and a kv head", fn);
    if (c->head_dim < 8 || c->head_dim % 8 || c->head_dim > 256)
        return invalid("%s: head_dim %d of a cache must be a multiple of 8 in [8, 256]", fn,
                       c->head_dim);
    if (!aligned_to(c->k, 16) || !aligned_to(c->v, 16))
        return invalid("%s: pages must be 16-byte aligned", fn);
    const long ps = c->page_stride, hs = c->head_stride, ss = c->slot_stride, hd = c->head_dim;
    if (ps % 8 || hs % 8 || ss % 8) return invalid("%s: cache strides must be multiples of 8", fn);
    if (ps < 0 || hs < 0 || ss < 0 || (c->num_pages > 1 && ps < hd) ||
        (c->num_kv_heads > 1 && hs < hd) || (c->page_size > 1 && ss < hd))
        return invalid("%s: cache strides smaller than a head", fn);
    return 0;
}

int check_paged_batch(const char* fn, const spb_paged_batch* b) {
    if (!b) return invalid("%s: null batch", fn);
    if (b->num_seqs < 0 || b->table_width < 0 || b->num_tokens < 0 || b->max_new < 0)
        return invalid("%s: negative size of the batch", fn);
    if (b->num_seqs > 65536) return invalid("%s: more than 65536 sequences", fn);
    if (b->num_seqs == 0 || b->num_tokens == 0) return 0;
    if (!b->token_starts || !b->kv_lens || (!b->page_table && b->table_width))
        return invalid("%s: null array of the batch", fn);
    return 0;
}

BatchArgs batch_args(const spb_paged_cache& c, const spb_paged_batch& b) {
    BatchArgs a;
    a.starts = b.token_starts;
    a.lens = b.kv_lens;
    a.table = b.page_table;
    a.seqs = b.num_seqs;
    a.width = b.table_width;
    a.tokens = b.num_tokens;
    a.pages = c.num_pages;
    const long cap = static_cast<long>(b.table_width) * c.page_size;
    a.capacity = static_cast<int>(cap < 0x7FFFFF00L ? cap : 0x7FFFFF00L);
    a.page = FastDiv(static_cast<uint32_t>(c.page_size));
    return a;
}

}  // namespace spb

using namespace spb;

extern "C" {

int spb_rope_inv_freq(double* inv_freq, float* scale, int rotary_dim, double theta, int scaling,
                      double factor, int original_positions, double beta_fast, double beta_slow) {
    clear_error();
    const char* fn = "spb_rope_inv_freq";
    if (!inv_freq) return invalid("%s: null pointer", fn);
    if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > 2 * kMaxHalf)
        return invalid("%s: rotary_dim %d must be even and in [2, %d]", fn, rotary_dim,
                       2 * kMaxHalf);
    if (!(theta > 1.0) || !std::isfinite(theta)) return invalid("%s: theta must be above 1", fn);
    if (scaling < SPB_ROPE_PLAIN || scaling > SPB_ROPE_YARN)
        return invalid("%s: unknown scaling %d", fn, scaling);
    if (scaling != SPB_ROPE_PLAIN && (!(factor > 0.0) || !std::isfinite(factor)))
        return invalid("%s: factor must be positive", fn);
    if (scaling == SPB_ROPE_NTK && rotary_dim == 2)
        return invalid("%s: NTK scaling needs rotary_dim > 2", fn);
    if (scaling == SPB_ROPE_YARN && (original_positions < 1 || !(beta_slow > 0.0) ||
                                     !(beta_fast > beta_slow) || !std::isfinite(beta_fast)))
        return invalid("%s: YaRN scaling needs original_positions >= 1, beta_fast > beta_slow > 0",
                       fn);
    const double d = rotary_dim;
    if (scaling == SPB_ROPE_NTK) theta *= std::pow(factor, d / (d - 2.0));
    double low = 0.0, high = 0.0;
    if (scaling == SPB_ROPE_YARN) {
        // index of the pair that turns `beta` times over the original positions
        auto index = [&](double beta) {
            return d * std::log(original_positions / (beta * 2.0 * M_PI)) / (2.0 * std::log(theta));
        };
        low = std::fmax(std::floor(index(beta_fast)), 0.0);
        high = std::fmin(std::ceil(index(beta_slow)), d - 1.0);
    }
    for (int i = 0; i < rotary_dim / 2; ++i) {
        double f = std::pow(theta, -2.0 * i / d);
        if (scaling == SPB_ROPE_LINEAR) f /= factor;
        if (scaling == SPB_ROPE_YARN) {
            const double r = (i - low) / std::fmax(high - low, 1e-3);
            const double ramp = std::fmin(std::fmax(r, 0.0), 1.0);
            f = f * (1.0 - ramp) + f / factor * ramp;
        }
        inv_freq[i] = f;
    }
    if (scale)
        *scale = scaling == SPB_ROPE_YARN && factor > 1.0
                     ? static_cast<float>(0.1 * std::log(factor) + 1.0) : 1.0f;
    return 0;
}

int spb_rope_tokens_f16(const uint16_t* x, uint16_t* output, const int* positions,
                        const spb_rope* rope, int num_tokens, int num_heads, int head_dim,
                        long x_stride, long output_stride, spb_stream_t stream) {
    return rope_tokens<F16>("spb_rope_tokens_f16", x, output, positions, rope, num_tokens,
                            num_heads, head_dim, x_stride, output_stride, stream);
}
int spb_rope_tokens_bf16(const uint16_t* x, uint16_t* output, const int* positions,
                         const spb_rope* rope, int num_tokens, int num_heads, int head_dim,
                         long x_stride, long output_stride, spb_stream_t stream) {
    return rope_tokens<BF16>("spb_rope_tokens_bf16", x, output, positions, rope, num_tokens,
                             num_heads, head_dim, x_stride, output_stride, stream);
}
int spb_qk_norm_rope_f16(const uint16_t* q, const uint16_t* k, uint16_t* q_output,
                         uint16_t* k_output, const float* q_weight, const float* k_weight,
                         const int* positions, const spb_rope* rope, int num_tokens,
                         int num_heads, int num_kv_heads, int head_dim, long q_stride,
                         long k_stride, long q_output_stride, long k_output_stride, float eps,
                         spb_stream_t stream) {
    return qk_norm_rope<F16>("spb_qk_norm_rope_f16", q, k, q_output, k_output, q_weight, k_weight,
                             positions, rope, num_tokens, num_heads, num_kv_heads, head_dim,
                             q_stride, k_stride, q_output_stride, k_output_stride, eps, stream);
}
int spb_qk_norm_rope_bf16(const uint16_t* q, const uint16_t* k, uint16_t* q_output,
                          uint16_t* k_output, const float* q_weight, const float* k_weight,
                          const int* positions, const spb_rope* rope, int num_tokens,
                          int num_heads, int num_kv_heads, int head_dim, long q_stride,
                          long k_stride, long q_output_stride, long k_output_stride, float eps,
                          spb_stream_t stream) {
    return qk_norm_rope<BF16>("spb_qk_norm_rope_bf16", q, k, q_output, k_output, q_weight,
                              k_weight, positions, rope, num_tokens, num_heads, num_kv_heads,
                              head_dim, q_stride, k_stride, q_output_stride, k_output_stride, eps,
                              stream);
}
int spb_paged_append_f16(const spb_paged_cache* cache, const spb_paged_batch* batch,
                         const uint16_t* k, const uint16_t* v, const uint16_t* q,
                         uint16_t* q_output, long k_stride, long v_stride, long q_stride,
                         long q_output_stride, int num_heads, const float* q_weight,
                         const float* k_weight, float eps, const spb_rope* rope,
                         spb_stream_t stream) {
    return paged_append<F16>("spb_paged_append_f16", cache, batch, k, v, q, q_output, k_stride,
                             v_stride, q_stride, q_output_stride, num_heads, q_weight, k_weight,
                             eps, rope, stream);
}
int spb_paged_append_bf16(const spb_paged_cache* cache, const spb_paged_batch* batch,
                          const uint16_t* k, const uint16_t* v, const uint16_t* q,
                          uint16_t* q_output, long k_stride, long v_stride, long q_stride,
                          long q_output_stride, int num_heads, const float* q_weight,
                          const float* k_weight, float eps, const spb_rope* rope,
                          spb_stream_t stream) {
    return paged_append<BF16>("spb_paged_append_bf16", cache, batch, k, v, q, q_output, k_stride,
                              v_stride, q_stride, q_output_stride, num_heads, q_weight, k_weight,
                              eps, rope, stream);
}

}  // extern "C"
