// adapters.hip -- low-rank adapters of many requests beside a shared projection:
// output[t] = base[t] + scale[a] * B[a] (A[a] x[t]), a = ids[t].
#include "common.hpp"
#include "paged.hpp"
#include "spbitnet_amd.h"

namespace spb {
namespace {

constexpr int kMaxSections = SPB_MAX_SECTIONS;
constexpr int kMaxRank = 256;
constexpr int kMaxSize = 1 << 20;  // tokens, rows and columns: indices and grids in 32 bits
constexpr int kBlock = 256;

struct Args {
    const uint16_t* a;
    const uint16_t* b;
    const float* scales;
    const int* ranks;
    const int* ids;
    const uint16_t* x;
    const uint16_t* base;
    uint16_t* out;
    float* h;  // [tokens][sections * rank]
    long a_adapter, a_row, b_adapter, b_row, xs, bs, os;
    int num, rank, cols, sections, tokens, rows;
    int end[kMaxSections];  // first row behind each section
};

__device__ __forceinline__ int rank_of(const Args& g, int a) {
    return g.ranks ? min(max(g.ranks[a], 0), g.rank) : g.rank;
}

// h[t][j] = A[a][j] . x[t], one wave each.
template <class T>
__global__ __launch_bounds__(kBlock) void shrink_kernel(Args g) {
    const int t = blockIdx.x, lane = threadIdx.x % kWave;
    const int j = blockIdx.y * (kBlock / kWave) + threadIdx.x / kWave;
    const int a = g.ids[t];
    if (a < 0 || a >= g.num || j >= g.sections * g.rank || j % g.rank >= rank_of(g, a)) return;
    const uint16_t* w = g.a + a * g.a_adapter + j * g.a_row;
    const uint16_t* x = g.x + t * g.xs;
    float s = 0.0f;
    for (int c = lane; c < g.cols; c += kWave) s += T::to_float(w[c]) * T::to_float(x[c]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, kWave);
    if (lane == 0) g.h[static_cast<long>(t) * (g.sections * g.rank) + j] = s;
}

template <class T>
__global__ __launch_bounds__(kBlock) void expand_kernel(Args g) {
    const int t = blockIdx.x, row = blockIdx.y * kBlock + threadIdx.x;
    if (row >= g.rows) return;
    const int a = g.ids[t];
    const uint16_t bits = g.base[t * g.bs + row];
    if (a < 0 || a >= g.num) {
        if (g.base != g.out) g.out[t * g.os + row] = bits;
        return;
    }
    int sec = 0;
    while (row >= g.end[sec]) ++sec;
    const uint16_t* w = g.b + a * g.b_adapter + row * g.b_row;
    const float* h = g.h + static_cast<long>(t) * (g.sections * g.rank) + sec * g.rank;
    const int r = rank_of(g, a);
    float s = 0.0f;
    for (int j = 0; j < r; ++j) s += T::to_float(w[j]) * h[j];
    g.out[t * g.os + row] = T::from_float(T::to_float(bits) + g.scales[a] * s);
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

size_t workspace_size(const spb_adapters& d, int tokens) {
    return sizeof(float) * d.num_sections * d.rank * static_cast<size_t>(tokens);
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
    const int waves = kBlock / kWave;
    hipLaunchKernelGGL(shrink_kernel<T>, dim3(tokens, (g.sections * g.rank + waves - 1) / waves),
                       dim3(kBlock), 0, st, g);
    if (int e = launch_status(fn)) return e;
    hipLaunchKernelGGL(expand_kernel<T>, dim3(tokens, (g.rows + kBlock - 1) / kBlock),
                       dim3(kBlock), 0, st, g);
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
