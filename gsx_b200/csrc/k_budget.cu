/*
 * Keeping a set of entries (a scene's Gaussians, the rows of key-value caches) within a budget by accumulated weight.
 *
 *   accumulate  out[g, j] = decay * score[g, j] + sum over r of weights[g, r, j]
 *   select      the ordered list of the entries that stay: the `first` first, the `recent` last, and of the others
 *               those with the largest scores (ties to the lowest index)
 *   gather      the kept rows of every field, in order, in one launch
 *
 * The selection is exact: scores become 32-bit keys whose unsigned order is the scores' order, a radix select (11,
 * 11 and 10 bits from the top) finds the key of the last kept entry and how many of its equals stay, and an ordered
 * compaction writes the list.  Groups of up to kCtaKeys entries run in one CTA with their keys in shared memory;
 * longer ones spread each step over many CTAs, the last CTA of a step (an integer ticket, nobody waits) doing the
 * step's scan.
 */
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/gsx_b200.h"
#include "gsx_b200_kernels.cuh"

int gsx_internal_fail(int code, const char *msg);

namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T, int VW>
struct alignas(sizeof(T) * VW) Pack {
    T v[VW];
};

/* entries of group g in use */
__device__ __forceinline__ uint32_t length_of(const int32_t *__restrict__ lengths, uint32_t g, uint32_t length)
{
    if(lengths == nullptr) return length;
    const int32_t n = __ldg(lengths + g);
    return n < 0 ? 0u : (uint32_t)n < length ? (uint32_t)n : length;
}

/* ------------------------------------------------------------------------------------------ */
/* accumulate */

/* A CTA owns kThreads / RG * VW columns of one group; RG threads share a column's rows (row r goes to thread
 * r mod RG) and are joined in shared memory in their order. */
template <typename T, int VW, int RG>
__global__ void __launch_bounds__(kThreads) accumulate_kernel(const float *score, uint64_t score_stride,
                                                              const T *__restrict__ weights, uint64_t group_stride,
                                                              uint64_t row_stride, uint32_t groups, uint32_t rows,
                                                              uint32_t length, const int32_t *__restrict__ lengths,
                                                              const int32_t *__restrict__ row_lengths, float decay,
                                                              float *out, uint64_t out_stride)
{
    constexpr int CT = kThreads / RG;
    constexpr int U = VW >= 8 ? 4 : 8;
    __shared__ float s_part[RG > 1 ? RG * CT * VW : 1];
    const int ct = threadIdx.x % CT, rg = threadIdx.x / CT;
    for(uint32_t g = blockIdx.y; g < groups; g += gridDim.y) {
        const uint32_t n = length_of(lengths, g, length);
        const uint32_t nr = length_of(row_lengths, g, rows);
        const uint32_t j = (blockIdx.x * (uint32_t)CT + (uint32_t)ct) * VW;
        float acc[VW] = {};
        if(j < n) {
            const T *w = weights + (uint64_t)g * group_stride + j;
            uint32_t r = (uint32_t)rg;
            for(; r + (U - 1) * RG < nr; r += U * RG) {
                Pack<T, VW> x[U];
#pragma unroll
                for(int u = 0; u < U; ++u)
                    x[u] = *reinterpret_cast<const Pack<T, VW> *>(w + (uint64_t)(r + u * RG) * row_stride);
#pragma unroll
                for(int u = 0; u < U; ++u)
#pragma unroll
                    for(int v = 0; v < VW; ++v) acc[v] += to_f32(x[u].v[v]);
            }
            for(; r < nr; r += RG) {
                const Pack<T, VW> x = *reinterpret_cast<const Pack<T, VW> *>(w + (uint64_t)r * row_stride);
#pragma unroll
                for(int v = 0; v < VW; ++v) acc[v] += to_f32(x.v[v]);
            }
        }
        if(RG > 1) {
            __syncthreads();
#pragma unroll
            for(int v = 0; v < VW; ++v) s_part[(rg * VW + v) * CT + ct] = acc[v];
            __syncthreads();
            if(rg == 0)
                for(int k = 1; k < RG; ++k)
#pragma unroll
                    for(int v = 0; v < VW; ++v) acc[v] += s_part[(k * VW + v) * CT + ct];
        }
        if(rg != 0) continue;
        const float *in = score + (uint64_t)g * score_stride;
        float *to = out + (uint64_t)g * out_stride;
#pragma unroll
        for(int v = 0; v < VW; ++v) {
            const uint32_t c = j + v;
            if(c < n) to[c] = decay == 0.0f ? acc[v] : fmaf(decay, in[c], acc[v]);
            else if(c < length && to != in) to[c] = in[c];
        }
    }
}

template <typename T, int VW>
void launch_accumulate(const float *score, uint64_t score_stride, const void *weights, uint64_t group_stride,
                       uint64_t row_stride, uint32_t groups, uint32_t rows, uint32_t length, const int32_t *lengths,
                       const int32_t *row_lengths, float decay, float *out, uint64_t out_stride, cudaStream_t stream)
{
    const T *w = static_cast<const T *>(weights);
    const unsigned gy = groups < 65535u ? groups : 65535u;
    auto blocks = [&](int rg) { return dim3((length + (kThreads / rg) * VW - 1) / ((kThreads / rg) * VW), gy); };
    if(rows >= 64)
        accumulate_kernel<T, VW, 8><<<blocks(8), kThreads, 0, stream>>>(score, score_stride, w, group_stride, row_stride, groups, rows,
                                                                        length, lengths, row_lengths, decay, out, out_stride);
    else
        accumulate_kernel<T, VW, 1><<<blocks(1), kThreads, 0, stream>>>(score, score_stride, w, group_stride, row_stride, groups, rows,
                                                                        length, lengths, row_lengths, decay, out, out_stride);
}

/* ------------------------------------------------------------------------------------------ */
/* select */

constexpr int kCtaThreads = 1024;
constexpr uint32_t kCtaKeys = 49152; /* 192 KB of keys */
constexpr int kBins = 2048;
constexpr int kPasses = 3;
__device__ constexpr int kShift[kPasses] = { 21, 10, 0 };
__device__ constexpr int kPassBits[kPasses] = { 11, 11, 10 };

/* unsigned order of the keys = order of the scores; NaN below everything, -0 equal to +0 */
__device__ __forceinline__ uint32_t key_of(float x)
{
    if(x != x) return 0u;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

/* inclusive scan over a block of any whole number of warps; s_warp: 32 words */
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *s_warp, uint32_t *total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for(int d = 1; d < 32; d <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, v, d);
        if(lane >= d) v += t;
    }
    __syncthreads();
    if(lane == 31) s_warp[warp] = v;
    __syncthreads();
    uint32_t before = 0, sum = 0;
    for(int w = 0; w < warps; ++w) {
        const uint32_t s = s_warp[w];
        before += w < warp ? s : 0u;
        sum += s;
    }
    if(total) *total = sum;
    return before + v;
}

/* The bin, from the top, in which the need-th largest element lies: s_out[0] = bin, s_out[1] = how many of the
 * bin's elements are still needed.  need >= 1 and at most the sum of the bins.  A block of kBins / PER threads. */
template <int PER, typename H>
__device__ __forceinline__ void find_bin(const H &hist, uint32_t need, uint32_t *s_warp, uint32_t *s_out)
{
    uint32_t c[PER], sum = 0;
    const int top = kBins - 1 - (int)threadIdx.x * PER; /* thread 0 owns the highest bins */
#pragma unroll
    for(int k = 0; k < PER; ++k) {
        c[k] = hist(top - k);
        sum += c[k];
    }
    uint32_t above = block_scan(sum, s_warp, nullptr) - sum;
#pragma unroll
    for(int k = 0; k < PER; ++k) {
        if(above < need && above + c[k] >= need) {
            s_out[0] = (uint32_t)(top - k);
            s_out[1] = need - above;
        }
        above += c[k];
    }
    __syncthreads();
}

struct Select {
    const float *score;
    uint64_t score_stride;
    const int32_t *lengths;
    uint32_t groups, length, first, recent, budget;
    int32_t *keep;
    uint64_t keep_stride;
    int32_t *kept;
    int32_t *drop;
    uint64_t drop_stride;
};

__device__ __forceinline__ bool is_protected(const Select &a, uint32_t n, uint32_t j)
{
    return j < a.first || j >= n - a.recent;
}

/* Ordered compaction of [begin, end): entries above the threshold (or protected) and the first `need` equal ones go
 * to keep, the others to drop.  gt0 / eq0: entries above / equal before `begin`.  get(j) gives 1 for above, 0 for
 * equal, -1 for below.  Each warp takes a contiguous share. */
template <typename Get>
__device__ __forceinline__ void compact(const Select &a, uint32_t g, uint32_t begin, uint32_t end, uint32_t gt0,
                                        uint32_t eq0, uint32_t need, const Get &get, uint32_t *s_warp)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const uint32_t span = end - begin;
    const uint32_t share = ((span + warps - 1) / warps + 31) / 32 * 32;
    const uint32_t w0 = begin + (share * warp < span ? share * warp : span);
    const uint32_t w1 = end - w0 < share ? end : w0 + share;
    uint32_t gt = 0, eq = 0;
    for(uint32_t j0 = w0; j0 < w1; j0 += 32) {
        const int t = j0 + lane < w1 ? get(j0 + lane) : -1;
        gt += __popc(__ballot_sync(0xffffffffu, t > 0));
        eq += __popc(__ballot_sync(0xffffffffu, t == 0));
    }
    __syncthreads();
    if(lane == 0) {
        s_warp[warp] = gt;
        s_warp[32 + warp] = eq;
    }
    __syncthreads();
    gt = gt0;
    eq = eq0;
    for(int w = 0; w < warp; ++w) {
        gt += s_warp[w];
        eq += s_warp[32 + w];
    }
    int32_t *keep = a.keep + (uint64_t)g * a.keep_stride;
    int32_t *drop = a.drop != nullptr ? a.drop + (uint64_t)g * a.drop_stride : nullptr;
    const unsigned lt = (1u << lane) - 1u;
    for(uint32_t j0 = w0; j0 < w1; j0 += 32) {
        const uint32_t j = j0 + lane;
        const int t = j < w1 ? get(j) : -1;
        const unsigned bg = __ballot_sync(0xffffffffu, t > 0), be = __ballot_sync(0xffffffffu, t == 0);
        const uint32_t g_before = gt + __popc(bg & lt), e_before = eq + __popc(be & lt);
        const uint32_t kept_before = g_before + (e_before < need ? e_before : need);
        if(j < w1) {
            if(t > 0 || (t == 0 && e_before < need)) keep[kept_before] = (int32_t)j;
            else if(drop != nullptr) drop[j - kept_before] = (int32_t)j;
        }
        gt += __popc(bg);
        eq += __popc(be);
    }
}

/* one CTA per group, keys in shared memory */
__global__ void __launch_bounds__(kCtaThreads) select_cta_kernel(const Select a)
{
    extern __shared__ __align__(16) uint32_t s_keys[];
    __shared__ uint32_t s_hist[kBins];
    __shared__ uint32_t s_warp[64];
    __shared__ uint32_t s_found[2];
    for(uint32_t g = blockIdx.x; g < a.groups; g += gridDim.x) {
        const uint32_t n = length_of(a.lengths, g, a.length);
        const float *score = a.score + (uint64_t)g * a.score_stride;
        if(threadIdx.x == 0) a.kept[g] = (int32_t)(n < a.budget ? n : a.budget);
        if(n <= a.budget) {
            for(uint32_t j = threadIdx.x; j < n; j += kCtaThreads) a.keep[(uint64_t)g * a.keep_stride + j] = (int32_t)j;
            continue;
        }
        __syncthreads(); /* the previous group's readers of s_keys are done */
        for(uint32_t j = threadIdx.x; j < n; j += kCtaThreads) s_keys[j] = key_of(score[j]);
        uint32_t need = a.budget - a.first - a.recent, prefix = 0;
        for(int p = 0; p < kPasses && need > 0; ++p) {
            for(int b = threadIdx.x; b < kBins; b += kCtaThreads) s_hist[b] = 0u;
            __syncthreads();
            const int shift = kShift[p], bits = kPassBits[p];
            for(uint32_t j = a.first + threadIdx.x; j < n - a.recent; j += kCtaThreads) {
                const uint32_t k = s_keys[j];
                if(p == 0 || k >> (shift + bits) == prefix) atomicAdd(&s_hist[k >> shift & ((1u << bits) - 1u)], 1u);
            }
            __syncthreads();
            find_bin<kBins / kCtaThreads>([&](int b) { return s_hist[b]; }, need, s_warp, s_found);
            prefix = prefix << bits | s_found[0];
            need = s_found[1];
            __syncthreads();
        }
        const uint32_t t = need > 0 ? prefix : 0xffffffffu; /* no key reaches 0xffffffff */
        __syncthreads();
        compact(a, g, 0u, n, 0u, 0u, need,
                [&](uint32_t j) {
                    const uint32_t k = s_keys[j];
                    return is_protected(a, n, j) || k > t ? 1 : k == t ? 0 : -1;
                },
                s_warp);
    }
}

/* Long groups.  Workspace of one group: kState words of state, kPasses * kBins of histogram (both cleared by the
 * caller), then two counts for each of the group's blocks. */
constexpr int kState = 32; /* [0] prefix, [1] need, [8..11] tickets */
constexpr int kSegThreads = 512;
constexpr uint32_t kSegLeast = 8192;

uint32_t long_blocks(uint32_t groups, uint32_t length)
{
    const uint32_t most = (length + kSegLeast - 1) / kSegLeast;
    uint32_t nb = groups < 148u * 2u ? 148u * 2u / groups : 1u;
    if(nb > most) nb = most;
    return nb ? nb : 1u;
}
uint64_t long_clear_words(uint32_t groups) { return (uint64_t)groups * (kState + kPasses * kBins); }
uint64_t long_words(uint32_t groups, uint32_t length)
{
    return long_clear_words(groups) + 2ull * groups * long_blocks(groups, length);
}

struct Long {
    uint32_t *state; /* groups * kState */
    uint32_t *hist;  /* groups * kPasses * kBins */
    uint32_t *counts; /* groups * blocks * 2 */
};

__device__ __forceinline__ void segment(uint32_t n, uint32_t &begin, uint32_t &end)
{
    const uint32_t len = ((n + gridDim.x - 1) / gridDim.x + 31u) / 32u * 32u;
    const uint64_t b = (uint64_t)blockIdx.x * len;
    begin = b < n ? (uint32_t)b : n;
    end = n - begin < len ? n : begin + len;
}

/* true in the block that is the last of its group to arrive */
__device__ __forceinline__ bool last_block(uint32_t *ticket)
{
    __shared__ bool s_last;
    __threadfence();
    __syncthreads();
    if(threadIdx.x == 0) s_last = atomicAdd(ticket, 1u) == gridDim.x - 1;
    __syncthreads();
    if(s_last) __threadfence();
    return s_last;
}

template <int P>
__global__ void __launch_bounds__(kSegThreads) select_hist_kernel(const Select a, const Long w)
{
    __shared__ uint32_t s_hist[kBins];
    __shared__ uint32_t s_warp[32];
    __shared__ uint32_t s_found[2];
    const uint32_t g = blockIdx.y;
    const uint32_t n = length_of(a.lengths, g, a.length);
    const uint32_t most = a.budget - a.first - a.recent;
    if(n <= a.budget || most == 0) return;
    uint32_t *state = w.state + (uint64_t)g * kState;
    const uint32_t prefix = P > 0 ? state[0] : 0u, need = P > 0 ? state[1] : most;
    for(int b = threadIdx.x; b < kBins; b += kSegThreads) s_hist[b] = 0u;
    __syncthreads();
    const float *score = a.score + (uint64_t)g * a.score_stride;
    constexpr int shift = kShift[P], bits = kPassBits[P];
    uint32_t begin, end;
    segment(n, begin, end);
    for(uint32_t j = begin + threadIdx.x; j < end; j += kSegThreads) {
        if(is_protected(a, n, j)) continue;
        const uint32_t k = key_of(__ldg(score + j));
        if(P == 0 || k >> ((shift + bits) & 31) == prefix) atomicAdd(&s_hist[k >> shift & ((1u << bits) - 1u)], 1u);
    }
    __syncthreads();
    uint32_t *hist = w.hist + ((uint64_t)g * kPasses + P) * kBins;
    for(int b = threadIdx.x; b < kBins; b += kSegThreads)
        if(s_hist[b]) atomicAdd(&hist[b], s_hist[b]);
    if(!last_block(&state[8 + P])) return;
    find_bin<kBins / kSegThreads>([&](int b) { return __ldcg(hist + b); }, need, s_warp, s_found);
    if(threadIdx.x == 0) {
        state[0] = prefix << bits | s_found[0];
        state[1] = s_found[1];
    }
}

/* threshold and number of equals that stay, of a group with n > budget */
__device__ __forceinline__ void threshold(const Select &a, const uint32_t *state, uint32_t &t, uint32_t &need)
{
    const bool any = a.budget > a.first + a.recent;
    t = any ? state[0] : 0xffffffffu;
    need = any ? state[1] : 0u;
}

/* per block: entries above and equal; the last block turns them into counts before each block */
__global__ void __launch_bounds__(kSegThreads) select_count_kernel(const Select a, const Long w)
{
    __shared__ uint32_t s_warp[32];
    const uint32_t g = blockIdx.y;
    const uint32_t n = length_of(a.lengths, g, a.length);
    if(n <= a.budget) return;
    uint32_t *state = w.state + (uint64_t)g * kState;
    uint32_t t, need;
    threshold(a, state, t, need);
    const float *score = a.score + (uint64_t)g * a.score_stride;
    uint32_t begin, end, gt = 0, eq = 0;
    segment(n, begin, end);
    for(uint32_t j = begin + threadIdx.x; j < end; j += kSegThreads) {
        const uint32_t k = key_of(__ldg(score + j));
        if(is_protected(a, n, j) || k > t) ++gt;
        else if(k == t) ++eq;
    }
    uint32_t gts, eqs;
    block_scan(gt, s_warp, &gts);
    block_scan(eq, s_warp, &eqs);
    uint32_t *counts = w.counts + (uint64_t)g * gridDim.x * 2;
    if(threadIdx.x == 0) {
        counts[2 * blockIdx.x] = gts;
        counts[2 * blockIdx.x + 1] = eqs;
    }
    if(!last_block(&state[11])) return;
    uint32_t g_run = 0, e_run = 0;
    for(uint32_t b0 = 0; b0 < gridDim.x; b0 += kSegThreads) {
        const uint32_t b = b0 + threadIdx.x;
        const uint32_t x = b < gridDim.x ? __ldcg(counts + 2 * b) : 0u, y = b < gridDim.x ? __ldcg(counts + 2 * b + 1) : 0u;
        uint32_t xs, ys;
        const uint32_t xi = block_scan(x, s_warp, &xs), yi = block_scan(y, s_warp, &ys);
        if(b < gridDim.x) {
            counts[2 * b] = g_run + xi - x;
            counts[2 * b + 1] = e_run + yi - y;
        }
        g_run += xs;
        e_run += ys;
    }
}

__global__ void __launch_bounds__(kSegThreads) select_write_kernel(const Select a, const Long w)
{
    __shared__ uint32_t s_warp[64];
    const uint32_t g = blockIdx.y;
    const uint32_t n = length_of(a.lengths, g, a.length);
    uint32_t begin, end;
    segment(n, begin, end);
    if(blockIdx.x == 0 && threadIdx.x == 0) a.kept[g] = (int32_t)(n < a.budget ? n : a.budget);
    if(n <= a.budget) {
        for(uint32_t j = begin + threadIdx.x; j < end; j += kSegThreads) a.keep[(uint64_t)g * a.keep_stride + j] = (int32_t)j;
        return;
    }
    uint32_t t, need;
    threshold(a, w.state + (uint64_t)g * kState, t, need);
    const uint32_t *counts = w.counts + ((uint64_t)g * gridDim.x + blockIdx.x) * 2;
    const float *score = a.score + (uint64_t)g * a.score_stride;
    compact(a, g, begin, end, counts[0], counts[1], need,
            [&](uint32_t j) {
                const uint32_t k = key_of(__ldg(score + j));
                return is_protected(a, n, j) || k > t ? 1 : k == t ? 0 : -1;
            },
            s_warp);
}

/* ------------------------------------------------------------------------------------------ */
/* gather */

struct Field {
    const unsigned char *src;
    unsigned char *dst;
    uint64_t src_outer, src_inner, src_row, dst_outer, dst_inner, dst_row; /* bytes */
    uint32_t row_bytes, unit, rows_per_block, first_block;
};
struct Fields {
    Field f[GSX_B200_GATHER_MAX_FIELDS];
    int count;
};
constexpr uint32_t kGatherBytes = 16384; /* of output per CTA */

template <typename W>
__device__ __forceinline__ void gather_tile(const Field &f, const unsigned char *src, unsigned char *dst,
                                            const int32_t *__restrict__ keep, uint32_t r0, uint32_t rows, uint32_t length,
                                            uint32_t *bad)
{
    const uint32_t per_row = f.row_bytes / (uint32_t)sizeof(W);
    const uint32_t total = rows * per_row;
    for(uint32_t i = threadIdx.x; i < total; i += kThreads) {
        const uint32_t r = i / per_row, k = i - r * per_row;
        const int32_t s = __ldg(keep + r0 + r);
        if(s < 0 || (uint32_t)s >= length) {
            if(bad != nullptr && k == 0) atomicExch(bad, 1u);
            continue;
        }
        reinterpret_cast<W *>(dst + (uint64_t)(r0 + r) * f.dst_row)[k] =
            __ldg(reinterpret_cast<const W *>(src + (uint64_t)s * f.src_row) + k);
    }
}

__global__ void __launch_bounds__(kThreads) budget_gather_kernel(const __grid_constant__ Fields fields, uint32_t groups,
                                                                 uint32_t inner, uint32_t length, uint32_t budget,
                                                                 const int32_t *__restrict__ keep, uint64_t keep_stride,
                                                                 const int32_t *__restrict__ kept,
                                                                 uint32_t *__restrict__ bad)
{
    int k = 0;
    while(k + 1 < fields.count && blockIdx.x >= fields.f[k + 1].first_block) ++k;
    const Field &f = fields.f[k];
    const uint32_t r0 = (blockIdx.x - f.first_block) * f.rows_per_block;
    for(uint32_t g = blockIdx.y; g < groups; g += gridDim.y) {
        const uint32_t n = length_of(kept, g, budget);
        if(r0 >= n) continue;
        const uint32_t rows = n - r0 < f.rows_per_block ? n - r0 : f.rows_per_block;
        const uint64_t o = g / inner, i = g - (uint32_t)o * inner;
        const unsigned char *src = f.src + o * f.src_outer + i * f.src_inner;
        unsigned char *dst = f.dst + o * f.dst_outer + i * f.dst_inner;
        const int32_t *list = keep + (uint64_t)g * keep_stride;
        switch(f.unit) {
        case 16: gather_tile<uint4>(f, src, dst, list, r0, rows, length, bad); break;
        case 8: gather_tile<uint2>(f, src, dst, list, r0, rows, length, bad); break;
        case 4: gather_tile<uint32_t>(f, src, dst, list, r0, rows, length, bad); break;
        case 2: gather_tile<uint16_t>(f, src, dst, list, r0, rows, length, bad); break;
        default: gather_tile<uint8_t>(f, src, dst, list, r0, rows, length, bad); break;
        }
    }
}

int launch_status()
{
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? GSX_B200_SUCCESS : gsx_internal_fail(GSX_B200_UNKNOWN, cudaGetErrorString(e));
}

bool overlap(const void *a, uint64_t a_bytes, const void *b, uint64_t b_bytes)
{
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + b_bytes && y < x + a_bytes;
}

} // namespace

extern "C" int gsx_b200_budget_accumulate(const float *score, uint64_t score_stride, const void *weights, int weight_type,
                                          uint64_t group_stride, uint64_t row_stride, uint64_t groups, uint64_t rows,
                                          uint64_t length, const int32_t *lengths, const int32_t *row_lengths, float decay,
                                          float *out, uint64_t out_stride, void *stream_)
{
    if(weight_type != GSX_B200_DATA_F32 && weight_type != GSX_B200_DATA_F16 && weight_type != GSX_B200_DATA_BF16)
        return gsx_internal_fail(GSX_B200_NOT_SUPPORTED, "weights are f32, f16 or bf16");
    if(groups > (uint64_t)INT32_MAX || rows > (uint64_t)INT32_MAX || length > (uint64_t)INT32_MAX)
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "groups, rows and length must be below 2^31");
    if(groups == 0 || length == 0) return GSX_B200_SUCCESS;
    if(score == nullptr || out == nullptr || (rows > 0 && weights == nullptr))
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "score, weights and out must be non-null");
    const uint64_t es = weight_type == GSX_B200_DATA_F32 ? 4 : 2;
    if((uintptr_t)score % 4 || (uintptr_t)out % 4 || (uintptr_t)weights % es)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "pointers must be aligned to their element type");
    if((groups > 1 && (score_stride < length || out_stride < length)) || (rows > 1 && row_stride < length))
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "strides must be at least length elements");
    if(score_stride > (1ull << 40) || out_stride > (1ull << 40) || group_stride > (1ull << 40) || row_stride > (1ull << 40))
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "strides must be at most 2^40 elements");
    const uint64_t score_bytes = 4 * ((groups - 1) * score_stride + length), out_bytes = 4 * ((groups - 1) * out_stride + length);
    if((score != out || (groups > 1 && score_stride != out_stride)) && overlap(score, score_bytes, out, out_bytes))
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "out must be score itself or not overlap it");
    if(rows > 0 && overlap(out, out_bytes, weights, es * ((groups - 1) * group_stride + (rows - 1) * row_stride + length)))
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "out must not overlap weights");
    cudaStream_t stream = (cudaStream_t)stream_;
    const bool vec = (uintptr_t)weights % 16 == 0 && (groups == 1 || group_stride * es % 16 == 0) &&
                     (rows <= 1 || row_stride * es % 16 == 0) && length * es % 16 == 0;
#define GSX_ACCUMULATE(T, VW)                                                                                          \
    launch_accumulate<T, VW>(score, score_stride, weights, group_stride, row_stride, (uint32_t)groups, (uint32_t)rows, \
                             (uint32_t)length, lengths, row_lengths, decay, out, out_stride, stream)
    if(weight_type == GSX_B200_DATA_F32) {
        if(vec) GSX_ACCUMULATE(float, 4);
        else GSX_ACCUMULATE(float, 1);
    } else if(weight_type == GSX_B200_DATA_F16) {
        if(vec) GSX_ACCUMULATE(__half, 8);
        else GSX_ACCUMULATE(__half, 1);
    } else {
        if(vec) GSX_ACCUMULATE(__nv_bfloat16, 8);
        else GSX_ACCUMULATE(__nv_bfloat16, 1);
    }
#undef GSX_ACCUMULATE
    return launch_status();
}

extern "C" uint64_t gsx_b200_budget_workspace_bytes(uint64_t groups, uint64_t length)
{
    if(groups == 0 || length <= kCtaKeys || groups > 65535 || length > (uint64_t)INT32_MAX) return 0;
    return 4 * long_words((uint32_t)groups, (uint32_t)length);
}

extern "C" int gsx_b200_budget_select(const float *score, uint64_t score_stride, uint64_t groups, uint64_t length,
                                      const int32_t *lengths, uint64_t first, uint64_t recent, uint64_t budget,
                                      int32_t *keep, uint64_t keep_stride, int32_t *kept, int32_t *drop,
                                      uint64_t drop_stride, void *workspace, uint64_t workspace_bytes, void *stream_)
{
    if(groups > (uint64_t)INT32_MAX || length > (uint64_t)INT32_MAX || budget > (uint64_t)INT32_MAX)
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "groups, length and budget must be below 2^31");
    if(length > kCtaKeys && groups > 65535)
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "at most 65535 groups of more than 49152 entries");
    if(first > budget || recent > budget - first)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "first + recent must be at most budget");
    if(groups == 0) return GSX_B200_SUCCESS;
    if(kept == nullptr || (length > 0 && score == nullptr) || (length > 0 && budget > 0 && keep == nullptr))
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "score, keep and kept must be non-null");
    if((uintptr_t)score % 4 || (uintptr_t)keep % 4 || (uintptr_t)kept % 4 || (uintptr_t)drop % 4)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "pointers must be aligned to 4 bytes");
    const uint64_t most = budget < length ? budget : length;
    if(groups > 1 && (score_stride < length || keep_stride < most || (drop != nullptr && drop_stride < length)))
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "strides must cover a group's entries");
    cudaStream_t stream = (cudaStream_t)stream_;
    Select a;
    a.score = score;
    a.score_stride = score_stride;
    a.lengths = lengths;
    a.groups = (uint32_t)groups;
    a.length = (uint32_t)length;
    a.first = (uint32_t)first;
    a.recent = (uint32_t)recent;
    a.budget = (uint32_t)budget;
    a.keep = keep;
    a.keep_stride = keep_stride;
    a.kept = kept;
    a.drop = drop;
    a.drop_stride = drop_stride;
    if(length <= kCtaKeys) {
        const cudaError_t e = cudaFuncSetAttribute(select_cta_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kCtaKeys * 4));
        if(e != cudaSuccess) return gsx_internal_fail(GSX_B200_UNKNOWN, cudaGetErrorString(e));
        select_cta_kernel<<<(unsigned)groups, kCtaThreads, (size_t)length * 4, stream>>>(a);
        return launch_status();
    }
    const uint64_t need = gsx_b200_budget_workspace_bytes(groups, length);
    if(workspace == nullptr || (uintptr_t)workspace % 4 || workspace_bytes < need)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "workspace must hold gsx_b200_budget_workspace_bytes bytes");
    Long w;
    w.state = static_cast<uint32_t *>(workspace);
    w.hist = w.state + (size_t)groups * kState;
    w.counts = w.state + long_clear_words(a.groups);
    const cudaError_t e = cudaMemsetAsync(workspace, 0, 4 * long_clear_words(a.groups), stream);
    if(e != cudaSuccess) return gsx_internal_fail(GSX_B200_UNKNOWN, cudaGetErrorString(e));
    const dim3 grid(long_blocks(a.groups, a.length), a.groups);
    if(length > budget) {
        if(budget > first + recent) {
            select_hist_kernel<0><<<grid, kSegThreads, 0, stream>>>(a, w);
            select_hist_kernel<1><<<grid, kSegThreads, 0, stream>>>(a, w);
            select_hist_kernel<2><<<grid, kSegThreads, 0, stream>>>(a, w);
        }
        select_count_kernel<<<grid, kSegThreads, 0, stream>>>(a, w);
    }
    select_write_kernel<<<grid, kSegThreads, 0, stream>>>(a, w);
    return launch_status();
}

extern "C" int gsx_b200_budget_gather(const gsx_b200_gather_field *fields, int32_t field_count, uint64_t outer,
                                      uint64_t inner, uint64_t length, uint64_t budget, const int32_t *keep,
                                      uint64_t keep_stride, const int32_t *kept, uint32_t *device_out_of_range,
                                      void *stream_)
{
    if(field_count < 0 || field_count > GSX_B200_GATHER_MAX_FIELDS)
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "field_count must be in [0, 32]");
    if(field_count > 0 && fields == nullptr) return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "fields must be non-null");
    if(outer >= (1ull << 31) || inner >= (1ull << 31) || outer * inner > (uint64_t)INT32_MAX ||
       length > (uint64_t)INT32_MAX || budget > (uint64_t)INT32_MAX)
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "outer * inner, length and budget must be below 2^31");
    if(outer * inner == 0 || budget == 0 || field_count == 0) return GSX_B200_SUCCESS;
    if(keep == nullptr || kept == nullptr) return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "keep and kept must be non-null");
    if(outer * inner > 1 && keep_stride < budget)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "keep_stride must be at least budget");
    Fields t;
    t.count = 0;
    uint64_t blocks = 0;
    struct Span {
        const void *p;
        uint64_t bytes;
    } src_span[GSX_B200_GATHER_MAX_FIELDS], dst_span[GSX_B200_GATHER_MAX_FIELDS];
    for(int i = 0; i < field_count; ++i) {
        const gsx_b200_gather_field &in = fields[i];
        if(in.row_bytes == 0) continue;
        if(in.row_bytes > (1ull << 31)) return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "rows of at most 2^31 bytes");
        if(in.dst == nullptr || (length > 0 && in.src == nullptr))
            return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "field pointers must be non-null");
        const uint64_t limit = 1ull << 42;
        if(in.src_outer_stride > limit || in.src_inner_stride > limit || in.src_row_stride > limit ||
           in.dst_outer_stride > limit || in.dst_inner_stride > limit || in.dst_row_stride > limit)
            return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "strides must be at most 2^42 bytes");
        if(budget > 1 && in.dst_row_stride < in.row_bytes)
            return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "dst_row_stride must be at least row_bytes");
        Field &f = t.f[t.count];
        f.src = static_cast<const unsigned char *>(in.src);
        f.dst = static_cast<unsigned char *>(in.dst);
        f.src_outer = in.src_outer_stride;
        f.src_inner = in.src_inner_stride;
        f.src_row = in.src_row_stride;
        f.dst_outer = in.dst_outer_stride;
        f.dst_inner = in.dst_inner_stride;
        f.dst_row = in.dst_row_stride;
        f.row_bytes = (uint32_t)in.row_bytes;
        const uint64_t all = (uint64_t)(uintptr_t)in.src | (uint64_t)(uintptr_t)in.dst | in.row_bytes | (outer > 1 ? in.src_outer_stride | in.dst_outer_stride : 0) |
                             (inner > 1 ? in.src_inner_stride | in.dst_inner_stride : 0) | in.src_row_stride | in.dst_row_stride;
        f.unit = 16;
        while(all % f.unit) f.unit /= 2;
        f.rows_per_block = f.row_bytes >= kGatherBytes ? 1u : kGatherBytes / f.row_bytes;
        f.first_block = (uint32_t)blocks;
        blocks += (budget + f.rows_per_block - 1) / f.rows_per_block;
        src_span[t.count] = { in.src, length == 0 ? 0 : (outer - 1) * f.src_outer + (inner - 1) * f.src_inner + (length - 1) * f.src_row + f.row_bytes };
        dst_span[t.count] = { in.dst, (outer - 1) * f.dst_outer + (inner - 1) * f.dst_inner + (budget - 1) * f.dst_row + f.row_bytes };
        ++t.count;
    }
    for(int i = 0; i < t.count; ++i)
        for(int j = 0; j < t.count; ++j) {
            if(overlap(src_span[i].p, src_span[i].bytes, dst_span[j].p, dst_span[j].bytes))
                return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "a field's dst must not overlap any field's src");
        }
    if(t.count == 0) return GSX_B200_SUCCESS;
    if(blocks > (uint64_t)INT32_MAX) return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "too many rows in one call");
    const uint64_t groups = outer * inner;
    budget_gather_kernel<<<dim3((unsigned)blocks, (unsigned)(groups < 65535 ? groups : 65535)), kThreads, 0, (cudaStream_t)stream_>>>(
        t, (uint32_t)groups, (uint32_t)inner, (uint32_t)length, (uint32_t)budget, keep, keep_stride, kept, device_out_of_range);
    return launch_status();
}
