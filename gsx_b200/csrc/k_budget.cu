/*
 * Keeping a set of entries (a scene's Gaussians, the rows of key-value caches) within a budget by accumulated weight.
 *
 *   accumulate  out[g, j] = decay * score[g, j] + sum over r of weights[g, r, j].  Reads every weight once; bound by DRAM
 *               (8 x 2048 x 8192 bf16: 41.6 us, 6.5 TB/s; 8 x 3M f32 onto one scene: 19.1 us, 6.3 TB/s).
 *   select      the ordered list of the entries that stay: the `first` first, the `recent` last, and of the others
 *               those with the largest scores (ties to the lowest index).  Bound by latency: each step needs the one
 *               before (32 groups of 32768: 17 us; 3M entries: 49 us in five launches over the whole GPU).
 *   gather      the kept rows of every field, in order, in one launch.  Bound by DRAM and the latency of list, then row
 *               (32 x 4096 rows of 2 x 256 bytes: 28.7 us, 134 MB; 2M Gaussians of 60 bytes: 61 us, 0.56 of DRAM's peak:
 *               a third of the rows between the kept ones is read with them).
 *
 * The selection is exact: scores become 32-bit keys whose unsigned order is the scores' order, a radix select (11,
 * 11 and 10 bits from the top; it ends early when a whole bin stays) finds the key of the last kept entry and how many
 * of its equals stay, and an ordered compaction writes the list.  Groups of up to kClusterKeys entries run in a cluster of
 * CTAs with their keys in shared memory; longer ones spread each step over the GPU, the last CTA of a step (an integer
 * ticket, nobody waits) doing the step's scan.
 */
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cooperative_groups.h>

#include "../../include/gsx_b200.h"
#include "gsx_b200_kernels.cuh"
#include "gsx_spans.h"

int gsx_internal_fail(int code, const char *msg);

namespace cg = cooperative_groups;

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

constexpr int kAccumulateCtas = 4; /* an SM */

/* U rows, hop elements apart, all in flight before the first is added: packs of VW elements, or (SPREAD) single elements
 * at VW places `apart` from the first */
template <typename T, int VW, int U, bool SPREAD>
__device__ __forceinline__ void add_rows(float (&acc)[VW], const T *__restrict__ w, uint64_t hop, const uint32_t (&apart)[VW])
{
    Pack<T, VW> x[U];
#pragma unroll
    for(int u = 0; u < U; ++u) {
        if(SPREAD)
#pragma unroll
            for(int v = 0; v < VW; ++v) x[u].v[v] = (w + u * hop)[apart[v]];
        else x[u] = *reinterpret_cast<const Pack<T, VW> *>(w + u * hop);
    }
#pragma unroll
    for(int u = 0; u < U; ++u)
#pragma unroll
        for(int v = 0; v < VW; ++v) acc[v] += to_f32(x[u].v[v]);
}

/* VW consecutive floats in accesses of up to 16 bytes */
template <int VW>
__device__ __forceinline__ void load_floats(float (&x)[VW], const float *from)
{
    constexpr int P = VW < 4 ? VW : 4;
#pragma unroll
    for(int q = 0; q < VW / P; ++q) {
        const Pack<float, P> y = reinterpret_cast<const Pack<float, P> *>(from)[q];
#pragma unroll
        for(int v = 0; v < P; ++v) x[q * P + v] = y.v[v];
    }
}

template <int VW>
__device__ __forceinline__ void store_floats(float *to, const float (&x)[VW])
{
    constexpr int P = VW < 4 ? VW : 4;
#pragma unroll
    for(int q = 0; q < VW / P; ++q) {
        Pack<float, P> y;
#pragma unroll
        for(int v = 0; v < P; ++v) y.v[v] = x[q * P + v];
        reinterpret_cast<Pack<float, P> *>(to)[q] = y;
    }
}

/* A cluster of CTAs owns kThreads / RG * VW columns of one group and deals their rows out: row r goes to the cluster's CTA
 * (r / RG) mod splits, thread row r mod RG.  A thread keeps U rows in flight; the RG threads of a column are joined in
 * shared memory, the CTAs in distributed shared memory, each in a fixed order.  SPREAD, for rows that no 4-byte access
 * fits: a thread's VW columns lie CT apart, so that the lanes' single elements stay side by side. */
template <typename T, int VW, int RG, bool SPREAD>
__global__ void __launch_bounds__(kThreads, kAccumulateCtas) accumulate_kernel(const float *score, uint64_t score_stride,
                                                              const T *__restrict__ weights, uint64_t group_stride,
                                                              uint64_t row_stride, uint32_t groups, uint32_t rows,
                                                              uint32_t length, const int32_t *__restrict__ lengths,
                                                              const int32_t *__restrict__ row_lengths, float decay,
                                                              float *out, uint64_t out_stride, bool wide_scores)
{
    constexpr int CT = kThreads / RG;
    constexpr int U = 8;
    constexpr bool kEarly = RG == 1; /* few rows: their scores are loaded before them */
    __shared__ float s_part[RG * CT * VW];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t splits = cluster.num_blocks(), split = cluster.block_rank();
    const int ct = threadIdx.x % CT, rg = threadIdx.x / CT;
    const uint32_t step = RG * splits, c0 = blockIdx.x / splits * (uint32_t)(CT * VW);
    const uint32_t j = SPREAD ? c0 + (uint32_t)ct : c0 + (uint32_t)ct * VW; /* the thread's first column */
    for(uint32_t g = blockIdx.y; g < groups; g += gridDim.y) {
        const uint32_t n = length_of(lengths, g, length);
        const uint32_t nr = length_of(row_lengths, g, rows);
        float acc[VW] = {}, before[VW] = {};
        const float *in = score + (uint64_t)g * score_stride;
        float *to = out + (uint64_t)g * out_stride;
        const bool wide = !SPREAD && wide_scores && j < n && n - j >= VW;
        if(kEarly && wide && split == 0 && decay != 0.0f) load_floats<VW>(before, in + j);
        if(j < n) {
            uint32_t apart[VW]; /* columns that are not in use are read in the place of the last */
#pragma unroll
            for(int v = 0; v < VW; ++v) apart[v] = j + v * CT < n ? v * CT : n - 1 - j;
            const T *w = weights + (uint64_t)g * group_stride + j + (uint64_t)(split * RG + (uint32_t)rg) * row_stride;
            const uint64_t hop = (uint64_t)step * row_stride;
            /* rows of this thread */
            int left = nr > split * RG + (uint32_t)rg ? (int)((nr - split * RG - (uint32_t)rg + step - 1) / step) : 0;
            for(; left >= U; left -= U, w += U * hop) add_rows<T, VW, U, SPREAD>(acc, w, hop, apart);
            if(left >= 4) {
                add_rows<T, VW, 4, SPREAD>(acc, w, hop, apart);
                left -= 4;
                w += 4 * hop;
            }
            if(left >= 2) {
                add_rows<T, VW, 2, SPREAD>(acc, w, hop, apart);
                left -= 2;
                w += 2 * hop;
            }
            if(left) add_rows<T, VW, 1, SPREAD>(acc, w, hop, apart);
        }
        if(RG > 1 || splits > 1) {
            __syncthreads();
#pragma unroll
            for(int v = 0; v < VW; ++v) s_part[(rg * VW + v) * CT + ct] = acc[v];
            __syncthreads();
            if(rg == 0) {
                for(int k = 1; k < RG; ++k)
#pragma unroll
                    for(int v = 0; v < VW; ++v) acc[v] += s_part[(k * VW + v) * CT + ct];
                if(splits > 1)
#pragma unroll
                    for(int v = 0; v < VW; ++v) s_part[v * CT + ct] = acc[v];
            }
        }
        if(splits > 1) {
            cluster.sync();
            if(split == 0 && rg == 0)
                for(uint32_t k = 1; k < splits; ++k) {
                    const float *other = cluster.map_shared_rank(s_part, k);
#pragma unroll
                    for(int v = 0; v < VW; ++v) acc[v] += other[v * CT + ct];
                }
            cluster.sync();
        }
        if(split != 0 || rg != 0) continue;
        if(wide) { /* 8 x 3M f16: 14 us, with scores one at a time 23 */
            if(!kEarly && decay != 0.0f) load_floats<VW>(before, in + j);
            if(decay != 0.0f)
#pragma unroll
                for(int v = 0; v < VW; ++v) acc[v] = fmaf(decay, before[v], acc[v]);
            store_floats<VW>(to + j, acc);
            continue;
        }
#pragma unroll
        for(int v = 0; v < VW; ++v) {
            const uint32_t c = SPREAD ? j + v * CT : j + v;
            if(c < n) to[c] = decay == 0.0f ? acc[v] : fmaf(decay, in[c], acc[v]);
            else if(c < length && to != in) to[c] = in[c];
        }
    }
}

/* Many rows that start at any element.  Rows a multiple of VW apart start at the same place of a 16-byte block, so with VW
 * thread rows every thread's rows do: it reads whole blocks, shift elements left of the CTA's columns, and the shift is
 * taken out where the thread rows are joined.  Of the CT * VW columns that the threads read, a CTA owns VW fewer.  A block
 * that reaches over the first or the last element of the weights is read by element.  8 x 2048 x 8191 bf16: 44 us, with
 * two-byte loads 73; with few rows the join costs more than it saves (8 x 3M f16 odd: 52 us, by element 25). */
template <typename T>
__global__ void __launch_bounds__(kThreads, kAccumulateCtas) accumulate_shifted_kernel(
    const float *score, uint64_t score_stride, const T *__restrict__ weights, uint64_t group_stride, uint64_t row_stride,
    uint32_t groups, uint32_t rows, uint32_t length, const int32_t *__restrict__ lengths,
    const int32_t *__restrict__ row_lengths, float decay, float *out, uint64_t out_stride)
{
    constexpr int VW = 16 / sizeof(T), RG = VW, CT = kThreads / RG, U = 8, OWN = (CT - 1) * VW;
    __shared__ __align__(16) float s_part[RG][CT * VW];
    __shared__ float s_sum[OWN];
    __shared__ uint32_t s_shift[RG];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t splits = cluster.num_blocks(), split = cluster.block_rank();
    const int ct = threadIdx.x % CT, rg = threadIdx.x / CT;
    const uint32_t step = RG * splits, c0 = blockIdx.x / splits * (uint32_t)OWN, row0 = split * RG + (uint32_t)rg;
    for(uint32_t g = blockIdx.y; g < groups; g += gridDim.y) {
        const uint32_t n = length_of(lengths, g, length);
        const uint32_t nr = length_of(row_lengths, g, rows);
        const T *w = weights + (uint64_t)g * group_stride + (uint64_t)row0 * row_stride + c0;
        const uint32_t shift = (uint32_t)((uintptr_t)w % 16) / (uint32_t)sizeof(T);
        const int64_t col = (int64_t)c0 + ct * VW - (int64_t)shift; /* the first column of the thread's block */
        w = w + ct * VW - shift;
        float acc[VW] = {};
        if(col < (int64_t)n) {
            const uint64_t hop = (uint64_t)step * row_stride;
            int left = nr > row0 ? (int)((nr - row0 + step - 1) / step) : 0;
            auto by_element = [&]() {
#pragma unroll
                for(int v = 0; v < VW; ++v)
                    if(col + v >= 0 && col + v < (int64_t)n) acc[v] += to_f32(w[v]);
                w += hop;
                --left;
            };
            if(left > 0 && col < 0 && g == 0 && row0 == 0) by_element();
            const bool last = left > 0 && col + VW > (int64_t)length && g == groups - 1 && nr == rows && (rows - 1 - row0) % step == 0;
            left -= last;
            constexpr uint32_t apart[VW] = {};
            for(; left >= U; left -= U, w += U * hop) add_rows<T, VW, U, false>(acc, w, hop, apart);
            if(left >= 4) {
                add_rows<T, VW, 4, false>(acc, w, hop, apart);
                left -= 4;
                w += 4 * hop;
            }
            if(left >= 2) {
                add_rows<T, VW, 2, false>(acc, w, hop, apart);
                left -= 2;
                w += 2 * hop;
            }
            if(left > 0) {
                add_rows<T, VW, 1, false>(acc, w, hop, apart);
                w += hop;
            }
            if(last) by_element();
        }
        __syncthreads();
        store_floats<VW>(&s_part[rg][ct * VW], acc);
        if(ct == 0) s_shift[rg] = shift;
        __syncthreads();
        const uint32_t t = threadIdx.x;
        float sum = 0.0f;
        if(t < (uint32_t)OWN)
#pragma unroll
            for(int k = 0; k < RG; ++k) sum += s_part[k][t + s_shift[k]];
        if(splits > 1) {
            if(t < (uint32_t)OWN) s_sum[t] = sum;
            cluster.sync();
            if(split == 0 && t < (uint32_t)OWN)
                for(uint32_t k = 1; k < splits; ++k) sum += cluster.map_shared_rank(s_sum, k)[t];
            cluster.sync();
        }
        if(split != 0 || t >= (uint32_t)OWN) continue;
        const float *in = score + (uint64_t)g * score_stride;
        float *to = out + (uint64_t)g * out_stride;
        const uint32_t c = c0 + t;
        if(c < n) to[c] = decay == 0.0f ? sum : fmaf(decay, in[c], sum);
        else if(c < length && to != in) to[c] = in[c];
    }
}

/* `cols` columns and `row_threads` rows at a time a CTA */
template <typename Kernel, typename... Args>
cudaError_t launch_split(Kernel kernel, uint32_t cols, uint32_t row_threads, uint32_t groups, uint32_t rows, uint32_t length,
                         cudaStream_t stream, Args... args)
{
    const uint32_t blocks = (length + cols - 1) / cols, gy = groups < 65535u ? groups : 65535u;
    /* split the rows further while the GPU is not full and a split keeps at least two rows a thread */
    uint32_t splits = 1;
    while(splits < 8 && (uint64_t)blocks * gy * splits * 2 <= 148 * kAccumulateCtas && rows >= splits * 2 * row_threads * 2) splits *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks * splits, gy);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, int VW, int RG, bool SPREAD>
cudaError_t launch_accumulate_rg(const float *score, uint64_t score_stride, const T *weights, uint64_t group_stride,
                                 uint64_t row_stride, uint32_t groups, uint32_t rows, uint32_t length,
                                 const int32_t *lengths, const int32_t *row_lengths, float decay, float *out,
                                 uint64_t out_stride, cudaStream_t stream)
{
    /* scores and out in packs where all of a group's start at 16 bytes */
    const bool wide = (((uintptr_t)score | (uintptr_t)out | (groups > 1 ? (score_stride | out_stride) * 4 : 0)) & 15) == 0;
    return launch_split(accumulate_kernel<T, VW, RG, SPREAD>, kThreads / RG * VW, RG, groups, rows, length, stream, score,
                        score_stride, weights, group_stride, row_stride, groups, rows, length, lengths, row_lengths, decay,
                        out, out_stride, wide);
}

/* `unit`: the widest access in bytes (up to 16) that every row's start and the length are multiples of */
template <typename T>
cudaError_t launch_accumulate(uint64_t unit, const float *score, uint64_t score_stride, const void *weights, uint64_t group_stride,
                              uint64_t row_stride, uint32_t groups, uint32_t rows, uint32_t length, const int32_t *lengths,
                              const int32_t *row_lengths, float decay, float *out, uint64_t out_stride, cudaStream_t stream)
{
    auto run = [&](auto launch) {
        return launch(score, score_stride, static_cast<const T *>(weights), group_stride, row_stride, groups, rows, length, lengths,
                      row_lengths, decay, out, out_stride, stream);
    };
    /* many rows: fewer columns to a CTA, whose threads share them (512 bytes of a row a CTA where it reads packs) */
    constexpr int W = 16 / sizeof(T);
    const bool many = rows >= 32;
    if(unit == 16) return many ? run(launch_accumulate_rg<T, W, 8, false>) : run(launch_accumulate_rg<T, W, 1, false>);
    if(unit == 8) return many ? run(launch_accumulate_rg<T, W / 2, 4, false>) : run(launch_accumulate_rg<T, W / 2, 1, false>);
    /* the shifted form reads whole blocks between the first and the last element: rows of at least a block, none in another */
    const uint64_t all_rows = (uint64_t)(rows - 1) * row_stride + length, all_groups = (uint64_t)(groups - 1) * group_stride + length;
    const bool apart = length >= (uint32_t)W &&
                       (groups == 1 || (group_stride >= length && (group_stride >= all_rows || row_stride >= all_groups)));
    if(many && apart)
        return launch_split(accumulate_shifted_kernel<T>, kThreads - W, W, groups, rows, length, stream, score, score_stride,
                            static_cast<const T *>(weights), group_stride, row_stride, groups, rows, length, lengths, row_lengths,
                            decay, out, out_stride);
    if(unit == 4 && sizeof(T) == 2 && !many) return run(launch_accumulate_rg<T, 2, 1, false>);
    if(many) return run(launch_accumulate_rg<T, 4, 4, true>);
    /* four columns a thread where that still fills the GPU, else one */
    if((uint64_t)groups * ((length + kThreads * 4 - 1) / (kThreads * 4)) >= 148 * kAccumulateCtas) return run(launch_accumulate_rg<T, 4, 1, true>);
    return run(launch_accumulate_rg<T, 1, 1, false>);
}

/* ------------------------------------------------------------------------------------------ */
/* select */

constexpr int kCtaThreads = 1024;
constexpr uint32_t kCtaKeys = 16384;
/* of the eight CTAs of a cluster; a group of 393216 took 48 us in a cluster (of 49152 keys a CTA) and 23 us spread over
 * the GPU, eight of 131072 25 and 30 us */
constexpr uint32_t kClusterKeys = 8 * kCtaKeys;
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
    const uint32_t mine = lane < warps ? s_warp[lane] : 0u;
    uint32_t incl = mine;
#pragma unroll
    for(int d = 1; d < 32; d <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, incl, d);
        if(lane >= d) incl += t;
    }
    if(total) *total = __shfl_sync(0xffffffffu, incl, 31);
    return v + __shfl_sync(0xffffffffu, incl - mine, warp);
}

/* The bin, from the top, in which the need-th largest element lies: s_out[0] = bin, s_out[1] = how many of the
 * bin's elements are still needed, s_out[2] = whether that is all of them.  need >= 1 and at most the sum of the bins.
 * A block of kBins / PER threads. */
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
            s_out[2] = need - above == c[k];
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

/* 1 for an entry that stays, 0 for one equal to the threshold, -1 for one below */
__device__ __forceinline__ int place_of(const Select &a, uint32_t n, uint32_t j, uint32_t key, uint32_t t)
{
    return is_protected(a, n, j) || key > t ? 1 : key == t ? 0 : -1;
}

/* A tile of compact(): four consecutive entries a thread.  kWhole: all lie before `end`.  kMiddle: none is protected. */
template <bool kWhole, bool kMiddle>
__device__ __forceinline__ void compact_tile(const Select &a, uint32_t n, uint32_t j0, uint32_t end, uint32_t &gt0, uint32_t &eq0,
                                             uint32_t t, uint32_t need, const uint32_t (&key)[4], int32_t *keep, int32_t *drop,
                                             uint32_t *s_warp)
{
    bool gt[4], eq[4];
    uint32_t sum = 0; /* above | equal << 16 */
#pragma unroll
    for(int k = 0; k < 4; ++k) {
        const bool in = kWhole || j0 + k < end;
        const bool forced = !kMiddle && is_protected(a, n, j0 + k);
        gt[k] = in && (forced || key[k] > t);
        eq[k] = in && !forced && key[k] == t;
        sum += (gt[k] ? 1u : 0u) + (eq[k] ? 0x10000u : 0u);
    }
    uint32_t all;
    const uint32_t before = block_scan(sum, s_warp, &all) - sum;
    uint32_t g = gt0 + (before & 0xffffu), e = eq0 + (before >> 16);
#pragma unroll
    for(int k = 0; k < 4; ++k) {
        const uint32_t kept_before = g + (e < need ? e : need);
        const bool stays = gt[k] || (eq[k] && e < need);
        if(stays) keep[kept_before] = (int32_t)(j0 + k);
        if(drop != nullptr && !stays && (kWhole || j0 + k < end)) drop[j0 + k - kept_before] = (int32_t)(j0 + k);
        g += gt[k] ? 1u : 0u;
        e += eq[k] ? 1u : 0u;
    }
    gt0 += all & 0xffffu;
    eq0 += all >> 16;
}

/* Ordered compaction of [begin, end): entries above the threshold (or protected) and the first `need` equal ones go
 * to keep, the others to drop.  gt0 / eq0: entries above / equal before `begin`.  load(j, key) gives the keys of four
 * consecutive entries, of which those behind `end` are not looked at. */
template <typename Load>
__device__ __forceinline__ void compact(const Select &a, uint32_t g, uint32_t n, uint32_t begin, uint32_t end, uint32_t gt0,
                                        uint32_t eq0, uint32_t t, uint32_t need, const Load &load, uint32_t *s_warp)
{
    int32_t *keep = a.keep + (uint64_t)g * a.keep_stride;
    int32_t *drop = a.drop != nullptr ? a.drop + (uint64_t)g * a.drop_stride : nullptr;
    const uint32_t tile = blockDim.x * 4;
    for(uint32_t base = begin; base < end; base += tile) {
        const uint32_t j0 = base + threadIdx.x * 4;
        const bool whole = end - base >= tile;
        uint32_t key[4] = {};
        load(j0, key, whole);
        if(whole && base >= a.first && base + tile <= n - a.recent)
            compact_tile<true, true>(a, n, j0, end, gt0, eq0, t, need, key, keep, drop, s_warp);
        else
            compact_tile<false, false>(a, n, j0, end, gt0, eq0, t, need, key, keep, drop, s_warp);
    }
}

/* Groups of up to kClusterKeys entries: a cluster of CTAs a group, each with its part of the keys in shared memory.
 * The first CTA adds up the histograms (integer atomics on distributed shared memory) and finds the bins. */
__global__ void __launch_bounds__(kCtaThreads) select_cluster_kernel(const Select a)
{
    extern __shared__ __align__(16) uint32_t s_keys[];
    __shared__ uint32_t s_hist[kBins];
    __shared__ uint32_t s_warp[32];
    __shared__ uint32_t s_found[3]; /* bin, how many of it are needed, whether that is all of them */
    __shared__ uint32_t s_counts;   /* this CTA's entries above | equal << 16 */
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank(), g = blockIdx.x / ctas;
    const uint32_t n = length_of(a.lengths, g, a.length);
    const uint32_t seg = ((n + ctas - 1) / ctas + 3u) / 4u * 4u;
    const uint32_t begin = seg * rank < n ? seg * rank : n, end = n - begin < seg ? n : begin + seg;
    const float *score = a.score + (uint64_t)g * a.score_stride;
    if(rank == 0 && threadIdx.x == 0) a.kept[g] = (int32_t)(n < a.budget ? n : a.budget);
    if(n <= a.budget) {
        for(uint32_t j = begin + threadIdx.x; j < end; j += kCtaThreads) a.keep[(uint64_t)g * a.keep_stride + j] = (int32_t)j;
        return;
    }
    uint32_t j0 = begin; /* whole rounds without a condition an entry, then the rest */
    for(; end - j0 >= kCtaThreads * 4; j0 += kCtaThreads * 4) {
        float x[4];
#pragma unroll
        for(int k = 0; k < 4; ++k) x[k] = __ldg(score + j0 + threadIdx.x + k * kCtaThreads);
#pragma unroll
        for(int k = 0; k < 4; ++k) s_keys[j0 + threadIdx.x + k * kCtaThreads - begin] = key_of(x[k]);
    }
    for(uint32_t j = j0 + threadIdx.x; j < end; j += kCtaThreads) s_keys[j - begin] = key_of(__ldg(score + j));
    uint32_t need = a.budget - a.first - a.recent, prefix = 0;
    uint32_t t = 0xffffffffu; /* no key reaches 0xffffffff */
    const uint32_t from = begin > a.first ? begin : a.first, to = end < n - a.recent ? end : n - a.recent;
    for(int p = 0; p < kPasses && need > 0; ++p) {
        for(int b = threadIdx.x; b < kBins; b += kCtaThreads) s_hist[b] = 0u;
        __syncthreads();
        const int shift = kShift[p], bits = kPassBits[p];
        for(uint32_t j = from + threadIdx.x; j < to; j += kCtaThreads) {
            const uint32_t k = s_keys[j - begin];
            if(p == 0 || k >> (shift + bits) == prefix) atomicAdd(&s_hist[k >> shift & ((1u << bits) - 1u)], 1u);
        }
        __syncthreads();
        if(ctas > 1) {
            cluster.sync();
            if(rank != 0) {
                uint32_t *hist0 = cluster.map_shared_rank(s_hist, 0);
                for(int b = threadIdx.x; b < kBins; b += kCtaThreads)
                    if(s_hist[b]) atomicAdd(hist0 + b, s_hist[b]);
            }
            cluster.sync();
        }
        if(rank == 0) {
            find_bin<kBins / kCtaThreads>([&](int b) { return s_hist[b]; }, need, s_warp, s_found);
            if(ctas > 1 && threadIdx.x > 0 && threadIdx.x < ctas) {
                uint32_t *other = cluster.map_shared_rank(s_found, threadIdx.x);
                other[0] = s_found[0];
                other[1] = s_found[1];
                other[2] = s_found[2];
            }
        }
        if(ctas > 1) cluster.sync();
        prefix = prefix << bits | s_found[0];
        need = s_found[1];
        t = prefix << shift;
        if(s_found[2] && t > 0) { /* all of the bin stay: the rest of its bits does not matter */
            --t;
            need = 0;
        }
        __syncthreads();
    }
    __syncthreads();
    uint32_t gt0 = 0, eq0 = 0;
    if(ctas > 1) {
        uint32_t gt = 0, eq = 0;
        for(uint32_t j = begin + threadIdx.x; j < end; j += kCtaThreads) {
            const int at = place_of(a, n, j, s_keys[j - begin], t);
            gt += at > 0;
            eq += at == 0;
        }
        uint32_t all;
        block_scan(gt | eq << 16, s_warp, &all);
        if(threadIdx.x == 0) s_counts = all; /* each at most kCtaKeys */
        cluster.sync();
        for(uint32_t k = 0; k < rank; ++k) {
            const uint32_t c = *cluster.map_shared_rank(&s_counts, k);
            gt0 += c & 0xffffu;
            eq0 += c >> 16;
        }
        cluster.sync(); /* nobody leaves while its counts are read */
    }
    compact(a, g, n, begin, end, gt0, eq0, t, need,
            [&](uint32_t j, uint32_t (&key)[4], bool) {
                if(j >= end) return;
                const uint4 v = *reinterpret_cast<const uint4 *>(s_keys + (j - begin));
                key[0] = v.x;
                key[1] = v.y;
                key[2] = v.z;
                key[3] = v.w;
            },
            s_warp);
}

/* Long groups.  Workspace of one group: kState words of state, kPasses * kBins of histogram (both cleared by the
 * caller), then two counts for each of the group's blocks. */
constexpr int kState = 32; /* [0] threshold so far, [1] equals needed, [2] bits still open, [8..11] tickets */
constexpr int kSegThreads = 512;
constexpr uint32_t kSegLeast = 4096;

uint32_t long_blocks(uint32_t groups, uint32_t length)
{
    const uint32_t most = (length + kSegLeast - 1) / kSegLeast;
    uint32_t nb = groups < 148u * 4u ? 148u * 4u / groups : 1u;
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
    __syncthreads();
    if(threadIdx.x == 0) { /* its fences stand for the block: what the others wrote is ordered by the barriers */
        __threadfence();
        s_last = atomicAdd(ticket, 1u) == gridDim.x - 1;
        __threadfence();
    }
    __syncthreads();
    return s_last;
}

/* f(entry, key) for the entries [begin, end) of a group, dealt to the threads, eight loads in flight; whole rounds without a
 * condition an entry (one makes a branch of each) */
template <typename F>
__device__ __forceinline__ void for_keys(const float *__restrict__ score, uint32_t begin, uint32_t end, const F &f)
{
    uint32_t j0 = begin;
    for(; end - j0 >= kSegThreads * 8; j0 += kSegThreads * 8) {
        float x[8];
#pragma unroll
        for(int k = 0; k < 8; ++k) x[k] = __ldg(score + j0 + threadIdx.x + k * kSegThreads);
#pragma unroll
        for(int k = 0; k < 8; ++k) f(j0 + threadIdx.x + k * kSegThreads, key_of(x[k]));
    }
    if(j0 >= end) return;
    float x[8]; /* entries behind the end are read in the place of the last */
#pragma unroll
    for(int k = 0; k < 8; ++k) {
        const uint32_t j = j0 + threadIdx.x + k * kSegThreads;
        x[k] = __ldg(score + (j < end ? j : end - 1));
    }
#pragma unroll
    for(int k = 0; k < 8; ++k)
        if(j0 + threadIdx.x + k * kSegThreads < end) f(j0 + threadIdx.x + k * kSegThreads, key_of(x[k]));
}

template <int P>
__global__ void __launch_bounds__(kSegThreads) select_hist_kernel(const Select a, const Long w)
{
    __shared__ uint32_t s_hist[kBins];
    __shared__ uint32_t s_warp[32];
    __shared__ uint32_t s_found[3];
    const uint32_t g = blockIdx.y;
    const uint32_t n = length_of(a.lengths, g, a.length);
    const uint32_t most = a.budget - a.first - a.recent;
    for(int b = threadIdx.x; b < kBins; b += kSegThreads) s_hist[b] = 0u;
    __syncthreads();
    gsx_pdl_trigger();
    gsx_pdl_wait();
    if(n <= a.budget || most == 0) return;
    uint32_t *state = w.state + (uint64_t)g * kState;
    const uint32_t prefix = P > 0 ? __ldcg(state) : 0u, need = P > 0 ? __ldcg(state + 1) : most;
    if(need == 0) return; /* the earlier bits decided */
    constexpr int shift = kShift[P], bits = kPassBits[P];
    uint32_t begin, end;
    segment(n, begin, end);
    if(begin < a.first) begin = a.first < end ? a.first : end;
    if(end > n - a.recent) end = n - a.recent > begin ? n - a.recent : begin;
    for_keys(a.score + (uint64_t)g * a.score_stride, begin, end, [&](uint32_t, uint32_t k) {
        if(P == 0 || (k ^ prefix) >> ((shift + bits) & 31) == 0) atomicAdd(&s_hist[k >> shift & ((1u << bits) - 1u)], 1u);
    });
    __syncthreads();
    uint32_t *hist = w.hist + ((uint64_t)g * kPasses + P) * kBins;
    for(int b = threadIdx.x; b < kBins; b += kSegThreads)
        if(s_hist[b]) atomicAdd(&hist[b], s_hist[b]);
    if(!last_block(&state[8 + P])) return;
    find_bin<kBins / kSegThreads>([&](int b) { return __ldcg(hist + b); }, need, s_warp, s_found);
    if(threadIdx.x == 0) {
        uint32_t t = prefix | s_found[0] << shift, left = s_found[1];
        if(s_found[2] && t > 0) { /* all of the bin stay: the rest of its bits does not matter */
            --t;
            left = 0;
        }
        state[0] = t;
        state[1] = left;
    }
}

/* threshold and number of equals that stay, of a group with n > budget */
__device__ __forceinline__ void threshold(const Select &a, const uint32_t *state, uint32_t &t, uint32_t &need)
{
    const bool any = a.budget > a.first + a.recent;
    t = any ? __ldcg(state) : 0xffffffffu;
    need = any ? __ldcg(state + 1) : 0u;
}

/* per block: entries above and equal; the last block turns them into counts before each block */
__global__ void __launch_bounds__(kSegThreads) select_count_kernel(const Select a, const Long w)
{
    __shared__ uint32_t s_warp[32];
    gsx_pdl_trigger();
    gsx_pdl_wait();
    const uint32_t g = blockIdx.y;
    const uint32_t n = length_of(a.lengths, g, a.length);
    if(n <= a.budget) return;
    uint32_t *state = w.state + (uint64_t)g * kState;
    uint32_t t, need;
    threshold(a, state, t, need);
    uint32_t begin, end, gt = 0, eq = 0;
    segment(n, begin, end);
    for_keys(a.score + (uint64_t)g * a.score_stride, begin, end, [&](uint32_t j, uint32_t k) {
        const int at = place_of(a, n, j, k, t);
        gt += at > 0;
        eq += at == 0;
    });
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
    __shared__ uint32_t s_warp[32];
    gsx_pdl_wait();
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
    const bool wide = (uintptr_t)(score + begin) % 16 == 0;
    compact(a, g, n, begin, end, __ldcg(counts), __ldcg(counts + 1), t, need,
            [&](uint32_t j, uint32_t (&key)[4], bool whole) {
                float x[4] = {};
                if(whole && wide) {
                    const float4 v = __ldg(reinterpret_cast<const float4 *>(score + j));
                    x[0] = v.x;
                    x[1] = v.y;
                    x[2] = v.z;
                    x[3] = v.w;
                } else {
#pragma unroll
                    for(int k = 0; k < 4; ++k)
                        if(j + k < end) x[k] = __ldg(score + j + k);
                }
#pragma unroll
                for(int k = 0; k < 4; ++k) key[k] = key_of(x[k]);
            },
            s_warp);
}

/* ------------------------------------------------------------------------------------------ */
/* gather */

struct Field {
    const unsigned char *src;
    unsigned char *dst;
    uint64_t src_outer, src_inner, dst_outer, dst_inner; /* bytes */
    uint32_t src_row, dst_row, row_bytes;
    uint32_t unit; /* bytes of an access, or 100 + the words of a short row */
    uint32_t first_block;
    uint32_t div_mul, div_shift; /* of the division by row_bytes / unit */
};
struct Fields {
    Field f[GSX_B200_GATHER_MAX_FIELDS];
    int count;
};

/* i / per_row for i < 2^31 by one multiplication (division by an invariant, Granlund and Montgomery 1994):
 * with 2^s >= d and m = floor(2^(31 + s) / d) + 1, i / d = i * m >> (31 + s) */
__device__ __forceinline__ uint32_t divide(uint32_t i, uint32_t mul, uint32_t shift)
{
    return shift ? __umulhi(i, mul) >> (shift - 1) : i;
}

/* What a CTA needs of a field and group.  The gathers below are functions of their own (not inlined), so that the widest
 * does not take registers from the others. */
struct Part {
    const unsigned char *src;
    unsigned char *dst;
    uint32_t src_row, dst_row, row_bytes, div_mul, div_shift;
};

/* A row that is not there is read in the place of row 0 and not stored: a load under a condition becomes a branch. */

/* row (of a list of n) that the list names, or UINT32_MAX for none; a name outside [0, length) sets outside */
__device__ __forceinline__ uint32_t named(uint32_t s, uint32_t r, uint32_t n, uint32_t length, bool &outside)
{
    if(r >= n) return UINT32_MAX;
    outside |= s >= length;
    return s < length ? s : UINT32_MAX;
}

/* A CTA's part of one field: accesses [first, first + kThreads * U) of a W each, all of a thread's in flight at once.
 * The list is read before its length is known (its places behind the length are not used). */
template <typename W, int U>
__device__ __noinline__ bool gather_part(const Part a, uint32_t part, const int32_t *__restrict__ keep,
                                         const int32_t *__restrict__ kept, uint32_t budget, uint32_t length)
{
    const unsigned char *__restrict__ src = a.src;
    unsigned char *__restrict__ dst = a.dst;
    const uint32_t per_row = a.row_bytes / (uint32_t)sizeof(W), src_row = a.src_row, dst_row = a.dst_row;
    const uint64_t first = (uint64_t)part * (kThreads * U);
    /* the part's first row, and accesses counted from the start of that */
    const uint32_t row0 = (uint32_t)(first / per_row), i0 = (uint32_t)(first - (uint64_t)row0 * per_row) + threadIdx.x;
    const uint32_t r0 = row0 + divide(i0, a.div_mul, a.div_shift), c0 = i0 - (r0 - row0) * per_row;
    const uint32_t dr = divide(kThreads, a.div_mul, a.div_shift), dc = kThreads - dr * per_row;
    auto next = [&](uint32_t &r, uint32_t &c) { /* the access kThreads further on */
        r += dr;
        c += dc;
        if(c >= per_row) {
            c -= per_row;
            ++r;
        }
    };
    uint32_t s[U], r = r0, c = c0;
    W x[U];
#pragma unroll
    for(int u = 0; u < U; ++u, next(r, c)) s[u] = r < budget ? (uint32_t)__ldg(keep + r) : UINT32_MAX;
    const uint32_t n = length_of(kept, 0, budget);
    if(row0 >= n) return false;
    bool outside = false;
    r = r0;
    c = c0;
#pragma unroll
    for(int u = 0; u < U; ++u, next(r, c)) {
        s[u] = named(s[u], r, n, length, outside);
        x[u] = __ldg(reinterpret_cast<const W *>(src + (uint64_t)(s[u] != UINT32_MAX ? s[u] : 0u) * src_row) + c);
    }
    r = r0;
    c = c0;
#pragma unroll
    for(int u = 0; u < U; ++u, next(r, c))
        if(s[u] != UINT32_MAX) reinterpret_cast<W *>(dst + (uint64_t)r * dst_row)[c] = x[u];
    return outside;
}

/* Short rows of WORDS 4-byte words into a contiguous, 16-byte aligned dst: a thread reads whole rows, shared memory
 * turns them into 16-byte stores (a word an access: 59 instructions a word and 88 us for the fields of a scene, this 30
 * and 61). */
constexpr int kShortRows = 1024; /* rows of a CTA */
constexpr uint32_t kShortWords = 8;
template <int WORDS>
__device__ __noinline__ bool gather_short(const Part a, uint32_t part, const int32_t *__restrict__ keep,
                                          const int32_t *__restrict__ kept, uint32_t budget, uint32_t length,
                                          uint32_t *s_tile)
{
    constexpr int U = kShortRows / kThreads;
    const unsigned char *__restrict__ src = a.src;
    const uint32_t row0 = part * kShortRows;
    uint32_t s[U], x[U][WORDS];
#pragma unroll
    for(int u = 0; u < U; ++u) {
        const uint32_t r = row0 + threadIdx.x + u * kThreads;
        s[u] = r < budget ? (uint32_t)__ldg(keep + r) : UINT32_MAX;
    }
    const uint32_t n = length_of(kept, 0, budget), src_row = a.src_row;
    if(row0 >= n) return false;
    bool outside = false;
#pragma unroll
    for(int u = 0; u < U; ++u) {
        s[u] = named(s[u], row0 + threadIdx.x + u * kThreads, n, length, outside);
        const uint32_t *from = reinterpret_cast<const uint32_t *>(src + (uint64_t)(s[u] != UINT32_MAX ? s[u] : 0u) * src_row);
#pragma unroll
        for(int w = 0; w < WORDS; ++w) x[u][w] = __ldg(from + w);
    }
    uint32_t *to = reinterpret_cast<uint32_t *>(a.dst) + (uint64_t)row0 * WORDS;
    if(__syncthreads_or(outside)) { /* some rows stay as they were */
#pragma unroll
        for(int u = 0; u < U; ++u)
            if(s[u] != UINT32_MAX)
#pragma unroll
                for(int w = 0; w < WORDS; ++w) to[(threadIdx.x + u * kThreads) * WORDS + w] = x[u][w];
        return outside;
    }
#pragma unroll
    for(int u = 0; u < U; ++u)
#pragma unroll
        for(int w = 0; w < WORDS; ++w) s_tile[(threadIdx.x + u * kThreads) * WORDS + w] = x[u][w];
    __syncthreads();
    const uint32_t words = (n - row0 < (uint32_t)kShortRows ? n - row0 : (uint32_t)kShortRows) * WORDS;
    for(uint32_t i = threadIdx.x; i < words / 4; i += kThreads)
        reinterpret_cast<uint4 *>(to)[i] = reinterpret_cast<const uint4 *>(s_tile)[i];
    if(threadIdx.x < words % 4) to[words / 4 * 4 + threadIdx.x] = s_tile[words / 4 * 4 + threadIdx.x];
    __syncthreads();
    return false;
}

/* accesses of a thread by their size: 16 KB of output a CTA in whole packs, less where rows need narrower accesses */
__host__ __device__ constexpr uint32_t gather_accesses(uint32_t unit) { return unit == 16 ? 4u : 8u; }

__global__ void __launch_bounds__(kThreads, 4) budget_gather_kernel(const __grid_constant__ Fields fields, uint32_t groups,
                                                                    uint32_t inner, uint32_t length, uint32_t budget,
                                                                    const int32_t *__restrict__ keep, uint64_t keep_stride,
                                                                    const int32_t *__restrict__ kept,
                                                                    uint32_t *__restrict__ bad)
{
    __shared__ __align__(16) uint32_t s_tile[kShortRows * kShortWords];
    if(length == 0) { /* no row to name */
        for(uint32_t g = blockIdx.y; g < groups; g += gridDim.y)
            if(bad != nullptr && threadIdx.x == 0 && length_of(kept, g, budget) > 0) atomicExch(bad, 1u);
        return;
    }
    int k = 0;
    while(k + 1 < fields.count && blockIdx.x >= fields.f[k + 1].first_block) ++k;
    const Field &f = fields.f[k];
    const uint32_t part = blockIdx.x - f.first_block;
    for(uint32_t g = blockIdx.y; g < groups; g += gridDim.y) {
        const uint32_t o = g / inner, i = g - o * inner;
        const Part a = { f.src + o * f.src_outer + i * f.src_inner, f.dst + o * f.dst_outer + i * f.dst_inner, f.src_row,
                         f.dst_row, f.row_bytes, f.div_mul, f.div_shift };
        const int32_t *list = keep + (uint64_t)g * keep_stride;
        bool outside;
        switch(f.unit) {
        case 101: outside = gather_short<1>(a, part, list, kept + g, budget, length, s_tile); break;
        case 102: outside = gather_short<2>(a, part, list, kept + g, budget, length, s_tile); break;
        case 103: outside = gather_short<3>(a, part, list, kept + g, budget, length, s_tile); break;
        case 104: outside = gather_short<4>(a, part, list, kept + g, budget, length, s_tile); break;
        case 105: outside = gather_short<5>(a, part, list, kept + g, budget, length, s_tile); break;
        case 106: outside = gather_short<6>(a, part, list, kept + g, budget, length, s_tile); break;
        case 107: outside = gather_short<7>(a, part, list, kept + g, budget, length, s_tile); break;
        case 108: outside = gather_short<8>(a, part, list, kept + g, budget, length, s_tile); break;
        case 16: outside = gather_part<uint4, gather_accesses(16)>(a, part, list, kept + g, budget, length); break;
        case 8: outside = gather_part<uint2, gather_accesses(8)>(a, part, list, kept + g, budget, length); break;
        case 4: outside = gather_part<uint32_t, gather_accesses(4)>(a, part, list, kept + g, budget, length); break;
        case 2: outside = gather_part<uint16_t, gather_accesses(2)>(a, part, list, kept + g, budget, length); break;
        default: outside = gather_part<uint8_t, gather_accesses(1)>(a, part, list, kept + g, budget, length); break;
        }
        if(outside && bad != nullptr) atomicExch(bad, 1u);
    }
}

int launch_status(cudaError_t e = cudaSuccess)
{
    const cudaError_t last = cudaGetLastError();
    if(e == cudaSuccess) e = last;
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
    if((uintptr_t)score % 4 || (uintptr_t)out % 4 || (uintptr_t)weights % es || (uintptr_t)lengths % 4 || (uintptr_t)row_lengths % 4)
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
    const GsxRows written(out, 4 * length, { { groups, 4 * out_stride } });
    if(gsx_rows_meet(written, { lengths, 4 * groups }) || gsx_rows_meet(written, { row_lengths, 4 * groups }))
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "out must not overlap lengths or row_lengths");
    cudaStream_t stream = (cudaStream_t)stream_;
    const uint64_t all = (uint64_t)(uintptr_t)weights | length * es | (groups > 1 ? group_stride * es : 0) | (rows > 1 ? row_stride * es : 0);
    uint64_t unit = 16;
    while(all % unit) unit /= 2;
    auto run = [&](auto launch) {
        return launch_status(launch(unit, score, score_stride, weights, group_stride, row_stride, (uint32_t)groups, (uint32_t)rows,
                                    (uint32_t)length, lengths, row_lengths, decay, out, out_stride, stream));
    };
    if(weight_type == GSX_B200_DATA_F32) return run(launch_accumulate<float>);
    if(weight_type == GSX_B200_DATA_F16) return run(launch_accumulate<__half>);
    return run(launch_accumulate<__nv_bfloat16>);
}

extern "C" uint64_t gsx_b200_budget_workspace_bytes(uint64_t groups, uint64_t length)
{
    if(groups == 0 || length <= kClusterKeys || groups > 65535 || length > (uint64_t)INT32_MAX) return 0;
    return 4 * long_words((uint32_t)groups, (uint32_t)length);
}

extern "C" int gsx_b200_budget_select(const float *score, uint64_t score_stride, uint64_t groups, uint64_t length,
                                      const int32_t *lengths, uint64_t first, uint64_t recent, uint64_t budget,
                                      int32_t *keep, uint64_t keep_stride, int32_t *kept, int32_t *drop,
                                      uint64_t drop_stride, void *workspace, uint64_t workspace_bytes, void *stream_)
{
    if(groups > (uint64_t)INT32_MAX || length > (uint64_t)INT32_MAX || budget > (uint64_t)INT32_MAX)
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "groups, length and budget must be below 2^31");
    if(groups > (length > kClusterKeys ? 65535u : 1u << 27))
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "at most 65535 groups of more than 131072 entries, 2^27 of fewer");
    if(first > budget || recent > budget - first)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "first + recent must be at most budget");
    if(groups == 0) return GSX_B200_SUCCESS;
    if(kept == nullptr || (length > 0 && score == nullptr) || (length > 0 && budget > 0 && keep == nullptr))
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "score, keep and kept must be non-null");
    if((uintptr_t)score % 4 || (uintptr_t)keep % 4 || (uintptr_t)kept % 4 || (uintptr_t)drop % 4 || (uintptr_t)lengths % 4)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "pointers must be aligned to 4 bytes");
    const uint64_t most = budget < length ? budget : length;
    if(groups > 1 && (score_stride < length || keep_stride < most || (drop != nullptr && drop_stride < length)))
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "strides must cover a group's entries");
    if(groups > 1 && (score_stride > (1ull << 40) || keep_stride > (1ull << 40) || (drop != nullptr && drop_stride > (1ull << 40))))
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "strides must be at most 2^40 elements");
    const uint64_t need = gsx_b200_budget_workspace_bytes(groups, length);
    /* scores and lengths are read again while the lists are written: by other CTAs of a group, and in the long form by every step */
    const GsxRows written[] = { { keep, 4 * most, { { groups, 4 * keep_stride } } },
                                { drop, length > budget ? 4 * (length - budget) : 0, { { groups, 4 * drop_stride } } },
                                { kept, 4 * groups },
                                { workspace, need } };
    const GsxRows read[] = { { score, 4 * length, { { groups, 4 * score_stride } } }, { lengths, 4 * groups } };
    for(int i = 0; i < 4; ++i) {
        for(const GsxRows &r : read)
            if(gsx_rows_meet(written[i], r))
                return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "keep, kept, drop and workspace must not overlap score or lengths");
        for(int j = 0; j < i; ++j)
            if(gsx_rows_meet(written[i], written[j]))
                return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "keep, kept, drop and workspace must not overlap one another");
    }
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
    if(length <= kClusterKeys) {
        /* as many CTAs as the keys need, and more while the GPU is not full (two an SM) and a part keeps 8192 entries
         * (barriers between more CTAs cost more than they save: 32 groups of 32768 took 20.7 us with parts of 4096,
         * 18.4 with 8192) */
        uint32_t ctas = 1;
        while(ctas < 8 && (length > (uint64_t)ctas * kCtaKeys || (groups * ctas * 2 <= 148 * 2 && length >= (uint64_t)ctas * 2 * 8192)))
            ctas *= 2;
        const size_t part = ((length + ctas - 1) / ctas + 3) / 4 * 4;
        cudaError_t e = gsx_allow_smem<select_cluster_kernel>(kCtaKeys * 4);
        if(e != cudaSuccess) return launch_status(e);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(groups * ctas));
        cfg.blockDim = dim3(kCtaThreads);
        cfg.dynamicSmemBytes = part * 4;
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ctas;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return launch_status(cudaLaunchKernelEx(&cfg, select_cluster_kernel, a));
    }
    if(workspace == nullptr || (uintptr_t)workspace % 4 || workspace_bytes < need)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "workspace must hold gsx_b200_budget_workspace_bytes bytes");
    Long w;
    w.state = static_cast<uint32_t *>(workspace);
    w.hist = w.state + (size_t)groups * kState;
    w.counts = w.state + long_clear_words(a.groups);
    const dim3 grid(long_blocks(a.groups, a.length), a.groups), block(kSegThreads);
    if(length <= budget) { /* every group keeps all */
        select_write_kernel<<<grid, block, 0, stream>>>(a, w);
        return launch_status();
    }
    cudaError_t e = cudaMemsetAsync(workspace, 0, 4 * long_clear_words(a.groups), stream);
    if(e == cudaSuccess && budget > first + recent) {
        select_hist_kernel<0><<<grid, block, 0, stream>>>(a, w);
        e = gsx_launch_pdl(select_hist_kernel<1>, grid, block, 0, stream, a, w);
        if(e == cudaSuccess) e = gsx_launch_pdl(select_hist_kernel<2>, grid, block, 0, stream, a, w);
        if(e == cudaSuccess) e = gsx_launch_pdl(select_count_kernel, grid, block, 0, stream, a, w);
    } else if(e == cudaSuccess) {
        select_count_kernel<<<grid, block, 0, stream>>>(a, w);
    }
    if(e == cudaSuccess) e = gsx_launch_pdl(select_write_kernel, grid, block, 0, stream, a, w);
    return launch_status(e);
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
    if((uintptr_t)keep % 4 || (uintptr_t)kept % 4 || (uintptr_t)device_out_of_range % 4)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "pointers must be aligned to 4 bytes");
    if(outer * inner > 1 && keep_stride < budget)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "keep_stride must be at least budget");
    if(outer * inner > 1 && keep_stride > (1ull << 40)) return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "keep_stride must be at most 2^40 elements");
    const GsxRows lists[] = { { keep, 4 * budget, { { outer * inner, 4 * keep_stride } } },
                              { kept, 4 * outer * inner },
                              { device_out_of_range, 4 } };
    Fields t;
    t.count = 0;
    uint64_t blocks = 0;
    struct Span {
        const void *p;
        uint64_t bytes;
    } src_span[GSX_B200_GATHER_MAX_FIELDS], dst_span[GSX_B200_GATHER_MAX_FIELDS];
    GsxRows dst_rows[GSX_B200_GATHER_MAX_FIELDS];
    for(int i = 0; i < field_count; ++i) {
        const gsx_b200_gather_field &in = fields[i];
        if(in.row_bytes == 0) continue;
        if(in.row_bytes > (1ull << 30)) return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "rows of at most 2^30 bytes");
        if(in.dst == nullptr || (length > 0 && in.src == nullptr))
            return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "field pointers must be non-null");
        const uint64_t limit = 1ull << 42;
        if(in.src_outer_stride > limit || in.src_inner_stride > limit || in.dst_outer_stride > limit || in.dst_inner_stride > limit ||
           in.src_row_stride > UINT32_MAX || in.dst_row_stride > UINT32_MAX)
            return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "group strides of at most 2^42 bytes, row strides below 2^32");
        if(budget > 1 && in.dst_row_stride < in.row_bytes)
            return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "dst_row_stride must be at least row_bytes");
        Field &f = t.f[t.count];
        f.src = static_cast<const unsigned char *>(in.src);
        f.dst = static_cast<unsigned char *>(in.dst);
        f.src_outer = in.src_outer_stride;
        f.src_inner = in.src_inner_stride;
        f.src_row = (uint32_t)in.src_row_stride;
        f.dst_outer = in.dst_outer_stride;
        f.dst_inner = in.dst_inner_stride;
        f.dst_row = (uint32_t)in.dst_row_stride;
        f.row_bytes = (uint32_t)in.row_bytes;
        const uint64_t all = (uint64_t)(uintptr_t)in.src | (uint64_t)(uintptr_t)in.dst | in.row_bytes | (outer > 1 ? in.src_outer_stride | in.dst_outer_stride : 0) |
                             (inner > 1 ? in.src_inner_stride | in.dst_inner_stride : 0) | in.src_row_stride | in.dst_row_stride;
        f.unit = 16;
        while(all % f.unit) f.unit /= 2;
        const uint64_t per_row = f.row_bytes / f.unit;
        f.div_shift = 0;
        while((1ull << f.div_shift) < per_row) ++f.div_shift;
        f.div_mul = f.div_shift ? (uint32_t)((1ull << (31 + f.div_shift)) / per_row + 1) : 0u;
        f.first_block = (uint32_t)blocks;
        const uint64_t dst_all = (uint64_t)(uintptr_t)in.dst | (outer > 1 ? in.dst_outer_stride : 0) | (inner > 1 ? in.dst_inner_stride : 0);
        uint64_t part = kThreads * gather_accesses(f.unit), accesses = budget * per_row;
        if(f.unit < 16 && f.unit >= 4 && f.row_bytes <= kShortWords * 4 && f.dst_row == f.row_bytes && dst_all % 16 == 0) {
            f.unit = 100 + f.row_bytes / 4;
            part = kShortRows;
            accesses = budget;
        }
        blocks += (accesses + part - 1) / part;
        if(blocks > (uint64_t)INT32_MAX) return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "too many rows in one call");
        src_span[t.count] = { in.src, length == 0 ? 0 : (outer - 1) * f.src_outer + (inner - 1) * f.src_inner + (length - 1) * (uint64_t)f.src_row + f.row_bytes };
        dst_span[t.count] = { in.dst, (outer - 1) * f.dst_outer + (inner - 1) * f.dst_inner + (budget - 1) * (uint64_t)f.dst_row + f.row_bytes };
        dst_rows[t.count] = GsxRows(in.dst, in.row_bytes, { { outer, f.dst_outer }, { inner, f.dst_inner }, { budget, f.dst_row } });
        if(!dst_rows[t.count].nested())
            return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "the rows and groups of a field's dst must not overlap");
        for(const GsxRows &r : lists)
            if(gsx_rows_meet(dst_rows[t.count], r))
                return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "a field's dst must not overlap keep, kept or the flag");
        ++t.count;
    }
    for(int i = 0; i < t.count; ++i)
        for(int j = 0; j < t.count; ++j) {
            /* keys and values may interleave in one buffer: rows, not spans */
            if(j < i && gsx_rows_meet(dst_rows[i], dst_rows[j]))
                return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "a field's dst must not overlap another's");
            if(overlap(src_span[i].p, src_span[i].bytes, dst_span[j].p, dst_span[j].bytes))
                return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "a field's dst must not overlap any field's src");
        }
    if(t.count == 0) return GSX_B200_SUCCESS;
    const uint64_t groups = outer * inner;
    budget_gather_kernel<<<dim3((unsigned)blocks, (unsigned)(groups < 65535 ? groups : 65535)), kThreads, 0, (cudaStream_t)stream_>>>(
        t, (uint32_t)groups, (uint32_t)inner, (uint32_t)length, (uint32_t)budget, keep, keep_stride, kept, device_out_of_range);
    return launch_status();
}
