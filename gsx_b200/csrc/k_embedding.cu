/*
 * Shared rows: out[n] = scale * table[index[n]], and the gradient of the table.
 *
 * The gradient grad_table[v] = scale * sum of grad_out[n] over the n with index[n] = v is summed in the order of
 * the positions n, grouped by row: a stable counting sort of the positions by row, then one sum per row.  No
 * floating-point atomics: the same inputs give the same bits.
 *
 *   sort    count <= kSmallCount: one CTA sorts (row, position) in shared memory by 8-bit digits.
 *           else, per digit of at most 12 bits: per-chunk digit counts, an exclusive scan over (digit, chunk), a
 *           scatter in which every warp ranks its own part of the chunk (__match_any_sync).  Tables of up to 4096
 *           rows need one pass.  Positions whose index is the padding row or out of range are dropped in the
 *           first pass.
 *   pieces  the sorted order is cut into pieces of kPiece positions; a piece that lies in one row is summed by a
 *           CTA of its own, so that a row which holds most of the positions is spread over the whole GPU.
 *   rows    a warp sums each row of up to kWarpMax positions, a CTA each longer one (its pieces' sums and the raw
 *           positions before and after them), scales, rounds once and stores.  Rows without positions get zeros.
 *
 * Sums are held in 32 bits: a row is split over the lanes that share its columns, then warps, then pieces, so no
 * chain of additions is longer than kPiece / 8 = 64 positions plus one term a piece.
 */
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/gsx_b200.h"
#include "gsx_b200_kernels.cuh"

int gsx_internal_fail(int code, const char *msg);

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPiece = 512;
constexpr int kWarpMax = 64;
constexpr int kSmallThreads = 1024;
constexpr int kSmallItems = 8;
constexpr int kSmallCount = kSmallThreads * kSmallItems;
constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxBits = 12;
constexpr int kMaxBins = 1 << kMaxBits;
constexpr uint64_t kMaxChunk = 32768; /* a warp's counts of one digit fit 16 bits */
constexpr int kChunks = 148;

/* ---- element types ---- */
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

/* VW elements that are loaded and stored with accesses of up to 16 bytes */
template <typename T, int VW>
struct alignas(sizeof(T) * VW > 16 ? 16 : sizeof(T) * VW) Pack {
    T v[VW];
};

/* ------------------------------------------------------------------------------------------ */
/* lookup */

/* rows of whole VW-element packs: one pack per thread and step */
template <typename T, typename O, typename I, int VW, int U>
__global__ void __launch_bounds__(kThreads) lookup_pack_kernel(const T *__restrict__ table, uint64_t rows,
                                                               uint32_t packs, uint64_t table_stride,
                                                               const I *__restrict__ index, uint64_t total, float scale,
                                                               O *__restrict__ out, uint64_t out_stride,
                                                               uint32_t *__restrict__ bad)
{
    const uint64_t w0 = (uint64_t)blockIdx.x * (kThreads * U) + threadIdx.x;
    uint64_t n[U];
    uint32_t c[U];
    I s[U];
    Pack<T, VW> x[U];
#pragma unroll
    for(int u = 0; u < U; ++u) {
        const uint64_t w = w0 + (uint64_t)u * kThreads;
        n[u] = total <= 0xffffffffull ? (uint64_t)((uint32_t)w / packs) : w / packs;
        c[u] = (uint32_t)(w - n[u] * packs);
        s[u] = w < total ? __ldg(index + n[u]) : (I)-1;
    }
#pragma unroll
    for(int u = 0; u < U; ++u)
        if(s[u] >= 0 && (uint64_t)s[u] < rows)
            x[u] = *reinterpret_cast<const Pack<T, VW> *>(table + (uint64_t)s[u] * table_stride + (uint64_t)c[u] * VW);
#pragma unroll
    for(int u = 0; u < U; ++u) {
        if(w0 + (uint64_t)u * kThreads >= total) continue;
        if(s[u] < 0 || (uint64_t)s[u] >= rows) {
            if(bad != nullptr && c[u] == 0) atomicExch(bad, 1u);
            continue;
        }
        Pack<O, VW> y;
#pragma unroll
        for(int k = 0; k < VW; ++k) y.v[k] = from_f32<O>(scale * to_f32(x[u].v[k]));
        *reinterpret_cast<Pack<O, VW> *>(out + n[u] * out_stride + (uint64_t)c[u] * VW) = y;
    }
}

/* any row: each thread makes OV consecutive elements of a contiguous out, across row borders */
template <typename T, typename O, typename I, int OV>
__global__ void __launch_bounds__(kThreads) lookup_flat_kernel(const T *__restrict__ table, uint64_t rows, uint32_t dim,
                                                               uint64_t table_stride, const I *__restrict__ index,
                                                               uint64_t total, float scale, O *__restrict__ out,
                                                               uint64_t out_stride, uint32_t *__restrict__ bad)
{
    const uint64_t e0 = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) * OV;
    if(e0 >= total) return;
    uint64_t n = total <= 0xffffffffull ? (uint64_t)((uint32_t)e0 / dim) : e0 / dim;
    uint32_t c = (uint32_t)(e0 - n * dim);
    const int m = total - e0 < (uint64_t)OV ? (int)(total - e0) : OV;
    I s = __ldg(index + n);
    bool whole = m == OV;
    Pack<O, OV> y;
    uint32_t ok = 0;
    uint64_t n_k = n;
    uint32_t c_k = c;
#pragma unroll
    for(int k = 0; k < OV; ++k) {
        if(k < m) {
            if(c_k == dim) {
                c_k = 0;
                s = __ldg(index + ++n_k);
            }
            if(s >= 0 && (uint64_t)s < rows) {
                y.v[k] = from_f32<O>(scale * to_f32(table[(uint64_t)s * table_stride + c_k]));
                ok |= 1u << k;
            } else {
                whole = false;
                if(bad != nullptr && c_k == 0) atomicExch(bad, 1u);
            }
            ++c_k;
        }
    }
    if(whole && OV > 1) {
        *reinterpret_cast<Pack<O, OV> *>(out + e0) = y; /* out_stride == dim */
        return;
    }
#pragma unroll
    for(int k = 0; k < OV; ++k) {
        if(k < m) {
            if(c == dim) {
                c = 0;
                ++n;
            }
            if(ok >> k & 1u) out[n * out_stride + c] = y.v[k];
            ++c;
        }
    }
}

template <typename T, typename O, typename I>
void launch_lookup(const void *table_, uint64_t rows, uint64_t dim, uint64_t table_stride, const void *index_,
                   uint64_t count, float scale, void *out_, uint64_t out_stride, uint32_t *bad, cudaStream_t stream)
{
    const T *table = static_cast<const T *>(table_);
    const I *index = static_cast<const I *>(index_);
    O *out = static_cast<O *>(out_);
    constexpr int VW = 16 / sizeof(T);
    constexpr int OV = 16 / sizeof(O);
    const bool packs = dim % VW == 0 && table_stride % VW == 0 && (uintptr_t)table % 16 == 0 &&
                       (out_stride * sizeof(O)) % 16 == 0 && (uintptr_t)out % 16 == 0 && dim % OV == 0;
    if(packs) {
        const uint64_t total = count * (dim / VW);
        if(total >= 148ull * 2048 * 2) {
            const uint64_t per = kThreads * 4;
            lookup_pack_kernel<T, O, I, VW, 4><<<(unsigned)((total + per - 1) / per), kThreads, 0, stream>>>(
                table, rows, (uint32_t)(dim / VW), table_stride, index, total, scale, out, out_stride, bad);
        } else {
            lookup_pack_kernel<T, O, I, VW, 1><<<(unsigned)((total + kThreads - 1) / kThreads), kThreads, 0, stream>>>(
                table, rows, (uint32_t)(dim / VW), table_stride, index, total, scale, out, out_stride, bad);
        }
        return;
    }
    const uint64_t total = count * dim;
    if(out_stride == dim && (uintptr_t)out % 16 == 0) {
        const uint64_t per = kThreads * OV;
        lookup_flat_kernel<T, O, I, OV><<<(unsigned)((total + per - 1) / per), kThreads, 0, stream>>>(
            table, rows, (uint32_t)dim, table_stride, index, total, scale, out, out_stride, bad);
    } else {
        lookup_flat_kernel<T, O, I, 1><<<(unsigned)((total + kThreads - 1) / kThreads), kThreads, 0, stream>>>(
            table, rows, (uint32_t)dim, table_stride, index, total, scale, out, out_stride, bad);
    }
}

/* ------------------------------------------------------------------------------------------ */
/* the sort of positions by row */

/* row of position i, or -1 where it takes no part */
template <typename I>
__device__ __forceinline__ int64_t row_of(const I *__restrict__ index, uint64_t i, uint64_t rows, int64_t padding,
                                          uint32_t *bad)
{
    const int64_t s = (int64_t)__ldg(index + i);
    if(s < 0 || (uint64_t)s >= rows) {
        if(bad != nullptr && s != padding) atomicExch(bad, 1u);
        return -1;
    }
    return s == padding ? -1 : s;
}

/* block-wide inclusive scan of one value per thread; s_warp holds one word per warp */
__device__ __forceinline__ uint32_t block_inclusive_scan(uint32_t v, uint32_t *s_warp, uint32_t *total)
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

/* all of a small sort in one CTA: keys (rows, ascending) and positions; *n_sorted = positions that take part */
template <typename I>
__global__ void __launch_bounds__(kSmallThreads) small_sort_kernel(const I *__restrict__ index, uint32_t count,
                                                                   uint64_t rows, int64_t padding,
                                                                   uint32_t *__restrict__ keys,
                                                                   uint32_t *__restrict__ pos,
                                                                   uint32_t *__restrict__ n_sorted,
                                                                   uint32_t *__restrict__ bad)
{
    extern __shared__ __align__(16) unsigned char smem[];
    uint32_t *s_key = reinterpret_cast<uint32_t *>(smem);         /* kSmallCount */
    uint32_t *s_pos = s_key + kSmallCount;                        /* kSmallCount */
    uint32_t *s_hist = s_pos + kSmallCount;                       /* 32 warps * 256 */
    uint32_t *s_warp = s_hist + 32 * 256;                         /* 32 */
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int items = (int)((count + kSmallThreads - 1) / kSmallThreads);
    const uint32_t wbase = (uint32_t)warp * 32u * (uint32_t)items + (uint32_t)lane;
    uint32_t k[kSmallItems], p[kSmallItems], rank[kSmallItems];
    uint32_t dropped = 0;
#pragma unroll
    for(int it = 0; it < kSmallItems; ++it) {
        k[it] = 0xffffffffu; /* after every row in each digit: behind the count, never written */
        p[it] = wbase + (uint32_t)it * 32u;
        if(it < items && p[it] < count) {
            const int64_t r = row_of(index, p[it], rows, padding, bad);
            if(r >= 0) k[it] = (uint32_t)r;
            else ++dropped;
        }
    }
    uint32_t all_dropped;
    block_inclusive_scan(dropped, s_warp, &all_dropped);
    if(threadIdx.x == 0) *n_sorted = count - all_dropped;
    /* the top digit's bits; dropped positions need a value above the last row */
    const int bits = 32 - __clz((uint32_t)(all_dropped ? rows : rows - 1));
    const int passes = bits == 0 ? 0 : (bits + 7) / 8;
    for(int pass = 0; pass < passes; ++pass) {
        const int shift = 8 * pass;
        for(int j = threadIdx.x; j < 32 * 256; j += kSmallThreads) s_hist[j] = 0u;
        __syncthreads();
        uint32_t *wh = s_hist + warp * 256;
#pragma unroll
        for(int it = 0; it < kSmallItems; ++it) {
            if(it < items) {
                const uint32_t d = (k[it] >> shift) & 255u;
                const unsigned peers = __match_any_sync(0xffffffffu, d);
                const int leader = __ffs(peers) - 1;
                uint32_t base = 0;
                if(lane == leader) {
                    base = wh[d];
                    wh[d] = base + (uint32_t)__popc(peers);
                }
                base = __shfl_sync(0xffffffffu, base, leader);
                rank[it] = base + (uint32_t)__popc(peers & ((1u << lane) - 1u));
                __syncwarp();
            }
        }
        __syncthreads();
        uint32_t sum = 0;
        if(threadIdx.x < 256) {
#pragma unroll
            for(int w = 0; w < 32; ++w) {
                const uint32_t c = s_hist[w * 256 + threadIdx.x];
                s_hist[w * 256 + threadIdx.x] = sum;
                sum += c;
            }
        }
        const uint32_t before = block_inclusive_scan(sum, s_warp, nullptr) - sum;
        if(threadIdx.x < 256) {
#pragma unroll
            for(int w = 0; w < 32; ++w) s_hist[w * 256 + threadIdx.x] += before;
        }
        __syncthreads();
#pragma unroll
        for(int it = 0; it < kSmallItems; ++it) {
            if(it < items) {
                const uint32_t to = wh[(k[it] >> shift) & 255u] + rank[it];
                s_key[to] = k[it];
                s_pos[to] = p[it];
            }
        }
        __syncthreads();
#pragma unroll
        for(int it = 0; it < kSmallItems; ++it) {
            if(it < items) {
                k[it] = s_key[wbase + (uint32_t)it * 32u];
                p[it] = s_pos[wbase + (uint32_t)it * 32u];
            }
        }
        __syncthreads();
    }
#pragma unroll
    for(int it = 0; it < kSmallItems; ++it) {
        const uint32_t i = wbase + (uint32_t)it * 32u;
        if(it < items && i < count - all_dropped) {
            keys[i] = k[it];
            pos[i] = p[it];
        }
    }
}

/* The part of a pass's input that chunk c of `chunks` covers: whole warps' shares of 32 positions. */
__device__ __forceinline__ void chunk_range(uint64_t n, uint32_t chunks, uint32_t c, uint64_t &begin, uint64_t &end)
{
    uint64_t len = (n + chunks - 1) / chunks;
    len = (len + kSortThreads - 1) / kSortThreads * kSortThreads;
    begin = (uint64_t)c * len < n ? (uint64_t)c * len : n;
    end = begin + len < n ? begin + len : n;
}

/* One digit of element i: of the index itself in the first pass (kFirst), of the pass's input pairs else.
 * Returns the digit, or -1 where the position takes no part. */
template <typename I, bool kFirst>
__device__ __forceinline__ int digit_at(const I *__restrict__ index, const uint2 *__restrict__ pairs, uint64_t i,
                                        uint64_t rows, int64_t padding, uint32_t *bad, int shift, uint32_t mask,
                                        uint32_t &key, uint32_t &p)
{
    if(kFirst) {
        const int64_t r = row_of(index, i, rows, padding, bad);
        if(r < 0) return -1;
        key = (uint32_t)r;
        p = (uint32_t)i;
    } else {
        const uint2 kp = __ldg(pairs + i);
        key = kp.x;
        p = kp.y;
    }
    return (int)((key >> shift) & mask);
}

/* digit counts of every chunk, and of all (totals, cleared by the caller) */
template <typename I, bool kFirst>
__global__ void __launch_bounds__(kSortThreads) digit_count_kernel(const I *__restrict__ index,
                                                                   const uint2 *__restrict__ pairs, uint64_t count,
                                                                   const uint32_t *__restrict__ n_pairs, uint64_t rows,
                                                                   int64_t padding, int shift, int bits,
                                                                   uint32_t *__restrict__ counts,
                                                                   uint32_t *__restrict__ totals,
                                                                   uint32_t *__restrict__ bad)
{
    __shared__ uint32_t s_hist[kMaxBins];
    const int bins = 1 << bits;
    for(int j = threadIdx.x; j < bins; j += kSortThreads) s_hist[j] = 0u;
    __syncthreads();
    uint64_t begin, end;
    chunk_range(kFirst ? count : (uint64_t)*n_pairs, gridDim.x, blockIdx.x, begin, end);
    for(uint64_t i = begin + threadIdx.x; i < end; i += kSortThreads) {
        uint32_t key, p;
        const int d = digit_at<I, kFirst>(index, pairs, i, rows, padding, bad, shift, (uint32_t)bins - 1u, key, p);
        if(d >= 0) atomicAdd(&s_hist[d], 1u);
    }
    __syncthreads();
    for(int j = threadIdx.x; j < bins; j += kSortThreads) {
        const uint32_t v = s_hist[j];
        counts[(uint64_t)blockIdx.x * bins + j] = v;
        if(v) atomicAdd(&totals[j], v);
    }
}

/* counts[c][d] -> first output place of chunk c's digit d; starts[d] = first place of digit d (starts[bins] = all).
 * A CTA owns 32 digits: 32 x 32 threads, each adding up a 32nd of the chunks. */
__global__ void __launch_bounds__(1024) digit_scan_kernel(uint32_t *__restrict__ counts, uint32_t chunks, int bins,
                                                          const uint32_t *__restrict__ totals,
                                                          uint32_t *__restrict__ starts, uint32_t *__restrict__ n_sorted)
{
    __shared__ uint32_t s_part[32][33];
    __shared__ uint32_t s_warp[32];
    __shared__ uint32_t s_base[32];
    const int dl = threadIdx.x & 31, cl = threadIdx.x >> 5;
    const int d0 = blockIdx.x * 32, d = d0 + dl;
    /* everything before this CTA's digits */
    uint32_t before = 0;
    for(int j = threadIdx.x; j < d0; j += 1024) before += totals[j];
    uint32_t base;
    block_inclusive_scan(before, s_warp, &base);
    const uint32_t per = (chunks + 31) / 32;
    const uint32_t c0 = (uint32_t)cl * per, c1 = c0 + per < chunks ? c0 + per : chunks;
    uint32_t sum = 0;
    if(d < bins)
        for(uint32_t c = c0; c < c1; ++c) sum += counts[(uint64_t)c * bins + d];
    s_part[cl][dl] = sum;
    if(cl == 0) {
        const uint32_t t = d < bins ? totals[d] : 0u;
        uint32_t v = t;
#pragma unroll
        for(int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
            if(dl >= o) v += u;
        }
        s_base[dl] = base + v - t;
        if(d < bins) starts[d] = base + v - t;
        if(d == bins - 1) {
            starts[bins] = base + v;
            *n_sorted = base + v;
        }
    }
    __syncthreads();
    uint32_t run = s_base[dl];
    for(int w = 0; w < cl; ++w) run += s_part[w][dl];
    if(d < bins)
        for(uint32_t c = c0; c < c1; ++c) {
            const uint32_t v = counts[(uint64_t)c * bins + d];
            counts[(uint64_t)c * bins + d] = run;
            run += v;
        }
}

/* each element to its place, in input order within a digit.  kLast writes positions (and keys, where the caller
 * needs them), the other passes write (key, position) pairs.  Shared memory: a 16-bit count of every digit for
 * each warp, which becomes the warp's next place within the chunk's run, and the chunk's first places. */
template <typename I, bool kFirst, bool kLast>
__global__ void __launch_bounds__(kSortThreads) digit_scatter_kernel(
    const I *__restrict__ index, const uint2 *__restrict__ pairs, uint64_t count, const uint32_t *__restrict__ n_pairs,
    uint64_t rows, int64_t padding, int shift, int bits, const uint32_t *__restrict__ places, uint2 *__restrict__ pairs_out,
    uint32_t *__restrict__ keys_out, uint32_t *__restrict__ pos_out)
{
    extern __shared__ __align__(16) unsigned char smem[];
    const int bins = 1 << bits;
    const int words = bins > 1 ? bins / 2 : 1;                            /* two counts a word */
    uint32_t *s_place = reinterpret_cast<uint32_t *>(smem);               /* bins */
    uint32_t *s_count = s_place + bins;                                   /* kSortWarps * words */
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for(int j = threadIdx.x; j < kSortWarps * words; j += kSortThreads) s_count[j] = 0u;
    for(int j = threadIdx.x; j < bins; j += kSortThreads) s_place[j] = places[(uint64_t)blockIdx.x * bins + j];
    __syncthreads();
    uint64_t begin, end;
    chunk_range(kFirst ? count : (uint64_t)*n_pairs, gridDim.x, blockIdx.x, begin, end);
    const uint64_t share = (end - begin + kSortThreads - 1) / kSortThreads * 32;
    const uint64_t w0 = begin + share * warp < end ? begin + share * warp : end;
    const uint64_t w1 = w0 + share < end ? w0 + share : end;
    uint32_t *mine = s_count + warp * words;
    uint16_t *mine16 = reinterpret_cast<uint16_t *>(mine);
    for(uint64_t i = w0 + lane; i < w1; i += 32) {
        uint32_t key, p;
        const int d = digit_at<I, kFirst>(index, pairs, i, rows, padding, nullptr, shift, (uint32_t)bins - 1u, key, p);
        if(d >= 0) atomicAdd(&mine[d >> 1], 1u << (16 * (d & 1)));
    }
    __syncthreads();
    /* counts -> exclusive prefix over the warps, both halves of a word at once (no half exceeds kMaxChunk) */
    for(int j = threadIdx.x; j < words; j += kSortThreads) {
        uint32_t run = 0;
#pragma unroll
        for(int w = 0; w < kSortWarps; ++w) {
            const uint32_t v = s_count[w * words + j];
            s_count[w * words + j] = run;
            run += v;
        }
    }
    __syncthreads();
    for(uint64_t i0 = w0; i0 < w1; i0 += 32) {
        const uint64_t i = i0 + lane;
        uint32_t key = 0, p = 0;
        int d = -1;
        if(i < w1) d = digit_at<I, kFirst>(index, pairs, i, rows, padding, nullptr, shift, (uint32_t)bins - 1u, key, p);
        const unsigned peers = __match_any_sync(0xffffffffu, d);
        const int leader = __ffs(peers) - 1;
        uint32_t base = 0;
        if(lane == leader && d >= 0) {
            base = mine16[d];
            mine16[d] = (uint16_t)(base + (uint32_t)__popc(peers));
        }
        base = __shfl_sync(0xffffffffu, base, leader);
        __syncwarp();
        if(d >= 0) {
            const uint32_t to = s_place[d] + base + (uint32_t)__popc(peers & ((1u << lane) - 1u));
            if(kLast) {
                pos_out[to] = p;
                if(keys_out != nullptr) keys_out[to] = key;
            } else {
                pairs_out[to] = make_uint2(key, p);
            }
        }
    }
}

/* ------------------------------------------------------------------------------------------ */
/* sums by row */

/* What the sums read: the sorted positions, and where each row's begin: starts[v] where the sort gives them
 * (tables of one pass), else the sorted keys, searched. */
struct Sorted {
    const uint32_t *pos;
    const uint32_t *keys;
    const uint32_t *starts;
    const uint32_t *n_sorted;
    uint64_t rows;
};

/* first place whose key is at least `row` */
__device__ __forceinline__ uint32_t first_of(const Sorted &s, uint32_t n, uint64_t row)
{
    if(row >= s.rows) return n;
    if(s.starts != nullptr) return __ldg(s.starts + row);
    uint32_t lo = 0, len = n;
    while(len > 0) {
        const uint32_t half = len / 2;
        if((uint64_t)__ldg(s.keys + lo + half) < row) {
            lo += half + 1;
            len -= half + 1;
        } else {
            len = half;
        }
    }
    return lo;
}

/* How a warp covers columns and positions: 2^clog lanes side by side take VW columns each (NR times, side by side),
 * the 32 >> clog groups of such lanes take every so-manieth position. */
template <typename GT, int VW, int NR>
__device__ __forceinline__ void add_positions(float (&acc)[NR * VW], const GT *__restrict__ grad, uint64_t stride,
                                              const uint32_t *__restrict__ pos, uint32_t s, uint32_t e, int lane,
                                              int clog, uint32_t col0, uint32_t dim)
{
    constexpr int U = NR * VW >= 16 ? 2 : 4;
    const int cl = 1 << clog, pl = 32 >> clog;
    const int cg = lane & (cl - 1), pg = lane >> clog;
    for(uint32_t base = s; base < e; base += 32) {
        const int m = e - base < 32u ? (int)(e - base) : 32;
        const uint32_t mine = lane < m ? __ldg(pos + base + lane) : 0u;
        for(int k = 0; k < m; k += pl * U) {
            Pack<GT, VW> x[U][NR];
            bool in[U];
#pragma unroll
            for(int u = 0; u < U; ++u) {
                const int at = k + u * pl + pg;
                const uint32_t q = __shfl_sync(0xffffffffu, mine, at & 31);
                in[u] = at < m;
#pragma unroll
                for(int r = 0; r < NR; ++r) {
                    const uint32_t c = col0 + (uint32_t)((r * cl + cg) * VW);
                    if(in[u] && c < dim)
                        x[u][r] = *reinterpret_cast<const Pack<GT, VW> *>(grad + (uint64_t)q * stride + c);
                }
            }
#pragma unroll
            for(int u = 0; u < U; ++u)
#pragma unroll
                for(int r = 0; r < NR; ++r) {
                    const uint32_t c = col0 + (uint32_t)((r * cl + cg) * VW);
                    if(in[u] && c < dim)
#pragma unroll
                        for(int v = 0; v < VW; ++v) acc[r * VW + v] += to_f32(x[u][r].v[v]);
                }
        }
    }
}

/* the groups' sums of a warp, added up (every lane of a column group gets the sum) */
template <int N>
__device__ __forceinline__ void join_groups(float (&acc)[N], int clog)
{
    for(int o = 1 << clog; o < 32; o <<= 1)
#pragma unroll
        for(int v = 0; v < N; ++v) acc[v] += __shfl_xor_sync(0xffffffffu, acc[v], o);
}

/* every warp's sums -> warp 0's, through shared memory, in the order of the warps */
template <int N>
__device__ __forceinline__ void join_warps(float (&acc)[N], float *s_join, int clog)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if(lane < (1 << clog))
#pragma unroll
        for(int v = 0; v < N; ++v) s_join[(warp * N + v) * 32 + lane] = acc[v];
    __syncthreads();
    if(warp == 0 && lane < (1 << clog))
        for(int w = 1; w < kWarps; ++w)
#pragma unroll
            for(int v = 0; v < N; ++v) acc[v] += s_join[(w * N + v) * 32 + lane];
}

/* partial[p] = sum of piece p, where the piece lies in one row */
template <typename GT, int VW, int NR>
__global__ void __launch_bounds__(kThreads) piece_sum_kernel(const GT *__restrict__ grad, uint64_t stride, Sorted sorted,
                                                             float *__restrict__ partial, uint32_t partial_stride,
                                                             uint32_t dim, int clog)
{
    __shared__ float s_join[kWarps * 32 * NR * VW];
    __shared__ int s_in_one;
    const uint32_t n = *sorted.n_sorted;
    const uint64_t b = (uint64_t)blockIdx.x * kPiece;
    if(b + kPiece > n) return;
    if(threadIdx.x == 0) {
        if(sorted.starts != nullptr) {
            /* last row that starts at or before b */
            uint64_t lo = 0, len = sorted.rows;
            while(len > 0) {
                const uint64_t half = len / 2;
                if((uint64_t)__ldg(sorted.starts + lo + half) <= b) {
                    lo += half + 1;
                    len -= half + 1;
                } else {
                    len = half;
                }
            }
            s_in_one = (lo < sorted.rows ? __ldg(sorted.starts + lo) : n) >= b + kPiece;
        } else {
            s_in_one = __ldg(sorted.keys + b) == __ldg(sorted.keys + b + kPiece - 1);
        }
    }
    __syncthreads();
    if(!s_in_one) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t col0 = blockIdx.y * (uint32_t)(NR * VW << clog);
    float acc[NR * VW] = {};
    constexpr uint32_t share = kPiece / kWarps;
    const uint32_t s = (uint32_t)b + share * (uint32_t)warp;
    add_positions<GT, VW, NR>(acc, grad, stride, sorted.pos, s, s + share, lane, clog, col0, dim);
    join_groups(acc, clog);
    join_warps(acc, s_join, clog);
    if(warp == 0 && lane < (1 << clog)) {
#pragma unroll
        for(int r = 0; r < NR; ++r) {
            const uint32_t c = col0 + (uint32_t)(((r << clog) + lane) * VW);
            if(c < dim)
#pragma unroll
                for(int v = 0; v < VW; ++v)
                    if(c + v < dim) partial[(uint64_t)blockIdx.x * partial_stride + c + v] = acc[r * VW + v];
        }
    }
}

template <typename TT, int VW, int NR>
__device__ __forceinline__ void store_row(const float (&acc)[NR * VW], TT *__restrict__ row, float scale, bool accumulate,
                                          int lane, int clog, uint32_t col0, uint32_t dim)
{
    if(lane >= (1 << clog)) return;
#pragma unroll
    for(int r = 0; r < NR; ++r) {
        const uint32_t c = col0 + (uint32_t)(((r << clog) + lane) * VW);
        if(c >= dim) continue;
        Pack<TT, VW> y;
        if(accumulate) y = *reinterpret_cast<const Pack<TT, VW> *>(row + c);
#pragma unroll
        for(int v = 0; v < VW; ++v)
            y.v[v] = from_f32<TT>(accumulate ? fmaf(scale, acc[r * VW + v], to_f32(y.v[v])) : scale * acc[r * VW + v]);
        *reinterpret_cast<Pack<TT, VW> *>(row + c) = y;
    }
}

/* grad_table[v] for the rows of this CTA (rows_per_cta from blockIdx.x on) and its columns (blockIdx.y) */
constexpr int kMaxRowsPerCta = 64;
template <typename GT, typename TT, int VW, int NR>
__global__ void __launch_bounds__(kThreads) row_sum_kernel(const GT *__restrict__ grad, uint64_t stride, Sorted sorted,
                                                           const float *__restrict__ partial, uint32_t partial_stride,
                                                           float scale, TT *__restrict__ table, uint64_t table_stride,
                                                           uint32_t dim, int clog, int rows_per_cta, bool accumulate)
{
    __shared__ uint32_t s_start[kMaxRowsPerCta + 1];
    __shared__ float s_join[kWarps * 32 * NR * VW];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t n = *sorted.n_sorted;
    const uint64_t row0 = (uint64_t)blockIdx.x * rows_per_cta;
    if((int)threadIdx.x <= rows_per_cta) s_start[threadIdx.x] = first_of(sorted, n, row0 + threadIdx.x);
    __syncthreads();
    const uint32_t col0 = blockIdx.y * (uint32_t)(NR * VW << clog);
    bool any_long = false;
    for(int r = 0; r < rows_per_cta; ++r) {
        const uint64_t v = row0 + r;
        if(v >= sorted.rows) break;
        const uint32_t s = s_start[r], e = s_start[r + 1];
        if(e - s > (uint32_t)kWarpMax) {
            any_long = true;
            continue;
        }
        if((r % kWarps) != warp || (accumulate && s == e)) continue;
        float acc[NR * VW] = {};
        add_positions<GT, VW, NR>(acc, grad, stride, sorted.pos, s, e, lane, clog, col0, dim);
        if(s != e) join_groups(acc, clog);
        store_row<TT, VW, NR>(acc, table + v * table_stride, scale, accumulate, lane, clog, col0, dim);
    }
    if(!any_long) return;
    for(int r = 0; r < rows_per_cta; ++r) {
        const uint64_t v = row0 + r;
        if(v >= sorted.rows) break;
        const uint32_t s = s_start[r], e = s_start[r + 1];
        if(e - s <= (uint32_t)kWarpMax) continue;
        float acc[NR * VW] = {};
        /* whole pieces inside the row were summed by piece_sum_kernel */
        const uint32_t p0 = (s + kPiece - 1) / kPiece, p1 = e / kPiece;
        const uint32_t head_end = p0 < p1 ? p0 * kPiece : e, tail = p0 < p1 ? p1 * kPiece : e;
        const uint32_t hshare = (head_end - s + kWarps - 1) / kWarps, tshare = (e - tail + kWarps - 1) / kWarps;
        const uint32_t h0 = s + hshare * warp < head_end ? s + hshare * warp : head_end;
        const uint32_t h1 = h0 + hshare < head_end ? h0 + hshare : head_end;
        add_positions<GT, VW, NR>(acc, grad, stride, sorted.pos, h0, h1, lane, clog, col0, dim);
        const int pg = lane >> clog, pl = 32 >> clog;
        for(uint32_t p = p0 + (uint32_t)(warp * pl + pg); p < p1; p += (uint32_t)(kWarps * pl)) {
#pragma unroll
            for(int k = 0; k < NR; ++k) {
                const uint32_t c = col0 + (uint32_t)(((k << clog) + (lane & ((1 << clog) - 1))) * VW);
#pragma unroll
                for(int w = 0; w < VW; ++w)
                    if(c + w < dim) acc[k * VW + w] += __ldg(partial + (uint64_t)p * partial_stride + c + w);
            }
        }
        const uint32_t t0 = tail + tshare * warp < e ? tail + tshare * warp : e;
        const uint32_t t1 = t0 + tshare < e ? t0 + tshare : e;
        add_positions<GT, VW, NR>(acc, grad, stride, sorted.pos, t0, t1, lane, clog, col0, dim);
        join_groups(acc, clog);
        join_warps(acc, s_join, clog);
        if(warp == 0) store_row<TT, VW, NR>(acc, table + v * table_stride, scale, accumulate, lane, clog, col0, dim);
    }
}

template <typename GT, typename TT, int VW, int NR>
void launch_sums(const GT *grad, uint64_t grad_stride, const Sorted &sorted, uint64_t count, float *partial,
                 float scale, TT *table, uint64_t table_stride, uint64_t dim, bool accumulate, cudaStream_t stream)
{
    int clog = 0;
    while(clog < 5 && ((uint64_t)(NR * VW) << clog) < dim) ++clog;
    const uint64_t cols = (uint64_t)(NR * VW) << clog;
    const unsigned tiles = (unsigned)((dim + cols - 1) / cols);
    if(count >= (uint64_t)kPiece)
        piece_sum_kernel<GT, VW, NR><<<dim3((unsigned)(count / kPiece), tiles), kThreads, 0, stream>>>(
            grad, grad_stride, sorted, partial, (uint32_t)dim, (uint32_t)dim, clog);
    /* few rows: one to a warp, so that they spread over the GPU; many: 64 share a CTA's searches */
    int rows_per_cta = kWarps;
    while(rows_per_cta < kMaxRowsPerCta && (sorted.rows / (uint64_t)rows_per_cta) * tiles > 148 * 16) rows_per_cta *= 2;
    const unsigned ctas = (unsigned)((sorted.rows + rows_per_cta - 1) / rows_per_cta);
    row_sum_kernel<GT, TT, VW, NR><<<dim3(ctas, tiles), kThreads, 0, stream>>>(
        grad, grad_stride, sorted, partial, (uint32_t)dim, scale, table, table_stride, (uint32_t)dim, clog, rows_per_cta,
        accumulate);
}

template <typename GT, typename TT>
void launch_sums_typed(const void *grad_, uint64_t grad_stride, const Sorted &sorted, uint64_t count, float *partial,
                       float scale, void *table_, uint64_t table_stride, uint64_t dim, bool accumulate,
                       cudaStream_t stream)
{
    const GT *grad = static_cast<const GT *>(grad_);
    TT *table = static_cast<TT *>(table_);
    constexpr int VW = 16 / sizeof(GT);
    constexpr uint64_t TA = VW * sizeof(TT) < 16 ? VW * sizeof(TT) : 16;
    if(dim % VW == 0 && grad_stride % VW == 0 && (uintptr_t)grad % 16 == 0 && (uintptr_t)table % TA == 0 &&
       (table_stride * sizeof(TT)) % TA == 0) {
        if(dim > 32 * VW) launch_sums<GT, TT, VW, 2>(grad, grad_stride, sorted, count, partial, scale, table, table_stride, dim, accumulate, stream);
        else launch_sums<GT, TT, VW, 1>(grad, grad_stride, sorted, count, partial, scale, table, table_stride, dim, accumulate, stream);
    } else {
        if(dim > 32) launch_sums<GT, TT, 1, 2>(grad, grad_stride, sorted, count, partial, scale, table, table_stride, dim, accumulate, stream);
        else launch_sums<GT, TT, 1, 1>(grad, grad_stride, sorted, count, partial, scale, table, table_stride, dim, accumulate, stream);
    }
}

/* ------------------------------------------------------------------------------------------ */
/* workspace: n_sorted | totals, starts | counts | pairs, keys, positions | partial sums */

struct Plan {
    int passes = 0; /* 0: the one-CTA sort */
    int bits[4] = {};
    uint32_t chunks = 0;
    size_t o_words = 0, o_starts = 0, o_counts = 0, o_pairs = 0, o_pairs2 = 0, o_keys = 0, o_pos = 0, o_partial = 0, bytes = 0;
};

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

Plan make_plan(uint64_t count, uint64_t rows, uint64_t dim)
{
    Plan p;
    size_t o = 256;
    if(count > (uint64_t)kSmallCount) {
        int bits = 0;
        while(bits < 32 && (rows - 1) >> bits) ++bits;
        if(bits == 0) bits = 1;
        p.passes = (bits + kMaxBits - 1) / kMaxBits;
        for(int i = 0; i < p.passes; ++i) {
            p.bits[i] = (bits + p.passes - 1 - i) / (p.passes - i);
            bits -= p.bits[i];
        }
        uint64_t chunks = (count + 4095) / 4096;
        if(chunks > (uint64_t)kChunks) chunks = kChunks;
        const uint64_t least = (count + kMaxChunk - kSortThreads - 1) / (kMaxChunk - kSortThreads);
        if(chunks < least) chunks = least;
        p.chunks = (uint32_t)chunks;
        p.o_words = o;
        o += align256(sizeof(uint32_t) * kMaxBins) * p.passes; /* totals of every pass */
        p.o_starts = o;
        o += align256(sizeof(uint32_t) * (kMaxBins + 1));
        p.o_counts = o;
        o += align256(sizeof(uint32_t) * chunks << p.bits[0]);
        if(p.passes > 1) {
            p.o_pairs = o;
            o += align256(sizeof(uint2) * count);
        }
        if(p.passes > 2) {
            p.o_pairs2 = o;
            o += align256(sizeof(uint2) * count);
        }
    }
    if(p.passes != 1) {
        p.o_keys = o;
        o += align256(sizeof(uint32_t) * count);
    }
    p.o_pos = o;
    o += align256(sizeof(uint32_t) * count);
    p.o_partial = o;
    o += align256(sizeof(float) * (count / kPiece) * dim);
    p.bytes = o;
    return p;
}

size_t small_smem() { return sizeof(uint32_t) * (2 * kSmallCount + 32 * 256 + 32); }
size_t scatter_smem(int bits)
{
    const size_t bins = (size_t)1 << bits;
    return sizeof(uint32_t) * (bins + kSortWarps * (bins > 1 ? bins / 2 : 1));
}

template <typename K>
cudaError_t allow_smem(K kernel, size_t bytes)
{
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <typename I, bool kFirst, bool kLast>
cudaError_t launch_pass(const I *index, const uint2 *pairs, uint64_t count, uint32_t *n_sorted, uint64_t rows,
                        int64_t padding, int shift, int bits, uint32_t chunks, uint32_t *totals, uint32_t *starts,
                        uint32_t *counts, uint2 *pairs_out, uint32_t *keys_out, uint32_t *pos_out, uint32_t *bad,
                        cudaStream_t stream)
{
    const cudaError_t e = allow_smem(digit_scatter_kernel<I, kFirst, kLast>, scatter_smem(kMaxBits));
    if(e != cudaSuccess) return e;
    const int bins = 1 << bits;
    digit_count_kernel<I, kFirst><<<chunks, kSortThreads, 0, stream>>>(index, pairs, count, n_sorted, rows, padding,
                                                                       shift, bits, counts, totals, bad);
    digit_scan_kernel<<<(bins + 31) / 32, 1024, 0, stream>>>(counts, chunks, bins, totals, starts, n_sorted);
    digit_scatter_kernel<I, kFirst, kLast><<<chunks, kSortThreads, scatter_smem(bits), stream>>>(
        index, pairs, count, n_sorted, rows, padding, shift, bits, counts, pairs_out, keys_out, pos_out);
    return cudaSuccess;
}

template <typename I>
cudaError_t launch_sort(const Plan &plan, unsigned char *ws, const void *index_, uint64_t count, uint64_t rows,
                        int64_t padding, uint32_t *bad, cudaStream_t stream)
{
    const I *index = static_cast<const I *>(index_);
    uint32_t *n_sorted = reinterpret_cast<uint32_t *>(ws);
    uint32_t *keys = plan.passes != 1 ? reinterpret_cast<uint32_t *>(ws + plan.o_keys) : nullptr;
    uint32_t *pos = reinterpret_cast<uint32_t *>(ws + plan.o_pos);
    if(plan.passes == 0) {
        const cudaError_t e = allow_smem(small_sort_kernel<I>, small_smem());
        if(e != cudaSuccess) return e;
        small_sort_kernel<I><<<1, kSmallThreads, small_smem(), stream>>>(index, (uint32_t)count, rows, padding, keys,
                                                                         pos, n_sorted, bad);
        return cudaSuccess;
    }
    const size_t each = align256(sizeof(uint32_t) * kMaxBins);
    cudaError_t e = cudaMemsetAsync(ws + plan.o_words, 0, each * plan.passes, stream);
    if(e != cudaSuccess) return e;
    uint32_t *starts = reinterpret_cast<uint32_t *>(ws + plan.o_starts);
    uint32_t *counts = reinterpret_cast<uint32_t *>(ws + plan.o_counts);
    uint2 *from = nullptr, *to = reinterpret_cast<uint2 *>(ws + plan.o_pairs);
    int shift = 0;
    for(int p = 0; p < plan.passes; ++p) {
        uint32_t *totals = reinterpret_cast<uint32_t *>(ws + plan.o_words + each * p);
        const bool first = p == 0, last = p == plan.passes - 1;
        if(first && last)
            e = launch_pass<I, true, true>(index, nullptr, count, n_sorted, rows, padding, shift, plan.bits[p], plan.chunks,
                                           totals, starts, counts, nullptr, keys, pos, bad, stream);
        else if(first)
            e = launch_pass<I, true, false>(index, nullptr, count, n_sorted, rows, padding, shift, plan.bits[p],
                                            plan.chunks, totals, starts, counts, to, nullptr, nullptr, bad, stream);
        else if(!last)
            e = launch_pass<I, false, false>(index, from, count, n_sorted, rows, padding, shift, plan.bits[p],
                                             plan.chunks, totals, starts, counts, to, nullptr, nullptr, bad, stream);
        else
            e = launch_pass<I, false, true>(index, from, count, n_sorted, rows, padding, shift, plan.bits[p],
                                            plan.chunks, totals, starts, counts, nullptr, keys, pos, bad, stream);
        if(e != cudaSuccess) return e;
        shift += plan.bits[p];
        from = to;
        to = reinterpret_cast<uint2 *>(ws + (p % 2 == 0 && plan.passes > 2 ? plan.o_pairs2 : plan.o_pairs));
    }
    return cudaSuccess;
}

bool float_type(int t) { return t == GSX_B200_DATA_F32 || t == GSX_B200_DATA_F16 || t == GSX_B200_DATA_BF16; }
uint64_t float_bytes(int t) { return t == GSX_B200_DATA_F32 ? 4 : 2; }

int launch_status(cudaError_t e)
{
    const cudaError_t last = cudaGetLastError();
    if(e == cudaSuccess) e = last;
    return e == cudaSuccess ? GSX_B200_SUCCESS : gsx_internal_fail(GSX_B200_UNKNOWN, cudaGetErrorString(e));
}

int check_shape(uint64_t rows, uint64_t dim, uint64_t stride_a, uint64_t stride_b, uint64_t count)
{
    if(rows > (uint64_t)INT32_MAX || dim > (uint64_t)INT32_MAX || count > (uint64_t)INT32_MAX)
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "rows, dim and count must be below 2^31");
    if(stride_a < dim || stride_b < dim)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "row strides must be at least dim elements");
    if(stride_a > (1ull << 40) || stride_b > (1ull << 40))
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "row strides must be at most 2^40 elements");
    return 0;
}

} // namespace

/* T is the element type named by `t`; the calls below are written out once per pair of types */
#define GSX_WITH_FLOAT_TYPE(t, T, ...)                            \
    do {                                                          \
        if((t) == GSX_B200_DATA_F32) { using T = float; __VA_ARGS__; }           \
        else if((t) == GSX_B200_DATA_F16) { using T = __half; __VA_ARGS__; }     \
        else { using T = __nv_bfloat16; __VA_ARGS__; }                           \
    } while(0)

extern "C" int gsx_b200_embedding_lookup(const void *table, int table_type, uint64_t rows, uint64_t dim,
                                         uint64_t table_stride, const void *index, int index_type, uint64_t count,
                                         float scale, void *out, int out_type, uint64_t out_stride,
                                         uint32_t *device_out_of_range, void *stream_)
{
    if(!float_type(table_type) || !float_type(out_type))
        return gsx_internal_fail(GSX_B200_NOT_SUPPORTED, "embedding tables and outputs are f32, f16 or bf16");
    if(index_type != GSX_B200_DATA_I32 && index_type != GSX_B200_DATA_I64)
        return gsx_internal_fail(GSX_B200_NOT_SUPPORTED, "embedding indices are i32 or i64");
    if(int rc = check_shape(rows, dim, table_stride, out_stride, count)) return rc;
    if(count == 0 || dim == 0) return GSX_B200_SUCCESS;
    if((rows > 0 && table == nullptr) || index == nullptr || out == nullptr)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "table, index and out must be non-null");
    if((uintptr_t)table % float_bytes(table_type) || (uintptr_t)out % float_bytes(out_type) ||
       (uintptr_t)index % (index_type == GSX_B200_DATA_I32 ? 4 : 8))
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "pointers must be aligned to their element type");
    if(count * dim / 256 > (uint64_t)INT32_MAX)
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "count * dim must be below 2^39");
    cudaStream_t stream = (cudaStream_t)stream_;
    GSX_WITH_FLOAT_TYPE(table_type, T, GSX_WITH_FLOAT_TYPE(out_type, O, {
        if(index_type == GSX_B200_DATA_I32)
            launch_lookup<T, O, int32_t>(table, rows, dim, table_stride, index, count, scale, out, out_stride,
                                         device_out_of_range, stream);
        else
            launch_lookup<T, O, int64_t>(table, rows, dim, table_stride, index, count, scale, out, out_stride,
                                         device_out_of_range, stream);
    }));
    return launch_status(cudaSuccess);
}

extern "C" uint64_t gsx_b200_embedding_workspace_bytes(uint64_t count, uint64_t rows, uint64_t dim)
{
    if(count > (uint64_t)INT32_MAX || rows > (uint64_t)INT32_MAX || dim > (uint64_t)INT32_MAX || rows == 0) return 0;
    return make_plan(count, rows, dim).bytes;
}

extern "C" int gsx_b200_embedding_backward(const void *grad_out, int grad_type, uint64_t grad_stride, const void *index,
                                           int index_type, uint64_t count, float scale, int64_t padding_row,
                                           void *grad_table, int table_type, uint64_t rows, uint64_t dim,
                                           uint64_t table_stride, int accumulate, void *workspace,
                                           uint64_t workspace_bytes, uint32_t *device_out_of_range, void *stream_)
{
    if(!float_type(grad_type) || !float_type(table_type))
        return gsx_internal_fail(GSX_B200_NOT_SUPPORTED, "embedding gradients are f32, f16 or bf16");
    if(index_type != GSX_B200_DATA_I32 && index_type != GSX_B200_DATA_I64)
        return gsx_internal_fail(GSX_B200_NOT_SUPPORTED, "embedding indices are i32 or i64");
    if(int rc = check_shape(rows, dim, grad_stride, table_stride, count)) return rc;
    if(dim > 65535ull * 32) return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "dim must be at most 2097120");
    if(padding_row >= (int64_t)rows) return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "padding_row must be below rows");
    if(dim == 0 || (rows == 0 && count == 0)) return GSX_B200_SUCCESS;
    if(rows == 0) return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "rows must be positive");
    if(grad_table == nullptr || workspace == nullptr || (count > 0 && (grad_out == nullptr || index == nullptr)))
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "grad_out, index, grad_table and workspace must be non-null");
    if((uintptr_t)grad_out % float_bytes(grad_type) || (uintptr_t)grad_table % float_bytes(table_type) ||
       (uintptr_t)index % (index_type == GSX_B200_DATA_I32 ? 4 : 8) || (uintptr_t)workspace % 16)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT,
                                 "pointers must be aligned to their element type, the workspace to 16 bytes");
    const Plan plan = make_plan(count, rows, dim);
    if(workspace_bytes < plan.bytes)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT,
                                 "workspace is smaller than gsx_b200_embedding_workspace_bytes");
    cudaStream_t stream = (cudaStream_t)stream_;
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    const cudaError_t e = index_type == GSX_B200_DATA_I32
                              ? launch_sort<int32_t>(plan, ws, index, count, rows, padding_row, device_out_of_range, stream)
                              : launch_sort<int64_t>(plan, ws, index, count, rows, padding_row, device_out_of_range, stream);
    if(e != cudaSuccess) return launch_status(e);
    Sorted sorted;
    sorted.pos = reinterpret_cast<const uint32_t *>(ws + plan.o_pos);
    sorted.keys = plan.passes != 1 ? reinterpret_cast<const uint32_t *>(ws + plan.o_keys) : nullptr;
    sorted.starts = plan.passes == 1 ? reinterpret_cast<const uint32_t *>(ws + plan.o_starts) : nullptr;
    sorted.n_sorted = reinterpret_cast<const uint32_t *>(ws);
    sorted.rows = rows;
    float *partial = reinterpret_cast<float *>(ws + plan.o_partial);
    GSX_WITH_FLOAT_TYPE(grad_type, GT, GSX_WITH_FLOAT_TYPE(table_type, TT, {
        launch_sums_typed<GT, TT>(grad_out, grad_stride, sorted, count, partial, scale, grad_table, table_stride, dim,
                                  accumulate != 0, stream);
    }));
    return launch_status(cudaSuccess);
}
