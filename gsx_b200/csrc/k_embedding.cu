/*
 * Shared rows: out[n] = scale * table[index[n]], and the gradient of the table.
 *
 * Lookup.  It reads the indices and the table's rows (mostly from L2) and writes out; what bounds it is the writing of
 * out and, for rows that are no whole number of packs, the instructions an element.  Three forms, by the row: packs of
 * 16, 8 or 4 bytes; up to four elements (a thread makes whole rows, small tables lie in shared memory); any other (lanes
 * side by side on a row's elements).
 *
 * Gradient.  grad_table[v] = scale * sum of grad_out[n] over the n with index[n] = v.  No floating-point atomics: the
 * order of the additions is fixed by the sizes, the types, and the alignment and strides that decide between packs and
 * single elements, so the same call gives the same bits.
 *   sort    a stable sort of (row, position) by the row's bits, in digits of at most 8.  Up to small_count positions: one
 *           CTA, in shared memory, while other CTAs write the table's zeros.  More: per digit the counts of up to 148 chunks,
 *           then a scatter in which every CTA adds up the chunks' counts itself and ranks its chunk in tiles.  Positions
 *           whose index is the padding row or out of range are dropped in the first pass.
 *   sums    every CTA takes as many sorted positions as the others, whatever their rows: rows of any popularity cost the
 *           same (a warp for each row took 3 to 4 times as long on skewed indices).  Groups of lanes walk runs of
 *           positions with the gradients of the next ones in flight; rows that cross runs or CTAs are joined in order.
 *   small tables of short rows skip the sort: CTAs with tables of sums in shared memory (own_table_kernel).
 * The kernels of a call are launched so that each starts while the one before ends (gsx_launch_pdl).
 *
 * Sums are held in 32 bits.  No chain of additions is longer than a run (128 positions), plus one term for every group
 * of a CTA (64), plus one for every CTA that a row crosses up to 16 of them, beyond that an eighth of them and eight.  In the
 * tables in shared memory a chain has the row's positions of a chunk (512, or a 296th of all where that is more, to the next
 * 32), plus an eighth of the chunks (37) and eight.
 */
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/gsx_b200.h"
#include "gsx_b200_kernels.cuh"

int gsx_internal_fail(int code, const char *msg);

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSmallThreads = 1024;
/* Positions a thread that one CTA sorts.  Of 4000 and 8100 positions in 4650 rows the whole gradient takes 20 and 28 us so,
 * 25 and 26 with the longer sort; a sort of all digits in one cluster of CTAs took 23 and 24.  Beside the zeros of a large
 * table the one CTA costs nothing: 8191 positions and 268 MB take 57 us, with the longer sort, whose four launches end
 * with their zeros, 67; 67 MB take 29 and 27. */
constexpr int kSmallItems = 5, kBesideItems = 8;
constexpr uint64_t kBesideTable = 1u << 25; /* elements */
constexpr uint64_t small_count(uint64_t rows, uint64_t dim)
{
    return (uint64_t)kSmallThreads * (rows * dim > kBesideTable ? kBesideItems : kSmallItems);
}
constexpr int kSortThreads = 1024;
constexpr int kSortItems = 8;
constexpr int kTile = kSortThreads * kSortItems; /* pairs that a CTA of the longer sort ranks at once */
constexpr int kMaxBits = 8;
constexpr int kMaxBins = 1 << kMaxBits;
constexpr int kChunks = 148; /* CTAs of a pass: one an SM */

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

/* an index as a row number, or a number no table has */
template <typename I>
__device__ __forceinline__ uint32_t row_number(I v)
{
    return sizeof(I) == 8 && ((uint64_t)v >> 32) != 0 ? UINT32_MAX : (uint32_t)v;
}

/* i / d for i < 2^31 by one multiplication (division by an invariant, Granlund and Montgomery 1994): with 2^s >= d
 * and m = floor(2^(31 + s) / d) + 1, i / d = i * m >> (31 + s) */
struct Divider {
    uint32_t mul, shift;
    explicit Divider(uint32_t d) : mul(0), shift(0)
    {
        while((1ull << shift) < d) ++shift;
        if(shift) mul = (uint32_t)((1ull << (31 + shift)) / d + 1);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t i) const { return shift ? __umulhi(i, mul) >> (shift - 1) : i; }
};

/* Rows of whole VW-element packs: a CTA makes U * kThreads packs of out in order, U of a thread in flight.  Packs behind the
 * end, and of rows that are not there, are read in the place of row 0 and not stored.  kDense: the rows of out have
 * no gaps. */
template <typename T, typename O, typename I, int VW, int U, bool kDense>
__global__ void __launch_bounds__(kThreads) lookup_pack_kernel(const T *__restrict__ table, uint32_t rows, uint32_t packs,
                                                               uint32_t stride_bytes, const I *__restrict__ index,
                                                               uint64_t count, uint64_t total, float scale,
                                                               O *__restrict__ out, uint64_t out_stride,
                                                               const Divider by_packs, uint32_t *__restrict__ bad)
{
    const uint64_t w0 = (uint64_t)blockIdx.x * (kThreads * U);
    const uint64_t n0 = total <= 0xffffffffull ? (uint64_t)((uint32_t)w0 / packs) : w0 / packs; /* the CTA's first row */
    const uint32_t c0 = (uint32_t)(w0 - n0 * packs) + threadIdx.x;
    const uint32_t left = total - w0 < kThreads * U ? (uint32_t)(total - w0) : kThreads * U;
    const uint32_t last = (uint32_t)(count - 1 - n0 < 0x7fffffffull ? count - 1 - n0 : 0x7fffffffull);
    const I *ix = index + n0;
    uint32_t n[U], s[U];
    Pack<T, VW> x[U];
#pragma unroll
    for(int u = 0; u < U; ++u) {
        n[u] = by_packs(c0 + u * kThreads);
        s[u] = row_number(__ldg(ix + (n[u] < last ? n[u] : last)));
    }
    if(rows == 0) {
        if(bad != nullptr) atomicExch(bad, 1u);
        return;
    }
    const unsigned char *bytes = reinterpret_cast<const unsigned char *>(table);
#pragma unroll
    for(int u = 0; u < U; ++u) {
        const unsigned char *row = bytes + (uint64_t)(s[u] < rows ? s[u] : 0u) * stride_bytes;
        x[u] = reinterpret_cast<const Pack<T, VW> *>(row)[c0 + u * kThreads - n[u] * packs];
    }
    bool all = true;
#pragma unroll
    for(int u = 0; u < U; ++u) {
        Pack<O, VW> y;
#pragma unroll
        for(int k = 0; k < VW; ++k) y.v[k] = from_f32<O>(scale * to_f32(x[u].v[k]));
        const bool in = threadIdx.x + u * kThreads < left;
        all &= s[u] < rows || !in;
        if(s[u] < rows && in) {
            if(kDense) (reinterpret_cast<Pack<O, VW> *>(out) + w0)[threadIdx.x + u * kThreads] = y;
            else reinterpret_cast<Pack<O, VW> *>(out + (n0 + n[u]) * out_stride)[c0 + u * kThreads - n[u] * packs] = y;
        }
    }
    if(!all && bad != nullptr) atomicExch(bad, 1u);
}

/* Rows of DIM <= 4 elements into an out without gaps: a thread makes R of them, whole 16-byte stores.  A lane an element
 * spends 30 instructions on each (place, index, row, element), this about 3.  kTable: the scaled table lies in shared
 * memory, where the rows of 32 lanes cost a few bank conflicts instead of a cache line each. */
constexpr size_t kShortTable = 100 * 1024;

template <typename T, typename O, typename I, int DIM, bool kTable>
__global__ void __launch_bounds__(kTable ? 1024 : kThreads) lookup_short_kernel(const T *__restrict__ table, uint32_t rows,
                                                                                uint32_t stride_bytes,
                                                                                const I *__restrict__ index, uint64_t count,
                                                                                float scale, O *__restrict__ out,
                                                                                uint32_t *__restrict__ bad)
{
    constexpr int R = 16 / sizeof(O);
    constexpr uint32_t kBlock = kTable ? 1024 : kThreads;
    extern __shared__ __align__(16) unsigned char smem[];
    O *s_table = reinterpret_cast<O *>(smem);
    const unsigned char *bytes = reinterpret_cast<const unsigned char *>(table);
    if(kTable) {
        for(uint32_t j = threadIdx.x; j < rows * DIM; j += kBlock)
            s_table[j] = from_f32<O>(scale * to_f32(reinterpret_cast<const T *>(bytes + (uint64_t)(j / DIM) * stride_bytes)[j % DIM]));
        __syncthreads();
    }
    const bool wide = (uintptr_t)index % 16 == 0;
    for(uint64_t t = (uint64_t)blockIdx.x * kBlock + threadIdx.x; t * R < count; t += (uint64_t)gridDim.x * kBlock) {
        const I *ix = index + t * R;
        uint32_t s[R];
        if(wide && t * R + R <= count) {
            constexpr int V = 16 / sizeof(I);
#pragma unroll
            for(int r = 0; r < R; r += V) {
                const Pack<I, V> v = *reinterpret_cast<const Pack<I, V> *>(ix + r);
#pragma unroll
                for(int k = 0; k < V; ++k) s[r + k] = row_number(v.v[k]);
            }
        } else {
#pragma unroll
            for(int r = 0; r < R; ++r) s[r] = t * R + r < count ? row_number(__ldg(ix + r)) : UINT32_MAX;
        }
        Pack<O, R> y[DIM]; /* R * DIM elements in order */
        bool all = true;
#pragma unroll
        for(int r = 0; r < R; ++r) {
            all &= s[r] < rows;
            if(s[r] < rows)
#pragma unroll
                for(int k = 0; k < DIM; ++k) {
                    const int e = r * DIM + k;
                    y[e / R].v[e % R] = kTable ? s_table[s[r] * DIM + k]
                                               : from_f32<O>(scale * to_f32(reinterpret_cast<const T *>(bytes + (uint64_t)s[r] * stride_bytes)[k]));
                }
        }
        O *to = out + t * R * DIM;
        if(all) {
#pragma unroll
            for(int k = 0; k < DIM; ++k) reinterpret_cast<Pack<O, R> *>(to)[k] = y[k];
            continue;
        }
#pragma unroll
        for(int r = 0; r < R; ++r) {
            if(s[r] < rows) {
#pragma unroll
                for(int k = 0; k < DIM; ++k) to[r * DIM + k] = y[(r * DIM + k) / R].v[(r * DIM + k) % R];
            } else if(bad != nullptr && t * R + r < count) {
                atomicExch(bad, 1u);
            }
        }
    }
}

/* Any row: 2^CLOG lanes take a row's elements side by side (NC of them each, 2^CLOG apart), a warp ROWS consecutive
 * rows, whose indices it loads at once and hands round, with U steps of rows in flight.  Longer rows than NC * 32 are cut
 * into tiles (y).  Elements and rows that are not there are read in the place of ones that are (a load under a condition
 * becomes a branch of some ten instructions) and not stored.  1M rows of 45 from 16-bit rows: 43 us, bound by the
 * instructions an element (0.66 of the issue slots); writing its 180 MB alone takes 28. */
template <typename T, typename O, typename I, int NC, int CLOG, int ROWS>
__global__ void __launch_bounds__(kThreads) lookup_warp_kernel(const T *__restrict__ table, uint32_t rows, uint32_t dim,
                                                               uint32_t stride_bytes, const I *__restrict__ index,
                                                               uint64_t count, float scale, O *__restrict__ out,
                                                               uint64_t out_stride, uint32_t *__restrict__ bad)
{
    constexpr int kSteps = ROWS >> (5 - CLOG), U = 8 / NC < kSteps ? 8 / NC : kSteps, per = 32 >> CLOG; /* rows a step */
    static_assert(kSteps % U == 0, "whole rounds");
    const int lane = threadIdx.x & 31;
    const uint64_t n0 = ((uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * ROWS;
    if(n0 >= count) return;
    const int left = count - n0 < ROWS ? (int)(count - n0) : ROWS;
    const uint32_t mine = lane < left ? row_number(__ldg(index + n0 + lane)) : UINT32_MAX;
    if(bad != nullptr && lane < left && mine >= rows) atomicExch(bad, 1u);
    if(rows == 0) return;
    const unsigned char *bytes = reinterpret_cast<const unsigned char *>(table);
    const uint64_t hop = out_stride * per;
    uint32_t tile = NC == 4 ? blockIdx.y : 0;
    do {
        const uint32_t c0 = tile * (NC << CLOG) + (lane & ((1 << CLOG) - 1));
        const unsigned char *from[NC];
        bool in[NC];
#pragma unroll
        for(int k = 0; k < NC; ++k) {
            const uint32_t c = c0 + (k << CLOG);
            in[k] = c < dim;
            from[k] = bytes + (uint64_t)(in[k] ? c : 0u) * sizeof(T);
        }
        O *to = out + (n0 + (lane >> CLOG)) * out_stride + c0;
#pragma unroll 1
        for(int j = 0; j < kSteps; j += U) {
            uint32_t s[U];
            T x[U][NC];
#pragma unroll
            for(int u = 0; u < U; ++u) {
                s[u] = __shfl_sync(0xffffffffu, mine, (j + u) * per + (lane >> CLOG));
                const uint32_t row = s[u] < rows ? s[u] : 0u;
#pragma unroll
                for(int k = 0; k < NC; ++k) x[u][k] = *reinterpret_cast<const T *>(from[k] + (uint64_t)row * stride_bytes);
            }
#pragma unroll
            for(int u = 0; u < U; ++u) {
#pragma unroll
                for(int k = 0; k < NC; ++k)
                    if(s[u] < rows && in[k]) to[k << CLOG] = from_f32<O>(scale * to_f32(x[u][k]));
                to += hop;
            }
        }
        tile += gridDim.y;
    } while(NC == 4 && tile * (uint64_t)(NC << CLOG) < dim);
}

template <typename T, typename O, typename I, int DIM>
cudaError_t launch_short(const T *table, uint32_t rows, uint32_t stride_bytes, const I *index, uint64_t count, float scale, O *out,
                         uint32_t *bad, cudaStream_t stream)
{
    constexpr uint64_t R = 16 / sizeof(O);
    const size_t bytes = (size_t)rows * DIM * sizeof(O);
    /* a small table that is read many times over: each of two CTAs an SM copies it to shared memory once */
    if(bytes <= kShortTable && count >= (uint64_t)rows * 64 && count >= (1u << 18)) {
        const cudaError_t e = gsx_allow_smem<lookup_short_kernel<T, O, I, DIM, true>>(kShortTable);
        if(e != cudaSuccess) return e;
        lookup_short_kernel<T, O, I, DIM, true><<<148 * 2, 1024, bytes, stream>>>(table, rows, stride_bytes, index, count, scale, out, bad);
        return cudaSuccess;
    }
    const uint64_t threads = (count + R - 1) / R;
    lookup_short_kernel<T, O, I, DIM, false><<<(unsigned)((threads + kThreads - 1) / kThreads), kThreads, 0, stream>>>(
        table, rows, stride_bytes, index, count, scale, out, bad);
    return cudaSuccess;
}

/* whether the call can move packs of VW elements; if so, it has */
template <typename T, typename O, typename I, int VW>
bool launch_packs(const T *table, uint64_t rows, uint64_t dim, uint64_t table_stride, const I *index, uint64_t count, float scale,
                  O *out, uint64_t out_stride, uint32_t *bad, cudaStream_t stream)
{
    constexpr uint64_t TA = alignof(Pack<T, VW>), OA = alignof(Pack<O, VW>);
    if(dim % VW != 0 || (uintptr_t)table % TA != 0 || table_stride * sizeof(T) % TA != 0 || (uintptr_t)out % OA != 0 ||
       out_stride * sizeof(O) % OA != 0)
        return false;
    const uint64_t total = count * (dim / VW);
    const Divider by_packs((uint32_t)(dim / VW));
    auto launch = [&](auto kernel, uint64_t per) {
        kernel<<<(unsigned)((total + per - 1) / per), kThreads, 0, stream>>>(table, (uint32_t)rows, (uint32_t)(dim / VW),
                                                                             (uint32_t)(table_stride * sizeof(T)), index, count,
                                                                             total, scale, out, out_stride, by_packs, bad);
    };
    const bool dense = out_stride == dim;
    if(total >= 148ull * 2048 * 2) {
        if(dense) launch(lookup_pack_kernel<T, O, I, VW, 4, true>, kThreads * 4);
        else launch(lookup_pack_kernel<T, O, I, VW, 4, false>, kThreads * 4);
    } else {
        if(dense) launch(lookup_pack_kernel<T, O, I, VW, 1, true>, kThreads);
        else launch(lookup_pack_kernel<T, O, I, VW, 1, false>, kThreads);
    }
    return true;
}

template <typename T, typename O, typename I>
cudaError_t launch_lookup(const void *table_, uint64_t rows, uint64_t dim, uint64_t table_stride, const void *index_,
                          uint64_t count, float scale, void *out_, uint64_t out_stride, uint32_t *bad, cudaStream_t stream)
{
    const T *table = static_cast<const T *>(table_);
    const I *index = static_cast<const I *>(index_);
    O *out = static_cast<O *>(out_);
    const uint32_t stride_bytes = (uint32_t)(table_stride * sizeof(T));
    if(dim <= 4 && out_stride == dim && (uintptr_t)out % 16 == 0) {
        switch(dim) {
        case 1: return launch_short<T, O, I, 1>(table, (uint32_t)rows, stride_bytes, index, count, scale, out, bad, stream);
        case 2: return launch_short<T, O, I, 2>(table, (uint32_t)rows, stride_bytes, index, count, scale, out, bad, stream);
        case 3: return launch_short<T, O, I, 3>(table, (uint32_t)rows, stride_bytes, index, count, scale, out, bad, stream);
        default: return launch_short<T, O, I, 4>(table, (uint32_t)rows, stride_bytes, index, count, scale, out, bad, stream);
        }
    }
    /* the widest pack of elements that every row is a whole number of, on both sides */
    constexpr int VW = 16 / sizeof(T);
    if(launch_packs<T, O, I, VW>(table, rows, dim, table_stride, index, count, scale, out, out_stride, bad, stream) ||
       launch_packs<T, O, I, VW / 2>(table, rows, dim, table_stride, index, count, scale, out, out_stride, bad, stream))
        return cudaSuccess;
    if(VW == 8 && launch_packs<T, O, I, VW == 8 ? 2 : VW>(table, rows, dim, table_stride, index, count, scale, out, out_stride, bad, stream))
        return cudaSuccess;
    auto launch = [&](auto kernel, uint64_t warp_rows, uint64_t tiles) {
        const uint64_t ctas = (count + kWarps * warp_rows - 1) / (kWarps * warp_rows);
        kernel<<<dim3((unsigned)ctas, (unsigned)(tiles < 65535 ? tiles : 65535)), kThreads, 0, stream>>>(
            table, (uint32_t)rows, (uint32_t)dim, stride_bytes, index, count, scale, out, out_stride, bad);
    };
    const uint64_t tiles = (dim + 127) / 128;
    if(dim <= 8) launch(lookup_warp_kernel<T, O, I, 1, 3, 32>, 32, 1);
    else if(dim <= 16) launch(lookup_warp_kernel<T, O, I, 1, 4, 32>, 32, 1);
    else if(dim <= 32) launch(lookup_warp_kernel<T, O, I, 1, 5, 32>, 32, 1);
    else if(dim <= 64) launch(lookup_warp_kernel<T, O, I, 2, 5, 32>, 32, 1);
    else if((count + 31) / 32 * tiles >= 148 * 32) launch(lookup_warp_kernel<T, O, I, 4, 5, 32>, 32, tiles);
    else launch(lookup_warp_kernel<T, O, I, 4, 5, 2>, 2, tiles); /* few long rows: 4 of 2709 took 69 us at 32 a warp */
    return cudaSuccess;
}

/* ------------------------------------------------------------------------------------------ */
/* rows of the gradient table */

struct Table {
    void *data;
    uint64_t stride; /* elements */
    uint64_t rows;
    float scale;
    int bytes; /* of an element */
    bool accumulate;
};

template <typename TT, int VW>
__device__ __forceinline__ void store_sums(const Table &t, uint64_t row, uint32_t c, const float (&sum)[VW])
{
    Pack<TT, VW> *to = reinterpret_cast<Pack<TT, VW> *>(static_cast<TT *>(t.data) + row * t.stride + c);
    Pack<TT, VW> y;
    if(t.accumulate) {
        y = *to;
#pragma unroll
        for(int v = 0; v < VW; ++v) y.v[v] = from_f32<TT>(fmaf(t.scale, sum[v], to_f32(y.v[v])));
    } else {
#pragma unroll
        for(int v = 0; v < VW; ++v) y.v[v] = from_f32<TT>(t.scale * sum[v]);
    }
    *to = y;
}

/* zeros in part `part` of `parts` of a table (16-byte stores where rows and addresses allow it) */
__device__ __forceinline__ void zero_rows(const Table &t, uint32_t dim, uint32_t part, uint32_t parts)
{
    const uint64_t es = t.bytes;
    uint64_t rows = t.rows, row = dim * es;
    const uint64_t step = t.stride * es;
    if(row == step) {
        row *= rows;
        rows = 1;
    }
    unsigned char *base = static_cast<unsigned char *>(t.data);
    const uint64_t tid = (uint64_t)part * blockDim.x + threadIdx.x, threads = (uint64_t)parts * blockDim.x;
    if(rows == 1) {
        const uint64_t head = (16 - ((uintptr_t)base & 15)) & 15, first = head < row ? head : row;
        const uint64_t vecs = (row - first) / 16;
        uint4 *v = reinterpret_cast<uint4 *>(base + first);
        for(uint64_t i = tid; i < vecs; i += threads) v[i] = make_uint4(0, 0, 0, 0);
        uint16_t *h = reinterpret_cast<uint16_t *>(base);
        if(tid < first / 2) h[tid] = 0;
        const uint64_t done = first + vecs * 16;
        if(tid < (row - done) / 2) h[done / 2 + tid] = 0;
        return;
    }
    const uint64_t warp = tid / 32, warps = threads / 32;
    const uint32_t lane = threadIdx.x & 31;
    const bool wide = (((uintptr_t)base | row | step) & 15) == 0;
    for(uint64_t r = warp; r < rows; r += warps) {
        unsigned char *to = base + r * step;
        if(wide)
            for(uint64_t i = lane; i < row / 16; i += 32) reinterpret_cast<uint4 *>(to)[i] = make_uint4(0, 0, 0, 0);
        else
            for(uint64_t i = lane; i < row / 2; i += 32) reinterpret_cast<uint16_t *>(to)[i] = 0;
    }
}

/* ------------------------------------------------------------------------------------------ */
/* the sort of positions by row */

/* Which positions take part: those whose index is a row and not the padding row (UINT32_MAX: none).  Any other index
 * than the padding row sets *bad. */
struct Use {
    uint32_t rows, padding;
    uint32_t *bad;
};

template <typename I>
__device__ __forceinline__ bool takes_part(I s, const Use &use, bool &outside)
{
    const bool in = sizeof(I) == 4 ? (uint32_t)s < use.rows : (uint64_t)s < (uint64_t)use.rows;
    outside |= !in;
    return in && (uint32_t)s != use.padding;
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

/* A tile of (row, position) pairs that a CTA ranks by one digit of at most 8 bits. */
constexpr int kHistRow = kMaxBins + 1; /* one more: elements that take no part */
template <int THREADS, int ITEMS, typename P = uint2>
struct SortShared {
    uint32_t hist[THREADS / 32][kHistRow];
    uint32_t before[kHistRow]; /* of a digit: the tile's pairs with smaller ones */
    uint32_t warp[32];
    alignas(16) P pair[THREADS * ITEMS]; /* the last: a launch may leave room for the tile that it uses */
};

/* a pair in eight bytes, or in four: a position in a tile of at most 2^kPlaceBits */
constexpr int kPlaceBits = 12;
__device__ __forceinline__ void set_pair(uint2 &to, uint32_t key, uint32_t pos) { to = make_uint2(key, pos); }
__device__ __forceinline__ void set_pair(uint32_t &to, uint32_t key, uint32_t pos) { to = key << kPlaceBits | pos; }

/* Ranks the tile's pairs (warp w holds elements 32 * items * w + 32 * it + lane) by digit, stable in element
 * order, and leaves them in s.pair in that order, without those with valid[it] false (their key is 0).
 * Returns, for threads below the number of digits, how many pairs have that digit.  Lanes with equal digits find one
 * another by one ballot per digit bit: __match_any_sync takes a step per distinct value on this GPU (a tile of 8192
 * ranked in 12 us with it, in 4 us with ballots).  No step is under a condition of the element: elements that take
 * no part have a digit of their own (with branches a tile took 2.5 times as many instructions). */
template <int THREADS, int ITEMS, typename P>
__device__ __forceinline__ uint32_t sort_tile(SortShared<THREADS, ITEMS, P> &s, const uint32_t (&key)[ITEMS],
                                              const uint32_t (&pos)[ITEMS], const bool (&valid)[ITEMS], int items, int shift,
                                              int bits)
{
    static_assert(THREADS >= kMaxBins, "a thread to each digit");
    constexpr int WARPS = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t bins = 1u << bits, mask = bins - 1u;
    for(uint32_t j = threadIdx.x; j < WARPS * kHistRow; j += THREADS) (&s.hist[0][0])[j] = 0u;
    __syncthreads();
    uint32_t *wh = s.hist[warp];
    uint32_t rank[ITEMS], digit[ITEMS];
    /* item by item: all ballots ahead of the counts took 3M x 3 into 4096 rows from 40 to 42 us */
#pragma unroll
    for(int it = 0; it < ITEMS; ++it) {
        if(it < items) {
            const uint32_t d = key[it] >> shift & mask;
            const unsigned all = __ballot_sync(0xffffffffu, valid[it]);
            unsigned peers = valid[it] ? all : ~all;
#pragma unroll
            for(int b = 0; b < kMaxBits; ++b) {
                if(b < bits) {
                    const int one = -(int)(d >> b & 1u); /* all ones where the bit is set */
                    peers &= ~(__ballot_sync(0xffffffffu, one != 0) ^ (unsigned)one);
                }
            }
            digit[it] = valid[it] ? d : bins;
            const uint32_t before = wh[digit[it]];
            rank[it] = before + (uint32_t)__popc(peers & ((1u << lane) - 1u));
            __syncwarp();
            wh[digit[it]] = before + (uint32_t)__popc(peers);
            __syncwarp();
        }
    }
    __syncthreads();
    /* counts -> places before each warp's, for every digit and the one of the elements that take no part; that is the last
     * and may find no thread of its own */
    auto warps_before = [&](uint32_t d) {
        uint32_t c[WARPS], sum = 0;
#pragma unroll
        for(int w = 0; w < WARPS; ++w) c[w] = s.hist[w][d];
#pragma unroll
        for(int w = 0; w < WARPS; ++w) {
            s.hist[w][d] = sum;
            sum += c[w];
        }
        return sum;
    };
    const uint32_t count = threadIdx.x < bins ? warps_before(threadIdx.x) : 0u;
    if(threadIdx.x == THREADS - 1) warps_before(bins);
    uint32_t total;
    const uint32_t upto = block_inclusive_scan(count, s.warp, &total);
    if(threadIdx.x < bins) s.before[threadIdx.x] = upto - count;
    if(threadIdx.x == THREADS - 1) s.before[bins] = total;
    __syncthreads();
#pragma unroll
    for(int it = 0; it < ITEMS; ++it)
        if(it < items && (sizeof(P) == 8 || valid[it])) set_pair(s.pair[s.before[digit[it]] + wh[digit[it]] + rank[it]], key[it], pos[it]);
    __syncthreads();
    return count;
}

/* all of a small sort in one CTA */
template <typename I, int ITEMS>
__global__ void __launch_bounds__(kSmallThreads) small_sort_kernel(const I *__restrict__ index, uint32_t count,
                                                                   const Use use, uint2 *__restrict__ pairs,
                                                                   uint32_t *__restrict__ n_sorted)
{
    extern __shared__ __align__(16) unsigned char smem[];
    auto &s = *reinterpret_cast<SortShared<kSmallThreads, ITEMS> *>(smem);
    gsx_pdl_trigger(); /* the zeros are written meanwhile */
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int items = (int)((count + kSmallThreads - 1) / kSmallThreads);
    const uint32_t wbase = (uint32_t)warp * 32u * (uint32_t)items + (uint32_t)lane;
    uint32_t k[ITEMS], p[ITEMS], used = 0;
    bool valid[ITEMS];
    I raw[ITEMS];
#pragma unroll
    for(int it = 0; it < ITEMS; ++it) {
        p[it] = wbase + (uint32_t)it * 32u;
        valid[it] = it < items && p[it] < count;
        raw[it] = count > 0 ? __ldg(index + (valid[it] ? p[it] : 0u)) : (I)0;
    }
    bool outside = false;
#pragma unroll
    for(int it = 0; it < ITEMS; ++it) {
        valid[it] &= takes_part(valid[it] ? raw[it] : (I)0, use, outside);
        k[it] = valid[it] ? (uint32_t)raw[it] : 0u;
        used += valid[it];
    }
    if(outside && use.bad != nullptr) atomicExch(use.bad, 1u);
    uint32_t n;
    block_inclusive_scan(used, s.warp, &n);
    if(threadIdx.x == 0) *n_sorted = n;
    const int bits = use.rows > 1 ? 32 - __clz((int)(use.rows - 1)) : 1;
    const int passes = (bits + kMaxBits - 1) / kMaxBits;
    for(int pass = 0, shift = 0; pass < passes; ++pass) {
        const int width = (bits - shift + passes - 1 - pass) / (passes - pass);
        sort_tile(s, k, p, valid, items, shift, width);
        shift += width;
#pragma unroll
        for(int it = 0; it < ITEMS; ++it) {
            const uint32_t i = wbase + (uint32_t)it * 32u;
            valid[it] = it < items && i < n;
            if(it < items) {
                const uint2 kp = s.pair[i];
                k[it] = kp.x;
                p[it] = kp.y;
            }
        }
        __syncthreads();
    }
#pragma unroll
    for(int it = 0; it < ITEMS; ++it)
        if(valid[it]) pairs[wbase + (uint32_t)it * 32u] = make_uint2(k[it], p[it]);
}

/* the table's zeros, beside small_sort_kernel; the last CTA ends after that.  268 MB: 39 us, 6.9 TB/s */
__global__ void __launch_bounds__(kThreads) zero_kernel(const Table table, uint32_t dim)
{
    gsx_pdl_trigger();
    zero_rows(table, dim, blockIdx.x, gridDim.x);
    if(blockIdx.x == gridDim.x - 1) gsx_pdl_wait();
}

/* The kernels from here on are launched before the one ahead of them has ended (gsx_launch_pdl) and read what it wrote
 * after gsx_pdl_wait: with __ldcg, since a read-only load may return what the SM's cache held before. */

/* The table's zeros, written beside the sort: each of its kernels has CTAs behind those of its chunks that write the part of
 * that kernel, while the others wait for counts and ranks (30000 positions into 67 MB: 311 us with the zeros in the four CTAs
 * of the first count, 35 so). */
struct Zeros {
    Table table;
    uint32_t dim, ctas, first, parts; /* parts of the table: CTAs of this kernel, the first one's part, all parts */
};

/* the part of a pass's input that belongs to this CTA */
__device__ __forceinline__ void chunk_range(uint32_t n, uint32_t chunks, uint32_t &begin, uint32_t &end)
{
    const uint32_t len = (n + chunks - 1) / chunks;
    begin = len * blockIdx.x < n ? len * blockIdx.x : n;
    end = n - begin < len ? n : begin + len;
}

/* Up to ITEMS elements of a pass's input, at first + it * step below end: of the indices themselves in the
 * first pass (kFirst), of sorted pairs else.  All loads are issued before the first is looked at. */
template <typename I, bool kFirst, int ITEMS>
__device__ __forceinline__ void load_elements(const I *__restrict__ index, const uint2 *__restrict__ pairs, uint32_t first,
                                              uint32_t step, int items, uint32_t end, const Use &use,
                                              uint32_t (&key)[ITEMS], uint32_t (&pos)[ITEMS],
                                              bool (&valid)[ITEMS])
{
    const uint32_t last = end - 1; /* elements behind the end are read in its place */
    if(kFirst) {
        I raw[ITEMS];
#pragma unroll
        for(int it = 0; it < ITEMS; ++it) {
            pos[it] = first + it * step;
            raw[it] = __ldg(index + (pos[it] < last ? pos[it] : last));
        }
        bool outside = false;
#pragma unroll
        for(int it = 0; it < ITEMS; ++it) {
            const bool in = it < items && pos[it] < end;
            valid[it] = takes_part(raw[it], use, outside) && in;
            key[it] = valid[it] ? (uint32_t)raw[it] : 0u;
        }
        if(outside && use.bad != nullptr) atomicExch(use.bad, 1u);
        return;
    }
#pragma unroll
    for(int it = 0; it < ITEMS; ++it) {
        const uint32_t i = first + it * step;
        valid[it] = it < items && i < end;
        const uint2 kp = __ldcg(pairs + (i < last ? i : last));
        key[it] = valid[it] ? kp.x : 0u;
        pos[it] = kp.y;
    }
}

/* counts[c][d] = elements of chunk c with digit d */
template <typename I, bool kFirst>
__global__ void __launch_bounds__(kSortThreads) digit_count_kernel(const I *__restrict__ index,
                                                                   const uint2 *__restrict__ pairs, uint32_t count,
                                                                   const uint32_t *__restrict__ n_pairs, const Use use,
                                                                   int shift, int bits, uint32_t chunks,
                                                                   uint32_t *__restrict__ counts, const Zeros zeros)
{
    __shared__ uint32_t s_hist[kHistRow];
    const uint32_t bins = 1u << bits;
    for(uint32_t j = threadIdx.x; j <= bins; j += kSortThreads) s_hist[j] = 0u;
    __syncthreads();
    gsx_pdl_trigger();
    if(blockIdx.x >= chunks) {
        zero_rows(zeros.table, zeros.dim, zeros.first + blockIdx.x - chunks, zeros.parts);
        return;
    }
    if(!kFirst) gsx_pdl_wait();
    uint32_t begin, end;
    chunk_range(kFirst ? count : __ldcg(n_pairs), chunks, begin, end);
    for(uint32_t i0 = begin; i0 < end; i0 += kTile) {
        uint32_t key[kSortItems], pos[kSortItems];
        bool in[kSortItems];
        load_elements<I, kFirst, kSortItems>(index, pairs, i0 + threadIdx.x, kSortThreads, kSortItems, end, use, key, pos, in);
#pragma unroll
        for(int it = 0; it < kSortItems; ++it)
            atomicAdd(&s_hist[in[it] ? key[it] >> shift & (bins - 1u) : bins], 1u);
    }
    __syncthreads();
    const uint32_t padded = bins < 4 ? 4 : bins; /* read four at a time */
    for(uint32_t j = threadIdx.x; j < padded; j += kSortThreads) counts[blockIdx.x * padded + j] = j < bins ? s_hist[j] : 0u;
}

/* every pair to its place, in input order within a digit.  Each CTA adds up the counts of all chunks itself. */
template <typename I, bool kFirst>
__global__ void __launch_bounds__(kSortThreads) digit_scatter_kernel(const I *__restrict__ index,
                                                                        const uint2 *__restrict__ pairs, uint32_t count,
                                                                        uint32_t *n_pairs, const Use use, int shift,
                                                                        int bits, uint32_t chunks,
                                                                        const uint32_t *__restrict__ counts,
                                                                        uint2 *__restrict__ out, const Zeros zeros)
{
    extern __shared__ __align__(16) unsigned char smem[];
    auto &s = *reinterpret_cast<SortShared<kSortThreads, kSortItems> *>(smem);
    __shared__ uint32_t s_place[kMaxBins]; /* of a digit: the next output place */
    __shared__ uint32_t s_to[kMaxBins];    /* .. less the place of its first pair in the tile */
    __shared__ uint32_t s_n;
    const uint32_t bins = 1u << bits, mask = bins - 1u;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    gsx_pdl_trigger();
    if(blockIdx.x >= chunks) {
        zero_rows(zeros.table, zeros.dim, zeros.first + blockIdx.x - chunks, zeros.parts);
        return;
    }
    gsx_pdl_wait();
    uint32_t begin, end;
    chunk_range(kFirst ? count : __ldcg(n_pairs), chunks, begin, end);
    uint32_t k[kSortItems], p[kSortItems];
    bool valid[kSortItems];
    auto load = [&](uint32_t i0) {
        const int items = end - i0 >= (uint32_t)kTile ? kSortItems : (int)((end - i0 + kSortThreads - 1) / kSortThreads);
        load_elements<I, kFirst, kSortItems>(index, pairs, i0 + (uint32_t)(warp * 32 * items + lane), 32, items, end, use, k, p, valid);
        return items;
    };
    int items = begin < end ? load(begin) : 0; /* on their way while the counts are added up */
    {
        /* four digits a thread, up to 32 chunks side by side: a load for each five of 148 chunks where one digit a thread
         * took 37 (the sort of 1M positions by 14 bits: 38 us, then 33) */
        const uint32_t quads = (bins + 3) / 4, q = threadIdx.x % quads, lanes = kSortThreads / quads;
        const uint32_t parts = lanes < 32 ? lanes : 32, part = threadIdx.x / quads;
        uint4 all4 = make_uint4(0, 0, 0, 0), before4 = all4;
        if(part < parts) {
#pragma unroll 5
            for(uint32_t c = part; c < chunks; c += parts) {
                const uint4 v = __ldcg(reinterpret_cast<const uint4 *>(counts) + (c * quads + q));
                const uint32_t m = c < blockIdx.x ? ~0u : 0u;
                all4 = make_uint4(all4.x + v.x, all4.y + v.y, all4.z + v.z, all4.w + v.w);
                before4 = make_uint4(before4.x + (v.x & m), before4.y + (v.y & m), before4.z + (v.z & m), before4.w + (v.w & m));
            }
        }
        uint4 *s_all = reinterpret_cast<uint4 *>(s.pair), *s_before = s_all + kSortThreads; /* of kSortThreads each */
        s_all[threadIdx.x] = all4;
        s_before[threadIdx.x] = before4;
        __syncthreads();
        uint32_t all = 0, before = 0;
        if(threadIdx.x < bins)
#pragma unroll 8
            for(uint32_t p = 0; p < parts; ++p) {
                all += reinterpret_cast<const uint32_t *>(s_all + p * quads)[threadIdx.x];
                before += reinterpret_cast<const uint32_t *>(s_before + p * quads)[threadIdx.x];
            }
        uint32_t n;
        const uint32_t smaller = block_inclusive_scan(all, s.warp, &n) - all;
        if(threadIdx.x < bins) s_place[threadIdx.x] = smaller + before;
        if(kFirst && blockIdx.x == 0 && threadIdx.x == 0) *n_pairs = n;
        __syncthreads();
    }
    for(uint32_t i0 = begin; i0 < end; i0 += kTile) {
        const uint32_t c = sort_tile(s, k, p, valid, items, shift, bits);
        if(threadIdx.x < bins) {
            s_to[threadIdx.x] = s_place[threadIdx.x] - s.before[threadIdx.x];
            s_place[threadIdx.x] += c;
            if(threadIdx.x == bins - 1) s_n = s.before[threadIdx.x] + c;
        }
        if(end - i0 > (uint32_t)kTile) items = load(i0 + kTile); /* on their way while this tile is written */
        __syncthreads();
        const uint32_t n = s_n;
        for(uint32_t j = threadIdx.x; j < n; j += kSortThreads) {
            const uint2 kp = s.pair[j];
            out[s_to[kp.x >> shift & mask] + j] = kp;
        }
        __syncthreads();
    }
}

/* ------------------------------------------------------------------------------------------ */
/* sums of sorted positions by row
 *
 * 1M x 45 f32 into 16384 rows: 57 us for 243 MB (a row of 180 bytes touches 64-byte pieces that it shares with its
 * neighbours) in random order, 0.52 of the DRAM's peak, bound by the latency of the gathers; 35 more for the sort.
 *
 * A CTA owns R consecutive sorted positions.  A group of 2^clog lanes, each with NR packs of VW columns, walks a run
 * of C of them in order, with the rows of the next positions in flight, and stores a row whenever the row number
 * changes.  A row that runs across groups is put together in shared memory (H: what a group has of a row that began
 * before it, T: of one that goes on after it), one that runs across CTAs in row_join_kernel. */

constexpr uint32_t kHead = 1, kWhole = 2, kTail = 4;
constexpr int kMaxRun = 128;
constexpr uint32_t kMaxPositions = 5120; /* of a CTA */

struct Runs {
    const uint2 *pairs;
    const uint32_t *n_sorted;
    float *head, *tail; /* [CTAs][dim]: sums of the CTA's first / last row where that crosses its ends */
    uint32_t dim;
    int clog, run; /* lanes of a group, positions of a group */
};

template <typename GT, typename TT, int VW, int NR>
__global__ void __launch_bounds__(kThreads, NR * VW <= 8 ? 4 : 2) run_sum_kernel(const GT *__restrict__ grad, uint32_t stride_bytes, const Runs a,
                                                              const Table table)
{
    /* packs that are not there are read in the place of the first, added and not stored (a load under a condition becomes
     * a branch); single elements of short rows are not, as the idle lanes' loads cost more */
    constexpr bool kClamp = NR * VW > 1;
    constexpr int kRegs = NR * VW * (int)sizeof(GT) / 4 > 0 ? NR * VW * (int)sizeof(GT) / 4 : 1;
    constexpr int U = kRegs <= 3 ? 8 : kRegs <= 8 ? 4 : 2; /* a divisor of 8, as runs are multiples of 8 */
    extern __shared__ __align__(16) unsigned char smem[];
    float *s_head = reinterpret_cast<float *>(smem);      /* groups * (NR * VW << clog) */
    float *s_tail = s_head + kThreads * NR * VW;
    /* each group's run and the pair behind it: an odd number of pairs, so that the groups of a warp read other banks */
    uint2 *s_pair = reinterpret_cast<uint2 *>(s_tail + kThreads * NR * VW);
    __shared__ uint32_t s_flags[kThreads / 4];
    __shared__ uint8_t s_ends[kMaxPositions / 8]; /* bit j: position j is the last of its row */
    gsx_pdl_trigger();
    gsx_pdl_wait();
    const uint32_t n = __ldcg(a.n_sorted);
    const int cl = 1 << a.clog, groups = kThreads >> a.clog, run = a.run;
    const uint32_t b0 = blockIdx.x * (uint32_t)(groups * run);
    if(b0 >= n) return;
    const uint32_t len = n - b0 < (uint32_t)(groups * run) ? n - b0 : (uint32_t)(groups * run);
    for(int j = threadIdx.x; j < groups * (run + 1); j += kThreads) {
        const uint32_t at = b0 + (uint32_t)(j - j / (run + 1));
        s_pair[j] = at < n ? __ldcg(a.pairs + at) : make_uint2(0xffffffffu, 0u); /* no row */
    }
    __syncthreads();
    for(int j = threadIdx.x; j < groups * run / 8; j += kThreads) {
        const uint2 *eight = s_pair + 8 * j + 8 * j / run;
        uint32_t key = eight[0].x, m = 0;
#pragma unroll
        for(int k = 0; k < 8; ++k) {
            const uint32_t next = eight[k + 1].x;
            m |= key != next ? 1u << k : 0u;
            key = next;
        }
        s_ends[j] = (uint8_t)m;
    }
    __syncthreads();
    const int group = (int)threadIdx.x >> a.clog, cg = (int)threadIdx.x & (cl - 1);
    const uint32_t col0 = blockIdx.y * (uint32_t)(NR * VW << a.clog);
    const int left = (int)len - group * run, r1 = left < run ? left : run; /* the group's positions */
    uint32_t flags = 0;
    if(r1 > 0) {
        const uint2 *mine = s_pair + group * (run + 1);
        const uint8_t *my_ends = s_ends + group * run / 8;
        float acc[NR][VW] = {};
        /* the current row began before the run */
        bool first = group > 0 ? mine[-2].x == mine[0].x : b0 > 0 && __ldcg(&a.pairs[b0 - 1].x) == mine[0].x;
        const unsigned char *base[NR];
        bool in[NR]; /* which of the lane's packs lie in the row */
#pragma unroll
        for(int r = 0; r < NR; ++r) {
            const uint32_t c = col0 + (uint32_t)((r * cl + cg) * VW);
            in[r] = c < a.dim;
            base[r] = reinterpret_cast<const unsigned char *>(grad + (!kClamp || in[r] ? c : 0u));
        }
        auto load = [&](Pack<GT, VW> (&x)[NR], int i) {
            const uint32_t p = mine[i].y;
#pragma unroll
            for(int r = 0; r < NR; ++r)
                if(kClamp || in[r]) x[r] = *reinterpret_cast<const Pack<GT, VW> *>(base[r] + (uint64_t)p * stride_bytes);
        };
        auto add = [&](const Pack<GT, VW> (&x)[NR]) {
#pragma unroll
            for(int r = 0; r < NR; ++r)
#pragma unroll
                for(int v = 0; v < VW; ++v) acc[r][v] += to_f32(x[r].v[v]);
        };
        /* the sums so far are all that the run has of `row`; `next` is the row behind them */
        auto finish = [&](uint32_t row, uint32_t next) {
            const bool open = next == row; /* the row goes on behind the run */
            if(first || open) {
                float *to = first ? s_head : s_tail;
                flags |= !first ? kTail : open ? kHead | kWhole : kHead;
#pragma unroll
                for(int r = 0; r < NR; ++r)
#pragma unroll
                    for(int v = 0; v < VW; ++v) to[(group * NR * cl + r * cl + cg) * VW + v] = acc[r][v];
            } else {
#pragma unroll
                for(int r = 0; r < NR; ++r)
                    if(in[r]) store_sums<TT, VW>(table, row, col0 + (uint32_t)((r * cl + cg) * VW), acc[r]);
            }
            first = false;
#pragma unroll
            for(int r = 0; r < NR; ++r)
#pragma unroll
                for(int v = 0; v < VW; ++v) acc[r][v] = 0.0f;
        };
        for(int i = 0; i < r1; i += U) {
            Pack<GT, VW> x[U][NR];
            uint32_t ends = (uint32_t)my_ends[i >> 3] >> (i & 7) & ((1u << U) - 1u);
            if(i + U >= r1) ends |= 1u << (r1 - 1 - i);
            if(ends == 0u) { /* all of one row, which goes on */
#pragma unroll
                for(int u = 0; u < U; ++u) load(x[u], i + u);
#pragma unroll
                for(int u = 0; u < U; ++u) add(x[u]);
                continue;
            }
#pragma unroll
            for(int u = 0; u < U; ++u)
                load(x[u], i + u < r1 ? i + u : i);
#pragma unroll
            for(int u = 0; u < U; ++u) {
                if(i + u < r1) add(x[u]);
                if(ends >> u & 1u) finish(mine[i + u].x, mine[i + u + 1].x);
            }
        }
    }
    if(cg == 0) s_flags[group] = flags;
    __syncthreads();
    /* rows across groups, one thread a column */
    const uint32_t cols = (uint32_t)(NR * VW << a.clog);
    const uint2 *last = s_pair + groups * (run + 1) - 2;
    const bool cta_tail = last[0].x == last[1].x && len == (uint32_t)(groups * run);
    for(uint32_t c = threadIdx.x; c < cols && col0 + c < a.dim; c += kThreads) {
        float cur = 0.0f;
        bool outside = true;
        for(int g = 0; g < groups; ++g) {
            const uint32_t f = s_flags[g];
            if(f & kHead) {
                cur += s_head[g * cols + c];
                if(!(f & kWhole)) {
                    if(outside) {
                        a.head[(uint64_t)blockIdx.x * a.dim + col0 + c] = cur;
                    } else {
                        const float one[1] = { cur };
                        store_sums<TT, 1>(table, s_pair[g * (run + 1)].x, col0 + c, one);
                    }
                    outside = false;
                }
            }
            if(f & kTail) {
                cur = s_tail[g * cols + c];
                outside = false;
            }
        }
        if(cta_tail) (outside ? a.head : a.tail)[(uint64_t)blockIdx.x * a.dim + col0 + c] = cur;
    }
}

/* Rows across CTAs of run_sum_kernel: the CTA (x) in which such a row begins adds up its parts.  Columns: 256 to a
 * CTA (y), a thread each, while the row has few parts; else 32 at a time, the parts dealt to the eight warps. */
constexpr uint32_t kFewParts = 16;
template <typename TT>
__global__ void __launch_bounds__(kThreads) row_join_kernel(const Runs a, const Table table)
{
    __shared__ float s_part[kWarps][32];
    gsx_pdl_wait();
    const uint32_t n = __ldcg(a.n_sorted);
    const uint32_t R = (uint32_t)(kThreads >> a.clog) * (uint32_t)a.run;
    const uint32_t b = blockIdx.x, b0 = b * R, b1 = b0 + R;
    if(b1 >= n) return;
    const uint32_t row = __ldcg(&a.pairs[b1 - 1].x);
    if(__ldcg(&a.pairs[b1].x) != row) return;
    if(b0 > 0 && __ldcg(&a.pairs[b0].x) == row && __ldcg(&a.pairs[b0 - 1].x) == row) return; /* began before */
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    /* the last CTA whose first position has the row: among the next 32, or by halving behind them */
    uint32_t lo = b + 1, hi = (n - 1) / R;
    const uint32_t look = lo + lane <= hi ? __ldcg(&a.pairs[(uint64_t)(lo + lane) * R].x) : UINT32_MAX;
    const unsigned same = __ballot_sync(0xffffffffu, look == row);
    if(same != 0xffffffffu) {
        hi = lo + (uint32_t)__ffs(~same) - 2; /* the first of them has the row */
        lo = hi;
    }
    while(lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if(__ldcg(&a.pairs[(uint64_t)mid * R].x) == row) lo = mid;
        else hi = mid - 1;
    }
    const uint32_t parts = lo - b;
    const uint32_t c0 = blockIdx.y * 256u;
    if(parts <= kFewParts) {
        const uint32_t c = c0 + threadIdx.x;
        if(c >= a.dim) return;
        float sum[1] = { __ldcg(a.tail + (uint64_t)b * a.dim + c) };
        for(uint32_t k = 1; k <= parts; ++k) sum[0] += __ldcg(a.head + (uint64_t)(b + k) * a.dim + c);
        store_sums<TT, 1>(table, row, c, sum);
        return;
    }
    for(uint32_t c1 = c0; c1 < a.dim && c1 < c0 + 256u; c1 += 32) {
        const uint32_t c = c1 + lane;
        float sum[1] = { 0.0f };
        if(c < a.dim) {
            if(warp == 0) sum[0] = __ldcg(a.tail + (uint64_t)b * a.dim + c);
#pragma unroll 8
            for(uint32_t k = 1 + warp; k <= parts; k += kWarps) sum[0] += __ldcg(a.head + (uint64_t)(b + k) * a.dim + c);
        }
        __syncthreads();
        s_part[warp][lane] = sum[0];
        __syncthreads();
        if(warp == 0 && c < a.dim) {
#pragma unroll
            for(int w = 1; w < kWarps; ++w) sum[0] += s_part[w][lane];
            store_sums<TT, 1>(table, row, c, sum);
        }
    }
}

/* ------------------------------------------------------------------------------------------ */
/* Small tables of short rows (a codebook of colours): the positions need not be sorted as a whole.  A CTA keeps a table of
 * sums in shared memory and walks a chunk of the positions in tiles.  It ranks a tile by the low 8 bits of the row while the
 * tile's gradients come into shared memory beside it, then the sums are added in that order: every row has one owner in
 * the CTA, so the order is fixed.  The CTAs' tables are then added up in the order of the chunks.
 *
 * 3M x 3 f32 into 4096 rows: 40 us, bound by the instructions and shared-memory accesses of ranking and walking (16 warps an
 * SM, as two tables fill its memory); the data alone takes 7.  Of the 64 us that it took before, a fifth went into loads
 * that all CTAs waited for at the same time: the next tile's indices now go to registers and its gradients to the L2
 * while this one is walked.  Gradients read by the walk itself, in sorted order, cost the same as staging them, but had
 * no room for that. */
constexpr int kOwnThreads = 256;
constexpr int kOwnItems = 16; /* positions a thread of a tile, at most */
constexpr uint32_t kOwnTile = kOwnThreads * kOwnItems;
static_assert(kOwnTile <= 1u << kPlaceBits, "a place of a tile fits a pair");
constexpr uint64_t kOwnLeast = 512; /* positions of a chunk */
constexpr size_t kOwnTable = 96 * 1024;
static_assert(kOwnTable / 4 <= 1u << (32 - kPlaceBits), "a row fits a pair");
constexpr size_t kOwnMemory = 113 * 1024; /* of a CTA: two an SM */
constexpr uint32_t kOwnLong = 64;
static_assert(kOwnThreads == kMaxBins, "thread t owns digit t");
using OwnShared = SortShared<kOwnThreads, kOwnItems, uint32_t>;

/* the most positions of a tile beside the table, with their pairs and gradients of gb bytes an element */
uint32_t own_fit(uint64_t rows, uint64_t dim, uint64_t gb)
{
    const uint64_t fixed = sizeof(OwnShared) - sizeof(uint32_t) * kOwnTile + 4 * rows * dim;
    const uint64_t fit = (kOwnMemory - fixed) / (sizeof(uint32_t) + dim * gb) / 32 * 32;
    return fit < kOwnTile ? (uint32_t)fit : kOwnTile;
}

/* tiles of equal length */
uint32_t own_tile(uint32_t len, uint32_t rows, uint32_t dim, size_t gb)
{
    const uint32_t most = own_fit(rows, dim, gb), tiles = (len + most - 1) / most;
    return ((len + tiles - 1) / tiles + 31) / 32 * 32;
}

/* whole multiples of 32 positions a chunk, so that tiles of dense rows start at 16 bytes */
__host__ __device__ constexpr uint32_t own_length(uint32_t count, uint32_t chunks)
{
    return ((count + chunks - 1) / chunks + 31u) / 32u * 32u;
}

/* Rows of DIM elements: thread t adds up the n pairs of digit t.  Lists of more than kOwnLong go to a warp, 32 at a time. */
template <typename GT, int DIM>
__device__ __forceinline__ void walk_lists(const OwnShared &s, const uint32_t *s_count, uint32_t n, uint32_t rows, const GT *s_grad,
                                           float *table)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto split = [&](uint32_t pair, float(&x)[DIM]) { /* its row in the table */
        const GT *g = s_grad + (pair & ((1u << kPlaceBits) - 1u)) * DIM;
#pragma unroll
        for(int c = 0; c < DIM; ++c) x[c] = to_f32(g[c]);
        return table + (pair >> kPlaceBits) * DIM;
    };
    const uint32_t first = s.before[threadIdx.x];
    if(n <= kOwnLong)
        for(uint32_t j = 0; j < n; j += 4) {
            float *to[4];
            float x[4][DIM];
#pragma unroll
            for(uint32_t u = 0; u < 4; ++u) to[u] = split(s.pair[first + (j + u < n ? j + u : n - 1)], x[u]);
#pragma unroll
            for(uint32_t u = 0; u < 4; ++u)
                if(j + u < n)
#pragma unroll
                    for(int c = 0; c < DIM; ++c) to[u][c] += x[u][c];
        }
    unsigned lists = __ballot_sync(0xffffffffu, s_count[lane * (kOwnThreads / 32) + warp] > kOwnLong);
    for(; lists != 0u; lists &= lists - 1u) {
        const int t = (__ffs(lists) - 1) * (kOwnThreads / 32) + warp;
        const uint32_t m = s_count[t], at = s.before[t];
        if(rows <= kMaxBins) { /* the list is one row's: the lanes add up theirs first */
            float sum[DIM] = {}, one = 0.0f;
#pragma unroll 4
            for(uint32_t j = lane; j < m; j += 32) {
                float x[DIM];
                split(s.pair[at + j], x);
#pragma unroll
                for(int c = 0; c < DIM; ++c) sum[c] += x[c];
            }
#pragma unroll
            for(int c = 0; c < DIM; ++c) {
#pragma unroll
                for(int o = 16; o > 0; o >>= 1) sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], o);
                one = lane == c ? sum[c] : one;
            }
            if(lane < DIM) table[t * DIM + lane] += one;
            continue;
        }
        /* the sums of a step's distinct rows one after another */
        for(uint32_t j = 0; j < m; j += 32) {
            const bool in = j + lane < m;
            float x[DIM];
            float *to = split(s.pair[at + (in ? j + lane : m - 1)], x);
            const uint32_t place = (uint32_t)(to - table);
            unsigned rest = __ballot_sync(0xffffffffu, in);
            while(rest != 0u) {
                const uint32_t one = __shfl_sync(0xffffffffu, place, __ffs(rest) - 1);
                const bool mine = in && place == one;
                float sum = 0.0f; /* lane c: of column c */
#pragma unroll
                for(int c = 0; c < DIM; ++c) {
                    float v = mine ? x[c] : 0.0f;
#pragma unroll
                    for(int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                    sum = lane == c ? v : sum;
                }
                if(lane < DIM) table[one + lane] += sum;
                rest &= ~__ballot_sync(0xffffffffu, mine);
            }
            __syncwarp();
        }
    }
}

/* Longer rows: groups of lanes side by side on the columns.  A group owns the digits whose pairs start in its equal share of
 * the tile (300k x 24 into 500 rows: 29 us; a thread for a digit's pairs, four columns at a time, took 61) and walks them as
 * they lie, storing a sum whenever the row changes. */
template <typename GT>
__device__ __forceinline__ void walk_columns(const OwnShared &s, const GT *s_grad, uint32_t dim, float *table)
{
    const int clog = dim > 16 ? 5 : dim > 8 ? 4 : 3;
    const uint32_t groups = kOwnThreads >> clog, group = threadIdx.x >> clog;
    const uint32_t share = (s.before[kMaxBins] + groups - 1) / groups;
    auto start = [&](uint32_t place) { /* of the first digit whose pairs start there or behind */
        uint32_t lo = 0, hi = kMaxBins;
        while(lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if(s.before[mid] < place) lo = mid + 1;
            else hi = mid;
        }
        return s.before[lo];
    };
    const uint32_t from = start(group * share), to = start((group + 1) * share);
    for(uint32_t c = threadIdx.x & ((1u << clog) - 1u); c < dim; c += 1u << clog) {
        uint32_t row = 0xffffffffu;
        float sum = 0.0f;
        for(uint32_t j = from; j < to; j += 8) {
            uint32_t pair[8];
            float x[8];
#pragma unroll
            for(uint32_t u = 0; u < 8; ++u) pair[u] = s.pair[j + u < to ? j + u : to - 1];
#pragma unroll
            for(uint32_t u = 0; u < 8; ++u) x[u] = to_f32(s_grad[(pair[u] & ((1u << kPlaceBits) - 1u)) * dim + c]);
#pragma unroll
            for(uint32_t u = 0; u < 8; ++u) {
                if(j + u >= to) break;
                if(pair[u] >> kPlaceBits != row) {
                    if(row != 0xffffffffu) table[row * dim + c] += sum;
                    row = pair[u] >> kPlaceBits;
                    sum = 0.0f;
                }
                sum += x[u];
            }
        }
        if(row != 0xffffffffu) table[row * dim + c] += sum;
    }
}

template <typename GT, typename I, int DIM>
__global__ void __launch_bounds__(kOwnThreads, 2) own_table_kernel(const GT *__restrict__ grad, uint32_t stride_bytes,
                                                                   const I *__restrict__ index, uint32_t count, const Use use,
                                                                   uint32_t tile, uint32_t any_dim, float *__restrict__ partial)
{
    const uint32_t dim = DIM > 0 ? DIM : any_dim;
    extern __shared__ __align__(16) unsigned char smem[];
    OwnShared &s = *reinterpret_cast<OwnShared *>(smem);
    const uint32_t size = use.rows * dim;
    GT *s_grad = reinterpret_cast<GT *>(smem + (sizeof(OwnShared) - sizeof(uint32_t) * (kOwnTile - tile)));
    float *table = reinterpret_cast<float *>(s_grad + tile * dim);
    uint32_t *s_count = s.hist[0]; /* of a digit: its pairs; the histograms are done with by then */
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned char *bytes = reinterpret_cast<const unsigned char *>(grad);
    const bool dense = stride_bytes == dim * sizeof(GT) && (uintptr_t)grad % 16 == 0;
    const uint32_t len = own_length(count, gridDim.x);
    const uint32_t begin = len * blockIdx.x < count ? len * blockIdx.x : count, end = count - begin < len ? count : begin + len;
    I raw[kOwnItems]; /* the indices of the next tile */
    auto fetch = [&](uint32_t i0) {
        const uint32_t here = end - i0 < tile ? end - i0 : tile, items = (here + kOwnThreads - 1) / kOwnThreads;
#pragma unroll
        for(uint32_t it = 0; it < kOwnItems; ++it) {
            const uint32_t i = i0 + (uint32_t)warp * 32u * items + it * 32u + (uint32_t)lane;
            raw[it] = __ldg(index + (it < items && i < end ? i : end - 1));
        }
    };
    if(begin < end) fetch(begin);
    for(uint32_t j = threadIdx.x; j < size; j += kOwnThreads) table[j] = 0.0f;
    for(uint32_t i0 = begin; i0 < end; i0 += tile) {
        const uint32_t here = end - i0 < tile ? end - i0 : tile;
        const int items = (int)((here + kOwnThreads - 1) / kOwnThreads);
        /* the tile's gradients, on their way while it is ranked, and the next one's as far as the L2 */
        if(dense) {
            const unsigned char *from = bytes + (uint64_t)i0 * (dim * sizeof(GT));
            unsigned char *to = reinterpret_cast<unsigned char *>(s_grad);
            const uint32_t all = here * dim * (uint32_t)sizeof(GT), whole = all / 16 * 16;
#pragma unroll 4
            for(uint32_t o = threadIdx.x * 16; o < whole; o += kOwnThreads * 16)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to + o)), "l"(from + o)
                             : "memory");
            asm volatile("cp.async.commit_group;" ::: "memory");
            const uint32_t o = whole + threadIdx.x * (uint32_t)sizeof(GT);
            if(o < all) *reinterpret_cast<GT *>(to + o) = *reinterpret_cast<const GT *>(from + o);
            const uint32_t rest = end - i0 - here, next = (rest < tile ? rest : tile) * dim * (uint32_t)sizeof(GT) / 16 * 16;
            if(threadIdx.x == 0 && next > 0)
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from + all), "r"(next) : "memory");
        } else {
            for(uint32_t j = threadIdx.x; j < here * dim; j += kOwnThreads)
                s_grad[j] = reinterpret_cast<const GT *>(bytes + (uint64_t)(i0 + j / dim) * stride_bytes)[j % dim];
        }
        uint32_t k[kOwnItems], p[kOwnItems];
        bool valid[kOwnItems], outside = false;
#pragma unroll
        for(int it = 0; it < kOwnItems; ++it) {
            p[it] = (uint32_t)(warp * 32 * items + it * 32 + lane);
            const bool in = it < items && p[it] < here;
            valid[it] = takes_part(raw[it], use, outside) && in; /* those behind the end repeat the last index */
            k[it] = valid[it] ? (uint32_t)raw[it] : 0u;
        }
        if(outside && use.bad != nullptr) atomicExch(use.bad, 1u);
        const uint32_t n = sort_tile(s, k, p, valid, items, 0, kMaxBits);
        s_count[threadIdx.x] = n;
        if(i0 + here < end) fetch(i0 + here);
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        if constexpr(DIM > 0) walk_lists<GT, DIM>(s, s_count, n, use.rows, s_grad, table);
        else walk_columns(s, s_grad, dim, table);
        __syncthreads();
    }
    __syncthreads();
    for(uint32_t j = threadIdx.x; j < size; j += kOwnThreads) partial[(uint64_t)blockIdx.x * size + j] = table[j];
}

/* the chunks' tables added up: 32 elements a CTA, an eighth of the chunks a warp */
template <typename TT>
__global__ void __launch_bounds__(kThreads) own_join_kernel(const float *partial, uint32_t size, uint32_t chunks, uint32_t dim,
                                                            const Table table)
{
    __shared__ float s_part[kWarps][32];
    gsx_pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t j = blockIdx.x * 32 + lane, per = (chunks + kWarps - 1) / kWarps;
    const uint32_t c0 = per * warp < chunks ? per * warp : chunks, c1 = c0 + per < chunks ? c0 + per : chunks;
    const float *from = partial + (j < size ? j : size - 1);
    float sum[1] = { 0.0f };
#pragma unroll 8
    for(uint32_t c = c0; c < c1; ++c) sum[0] += __ldcg(from + (uint64_t)c * size);
    s_part[warp][lane] = sum[0];
    __syncthreads();
    if(warp != 0 || j >= size) return;
#pragma unroll
    for(int w = 1; w < kWarps; ++w) sum[0] += s_part[w][lane];
    if(table.accumulate && sum[0] == 0.0f) return; /* rows that no index names stay as they are, to the bit */
    store_sums<TT, 1>(table, j / dim, j % dim, sum);
}

/* Chunks of a call that takes this path, or 0: the table fits and leaves room for a tile that is worth its fixed steps.
 * Measured against the sort of all positions (us, here / there): 3M x 3 into 4096 rows 40 / 104, into 1 row 36 / 75;
 * 300k x 3 into 4096 14 / 35; 1000 x 3 into 4096 8 / 14; 2.5M x 15 into 1000 122 / 140; 20000 x 24 into 500 14 / 23.  Rows
 * whose tiles would be shorter than 512: 300k x 45 into 300 50 / 40, 2.5M x 24 into 800 231 / 163; but with few columns and
 * positions 20000 x 24 into 800 17 / 22, 100k x 15 into 1278 20 / 27.  1024 positions a chunk: 1000 x 15 into 1000 17 us,
 * with 512 10. */
uint32_t own_chunks(uint64_t count, uint64_t rows, uint64_t dim)
{
    if(rows * dim * 4 > kOwnTable || own_fit(rows, dim, 4) < (count <= 1u << 18 && dim <= 24 ? 256u : 512u)) return 0;
    const uint64_t chunks = (count + kOwnLeast - 1) / kOwnLeast;
    return (uint32_t)(chunks < 296 ? chunks : 296);
}

/* ------------------------------------------------------------------------------------------ */
/* workspace: n_sorted | counts | pairs, pairs | sums of rows across CTAs */

struct Plan {
    int passes = 0; /* 0: the one-CTA sort */
    int bits[4] = {};
    uint32_t chunks = 0;
    uint32_t own = 0; /* chunks of the path with tables in shared memory */
    /* the sums */
    int clog = 0, nr = 1, run = 8;
    uint32_t ctas = 0, tiles = 1;
    size_t o_counts = 0, o_pairs[2] = {}, o_head = 0, o_tail = 0, bytes = 0;
};

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

/* How the sums lay lanes over columns: packs of a row over 2^clog lanes and NR packs a lane, as few idle ones as
 * possible (fewer packs a lane where that is equal); rows of more than 32 lanes take several CTAs side by side. */
void plan_sums(Plan &p, uint64_t count, uint64_t packs)
{
    uint64_t best = UINT64_MAX;
    for(int nr = 1; nr <= 3; ++nr)
        for(int clog = 2; clog <= 5; ++clog) {
            const uint64_t slots = (uint64_t)nr << clog;
            const uint64_t tiles = (packs + slots - 1) / slots;
            if(tiles > 1 && (clog < 5 || nr > 2)) continue;
            const uint64_t cost = tiles * slots * 16 + (uint64_t)nr;
            if(cost < best) {
                best = cost;
                p.nr = nr;
                p.clog = clog;
                p.tiles = (uint32_t)tiles;
            }
        }
    const uint64_t groups = kThreads >> p.clog;
    /* one wave of CTAs with equal work (four an SM): a second, partly filled wave costs more than the longer runs */
    uint64_t run = (count * p.tiles + groups * 592 - 1) / (groups * 592);
    run = (run + 7) / 8 * 8;
    if(run < 8) run = 8;
    if(run > (uint64_t)kMaxRun) run = kMaxRun;
    if(run > kMaxPositions / groups) run = kMaxPositions / groups;
    p.run = (int)run;
    p.ctas = (uint32_t)((count + groups * run - 1) / (groups * run));
}

/* The layout of one call.  `vec`: elements of a pack.  The sizes do not depend on it or on the pointers, which
 * gsx_b200_embedding_workspace_bytes does not know: they are those of the larger choice. */
Plan make_plan(uint64_t count, uint64_t rows, uint64_t dim, uint64_t vec)
{
    Plan p;
    size_t o = 256;
    p.own = own_chunks(count, rows, dim);
    if(p.own) {
        p.o_head = o;
        p.bytes = o + sizeof(float) * p.own * rows * dim;
        return p;
    }
    if(count > small_count(rows, dim)) {
        int bits = 1;
        while(bits < 32 && (rows - 1) >> bits) ++bits;
        p.passes = (bits + kMaxBits - 1) / kMaxBits;
        for(int i = 0; i < p.passes; ++i) {
            p.bits[i] = (bits + p.passes - 1 - i) / (p.passes - i);
            bits -= p.bits[i];
        }
        /* an element a thread first, then more of them: 10659 positions in 11 chunks, not in two */
        const uint64_t chunks = (count + kSortThreads - 1) / kSortThreads;
        p.chunks = (uint32_t)(chunks < (uint64_t)kChunks ? chunks : kChunks);
        p.o_counts = o;
        o += align256(sizeof(uint32_t) * p.chunks * kMaxBins);
    }
    p.o_pairs[0] = o;
    o += align256(sizeof(uint2) * count);
    p.o_pairs[1] = o;
    if(p.passes > 1) o += align256(sizeof(uint2) * count);
    /* every CTA of the sums has at least 64 positions (8 groups of 8) */
    const size_t ends = align256(sizeof(float) * ((count + 63) / 64) * dim);
    p.o_head = o;
    p.o_tail = o + ends;
    p.bytes = o + 2 * ends;
    plan_sums(p, count, (dim + vec - 1) / vec);
    return p;
}

template <typename I, bool kFirst>
cudaError_t launch_pass(const I *index, const uint2 *pairs, uint32_t count, uint32_t *n_sorted, const Use &use, int shift,
                        int bits, uint32_t chunks, uint32_t *counts, uint2 *out, Zeros zeros, cudaStream_t stream)
{
    constexpr size_t smem = sizeof(SortShared<kSortThreads, kSortItems>);
    cudaError_t e = gsx_allow_smem<digit_scatter_kernel<I, kFirst>>(smem);
    if(e != cudaSuccess) return e;
    if(kFirst)
        digit_count_kernel<I, true><<<chunks + zeros.ctas, kSortThreads, 0, stream>>>(index, pairs, count, n_sorted, use, shift,
                                                                                      bits, chunks, counts, zeros);
    else
        e = gsx_launch_pdl(digit_count_kernel<I, false>, dim3(chunks + zeros.ctas), dim3(kSortThreads), 0, stream, index, pairs,
                           count, n_sorted, use, shift, bits, chunks, counts, zeros);
    Use quiet = use; /* indices are reported once, by the count */
    quiet.bad = nullptr;
    zeros.first += zeros.ctas;
    if(e == cudaSuccess)
        e = gsx_launch_pdl(digit_scatter_kernel<I, kFirst>, dim3(chunks + zeros.ctas), dim3(kSortThreads), smem, stream, index,
                           pairs, count, n_sorted, quiet, shift, bits, chunks, counts, out, zeros);
    return e;
}

template <typename I, int ITEMS>
cudaError_t launch_small_sort(const I *index, uint32_t count, const Use &use, uint2 *pairs, uint32_t *n_sorted, cudaStream_t stream)
{
    constexpr size_t smem = sizeof(SortShared<kSmallThreads, ITEMS>);
    const cudaError_t e = gsx_allow_smem<small_sort_kernel<I, ITEMS>>(smem);
    if(e != cudaSuccess) return e;
    small_sort_kernel<I, ITEMS><<<1, kSmallThreads, smem, stream>>>(index, count, use, pairs, n_sorted);
    return cudaSuccess;
}

/* sorted pairs end up in *out_pairs; the table's rows are zero afterwards (unless it accumulates) */
template <typename I>
cudaError_t launch_sort(const Plan &plan, unsigned char *ws, const void *index_, uint32_t count, const Use &use,
                        const Table &table, uint32_t dim, const uint2 **out_pairs, cudaStream_t stream)
{
    const I *index = static_cast<const I *>(index_);
    uint32_t *n_sorted = reinterpret_cast<uint32_t *>(ws);
    uint2 *pairs[2] = { reinterpret_cast<uint2 *>(ws + plan.o_pairs[0]), reinterpret_cast<uint2 *>(ws + plan.o_pairs[1]) };
    if(plan.passes == 0) {
        *out_pairs = pairs[0];
        cudaError_t e = count <= (uint32_t)(kSmallThreads * kSmallItems)
                            ? launch_small_sort<I, kSmallItems>(index, count, use, pairs[0], n_sorted, stream)
                            : launch_small_sort<I, kBesideItems>(index, count, use, pairs[0], n_sorted, stream);
        if(e == cudaSuccess && !table.accumulate) {
            /* 16 KB of zeros a CTA: many short CTAs write 15% faster than one wave of long ones (6.9 against 6.0 TB/s) */
            const uint64_t ctas = (table.rows * dim * table.bytes + 16383) / 16384;
            e = gsx_launch_pdl(zero_kernel, dim3((unsigned)(ctas < (1u << 30) ? ctas : 1u << 30)), dim3(kThreads), 0, stream,
                               table, dim);
        }
        return e;
    }
    uint32_t *counts = reinterpret_cast<uint32_t *>(ws + plan.o_counts);
    Zeros zeros = { table, dim, 0, 0, 0 };
    if(!table.accumulate) { /* 64 KB a CTA, an equal part of them in each of the kernels */
        const uint32_t kernels = 2u * (uint32_t)plan.passes;
        const uint64_t ctas = (table.rows * dim * table.bytes + 65535) / 65536 / kernels + 1;
        zeros.ctas = (uint32_t)(ctas < (1u << 24) ? ctas : 1u << 24);
        zeros.parts = zeros.ctas * kernels;
    }
    for(int p = 0, shift = 0; p < plan.passes; shift += plan.bits[p], ++p) {
        uint2 *to = pairs[p & 1];
        const cudaError_t e = p == 0 ? launch_pass<I, true>(index, nullptr, count, n_sorted, use, shift, plan.bits[p],
                                                            plan.chunks, counts, to, zeros, stream)
                                     : launch_pass<I, false>(index, pairs[(p - 1) & 1], count, n_sorted, use, shift, plan.bits[p],
                                                             plan.chunks, counts, to, zeros, stream);
        zeros.first += 2 * zeros.ctas;
        if(e != cudaSuccess) return e;
        *out_pairs = to;
    }
    return cudaSuccess;
}

template <typename GT, typename TT, int VW, int NR>
cudaError_t launch_runs(const GT *grad, uint64_t stride, const Plan &plan, const Runs &runs, const Table &table,
                        cudaStream_t stream)
{
    const size_t fixed = sizeof(float) * 2 * kThreads * NR * VW;
    const cudaError_t e = gsx_allow_smem<run_sum_kernel<GT, TT, VW, NR>>(fixed + sizeof(uint2) * (kMaxPositions + kThreads / 4));
    if(e != cudaSuccess) return e;
    return gsx_launch_pdl(run_sum_kernel<GT, TT, VW, NR>, dim3(plan.ctas, plan.tiles), dim3(kThreads),
                          fixed + sizeof(uint2) * (size_t)(kThreads >> plan.clog) * (plan.run + 1), stream, grad,
                          (uint32_t)(stride * sizeof(GT)), runs, table);
}

template <typename GT, typename TT>
cudaError_t launch_sums(const void *grad_, uint64_t stride, uint64_t vec, const Plan &plan, const Runs &runs,
                        const Table &table, cudaStream_t stream)
{
    const GT *grad = static_cast<const GT *>(grad_);
    constexpr int VW = 16 / sizeof(GT);
    cudaError_t e;
    if(vec == (uint64_t)VW)
        e = plan.nr == 1 ? launch_runs<GT, TT, VW, 1>(grad, stride, plan, runs, table, stream)
            : plan.nr == 2 ? launch_runs<GT, TT, VW, 2>(grad, stride, plan, runs, table, stream)
                           : launch_runs<GT, TT, VW, 3>(grad, stride, plan, runs, table, stream);
    else
        e = plan.nr == 1 ? launch_runs<GT, TT, 1, 1>(grad, stride, plan, runs, table, stream)
            : plan.nr == 2 ? launch_runs<GT, TT, 1, 2>(grad, stride, plan, runs, table, stream)
                           : launch_runs<GT, TT, 1, 3>(grad, stride, plan, runs, table, stream);
    if(e == cudaSuccess && plan.ctas > 1)
        e = gsx_launch_pdl(row_join_kernel<TT>, dim3(plan.ctas - 1, (runs.dim + 255) / 256), dim3(kThreads), 0, stream, runs, table);
    return e;
}

template <typename GT, typename TT, typename I>
cudaError_t launch_own(const void *grad, uint64_t stride, const void *index, uint32_t count, const Use &use, const Plan &plan,
                       float *partial, const Table &table, uint32_t dim, cudaStream_t stream)
{
    const uint32_t size = (uint32_t)table.rows * dim;
    const uint32_t tile = own_tile(own_length(count, plan.own), (uint32_t)table.rows, dim, sizeof(GT));
    auto launch = [&](auto kernel, cudaError_t e) {
        if(e != cudaSuccess) return e;
        const size_t smem = sizeof(OwnShared) - sizeof(uint32_t) * (kOwnTile - tile) + (size_t)tile * dim * sizeof(GT) + 4 * (size_t)size;
        kernel<<<plan.own, kOwnThreads, smem, stream>>>(static_cast<const GT *>(grad), (uint32_t)(stride * sizeof(GT)),
                                                        static_cast<const I *>(index), count, use, tile, dim, partial);
        return cudaSuccess;
    };
    cudaError_t e;
    switch(dim) {
    case 1: e = launch(own_table_kernel<GT, I, 1>, gsx_allow_smem<own_table_kernel<GT, I, 1>>(kOwnMemory)); break;
    case 2: e = launch(own_table_kernel<GT, I, 2>, gsx_allow_smem<own_table_kernel<GT, I, 2>>(kOwnMemory)); break;
    case 3: e = launch(own_table_kernel<GT, I, 3>, gsx_allow_smem<own_table_kernel<GT, I, 3>>(kOwnMemory)); break;
    case 4: e = launch(own_table_kernel<GT, I, 4>, gsx_allow_smem<own_table_kernel<GT, I, 4>>(kOwnMemory)); break;
    default: e = launch(own_table_kernel<GT, I, 0>, gsx_allow_smem<own_table_kernel<GT, I, 0>>(kOwnMemory)); break;
    }
    if(e != cudaSuccess) return e;
    return gsx_launch_pdl(own_join_kernel<TT>, dim3((size + 31) / 32), dim3(kThreads), 0, stream, (const float *)partial, size,
                          plan.own, dim, table);
}

bool float_type(int t) { return t == GSX_B200_DATA_F32 || t == GSX_B200_DATA_F16 || t == GSX_B200_DATA_BF16; }
uint64_t float_bytes(int t) { return t == GSX_B200_DATA_F32 ? 4 : 2; }

int launch_status(cudaError_t e)
{
    const cudaError_t last = cudaGetLastError();
    if(e == cudaSuccess) e = last;
    return e == cudaSuccess ? GSX_B200_SUCCESS : gsx_internal_fail(GSX_B200_UNKNOWN, cudaGetErrorString(e));
}

/* whether two spans of rows share bytes */
bool overlap(const void *a, uint64_t a_rows, uint64_t a_step, uint64_t a_row, const void *b, uint64_t b_rows, uint64_t b_step,
             uint64_t b_row)
{
    if(a_rows == 0 || b_rows == 0) return false;
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + (b_rows - 1) * b_step + b_row && y < x + (a_rows - 1) * a_step + a_row;
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
       (uintptr_t)index % (index_type == GSX_B200_DATA_I32 ? 4 : 8) || (uintptr_t)device_out_of_range % 4)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "pointers must be aligned to their element type");
    if(table_stride * float_bytes(table_type) > 0xffffffffull)
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "table_stride must be below 4 GiB");
    if(count * dim / 256 > (uint64_t)INT32_MAX)
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "count * dim must be below 2^39");
    const uint64_t tb = float_bytes(table_type), ob = float_bytes(out_type), ib = index_type == GSX_B200_DATA_I32 ? 4 : 8;
    if(overlap(out, count, out_stride * ob, dim * ob, table, rows, table_stride * tb, dim * tb) ||
       overlap(out, count, out_stride * ob, dim * ob, index, 1, 0, count * ib))
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "out must not overlap table or index");
    cudaStream_t stream = (cudaStream_t)stream_;
    cudaError_t e = cudaSuccess;
    GSX_WITH_FLOAT_TYPE(table_type, T, GSX_WITH_FLOAT_TYPE(out_type, O, {
        e = index_type == GSX_B200_DATA_I32 ? launch_lookup<T, O, int32_t>(table, rows, dim, table_stride, index, count, scale, out,
                                                                           out_stride, device_out_of_range, stream)
                                            : launch_lookup<T, O, int64_t>(table, rows, dim, table_stride, index, count, scale, out,
                                                                           out_stride, device_out_of_range, stream);
    }));
    return launch_status(e);
}

extern "C" uint64_t gsx_b200_embedding_workspace_bytes(uint64_t count, uint64_t rows, uint64_t dim)
{
    if(count > (uint64_t)INT32_MAX || rows > (uint64_t)INT32_MAX || dim > (uint64_t)INT32_MAX || rows == 0) return 0;
    return make_plan(count, rows, dim, 1).bytes;
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
    if(grad_stride * float_bytes(grad_type) > 0xffffffffull)
        return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "grad_stride must be below 4 GiB");
    if(padding_row >= (int64_t)rows) return gsx_internal_fail(GSX_B200_OUT_OF_RANGE, "padding_row must be below rows");
    if(dim == 0 || (rows == 0 && count == 0)) return GSX_B200_SUCCESS;
    if(rows == 0) return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "rows must be positive");
    if(grad_table == nullptr || workspace == nullptr || (count > 0 && (grad_out == nullptr || index == nullptr)))
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "grad_out, index, grad_table and workspace must be non-null");
    if((uintptr_t)grad_out % float_bytes(grad_type) || (uintptr_t)grad_table % float_bytes(table_type) ||
       (uintptr_t)index % (index_type == GSX_B200_DATA_I32 ? 4 : 8) || (uintptr_t)device_out_of_range % 4 || (uintptr_t)workspace % 16)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT,
                                 "pointers must be aligned to their element type, the workspace to 16 bytes");
    if(!(scale - scale == 0.0f)) return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "scale must be finite");
    {
        const uint64_t tb = float_bytes(table_type), ob = float_bytes(grad_type), ib = index_type == GSX_B200_DATA_I32 ? 4 : 8;
        if(overlap(grad_table, rows, table_stride * tb, dim * tb, grad_out, count, grad_stride * ob, dim * ob) ||
           overlap(grad_table, rows, table_stride * tb, dim * tb, index, 1, 0, count * ib))
            return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "grad_table must not overlap grad_out or index");
    }
    Table table;
    table.data = grad_table;
    table.stride = table_stride;
    table.rows = rows;
    table.scale = scale;
    table.bytes = (int)float_bytes(table_type);
    table.accumulate = accumulate != 0;
    const uint64_t gb = float_bytes(grad_type), pack = 16 / gb;
    const uint64_t tb = float_bytes(table_type) * pack < 16 ? float_bytes(table_type) * pack : 16;
    const bool packs = dim % pack == 0 && grad_stride % pack == 0 && (uintptr_t)grad_out % 16 == 0 &&
                       (uintptr_t)grad_table % tb == 0 && table_stride * float_bytes(table_type) % tb == 0;
    const uint64_t vec = packs ? pack : 1;
    const Plan plan = make_plan(count, rows, dim, vec);
    if(workspace_bytes < plan.bytes)
        return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT,
                                 "workspace is smaller than gsx_b200_embedding_workspace_bytes");
    {
        const uint64_t tb = float_bytes(table_type), ob = float_bytes(grad_type), ib = index_type == GSX_B200_DATA_I32 ? 4 : 8;
        if(overlap(workspace, 1, 0, plan.bytes, grad_table, rows, table_stride * tb, dim * tb) ||
           overlap(workspace, 1, 0, plan.bytes, grad_out, count, grad_stride * ob, dim * ob) ||
           overlap(workspace, 1, 0, plan.bytes, index, 1, 0, count * ib))
            return gsx_internal_fail(GSX_B200_INVALID_ARGUMENT, "workspace must not overlap grad_table, grad_out or index");
    }
    cudaStream_t stream = (cudaStream_t)stream_;
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    const Use use = { (uint32_t)rows, padding_row < 0 ? UINT32_MAX : (uint32_t)padding_row, device_out_of_range };
    cudaError_t e = cudaSuccess;
    if(plan.own) {
        GSX_WITH_FLOAT_TYPE(grad_type, GT, GSX_WITH_FLOAT_TYPE(table_type, TT, {
            float *partial = reinterpret_cast<float *>(ws + plan.o_head);
            e = index_type == GSX_B200_DATA_I32
                    ? launch_own<GT, TT, int32_t>(grad_out, grad_stride, index, (uint32_t)count, use, plan, partial, table, (uint32_t)dim, stream)
                    : launch_own<GT, TT, int64_t>(grad_out, grad_stride, index, (uint32_t)count, use, plan, partial, table, (uint32_t)dim, stream);
        }));
        return launch_status(e);
    }
    Runs runs;
    e = index_type == GSX_B200_DATA_I32
            ? launch_sort<int32_t>(plan, ws, index, (uint32_t)count, use, table, (uint32_t)dim, &runs.pairs, stream)
            : launch_sort<int64_t>(plan, ws, index, (uint32_t)count, use, table, (uint32_t)dim, &runs.pairs, stream);
    if(e != cudaSuccess || count == 0) return launch_status(e);
    runs.n_sorted = reinterpret_cast<const uint32_t *>(ws);
    runs.head = reinterpret_cast<float *>(ws + plan.o_head);
    runs.tail = reinterpret_cast<float *>(ws + plan.o_tail);
    runs.dim = (uint32_t)dim;
    runs.clog = plan.clog;
    runs.run = plan.run;
    GSX_WITH_FLOAT_TYPE(grad_type, GT, GSX_WITH_FLOAT_TYPE(table_type, TT, {
        e = launch_sums<GT, TT>(grad_out, grad_stride, vec, plan, runs, table, stream);
    }));
    return launch_status(e);
}
