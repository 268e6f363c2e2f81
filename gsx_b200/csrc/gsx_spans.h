/*
 * Host-side test of whether two strided sets of bytes share one: what a call's outputs must not do.
 */
#ifndef GSX_SPANS_H
#define GSX_SPANS_H

#include <stdint.h>

#include <initializer_list>

/* `bytes` consecutive bytes at `at` and at every combination of up to three steps from there (a row, its group, its outer group) */
struct GsxRows {
    struct Dim {
        uint64_t count, step;
    };
    int64_t at;
    uint64_t bytes;
    Dim dim[3]; /* those of more than one place, the longest step first */
    int dims;
    bool empty;
    static constexpr uint64_t kMost = 1ull << 62; /* longer steps and extents count as this, so that no sum wraps */

    GsxRows() : at(0), bytes(0), dims(0), empty(true) {}
    GsxRows(const void *p, uint64_t row_bytes, std::initializer_list<Dim> all = {}) : at((int64_t)(uintptr_t)p), bytes(row_bytes), dims(0)
    {
        empty = p == nullptr || row_bytes == 0;
        for(const Dim &d : all) {
            empty |= d.count == 0;
            if(d.count <= 1 || dims == 3) continue;
            int k = dims++;
            const uint64_t step = d.step < kMost ? d.step : kMost;
            for(; k > 0 && dim[k - 1].step < step; --k) dim[k] = dim[k - 1];
            dim[k] = { d.count, step };
        }
    }
    /* bytes from the first to the last of what lies under dimensions i and further */
    uint64_t extent(int i) const
    {
        unsigned __int128 n = bytes;
        for(int k = i; k < dims; ++k) n += (unsigned __int128)(dim[k].count - 1) * dim[k].step;
        return n < kMost ? (uint64_t)n : kMost;
    }
    /* every step is at least as long as what lies under it, so no byte is in two places */
    bool nested() const
    {
        for(int k = 0; !empty && k < dims; ++k)
            if(dim[k].step < extent(k + 1)) return false;
        return true;
    }
};

/* whether a (from its dimension i on, at x) and b (j, y) share a byte; both nested.  Where it would take more than `left`
 * steps to tell, they count as sharing one: steps of different lengths that interleave many times over. */
inline bool gsx_rows_meet(const GsxRows &a, int i, int64_t x, const GsxRows &b, int j, int64_t y, int &left)
{
    const int64_t ea = (int64_t)a.extent(i), eb = (int64_t)b.extent(j);
    if(x + ea <= y || y + eb <= x) return false;
    if(i == a.dims && j == b.dims) return true;
    if(--left < 0) return true;
    /* x / s rounded down */
    auto floor_div = [](int64_t v, int64_t s) { return v / s - (v % s < 0); };
    if(i < a.dims && j < b.dims && a.dim[i].step == b.dim[j].step) {
        /* what lies under place k of a and place l of b: it only matters how far l - k is */
        const int64_t s = (int64_t)a.dim[i].step, ia = (int64_t)a.extent(i + 1), ib = (int64_t)b.extent(j + 1), d = y - x;
        int64_t lo = floor_div(-ib - d, s) + 1, hi = floor_div(ia - d - 1, s); /* -ib < d + t * s < ia */
        if(lo < -((int64_t)a.dim[i].count - 1)) lo = -((int64_t)a.dim[i].count - 1);
        if(hi > (int64_t)b.dim[j].count - 1) hi = (int64_t)b.dim[j].count - 1;
        for(int64_t t = lo; t <= hi; ++t)
            if(gsx_rows_meet(a, i + 1, x, b, j + 1, y + t * s, left)) return true;
        return false;
    }
    if(i == a.dims || (j < b.dims && b.dim[j].step > a.dim[i].step)) return gsx_rows_meet(b, j, y, a, i, x, left);
    /* the places of a's longest step under which something reaches into b */
    const int64_t s = (int64_t)a.dim[i].step, ia = (int64_t)a.extent(i + 1);
    int64_t lo = floor_div(y - ia - x, s) + 1, hi = floor_div(y + eb - 1 - x, s); /* y - ia < x + t * s < y + eb */
    if(lo < 0) lo = 0;
    if(hi > (int64_t)a.dim[i].count - 1) hi = (int64_t)a.dim[i].count - 1;
    for(int64_t t = lo; t <= hi; ++t)
        if(gsx_rows_meet(a, i + 1, x + t * s, b, j, y, left)) return true;
    return false;
}

inline bool gsx_rows_meet(const GsxRows &a, const GsxRows &b)
{
    int left = 4096;
    return !a.empty && !b.empty && gsx_rows_meet(a, 0, a.at, b, 0, b.at, left);
}

#endif
