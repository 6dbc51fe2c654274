// Keys and values in pages (tah_pages, include/tah.h): the pool as the kernels see it, and where a row of a table lies.
#pragma once

#include "common.hpp"

namespace tah {

// A pool on the card with its tables' pages. A page is heads parts of head_bytes: keys [rows][hd], values [hd][rows], then for
// ints the key and the value steps [rows].
struct PageSet {
    uint8_t *pool;
    const int32_t *table;
    int heads, hd, rows, log_rows;
    int pages, tables, ld;
    size_t head_bytes, page_bytes;
};

__host__ __device__ constexpr int page_width(int fmt) { return fmt == TAH_KV_F32 ? 4 : (fmt == TAH_KV_I16 ? 2 : 1); }

// the page of row `at` of table t, or -1 where it has none
__device__ __forceinline__ int page_of(const PageSet &p, int t, long at) {
    const long i = at >> p.log_rows;
    if (at < 0 || i >= p.ld) return -1;
    const int id = p.table[(size_t)t * p.ld + i];
    return (unsigned)id < (unsigned)p.pages ? id : -1;
}

// the last t in [0, tables) with offsets[t] <= r (0 if there is none): the table of row r where its rows begin at offsets[t]
__device__ __forceinline__ int table_of(const int32_t *offsets, int tables, int r) {
    int lo = 0, hi = tables;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid] <= r)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// The rows of a call into pages (k, v read) or from them (k, v written).
void pages_rows(hipStream_t s, int fmt, const PageSet &p, const int32_t *starts, const int32_t *offsets, float *k, float *v,
                int rows, size_t row_ld, bool write);

// The queries' attention (pages_attend.hip), work of pages_attend_work_bytes (which refuses calls that are too large).
size_t pages_attend_work_bytes(int fmt, const PageSet &p, int nq, int heads);
void pages_attend(hipStream_t s, int fmt, const PageSet &p, const int32_t *lengths, const float *q, const int32_t *offsets, int nq,
                  int heads, bool causal, size_t q_ld, float *out, void *work);

}  // namespace tah
