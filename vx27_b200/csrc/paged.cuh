// The paged KV cache's address arithmetic and argument checks (include/vx27_paged.h).
#pragma once
#include "common.cuh"

namespace vx27 {

constexpr int PG_HD = 256;

// Pool of pages, bf16 [n_pages][nkv][1 << ps_log][256].
struct PagePool {
    int n_pages, nkv, ps_log;
    // Row of slot `slot`, KV head h, in page `page` (counted in rows of 256 elements).
    __host__ __device__ size_t row(int page, int h, int slot) const {
        return (((size_t)page * nkv + h) << ps_log) + (slot & ((1 << ps_log) - 1));
    }
    __device__ bool has(int page) const { return (unsigned)page < (unsigned)n_pages; }
};

// Which of the n slots up to and with its own a token attends to: [0, sink_end) and
// [win_begin, n). Without a window win_begin is 0 and sink_end 0.
struct SeenSlots {
    int n, win_begin, sink_end;
    __host__ __device__ SeenSlots(int n_, int window, int sinks) : n(n_) {
        win_begin = window > 0 && n > window ? n - window : 0;
        sink_end = sinks < win_begin ? sinks : win_begin;
    }
    __host__ __device__ bool sees(int j) const {
        return j < n && (j >= win_begin || j < sink_end);
    }
};

// log2 of a supported page size, -1 for others.
inline int page_size_log(int page_size) {
    for (int l = 4; l <= 8; l++)
        if (page_size == 1 << l) return l;
    return -1;
}

// The checks that every call over a pool makes.
inline int check_pool(const char *fn, const void *k, const void *v, int n_pages, int page_size,
                      const void *table, int max_pages, int nkv, int hd, char *err,
                      size_t errlen) {
    if (hd != PG_HD) return fail(err, errlen, "%s: hd=%d unsupported (256 only)", fn, hd);
    if (page_size_log(page_size) < 0)
        return fail(err, errlen, "%s: page_size=%d (16, 32, 64, 128 or 256)", fn, page_size);
    if (nkv <= 0 || nkv > 65535 || n_pages <= 0 || max_pages <= 0)
        return fail(err, errlen, "%s: bad shape nkv=%d n_pages=%d max_pages=%d", fn, nkv, n_pages,
                    max_pages);
    // rows are 32-bit coordinates of the tensor maps, slots 32-bit everywhere
    if ((long long)n_pages * nkv * page_size > 0x7fffffffLL - 256 ||
        (long long)max_pages * page_size > 0x7fffffffLL - 256)
        return fail(err, errlen, "%s: %d pages of %d slots, %d pages a sequence: over 2^31 rows",
                    fn, n_pages, page_size, max_pages);
    if (!k || !v || !table) return fail(err, errlen, "%s: null pointer argument", fn);
    if (((uintptr_t)k | (uintptr_t)v) & 15)
        return fail(err, errlen, "%s: k_pages and v_pages must be 16-byte aligned", fn);
    return 0;
}

inline int check_heads(const char *fn, int nq, int nkv, char *err, size_t errlen) {
    if (nq <= 0 || nkv <= 0 || nq % nkv || nq / nkv > 8)
        return fail(err, errlen, "%s: nq=%d, nkv=%d (1 to 8 query heads per KV head)", fn, nq, nkv);
    return 0;
}

inline int check_window(const char *fn, int window, int sinks, char *err, size_t errlen) {
    if (window < 0 || sinks < 0 || (!window && sinks))
        return fail(err, errlen, "%s: window=%d, sinks=%d (sinks need a window, neither is negative)",
                    fn, window, sinks);
    return 0;
}

}  // namespace vx27
