// paged.h - what the kernels of the paged key / value cache share: the row -> sequence search, the key -> page arithmetic.
#pragma once
#include "common.h"
#include <initializer_list>

namespace mm {

// q = n / d for 0 <= n < 2^31 without a division: with l = ceil(log2 d) and m = floor(2^32 (2^l - d) / d) + 1,
// n / d = (mulhi(m, n) + n) >> l exactly (m / 2^32 + 1 is 2^l / d rounded up by less than 2^l / 2^32).  mulhi(m, n) < n, so the
// sum stays below 2^32.
struct FastDiv {
    uint32_t d, m, l;
};
inline FastDiv make_fastdiv(int d) {
    FastDiv f;
    f.d = (uint32_t)d;
    f.l = 0;
    while ((1ull << f.l) < (uint64_t)d) ++f.l;
    f.m = (uint32_t)((((1ull << f.l) - (uint64_t)d) << 32) / (uint64_t)d + 1);
    return f;
}
__device__ __forceinline__ uint32_t fdiv(uint32_t n, const FastDiv& f) { return (__umulhi(f.m, n) + n) >> f.l; }

// A key's place in the cache while a thread walks the keys of a sequence in equal steps: its page's index in the block table and
// the bytes from the page's start to its slot.  A step of n keys is n / page_size pages and n % page_size slots, so that moving on
// takes two additions and a conditional carry, and no division or multiplication.
struct PageStep {
    uint32_t pages, bytes;  // n / page_size, (n % page_size) slots in bytes
};
__device__ __forceinline__ PageStep page_step(uint32_t n, const FastDiv& f, uint32_t slot_bytes) {
    const uint32_t p = fdiv(n, f);
    return PageStep{p, (n - p * f.d) * slot_bytes};
}
struct PageCursor {
    uint32_t page, byte;
    __device__ __forceinline__ void set(uint32_t key, const FastDiv& f, uint32_t slot_bytes) {
        page = fdiv(key, f);
        byte = (key - page * f.d) * slot_bytes;
    }
    __device__ __forceinline__ void move(const PageStep& s, uint32_t page_bytes) {
        page += s.pages;
        byte += s.bytes;
        const bool c = byte >= page_bytes;
        byte -= c ? page_bytes : 0u;
        page += c ? 1u : 0u;
    }
};

// The sequence of packed row `row` in cu[0 .. n]: the number of i with cu[i + 1] <= row, found by a whole wave, 64 boundaries a
// step (one step up to 64 sequences, two up to 4096).  n when the row is behind the last sequence; the caller also checks
// cu[s] <= row.  Whatever cu holds, only cu[1 .. n] is read and the result is in [0, n].
__device__ __forceinline__ int find_seq(const int32_t* __restrict__ cu, int n, int row, int lane) {
    int lo = 0;
    for (;;) {
        const int step = (n + 63) >> 6;
        const int i = lane * step + step - 1;  // the last boundary of this lane's group
        const bool below = i < n && cu[lo + i + 1] <= row;
        const int g = __popcll(__ballot(below));  // groups that lie wholly before the row
        lo += g * step;
        n -= g * step;
        if (step == 1 || n <= 0) return lo;
        n = n < step ? n : step;
    }
}

// Host side: do operands share memory?  An operand is rows x heads runs of `width` bytes, strides in bytes.
struct Runs {
    const void* p;
    int64_t row, head, width;
    int rows, heads;
    int64_t first() const { return (int64_t)(uintptr_t)p + (row < 0 ? (rows - 1) * row : 0) + (head < 0 ? (heads - 1) * head : 0); }
    int64_t end() const { return (int64_t)(uintptr_t)p + (row > 0 ? (rows - 1) * row : 0) + (head > 0 ? (heads - 1) * head : 0) + width; }
    bool same(const Runs& o) const { return p == o.p && heads == o.heads && (rows == 1 || row == o.row) && (heads == 1 || head == o.head); }
};
// |d + n row| < width for some |n| < rows: two runs d apart, or some rows further on
inline bool meets(int64_t d, int64_t row, int rows, int64_t width) {
    int64_t near = row == 0 ? 0 : -d / row;
    near = near < 1 - rows ? 1 - rows : near > rows - 1 ? rows - 1 : near;
    for (int64_t n = near - 1; n <= near + 1; ++n)
        if (n > -rows && n < rows && d + n * row < width && d + n * row > -width) return true;
    return false;
}
inline bool overlaps_itself(const Runs& a) {
    const int64_t row = a.row < 0 ? -a.row : a.row, head = a.head < 0 ? -a.head : a.head;
    if (a.rows > 1 && row < a.width) return true;
    if (a.heads > 1 && head < a.width) return true;
    if (a.rows == 1 || a.heads == 1 || row >= (a.heads - 1) * head + a.width || head >= (a.rows - 1) * row + a.width) return false;
    for (int i = 1; i < a.heads; ++i)
        if (meets(i * a.head, a.row, a.rows, a.width)) return true;
    return false;
}
// Exact for operands of the same rows and row stride (slices of one tensor); others count as overlapping if the stretches of memory they span do.
inline bool overlap(const Runs& a, const Runs& b) {
    if (a.end() <= b.first() || b.end() <= a.first()) return false;
    if (a.rows != b.rows || a.width != b.width || (a.rows > 1 && a.row != b.row)) return true;
    const int64_t d = (int64_t)(uintptr_t)a.p - (int64_t)(uintptr_t)b.p;
    if (a.head == b.head && a.head >= 2 * a.width && a.row % a.head == 0) {  // e.g. [rows, heads, 3, hn]: places within a head
        const int64_t at = (d % a.head + a.head) % a.head;
        if (at >= a.width && at <= a.head - a.width) return false;
    }
    if (a.head != b.head && (int64_t)a.heads * b.heads > 1 << 16) return true;  // not worth the search
    for (int i = 0; i < a.heads; ++i)
        for (int j = 0; j < b.heads; ++j) {
            if (a.head == b.head && i > 0 && j > 0) break;  // the difference i - j has been seen
            if (meets(d + i * a.head - j * b.head, a.row, a.rows, a.width)) return true;
        }
    return false;
}

inline int check_paged(const char* fn, const mm_paged_kv* kv, const mm_paged_step* st, int rows) {
    MM_CHECK_ARG(kv && st, "%s: null cache or step", fn);
    MM_CHECK_ARG(kv->k && kv->v && (st->seqs == 0 || (st->block_table && st->cu_new && st->kv_lens)), "%s: null pointer", fn);
    MM_CHECK_ARG(kv->hn == 64 || kv->hn == 128, "%s: head size %d not supported (64 or 128)", fn, kv->hn);
    MM_CHECK_ARG(kv->num_pages > 0 && kv->page_size > 0 && kv->heads > 0 && rows >= 0 && st->seqs >= 0 && st->max_pages > 0,
                 "%s: pages=%d page_size=%d heads=%d rows=%d seqs=%d max_pages=%d out of range", fn, kv->num_pages, kv->page_size,
                 kv->heads, rows, st->seqs, st->max_pages);
    MM_CHECK_ARG((int64_t)st->max_pages * kv->page_size < (int64_t)1 << 30, "%s: %d pages of %d slots exceed 2^30 positions", fn,
                 st->max_pages, kv->page_size);
    MM_CHECK_ARG(st->max_new >= 0 && st->max_kv >= 0 && st->table_stride >= st->max_pages,
                 "%s: max_new=%d max_kv=%d table_stride=%lld out of range", fn, st->max_new, st->max_kv, (long long)st->table_stride);
    MM_CHECK_ARG(aligned16(kv->k) && aligned16(kv->v), "%s: the cache must be 16-byte aligned", fn);
    for (int64_t x : {kv->page, kv->head, kv->slot})
        MM_CHECK_ARG(x > 0 && x % 8 == 0 && x < (int64_t)1 << 31, "%s: cache stride %lld must be a multiple of 8 in (0, 2^31)", fn, (long long)x);
    MM_CHECK_ARG(kv->page_size * kv->slot < (int64_t)1 << 30, "%s: a page's slots span 2^30 elements or more", fn);
    return MM_OK;
}

}  // namespace mm
