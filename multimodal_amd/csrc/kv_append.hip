// kv_append.hip - new keys and values into the pages of a cache, the rotary embedding applied on the way.
//
// y[0 : d] = x[0 : d] cos[p] + rotate_half(x[0 : d]) sin[p] for keys and queries (reference
// megatron/model/positional_embeddings.py:69-92; rotate_half(x) = [-x2 | x1] of the two halves), v copied, p the row's position.
// Products and sum stay in fp32 and are rounded once (the training path rounds each product as the eager reference does).
//
// Bound by HBM: every element is read once and written once.  A work item is two chunks of W elements of one head's row - for a
// rotated head the chunk and its partner half a rotation further, so that the rotation needs no exchange between lanes; the
// lanes of a head's row are neighbours, so every access is a contiguous run of at least d bytes.  W = 8 (16-byte accesses) when
// rows and rotation allow it, else W = 1.
// Measured: 4 prompts of 2001 .. 2048 tokens, 32 + 2 x 32 heads of 128: 76 us, 399 MB at 5.3 TB/s, what a large copy reaches; 16 of
// 2048, 32 + 2 x 8 heads: 159 us, 806 MB at 5.1 TB/s; 256 rows of one token 4.6 us, one row 2.6 us, the latency of sequence ->
// length -> page.
#include "common.h"
#include "paged.h"

namespace mm {

struct AppendArgs {
    mm_paged_kv kv;
    mm_paged_step st;
    const u16 *k, *v, *q;
    u16* q_out;
    int64_t k_row, k_head, v_row, v_head, q_row, q_head, qo_row, qo_head;
    const void *cos, *sin;
    int nq, rows, rot_d, table_rows;
    FastDiv page;
};

template <typename T, int W> __device__ __forceinline__ void load_chunk(const u16* __restrict__ p, float (&f)[W]) {
    if constexpr (W == 8) unpack8<T>(*reinterpret_cast<const u32x4*>(p), f);
    else f[0] = to_f32<T>(*p);
}
template <int W> __device__ __forceinline__ void load_chunk_f32(const float* __restrict__ p, float (&f)[W]) {
    if constexpr (W == 8) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = a[i], f[4 + i] = b[i];
    } else f[0] = *p;
}
template <typename T, int W> __device__ __forceinline__ void store_chunk(u16* __restrict__ p, const float (&f)[W]) {
    if constexpr (W == 8) *reinterpret_cast<u32x4*>(p) = pack8<T>(f);
    else *p = from_f32<T>(f[0]);
}

// Where a row goes: its position, and the elements from the first page to its slot of head 0; -1: no such place, -2: padding, the
// row belongs to no sequence.
struct RowPlace {
    int64_t slot;
    int pos;
};
__device__ __forceinline__ bool is_padding(const AppendArgs& a, int row, int seq) { return seq >= a.st.seqs || a.st.cu_new[seq] > row; }
__device__ __forceinline__ RowPlace place_of(const AppendArgs& a, int row, int seq) {
    const int64_t pos64 = (int64_t)a.st.kv_lens[seq] - a.st.cu_new[seq + 1] + row;
    const bool ok = pos64 >= 0 && pos64 < (int64_t)a.st.max_pages * a.kv.page_size && (a.rot_d == 0 || pos64 < a.table_rows);
    const int pos = ok ? (int)pos64 : 0;
    const int pi = (int)fdiv((uint32_t)pos, a.page);
    const int page = a.st.block_table[(int64_t)seq * a.st.table_stride + pi];
    if (!ok || page < 0 || page >= a.kv.num_pages) return RowPlace{-1, 0};
    return RowPlace{(int64_t)page * a.kv.page + (int64_t)(pos - pi * a.kv.page_size) * a.kv.slot, pos};
}

// one work item: its two chunks loaded (a row that is no padding can be read before it is known where it goes), then rotated and stored
template <typename T, typename TT, int W, int HN> struct Item {
    static constexpr int IPH = HN / (2 * W);  // items per head
    int slot, c1, c2;
    bool rot;
    float x1[W], x2[W];
    __device__ __forceinline__ bool load(const AppendArgs& a, int row, int item) {
        slot = item / IPH;
        const int c = item % IPH, nkv = a.kv.heads, hc = a.rot_d / (2 * W);  // chunks per half of the rotated dims
        if (slot >= a.nq + 2 * nkv) return false;
        const u16* src;
        if (slot < a.nq) src = a.q + (int64_t)row * a.q_row + (int64_t)slot * a.q_head;
        else if (slot < a.nq + nkv) src = a.k + (int64_t)row * a.k_row + (int64_t)(slot - a.nq) * a.k_head;
        else src = a.v + (int64_t)row * a.v_row + (int64_t)(slot - a.nq - nkv) * a.v_head;
        rot = slot < a.nq + nkv && c < hc;
        // the item's two chunks: partners in the rotated part; behind it (everywhere for an unrotated row) neighbours
        c1 = rot ? c : 2 * c, c2 = rot ? c + hc : 2 * c + 1;
        load_chunk<T, W>(src + c1 * W, x1);
        load_chunk<T, W>(src + c2 * W, x2);
        return true;
    }
    __device__ __forceinline__ void store(const AppendArgs& a, int row, const RowPlace& to) {
        u16* dst;
        if (slot < a.nq) dst = a.q_out + (int64_t)row * a.qo_row + (int64_t)slot * a.qo_head;
        else {
            if (to.slot < 0) return;  // no place for it
            const bool is_k = slot < a.nq + a.kv.heads;
            dst = (u16*)(is_k ? a.kv.k : a.kv.v) + to.slot + (int64_t)(slot - a.nq - (is_k ? 0 : a.kv.heads)) * a.kv.head;
        }
        if (rot) {
            float k1[W], k2[W], s1[W], s2[W];
            const TT* ct = (const TT*)a.cos + (int64_t)to.pos * a.rot_d;
            const TT* st = (const TT*)a.sin + (int64_t)to.pos * a.rot_d;
            if constexpr (sizeof(TT) == 4) {
                load_chunk_f32<W>(ct + c1 * W, k1), load_chunk_f32<W>(ct + c2 * W, k2);
                load_chunk_f32<W>(st + c1 * W, s1), load_chunk_f32<W>(st + c2 * W, s2);
            } else {
                load_chunk<T, W>(ct + c1 * W, k1), load_chunk<T, W>(ct + c2 * W, k2);
                load_chunk<T, W>(st + c1 * W, s1), load_chunk<T, W>(st + c2 * W, s2);
            }
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float y1 = fmaf(x1[j], k1[j], -(x2[j] * s1[j])), y2 = fmaf(x2[j], k2[j], x1[j] * s2[j]);
                x1[j] = y1;
                x2[j] = y2;
            }
        }
        if (to.slot < 0)  // only queries come here: a row without a place must not pass for a number
#pragma unroll
            for (int j = 0; j < W; ++j) x1[j] = x2[j] = __builtin_nanf("");
        store_chunk<T, W>(dst + c1 * W, x1);
        store_chunk<T, W>(dst + c2 * W, x2);
    }
};

// Few rows: block b moves items [256 i, 256 i + 256) of row b / parts, i = b % parts (all of one row, so that the sequence search
// and the page look-up are uniform over the block)
template <typename T, typename TT, int W, int HN>
__global__ __launch_bounds__(256) void paged_kv_append_k(const AppendArgs a, int parts) {
    const int row = blockIdx.x / parts;
    const int seq = find_seq(a.st.cu_new, a.st.seqs, row, threadIdx.x & 63);
    if (is_padding(a, row, seq)) return;
    Item<T, TT, W, HN> it;
    const bool live = it.load(a, row, (blockIdx.x - row * parts) * 256 + threadIdx.x);
    const RowPlace to = place_of(a, row, seq);
    if (live) it.store(a, row, to);
}
// Many rows: a block moves `per` rows, whose places are looked up side by side, one lane each
template <typename T, typename TT, int W, int HN>
__global__ __launch_bounds__(256) void paged_kv_append_rows_k(const AppendArgs a, int per, FastDiv items) {
    __shared__ RowPlace places[64];
    const int row0 = blockIdx.x * per, n = min(per, a.rows - row0), tid = threadIdx.x;
    if (tid < 64) {
        int seq = find_seq(a.st.cu_new, a.st.seqs, row0, tid);
        if (tid < n) {
            // the row's own sequence: rarely far behind the first row's; sequences without rows may lie between
            int step = 0;
            while (step < 4 && seq < a.st.seqs && a.st.cu_new[seq + 1] <= row0 + tid) ++seq, ++step;
            for (int left = step == 4 ? a.st.seqs - seq : 0; left > 0;) {
                const int half = left >> 1;
                if (a.st.cu_new[seq + half + 1] <= row0 + tid) seq += half + 1, left -= half + 1;
                else left = half;
            }
            places[tid] = is_padding(a, row0 + tid, seq) ? RowPlace{-2, 0} : place_of(a, row0 + tid, seq);
        }
    }
    __syncthreads();
    const int total = n * (int)items.d;
    constexpr int U = 2;
    for (int i0 = tid; i0 < total; i0 += 256 * U) {
        Item<T, TT, W, HN> it[U];
        RowPlace to[U];
        int row[U];
        bool live[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 256 * u;
            live[u] = i < total;
            if (!live[u]) continue;
            const int r = (int)fdiv((uint32_t)i, items);
            row[u] = row0 + r;
            to[u] = places[r];
            live[u] = to[u].slot != -2 && it[u].load(a, row[u], i - r * (int)items.d);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (live[u]) it[u].store(a, row[u], to[u]);
    }
}

template <typename T, typename TT, int W, int HN> static int launch_append_hn(const AppendArgs& a, hipStream_t st) {
    const int items = (a.nq + 2 * a.kv.heads) * (HN / (2 * W));
    // One row a block leaves lanes idle where its items are few, or a little over 256; then several rows share one, once that leaves
    // 4 blocks a CU.  bf16, us with 1 / 2 / 8 rows a block (the kept one in brackets; 8 from 8192 rows on), at 4096, 8192 and
    // 32768 rows:
    //   72 items (16 / 1 of 64; 38 MB at 8192 rows): [8.5] / 7.9 / 8.5, 13.9 / 13.4 / [10.6], 42.4 / 40.8 / [29.0]
    //   96 items (16 / 4 of 64; 51 MB at 8192 rows): [8.7] / 8.4 / 8.7, 14.5 / 14.6 / [12.5], 43.1 / 42.4 / [35.5]
    //   112 items (24 / 2 of 64; 59 MB at 8192 rows): [9.1] / 9.0 / 9.1, [15.0] / 16.3 / 14.7, [44.6] / 45.6 / 40.2
    //   144 items (32 / 2 of 64; 76 MB at 8192 rows): [10.2] / 10.9 / 10.2, [16.7] / 19.0 / 17.4, [72.8] / 82.1 / 68.6
    //   160 items (32 / 4 of 64; 84 MB at 8192 rows): [10.6] / 11.5 / 10.7, [17.2] / 19.6 / 18.3, [75.5] / 85.1 / 76.4
    //   192 items (16 / 16 of 64; 101 MB at 8192 rows): [11.4] / 13.0 / 11.5, [18.4] / 21.0 / 19.8, [86.7] / 96.0 / 91.3
    //   224 items (24 / 2 of 128; 118 MB at 8192 rows): [13.3] / 14.9 / 13.3, [22.2] / 24.8 / 23.1, [91.2] / 101.9 / 104.1
    //   256 items (24 / 4 of 128; 135 MB at 8192 rows): [15.0] / 16.9 / 14.8, [24.8] / 28.6 / 26.1, [100.9] / 113.0 / 117.9
    //   288 items (32 / 2 of 128; 152 MB at 8192 rows): 21.1 / [18.2] / 21.1, 37.0 / [29.2] / 28.2, 159.5 / [131.3] / 130.9
    //   384 items (32 / 8 of 128; 202 MB at 8192 rows): 22.1 / [21.0] / 22.0, 39.0 / [35.6] / 35.4, 170.2 / [159.5] / 171.4
    //   768 items (32 / 32 of 128; 404 MB at 8192 rows): [33.0] / 36.0 / 33.2, [75.9] / 88.3 / 89.5
    // (Data below 256 MB may come from the Infinity Cache: the calls timed repeat on the same rows.)  Between 97 and 256 items 8 rows a
    // block win by up to 10 % at 32768 rows of 112 and 144 items and lose as much from 192 on or at 8192 rows.  The narrow path is
    // short of loads in flight: 1536 items of 64 with 20 rotated dims 61 -> 44.6.
    const int per = items <= 96 ? 8 : W == 1 || (items > 256 && items <= 384) ? 2 : 1;
    const bool shared = per > 1 && a.rows / per >= 1024;
    const int parts = shared ? 1 : (items + 255) / 256;
    const int64_t blocks = shared ? ((int64_t)a.rows + per - 1) / per : (int64_t)parts * a.rows;
    MM_CHECK_ARG(blocks < (int64_t)1 << 24, "mm_paged_kv_append: %d rows of %d items exceed the grid limit", a.rows, items);
    if (a.nq) {  // items of a row are moved by different lanes, rows by different workgroups: in place, or apart
        const auto runs = [&](const void* p, int64_t row, int64_t head, int heads) { return Runs{p, 2 * row, 2 * head, 2 * HN, a.rows, heads}; };
        const Runs out = runs(a.q_out, a.qo_row, a.qo_head, a.nq), q = runs(a.q, a.q_row, a.q_head, a.nq);
        MM_CHECK_ARG(!overlaps_itself(out), "mm_paged_kv_append: q_out overlaps itself");
        MM_CHECK_ARG(out.same(q) || !overlap(out, q), "mm_paged_kv_append: q_out overlaps q in part");
        MM_CHECK_ARG(!overlap(out, runs(a.k, a.k_row, a.k_head, a.kv.heads)) && !overlap(out, runs(a.v, a.v_row, a.v_head, a.kv.heads)),
                     "mm_paged_kv_append: q_out overlaps k or v");
    }
    if (shared) paged_kv_append_rows_k<T, TT, W, HN><<<(unsigned)blocks, 256, 0, st>>>(a, per, make_fastdiv(items));
    else paged_kv_append_k<T, TT, W, HN><<<(unsigned)blocks, 256, 0, st>>>(a, parts);
    MM_CHECK_LAUNCH();
    return MM_OK;
}
template <typename T, typename TT, int W> static int launch_append(const AppendArgs& a, hipStream_t st) {
    return a.kv.hn == 64 ? launch_append_hn<T, TT, W, 64>(a, st) : launch_append_hn<T, TT, W, 128>(a, st);
}

}  // namespace mm

using namespace mm;

extern "C" int mm_paged_kv_append(const mm_paged_kv* kv, const mm_paged_step* step, const void* k, int64_t k_row, int64_t k_head,
                                  const void* v, int64_t v_row, int64_t v_head, const void* q, int64_t q_row, int64_t q_head,
                                  void* q_out, int64_t qo_row, int64_t qo_head, int nq, int rows, const void* cos, const void* sin,
                                  int rot_d, int table_rows, int table_fp32, void* stream) {
    const char* fn = "mm_paged_kv_append";
    if (int rc = check_paged(fn, kv, step, rows)) return rc;
    MM_CHECK_ARG(rows == 0 || (k && v), "%s: null pointer", fn);
    if (!q) nq = 0;
    MM_CHECK_ARG(!q || (q_out && nq > 0 && nq < 1 << 20), "%s: queries need q_out and a head count, got %d", fn, nq);
    MM_CHECK_ARG(rot_d >= 0 && rot_d <= kv->hn && rot_d % 2 == 0, "%s: rotary dims %d must be even and at most %d", fn, rot_d, kv->hn);
    MM_CHECK_ARG(rot_d == 0 || (cos && sin && table_rows > 0), "%s: rotation needs cos / sin tables", fn);
    if (rows == 0 || step->seqs == 0) return MM_OK;
    AppendArgs a{*kv, *step, (const u16*)k, (const u16*)v, (const u16*)q, (u16*)q_out, k_row, k_head, v_row, v_head, q_row, q_head,
                 qo_row, qo_head, cos, sin, nq, rows, rot_d, table_rows, make_fastdiv(kv->page_size)};
    bool wide = rot_d % 16 == 0 && aligned16(k) && aligned16(v) && aligned16(q) && aligned16(q_out) && aligned16(cos) && aligned16(sin);
    for (int64_t x : {k_row, k_head, v_row, v_head, q ? q_row : 0, q ? q_head : 0, q ? qo_row : 0, q ? qo_head : 0}) wide = wide && x % 8 == 0;
    hipStream_t st = (hipStream_t)stream;
    return dispatch_dtype(kv->dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (wide) return table_fp32 ? launch_append<T, float, 8>(a, st) : launch_append<T, u16, 8>(a, st);
        return table_fp32 ? launch_append<T, float, 1>(a, st) : launch_append<T, u16, 1>(a, st);
    });
}
