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
// Measured: 4 prompts of 2001 .. 2048 tokens, 32 + 2 x 32 heads of 128: 75.3 us, 399 MB at 5.3 TB/s, what a large copy reaches; 256 rows of one token 4.6 us, one row 2.7 us, the latency of
// sequence -> length -> page -> row.
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

// block b moves items [256 i, 256 i + 256) of row b / parts, i = b % parts (all of one row, so that the sequence search and the
// page look-up are uniform over the block)
template <typename T, typename TT, int W, int HN>
__global__ __launch_bounds__(256) void paged_kv_append_k(const AppendArgs a, int parts) {
    constexpr int IPH = HN / (2 * W);  // items per head
    const int row = blockIdx.x / parts;
    const int seq = find_seq(a.st.cu_new, a.st.seqs, row, threadIdx.x & 63);
    if (seq >= a.st.seqs || a.st.cu_new[seq] > row) return;  // padding: belongs to no sequence
    const int64_t pos64 = (int64_t)a.st.kv_lens[seq] - a.st.cu_new[seq + 1] + row;
    bool ok = pos64 >= 0 && pos64 < (int64_t)a.st.max_pages * a.kv.page_size && (a.rot_d == 0 || pos64 < a.table_rows);
    const int pos = ok ? (int)pos64 : 0;
    const int pi = (int)fdiv((uint32_t)pos, a.page);
    const int page = a.st.block_table[(int64_t)seq * a.st.table_stride + pi];
    ok = ok && page >= 0 && page < a.kv.num_pages;

    const int item = (blockIdx.x - row * parts) * 256 + threadIdx.x;
    const int slot = item / IPH, c = item % IPH;
    const int nkv = a.kv.heads;
    if (slot >= a.nq + 2 * nkv) return;
    const int hc = a.rot_d / (2 * W);  // chunks per half of the rotated dims
    const u16* src;
    u16* dst;
    bool rot = hc > 0;
    if (slot < a.nq) {
        src = a.q + (int64_t)row * a.q_row + (int64_t)slot * a.q_head;
        dst = a.q_out + (int64_t)row * a.qo_row + (int64_t)slot * a.qo_head;
    } else {
        if (!ok) return;  // no place for it
        const bool is_k = slot < a.nq + nkv;
        const int h = slot - a.nq - (is_k ? 0 : nkv);
        const int off = pos - pi * a.kv.page_size;
        rot = rot && is_k;
        src = is_k ? a.k + (int64_t)row * a.k_row + (int64_t)h * a.k_head : a.v + (int64_t)row * a.v_row + (int64_t)h * a.v_head;
        dst = (u16*)(is_k ? a.kv.k : a.kv.v) + (int64_t)page * a.kv.page + (int64_t)h * a.kv.head + (int64_t)off * a.kv.slot;
    }
    rot = rot && c < hc;
    // the item's two chunks: partners in the rotated part; behind it (everywhere for an unrotated row) neighbours
    const int c1 = rot ? c : 2 * c, c2 = rot ? c + hc : 2 * c + 1;
    float x1[W], x2[W];
    load_chunk<T, W>(src + c1 * W, x1);
    load_chunk<T, W>(src + c2 * W, x2);
    if (rot) {
        float k1[W], k2[W], s1[W], s2[W];
        const TT* ct = (const TT*)a.cos + (int64_t)pos * a.rot_d;
        const TT* st = (const TT*)a.sin + (int64_t)pos * a.rot_d;
        if constexpr (sizeof(TT) == 4) {
            load_chunk_f32<W>(ct + c1 * W, k1), load_chunk_f32<W>(ct + c2 * W, k2);
            load_chunk_f32<W>(st + c1 * W, s1), load_chunk_f32<W>(st + c2 * W, s2);
        } else {
            load_chunk<T, W>(ct + c1 * W, k1), load_chunk<T, W>(ct + c2 * W, k2);
            load_chunk<T, W>(st + c1 * W, s1), load_chunk<T, W>(st + c2 * W, s2);
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const float y1 = x1[j] * k1[j] - x2[j] * s1[j], y2 = x2[j] * k2[j] + x1[j] * s2[j];
            x1[j] = y1;
            x2[j] = y2;
        }
    }
    if (!ok)  // only queries come here: a row without a place must not pass for a number
#pragma unroll
        for (int j = 0; j < W; ++j) x1[j] = x2[j] = __builtin_nanf("");
    store_chunk<T, W>(dst + c1 * W, x1);
    store_chunk<T, W>(dst + c2 * W, x2);
}

template <typename T, typename TT, int W> static int launch_append(const AppendArgs& a, hipStream_t st) {
    const int items = (a.nq + 2 * a.kv.heads) * (a.kv.hn / (2 * W));
    const int parts = (items + 255) / 256;
    MM_CHECK_ARG((int64_t)parts * a.rows < (int64_t)1 << 24, "mm_paged_kv_append: %d rows of %d items exceed the grid limit", a.rows, items);
    if (a.kv.hn == 64) paged_kv_append_k<T, TT, W, 64><<<parts * a.rows, 256, 0, st>>>(a, parts);
    else paged_kv_append_k<T, TT, W, 128><<<parts * a.rows, 256, 0, st>>>(a, parts);
    MM_CHECK_LAUNCH();
    return MM_OK;
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
