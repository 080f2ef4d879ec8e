// paged_attention.hip - attention of a step's new tokens over a paged key / value cache, for gfx950.
//
// Row j of a sequence that brings n rows and has len tokens afterwards sits at position p = len - n + j and sees keys 0 .. p:
// out = softmax(scale q k^T) v, lse = ln sum exp(scale q k^T) (reference: ParallelSelfAttention.attention with layer_past,
// megatron/model/transformer.py:315-416, 602-610).  The group = nq / heads query heads of one key head and the n new tokens
// together are the "rows" of one (sequence, key head): row r = token r / group, query head kh * group + r % group, so that a
// key or value tile is read once for all of them.
//
// Softmax runs in the exp2 domain with fp32 statistics in one pass over the keys; products accumulate in fp32; the
// probabilities (at most 2^kLag, see there) are rounded to the cache's dtype for the matrix instruction of P V and the row sum takes
// them unrounded.  The few-row form, whose matrix unit is idle, takes what that rounding leaves over in a second instruction, so
// that nothing is lost: bf16 outputs are 0.0017 (relative, over all elements) from the definition, which is their own rounding.  The
// many-row form does not, as the training forward does not: 0.0021 (prompts at head size 64) and 0.0023 (a chunk at 128), fp16 0.00029
// against 0.00021.  With the second instruction its outputs were as near as the few-row form's, at a fifth to a third more time (4 x
// 2048 tokens, 16 heads of 64: 64.7 -> 78.5 us; 1024 over 17k, 32 / 8 heads of 128: 301 -> 401; 12 sequences, 18 heads of 128: 60.9 ->
// 77.1).  Which form a sequence takes follows from its rows per key head (kFewRows) alone, never from what else is in the step.
//
// Masked places never matter: a score behind a row's position is replaced by -inf (not added to), value rows behind the
// sequence's end are zeroed on their way into LDS, and where a tile holds keys that some of its rows do not see, infinities and
// NaN in the values are taken out of the matrix product (0 * inf would spread them to those rows) and added at the end to
// the rows that do see them: p * v is +-inf or NaN whatever p > 0 is.  Tiles that all rows see go unchecked; if an output is not
// finite at the end, the keys are gone through once more with every tile checked, because there p may have rounded to 0.
#include "common.h"
#include "mfma32.h"
#include "attn_common.h"
#include "paged.h"

namespace mm {

struct PagedAttnArgs {
    mm_paged_kv kv;
    mm_paged_step st;
    const u16* q;
    u16* out;
    float* lse;
    int64_t q_row, q_head, o_row, o_head, l_row;
    int nq, group, rows;
    float scale_log2e;
    FastDiv page, grp;
    int few_chunk, few_splits, many_chunk, many_splits;  // keys per split (a multiple of the tiles) and splits, by kind of sequence
    // More than one split: unnormalised outputs [splits, .., hn] and (max, sum) [splits, .., 2] of [seqs, heads, few_rows] in the few-row
    // form and of [rows, nq] in the other, so that a long chunk beside single tokens is not kept once a split of theirs.
    int few_rows;
    float *few_o, *few_ml, *many_o, *many_ml;
};

// How far a score may exceed the running reference of a row's exponentials (in powers of two) before the row is rescaled
constexpr float kLag = 8.f;

constexpr int kFewRows = 16;  // sequences with at most so many rows per key head take the few-row form

// {first row, new rows, length} of a sequence; false: nothing to do
struct SeqInfo {
    int beg, n, len;
};
// A sequence that breaks the step's bounds has its rows set to NaN (by the workgroups with writer set) and is skipped.
template <int HD>
__device__ __forceinline__ bool seq_info(const PagedAttnArgs& a, int seq, int kh, bool writer, SeqInfo& s) {
    s.beg = a.st.cu_new[seq];
    const int end = a.st.cu_new[seq + 1];
    s.len = max(a.st.kv_lens[seq], 0);
    if (end <= s.beg) return false;
    if (s.beg >= 0 && end <= a.rows && end - s.beg <= a.st.max_new && s.len <= a.st.max_kv &&
        s.len <= a.st.max_pages * (int)a.page.d) {
        s.n = end - s.beg;
        return true;
    }
    if (writer) {
        const int b = s.beg < 0 ? 0 : s.beg, e = end < a.rows ? end : a.rows;
        const float nan = __builtin_nanf("");
        for (int64_t i = threadIdx.x; i < (int64_t)(e - b) * a.group * HD; i += blockDim.x) {
            const int row = b + (int)(i / (a.group * HD)), x = (int)(i % (a.group * HD)), h = kh * a.group + x / HD;
            a.out[(int64_t)row * a.o_row + (int64_t)h * a.o_head + x % HD] = 0x7fff;  // a NaN in both 16-bit types
            if (x % HD == 0) a.lse[(int64_t)row * a.l_row + h] = nan;
        }
    }
    return false;
}

__device__ __forceinline__ uint32_t nonfinite2(uint32_t v, uint32_t expm) {  // mask 0xffff per 16-bit value whose exponent is all ones
    return ((v & expm) == expm ? 0xffffu : 0u) | (((v >> 16) & expm) == expm ? 0xffff0000u : 0u);
}
template <typename T> constexpr uint32_t exp_mask();
template <> constexpr uint32_t exp_mask<BF16>() { return 0x7f80u; }
template <> constexpr uint32_t exp_mask<F16>() { return 0x7c00u; }
// takes infinities and NaN out of a 16-byte chunk; true if there were any
template <typename T> __device__ __forceinline__ bool take_nonfinite(u32x4& v) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t m = nonfinite2(v[i], exp_mask<T>());
        v[i] &= ~m;
        any |= m;
    }
    return any != 0;
}
__device__ __forceinline__ uint32_t scalar(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
// the infinity or NaN at p, else 0
template <typename T> __device__ __forceinline__ float only_nonfinite(const u16* __restrict__ p) {
    const u16 v = *p;
    return (v & exp_mask<T>()) == exp_mask<T>() ? to_f32<T>(v) : 0.f;
}
__device__ __forceinline__ bool nonfinite(float x) { return !(x - x == 0.f); }
// w * x where w stands for a positive weight that may have become 0
__device__ __forceinline__ float weigh(float w, float x) { return w != 0.f ? w * x : nonfinite(x) ? x : 0.f; }
// the same of a sum of weights: a NaN stays
__device__ __forceinline__ float weigh_sum(float w, float l) { return w == 0.f && l == l ? 0.f : w * l; }
// add(key, its value row) for the keys of [k0, k1) whose value rows hold infinities or NaN; a whole wave calls it
template <typename T, int HD, typename F>
__device__ __forceinline__ void each_nonfinite(const PagedAttnArgs& a, const int32_t* __restrict__ bt, int kh, int k0, int k1, F&& add) {
    constexpr int CPR = HD / 8, KEYS = 64 / CPR;  // lanes a key, keys a step
    const int lane = threadIdx.x & 63;
    auto row_of = [&](int key) -> const u16* {  // NULL: its page does not exist
        const int pi = (int)fdiv((uint32_t)key, a.page), pg = bt[pi];
        if ((uint32_t)pg >= (uint32_t)a.kv.num_pages) return nullptr;
        return (const u16*)a.kv.v + (int64_t)pg * a.kv.page + (int64_t)kh * a.kv.head + (int64_t)(key - pi * (int)a.page.d) * a.kv.slot;
    };
    for (int base = k0; base < k1; base += KEYS) {
        bool any = false;
        if (base + lane / CPR < k1) {
            const u16* vp = row_of(base + lane / CPR);
            if (vp) {
                u32x4 v = *reinterpret_cast<const u32x4*>(vp + 8 * (lane % CPR));
                any = take_nonfinite<T>(v);
            }
        }
        const uint64_t b = __ballot(any);
        for (int i = 0; i < KEYS && b; ++i)
            if ((b >> (CPR * i)) & ((1ull << CPR) - 1)) add(base + i, row_of(base + i));
    }
}

template <typename T> struct M16;
template <> struct M16<BF16> {
    typedef bf16x8 frag;
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct M16<F16> {
    typedef f16x8 frag;
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// =====================================================================================  few rows: at most 16 per (sequence, key head)
// Bound by the cache's bytes.  A wave works alone on 32-key tiles (the NW waves of a workgroup take them in turn, a grid
// dimension splits long sequences further) and keeps a tile of keys and values in flight in registers:
//   S^T[key][row] = K Q^T: mfma 16x16x32, the keys straight from global memory as the A operand (lane = key, 16 bytes of dims);
//   softmax over the keys of a column: 8 registers and the four 16-lane groups;
//   O^T[dim][row] += V^T P^T: P^T is S^T's registers as they stand - register j of sub-tile t in group g is key 16 t + 4 g + j,
//   and the V^T operand takes its keys in that order - V through a wave-private LDS tile, read transposed (ds_read_b64_tr_b16).
// Measured: 64 sequences of 5 .. 2047 keys, 32 heads of 128 in bf16: 198 us, 1.08 GB at 5.5 TB/s; 2 of 99k and 131k, 32 / 4 heads: 97 us
// with the joining, 5.2 TB/s (90 without, 0.51 GB at 5.7); one of 701, 16 heads of 64: 9.5 us, the latency of one workgroup's chain
// of loads.
// The LDS rows are unpadded; the 32-byte units of a row are XOR-ed with the row so that the transposed reads (16 rows, one unit
// each) and the writes (16 rows, two units each) spread evenly over the banks.
template <int HD> __device__ __forceinline__ int v_off(int row, int byte) {
    const int unit = byte >> 5;
    const int swz = HD == 128 ? (row & 7) : ((row >> 1) & 3);
    return row * (HD * 2) + ((unit ^ swz) << 5) + (byte & 31);
}

template <int HD, int NW> constexpr int few_lds() {  // V tiles; then floats of the final exchange; rows' maxima and sums
    return (NW * 32 * HD * 2 > NW * 16 * (HD + 4) * 4 ? NW * 32 * HD * 2 : NW * 16 * (HD + 4) * 4) + 2 * NW * 16 * 4;
}
// The page ids of a wave's first tile: they need nothing but the block table, so their load goes out with those of the sequence's
// rows and length.
template <int NW> struct FewStart {
    PageCursor cur[2];
    int pid[2];
    __device__ __forceinline__ FewStart(const PagedAttnArgs& a, int seq, int split) {
        const int32_t* bt = a.st.block_table + (int64_t)seq * a.st.table_stride;
        set(a, split);
#pragma unroll
        for (int t = 0; t < 2; ++t) pid[t] = bt[min(cur[t].page, (uint32_t)a.st.max_pages - 1)];
    }
    __device__ __forceinline__ void set(const PagedAttnArgs& a, int split) {
        const int key = split * a.few_chunk + (int)scalar(threadIdx.x >> 6) * 32 + (threadIdx.x & 15);
#pragma unroll
        for (int t = 0; t < 2; ++t) cur[t].set((uint32_t)(key + 16 * t), a.page, 2 * (uint32_t)a.kv.slot);
    }
};
template <typename T, int HD, int NW>
__device__ __forceinline__ void paged_attn_few(const PagedAttnArgs& a, char* smem, const SeqInfo& s, int seq, int kh, int split,
                                               FewStart<NW>& start) {
    typedef typename M16<T>::frag frag;
    constexpr int NC = HD / 32;  // 16-byte chunks of a key per lane = k-steps of Q K^T
    constexpr int NDB = HD / 16;
    constexpr int VB = 32 * HD * 2, RS = HD + 4;  // bytes of a wave's V tile; floats per row of the final exchange
    float (*sm_m)[16] = reinterpret_cast<float (*)[16]>(smem + few_lds<HD, NW>() - 2 * NW * 16 * 4);
    float (*sm_l)[16] = sm_m + NW;
    const int tid = threadIdx.x, wave = (int)scalar(tid >> 6), lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int R = s.n * a.group;
    const int c0 = split * a.few_chunk, c1 = min(c0 + a.few_chunk, s.len);
    if (split > 0 && c0 >= s.len) return;  // the joining kernel knows

    const int rc = r < R ? r : R - 1;
    const int tok = (int)fdiv((uint32_t)rc, a.grp), qh = kh * a.group + rc - tok * a.group;
    const int limit = s.len - s.n + tok, min_limit = s.len - s.n;
    const u16* qp = a.q + (int64_t)(s.beg + tok) * a.q_row + (int64_t)qh * a.q_head;
    frag qf[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) qf[i] = *reinterpret_cast<const frag*>(qp + 32 * i + 8 * g);

    const int32_t* bt = a.st.block_table + (int64_t)seq * a.st.table_stride;
    const char* kb = (const char*)((const u16*)a.kv.k + (int64_t)kh * a.kv.head + 8 * g);
    const int64_t k_to_v = (const char*)a.kv.v - (const char*)a.kv.k;
    const uint32_t page_stride = 2 * (uint32_t)a.kv.page, slot_bytes = 2 * (uint32_t)a.kv.slot, page_bytes = slot_bytes * a.page.d;
    const PageStep stride = page_step(NW * 32, a.page, slot_bytes);
    // Behind a sequence's end its table may hold anything: the keys there are fetched from a page that exists and masked.
    const uint32_t last_page = (uint32_t)a.st.max_pages - 1;

    u32x4 kr[2][NC], vr[2][NC];
    PageCursor (&cur)[2] = start.cur;
    int (&pid)[2] = start.pid;
    uint32_t at[2];    // bytes from the page's start to this lane's key of sub-tile t
    uint32_t bad = 0;  // bit t: it is in a page the cache does not have
    auto move_on = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            at[t] = cur[t].byte;
            cur[t].move(stride, page_bytes);
        }
    };
    auto fetch_pid = [&]() __attribute__((always_inline)) {  // page ids of the cursor's keys; the cursor moves on to the next tile
#pragma unroll
        for (int t = 0; t < 2; ++t) pid[t] = bt[min(cur[t].page, last_page)];
        move_on();
    };
    auto fetch = [&]() __attribute__((always_inline)) {  // keys and values of the tile whose page ids are here
        bad = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const bool b = (uint32_t)pid[t] >= (uint32_t)a.kv.num_pages;
            bad |= b ? 1u << t : 0u;
            const char* kp = kb + (uint64_t)(b ? 0u : (uint32_t)pid[t]) * page_stride + at[t];
            const char* vp = kp + k_to_v;
#pragma unroll
            for (int i = 0; i < NC; ++i) kr[t][i] = *reinterpret_cast<const u32x4*>(kp + 64 * i);
#pragma unroll
            for (int i = 0; i < NC; ++i) vr[t][i] = *reinterpret_cast<const u32x4*>(vp + 64 * i);
        }
    };

    f32x4 o[NDB];
    float m_run, l_run;
    char* vs = smem + wave * VB;
    const int kt0 = c0 + wave * 32;
    bool taken = false;  // values that are not finite have been taken out of the products
    for (bool check_all = false;; check_all = true) {
#pragma unroll
    for (int d = 0; d < NDB; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_run = -INFINITY, l_run = 0.f;
    if (kt0 < c1) {
        move_on();
        fetch();
        fetch_pid();
    }
    for (int kt = kt0; kt < c1; kt += NW * 32) {
        // the tile's values into LDS, its keys into the matrix unit; then its registers take the next tile
        const bool part = check_all || kt + 31 > min_limit;  // some row does not see all of it (wave-uniform)
        const uint64_t badk[2] = {__ballot(bad & 1), __ballot(bad & 2)};
        if (part) {
            bool any = false;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    if (kt + 16 * t + r >= s.len) vr[t][i] = u32x4{0, 0, 0, 0};
                    any |= take_nonfinite<T>(vr[t][i]);
                }
            taken |= __any(any);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < NC; ++i) *reinterpret_cast<u32x4*>(vs + v_off<HD>(16 * t + r, 64 * i + 16 * g)) = vr[t][i];
        f32x4 sc[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < NC; ++i) sc[t] = M16<T>::run(__builtin_bit_cast(frag, kr[t][i]), qf[i], sc[t]);
        }
        if (kt + NW * 32 < c1) {
            fetch();
            fetch_pid();
        }
        if (badk[0] | badk[1]) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if ((badk[t] >> (4 * g + j)) & 1) sc[t][j] = __builtin_nanf("");
        }
        if (part) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (kt + 16 * t + 4 * g + j > limit) sc[t][j] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])), fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = half_max(mx);
        const float m_tile = mx * a.scale_log2e;
        if (__any(m_tile > m_run + kLag)) {
            const float m_new = fmaxf(m_run, m_tile);
            const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
            l_run *= alpha;
#pragma unroll
            for (int d = 0; d < NDB; ++d) o[d] *= alpha;
            m_run = m_new;
        }
        const float m_use = m_run == -INFINITY ? 0.f : m_run;  // no key seen yet: every p is exp2(-inf) = 0
        float p[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                p[t][j] = fast_exp2(sc[t][j] * a.scale_log2e - m_use);
                l_run += p[t][j];
            }
        // The matrix unit takes probabilities in the cache's 16 bits.  It is idle most of the time here, so it takes what their
        // rounding leaves over as well: the output is then good to its own rounding (relative error of bf16 outputs 0.0022 -> 0.0017).
        u32x4 pw, pr;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a0 = p[i >> 1][2 * (i & 1)], a1 = p[i >> 1][2 * (i & 1) + 1];
            pw[i] = pack2<T>(a0, a1);
            pr[i] = pack2<T>(a0 - to_f32<T>((u16)(pw[i] & 0xffffu)), a1 - to_f32<T>((u16)(pw[i] >> 16)));
        }
        const frag pf = __builtin_bit_cast(frag, pw), pfr = __builtin_bit_cast(frag, pr);
        // V^T operand: lane (dim r of block d, group g) takes keys 4 g .. 4 g + 3 of both sub-tiles
#pragma unroll
        for (int d = 0; d < NDB; ++d) {
            const int row = 4 * g + (r >> 2), byte = 32 * d + 8 * (r & 3);
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vs + v_off<HD>(row, byte)));
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vs + v_off<HD>(row + 16, byte)));
            const s16x8 v = s16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            o[d] = M16<T>::run(__builtin_bit_cast(frag, v), pfr, M16<T>::run(__builtin_bit_cast(frag, v), pf, o[d]));
        }
    }
    float bad_out = 0.f;  // NaN if an output is not finite
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) bad_out = fmaf(o[d][j], 0.f, bad_out);
    if (check_all || !__any(bad_out != bad_out)) break;
    start.set(a, split);
#pragma unroll
    for (int t = 0; t < 2; ++t) pid[t] = bt[min(cur[t].page, last_page)];
    }
    if (taken) {
        for (int kt = kt0; kt < c1; kt += NW * 32)
            each_nonfinite<T, HD>(a, bt, kh, kt, min(kt + 32, c1), [&](int key, const u16* vp) {
                if (key > limit) return;
#pragma unroll
                for (int d = 0; d < NDB; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[d][j] += only_nonfinite<T>(vp + 16 * d + 4 * g + j);
            });
    }

    // join the waves: rows' maxima and sums, then the weighted outputs
    l_run += __shfl_xor(l_run, 16, 64);
    l_run = half_sum(l_run);
    __syncthreads();  // every wave has read its V tile
    float* red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int d = 0; d < NDB; ++d) *reinterpret_cast<f32x4*>(red + (wave * 16 + r) * RS + 16 * d + 4 * g) = o[d];
    if (g == 0) {
        sm_m[wave][r] = m_run;
        sm_l[wave][r] = l_run;
    }
    __syncthreads();
    for (int i = tid; i < R * (HD / 8); i += NW * 64) {
        const int row = i / (HD / 8), d0 = (i % (HD / 8)) * 8;
        float M = -INFINITY, L = 0.f, acc[8];
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sm_m[w][row]);
        const float mu = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {  // a wave without a key has the maximum -inf and zeros
            const float al = fast_exp2(sm_m[w][row] - mu);
            L += weigh_sum(al, sm_l[w][row]);
            const float* src = red + (w * 16 + row) * RS + d0;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += weigh(al, src[e]);
        }
        const int t = (int)fdiv((uint32_t)row, a.grp), h = kh * a.group + row - t * a.group, grow = s.beg + t;
        if (a.few_splits == 1) {
            const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] *= inv;
            *reinterpret_cast<u32x4*>(a.out + (int64_t)grow * a.o_row + (int64_t)h * a.o_head + d0) = pack8<T>(acc);
            if (d0 == 0) a.lse[(int64_t)grow * a.l_row + h] = (M + __log2f(L)) * kLn2;
        } else {
            const int64_t at = (((int64_t)split * a.st.seqs + seq) * a.kv.heads + kh) * a.few_rows + row;
            f32x4* dst = reinterpret_cast<f32x4*>(a.few_o + at * HD + d0);
            dst[0] = f32x4{acc[0], acc[1], acc[2], acc[3]};
            dst[1] = f32x4{acc[4], acc[5], acc[6], acc[7]};
            if (d0 == 0) {
                a.few_ml[2 * at] = M;
                a.few_ml[2 * at + 1] = L;
            }
        }
    }
}

// =====================================================================================  many rows
// Bound by the matrix unit and the softmax's vector work, as the training forward (attention.hip), whose tile walk it shares: a
// wave owns 32 rows on the lane index of mfma 32x32x16 score tiles; keys and values come in 64-key tiles, global -> registers ->
// double-buffered LDS, one barrier a tile; page ids are fetched a tile further ahead, so that no load waits for another.  Row
// blocks with the most keys start first.
// Measured: 1024 tokens over 17k, 32 / 8 heads of 128: 282 us with the joining, 980 TFLOP/s; 4 x 2048 tokens, 16 heads of 64: 57
// us, 600 TFLOP/s of what the causal mask leaves (on other boards, or after many calls without a pause, up to 301 and 65).  The
// occupancy bounds leave 7 registers spilled, written ahead of the tile loops and read behind them or once a pass, never inside.  A
// wave's 64-key tile at 128 takes 4070 cycles beside a second wave on its SIMD: 1024 of matrix instructions, about 900 of softmax,
// 350 .. 550 each for issuing the loads and writing LDS, the rest waiting for the other wave, whose matrix instructions hold the
// vector unit up (8 cycles each) and the other way round.  The clock falls with the work per cycle (1.88 GHz here, 1.73 at head
// size 64; a schedule of 4440 cycles a tile ran at 2.03).
// LDS rows are unpadded; the 16-byte chunks of a row are XOR-ed with the row so that the row reads (16 rows, one chunk) and the
// transposed reads (4 rows, 4 chunks) both meet all banks once.
template <int HD> struct KvTile {
    static constexpr int ROWB = HD * 2, BYTES = 64 * ROWB, CPR = HD / 8;
    static __device__ __forceinline__ int swz(int row) {
        if constexpr (HD == 64) return (((row >> 1) & 1) << 2) | ((row >> 1) & 2) | ((row >> 3) & 1);
        else return ((row & 3) << 2) | ((row >> 2) & 3);
    }
    static __device__ __forceinline__ int off(int row, int chunk) { return row * ROWB + ((chunk ^ swz(row)) << 4); }
};

template <int HD> constexpr int many_lds() { return 4 * KvTile<HD>::BYTES + 48; }
template <typename T, int HD, int NWV>
__device__ __forceinline__ void paged_attn_many(const PagedAttnArgs& a, char* smem, const SeqInfo& s, int seq, int kh, int row_block, int split) {
    typedef KvTile<HD> TL;
    typedef typename M32<T>::frag frag;
    constexpr int NDS = HD / 16, NDB = HD / 32, NT = 64 * NWV, NCH = 64 * TL::CPR / NT, ROWS = 32 * NWV;
    constexpr bool AHEAD = HD == 64 || NWV == 8;
    constexpr int KG = HD == 128 ? 2 : 4;  // key fragments read ahead
    auto fence = []() __attribute__((always_inline)) {
        if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
    };
    // two stages of K | V, then per ring slot (tile & 3) a 64-bit mask of the keys in pages the cache does not have, and whether
    // values that are not finite have been taken out of the products, and whether an output is not finite
    unsigned long long* flags = reinterpret_cast<unsigned long long*>(smem + 4 * TL::BYTES);
    int* taken = reinterpret_cast<int*>(flags + 4);
    int* bad_out = taken + 1;
    const int tid = threadIdx.x, wave = (int)scalar(tid >> 6), lane = tid & 63, r = lane & 31, hh = lane >> 5;
    const int r0 = row_block * ROWS;
    const int R = s.n * a.group;
    if (r0 >= R) return;
    const int c0 = split * a.many_chunk;
    if (split > 0 && c0 >= s.len) return;  // the joining kernel knows

    const int past = s.len - s.n;
    const int row = r0 + wave * 32 + r, rc = row < R ? row : R - 1;
    const int tok = (int)fdiv((uint32_t)rc, a.grp), qh = kh * a.group + rc - tok * a.group;
    const int limit = past + tok;
    const u16* qp = a.q + (int64_t)(s.beg + tok) * a.q_row + (int64_t)qh * a.q_head;
    frag qf[NDS];
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) qf[ds] = *reinterpret_cast<const frag*>(qp + 16 * ds + 8 * hh);

    const int wr0 = r0 + wave * 32;
    const int blk_first = past + (int)fdiv((uint32_t)r0, a.grp);
    const int blk_last = past + (int)fdiv((uint32_t)min(r0 + ROWS - 1, R - 1), a.grp);
    const int wave_first = past + (int)fdiv((uint32_t)min(wr0, R - 1), a.grp);
    const int wave_last = wr0 < R ? past + (int)fdiv((uint32_t)min(wr0 + 31, R - 1), a.grp) : -1;
    const int c1 = min(c0 + a.many_chunk, blk_last + 1);
    const int ntiles = c1 > c0 ? (c1 - c0 + 63) >> 6 : 0;

    const int32_t* bt = a.st.block_table + (int64_t)seq * a.st.table_stride;
    const int trow = tid / TL::CPR, tch = tid % TL::CPR;  // this thread's first row and its 16-byte chunk of a tile
    constexpr int RSTEP = NT / TL::CPR;
    const int st0 = TL::off(trow, tch);  // RSTEP is a multiple of 16 rows: the swizzle of all the thread's rows is the same
    const char* kb = (const char*)((const u16*)a.kv.k + (int64_t)kh * a.kv.head + tch * 8);
    const int64_t k_to_v = (const char*)a.kv.v - (const char*)a.kv.k;
    const uint32_t page_stride = 2 * (uint32_t)a.kv.page, slot_bytes = 2 * (uint32_t)a.kv.slot, page_bytes = slot_bytes * a.page.d;
    const PageStep stride = page_step(64, a.page, slot_bytes);
    const uint32_t last_page = s.len > 0 ? fdiv((uint32_t)s.len - 1, a.page) : 0;  // behind it the table is not the sequence's
    u32x4 kreg[NCH], vreg[NCH];
    PageCursor pos[NCH];
    int pid[NCH];
    uint32_t at[NCH];
    uint32_t bad = 0;
    auto fetch_pid = [&]() __attribute__((always_inline)) {  // page ids of the cursor's keys; the cursor moves on to the next tile
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            pid[i] = bt[min(pos[i].page, last_page)];
            at[i] = pos[i].byte;
            pos[i].move(stride, page_bytes);
        }
    };
    auto fetch = [&]() __attribute__((always_inline)) {  // keys and values of the tile whose page ids are here
        bad = 0;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const bool b = (uint32_t)pid[i] >= (uint32_t)a.kv.num_pages;
            bad |= b ? 1u << i : 0u;
            const char* kp = kb + (uint64_t)(b ? 0u : (uint32_t)pid[i]) * page_stride + at[i];
            kreg[i] = *reinterpret_cast<const u32x4*>(kp);
            vreg[i] = *reinterpret_cast<const u32x4*>(kp + k_to_v);
        }
    };
    bool check_all = false;
    // registers -> LDS stage of tile j; where some row of the block does not see the whole tile, the values behind the end become
    // zero and the non-finite ones are taken out
    auto put = [&](char* ks, int j) __attribute__((always_inline)) {
        const int kv0 = c0 + j * 64;
        if (check_all || kv0 + 63 > blk_first) {
            bool any = false;
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int key = trow + RSTEP * i;
                if (kv0 + key >= s.len) vreg[i] = u32x4{0, 0, 0, 0};
                any |= take_nonfinite<T>(vreg[i]);
            }
            if (any) *taken = 1;
        }
        if (__ballot(bad != 0)) {
#pragma unroll
            for (int i = 0; i < NCH; ++i)
                if ((bad >> i) & 1) atomicOr(flags + (j & 3), 1ull << (trow + RSTEP * i));
        }
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            *reinterpret_cast<u32x4*>(ks + st0 + i * RSTEP * TL::ROWB) = kreg[i];
            *reinterpret_cast<u32x4*>(ks + TL::BYTES + st0 + i * RSTEP * TL::ROWB) = vreg[i];
        }
    };

    f32x16 o[NDB];
    float m_run, l_run;
    // this lane's fragments: row reads of K (chunk 2 ds + hh of row r), transposed reads of V (as tr_frag in mfma32.h)
    const int ka0 = TL::off(r, hh);
    const int tg = lane >> 4, tq = (lane & 15) >> 2, tp = lane & 3;
    const int va0 = TL::off(4 * hh + tq, 2 * (tg & 1) + (tp >> 1)) + (tp & 1) * 8;
    auto k_frag = [&](const char* ks, int t, int ds) __attribute__((always_inline)) -> frag { return *reinterpret_cast<const frag*>(ks + ((ka0 ^ (ds << 5)) + t * 32 * TL::ROWB)); };
    auto v_frag = [&](const char* vs, int kb16, int d) __attribute__((always_inline)) -> frag {  // keys kb16 .. kb16 + 15 (a multiple of 16), dims 32 d .. 32 d + 31
        // rows 8 further on flip one bit of the swizzle (row bit 3): bit 1 of the chunk at head size 128, bit 0 at 64
        const char* pa = vs + ((va0 ^ (d << 6)) + kb16 * TL::ROWB);
        const char* pb = vs + ((va0 ^ (d << 6) ^ (HD == 64 ? 16 : 32)) + (kb16 + 8) * TL::ROWB);
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)pa);
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)pb);
        const s16x8 v = s16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        return __builtin_bit_cast(frag, v);
    };
    auto tile_step = [&](const int j, auto parity) __attribute__((always_inline)) {
        constexpr int cur = decltype(parity)::value;
        const char* ks = smem + cur * 2 * TL::BYTES;
        const char* vs = ks + TL::BYTES;
        const int kv0 = c0 + j * 64;
        if (j + 1 < ntiles) {
            fetch();
            fetch_pid();
        }
        if (tid == 0) flags[(j + 2) & 3] = 0;  // read in tile j - 2, written for tile j + 2 behind this tile's barrier
        const u32x2 fl = *reinterpret_cast<const u32x2*>(flags + (j & 3));
        const uint32_t badk[2] = {scalar(fl[0]), scalar(fl[1])};
        if (kv0 <= wave_last) {
            f32x16 sacc[2];
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) sacc[t][i] = 0.f;
            frag kf[2][KG], vf[2][NDB];
            auto load_k = [&](int grp, frag (&f)[KG]) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < KG; ++i) f[i] = k_frag(ks, (grp * KG + i) & 1, (grp * KG + i) >> 1);
                fence();
            };
            auto load_v = [&](int grp, frag (&f)[NDB]) __attribute__((always_inline)) {
#pragma unroll
                for (int d = 0; d < NDB; ++d) f[d] = v_frag(vs, 16 * grp, d);
                fence();
            };
            // Fragments are read from LDS a group ahead of the matrix instructions that take them (the fences keep the compiler from
            // moving the reads back to their use, where each waits out the LDS latency), the first values' behind the softmax: 1024
            // tokens over 17k, 32 / 8 heads of 128: 325 -> 300 us.  In 4 waves of 128 it takes registers that are not there (32 x 100 tokens
            // over 1.8k, 16 heads: 115 -> 123): the compiler's order stays.
            fence();
            load_k(0, kf[0]);
#pragma unroll
            for (int grp = 0; grp < 2 * NDS / KG; ++grp) {
                if (grp + 1 < 2 * NDS / KG) load_k(grp + 1, kf[(grp + 1) & 1]);
                else load_v(0, vf[0]);
#pragma unroll
                for (int i = 0; i < KG; ++i) sacc[(grp * KG + i) & 1] = M32<T>::run(kf[grp & 1][i], qf[(grp * KG + i) >> 1], sacc[(grp * KG + i) & 1]);
                fence();
            }
            __builtin_amdgcn_s_setprio(0);
            if (badk[0] | badk[1]) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint32_t b = badk[t] >> (4 * hh);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if ((b >> acc_row(i, 0)) & 1) sacc[t][i] = __builtin_nanf("");
                }
            }
            if (kv0 + 63 > wave_first) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (kv0 + 32 * t + acc_row(i, hh) > limit) sacc[t][i] = -INFINITY;
            }
            float rmax = fmaxf(sacc[0][0], sacc[1][0]);
#pragma unroll
            for (int i = 1; i < 16; ++i) rmax = fmaxf(fmaxf(rmax, sacc[0][i]), sacc[1][i]);
            rmax = half_max(rmax);
            // The reference value of the exponentials only moves when a score exceeds it by more than kLag: probabilities are then
            // at most 2^kLag, their relative rounding is the same, and most tiles need no rescaling.
            const float m_tile = rmax * a.scale_log2e;
            if (__any(m_tile > m_run + kLag)) {
                const float m_new = fmaxf(m_run, m_tile);
                const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < NDB; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
                m_run = m_new;
            }
            const float m_use = m_run == -INFINITY ? 0.f : m_run;  // no key seen yet: every p is exp2(-inf) = 0
            float lsum = 0.f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    sacc[t][i] = fast_exp2(sacc[t][i] * a.scale_log2e - m_use);
                    lsum += sacc[t][i];
                }
            l_run += lsum;
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    if (2 * t + s2 < 3) load_v(2 * t + s2 + 1, vf[(s2 + 1) & 1]);
                    const frag pf = M32<T>::cvt8(sacc[t][8 * s2], sacc[t][8 * s2 + 1], sacc[t][8 * s2 + 2], sacc[t][8 * s2 + 3],
                                                 sacc[t][8 * s2 + 4], sacc[t][8 * s2 + 5], sacc[t][8 * s2 + 6], sacc[t][8 * s2 + 7]);
#pragma unroll
                    for (int d = 0; d < NDB; ++d) o[d] = M32<T>::run(vf[s2][d], pf, o[d]);
                    fence();
                }
            __builtin_amdgcn_s_setprio(0);
        }
        if (j + 1 < ntiles) put(smem + (cur ^ 1) * 2 * TL::BYTES, j + 1);
        __syncthreads();
    };
    for (;; check_all = true) {
        int first = trow;
        asm volatile("" : "+v"(first));  // computed anew for the second pass, not held in registers through the first
#pragma unroll
        for (int i = 0; i < NDB; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
        m_run = -INFINITY, l_run = 0.f;
        if (tid < 4) flags[tid] = 0;
        if (tid < 2) taken[tid] = 0;
        __syncthreads();
        if (ntiles > 0) {
#pragma unroll
            for (int i = 0; i < NCH; ++i) pos[i].set((uint32_t)(c0 + first + RSTEP * i), a.page, slot_bytes);
            fetch_pid();
            fetch();
            fetch_pid();
            put(smem, 0);
        }
        __syncthreads();
#pragma unroll
        for (int ds = 0; ds < NDS; ++ds) pin(qf[ds]);
        for (int j = 0; j < ntiles; j += 2) {
            tile_step(j, std::integral_constant<int, 0>{});
            if (j + 1 < ntiles) tile_step(j + 1, std::integral_constant<int, 1>{});
        }
        if (check_all) break;
        float b = 0.f;  // NaN if an output is not finite
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) b = fmaf(o[d][i], 0.f, b);
        if (b != b) *bad_out = 1;
        __syncthreads();
        if (!scalar((uint32_t)*bad_out)) break;
        __syncthreads();  // everyone has read it
    }
    if (scalar((uint32_t)*taken))
        each_nonfinite<T, HD>(a, bt, kh, c0, min(c1, wave_last + 1), [&](int key, const u16* vp) {
            if (key > limit) return;
#pragma unroll
            for (int d = 0; d < NDB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] += only_nonfinite<T>(vp + 32 * d + acc_row(i, hh));
        });

    const float l_tot = half_sum(l_run);
    if (row >= R) return;
    const int grow = s.beg + tok;
    if (a.many_splits == 1) {
        const float inv = l_tot == 0.f ? 0.f : 1.0f / l_tot;
        u16* orow = a.out + (int64_t)grow * a.o_row + (int64_t)qh * a.o_head;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4)
                *reinterpret_cast<u32x2*>(orow + 32 * d + 8 * g4 + 4 * hh) =
                    u32x2{pack2<T>(o[d][4 * g4] * inv, o[d][4 * g4 + 1] * inv), pack2<T>(o[d][4 * g4 + 2] * inv, o[d][4 * g4 + 3] * inv)};
        if (hh == 0) a.lse[(int64_t)grow * a.l_row + qh] = (m_run + __log2f(l_tot)) * kLn2;
    } else {
        const int64_t at = ((int64_t)split * a.rows + grow) * a.nq + qh;
        float* orow = a.many_o + at * HD;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4)
                *reinterpret_cast<f32x4*>(orow + 32 * d + 8 * g4 + 4 * hh) = f32x4{o[d][4 * g4], o[d][4 * g4 + 1], o[d][4 * g4 + 2], o[d][4 * g4 + 3]};
        if (hh == 0) {
            a.many_ml[2 * at] = m_run;
            a.many_ml[2 * at + 1] = l_tot;
        }
    }
}

// =====================================================================================  the kernels
// Every sequence has at most kFewRows rows (token steps).  Grid: (sequence, key head), split.
template <typename T, int HD, int NW> __global__ __launch_bounds__(NW * 64) void paged_attn_few_k(const PagedAttnArgs a) {
    __shared__ __attribute__((aligned(16))) char smem[few_lds<HD, NW>()];
    const int seq = blockIdx.x / a.kv.heads, kh = blockIdx.x % a.kv.heads;
    FewStart<NW> start(a, seq, blockIdx.y);
    SeqInfo s;
    if (seq_info<HD>(a, seq, kh, blockIdx.y == 0, s)) paged_attn_few<T, HD, NW>(a, smem, s, seq, kh, blockIdx.y, start);
}
// Any step: each sequence in the form its rows call for, so that single tokens next to a chunk of a prompt run at the cache's
// bandwidth beside it.  Grid: (sequence, key head), then row blocks times splits - the row blocks with the most keys first.
template <typename T, int HD, int NW>
__global__ __launch_bounds__(NW * 64, (HD == 64 ? 3 : 2)) void paged_attn_any_k(const PagedAttnArgs a, int row_blocks) {
    constexpr int LDS = few_lds<HD, NW>() > many_lds<HD>() ? few_lds<HD, NW>() : many_lds<HD>();
    __shared__ __attribute__((aligned(16))) char smem[LDS];
    const int seq = blockIdx.x / a.kv.heads, kh = blockIdx.x % a.kv.heads;
    SeqInfo s;
    if (!seq_info<HD>(a, seq, kh, blockIdx.y == 0, s)) return;
    if (s.n * a.group <= kFewRows) {
        if ((int)blockIdx.y >= a.few_splits) return;
        FewStart<NW> start(a, seq, blockIdx.y);
        paged_attn_few<T, HD, NW>(a, smem, s, seq, kh, blockIdx.y, start);
    } else {
        const int split = blockIdx.y / row_blocks, rb = blockIdx.y % row_blocks;
        if (split < a.many_splits) paged_attn_many<T, HD, NW>(a, smem, s, seq, kh, row_blocks - 1 - rb, split);
    }
}

// =====================================================================================  joining the splits
// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s, always in the same order.  One wave per row and head; its 2 (head size 64: 4)
// groups of lanes take the splits in turn.  Bound by the latency of loads that follow from each other (the results
// come from other XCDs' caches): the first partial results are asked for before it is known which of them exist - all of them have
// their place in the workspace.  32768 rows and heads of 2 splits (1024 tokens, 32 heads of 128): 16 us, 42 MB at 2.6 TB/s; 64 of 32
// splits (2 tokens over 131k keys): 7 us.  (One split after the other behind a pass over the maxima: 23 and 8.7.)
template <typename T, int HD, bool few> __device__ __forceinline__ void join_rows(const PagedAttnArgs& a, int64_t id) {
    constexpr int LANES = HD / 4, GROUPS = 64 / LANES, U = few ? 4 : 1;  // a chunk of a prompt is rarely split more than GROUPS times
    const int lane = threadIdx.x & 63, g = lane / LANES, x = lane % LANES;
    const int64_t step = few ? (int64_t)a.st.seqs * a.kv.heads * a.few_rows : (int64_t)a.rows * a.nq;  // ids, and partial results a split
    if (id >= step) return;
    const int chunk = few ? a.few_chunk : a.many_chunk, splits = few ? a.few_splits : a.many_splits;
    const f32x4* ws_o = reinterpret_cast<const f32x4*>((few ? a.few_o : a.many_o) + id * HD) + x;
    const f32x2* ws_ml = reinterpret_cast<const f32x2*>(few ? a.few_ml : a.many_ml) + id;
    f32x2 ml[U];
    f32x4 v[U];
    auto load = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = min(i0 + u * GROUPS + g, splits - 1) * step;
            ml[u] = ws_ml[i];
            v[u] = ws_o[i * (HD / 4)];
        }
    };
    load(0);

    const int seq = few ? (int)(id / (a.kv.heads * a.few_rows)) : find_seq(a.st.cu_new, a.st.seqs, (int)(id / a.nq), lane);
    if (seq >= a.st.seqs) return;
    const int beg = a.st.cu_new[seq], end = a.st.cu_new[seq + 1], len = a.st.kv_lens[seq];
    // rows that the main kernel has not written or has handled itself (seq_info), and rows of the other form: nothing to join
    if (beg < 0 || end <= beg || end > a.rows || end - beg > a.st.max_new || len > a.st.max_kv || len > a.st.max_pages * (int)a.page.d) return;
    const int R = (end - beg) * a.group;
    if ((R <= kFewRows) != few) return;
    int row, h;
    if (few) {
        const int r = (int)(id % a.few_rows), kh = (int)(id / a.few_rows) % a.kv.heads, tok = (int)fdiv((uint32_t)r, a.grp);
        if (r >= R) return;
        row = beg + tok, h = kh * a.group + r - tok * a.group;
    } else {
        row = (int)(id / a.nq), h = (int)(id % a.nq);
        if (beg > row) return;
    }
    const int ns = len > chunk ? min(splits, (len - 1) / chunk + 1) : 1;
    float M = -INFINITY, L = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0;;) {
        float top = M;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * GROUPS + g < ns) top = fmaxf(top, ml[u][0]);
        const float mu = top == -INFINITY ? 0.f : top, alpha = fast_exp2(M - mu);
        M = top;
        L = weigh_sum(alpha, L);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = weigh(alpha, acc[e]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u * GROUPS + g >= ns) continue;
            const float w = fast_exp2(ml[u][0] - mu);
            L += weigh_sum(w, ml[u][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += weigh(w, v[u][e]);
        }
        i0 += GROUPS * U;
        if (i0 >= ns) break;
        load(i0);
    }
    float top = M;
#pragma unroll
    for (int d = LANES; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
    const float w = fast_exp2(M - (top == -INFINITY ? 0.f : top));
    L = weigh_sum(w, L);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = weigh(w, acc[e]);
#pragma unroll
    for (int d = LANES; d < 64; d *= 2) {
        L += __shfl_xor(L, d, 64);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], d, 64);
    }
    if (g != 0) return;
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    *reinterpret_cast<u32x2*>(a.out + (int64_t)row * a.o_row + (int64_t)h * a.o_head + 4 * x) =
        u32x2{pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv)};
    if (x == 0) a.lse[(int64_t)row * a.l_row + h] = (top + __log2f(L)) * kLn2;
}

// The first few_blocks blocks join the few-row form's [seqs, heads, few_rows], the others the many-row form's [rows, nq].
template <typename T, int HD> __global__ __launch_bounds__(256) void paged_attn_join_k(const PagedAttnArgs a, int few_blocks) {
    const int b = blockIdx.x, wave = threadIdx.x >> 6;
    if (b < few_blocks) join_rows<T, HD, true>(a, (int64_t)b * 4 + wave);
    else join_rows<T, HD, false>(a, (int64_t)(b - few_blocks) * 4 + wave);
}

// ---- launch plan, from the step's bounds alone (a captured step keeps it)
struct PagedPlan {
    bool few;
    int waves, row_blocks, few_chunk, few_splits, many_chunk, many_splits;
    int few_rows;
    // rows of partial results
    int64_t few_partials(const mm_paged_kv& kv, const mm_paged_step& st) const { return few_splits > 1 ? (int64_t)few_splits * st.seqs * kv.heads * few_rows : 0; }
    int64_t many_partials(int rows, int nq) const { return many_splits > 1 ? (int64_t)many_splits * rows * nq : 0; }
    size_t bytes(const mm_paged_kv& kv, const mm_paged_step& st, int rows, int nq) const {
        return (size_t)(few_partials(kv, st) + many_partials(rows, nq)) * (kv.hn + 2) * sizeof(float);
    }
};
// Splits while a launch has too few workgroups: as many as keep one resident set (`target`), none shorter than `least` keys
static void split_keys(int64_t wgs, int64_t target, int64_t least, int64_t gran, int max_kv, int& chunk, int& splits) {
    int64_t ns = wgs > 0 ? target / wgs : 1;
    const int64_t cap = (max_kv + least - 1) / least;
    if (ns > cap) ns = cap;
    if (ns < 1) ns = 1;
    int64_t c = (max_kv + ns - 1) / ns;
    c = (c + gran - 1) / gran * gran;
    if (c < gran) c = gran;
    chunk = (int)c;
    splits = max_kv > 0 ? (int)((max_kv + c - 1) / c) : 1;
}
static PagedPlan plan(const mm_paged_kv& kv, const mm_paged_step& st, int nq) {
    PagedPlan p;
    const int group = nq / kv.heads;
    const int64_t rows = (int64_t)st.max_new * group, pairs = (int64_t)st.seqs * kv.heads;
    p.few = rows <= kFewRows;
    p.few_rows = p.few ? (int)rows : kFewRows;
    // Few rows: one workgroup of 8 waves a CU.  With more, smaller ones the same bytes are in flight in more places at once: 2 x 131071
    // keys of 4 heads of 128: 162 us with 1024 workgroups of 4 waves, 133 with 512, 112 with 256 of 8.  Where the keys and values are
    // few (64 MB), the chain of loads and the waves' exchange count, and 4 waves do it sooner: 100 keys of 16 heads of 64 6.45 -> 5.7 us,
    // 1023 of 32 heads of 128 15.9 -> 15.3, 8191 of 16 heads of 64 13.6 -> 13.1; 65000 of 8 heads of 128, 266 MB, 52.4 -> 54.9.
    // Many rows: 128 a workgroup.  At head size 128 the registers hold two waves a SIMD whatever the workgroup's size, and one of 8
    // waves fetches each tile once for 256 rows: 1024 tokens over 17k, 32 / 8 heads: 337 -> 314 us.  At 64 three waves a SIMD fit,
    // which 8-wave workgroups cannot use: 59 us against 70 (4 x 2048 tokens, 16 heads).
    p.waves = p.few ? (pairs * st.max_kv * kv.hn <= 1 << 24 ? 4 : 8) : kv.hn == 128 && rows > 128 ? 8 : 4;
    p.row_blocks = p.few ? 1 : (int)((rows + 32 * p.waves - 1) / (32 * p.waves));
    // A token step's split pays for its second launch (about 2 us) once a workgroup's keys and values exceed 256 KB (one CU takes in
    // some 130 GB/s): 700 keys of 64 in one piece 9.7 us, in two 11.2; 1023 of 128 in one 19, in two 15; 2047 of 64 in two 15, in
    // four 11.7.  Beside chunks of prompts, whose rows the joining launch passes over too, from four times that.
    p.few_chunk = (st.max_kv + 32 * p.waves - 1) / (32 * p.waves) * (32 * p.waves), p.few_splits = 1;
    if ((int64_t)st.max_kv * kv.hn > (p.few ? 65536 : 262144)) split_keys(pairs, 2048 / p.waves, 512, 32 * p.waves, st.max_kv, p.few_chunk, p.few_splits);
    p.many_chunk = 64, p.many_splits = 1;
    if (!p.few) split_keys(pairs * p.row_blocks, 2048 / p.waves, 512, 64, st.max_kv, p.many_chunk, p.many_splits);
    return p;
}

template <typename T, int HD> static int launch_paged_attn(const PagedAttnArgs& a, const PagedPlan& p, hipStream_t st) {
    const Runs out = {a.out, 2 * a.o_row, 2 * a.o_head, 2 * HD, a.rows, a.nq}, q = {a.q, 2 * a.q_row, 2 * a.q_head, 2 * HD, a.rows, a.nq};
    const Runs lse = {a.lse, 4 * a.l_row, 0, 4 * (int64_t)a.nq, a.rows, 1};
    MM_CHECK_ARG(!overlaps_itself(out) && !overlaps_itself(lse), "mm_paged_attn_fwd: out or lse overlaps itself");
    // a workgroup has read its rows' queries before it, or the joining launch, writes their outputs
    MM_CHECK_ARG(out.same(q) || !overlap(out, q), "mm_paged_attn_fwd: out overlaps q in part");
    MM_CHECK_ARG(!overlap(lse, q) && !overlap(lse, out), "mm_paged_attn_fwd: lse overlaps q or out");
    const unsigned bx = (unsigned)(a.st.seqs * a.kv.heads);
    const int many = p.row_blocks * p.many_splits;
    const dim3 grid(bx, p.few ? p.few_splits : (p.few_splits > many ? p.few_splits : many));
    if (p.few && p.waves == 4) paged_attn_few_k<T, HD, 4><<<grid, 256, 0, st>>>(a);
    else if (p.few) paged_attn_few_k<T, HD, 8><<<grid, 512, 0, st>>>(a);
    else if constexpr (HD == 128) {
        if (p.waves == 8) paged_attn_any_k<T, 128, 8><<<grid, 512, 0, st>>>(a, p.row_blocks);
        else paged_attn_any_k<T, 128, 4><<<grid, 256, 0, st>>>(a, p.row_blocks);
    } else paged_attn_any_k<T, 64, 4><<<grid, 256, 0, st>>>(a, p.row_blocks);
    MM_CHECK_LAUNCH();
    if (p.few_splits > 1 || p.many_splits > 1) {
        const int64_t few_blocks = p.few_splits > 1 ? ((int64_t)bx * p.few_rows + 3) / 4 : 0;
        const int64_t many_blocks = p.many_splits > 1 ? ((int64_t)a.rows * a.nq + 3) / 4 : 0;
        paged_attn_join_k<T, HD><<<(unsigned)(few_blocks + many_blocks), 256, 0, st>>>(a, (int)few_blocks);
        MM_CHECK_LAUNCH();
    }
    return MM_OK;
}

static int check_paged_attn(const char* fn, const mm_paged_kv* kv, const mm_paged_step* st, int nq, int rows) {
    if (int rc = check_paged(fn, kv, st, rows)) return rc;
    MM_CHECK_ARG(nq > 0 && nq % kv->heads == 0 && nq < 1 << 20, "%s: %d query heads are no multiple of %d key heads", fn, nq, kv->heads);
    MM_CHECK_ARG((int64_t)st->max_new * (nq / kv->heads) < (int64_t)1 << 30 && (int64_t)st->max_new * (nq / kv->heads) / 128 < 16000,
                 "%s: max_new=%d rows of %d heads exceed the grid limit", fn, st->max_new, nq);
    MM_CHECK_ARG((int64_t)st->seqs * kv->heads < (int64_t)1 << 23 && (int64_t)rows * nq < (int64_t)1 << 31,
                 "%s: %d sequences, %d rows exceed the grid limit", fn, st->seqs, rows);
    MM_CHECK_ARG(st->max_kv < 1 << 30, "%s: max_kv=%d exceeds 2^30", fn, st->max_kv);
    return MM_OK;
}

}  // namespace mm

using namespace mm;

extern "C" size_t mm_paged_attn_workspace_bytes(const mm_paged_kv* kv, const mm_paged_step* step, int nq, int rows) {
    if (check_paged_attn("mm_paged_attn_workspace_bytes", kv, step, nq, rows) != MM_OK) return 0;
    const PagedPlan p = plan(*kv, *step, nq);
    return p.bytes(*kv, *step, rows, nq);
}

extern "C" int mm_paged_attn_fwd(const mm_paged_kv* kv, const mm_paged_step* step, void* out, int64_t o_row, int64_t o_head, float* lse,
                                 int64_t l_row, const void* q, int64_t q_row, int64_t q_head, int nq, int rows, float softmax_scale,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    const char* fn = "mm_paged_attn_fwd";
    if (int rc = check_paged_attn(fn, kv, step, nq, rows)) return rc;
    if (rows == 0 || step->seqs == 0 || step->max_new == 0) return MM_OK;
    MM_CHECK_ARG(out && lse && q, "%s: null pointer", fn);
    MM_CHECK_ARG(aligned16(q) && aligned16(out) && q_row % 8 == 0 && q_head % 8 == 0 && o_row % 8 == 0 && o_head % 8 == 0,
                 "%s: q / out must be 16-byte aligned with strides a multiple of 8", fn);
    MM_CHECK_ARG(softmax_scale > 0.f, "%s: softmax_scale %g must be positive", fn, (double)softmax_scale);
    const PagedPlan p = plan(*kv, *step, nq);
    const size_t need = p.bytes(*kv, *step, rows, nq);
    MM_CHECK_ARG(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need),
                 "%s: workspace of %zu bytes needed (16-byte aligned), got %zu", fn, need, workspace ? workspace_bytes : (size_t)0);
    const int64_t partials = (p.few_splits > 1 ? (int64_t)step->seqs * kv->heads * p.few_rows : 0) + (p.many_splits > 1 ? (int64_t)rows * nq : 0);
    MM_CHECK_ARG(partials < (int64_t)1 << 26, "%s: %lld joined rows exceed the grid limit", fn, (long long)partials);
    PagedAttnArgs a{};
    a.kv = *kv;
    a.st = *step;
    a.q = (const u16*)q, a.out = (u16*)out, a.lse = lse;
    a.q_row = q_row, a.q_head = q_head, a.o_row = o_row, a.o_head = o_head, a.l_row = l_row;
    a.nq = nq, a.group = nq / kv->heads, a.rows = rows;
    a.scale_log2e = softmax_scale * kLog2e;
    a.page = make_fastdiv(kv->page_size), a.grp = make_fastdiv(a.group);
    a.few_chunk = p.few_chunk, a.few_splits = p.few_splits, a.many_chunk = p.many_chunk, a.many_splits = p.many_splits;
    a.few_rows = p.few_rows;
    if (need) {
        a.few_o = (float*)workspace;
        a.many_o = a.few_o + p.few_partials(*kv, *step) * kv->hn;
        a.few_ml = a.many_o + p.many_partials(rows, nq) * kv->hn;
        a.many_ml = a.few_ml + p.few_partials(*kv, *step) * 2;
    }
    hipStream_t st = (hipStream_t)stream;
    return dispatch_dtype(kv->dtype, [&](auto t) -> int {
        using T = decltype(t);
        return kv->hn == 64 ? launch_paged_attn<T, 64>(a, p, st) : launch_paged_attn<T, 128>(a, p, st);
    });
}
