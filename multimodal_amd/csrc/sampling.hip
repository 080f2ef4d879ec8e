// sampling.hip - the next token of each row of logits: temperature, top-k, top-p, min-p and a given random number
// (reference: filter_logits + multinomial of megatron/text_generation_utils.py).
//
// The tokens of a row are ordered by descending logit, ties by ascending index; token t weighs w = exp((x_t - max) / temperature).
// Every filter keeps a prefix of that order, so each is a bound on the running weight: Z_k (the first k tokens), Z_p (up to the
// token whose running weight first exceeds top_p Z_k), Z_m (w >= min_p), and the token drawn is the first whose running
// weight exceeds u min(Z_k, Z_p, Z_m).  No sort is needed: a 16-bit logit has 65536 values at most, so a histogram over the
// values, in order, holds the whole distribution exactly - counts are integers, one weight per value in 64 bits - and the token is
// the j-th by index of one value.  Sums run in a fixed order: the result does not depend on scheduling, and a border of two tokens
// is off by about 1e-15 of the weight.  The running sums of neighbours are added up in different orders and so may differ either way
// by that much; a random number below 1 stays 2^-24 of the weight away from the end, but the last token kept, which one of 1 or
// more asks for, is found by counting tokens instead.
//
// One workgroup of 16 waves per row.  Its histogram (a count of a non-negative value in the low half of a word, of a negative one
// in the high half; 130 KB) fills most of a CU's LDS.  Steps: (1) the row into registers, each wave a contiguous 16th of it (the
// search by index needs that), one LDS atomic per logit as it arrives, and its largest value; (2) count and weight of every 64
// neighbouring values ("chunk"), one thread a chunk: the values of a chunk share their exponent and are evenly spaced, so their weights
// are a geometric sequence and the chunk's weight is a polynomial, sum n_i r^i, by Horner's rule - two exponentials a chunk instead of
// one a value.  A chunk takes 65 words of LDS, so that 64 lanes walking 64 chunks in step meet 64 banks; (3) a scan over the 1024
// chunks; (4) one wave finds the borders: 64-way search for the chunk, a scan over its 64 values; (5) the j-th match of the value found.
// With a top-k of at most 512, what can be among the first k is listed and ranked instead of counted.
// Rows of more than 65528 logits (BIG) could overflow 16-bit counts: they count non-negative and negative values one after the
// other in 32 bits, re-read the row instead of keeping it, and recount a chunk when a border falls into it.
//
// Bound by a row's chain of steps in one CU, not by HBM.  50304 fp16 logits, cycles: row and LDS atomics (1024 wave instructions) 11400,
// chunk sums 5300 (vector instructions), scan 1600, borders 4300, match 2400; the list instead of all of that 12000.  Kernel times:
// one row of bf16 with top-k 40: 8.4 us; 64 rows, top-p and min-p: 15 us; 512 rows with parameters of their own (two
// rows a CU after each other): 30 us, 51.5 MB at 1.7 TB/s.  BIG rows, read again for every recount: 64 of 65529 47 us (65528: 16), 64 of
// 128256 78 us, 190 of them 95.
#include "common.h"

namespace mm {

struct SampleArgs {
    const u16* logits;
    int64_t row_stride;
    const float* u;
    int64_t* out;
    int vocab;
    float temperature, top_p, min_p;
    int top_k;
    const float *temperature_v, *top_p_v, *min_p_v;  // per row, or NULL: the scalar
    const int32_t* top_k_v;
};

constexpr int kSampleThreads = 1024, kSampleWaves = 16, kChunks = 1024, kSampleSteps = 8, kListed = 1024;

// A 16-bit logit's place in descending order: non-negative b -> 0x7fff - b, negative b (sign bit set) -> b.  Two at a time.
// -0 (0x8000) becomes a value of its own next to +0 (0x7fff); they are merged where it matters.
__device__ __forceinline__ uint32_t order2(uint32_t v) {
    typedef __attribute__((ext_vector_type(2))) short ss2;
    const uint32_t negative = __builtin_bit_cast(uint32_t, __builtin_bit_cast(ss2, v) >> 15);
    return v ^ (0x7fff7fffu & ~negative);
}
constexpr int kPlusZero = 0x7fff, kMinusZero = 0x8000;
template <typename T> constexpr int inf_bits();
template <> constexpr int inf_bits<BF16>() { return 0x7f80; }
template <> constexpr int inf_bits<F16>() { return 0x7c00; }
template <typename T> constexpr int plus_inf() { return 0x7fff - inf_bits<T>(); }   // smaller: NaN
template <typename T> constexpr int minus_inf() { return 0x8000 + inf_bits<T>(); }  // larger: NaN
template <typename T> __device__ __forceinline__ float order_value(int dk) { return to_f32<T>((u16)(dk < 0x8000 ? 0x7fff - dk : dk)); }

// the weights of a row
template <typename T> struct Weights {
    int dmax;  // the largest value's place
    double xmax, inv_t;
    __device__ __forceinline__ double at(int dk) const {
        if (dk == dmax) return 1.0;
        const double x = (double)order_value<T>(dk);
        if (x == -(double)INFINITY || xmax == (double)INFINITY) return 0.0;
        return exp(fmax((x - xmax) * inv_t, -800.0));
    }
};

// Inclusive scans over a wave by DPP (row shifts inside 16 lanes, then the row broadcasts): no LDS round trips.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ double dpp_d(double v) {
    const unsigned long long b = __double_as_longlong(v);
    const uint32_t lo = dpp_u<CTRL, ROWS>((uint32_t)b), hi = dpp_u<CTRL, ROWS>((uint32_t)(b >> 32));
    return __longlong_as_double(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ uint32_t scan_u(uint32_t v) {
    v += dpp_u<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
    v += dpp_u<0x112, 0xf>(v);
    v += dpp_u<0x114, 0xf>(v);
    v += dpp_u<0x118, 0xf>(v);
    v += dpp_u<0x142, 0xa>(v);  // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3
    v += dpp_u<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ double scan_d(double v) {
    v += dpp_d<0x111, 0xf>(v);
    v += dpp_d<0x112, 0xf>(v);
    v += dpp_d<0x114, 0xf>(v);
    v += dpp_d<0x118, 0xf>(v);
    v += dpp_d<0x142, 0xa>(v);
    v += dpp_d<0x143, 0xc>(v);
    return v;
}
// minimum over a wave of two 16-bit numbers at once, in the last lane; row_min over each 16 lanes, in the last lane of the row
typedef __attribute__((ext_vector_type(2))) unsigned short us2;
__device__ __forceinline__ us2 pk_min(us2 a, us2 b) { return __builtin_elementwise_min(a, b); }
template <int CTRL, int ROWS> __device__ __forceinline__ us2 dpp_min(us2 v) {
    const int o = __builtin_amdgcn_update_dpp(-1, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false);
    return pk_min(v, __builtin_bit_cast(us2, o));
}
__device__ __forceinline__ us2 row_min(us2 v) {
    v = dpp_min<0x111, 0xf>(v);
    v = dpp_min<0x112, 0xf>(v);
    v = dpp_min<0x114, 0xf>(v);
    return dpp_min<0x118, 0xf>(v);
}
__device__ __forceinline__ us2 wave_min2(us2 v) { return dpp_min<0x143, 0xc>(dpp_min<0x142, 0xa>(row_min(v))); }
__device__ __forceinline__ uint32_t row_sum_u(uint32_t v) {
    v += dpp_u<0x111, 0xf>(v);
    v += dpp_u<0x112, 0xf>(v);
    v += dpp_u<0x114, 0xf>(v);
    return v + dpp_u<0x118, 0xf>(v);
}
__device__ __forceinline__ double row_sum_d(double v) {
    v += dpp_d<0x111, 0xf>(v);
    v += dpp_d<0x112, 0xf>(v);
    v += dpp_d<0x114, 0xf>(v);
    return v + dpp_d<0x118, 0xf>(v);
}
__device__ __forceinline__ double lane_d(double v, int l) {
    const unsigned long long b = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)b, l), hi = __builtin_amdgcn_readlane((uint32_t)(b >> 32), l);
    return __longlong_as_double(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ uint32_t lane_u(uint32_t v, int l) { return __builtin_amdgcn_readlane(v, l); }

struct SampleShared {
    uint32_t hist[512 * 65];  // value dk: word hist_word(dk), low half below 0x8000
    double mass[kChunks];    // then its inclusive scan
    uint32_t count[kChunks];
    double wave_mass[kSampleWaves];
    uint32_t wave_count[kSampleWaves];
    us2 wave_ends[kSampleWaves];
    double min_p_mass;
    int dk, j;
    uint32_t one_chunk[64];
    uint32_t listed;
    // the list of a top-k's candidates and its ranking take the histogram's place
    __device__ __forceinline__ uint64_t* list() { return reinterpret_cast<uint64_t*>(hist); }
    __device__ __forceinline__ uint64_t* sorted() { return reinterpret_cast<uint64_t*>(hist) + kListed; }
};

__device__ __forceinline__ int hist_word(int dk) { return (dk & 0x7fff) + ((dk >> 6) & 511); }

// the first of 1024 entries with pred(entry), which holds from there on (the last one if it never does); a whole wave calls it
template <typename F> __device__ __forceinline__ int first_of(F&& pred) {
    const int lane = threadIdx.x & 63;
    uint64_t b = __ballot(pred(16 * lane + 15));
    const int blk = b ? __builtin_ctzll(b) : 63;
    b = __ballot(lane < 16 && pred(16 * blk + (lane & 15)));
    return 16 * blk + (b ? __builtin_ctzll(b) : 15);
}

template <typename T, bool BIG> __global__ __launch_bounds__(kSampleThreads) void sample_tokens_k(const SampleArgs a) {
    __shared__ __attribute__((aligned(16))) SampleShared sm;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, row = blockIdx.x;
    constexpr uint32_t kNone = (uint32_t)minus_inf<T>() * 0x10001u;  // two -inf, in the order
    // The row as 16-byte aligned chunks: `lead` elements of the first one and the end of the last belong to no token and become
    // -inf.  (An aligned chunk that holds one element of the row lies in the allocation's own 16-byte granule.)
    const u16* rp = a.logits + (int64_t)row * a.row_stride;
    const int lead = (int)(((uintptr_t)rp & 15) >> 1);
    const u32x4* base = reinterpret_cast<const u32x4*>(rp - lead);
    const int nch = (int)(((int64_t)lead + a.vocab + 7) >> 3);
    const int seg = (nch + kSampleWaves - 1) / kSampleWaves;
    const int ch0 = wave * seg, ch1 = min(ch0 + seg, nch);
    const int steps = (seg + 63) >> 6;

    auto ordered = [&](u32x4 v, int ch) -> u32x4 {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = order2(v[i]);
        if (ch == 0 || ch == nch - 1) {
            const int e0 = ch * 8 - lead;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (e0 + 2 * i < 0 || e0 + 2 * i >= a.vocab) v[i] = (v[i] & 0xffff0000u) | (kNone & 0xffffu);
                if (e0 + 2 * i + 1 < 0 || e0 + 2 * i + 1 >= a.vocab) v[i] = (v[i] & 0xffffu) | (kNone & 0xffff0000u);
            }
        }
        return v;
    };
    u32x4 reg[BIG ? 1 : kSampleSteps];
    if constexpr (!BIG) {
#pragma unroll
        for (int s = 0; s < kSampleSteps; ++s) {
            reg[s] = u32x4{kNone, kNone, kNone, kNone};
            if (s < steps && ch0 + 64 * s + lane < ch1) reg[s] = base[ch0 + 64 * s + lane];
        }
    }
    const float u = a.u[row];
    const float temp = a.temperature_v ? a.temperature_v[row] : a.temperature;
    const float p = a.top_p_v ? a.top_p_v[row] : a.top_p, mp = a.min_p_v ? a.min_p_v[row] : a.min_p;
    const int k = a.top_k_v ? a.top_k_v[row] : a.top_k;
    const bool greedy = !(temp > 0.f);
    const bool last = !(u < 1.f);  // (or NaN) the last token kept
    // a token is kept whose weight is at least this, and not 0
    const double floor_w = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;
    auto clear_hist = [&]() {
        u32x4* h = reinterpret_cast<u32x4*>(sm.hist);
        for (int i = tid; i < 512 * 65 / 4; i += kSampleThreads) h[i] = u32x4{0, 0, 0, 0};
    };
    const bool try_list = !BIG && !greedy && k > 0 && k <= kSampleThreads / 2;
    if (!greedy && !try_list) clear_hist();
    us2 lo2 = {0xffff, 0xffff}, hi2 = {0, 0};
    auto ends_of = [&](uint32_t o) {
        lo2 = pk_min(lo2, __builtin_bit_cast(us2, o));
        hi2 = __builtin_elementwise_max(hi2, __builtin_bit_cast(us2, o));
    };
    auto count2 = [&](uint32_t o) {  // hist_word of both halves at once
        const uint32_t w = (o & 0x7fff7fffu) + ((o >> 6) & 0x01ff01ffu);
        uint32_t s0 = __builtin_amdgcn_ubfe(o, 15, 1), s1 = o >> 31;
        asm("" : "+v"(s0), "+v"(s1));  // keep the signs numbers: a compare and a select each cost more
        atomicAdd(&sm.hist[w & 0xffffu], __umul24(s0, 0xffffu) + 1u);
        atomicAdd(&sm.hist[w >> 16], __umul24(s1, 0xffffu) + 1u);
    };
    if constexpr (!BIG) {
        if (!greedy && !try_list) {  // counted as it arrives: the vector work hides behind the LDS atomics
            __syncthreads();
#pragma unroll
            for (int s = 0; s < kSampleSteps; ++s)
                if (s < steps && ch0 + 64 * s + lane < ch1) {
                    reg[s] = ordered(reg[s], ch0 + 64 * s + lane);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        count2(reg[s][i]);
                        ends_of(reg[s][i]);
                    }
                }
        } else {
#pragma unroll
            for (int s = 0; s < kSampleSteps; ++s)
                if (s < steps && ch0 + 64 * s + lane < ch1) {
                    reg[s] = ordered(reg[s], ch0 + 64 * s + lane);
#pragma unroll
                    for (int i = 0; i < 4; ++i) ends_of(reg[s][i]);
                }
        }
    }
    // f(two places in the order) over this thread's logits
    auto each2 = [&](auto&& f) {
        if constexpr (BIG) {
            for (int ch = ch0 + lane; ch < ch1; ch += 64) {
                const u32x4 v = ordered(base[ch], ch);
#pragma unroll
                for (int i = 0; i < 4; ++i) f(v[i]);
            }
        } else {
#pragma unroll
            for (int s = 0; s < kSampleSteps; ++s)
                if (s < steps && ch0 + 64 * s + lane < ch1) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) f(reg[s][i]);
                }
        }
    };

    if constexpr (BIG) each2(ends_of);
    hi2 = ~hi2;
    const us2 mine2 = pk_min(us2{lo2[0], hi2[0]}, us2{lo2[1], hi2[1]});  // {smallest, complement of the largest} place of this thread
    {
        const us2 w2 = wave_min2(mine2);
        if (lane == 63) sm.wave_ends[wave] = w2;
    }
    __syncthreads();
    const us2 ends = __builtin_bit_cast(us2, lane_u(__builtin_bit_cast(uint32_t, row_min(sm.wave_ends[lane & 15])), 15));
    int lo = ends[0];
    const int hi = 0xffff - ends[1];
    if (lo < plus_inf<T>() || hi > minus_inf<T>() || lo >= minus_inf<T>()) {  // a NaN, or nothing but -inf: no token
        if (tid == 0) a.out[row] = -1;
        return;
    }
    if (lo == kMinusZero) lo = kPlusZero;

    int dk = lo, j = 0;  // the token: the j-th by index of the value with this place
    if (!greedy) {
        const Weights<T> wt{lo, (double)order_value<T>(lo), 1.0 / (double)temp};
        // values below max - 50 T weigh less than 2^-72 each: nothing of them reaches a 64-bit sum that holds the largest's 1 (but
        // the last token kept may be one of them)
        const float xlow = (float)(wt.xmax - 50.0 * (double)temp);
        int dlow = minus_inf<T>();
        if (xlow > -INFINITY && !last) {
            const u16 b = from_f32<T>(xlow);
            dlow = min(dlow, ((b & 0x8000) ? (int)b : 0x7fff - (int)b) + 1);
        }
        const int clo = lo >> 6;
        sm.count[tid] = 0;
        sm.mass[tid] = 0.0;
        bool listed = false;
        if (try_list) {
            // The k-th largest of the threads' largest logits bounds the k-th largest logit from below: what lies in a later chunk
            // is not among the first k (50304 logits, k = 64: some 0.3 % are left).
            __syncthreads();
            atomicAdd(&sm.count[mine2[0] >> 6], 1u);
            __syncthreads();
            const uint32_t n = sm.count[tid], c = scan_u(n);
            if (lane == 63) sm.wave_count[wave] = c;
            if (tid == 0) sm.listed = 0;
            __syncthreads();
            const uint32_t w = sm.wave_count[lane & 15];
            const uint32_t upto = c + lane_u(row_sum_u((lane & 15) < wave ? w : 0u), 15);
            if (upto >= (uint32_t)k && upto - n < (uint32_t)k) {  // one thread
                sm.dk = tid;
                sm.j = (int)((uint32_t)k - (upto - n));  // the how manieth of this chunk's maxima
            }
            if (tid < 64) sm.one_chunk[tid] = 0;
            __syncthreads();
            const int bc = __builtin_amdgcn_readfirstlane(sm.dk);
            if ((int)(mine2[0] >> 6) == bc) atomicAdd(&sm.one_chunk[mine2[0] & 63], 1u);
            __syncthreads();
            const uint64_t at_k = __ballot(scan_u(sm.one_chunk[lane]) >= (uint32_t)sm.j);
            dlow = min(dlow, 64 * bc + (int)__builtin_ctzll(at_k));
            if (dlow == kPlusZero) dlow = kMinusZero;  // the two zeros tie
            sm.count[tid] = 0;
            // What is left is listed (in no order) and, if the list holds it, ranked: place and index make one number
            const us2 beyond = {(unsigned short)(dlow + 1), (unsigned short)(dlow + 1)};
            auto list = [&](uint32_t o, int e) {
                const us2 in = __builtin_elementwise_sub_sat(beyond, __builtin_bit_cast(us2, o));  // not 0: at or before dlow
                if (__builtin_bit_cast(uint32_t, in) != 0) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (in[i] == 0) continue;
                        uint32_t d = i ? o >> 16 : o & 0xffffu;
                        if (d == (uint32_t)kMinusZero) d = kPlusZero;
                        const uint32_t at = atomicAdd(&sm.listed, 1u);
                        if (at < kListed) sm.list()[at] = ((uint64_t)d << 32) | (uint32_t)(e + i);
                    }
                }
            };
#pragma unroll
            for (int s = 0; s < kSampleSteps; ++s)
                if (s < steps && ch0 + 64 * s + lane < ch1) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) list(reg[s < (BIG ? 1 : kSampleSteps) ? s : 0][i], (ch0 + 64 * s + lane) * 8 - lead + 2 * i);
                }
            __syncthreads();
            const int m = __builtin_amdgcn_readfirstlane((int)sm.listed);
            listed = m <= kListed;
            if (listed) {
                if (64 * wave < m) {
                    const uint64_t key = sm.list()[min(tid, m - 1)];
                    int rank = 0;
#pragma unroll 8
                    for (int i = 0; i < m; ++i) rank += sm.list()[i] < key ? 1 : 0;
                    if (tid < m) sm.sorted()[rank] = key;
                }
                __syncthreads();
                // weights in order; their running sum
                double wgt = 0.0;
                if (tid < m && tid < k) wgt = wt.at((int)(sm.sorted()[tid] >> 32));
                const double c2 = scan_d(wgt);
                const uint64_t heavy = __ballot(wgt >= floor_w && wgt > 0.0);
                if (lane == 63) {
                    sm.wave_mass[wave] = c2;
                    sm.wave_count[wave] = __popcll(heavy);
                }
                __syncthreads();
                sm.mass[tid] = c2 + lane_d(row_sum_d((lane & 15) < wave ? sm.wave_mass[lane & 15] : 0.0), 15);
                __syncthreads();
                if (wave == 0) {
                    double z = sm.mass[kChunks - 1], zp = z;
                    int end = max((int)lane_u(row_sum_u(sm.wave_count[lane & 15]), 15), 1) - 1;  // the last one kept
                    if (mp > 0.f) zp = fmin(zp, sm.mass[end]);
                    if (p > 0.f && p < 1.f) {
                        const int at = first_of([&](int i) { return sm.mass[i] > (double)p * z; });
                        zp = fmin(zp, sm.mass[at]);
                        end = min(end, at);
                    }
                    zp = fmax(zp, 1.0);
                    const double t = (double)u * zp;
                    const int f = last ? end : min(first_of([&](int i) { return sm.mass[i] > t; }), end);
                    if (lane == 0) a.out[row] = (int64_t)(uint32_t)sm.sorted()[f];
                }
                return;
            }
        }
        const int chi = dlow >> 6;
        // count and weight of chunk tid, chunks first .. last being in the histogram (BIG: half a histogram of whole words)
        auto chunk_sums = [&](int first, int last) {
            if (64 * wave + 63 < first || 64 * wave > last) return;  // none of this wave's chunks
            const uint32_t* h = sm.hist + (tid & 511) * 65;
            const int sh = BIG || tid < 512 ? 0 : 16;
            const uint32_t mask = BIG ? 0xffffffffu : 0xffffu;
            // the chunk's values are x0 - i ulp; weights e^((x0 - max) / T) r^i with r = e^(-ulp / T).  The largest value's own chunk
            // counts from that value, so that no power exceeds 1
            const bool top = tid == clo;
            const int i0 = top ? lo & 63 : 0, d0 = 64 * tid + i0;
            const int bits = d0 < 0x8000 ? 0x7fff - d0 : d0 & 0x7fff;  // magnitude of x0
            const double x0 = (double)order_value<T>(d0);
            const int e = max(bits >> (inf_bits<T>() == 0x7f80 ? 7 : 10), 1) - (inf_bits<T>() == 0x7f80 ? 127 + 7 : 15 + 10);
            const double r = exp(fmax(-ldexp(1.0, e) * wt.inv_t, -800.0));
            const bool none = x0 == -(double)INFINITY || (wt.xmax == (double)INFINITY && !top);
            const double first_w = top ? 1.0 : none ? 0.0 : exp(fmax((x0 - wt.xmax) * wt.inv_t, -800.0));
            double acc = 0.0;
            uint32_t n = 0;
            if (clo >> 6 == wave) {  // the wave of the top chunk
#pragma unroll 16
                for (int i = 63; i >= 0; --i) {
                    const uint32_t c = (h[i] >> sh) & mask;
                    n += c;
                    acc = i >= i0 ? fma(acc, r, (double)c) : acc;
                }
            } else {
#pragma unroll 16
                for (int i = 63; i >= 0; --i) {
                    const uint32_t c = (h[i] >> sh) & mask;
                    n += c;
                    acc = fma(acc, r, (double)c);
                }
            }
            if (tid >= first && tid <= last) {
                sm.count[tid] = n;
                sm.mass[tid] = acc * first_w;
            }
        };
        if constexpr (!BIG) {
            if (try_list) {  // the list has been where the counts go
                __syncthreads();
                clear_hist();
                __syncthreads();
                each2(count2);
            }
            __syncthreads();
            if (tid == 0) {  // -0 is +0
                const uint32_t z = sm.hist[hist_word(kMinusZero)] >> 16;
                sm.hist[hist_word(kMinusZero)] &= 0xffffu;
                sm.hist[hist_word(kPlusZero)] += z;
            }
            __syncthreads();
            chunk_sums(clo, chi);
        } else {
            for (int half = 0; half < 2; ++half) {
                if (half == 1) {
                    __syncthreads();
                    clear_hist();
                    __syncthreads();
                }
                auto one = [&](int d) {
                    if (d == kMinusZero) d = kPlusZero;
                    if ((d >> 15) == half) atomicAdd(&sm.hist[hist_word(d)], 1u);
                };
                each2([&](uint32_t o) {
                    one((int)(o & 0xffffu));
                    one((int)(o >> 16));
                });
                __syncthreads();
                chunk_sums(max(clo, 512 * half), min(chi, 512 * half + 511));
            }
        }
        __syncthreads();
        {   // inclusive scans over the chunks
            const uint32_t c = scan_u(sm.count[tid]);
            const double m = scan_d(sm.mass[tid]);
            if (lane == 63) {
                sm.wave_count[wave] = c;
                sm.wave_mass[wave] = m;
            }
            __syncthreads();
            const bool ahead = (lane & 15) < wave;
            sm.count[tid] = c + lane_u(row_sum_u(ahead ? sm.wave_count[lane & 15] : 0u), 15);
            sm.mass[tid] = m + lane_d(row_sum_d(ahead ? sm.wave_mass[lane & 15] : 0.0), 15);
            __syncthreads();
        }

        // Borders.  One wave, a second one for min-p beside it (BIG: every wave alike, because recounting a chunk takes the whole
        // workgroup).
        {
            auto counts = [&](int c) __attribute__((always_inline)) -> uint32_t {
                if constexpr (!BIG) return (sm.hist[(c & 511) * 65 + lane] >> (c < 512 ? 0 : 16)) & 0xffffu;
                __syncthreads();
                if (tid < 64) sm.one_chunk[tid] = 0;
                __syncthreads();
                auto one = [&](int d) {
                    if (d == kMinusZero) d = kPlusZero;
                    if ((d >> 6) == c) atomicAdd(&sm.one_chunk[d & 63], 1u);
                };
                each2([&](uint32_t o) {
                    one((int)(o & 0xffffu));
                    one((int)(o >> 16));
                });
                __syncthreads();
                return sm.one_chunk[lane];
            };
            // the first token whose running weight exceeds t: value, how many tokens of that value are ahead of it, and the running
            // weight up to and with it
            struct Found {
                int dk, j;
                double upto;
            };
            auto find = [&](double t) __attribute__((always_inline)) -> Found {
                int c = first_of([&](int i) { return sm.mass[i] > t; });
                uint32_t n = counts(c);
                if (__ballot(n != 0) == 0) {
                    // an empty chunk: rounding put t between the sums of chunks without a token between them, or t is below 0.  The
                    // chunk that holds the last token up to here, or the first of all
                    const uint32_t upto = max(sm.count[c], 1u);
                    c = first_of([&](int i) { return sm.count[i] >= upto; });
                    n = counts(c);
                }
                const double ahead = c ? sm.mass[c - 1] : 0.0;
                const double w = n ? wt.at(64 * c + lane) : 0.0;
                const double incl = ahead + scan_d((double)n * w);
                const uint64_t any = __ballot(n != 0);
                const uint64_t over = __ballot(n != 0 && incl > t);
                const int l = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
                const double before = incl - (double)n * w, last = (double)(n ? n - 1 : 0);
                const double jj = over ? fmin(fmax(floor((t - before) / w), 0.0), last) : last;
                const double up = before + (jj + 1.0) * w;
                return Found{64 * c + l, (int)lane_u((uint32_t)(int)jj, l), lane_d(up, l)};
            };
            // the first value that weighs too little to be kept: 64-way search in the order
            auto first_below = [&]() __attribute__((always_inline)) -> int {
                int from = lo, span = 65536 - lo;
                while (span > 0) {
                    const int st = (span + 63) >> 6, at = from + lane * st + st - 1;
                    const double w = wt.at(min(at, minus_inf<T>()));
                    const bool kept = lane * st + st - 1 < span && w >= floor_w && w > 0.0;
                    const int g = __popcll(__ballot(kept));
                    from += g * st;
                    span -= g * st;
                    if (st == 1) break;
                    span = min(span, st);
                }
                return from;
            };
            auto min_p_mass = [&]() -> double {
                const int from = first_below();
                const int c = min(from, 65535) >> 6;
                const uint32_t n = counts(c);
                const double w = n ? wt.at(64 * c + lane) : 0.0;
                const double mi = scan_d(64 * c + lane < from ? (double)n * w : 0.0);
                return (c ? sm.mass[c - 1] : 0.0) + lane_d(mi, 63);
            };
            if (!BIG && wave == 1 && mp > 0.f) {
                const double m = min_p_mass();
                if (lane == 0) sm.min_p_mass = m;
            }
            // the number of tokens of the values ahead of this one
            auto tokens_ahead = [&](int d) __attribute__((always_inline)) -> uint32_t {
                const int c = min(d, 65535) >> 6;
                const uint32_t n = counts(c);
                return (c ? sm.count[c - 1] : 0u) + lane_u(scan_u(64 * c + lane < d ? n : 0u), 63);
            };
            double zp = 0.0;
            uint32_t kept = sm.count[kChunks - 1];  // how many tokens (`last` alone needs it)
            if (BIG || wave == 0) {
                double z = sm.mass[kChunks - 1];
                if (k > 0 && (uint32_t)k < kept) {
                    kept = (uint32_t)k;
                    const int c = first_of([&](int i) { return sm.count[i] >= (uint32_t)k; });
                    const uint32_t n = counts(c);
                    const double w = n ? wt.at(64 * c + lane) : 0.0;
                    const uint32_t ci = (c ? sm.count[c - 1] : 0u) + scan_u(n);
                    const double mi = (c ? sm.mass[c - 1] : 0.0) + scan_d((double)n * w);
                    const uint64_t over = __ballot(n != 0 && ci >= (uint32_t)k);
                    const int l = over ? __builtin_ctzll(over) : 63;
                    z = fmin(z, lane_d(mi - (double)(ci - (uint32_t)k) * w, l));
                }
                zp = z;
                if (p > 0.f && p < 1.f) {
                    const Found f = find((double)p * z);
                    zp = fmin(zp, f.upto);
                    if (last) kept = min(kept, tokens_ahead(f.dk) + (uint32_t)f.j + 1);
                }
                if (last) kept = min(kept, tokens_ahead(first_below()));
            }
            if (!BIG) __syncthreads();
            if (BIG || wave == 0) {
                int fdk, fj;
                if (last) {
                    const int c = first_of([&](int i) { return sm.count[i] >= kept; });
                    const uint32_t n = counts(c), upto = (c ? sm.count[c - 1] : 0u) + scan_u(n);
                    const int l = __builtin_ctzll(__ballot(upto >= kept));
                    fdk = 64 * c + l;
                    fj = (int)(kept - 1 - lane_u(upto - n, l));
                } else {
                    if (mp > 0.f) zp = fmin(zp, BIG ? min_p_mass() : sm.min_p_mass);
                    const Found f = find((double)u * fmax(zp, 1.0));
                    fdk = f.dk;
                    fj = f.j;
                }
                if (BIG || lane == 0) {
                    sm.dk = fdk;
                    sm.j = fj;
                }
            }
        }
        __syncthreads();
        dk = __builtin_amdgcn_readfirstlane(sm.dk);
        j = __builtin_amdgcn_readfirstlane(sm.j);
    }

    // the j-th token with this value, by index: matches per wave, then per 64-lane step, then per lane
    const uint32_t want = (uint32_t)dk * 0x10001u;
    auto matches = [&](uint32_t o) -> uint32_t {  // bit 0: the first of two matches, bit 1: the second
        const uint32_t x = o ^ want;
        uint32_t m = ((x & 0xffffu) == 0 ? 1u : 0u) | ((x >> 16) == 0 ? 2u : 0u);
        if (dk == kPlusZero) m |= ((o & 0xffffu) == kMinusZero ? 1u : 0u) | ((o >> 16) == kMinusZero ? 2u : 0u);
        return m;
    };
    uint32_t mine = 0;
    if (dk == kPlusZero || BIG) {
        each2([&](uint32_t o) { mine += __popc(matches(o)); });
    } else {  // both halves of a word at once: 1 - 0 where they are equal, else 1 - 1 or more, saturated
        us2 equal = {0, 0};
        each2([&](uint32_t o) { equal += __builtin_elementwise_sub_sat(us2{1, 1}, __builtin_bit_cast(us2, o ^ want)); });
        mine = (uint32_t)equal[0] + equal[1];
    }
    const uint32_t tot = lane_u(scan_u(mine), 63);
    if (lane == 0) sm.wave_count[wave] = tot;  // its readers of the scan above have passed a barrier since
    __syncthreads();
    const uint32_t before = lane_u(row_sum_u((lane & 15) < wave ? sm.wave_count[lane & 15] : 0u), 15);
    if ((uint32_t)j < before || (uint32_t)j >= before + tot) return;  // another wave has it
    uint32_t left = (uint32_t)j - before;
    bool done = false;
    auto locate = [&](u32x4 v, int ch) {  // one 64-lane step; lanes without a chunk hold no match
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) bits |= matches(v[i]) << (2 * i);
        if (done || __ballot(bits != 0) == 0) return;
        const uint32_t incl = scan_u(__popc(bits)), sum = lane_u(incl, 63);
        if (left >= sum) {
            left -= sum;
            return;
        }
        uint32_t excl = incl - __popc(bits);
        if (left >= excl && left < incl) {
            for (; excl < left; ++excl) bits &= bits - 1;
            a.out[row] = ch * 8 - lead + __builtin_ctz(bits);
        }
        done = true;
    };
    if constexpr (BIG) {
        for (int s = 0; s < steps && !done; ++s) {
            const int ch = ch0 + 64 * s + lane;
            u32x4 v = {kNone, kNone, kNone, kNone};
            if (ch < ch1) v = ordered(base[ch], ch);
            locate(v, ch);
        }
    } else {
#pragma unroll
        for (int s = 0; s < kSampleSteps; ++s)
            if (s < steps) locate(reg[s], ch0 + 64 * s + lane);
    }
}

// =====================================================================================  every row greedy
// One workgroup a row: the largest value and the first 16-byte chunk that holds it, then the index inside that chunk.  3125 rows of
// 8000 logits: 11 us, 50 MB at 4.4 TB/s (from the Infinity Cache as well as from HBM); 50000 of 500: 57 us - three quarters of the
// lanes have no chunk, and a row's join and second look at its chunk wait for each other.
template <typename T, int THREADS> __global__ __launch_bounds__(THREADS) void sample_greedy_k(const SampleArgs a) {
    constexpr int WAVES = THREADS / 64;
    __shared__ unsigned long long best_of[WAVES];
    __shared__ uint32_t nan_of[WAVES];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, row = blockIdx.x;
    const u16* rp = a.logits + (int64_t)row * a.row_stride;
    const int lead = (int)(((uintptr_t)rp & 15) >> 1);
    const u32x4* base = reinterpret_cast<const u32x4*>(rp - lead);
    const int nch = (int)(((int64_t)lead + a.vocab + 7) >> 3);
    auto place = [&](const u32x4& v, int ch, int i) -> uint32_t {  // of element i of a chunk; what belongs to no token: -inf
        const int e = ch * 8 - lead + i;
        const uint32_t o = order2(v[i >> 1]), d = i & 1 ? o >> 16 : o & 0xffffu;
        return e < 0 || e >= a.vocab ? (uint32_t)minus_inf<T>() : d;
    };
    uint32_t best = 0xffffu, at = 0, worst = 0;
    for (int ch = tid; ch < nch; ch += THREADS) {
        const u32x4 v = base[ch];
        uint32_t lo, hi;
        if (ch == 0 || ch == nch - 1) {
            lo = 0xffffu, hi = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) lo = min(lo, place(v, ch, i)), hi = max(hi, place(v, ch, i));
        } else {
            us2 l = {0xffff, 0xffff}, h = {0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const us2 o = __builtin_bit_cast(us2, order2(v[i]));
                l = pk_min(l, o);
                h = __builtin_elementwise_max(h, o);
            }
            lo = min(l[0], l[1]), hi = max(h[0], h[1]);
        }
        if (lo == (uint32_t)kMinusZero) lo = kPlusZero;
        if (lo < best) best = lo, at = (uint32_t)ch;
        worst = max(worst, hi);
    }
    unsigned long long key = ((unsigned long long)best << 32) | at;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const unsigned long long o = __shfl_xor(key, d, 64);
        key = o < key ? o : key;
    }
    const bool nan = __ballot(worst > (uint32_t)minus_inf<T>()) != 0;
    if (lane == 0) best_of[wave] = key, nan_of[wave] = nan ? 1 : 0;
    __syncthreads();
    if (tid != 0) return;
    uint32_t any_nan = 0;
    for (int w = 0; w < WAVES; ++w) {
        key = best_of[w] < key ? best_of[w] : key;
        any_nan |= nan_of[w];
    }
    const uint32_t lo = (uint32_t)(key >> 32);
    if (any_nan || lo < (uint32_t)plus_inf<T>() || lo >= (uint32_t)minus_inf<T>()) {
        a.out[row] = -1;
        return;
    }
    const int ch = (int)(uint32_t)key;
    const u32x4 v = base[ch];
    int first = 7;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        const uint32_t d = place(v, ch, i);
        if (d == lo || (lo == (uint32_t)kPlusZero && d == (uint32_t)kMinusZero)) first = i;
    }
    a.out[row] = ch * 8 - lead + first;
}

// =====================================================================================  small vocabularies
// One wave a row of up to 64 EPL - 7 logits: place and index make a 32-bit key, a bitonic sort over the wave orders them (lane l
// holds the keys l EPL .. l EPL + EPL - 1), and what follows is the definition: weights in that order, their running sum, borders by
// ballots.  Only the first top_k weights are computed.  Bound by vector instructions: 50000 rows of 500 logits with top-p 145 us
// (the exponentials and the sort about even), with top-k 20 111 us.
template <typename T, int EPL> __global__ __launch_bounds__(256) void sample_small_k(const SampleArgs a, int rows) {
    __shared__ uint32_t sorted_of[4][64 * EPL];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const bool live = (int64_t)blockIdx.x * 4 + wave < rows;
    const int row = live ? blockIdx.x * 4 + wave : rows - 1;  // a wave behind the last row repeats it and writes nothing
    const u16* rp = a.logits + (int64_t)row * a.row_stride;
    const int lead = (int)(((uintptr_t)rp & 15) >> 1);
    const u32x4* base = reinterpret_cast<const u32x4*>(rp - lead);
    const int nch = (lead + a.vocab + 7) >> 3;
    uint32_t key[EPL];
    bool nan = false;
#pragma unroll
    for (int s = 0; s < EPL / 8; ++s) {
        const int ch = 64 * s + lane;
        u32x4 v = {0, 0, 0, 0};
        if (ch < nch) v = base[ch];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = ch * 8 - lead + i;
            const uint32_t o = order2(v[i >> 1]);
            uint32_t d = i & 1 ? o >> 16 : o & 0xffffu;
            const bool valid = e >= 0 && e < a.vocab;
            nan |= valid && (d < (uint32_t)plus_inf<T>() || d > (uint32_t)minus_inf<T>());
            if (d == (uint32_t)kMinusZero) d = kPlusZero;
            key[8 * s + i] = valid ? (d << 16) | (uint32_t)e : 0xffffffffu;
        }
    }
    const float u = a.u[row];
    const float temp = a.temperature_v ? a.temperature_v[row] : a.temperature;
    const float p = a.top_p_v ? a.top_p_v[row] : a.top_p, mp = a.min_p_v ? a.min_p_v[row] : a.min_p;
    const int k = a.top_k_v ? a.top_k_v[row] : a.top_k;

    // Bitonic sort: runs of `size` keys alternate in direction; a descending run is sorted ascending with all bits flipped
#pragma unroll
    for (int size = 2; size <= 64 * EPL; size *= 2) {
        uint32_t flip[2] = {0, 0};  // by the key's place in the lane where a run is shorter than a lane's keys
        if (size >= EPL) flip[0] = flip[1] = size < 64 * EPL && (lane & (size / EPL)) ? 0xffffffffu : 0u;
        else flip[1] = 0xffffffffu;
#pragma unroll
        for (int r = 0; r < EPL; ++r) key[r] ^= flip[(r & size) ? 1 : 0];
#pragma unroll
        for (int stride = size / 2; stride > 0; stride /= 2) {
            if (stride >= EPL) {
                const bool low = (lane & (stride / EPL)) == 0;
#pragma unroll
                for (int r = 0; r < EPL; ++r) {
                    const uint32_t o = (uint32_t)__shfl_xor((int)key[r], stride / EPL, 64);
                    key[r] = low ? min(key[r], o) : max(key[r], o);
                }
            } else {
#pragma unroll
                for (int r = 0; r < EPL; ++r)
                    if ((r & stride) == 0) {
                        const uint32_t x = key[r], y = key[r + stride];
                        key[r] = min(x, y), key[r + stride] = max(x, y);
                    }
            }
        }
#pragma unroll
        for (int r = 0; r < EPL; ++r) key[r] ^= flip[(r & size) ? 1 : 0];
    }
    uint32_t* sorted = sorted_of[wave];
#pragma unroll
    for (int r = 0; r < EPL; ++r) sorted[lane * EPL + r] = key[r];
    __syncthreads();

    const uint32_t first = lane_u(key[0], 0);
    const int lo = (int)(first >> 16);
    int64_t token = (int64_t)(first & 0xffffu);
    if (__ballot(nan) || lo >= minus_inf<T>()) token = -1;  // a NaN, or nothing but -inf: no token
    else if (temp > 0.f) {
        const Weights<T> wt{lo, (double)order_value<T>(lo), 1.0 / (double)temp};
        const int kept = k > 0 && k < a.vocab ? k : a.vocab;
        const double floor_w = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;
        double run[EPL], z = 0.0;  // running weights of keys 64 j + lane
        int heavy = 0;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            run[j] = z;
            if (64 * j >= kept) continue;
            const double w = 64 * j + lane < kept ? wt.at((int)(sorted[64 * j + lane] >> 16)) : 0.0;
            heavy += __popcll(__ballot(w >= floor_w && w > 0.0));
            run[j] = z + scan_d(w);
            z = lane_d(run[j], 63);
        }
        // the first key whose running weight exceeds t (the last one kept if none does), and that weight
        auto find = [&](double t, double& upto) -> int {
            int at = kept - 1;
            upto = z;
#pragma unroll
            for (int j = EPL - 1; j >= 0; --j) {
                const uint64_t b = __ballot(64 * j + lane < kept && run[j] > t);
                if (b) {
                    const int l = __builtin_ctzll(b);
                    at = 64 * j + l;
                    upto = lane_d(run[j], l);
                }
            }
            return at;
        };
        double zp = z, upto;
        int end = max(heavy, 1) - 1;  // the last one kept
        if (mp > 0.f) {
#pragma unroll
            for (int j = 0; j < EPL; ++j)
                if (end >> 6 == j) zp = fmin(zp, lane_d(run[j], end & 63));
        }
        if (p > 0.f && p < 1.f) {
            end = min(end, find((double)p * z, upto));
            zp = fmin(zp, upto);
        }
        // a random number of 1 or more, or NaN: the last one kept
        if (u < 1.f) end = min(end, find((double)u * fmax(zp, 1.0), upto));
        token = (int64_t)(sorted[end] & 0xffffu);
    }
    if (live && lane == 0) a.out[row] = token;
}

}  // namespace mm

using namespace mm;

extern "C" int mm_sample_tokens(int64_t* tokens, const void* logits, int64_t row_stride, const float* u, int rows, int vocab,
                                float temperature, const float* temperature_rows, int top_k, const int32_t* top_k_rows, float top_p,
                                const float* top_p_rows, float min_p, const float* min_p_rows, int dtype, void* stream) {
    const char* fn = "mm_sample_tokens";
    MM_CHECK_ARG(rows >= 0 && rows < 1 << 22 && vocab > 0 && vocab < 1 << 30, "%s: rows=%d vocab=%d out of range", fn, rows, vocab);
    if (rows == 0) return MM_OK;
    MM_CHECK_ARG(tokens && logits && u, "%s: null pointer", fn);
    MM_CHECK_ARG(((uintptr_t)logits & 1) == 0, "%s: logits must be 2-byte aligned", fn);
    SampleArgs a{(const u16*)logits, row_stride, u, tokens, vocab, temperature, top_p, min_p, top_k, temperature_rows, top_p_rows,
                 min_p_rows, top_k_rows};
    hipStream_t st = (hipStream_t)stream;
    return dispatch_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        // Where the scalar temperature says that every row is greedy, nothing needs the histogram (50000 rows of 500 484 -> 57 us,
        // 3125 of 8000 38 -> 12).  Workgroups of 256 or 1024 threads, us: 1 row of 8000 4.4 / 4.4, of 16384 5.2 / 4.6, of 32000 6.8
        // / 5.1, 512 rows of 8000 5.3 / 5.8, of 16384 6.1 / 6.4, of 20000 8.0 / 6.3, of 50304 14.8 / 11.6, 1525 rows of 16384 11.6
        // / 15.6; only beyond some 800 rows of 20000 .. 32000 are the smaller ones ahead again (1250 of 20000 10.9 / 14.0, 781 of
        // 32000 11.5 / 13.1). The histogram's workgroups cost the same however small the vocabulary; a wave's sort of a small row
        // takes longer the more keys a lane has, but 16 and more rows share a CU: 505 logits always (50000 rows of 500, top-p 1641
        // -> 145 us, 64 rows 10.4 -> 9.5), 1017 from two rows a CU on (64 rows 10.4 against 16.6, 300 rows 19.0 -> 16.8), 2041 from
        // five on (300 rows of 2000 18.9 against 31, 2000 rows 73 -> 47).  16-bit counts and kSampleSteps 16-byte chunks per thread
        // hold 65535 logits.
        if (!temperature_rows && !(temperature > 0.f)) {
            if (vocab <= 16384) sample_greedy_k<T, 256><<<rows, 256, 0, st>>>(a);
            else sample_greedy_k<T, 1024><<<rows, 1024, 0, st>>>(a);
        } else if (vocab <= 64 * 8 - 7) sample_small_k<T, 8><<<(rows + 3) / 4, 256, 0, st>>>(a, rows);
        else if (vocab <= 64 * 16 - 7 && rows > 256) sample_small_k<T, 16><<<(rows + 3) / 4, 256, 0, st>>>(a, rows);
        else if (vocab <= 64 * 32 - 7 && rows > 1024) sample_small_k<T, 32><<<(rows + 3) / 4, 256, 0, st>>>(a, rows);
        else if (vocab <= 65528) sample_tokens_k<T, false><<<rows, kSampleThreads, 0, st>>>(a);
        else sample_tokens_k<T, true><<<rows, kSampleThreads, 0, st>>>(a);
        MM_CHECK_LAUNCH();
        return MM_OK;
    });
}
