// sampling.hip - the next token of each row of logits: temperature, top-k, top-p, min-p and a given random number
// (reference: filter_logits + multinomial of megatron/text_generation_utils.py).
//
// The tokens of a row are ordered by descending logit, ties by ascending index; token t weighs w = exp((x_t - max) / temperature).
// Every filter keeps a prefix of that order, so each is a bound on the running weight: Z_k (the first k tokens), Z_p (up to the
// token whose running weight first exceeds top_p Z_k), Z_m (w >= min_p), and the token drawn is the first whose running
// weight exceeds u min(Z_k, Z_p, Z_m).  No sort is needed: a 16-bit logit has 65536 values at most, so a histogram over the
// values, in order, holds the whole distribution exactly - counts are integers, one weight per value in 64 bits - and the token is
// the j-th by index of one value.  Sums run in a fixed order: the result does not depend on scheduling, and a border of two tokens
// is off by about 1e-15 of the weight.
//
// One workgroup of 16 waves per row.  Its histogram (32768 words: a count of a non-negative value in the low half, of a negative
// one in the high half; 128 KB) fills most of a CU's LDS.  Steps: (1) the row into registers, each wave a contiguous 16th of it
// (the search by index needs that), and its largest value; (2) one LDS atomic per logit; (3) per 64 neighbouring values ("chunk")
// count and weight, one wave a chunk, empty chunks and weights below e^-50 skipped; (4) a scan over the 1024 chunks; (5) one wave
// finds the borders: 64-way search for the chunk, a scan over its 64 values; (6) the j-th match of the value found.
// Rows of more than 65535 logits (BIG) could overflow 16-bit counts: they count non-negative and negative values one after the
// other in 32 bits, re-read the row instead of keeping it, and recount a chunk when a border falls into it.
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

constexpr int kSampleThreads = 1024, kSampleWaves = 16, kChunks = 1024, kSampleSteps = 8;

// A 16-bit logit's place in descending order: non-negative b -> 0x7fff - b, negative b (sign bit set) -> b.  Two at a time.
// -0 (0x8000) becomes a value of its own next to +0 (0x7fff); they are merged where it matters.
__device__ __forceinline__ uint32_t order2(uint32_t v) { return v ^ 0x7fff7fffu ^ (((v >> 15) & 0x00010001u) * 0x7fffu); }
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

__device__ __forceinline__ double shfl_up_d(double v, int o) {
    const unsigned long long b = __double_as_longlong(v);
    const uint32_t lo = __shfl_up((uint32_t)b, o, 64), hi = __shfl_up((uint32_t)(b >> 32), o, 64);
    return __longlong_as_double(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double shfl_d(double v, int l) {
    const unsigned long long b = __double_as_longlong(v);
    const uint32_t lo = __shfl((uint32_t)b, l, 64), hi = __shfl((uint32_t)(b >> 32), l, 64);
    return __longlong_as_double(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ uint32_t scan_u(uint32_t v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(v, o, 64);
        if (lane >= o) v += x;
    }
    return v;
}
__device__ __forceinline__ double scan_d(double v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double x = shfl_up_d(v, o);
        if (lane >= o) v += x;
    }
    return v;
}

struct SampleShared {
    uint32_t hist[32768];
    double mass[kChunks];    // then its inclusive scan
    uint32_t count[kChunks];
    double wave_mass[kSampleWaves];
    uint32_t wave_count[kSampleWaves];
    int wave_min[kSampleWaves], wave_max[kSampleWaves];
    int dk, j;
    uint32_t one_chunk[64];  // BIG
};

template <typename T, bool BIG> __global__ __launch_bounds__(kSampleThreads) void sample_tokens_k(const SampleArgs a) {
    __shared__ __attribute__((aligned(16))) SampleShared sm;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, row = blockIdx.x;
    // The row as 16-byte aligned chunks: `lead` elements of the first one and the end of the last belong to no token.  (An aligned
    // chunk that holds one element of the row lies in the allocation's own 16-byte granule.)
    const u16* rp = a.logits + (int64_t)row * a.row_stride;
    const int lead = (int)(((uintptr_t)rp & 15) >> 1);
    const u32x4* base = reinterpret_cast<const u32x4*>(rp - lead);
    const int nch = (int)(((int64_t)lead + a.vocab + 7) >> 3);
    const int seg = (nch + kSampleWaves - 1) / kSampleWaves;
    const int ch0 = wave * seg, ch1 = min(ch0 + seg, nch);
    const int steps = (seg + 63) >> 6;

    u32x4 reg[BIG ? 1 : kSampleSteps];
    if constexpr (!BIG) {
#pragma unroll
        for (int s = 0; s < kSampleSteps; ++s)
            if (s < steps && ch0 + 64 * s + lane < ch1) reg[s] = base[ch0 + 64 * s + lane];
    }
    // f(place in the order, element index) for this thread's elements in ascending index
    auto each = [&](auto&& f) {
        auto chunk = [&](u32x4 v, int ch) {
            const int e0 = ch * 8 - lead;
            const bool whole = e0 >= 0 && e0 + 8 <= a.vocab;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t o = order2(v[i]);
                if (whole || (e0 + 2 * i >= 0 && e0 + 2 * i < a.vocab)) f((int)(o & 0xffffu), e0 + 2 * i);
                if (whole || (e0 + 2 * i + 1 >= 0 && e0 + 2 * i + 1 < a.vocab)) f((int)(o >> 16), e0 + 2 * i + 1);
            }
        };
        if constexpr (BIG) {
            for (int ch = ch0 + lane; ch < ch1; ch += 64) chunk(base[ch], ch);
        } else {
#pragma unroll
            for (int s = 0; s < kSampleSteps; ++s)
                if (s < steps && ch0 + 64 * s + lane < ch1) chunk(reg[s], ch0 + 64 * s + lane);
        }
    };

    const float temp = a.temperature_v ? a.temperature_v[row] : a.temperature;
    const bool greedy = !(temp > 0.f);
    auto clear_hist = [&]() {
        u32x4* h = reinterpret_cast<u32x4*>(sm.hist);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[tid + kSampleThreads * i] = u32x4{0, 0, 0, 0};
    };
    if (!greedy) clear_hist();
    int lo = 0xffff, hi = 0;
    each([&](int dk, int) {
        lo = min(lo, dk);
        hi = max(hi, dk);
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor(lo, o, 64));
        hi = max(hi, __shfl_xor(hi, o, 64));
    }
    if (lane == 0) {
        sm.wave_min[wave] = lo;
        sm.wave_max[wave] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) {
        lo = min(lo, sm.wave_min[w]);
        hi = max(hi, sm.wave_max[w]);
    }
    if (lo < plus_inf<T>() || hi > minus_inf<T>() || lo >= minus_inf<T>()) {  // a NaN, or nothing but -inf: no token
        if (tid == 0) a.out[row] = -1;
        return;
    }
    if (lo == kMinusZero) lo = kPlusZero;

    int dk = lo, j = 0;  // the token: the j-th by index of the value with this place
    if (!greedy) {
        const Weights<T> wt{lo, (double)order_value<T>(lo), 1.0 / (double)temp};
        // values below max - 50 T weigh less than 2^-72 each: nothing of them reaches a 64-bit sum that holds the largest's 1
        const float xlow = (float)(wt.xmax - 50.0 * (double)temp);
        int dlow = minus_inf<T>();
        if (xlow > -INFINITY) {
            const u16 b = from_f32<T>(xlow);
            dlow = min(dlow, ((b & 0x8000) ? (int)b : 0x7fff - (int)b) + 1);
        }
        const int clo = lo >> 6, chi = dlow >> 6;
        sm.count[tid] = 0;
        sm.mass[tid] = 0.0;
        auto chunk_sums = [&](int first, int last, auto&& counts) {  // chunks first .. last: one wave each
            for (int c = first + wave; c <= last; c += kSampleWaves) {
                const uint32_t n = counts(c);
                if (__ballot(n != 0) == 0) continue;
                uint32_t cn = n;
                double m = n ? (double)n * wt.at(64 * c + lane) : 0.0;
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) {
                    cn += __shfl_xor(cn, o, 64);
                    const unsigned long long b = __double_as_longlong(m);
                    const uint32_t l = __shfl_xor((uint32_t)b, o, 64), h = __shfl_xor((uint32_t)(b >> 32), o, 64);
                    m += __longlong_as_double(((unsigned long long)h << 32) | l);
                }
                if (lane == 0) {
                    sm.count[c] = cn;
                    sm.mass[c] = m;
                }
            }
        };
        auto resident = [&](int c) -> uint32_t { return (sm.hist[((c & 511) << 6) + lane] >> (c < 512 ? 0 : 16)) & 0xffffu; };
        if constexpr (!BIG) {
            each([&](int d, int) { atomicAdd(&sm.hist[d & 0x7fff], d < 0x8000 ? 1u : 0x10000u); });
            __syncthreads();
            if (tid == 0) {  // -0 is +0: word 0x7fff low half takes word 0 high half
                const uint32_t z = sm.hist[0] >> 16;
                sm.hist[0] &= 0xffffu;
                sm.hist[kPlusZero] += z;
            }
            __syncthreads();
            chunk_sums(clo, chi, resident);
        } else {
            for (int half = 0; half < 2; ++half) {
                if (half == 1) {
                    __syncthreads();
                    clear_hist();
                    __syncthreads();
                }
                each([&](int d, int) {
                    if (d == kMinusZero) d = kPlusZero;
                    if ((d >> 15) == half) atomicAdd(&sm.hist[d & 0x7fff], 1u);
                });
                __syncthreads();
                chunk_sums(max(clo, 512 * half), min(chi, 512 * half + 511), [&](int c) -> uint32_t { return sm.hist[((c & 511) << 6) + lane]; });
            }
        }
        __syncthreads();
        {   // inclusive scans over the chunks
            uint32_t c = scan_u(sm.count[tid], lane);
            double m = scan_d(sm.mass[tid], lane);
            if (lane == 63) {
                sm.wave_count[wave] = c;
                sm.wave_mass[wave] = m;
            }
            __syncthreads();
            double bm = 0.0;
            uint32_t bc = 0;
            for (int w = 0; w < wave; ++w) {
                bc += sm.wave_count[w];
                bm += sm.wave_mass[w];
            }
            sm.count[tid] = c + bc;
            sm.mass[tid] = m + bm;
            __syncthreads();
        }

        // Borders.  One wave (BIG: every wave alike, because recounting a chunk takes the whole workgroup).
        if (BIG || wave == 0) {
            auto counts = [&](int c) -> uint32_t {
                if constexpr (!BIG) return resident(c);
                __syncthreads();
                if (tid < 64) sm.one_chunk[tid] = 0;
                __syncthreads();
                each([&](int d, int) {
                    if (d == kMinusZero) d = kPlusZero;
                    if ((d >> 6) == c) atomicAdd(&sm.one_chunk[d & 63], 1u);
                });
                __syncthreads();
                return sm.one_chunk[lane];
            };
            auto first_chunk = [&](auto&& pred) -> int {  // the first chunk with pred(inclusive scan); pred holds from there on
                uint64_t b = __ballot(pred(16 * lane + 15));
                const int blk = b ? __builtin_ctzll(b) : 63;
                b = __ballot(lane < 16 && pred(16 * blk + lane));
                return 16 * blk + (b ? __builtin_ctzll(b) : 15);
            };
            // the first token whose running weight exceeds t: value, how many tokens of that value are ahead of it, and the running
            // weight up to and with it
            struct Found {
                int dk, j;
                double upto;
            };
            auto find = [&](double t) -> Found {
                const int c = first_chunk([&](int i) { return sm.mass[i] > t; });
                const double ahead = c ? sm.mass[c - 1] : 0.0;
                const uint32_t n = counts(c);
                const double w = n ? wt.at(64 * c + lane) : 0.0;
                const double incl = ahead + scan_d((double)n * w, lane);
                uint64_t any = __ballot(n != 0);
                if (!any) return Found{lo, 0, 1.0};  // rounding put t between two chunks' sums
                const uint64_t over = __ballot(n != 0 && incl > t);
                const int l = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
                const double before = incl - (double)n * w;
                double jj = floor((t - before) / w);
                jj = fmin(fmax(jj, 0.0), (double)(n ? n - 1 : 0));
                if (!over) jj = (double)(n ? n - 1 : 0);
                const double up = before + (jj + 1.0) * w;
                return Found{64 * c + l, __shfl((int)jj, l, 64), shfl_d(up, l)};
            };
            const double total = sm.mass[kChunks - 1];
            double z = total;
            const int k = a.top_k_v ? a.top_k_v[row] : a.top_k;
            if (k > 0 && (uint32_t)k < sm.count[kChunks - 1]) {
                const int c = first_chunk([&](int i) { return sm.count[i] >= (uint32_t)k; });
                const uint32_t n = counts(c);
                const double w = n ? wt.at(64 * c + lane) : 0.0;
                const uint32_t ci = (c ? sm.count[c - 1] : 0u) + scan_u(n, lane);
                const double mi = (c ? sm.mass[c - 1] : 0.0) + scan_d((double)n * w, lane);
                const uint64_t over = __ballot(n != 0 && ci >= (uint32_t)k);
                const int l = over ? __builtin_ctzll(over) : 63;
                z = fmin(z, shfl_d(mi - (double)(ci - (uint32_t)k) * w, l));
            }
            const float p = a.top_p_v ? a.top_p_v[row] : a.top_p, mp = a.min_p_v ? a.min_p_v[row] : a.min_p;
            double zp = z;
            if (p > 0.f && p < 1.f) zp = fmin(zp, find((double)p * z).upto);
            if (mp > 0.f) {
                // the first value whose weight is below min_p: 64-way search in the order
                const double floor_w = fmin((double)mp, 1.0);
                int from = lo, span = 65536 - lo;
                while (span > 0) {
                    const int st = (span + 63) >> 6, at = from + lane * st + st - 1;
                    const bool kept = lane * st + st - 1 < span && wt.at(min(at, minus_inf<T>())) >= floor_w;
                    const int g = __popcll(__ballot(kept));
                    from += g * st;
                    span -= g * st;
                    if (st == 1) break;
                    span = min(span, st);
                }
                const int c = min(from, 65535) >> 6;
                const uint32_t n = counts(c);
                const double w = n ? wt.at(64 * c + lane) : 0.0;
                const double mi = scan_d(64 * c + lane < from ? (double)n * w : 0.0, lane);
                zp = fmin(zp, (c ? sm.mass[c - 1] : 0.0) + shfl_d(mi, 63));
            }
            zp = fmax(zp, 1.0);
            double t = (double)a.u[row] * zp;
            if (!(t < zp)) t = __longlong_as_double(__double_as_longlong(zp) - 1);  // u of 1 or more: the last token kept
            const Found f = find(t);
            if (BIG || lane == 0) {
                sm.dk = f.dk;
                sm.j = f.j;
            }
        }
        __syncthreads();
        dk = sm.dk;
        j = sm.j;
    }

    // the j-th token with this value, by index: matches per wave, then per 64-lane step, then per lane
    auto is_match = [&](int d) { return d == dk || (dk == kPlusZero && d == kMinusZero); };
    uint32_t mine = 0;
    each([&](int d, int) { mine += is_match(d) ? 1u : 0u; });
    uint32_t tot = mine;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) tot += __shfl_xor(tot, o, 64);
    __syncthreads();
    if (lane == 0) sm.wave_count[wave] = tot;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; ++w) before += sm.wave_count[w];
    if ((uint32_t)j < before || (uint32_t)j >= before + tot) return;  // another wave has it
    uint32_t left = (uint32_t)j - before;
    for (int s = 0; s < steps; ++s) {
        const int ch = ch0 + 64 * s + lane;
        uint32_t bits = 0;
        int e0 = 0;
        if (ch < ch1) {
            const u32x4 v = base[ch];
            e0 = ch * 8 - lead;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t o = order2(v[i >> 1]);
                const int d = (int)((i & 1) ? o >> 16 : o & 0xffffu);
                if (e0 + i >= 0 && e0 + i < a.vocab && is_match(d)) bits |= 1u << i;
            }
        }
        const uint32_t incl = scan_u(__popc(bits), lane), sum = __shfl(incl, 63, 64);
        if (left >= sum) {
            left -= sum;
            continue;
        }
        uint32_t excl = incl - __popc(bits);
        if (left >= excl && left < incl) {
            for (; excl < left; ++excl) bits &= bits - 1;
            a.out[row] = e0 + __builtin_ctz(bits);
        }
        return;
    }
}

}  // namespace mm

using namespace mm;

extern "C" int mm_sample_tokens(int64_t* tokens, const void* logits, int64_t row_stride, const float* u, int rows, int vocab,
                                float temperature, const float* temperature_rows, int top_k, const int32_t* top_k_rows, float top_p,
                                const float* top_p_rows, float min_p, const float* min_p_rows, int dtype, void* stream) {
    const char* fn = "mm_sample_tokens";
    MM_CHECK_ARG(rows >= 0 && vocab > 0 && vocab < 1 << 30, "%s: rows=%d vocab=%d out of range", fn, rows, vocab);
    if (rows == 0) return MM_OK;
    MM_CHECK_ARG(tokens && logits && u, "%s: null pointer", fn);
    MM_CHECK_ARG(((uintptr_t)logits & 1) == 0, "%s: logits must be 2-byte aligned", fn);
    SampleArgs a{(const u16*)logits, row_stride, u, tokens, vocab, temperature, top_p, min_p, top_k, temperature_rows, top_p_rows,
                 min_p_rows, top_k_rows};
    hipStream_t st = (hipStream_t)stream;
    return dispatch_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        // 16-bit counts and kSampleSteps 16-byte chunks per thread hold 65535 logits
        if (vocab <= 65528) sample_tokens_k<T, false><<<rows, kSampleThreads, 0, st>>>(a);
        else sample_tokens_k<T, true><<<rows, kSampleThreads, 0, st>>>(a);
        MM_CHECK_LAUNCH();
        return MM_OK;
    });
}
