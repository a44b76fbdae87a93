// Token sampling: temperature, top-k, top-p, min-p and a given uniform number a row.
//
// Weights w = exp((x - max) / T) are held as 64-bit fixed point (2^-44 for vocabularies of 2^18, finer for
// smaller ones: a sum stays below 2^63): integer sums have no order, and a row's result is the same bits on every
// run.  A slice's sums are taken against its own maximum, to 2^-51 of it, and brought to the row's as a whole, which
// rounds them to half a unit; a slice whose largest token rounds to nothing has none.  No row is sorted: the last
// kept token is found from a histogram over the distance to the maximum, then from the tokens of the one bin that
// holds it.
//
// sample_slice_kernel, a workgroup for 8192 tokens of a row, reads the logits once into registers: the slice's
// maximum, and against it the tokens' weights, their sum, the histogram (256 bins of 1/8 in x / T on a grid that
// all slices share) and the tokens' indexes, sorted by bin as they are counted.  sample_row_kernel, a workgroup a
// row: the slices' sums brought to the row's maximum (a slice that holds the maximum exactly, so that equal logits
// stay equal weights), the bin of the last kept token, its tokens by the slices' lists into LDS, the border among
// them, and the sums along the index down to the token.
//
// Bound: the slices by the bytes of the logits where a row is not filtered (256 rows of 131072 in fp32: 36 us for
// 134 MB), by fp64 arithmetic, the histogram's atomics and the lists' stores side by side where it is (65 us); the
// rows by a chain of some twelve steps that wait for each other (16 to 38 us, whatever the rows).  The lists
// cost the slices 2 bytes a token and save the rows a second look at their logits: 48 rows with all filters 69
// -> 57 us, 64 rows whose bin holds more than LDS does 186 -> 84, 256 rows 107 -> 104.
#include "launch.h"
#include "sample.h"

namespace pgmoe {

constexpr int kSlice = 8192;                   // tokens of a slice: 16 a thread, four workgroups a CU
constexpr int kThreads = 512;                  // 1024 for a row: 26.0 us for one row (25.1 with 512), 256 rows 106 (104)
constexpr int kWaves = kThreads / 64;
constexpr int kPer = kSlice / kThreads;        // tokens of a thread
constexpr int kBins = 256;                     // of the distance; the last holds all that lies further
constexpr int kCopies = 4;                     // of a slice's histogram, by lane: equal bins of a wave meet less often
constexpr float kPerNat = 8.0f;                // bins a unit of x / T
constexpr int kDigitBits = 9;                  // of a level of the descent
constexpr int kDigits = 1 << kDigitBits;
constexpr int kList = 7168;                    // tokens of one bin that fit LDS, two workgroups a CU
constexpr int kHeld = 12;                      // histogram entries that a thread keeps: 24 slices
constexpr int kMaxSlices = kMaxVocab / kSlice;

struct Slice {
    uint64_t sum;  // of weights against the slice's maximum
    float max;
    int first;  // lowest index of the maximum
};
struct Layout {
    int64_t slices, cnt, wgt, off, idx, total;
};
static __host__ __device__ Layout layout(int rows, int vocab) {
    const int64_t n = (int64_t)rows * ((vocab + kSlice - 1) / kSlice);
    Layout o;
    o.slices = 0;
    o.wgt = (n * (int64_t)sizeof(Slice) + 255) / 256 * 256;
    o.cnt = o.wgt + n * kBins * 8;
    o.off = o.cnt + n * kBins * 4;
    o.idx = o.off + n * kBins * 2;
    o.total = o.idx + n * kSlice * 2;
    return o;
}

// A monotone 32-bit key: a > b as floats exactly if key(a) > key(b); +0 and -0 share one.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Eight consecutive logits as they lie in memory.
template <int DT>
struct Eight {
    static constexpr int SZ = DT == PGMOE_DT_F32 ? 4 : 2;
    uint4 v[SZ / 2];
    // aligned and inside the row: straight loads, nothing that waits for them
    __device__ __forceinline__ void load(const void* logits, int64_t at) {
        const uint4* p = (const uint4*)((const uint8_t*)logits + at * SZ);
#pragma unroll
        for (int i = 0; i < SZ / 2; ++i) v[i] = p[i];
    }
    // any alignment; -inf behind the last
    __device__ __forceinline__ void load_checked(const SampleArgs& A, int64_t row, int i) {
        uint32_t* w = (uint32_t*)v;
        if constexpr (DT == PGMOE_DT_F32) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                w[j] = i + j < A.vocab ? ((const uint32_t*)A.logits)[row + i + j] : 0xff800000u;
        } else {
            constexpr uint32_t out = DT == PGMOE_DT_F16 ? 0xfc00 : 0xff80;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t a = i + 2 * j < A.vocab ? ((const uint16_t*)A.logits)[row + i + 2 * j] : out;
                const uint32_t b = i + 2 * j + 1 < A.vocab ? ((const uint16_t*)A.logits)[row + i + 2 * j + 1] : out;
                w[j] = a | b << 16;
            }
        }
    }
    __device__ __forceinline__ float operator[](int j) const {
        const uint32_t* w = (const uint32_t*)v;
        if constexpr (DT == PGMOE_DT_F32)
            return __builtin_bit_cast(float, w[j]);
        else if constexpr (DT == PGMOE_DT_F16)
            return h2f((uint16_t)(w[j >> 1] >> (16 * (j & 1))));
        else
            return __builtin_bit_cast(float, j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
    }
};
template <int DT>
__device__ __forceinline__ float one_logit(const SampleArgs& A, int64_t at) {
    if constexpr (DT == PGMOE_DT_F32)
        return ((const float*)A.logits)[at];
    else if constexpr (DT == PGMOE_DT_F16)
        return h2f(((const uint16_t*)A.logits)[at]);
    else
        return __builtin_bit_cast(float, (uint32_t)((const uint16_t*)A.logits)[at] << 16);
}
// A thread's tokens of slice s (kPer / 8 times eight), -inf where there are none.
template <int DT>
__device__ __forceinline__ void load_slice(const SampleArgs& A, int64_t row, int s, bool aligned, Eight<DT> (&x)[kPer / 8]) {
    if (aligned && (s + 1) * kSlice <= A.vocab) {
#pragma unroll
        for (int j = 0; j < kPer / 8; ++j) x[j].load(A.logits, row + s * kSlice + (j * kThreads + (int)threadIdx.x) * 8);
    } else {
#pragma unroll
        for (int j = 0; j < kPer / 8; ++j) x[j].load_checked(A, row, s * kSlice + (j * kThreads + (int)threadIdx.x) * 8);
    }
}
template <int DT>
__device__ __forceinline__ bool row_aligned(const SampleArgs& A, int64_t row) {
    return (((uintptr_t)A.logits + row * Eight<DT>::SZ) & 15) == 0;
}

// The settings of a row.
struct Settings {
    double inv_t, top_p, min_p;
    uint64_t top_k;
    bool greedy, filters;
    __device__ Settings(const SampleArgs& A, int r) {
        const double t = A.P.temperatures ? (double)A.P.temperatures[r] : A.P.temperature;
        top_p = A.P.top_ps ? (double)A.P.top_ps[r] : A.P.top_p;
        min_p = A.P.min_ps ? (double)A.P.min_ps[r] : A.P.min_p;
        const int k = A.P.top_ks ? A.P.top_ks[r] : A.P.top_k;
        greedy = !(t > 0.0);
        inv_t = greedy ? 1.0 : 1.0 / t;
        top_k = k > 0 && k < A.vocab ? (uint64_t)k : ~0ull;
        filters = !greedy && (top_k != ~0ull || top_p < 1.0 || min_p > 0.0);
    }
};

// w = exp((x - top) / T) = 2^(q / 256) e^g with |g| <= ln 2 / 512: a table of 256 powers and four terms of the
// series, relative error 2^-50; fixed point by adding 2^52.  No branch: several tokens are under way at a time.
constexpr int kPowers = 256;
struct Weigh {
    const double* powers;  // 2^(i / 256), LDS
    float top;
    double k;  // 256 log2(e) / T
    int shift;
    __device__ __forceinline__ Weigh(const double* powers_, float top_, double inv_t, int shift_)
        : powers(powers_), top(top_), k(inv_t * 369.32993046757464), shift(shift_) {}
    // 2^shift w; 2^(shift - 64) for less than that, -inf, NaN, and everything beside +inf
    __device__ __forceinline__ double scaled(float x, int shift_) const {
        const double t = x == top ? 0.0 : __builtin_fmax(((double)x - (double)top) * k, -16384.0);
        const double q = __builtin_rint(t);
        const double g = (t - q) * 0.0027076061740622863;
        double p = __builtin_fma(g, 1.0 / 24.0, 1.0 / 6.0);
        p = __builtin_fma(p, g, 0.5);
        p = __builtin_fma(p, g, 1.0);
        p = __builtin_fma(p, g, 1.0);
        const int n = (int)q;
        return __builtin_ldexp(powers[n & (kPowers - 1)] * p, (n >> 8) + shift_);
    }
    __device__ __forceinline__ double w(float x) const { return scaled(x, 0); }
    __device__ __forceinline__ uint64_t fix(float x) const {
        const double v = scaled(x, shift) + 4503599627370496.0;
        return __builtin_bit_cast(uint64_t, v) & 0xfffffffffffffull;
    }
};
__device__ __forceinline__ void fill_powers(double* p, int tid) {
    if (tid < kPowers) p[tid] = exp2((double)tid / kPowers);
}

// The grid of the histogram: bins of 1/8 in x / T, counted down from the bin of `top`.
struct Grid {
    float g, top, at;
    __device__ __forceinline__ Grid(float top_, double inv_t) : g((float)inv_t * kPerNat), top(top_), at(floorf(top_ * g)) {}
    __device__ __forceinline__ int bin(float x) const {
        const float d = at - floorf(x * g);
        return x == top ? 0 : d < (float)(kBins - 1) ? (int)d : kBins - 1;  // NaN: the last
    }
};

__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor((unsigned long long)v, d);
    return v;
}

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) { return __shfl((unsigned long long)v, lane); }
// Sum over the lanes below this one, and over all.
__device__ __forceinline__ uint64_t wave_before(uint64_t v, uint64_t* all) {
    const int lane = threadIdx.x & 63;
    uint64_t x = v;
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t p = __shfl_up((unsigned long long)x, d);
        if (lane >= d) x += p;
    }
    *all = shfl64(x, 63);
    return x - v;
}

template <int DT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(8))) void sample_slice_kernel(const SampleArgs A) {
    constexpr int G = 8, N = kPer / G;  // groups of 8 tokens a thread
    __shared__ __attribute__((aligned(16))) uint32_t cnt[kBins * kCopies];
    __shared__ unsigned long long wgt[kBins * kCopies];
    __shared__ double powers[kPowers];
    __shared__ float s_max[kWaves];
    __shared__ uint64_t s_sum[kWaves];
    __shared__ __attribute__((aligned(16))) uint16_t off[kBins * kCopies];  // where a bin's tokens begin in idx
    __shared__ int s_all;
    __shared__ __attribute__((aligned(16))) uint16_t idx[kSlice];  // the tokens by bin
    __shared__ int s_first;
    const int r = blockIdx.x, slice = blockIdx.y, tid = threadIdx.x, lane = tid & 63, base = slice * kSlice;
    const int64_t row = (int64_t)r * A.row_stride;
    Eight<DT> x[N];
    load_slice<DT>(A, row, slice, row_aligned<DT>(A, row), x);
    const Settings S(A, r);
    fill_powers(powers, tid);
    if (tid == 0) s_first = 0x7fffffff;
    for (int i = tid; i < kBins * kCopies; i += kThreads) cnt[i] = 0, wgt[i] = 0;
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < G; ++e) mx = fmaxf(mx, x[j][e]);
    mx = wave_max(mx);
    if (lane == 0) s_max[tid >> 6] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) mx = fmaxf(mx, s_max[i]);

    const int64_t at = (int64_t)r * gridDim.y + slice;
    const Layout o = layout(A.rows, A.vocab);
    Slice* out = (Slice*)((uint8_t*)A.ws + o.slices) + at;
    if (S.greedy || mx == -INFINITY) {
        int first = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < G; ++e)
                if (x[j][e] == mx) {
                    const int i = base + (j * kThreads + tid) * G + e;
                    first = i < first ? i : first;
                }
        if (first != 0x7fffffff) atomicMin(&s_first, first);
        __syncthreads();
        if (tid == 0) *out = Slice{0, mx, s_first};
    } else {
        const Weigh W(powers, mx, S.inv_t, A.shift);
        const Grid g(mx, S.inv_t);
        uint64_t sum = 0;
        uint32_t rank[N][G];  // of a token within its bin, in no order, beside the bin; 0xffff: no token
        if (S.filters) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                uint32_t b[G];
#pragma unroll
                for (int e = 0; e < G; ++e) b[e] = g.bin(x[j][e]) * kCopies + lane % kCopies;
#pragma unroll
                for (int e = 0; e < G; ++e) {
                    rank[j][e] = 0xffff;
                    if (x[j][e] > -INFINITY) rank[j][e] = atomicAdd(&cnt[b[e]], 1u);
                }
#pragma unroll
                for (int e = 0; e < G; ++e) rank[j][e] |= b[e] << 16;
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            uint64_t f[G];
#pragma unroll
            for (int e = 0; e < G; ++e) f[e] = W.fix(x[j][e]), sum += f[e];
            if (S.filters) {
#pragma unroll
                for (int e = 0; e < G; ++e)
                    if (f[e]) atomicAdd(&wgt[rank[j][e] >> 16], (unsigned long long)f[e]);
            }
        }
        sum = wave_sum(sum);
        if (lane == 0) s_sum[tid >> 6] = sum;
        __syncthreads();
        if (tid == 0) {
            sum = 0;
            for (int i = 0; i < kWaves; ++i) sum += s_sum[i];
            *out = Slice{sum, mx, 0};
        }
        if (S.filters) {
            if (tid < 64) {
                constexpr int B = kBins * kCopies / 64;
                uint32_t n[B], own = 0;
#pragma unroll
                for (int i = 0; i < B; ++i) n[i] = cnt[lane * B + i], own += n[i];
                uint32_t at = own;
                for (int d = 1; d < 64; d <<= 1) {
                    const uint32_t p = __shfl_up(at, d);
                    if (lane >= d) at += p;
                }
                if (lane == 63) s_all = (int)at;
                at -= own;
#pragma unroll
                for (int i = 0; i < B; ++i) off[lane * B + i] = (uint16_t)at, at += n[i];
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < N; ++j)
#pragma unroll
                for (int e = 0; e < G; ++e)
                    if ((rank[j][e] & 0xffff) != 0xffff)
                        idx[off[rank[j][e] >> 16] + (rank[j][e] & 0xffff)] = (uint16_t)((j * kThreads + tid) * G + e);
            __syncthreads();
            uint4* to = (uint4*)((uint16_t*)((uint8_t*)A.ws + o.idx) + at * kSlice);
            for (int i = tid; i * 8 < s_all; i += kThreads) to[i] = ((const uint4*)idx)[i];
        }
    }
    if (S.filters) {
        if (mx == -INFINITY) {
            for (int i = tid; i < kBins * kCopies; i += kThreads) off[i] = 0;
            __syncthreads();
        }
        if (tid < kBins) {
            uint32_t c = 0;
            uint64_t w = 0;
#pragma unroll
            for (int i = 0; i < kCopies; ++i) c += cnt[tid * kCopies + i], w += wgt[tid * kCopies + i];
            ((uint32_t*)((uint8_t*)A.ws + o.cnt))[at * kBins + tid] = c;
            ((uint64_t*)((uint8_t*)A.ws + o.wgt))[at * kBins + tid] = w;
            ((uint16_t*)((uint8_t*)A.ws + o.off))[at * kBins + tid] = off[tid * kCopies];
        }
    }
}

// The least key above `out` of which `in` (which is true, as all above the border are) holds: a wave tries 64 keys
// around `near`, and bisects where the border lies elsewhere.
template <class In>
__device__ __forceinline__ uint32_t first_that(uint32_t near, uint32_t out, uint32_t top, In&& in) {
    const int lane = threadIdx.x & 63;
    if (near > out + 32 && near < top && top - near > 32) {
        const uint64_t m = __ballot(in(near - 32 + lane));
        if (m && !(m & 1)) return near - 32 + __builtin_ctzll(m);
    }
    while (top - out > 1) {
        const uint32_t mid = out + (top - out) / 2;
        (in(mid) ? top : out) = mid;
    }
    return top;
}

// Where the order of the tokens leaves the kept ones, among N places (bins or digits) a lane of one wave, in
// order: the first place that is not kept whole, with the count and weight before it; -1: all are.
template <int N>
struct Border {
    int place;
    uint64_t cb, wb, all;
    template <class Stop>
    __device__ __forceinline__ Border(const uint64_t (&c)[N], const uint64_t (&w)[N], uint64_t cb0, uint64_t wb0,
                                      Stop&& stop) {
        const int lane = threadIdx.x & 63;
        uint64_t cs = 0, ws = 0, unused;
#pragma unroll
        for (int i = 0; i < N; ++i) cs += c[i], ws += w[i];
        uint64_t c1 = cb0 + wave_before(cs, &unused), w1 = wb0 + wave_before(ws, &all);
        int at = -1;
        uint64_t ca = 0, wa = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (at < 0 && c[i] && stop(lane * N + i, c1 + c[i], w1 + w[i], all)) at = lane * N + i, ca = c1, wa = w1;
            c1 += c[i], w1 += w[i];
        }
        const uint64_t who = __ballot(at >= 0);
        const int l = who ? __builtin_ctzll(who) : 0;
        place = who ? __shfl(at, l) : -1;
        cb = shfl64(ca, l), wb = shfl64(wa, l);
    }
};

// Two workgroups a CU: 1024 rows of 32000 take 110 us in all, 125 with the registers of one (one row 25.3, 25.0).
template <int DT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4))) void sample_row_kernel(const SampleArgs A) {
    constexpr int kLaneSlices = kMaxSlices / 64;
    __shared__ uint2 few[64];
    __shared__ uint2 list[kList];  // (key, index) of the tokens of the last kept one's bin
    __shared__ unsigned long long wsum[2][kDigits];
    __shared__ uint32_t cnt[2][kDigits];
    __shared__ unsigned long long slice_w[kMaxSlices];  // what a slice keeps
    __shared__ uint32_t slice_n[kMaxSlices];            // its tokens of key `edge`
    __shared__ double slice_s[kMaxSlices];  // the slice's weights to the row's: exp((its max - max) / T)
    __shared__ float slice_d[kMaxSlices];   // the slice's bins to the row's
    __shared__ double powers[kPowers];
    __shared__ uint64_t red[kWaves][2];
    __shared__ int s_n;
    __shared__ uint32_t s_lo, s_hi;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, V = A.vocab;
    const int slices = (V + kSlice - 1) / kSlice;
    const int64_t row = (int64_t)r * A.row_stride;
    const Layout o = layout(A.rows, V);
    const Slice* sl = (const Slice*)((uint8_t*)A.ws + o.slices) + (int64_t)r * slices;
    const uint32_t* hc = (const uint32_t*)((uint8_t*)A.ws + o.cnt) + (int64_t)r * slices * kBins;
    const uint64_t* hw = (const uint64_t*)((uint8_t*)A.ws + o.wgt) + (int64_t)r * slices * kBins;
    const Settings S(A, r);
    const bool aligned = row_aligned<DT>(A, row);

    // every wave holds the slices' maxima, so that the row's needs no meeting
    float mx = -INFINITY;
    int first = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < kLaneSlices; ++i)
        if (64 * i + lane < slices) mx = fmaxf(mx, sl[64 * i + lane].max);
    uint32_t hold_c[kHeld];
    uint64_t hold_w[kHeld];
    if (S.filters) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int e = i * kThreads + tid;
            hold_c[i] = e < slices * kBins ? hc[e] : 0;
            hold_w[i] = e < slices * kBins ? hw[e] : 0;
        }
    }
    fill_powers(powers, tid);
    mx = wave_max(mx);
    if (mx == -INFINITY) {
        if (tid == 0) {
            A.token[r] = -1;
            if (A.logprob) A.logprob[r] = -INFINITY;
        }
        return;
    }
    if (S.greedy) {
#pragma unroll
        for (int i = 0; i < kLaneSlices; ++i)
            if (64 * i + lane < slices && sl[64 * i + lane].max == mx) {
                const int f = sl[64 * i + lane].first;
                first = f < first ? f : first;
            }
        for (int d = 32; d; d >>= 1) {
            const int f = __shfl_xor(first, d);
            first = f < first ? f : first;
        }
        if (tid == 0) {
            A.token[r] = first;
            if (A.logprob) A.logprob[r] = 0.0f;
        }
        return;
    }
    const Weigh W(powers, mx, S.inv_t, A.shift);
    const Grid g(mx, S.inv_t);
    auto to_row = [&](uint64_t w, int s) { return slice_s[s] == 1.0 ? w : (uint64_t)llrint((double)w * slice_s[s]); };
    for (int i = tid; i < kDigits; i += kThreads) cnt[0][i] = cnt[1][i] = 0, wsum[0][i] = wsum[1][i] = 0;
    if (tid == 0) s_n = 0, s_lo = 0xffffffffu, s_hi = 0;
    __syncthreads();  // the powers
    if (tid < slices) {
        const Slice m = sl[tid];
        const bool top = m.max == mx;
        // A slice whose largest logit has no weight has none, whatever its tokens' small ones add up to: where a slice
        // has a sum, one token of it at least can be drawn.
        const double f = top ? 1.0 : W.fix(m.max) ? W.w(m.max) : 0.0;
        slice_s[tid] = f;
        slice_d[tid] = top ? 0.0f : g.at - floorf(m.max * g.g);
        slice_w[tid] = S.filters ? 0 : f == 1.0 ? m.sum : (uint64_t)llrint((double)m.sum * f);
        slice_n[tid] = 0;
    }
    __syncthreads();

    // The last kept token: key `edge`, of which the first `ties` in index order are kept; every greater key is.
    uint32_t edge = 0;
    uint64_t ties = 0;
    if (S.filters) {
        auto row_bin = [&](int s, int b) {
            const float d = (float)b + slice_d[s];
            return d < (float)(kBins - 1) ? (int)d : kBins - 1;
        };
        auto entries = [&](auto&& take) {  // the slices' histograms, entry by entry
#pragma unroll
            for (int i = 0; i < kHeld; ++i)
                if (hold_c[i]) take(i * kThreads + tid, hold_c[i], hold_w[i]);
            for (int e = kHeld * kThreads + tid; e < slices * kBins; e += kThreads)
                if (hc[e]) take(e, hc[e], hw[e]);
        };
        entries([&](int e, uint32_t c, uint64_t w) {
            const int s = e / kBins, b = row_bin(s, e % kBins);
            atomicAdd(&cnt[0][b], c);
            atomicAdd(&wsum[0][b], (unsigned long long)to_row(w, s));
        });
        // the least key that min_p keeps: the border of w >= min_p, near its logarithm
        uint32_t least = 0;
        int least_bin = kBins;
        if (S.min_p >= 1.0) {
            least = key_of(mx) + (S.min_p > 1.0);
            least_bin = 0;
        } else if (S.min_p > 0.0) {
            least = first_that(key_of((float)((double)mx + log(S.min_p) / S.inv_t)), key_of(-INFINITY), key_of(mx),
                               [&](uint32_t k) { return W.w(of_key(k)) >= S.min_p; });
            least_bin = g.bin(of_key(least));
        }
        __syncthreads();
        uint64_t target = ~0ull, cb, wb;
        int bin;
        {
            constexpr int N = kBins / 64;
            uint64_t c[N], w[N];
#pragma unroll
            for (int i = 0; i < N; ++i) c[i] = cnt[0][lane * N + i], w[i] = wsum[0][lane * N + i];
            auto aim = [&](uint64_t all) {
                return S.top_p < 1.0 ? (S.top_p > 0.0 ? (uint64_t)ceil(S.top_p * (double)all) : 0) : ~0ull;
            };
            const Border<N> B(c, w, 0, 0, [&](int b, uint64_t ce, uint64_t we, uint64_t all) {
                return ce >= S.top_k || we >= aim(all) || b >= least_bin;
            });
            target = aim(B.all);
            bin = B.place, cb = B.cb, wb = B.wb;
        }
        const bool some = bin >= 0;
        const int cnt_bin = some ? (int)cnt[0][bin] : 0;
        const bool light = some && cb && !wsum[0][bin];  // which of its tokens are kept changes nothing: none is
        const bool listed = cnt_bin <= kList;
        __syncthreads();
        for (int i = tid; i < kBins; i += kThreads) cnt[0][i] = 0, wsum[0][i] = 0;
        // what each slice keeps above the bin
        entries([&](int e, uint32_t c, uint64_t w) {
            const int s = e / kBins, b = row_bin(s, e % kBins);
            if (!some || b < bin) atomicAdd(&slice_w[s], (unsigned long long)to_row(w, s));
        });
        __syncthreads();
        if (some) {
            // A slice's list has the bin's tokens in a row, from `first`, n of them: a lane knows kLaneSlices slices,
            // a wave reads every kWaves-th, with the `before` earlier slices' ones numbered first
            int n[kLaneSlices], first[kLaneSlices], before;
            {
                uint64_t own = 0, unused;
#pragma unroll
                for (int i = 0; i < kLaneSlices; ++i) {
                    const int s = lane * kLaneSlices + i;
                    n[i] = first[i] = 0;
                    if (s < slices) {
                        const uint32_t* sc = hc + s * kBins;
                        const uint16_t* so = (const uint16_t*)((uint8_t*)A.ws + o.off) + ((int64_t)r * slices + s) * kBins;
                        const float b = (float)bin - slice_d[s];
                        if (bin == kBins - 1) {  // all that lies that far
                            first[i] = so[b > 0.0f ? (int)b : 0];
                            n[i] = so[kBins - 1] + (int)sc[kBins - 1] - first[i];
                        } else if (b >= 0.0f) {
                            first[i] = so[(int)b];
                            n[i] = (int)sc[(int)b];
                        }
                    }
                    own += n[i];
                }
                before = (int)wave_before(own, &unused);
            }
            auto read_bin = [&](auto&& take) {  // the bin's tokens from memory: number, key, index
                for (int s = tid >> 6; s < slices; s += kWaves) {
                    const int l = s / kLaneSlices;
                    int at = __shfl(before, l), ns = 0, fs = 0;
#pragma unroll
                    for (int i = 0; i < kLaneSlices; ++i) {
                        const int ni = __shfl(n[i], l), fi = __shfl(first[i], l);
                        at += i < s % kLaneSlices ? ni : 0;
                        if (i == s % kLaneSlices) ns = ni, fs = fi;
                    }
                    const uint16_t* from = (const uint16_t*)((uint8_t*)A.ws + o.idx) + ((int64_t)r * slices + s) * kSlice + fs;
                    constexpr int U = 8;  // of them on their way at a time
                    for (int k = lane; k < ns; k += 64 * U) {
                        int t[U];
                        float y[U];
#pragma unroll
                        for (int q = 0; q < U; ++q) t[q] = s * kSlice + from[k + 64 * q < ns ? k + 64 * q : k];
#pragma unroll
                        for (int q = 0; q < U; ++q) y[q] = one_logit<DT>(A, row + t[q]);
#pragma unroll
                        for (int q = 0; q < U; ++q)
                            if (k + 64 * q < ns) take(at + k + 64 * q, key_of(y[q]), t[q]);
                    }
                }
            };
            auto meet = [&](uint32_t l, uint32_t h) {  // the least and greatest key of the workgroup
                for (int d = 32; d; d >>= 1) {
                    const uint32_t p = __shfl_xor(l, d), q = __shfl_xor(h, d);
                    l = p < l ? p : l;
                    h = q > h ? q : h;
                }
                if (lane == 0 && l <= h) atomicMin(&s_lo, l), atomicMax(&s_hi, h);
            };
            uint32_t lo = 0xffffffffu, hi = 0;
            read_bin([&](int i, uint32_t k, int t) {
                if (listed) list[i] = make_uint2(k, (uint32_t)t);
                lo = k < lo ? k : lo;
                hi = k > hi ? k : hi;
            });
            meet(lo, hi);
            __syncthreads();
            lo = s_lo, hi = s_hi;
            auto scan = [&](auto&& take) {  // every token of the bin, in no order
                if (listed)
                    for (int i = tid; i < cnt_bin; i += kThreads) take(list[i].x, (int)list[i].y);
                else
                    read_bin([&](int, uint32_t k, int t) { take(k, t); });
            };
            constexpr int N = kDigits / 64;
            int buf = 0;
            bool open = true;  // the border lies in what is left; else all of that is kept
            auto border = [&](auto&& below) {  // among the digits of cnt[buf], the greatest first; below: min_p ends there
                uint64_t c[N], w[N];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int d = kDigits - 1 - (lane * N + i);
                    c[i] = cnt[buf][d], w[i] = wsum[buf][d];
                }
                const Border<N> B(c, w, cb, wb, [&](int p, uint64_t ce, uint64_t we, uint64_t) {
                    return ce >= S.top_k || we >= target || below(kDigits - 1 - p);
                });
                open = B.place >= 0;
                if (open) cb = B.cb, wb = B.wb, ties = cnt[buf][kDigits - 1 - B.place];
                return kDigits - 1 - B.place;
            };
            auto turn = [&]() {  // to the other buffer; this one, which every wave has left, is cleared
                __syncthreads();
                for (int i = tid; i < kDigits; i += kThreads) cnt[buf][i] = 0, wsum[buf][i] = 0;
                buf ^= 1;
            };
            // first by the place within the bin, which spreads keys of any exponent (the last bin has none)
            int part = -1;
            auto part_of = [&](uint32_t u) {
                const float v = of_key(u) * g.g;
                const int d = (int)((v - floorf(v)) * kDigits);
                return d < 0 ? 0 : d < kDigits ? d : kDigits - 1;
            };
            auto mine = [&](uint32_t u) { return part < 0 || part_of(u) == part; };
            // up to 64 tokens: each wave ranks them by key and index; the kept ones are the first of that order
            bool settled = false;
            auto rank = [&](uint2 e, int n) {
                const uint64_t f = lane < n ? W.fix(of_key(e.x)) : 0;
                uint64_t before = wb;
                int ahead = 0;
                for (int j = 0; j < n; ++j) {
                    const uint32_t k = __builtin_amdgcn_readlane(e.x, j), i = __builtin_amdgcn_readlane(e.y, j);
                    const uint64_t w = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)f, j) |
                                       (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(f >> 32), j) << 32;
                    const bool first = k > e.x || (k == e.x && i < e.y);
                    ahead += first;
                    before += first ? w : 0;
                }
                const bool keep = lane < n && ((cb == 0 && ahead == 0) ||
                                               (cb + ahead < S.top_k && before < target && e.x >= least));
                const uint64_t kept = __ballot(keep);
                uint32_t k = keep ? e.x : 0xffffffffu, top = lane < n ? e.x : 0;
                for (int d = 32; d; d >>= 1) {
                    const uint32_t p = __shfl_xor(k, d), q = __shfl_xor(top, d);
                    k = p < k ? p : k;
                    top = q > top ? q : top;
                }
                edge = kept ? k : top;
                ties = kept ? __popcll(__ballot(keep && e.x == edge)) : 0;
                settled = true;
            };
            ties = cnt_bin;
            edge = lo - 1;
            if (light) {
                edge = hi;
                ties = 0;
                settled = true;
            } else if (cnt_bin <= 64) {
                rank(lane < cnt_bin ? list[lane] : make_uint2(0u, 0u), cnt_bin);
            } else if (bin < kBins - 1 && lo < hi) {
                scan([&](uint32_t u, int) {
                    atomicAdd(&cnt[buf][part_of(u)], 1u);
                    atomicAdd(&wsum[buf][part_of(u)], (unsigned long long)W.fix(of_key(u)));
                });
                __syncthreads();
                const int least_part = least_bin > bin ? -1 : least_bin < bin || S.min_p > 1.0 ? kDigits : part_of(least);
                part = border([&](int d) { return d <= least_part; });
                if (open && ties <= 64) {
                    if (tid == 0) s_n = 0;
                    __syncthreads();
                    scan([&](uint32_t u, int i) {
                        if (mine(u)) few[atomicAdd(&s_n, 1)] = make_uint2(u, (uint32_t)i);
                    });
                    __syncthreads();
                    rank(lane < (int)ties ? few[lane] : make_uint2(0u, 0u), (int)ties);
                } else if (open) {
                    if (tid == 0) s_lo = 0xffffffffu, s_hi = 0;
                    turn();
                    uint32_t l = 0xffffffffu, h = 0;
                    scan([&](uint32_t u, int) {
                        if (!mine(u)) return;
                        l = u < l ? u : l;
                        h = u > h ? u : h;
                    });
                    meet(l, h);
                    __syncthreads();
                    lo = s_lo, hi = s_hi;
                }
            }
            if (open && !settled) {
                // then by key - lo, nine bits a level from the highest that the keys left use
                int low = 0;
                while (low < 32 && (hi - lo) >> low) low += kDigitBits;
                uint32_t from = lo;  // the least key of what is left
                edge = lo;
                while (low > 0 && open) {
                    const int sh = low - kDigitBits;
                    scan([&](uint32_t u, int) {
                        const uint32_t d = u - from;
                        if (u >= from && (low >= 32 || d >> low == 0) && mine(u)) {
                            atomicAdd(&cnt[buf][d >> sh], 1u);
                            atomicAdd(&wsum[buf][d >> sh], (unsigned long long)W.fix(of_key(u)));
                        }
                    });
                    __syncthreads();
                    const int d = border([&](int i) { return from + ((uint32_t)i << sh) < least; });
                    if (open) {
                        from += (uint32_t)d << sh;
                        low = sh;
                        edge = from;
                    } else {
                        edge = from - 1;  // what is left lies above; lower digits, parts and bins at this or below
                    }
                    if (low > 0 && open) turn();
                }
            }
            if (settled) {
            } else if (open) {  // one key is left: how many of it are kept
                const uint64_t f = W.fix(of_key(edge));
                if (S.top_k != ~0ull) ties = ties < S.top_k - cb ? ties : S.top_k - cb;
                if (f && target != ~0ull) {
                    const uint64_t m = target > wb ? (target - wb + f - 1) / f : 0;
                    ties = ties < m ? ties : m;
                }
                if (edge < least) ties = 0;
                if (cb == 0 && ties == 0) ties = 1;
            } else {
                ties = 0;
            }
            scan([&](uint32_t u, int i) {
                if (u > edge) atomicAdd(&slice_w[i / kSlice], (unsigned long long)W.fix(of_key(u)));
                if (u == edge) atomicAdd(&slice_n[i / kSlice], 1u);
            });
            __syncthreads();
        }
    }

    // Along the index, equal ones of key `edge` until `ties` are used up: the slice that holds the token ...
    const uint64_t fe = ties ? W.fix(of_key(edge)) : 0;
    double u = (double)A.u[r];
    u = u > 0.0 ? (u < 1.0 ? u : 1.0) : 0.0;
    uint64_t total, goal, nb;
    int slice;
    {
        uint64_t w[kLaneSlices], n[kLaneSlices], ws = 0, ns = 0, unused;
#pragma unroll
        for (int i = 0; i < kLaneSlices; ++i) {
            const int s = lane * kLaneSlices + i;
            w[i] = s < slices ? slice_w[s] : 0, n[i] = s < slices ? slice_n[s] : 0;
            ws += w[i], ns += n[i];
        }
        uint64_t n0 = wave_before(ns, &unused), w0 = wave_before(ws, &total);
        total += (ties < unused ? ties : unused) * fe;
        goal = (uint64_t)floor(u * (double)total);
        goal = goal < total ? goal : total - 1;  // u of one and above: the last kept token
        int mine = -1;
        uint64_t mg = 0, mn = 0;
#pragma unroll
        for (int i = 0; i < kLaneSlices; ++i) {
            const uint64_t a = w0 + (n0 < ties ? n0 : ties) * fe;
            const uint64_t n1 = n0 + n[i], z = w0 + w[i] + (n1 < ties ? n1 : ties) * fe;
            if (a <= goal && goal < z) mine = lane * kLaneSlices + i, mg = goal - a, mn = n0;
            n0 = n1, w0 += w[i];
        }
        const uint64_t who = __ballot(mine >= 0);
        const int l = who ? __builtin_ctzll(who) : 0;
        slice = who ? __shfl(mine, l) : 0;
        goal = shfl64(mg, l);  // within the slice
        nb = shfl64(mn, l);    // equal ones before it
    }
    // ... then the token
    const int i0 = slice * kSlice + tid * kPer;
    float x[kPer];
#pragma unroll
    for (int j = 0; j < kPer / 8; ++j) {
        Eight<DT> v;
        if (aligned && i0 + kPer <= V)
            v.load(A.logits, row + i0 + 8 * j);
        else
            v.load_checked(A, row, i0 + 8 * j);
#pragma unroll
        for (int q = 0; q < 8; ++q) x[8 * j + q] = v[q];
    }
    uint64_t f[kPer], w = 0, n = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const uint32_t k = x[e] > -INFINITY ? key_of(x[e]) : 0;
        f[e] = k > edge ? W.fix(x[e]) : 0;
        w += f[e];
        n += k && k == edge;
    }
    uint64_t wa, na;
    uint64_t w0 = wave_before(w, &wa), n0 = nb + wave_before(n, &na);
    if (lane == 0) red[tid >> 6][0] = wa, red[tid >> 6][1] = na;
    __syncthreads();
    uint64_t sw = 0, sn = nb;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (i < (tid >> 6)) w0 += red[i][0], n0 += red[i][1];
        sw += red[i][0], sn += red[i][1];
    }
    auto kept = [&](uint64_t before) { return ((before < ties ? before : ties) - (nb < ties ? nb : ties)) * fe; };
    const uint64_t all = sw + kept(sn);
    // the slice's sum was rounded apart from its tokens', by some units of 2^-shift
    goal = goal < all ? goal : all - 1;
    uint64_t at = w0 + kept(n0);
    if (at <= goal && goal < w0 + w + kept(n0 + n)) {
        int tok = -1;
        float xt = 0.0f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            at += f[e];
            if (x[e] > -INFINITY && key_of(x[e]) == edge) at += n0++ < ties ? fe : 0;
            if (tok < 0 && at > goal) tok = i0 + e, xt = x[e];
        }
        A.token[r] = tok;
        if (A.logprob) {
            const double d = xt == mx ? 0.0 : ((double)xt - (double)mx) * S.inv_t;
            A.logprob[r] = (float)(d - log(__builtin_ldexp((double)total, -A.shift)));
        }
    }
}

size_t sample_ws_bytes(int rows, int vocab) { return (size_t)layout(rows, vocab).total; }

int launch_sample(const SampleArgs& A, hipStream_t st) {
    if (A.rows == 0) return PGMOE_OK;
    const dim3 slices(A.rows, (A.vocab + kSlice - 1) / kSlice), rows(A.rows), block(kThreads);
#define SAMPLE(DT)                                                              \
    do {                                                                        \
        PG_LAUNCH((sample_slice_kernel<DT>), slices, block, 0, st, A);          \
        PG_LAUNCH((sample_row_kernel<DT>), rows, block, 0, st, A);              \
    } while (0)
    if (A.dtype == PGMOE_DT_F32)
        SAMPLE(PGMOE_DT_F32);
    else if (A.dtype == PGMOE_DT_F16)
        SAMPLE(PGMOE_DT_F16);
    else
        SAMPLE(PGMOE_DT_BF16);
#undef SAMPLE
    return check_launch("sample");
}

}  // namespace pgmoe
