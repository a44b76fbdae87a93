// Token sampling: temperature, top-k, top-p, min-p and a given uniform number a row.
//
// Weights w = exp((x - max) / T) are held as 64-bit fixed point (2^-44 for vocabularies of 2^18, finer for
// smaller ones: a sum stays below 2^63): integer sums have no order, and a row's result is the same bits however it is cut.  No
// row is sorted: the last kept token is found from a histogram over the distance to the maximum, then by a
// radix descent over the float keys of the one bin that holds it.
//
// slice_kernel, a workgroup for 8192 tokens of a row, reads the logits once into registers: the slice's
// maximum, and against it the tokens' weights, their sum and the histogram (256 bins of 1/8 in x / T on a grid
// that all slices share).  row_kernel, a workgroup a row: the slices' sums brought to the row's maximum (a
// slice that holds the maximum exactly, so that equal logits stay equal weights), the bin of the last kept
// token, its tokens read again into LDS, the descent, and the sums along the index down to the token.
#include "launch.h"
#include "sample.h"

namespace pgmoe {

constexpr int kSlice = 8192;                   // tokens of a slice
constexpr int kSliceThreads = 256;
constexpr int kRowThreads = 1024;
constexpr int kPer = kSlice / kRowThreads;     // consecutive tokens of a row_kernel thread
constexpr int kBins = 256;                     // of the distance; the last holds all that lies further
constexpr float kPerNat = 8.0f;                // bins a unit of x / T
constexpr int kDigits = 2048;
constexpr int kList = 6144;                    // tokens of one bin that fit LDS
constexpr int kMaxSlices = kMaxVocab / kSlice;

struct Slice {
    uint64_t sum;  // of weights against the slice's maximum
    float max;
    int first;  // lowest index of the maximum
};
struct Layout {
    int64_t slices, cnt, wgt, total;
};
static __host__ __device__ Layout layout(int rows, int vocab) {
    const int64_t n = (int64_t)rows * ((vocab + kSlice - 1) / kSlice);
    Layout o;
    o.slices = 0;
    o.wgt = (n * (int64_t)sizeof(Slice) + 255) / 256 * 256;
    o.cnt = o.wgt + n * kBins * 8;
    o.total = o.cnt + n * kBins * 4;
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

// N consecutive logits from element i of a row on, -inf behind the last.
template <int N>
__device__ __forceinline__ void load_logits(const SampleArgs& A, int64_t row, int i, float (&x)[N]) {
    const int64_t at = row + i;
    if (A.dtype == PGMOE_DT_F32) {
        const float* p = (const float*)A.logits + at;
        if (i + N <= A.vocab && ((uintptr_t)p & 15) == 0) {
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                const float4 v = *(const float4*)(p + j);
                x[j] = v.x, x[j + 1] = v.y, x[j + 2] = v.z, x[j + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = i + j < A.vocab ? p[j] : -INFINITY;
        }
        return;
    }
    const uint16_t* p = (const uint16_t*)A.logits + at;
    uint16_t h[N];
    if (i + N <= A.vocab && ((uintptr_t)p & 15) == 0) {
#pragma unroll
        for (int j = 0; j < N; j += 8) {
            const uint4 v = *(const uint4*)(p + j);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 8; ++k) h[j + k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) h[j] = i + j < A.vocab ? p[j] : A.dtype == PGMOE_DT_F16 ? 0xfc00 : 0xff80;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = A.dtype == PGMOE_DT_F16 ? h2f(h[j]) : __builtin_bit_cast(float, (uint32_t)h[j] << 16);
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

// w = exp((x - top) / T) = 2^(q / 32) e^g with |g| <= ln 2 / 64: a table of 32 powers and five terms of the
// series, relative error 2^-48; fixed point by adding 2^52.
struct Weigh {
    const double* powers;  // 2^(i / 32), LDS
    float top;
    double k32;  // 32 log2(e) / T
    int shift;
    __device__ __forceinline__ Weigh(const double* powers_, float top_, double inv_t, int shift_)
        : powers(powers_), top(top_), k32(inv_t * 46.16624130844683), shift(shift_) {}
    __device__ __forceinline__ double scaled(float x, int shift_) const {
        if (x == top) return __builtin_ldexp(1.0, shift_);
        const double t = ((double)x - (double)top) * k32;
        if (!(t > -2048.0)) return 0.0;  // also -inf, NaN, and everything beside +inf; 2^-64
        const double q = __builtin_rint(t);
        const double g = (t - q) * 0.021660849392498290;
        double p = __builtin_fma(g, 1.0 / 120.0, 1.0 / 24.0);
        p = __builtin_fma(p, g, 1.0 / 6.0);
        p = __builtin_fma(p, g, 0.5);
        p = __builtin_fma(p, g, 1.0);
        p = __builtin_fma(p, g, 1.0);
        const int n = (int)q;
        return __builtin_ldexp(powers[n & 31] * p, (n >> 5) + shift_);
    }
    __device__ __forceinline__ double w(float x) const { return scaled(x, 0); }
    __device__ __forceinline__ uint64_t fix(float x) const {
        const double v = scaled(x, shift) + 4503599627370496.0;
        return __builtin_bit_cast(uint64_t, v) & 0xfffffffffffffull;
    }
};
__device__ __forceinline__ void fill_powers(double* p, int tid) {
    if (tid < 32) p[tid] = exp2((double)tid / 32.0);
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

__global__ __launch_bounds__(kSliceThreads) void sample_slice_kernel(const SampleArgs A) {
    constexpr int G = 8, N = kSlice / kSliceThreads / G;  // groups of 8 tokens a thread
    __shared__ uint32_t cnt[kBins];
    __shared__ unsigned long long wgt[kBins];
    __shared__ double powers[32];
    __shared__ float s_max[kSliceThreads / 64];
    __shared__ uint64_t s_sum[kSliceThreads / 64];
    __shared__ int s_first;
    const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63, base = blockIdx.x * kSlice;
    const int64_t row = (int64_t)r * A.row_stride;
    float x[N][G];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int i = base + (j * kSliceThreads + tid) * G;
        if (i < A.vocab)
            load_logits<G>(A, row, i, x[j]);
        else
            for (int e = 0; e < G; ++e) x[j][e] = -INFINITY;
    }
    const Settings S(A, r);
    fill_powers(powers, tid);
    if (tid == 0) s_first = 0x7fffffff;
    cnt[tid] = 0, wgt[tid] = 0;
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < G; ++e) mx = fmaxf(mx, x[j][e]);
    mx = wave_max(mx);
    if (lane == 0) s_max[tid >> 6] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSliceThreads / 64; ++i) mx = fmaxf(mx, s_max[i]);

    const int64_t at = (int64_t)r * gridDim.x + blockIdx.x;
    const Layout o = layout(A.rows, A.vocab);
    Slice* out = (Slice*)((uint8_t*)A.ws + o.slices) + at;
    if (S.greedy || mx == -INFINITY) {
        int first = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < G; ++e)
                if (x[j][e] == mx) {
                    const int i = base + (j * kSliceThreads + tid) * G + e;
                    first = i < first ? i : first;
                }
        if (first != 0x7fffffff) atomicMin(&s_first, first);
        __syncthreads();
        if (tid == 0) *out = Slice{0, mx, s_first};
    } else {
        const Weigh W(powers, mx, S.inv_t, A.shift);
        const Grid g(mx, S.inv_t);
        uint64_t sum = 0;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < G; ++e) {
                const uint64_t f = W.fix(x[j][e]);
                sum += f;
                if (S.filters && x[j][e] > -INFINITY) {
                    const int b = g.bin(x[j][e]);
                    atomicAdd(&cnt[b], 1u);
                    if (f) atomicAdd(&wgt[b], (unsigned long long)f);
                }
            }
        sum = wave_sum(sum);
        if (lane == 0) s_sum[tid >> 6] = sum;
        __syncthreads();
        if (tid == 0) *out = Slice{s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3], mx, 0};
    }
    if (S.filters) {
        __syncthreads();
        ((uint32_t*)((uint8_t*)A.ws + o.cnt))[at * kBins + tid] = cnt[tid];
        ((uint64_t*)((uint8_t*)A.ws + o.wgt))[at * kBins + tid] = wgt[tid];
    }
}

__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* s) {
    __syncthreads();
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
    for (int i = 0; i < kRowThreads / 64; ++i) t += s[i];
    return t;
}
// Sums of two values over the threads below this one.
__device__ __forceinline__ void block_before(uint64_t& a, uint64_t& b, uint64_t (*s)[2]) {
    __syncthreads();
    const int lane = threadIdx.x & 63;
    uint64_t x = a, y = b;
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t p = __shfl_up((unsigned long long)x, d), q = __shfl_up((unsigned long long)y, d);
        if (lane >= d) x += p, y += q;
    }
    if (lane == 63) s[threadIdx.x >> 6][0] = x, s[threadIdx.x >> 6][1] = y;
    __syncthreads();
    a = x - a, b = y - b;
    for (int i = 0; i < (int)(threadIdx.x >> 6); ++i) a += s[i][0], b += s[i][1];
}

__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(const SampleArgs A) {
    __shared__ uint2 list[kList];  // (key, index) of the tokens of the last kept one's bin
    __shared__ unsigned long long wsum[kDigits];
    __shared__ uint32_t cnt[kDigits];
    __shared__ unsigned long long slice_w[kMaxSlices];
    __shared__ double slice_s[kMaxSlices];  // the slice's weights to the row's: exp((its max - max) / T)
    __shared__ float slice_d[kMaxSlices];   // the slice's bins to the row's
    __shared__ uint32_t slice_n[kMaxSlices];
    __shared__ double powers[32];
    __shared__ uint64_t red[kRowThreads / 64][2];
    __shared__ float redf[kRowThreads / 64];
    __shared__ int s_bin, s_n, s_first, s_slice;
    __shared__ uint64_t s_cb, s_wb;
    const int r = blockIdx.x, tid = threadIdx.x, V = A.vocab;
    const int slices = (V + kSlice - 1) / kSlice;
    const int64_t row = (int64_t)r * A.row_stride;
    const Layout o = layout(A.rows, V);
    const Slice* sl = (const Slice*)((uint8_t*)A.ws + o.slices) + (int64_t)r * slices;
    const uint32_t* hc = (const uint32_t*)((uint8_t*)A.ws + o.cnt) + (int64_t)r * slices * kBins;
    const uint64_t* hw = (const uint64_t*)((uint8_t*)A.ws + o.wgt) + (int64_t)r * slices * kBins;
    const Settings S(A, r);

    Slice mine{0, -INFINITY, 0x7fffffff};
    if (tid < slices) mine = sl[tid];
    fill_powers(powers, tid);
    if (tid == 0) s_first = 0x7fffffff, s_n = 0, s_bin = 0x7fffffff;
    float mx = wave_max(mine.max);
    if ((tid & 63) == 0) redf[tid >> 6] = mx;
    __syncthreads();
    for (int i = 0; i < kRowThreads / 64; ++i) mx = fmaxf(mx, redf[i]);
    if (mx == -INFINITY) {
        if (tid == 0) {
            A.token[r] = -1;
            if (A.logprob) A.logprob[r] = -INFINITY;
        }
        return;
    }
    if (S.greedy) {
        if (mine.max == mx) atomicMin(&s_first, mine.first);
        __syncthreads();
        if (tid == 0) {
            A.token[r] = s_first;
            if (A.logprob) A.logprob[r] = 0.0f;
        }
        return;
    }
    const Weigh W(powers, mx, S.inv_t, A.shift);
    const Grid g(mx, S.inv_t);
    auto to_row = [&](uint64_t w, int s) { return slice_s[s] == 1.0 ? w : (uint64_t)llrint((double)w * slice_s[s]); };
    if (tid < slices) {
        const bool top = mine.max == mx;
        slice_s[tid] = top ? 1.0 : mine.max == -INFINITY || mx == INFINITY ? 0.0 : exp(((double)mine.max - (double)mx) * S.inv_t);
        slice_d[tid] = top ? 0.0f : g.at - floorf(mine.max * g.g);
        slice_w[tid] = to_row(mine.sum, tid);  // without filters: everything is kept
        slice_n[tid] = 0;
    }
    __syncthreads();

    // The last kept token: key `edge`, of which the first `ties` in index order are kept; every greater key is.
    uint32_t edge = 0;
    uint64_t ties = 0;
    if (S.filters) {
        for (int i = tid; i < kBins; i += kRowThreads) cnt[i] = 0, wsum[i] = 0;
        __syncthreads();
        auto row_bin = [&](int s, int b) {
            const float d = (float)b + slice_d[s];
            return d < (float)(kBins - 1) ? (int)d : kBins - 1;
        };
        for (int i = tid; i < slices * kBins; i += kRowThreads) {
            const int s = i / kBins;
            const uint32_t c = hc[i];
            if (c && sl[s].max > -INFINITY) {
                const int b = row_bin(s, i % kBins);
                atomicAdd(&cnt[b], c);
                atomicAdd(&wsum[b], (unsigned long long)to_row(hw[i], s));
            }
        }
        // the least key that min_p keeps: bisection to the border of w >= min_p, from its logarithm
        uint32_t least = 0;
        int least_bin = kBins;
        if (S.min_p >= 1.0) {
            least = key_of(mx) + (S.min_p > 1.0);
            least_bin = 0;
        } else if (S.min_p > 0.0) {
            const uint32_t k = key_of((float)((double)mx + log(S.min_p) / S.inv_t));
            uint32_t out = key_of(-INFINITY), in = key_of(mx);  // falls short, is kept
            if (k > out + 8 && k < in && !(W.w(of_key(k - 8)) >= S.min_p)) out = k - 8;
            if (k > out && k + 8 < in && W.w(of_key(k + 8)) >= S.min_p) in = k + 8;
            while (in - out > 1) {
                const uint32_t mid = out + (in - out) / 2;
                (W.w(of_key(mid)) >= S.min_p ? in : out) = mid;
            }
            least = in;
            least_bin = g.bin(of_key(least));
        }
        __syncthreads();
        const uint64_t all = block_sum(tid < kBins ? wsum[tid] : 0, (uint64_t*)red);
        const uint64_t target = S.top_p < 1.0 ? (S.top_p > 0.0 ? (uint64_t)ceil(S.top_p * (double)all) : 0) : ~0ull;
        uint64_t cb, wb;
        {
            const uint64_t c = tid < kBins ? cnt[tid] : 0, w = tid < kBins ? wsum[tid] : 0;
            uint64_t c0 = c, w0 = w;
            block_before(c0, w0, red);
            if (c && (c0 + c >= S.top_k || w0 + w >= target || tid >= least_bin)) atomicMin(&s_bin, tid);
            __syncthreads();
            if (tid == s_bin) s_cb = c0, s_wb = w0;
        }
        __syncthreads();
        const int bin = s_bin;
        if (bin < kBins) {
            cb = s_cb, wb = s_wb;
            const bool listed = cnt[bin] <= kList;
            // what each slice keeps above the bin, and the bin's tokens
            if (tid < slices) slice_w[tid] = 0;
            __syncthreads();
            for (int i = tid; i < slices * kBins; i += kRowThreads) {
                const int s = i / kBins;
                if (hc[i] && sl[s].max > -INFINITY && row_bin(s, i % kBins) < bin)
                    atomicAdd(&slice_w[s], (unsigned long long)to_row(hw[i], s));
            }
            auto scan = [&](auto&& take) {  // every token of the bin, in no order
                if (listed) {
                    for (int i = tid; i < s_n && i < kList; i += kRowThreads) take(list[i].x, (int)list[i].y);
                } else {
                    for (int s = 0; s < slices; ++s) {
                        float x[kPer];
                        const int i0 = s * kSlice + tid * kPer;
                        if (i0 >= V) continue;
                        load_logits<kPer>(A, row, i0, x);
#pragma unroll
                        for (int e = 0; e < kPer; ++e)
                            if (x[e] > -INFINITY && g.bin(x[e]) == bin) take(key_of(x[e]), i0 + e);
                    }
                }
            };
            if (listed) {
#pragma unroll 4
                for (int s = 0; s < slices; ++s) {
                    // only slices that have tokens there
                    const float b = (float)bin - slice_d[s];
                    if (bin < kBins - 1 && (!(b >= 0.0f) || !hc[s * kBins + (int)b])) continue;
                    float x[kPer];
                    const int i0 = s * kSlice + tid * kPer;
                    if (i0 >= V) continue;
                    load_logits<kPer>(A, row, i0, x);
#pragma unroll
                    for (int e = 0; e < kPer; ++e)
                        if (x[e] > -INFINITY && g.bin(x[e]) == bin) {
                            const int at = atomicAdd(&s_n, 1);
                            if (at < kList) list[at] = make_uint2(key_of(x[e]), (uint32_t)(i0 + e));
                        }
                }
            }
            __syncthreads();
            uint32_t prefix = 0;
            int low = 32;  // bits below the prefix
            const int bits[3] = {11, 11, 10};
            bool whole = false;
            for (int level = 0; level < 3 && !whole; ++level) {
                const int sh = low - bits[level], n = 1 << bits[level];
                for (int i = tid; i < n; i += kRowThreads) cnt[i] = 0, wsum[i] = 0;
                if (tid == 0) s_bin = -1;
                __syncthreads();
                scan([&](uint32_t u, int) {
                    if (level == 0 || (u >> low) == prefix) {
                        const int d = (u >> sh) & (n - 1);
                        atomicAdd(&cnt[d], 1u);
                        atomicAdd(&wsum[d], (unsigned long long)W.fix(of_key(u)));
                    }
                });
                __syncthreads();
                // thread i holds digits n - 1 - 2 i and n - 2 - 2 i: the order of the tokens
                uint64_t c[2] = {0, 0}, w[2] = {0, 0};
                for (int q = 0; q < 2; ++q) {
                    const int d = n - 1 - 2 * tid - q;
                    if (d >= 0) c[q] = cnt[d], w[q] = wsum[d];
                }
                uint64_t c0 = c[0] + c[1], w0 = w[0] + w[1];
                block_before(c0, w0, red);
                c0 += cb, w0 += wb;
                uint64_t c1 = c0, w1 = w0;
                for (int q = 0; q < 2; ++q) {
                    const int d = n - 1 - 2 * tid - q;
                    if (d >= 0 && c[q]) {
                        const uint32_t lowest = (low == 32 ? 0u : prefix << low) | (uint32_t)d << sh;
                        if (c1 + c[q] >= S.top_k || w1 + w[q] >= target || lowest < least) atomicMax(&s_bin, d);
                    }
                    c1 += c[q], w1 += w[q];
                }
                __syncthreads();
                whole = s_bin < 0;  // every token of this prefix is kept, and none below it
                if (whole) {
                    // the greatest key below the bin's: keys of lower bins are smaller than the bin's least
                    uint32_t lowest = 0xffffffffu;
                    scan([&](uint32_t u, int) {
                        if (level == 0 || (u >> low) == prefix) lowest = u < lowest ? u : lowest;
                    });
                    if (tid == 0) s_first = -1;  // as unsigned: the greatest
                    __syncthreads();
                    atomicMin((unsigned*)&s_first, lowest);
                    __syncthreads();
                    edge = (uint32_t)s_first - 1u;
                    ties = 0;
                    break;
                }
                for (int q = 0; q < 2; ++q) {
                    if (n - 1 - 2 * tid - q == s_bin) s_cb = c0, s_wb = w0;
                    c0 += c[q], w0 += w[q];
                }
                __syncthreads();
                prefix = (low == 32 ? 0u : prefix << bits[level]) | (uint32_t)s_bin;
                low = sh;
                cb = s_cb, wb = s_wb;
                if (level == 2) {
                    edge = prefix;
                    const uint64_t f = W.fix(of_key(edge));
                    ties = cnt[s_bin];
                    if (S.top_k != ~0ull) ties = ties < S.top_k - cb ? ties : S.top_k - cb;
                    if (f && target != ~0ull) {
                        const uint64_t m = target > wb ? (target - wb + f - 1) / f : 0;
                        ties = ties < m ? ties : m;
                    }
                    if (edge < least) ties = 0;
                    if (cb == 0 && ties == 0) ties = 1;
                }
                __syncthreads();
            }
            scan([&](uint32_t u, int i) {
                if (u > edge) atomicAdd(&slice_w[i / kSlice], (unsigned long long)W.fix(of_key(u)));
                if (u == edge) atomicAdd(&slice_n[i / kSlice], 1u);
            });
            __syncthreads();
        }
    }

    // Along the index: the slice that holds the token, then the token.
    const uint64_t fe = W.fix(of_key(edge));
    auto tied = [&](uint64_t before, uint64_t n) {  // how many of n equal ones behind `before` others are kept
        const uint64_t a = before < ties ? before : ties, b = before + n < ties ? before + n : ties;
        return b - a;
    };
    double u = (double)A.u[r];
    u = u > 0.0 ? (u < 1.0 ? u : 1.0) : 0.0;
    uint64_t total;
    {
        const uint64_t n = tid < slices ? slice_n[tid] : 0, w = tid < slices ? slice_w[tid] : 0;
        uint64_t nb = n, unused = 0;
        block_before(nb, unused, red);
        const uint64_t m = w + tied(nb, n) * fe;
        total = block_sum(m, (uint64_t*)red);
        uint64_t goal = (uint64_t)floor(u * (double)total);
        goal = goal < total ? goal : total - 1;  // u of one and above: the last kept token
        uint64_t at = m;
        unused = 0;
        block_before(at, unused, red);
        if (tid == 0) s_slice = slices - 1;
        __syncthreads();
        if (at <= goal && at + m > goal) s_slice = tid, s_wb = goal - at, s_cb = nb;
    }
    __syncthreads();
    const int i0 = s_slice * kSlice + tid * kPer;
    const uint64_t goal = s_wb;  // within the slice
    float x[kPer];
    if (i0 < V)
        load_logits<kPer>(A, row, i0, x);
    else
        for (int e = 0; e < kPer; ++e) x[e] = -INFINITY;
    uint64_t w = 0, n = 0;
    int last = -1;  // of this thread's kept tokens
#pragma unroll
    for (int e = 0; e < kPer; ++e)
        if (x[e] > -INFINITY) {
            const uint32_t k = key_of(x[e]);
            if (k > edge) w += W.fix(x[e]);
            n += k == edge;
        }
    uint64_t nb = n, unused = 0;
    block_before(nb, unused, red);
    nb += s_cb;
    const uint64_t m = w + tied(nb, n) * fe;
    uint64_t at = m;
    unused = 0;
    block_before(at, unused, red);
    // the slice's sum was rounded apart from its tokens' by some units of 2^-44: the last kept one then
    if (tid == 0) s_first = -1, s_n = 0x7fffffff;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        if (!(x[e] > -INFINITY)) continue;
        const uint32_t k = key_of(x[e]);
        const uint64_t f = k > edge ? W.fix(x[e]) : k == edge && nb < ties ? fe : 0;
        nb += k == edge;
        at += f;
        if (f) last = i0 + e;
        if (f && at > goal) {
            atomicMin(&s_n, i0 + e);
            break;
        }
    }
    if (last >= 0) atomicMax(&s_first, last);
    __syncthreads();
    const int tok = s_n != 0x7fffffff ? s_n : s_first;
    if (tok >= i0 && tok < i0 + kPer) {
#pragma unroll
        for (int e = 0; e < kPer; ++e)
            if (tok == i0 + e) {
                A.token[r] = tok;
                if (A.logprob) {
                    const double d = x[e] == mx ? 0.0 : ((double)x[e] - (double)mx) * S.inv_t;
                    A.logprob[r] = (float)(d - log(__builtin_ldexp((double)total, -A.shift)));
                }
            }
    }
}

size_t sample_ws_bytes(int rows, int vocab) { return (size_t)layout(rows, vocab).total; }

int launch_sample(const SampleArgs& A, hipStream_t st) {
    if (A.rows == 0) return PGMOE_OK;
    PG_LAUNCH(sample_slice_kernel, dim3((A.vocab + kSlice - 1) / kSlice, A.rows), dim3(kSliceThreads), 0, st, A);
    PG_LAUNCH(sample_row_kernel, dim3(A.rows), dim3(kRowThreads), 0, st, A);
    return check_launch("sample");
}

}  // namespace pgmoe
