// Token sampling: temperature, top-k, top-p, min-p and a given uniform number a row.
//
// The simplest right form: one workgroup a row, which it reads from memory once for the maximum, once for
// each digit of a radix descent to the last kept token, and once for the sums along the index.
#include "launch.h"
#include "sample.h"

namespace pgmoe {

constexpr int kSampleThreads = 1024;
constexpr int kPer = 8;  // consecutive tokens of a thread
constexpr int kTile = kSampleThreads * kPer;
constexpr int kBins = 2048;
constexpr int kMaxTiles = kMaxVocab / kTile;

__device__ __forceinline__ float logit(const void* p, int dt, int64_t i) {
    if (dt == PGMOE_DT_F32) return ((const float*)p)[i];
    const uint16_t u = ((const uint16_t*)p)[i];
    return dt == PGMOE_DT_F16 ? h2f(u) : __builtin_bit_cast(float, (uint32_t)u << 16);
}
// A monotone 32-bit key: a > b as floats exactly if key(a) > key(b); +0 and -0 share one.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct Weigh {
    float mx;
    double inv_t;
    int shift;
    __device__ double w(float x) const {  // 0 for NaN and below everything that counts
        if (x == mx) return 1.0;
        if (!(x > -INFINITY) || mx == INFINITY) return 0.0;
        return exp(((double)x - (double)mx) * inv_t);
    }
    __device__ uint64_t fix(float x) const { return (uint64_t)llrint(ldexp(w(x), shift)); }
};

__device__ uint64_t block_sum(uint64_t v, uint64_t* s) {
    __syncthreads();
    for (int d = 32; d; d >>= 1) v += __shfl_xor((unsigned long long)v, d);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
    for (int i = 0; i < kSampleThreads / 64; ++i) t += s[i];
    return t;
}
// Sum over the threads below this one.
__device__ uint64_t block_before(uint64_t v, uint64_t* s) {
    __syncthreads();
    const int lane = threadIdx.x & 63;
    uint64_t inc = v;
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up((unsigned long long)inc, d);
        if (lane >= d) inc += o;
    }
    if (lane == 63) s[threadIdx.x >> 6] = inc;
    __syncthreads();
    uint64_t t = inc - v;
    for (int i = 0; i < (int)(threadIdx.x >> 6); ++i) t += s[i];
    return t;
}

__global__ __launch_bounds__(kSampleThreads) void sample_row_kernel(const SampleArgs A) {
    __shared__ uint32_t cnt[kBins];
    __shared__ unsigned long long wsum[kBins];
    __shared__ uint64_t red[kSampleThreads / 64];
    __shared__ float redf[kSampleThreads / 64];
    __shared__ uint64_t tile_w[kMaxTiles];
    __shared__ uint32_t tile_n[kMaxTiles];
    __shared__ int s_bin, s_tile;
    __shared__ uint64_t s_cb, s_wb;
    const int r = blockIdx.x, tid = threadIdx.x, V = A.vocab;
    const int64_t row = (int64_t)r * A.row_stride;
    const double temp = A.P.temperatures ? (double)A.P.temperatures[r] : A.P.temperature;
    const double top_p = A.P.top_ps ? (double)A.P.top_ps[r] : A.P.top_p;
    const double min_p = A.P.min_ps ? (double)A.P.min_ps[r] : A.P.min_p;
    int top_k = A.P.top_ks ? A.P.top_ks[r] : A.P.top_k;
    const bool greedy = !(temp > 0.0);
    if (greedy) top_k = 1;
    const uint64_t k = top_k > 0 ? (uint64_t)top_k : ~0ull;

    float mx = -INFINITY;
    for (int i = tid; i < V; i += kSampleThreads) mx = fmaxf(mx, logit(A.logits, A.dtype, row + i));
    mx = wave_max(mx);
    if ((tid & 63) == 0) redf[tid >> 6] = mx;
    __syncthreads();
    for (int i = 0; i < kSampleThreads / 64; ++i) mx = fmaxf(mx, redf[i]);
    if (mx == -INFINITY) {
        if (tid == 0) {
            A.token[r] = -1;
            if (A.logprob) A.logprob[r] = -INFINITY;
        }
        return;
    }
    const Weigh W{mx, greedy ? 1.0 : 1.0 / temp, A.shift};

    // The last kept token: key `edge`, of which the first `ties` in index order are kept; every greater key is.
    uint32_t edge = 0;
    uint64_t ties = 0;
    if (k != ~0ull || top_p < 1.0 || min_p > 0.0) {
        uint64_t cb = 0, wb = 0, target = ~0ull;
        uint32_t prefix = 0;
        int low = 32;  // bits below the prefix
        const int bits[3] = {11, 11, 10};
        for (int level = 0; level < 3; ++level) {
            const int sh = low - bits[level], n = 1 << bits[level];
            for (int i = tid; i < n; i += kSampleThreads) cnt[i] = 0, wsum[i] = 0;
            __syncthreads();
            for (int i = tid; i < V; i += kSampleThreads) {
                const float x = logit(A.logits, A.dtype, row + i);
                const uint32_t u = key_of(x);
                if (x > -INFINITY && (level == 0 || (u >> low) == prefix)) {
                    const int bin = (u >> sh) & (n - 1);
                    atomicAdd(&cnt[bin], 1u);
                    atomicAdd(&wsum[bin], (unsigned long long)W.fix(x));
                }
            }
            if (tid == 0) s_bin = -1;
            __syncthreads();
            if (level == 0 && top_p < 1.0) {
                const uint64_t all = block_sum(wsum[tid] + wsum[tid + kSampleThreads], red);
                target = top_p > 0.0 ? (uint64_t)ceil(top_p * (double)all) : 0;
            }
            // thread i holds bins n - 1 - 2 i and n - 2 - 2 i: the order of the tokens
            uint64_t c[2] = {0, 0}, w[2] = {0, 0};
            for (int q = 0; q < 2; ++q) {
                const int bin = n - 1 - 2 * tid - q;
                if (bin >= 0) c[q] = cnt[bin], w[q] = wsum[bin];
            }
            uint64_t c0 = cb + block_before(c[0] + c[1], red), w0 = wb + block_before(w[0] + w[1], red);
            for (int q = 0; q < 2; ++q) {
                const int bin = n - 1 - 2 * tid - q;
                if (bin >= 0 && c[q]) {
                    const uint32_t least = (low == 32 ? 0u : prefix << low) | (uint32_t)bin << sh;
                    if (c0 + c[q] >= k || w0 + w[q] >= target || (min_p > 0.0 && !(W.w(of_key(least)) >= min_p)))
                        atomicMax(&s_bin, bin);
                }
                c0 += c[q], w0 += w[q];
            }
            __syncthreads();
            if (s_bin < 0) {  // every token of this prefix is kept
                edge = low == 32 ? 0u : (prefix << low) - 1u;
                ties = 0;
                break;
            }
            c0 -= c[0] + c[1], w0 -= w[0] + w[1];
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
                const float x = of_key(edge);
                const uint64_t f = W.fix(x);
                ties = cnt[s_bin];
                if (k != ~0ull) ties = ties < k - cb ? ties : k - cb;
                if (f && target != ~0ull) {
                    const uint64_t m = target > wb ? (target - wb + f - 1) / f : 0;
                    ties = ties < m ? ties : m;
                }
                if (min_p > 0.0 && !(W.w(x) >= min_p)) ties = 0;
                if (cb == 0 && ties == 0) ties = 1;
            }
            __syncthreads();
        }
    }

    // Sums along the index, a tile at a time; then the one tile that holds the token.
    const uint64_t fe = W.fix(of_key(edge));
    const int tiles = (V + kTile - 1) / kTile;
    for (int g = 0; g < tiles; ++g) {
        uint64_t w = 0, n = 0;
        for (int q = 0; q < kPer; ++q) {
            const int i = g * kTile + tid * kPer + q;
            const float x = i < V ? logit(A.logits, A.dtype, row + i) : -INFINITY;
            const uint32_t u = key_of(x);
            if (x > -INFINITY) {
                if (u > edge) w += W.fix(x);
                n += u == edge;
            }
        }
        w = block_sum(w, red);
        n = block_sum(n, red);
        if (tid == 0) tile_w[g] = w, tile_n[g] = (uint32_t)n;
    }
    __syncthreads();
    uint64_t total = 0, nb = 0;
    for (int g = 0; g < tiles; ++g) {
        const uint64_t e = nb + tile_n[g] < ties ? nb + tile_n[g] : ties, f = nb < ties ? nb : ties;
        total += tile_w[g] + (e - f) * fe;
        nb += tile_n[g];
    }
    double u = (double)A.u[r];
    u = u > 0.0 ? (u < 1.0 ? u : 1.0) : 0.0;
    uint64_t goal = (uint64_t)floor(u * (double)total);
    if (goal >= total) goal = total - 1;  // u of one and above: the last kept token
    if (tid == 0) {
        uint64_t at = 0;
        nb = 0;
        int g = 0;
        for (; g < tiles; ++g) {
            const uint64_t e = nb + tile_n[g] < ties ? nb + tile_n[g] : ties, f = nb < ties ? nb : ties;
            const uint64_t w = tile_w[g] + (e - f) * fe;
            if (at + w > goal) break;
            at += w;
            nb += tile_n[g];
        }
        s_tile = g, s_wb = at, s_cb = nb;
    }
    __syncthreads();
    const int i0 = s_tile * kTile + tid * kPer;
    uint64_t w = 0, n = 0;
    float x[kPer];
    for (int q = 0; q < kPer; ++q) {
        x[q] = i0 + q < V ? logit(A.logits, A.dtype, row + i0 + q) : -INFINITY;
        if (x[q] > -INFINITY) {
            if (key_of(x[q]) > edge) w += W.fix(x[q]);
            n += key_of(x[q]) == edge;
        }
    }
    nb = s_cb + block_before(n, red);
    uint64_t mine = w;
    {
        const uint64_t e = nb + n < ties ? nb + n : ties, f = nb < ties ? nb : ties;
        mine += (e - f) * fe;
    }
    uint64_t at = s_wb + block_before(mine, red);
    if (at <= goal && at + mine > goal) {
        for (int q = 0; q < kPer; ++q) {
            if (!(x[q] > -INFINITY)) continue;
            const uint32_t kx = key_of(x[q]);
            const uint64_t f = kx > edge ? W.fix(x[q]) : kx == edge && nb < ties ? fe : 0;
            nb += kx == edge;
            at += f;
            if (at > goal) {
                A.token[r] = i0 + q;
                if (A.logprob) {
                    const double d = x[q] == mx ? 0.0 : ((double)x[q] - (double)mx) * W.inv_t;
                    A.logprob[r] = greedy ? 0.0f : (float)(d - log(ldexp((double)total, -A.shift)));
                }
                break;
            }
        }
    }
}

size_t sample_ws_bytes(int rows, int vocab) { return 0; }

int launch_sample(const SampleArgs& A, hipStream_t st) {
    if (A.rows == 0) return PGMOE_OK;
    PG_LAUNCH(sample_row_kernel, dim3(A.rows), dim3(kSampleThreads), 0, st, A);
    return check_launch("sample");
}

}  // namespace pgmoe
