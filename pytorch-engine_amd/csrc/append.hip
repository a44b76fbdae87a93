// Rotary positions and per-head RMSNorm on the way into a paged KV cache.
//
// For token t of sequence b with own index j (position p = prefix + j), head by head:
//   x' = x * (1 / sqrt(mean(x^2) + eps)) * w                      (q and k, with norm weights)
//   a_i = 2 pi frac(p * turns[i]);  (x1, x2) -> (x1 cos a - x2 sin a, x2 cos a + x1 sin a) * attn_factor
// q goes to q_out, k and v to row j of the sequence's pages, each value rounded once.  The position
// times turns[i] is formed and reduced to (-1/2, 1/2] turn in float64: a float32 product at position 10^6
// is off by up to 0.06 rad, the float64 one by 10^-9.
//
// A workgroup takes one token and up to 4 waves' worth of head rows: a row is D / 8 lanes of 8 values
// (16-byte loads and stores of 16-bit types), so a wave holds 4 rows of 128.  The cosines of the token are
// computed once a workgroup into LDS.  HBM-bound from some thousand tokens on (4300 tokens of 48 rows of 128,
// fp16: 26 us, 4.0 TB/s), a chain of latencies (sequence, page id, row) below (64 tokens: 3.4 us).  Three rows a
// thread, all on their way at once, measured the same there and slower for 640 tokens (8.4 us against 6.8);
// workgroups of 512 threads 29.9 us, of 64 28, loads that leave the caches alone 33.
#include "kv.h"
#include "launch.h"

namespace pgmoe {

constexpr int kAppendThreads = 256;
constexpr int kMaxHalf = 128;  // rot_dim / 2 at head_dim 256

struct AppendArgs {
    KvCache C;
    KvBatch B;
    const void* src[3];
    int64_t tok[3], head[3];
    int sdt, T, hq, rot, interleaved;
    const double* turns;
    float attn_factor, eps;
    const float* norm[2];
    uint16_t* q_out;
};

__device__ __forceinline__ void load8(const void* p, int dt, int64_t at, float (&x)[8]) {
    if (dt == PGMOE_DT_F32) {
        const float4* q = (const float4*)((const float*)p + at);
        const float4 a = q[0], b = q[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        return;
    }
    const uint4 u = *(const uint4*)((const uint16_t*)p + at);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (dt == PGMOE_DT_F16) {
            x[2 * i] = lo_half(w[i]);
            x[2 * i + 1] = hi_half(w[i]);
        } else {
            x[2 * i] = __builtin_bit_cast(float, w[i] << 16);
            x[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
        }
    }
}

template <int D, bool BF16>
__global__ __launch_bounds__(kAppendThreads) void rope_append_kernel(const AppendArgs A) {
    constexpr int LPR = D / 8;              // lanes a row
    constexpr int RPB = kAppendThreads / LPR;  // rows a workgroup
    __shared__ float2 s_turn[kMaxHalf];
    __shared__ int s_cnt[kAppendThreads / 64];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int row = blockIdx.y * RPB + tid / LPR, e0 = (tid % LPR) * 8;
    const int rows = A.hq + 2 * A.C.heads;

    // the row's values are on their way while its place is looked up
    const int kind = row < A.hq ? 0 : row < A.hq + A.C.heads ? 1 : 2;
    const int h = kind == 0 ? row : kind == 1 ? row - A.hq : row - A.hq - A.C.heads;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (row < rows) load8(A.src[kind], A.sdt, (int64_t)t * A.tok[kind] + (int64_t)h * A.head[kind] + e0, x);

    int b = t, lo = t, hi = t + 1;
    if (A.B.q_start) {  // the last sequence that begins at or before t
        int n = 0;
        for (int i = tid; i < A.B.seqs; i += kAppendThreads) n += A.B.q_start[i] <= t;
        n = (int)group_sum<64>((float)n);  // at most 4096: exact
        if (lane == 0) s_cnt[tid >> 6] = n;
        __syncthreads();
        b = s_cnt[0] + s_cnt[1] + s_cnt[2] + s_cnt[3] - 1;
        if (b < 0) return;
        seq_tokens(A.B, b, A.T, lo, hi);
    }
    if (b >= A.B.seqs || t < lo || t >= hi) return;  // behind the last sequence
    int len = A.B.lens[b];
    len = len < 0 ? 0 : len;
    const int64_t j = (int64_t)len - (hi - t);
    const int half = A.rot >> 1;
    if (tid < half) {
        const double a = (double)(A.B.prefix + j) * A.turns[tid];
        float s, c;
        sincospif(2.0f * (float)(a - rint(a)), &s, &c);
        s_turn[tid] = make_float2(c * A.attn_factor, s * A.attn_factor);
    }
    if (half) __syncthreads();

    if (kind < 2) {
        const float* w = A.norm[kind];
        if (w) {
            float sq = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) sq = __builtin_fmaf(x[i], x[i], sq);
            sq = group_sum<LPR>(sq);
            const float r = 1.0f / sqrtf(sq / (float)D + A.eps);
            const float4 w0 = *(const float4*)(w + e0), w1 = *(const float4*)(w + e0 + 4);
            const float wv[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * r * wv[i];
        }
        if (A.interleaved) {
            if (e0 < A.rot) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 cs = s_turn[(e0 >> 1) + i];
                    const float p = x[2 * i], q = x[2 * i + 1];
                    x[2 * i] = p * cs.x - q * cs.y;
                    x[2 * i + 1] = q * cs.x + p * cs.y;
                }
            }
        } else if (A.rot) {
            // the other half of the pair sits half / 8 lanes away (half is a multiple of 8)
            const bool first = e0 < half, in = e0 < A.rot;
            const int other = in ? (first ? lane + (half >> 3) : lane - (half >> 3)) : lane;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = __shfl(x[i], other);
                if (in) {
                    const float2 cs = s_turn[(first ? e0 : e0 - half) + i];
                    x[i] = first ? x[i] * cs.x - y * cs.y : x[i] * cs.x + y * cs.y;
                }
            }
        }
    }
    if (row >= rows) return;
    uint4 o;
    uint32_t* ow = (uint32_t*)&o;
#pragma unroll
    for (int i = 0; i < 4; ++i) ow[i] = to16<BF16>(x[2 * i]) | (uint32_t)to16<BF16>(x[2 * i + 1]) << 16;
    if (kind == 0) {
        *(uint4*)(A.q_out + ((int64_t)t * A.hq + h) * D + e0) = o;
        return;
    }
    const int64_t pi = j >> A.C.page_shift;
    if (j < 0 || pi >= A.B.max_pages) return;
    const int page = A.B.table[(int64_t)b * A.B.table_stride + pi];
    if (page < 0 || page >= A.C.n_pages) return;
    const int64_t at = (int64_t)page * A.C.page_stride + (int64_t)h * A.C.head_stride +
                       (j & ((1 << A.C.page_shift) - 1)) * A.C.row_stride + e0;
    *(uint4*)((kind == 1 ? A.C.k : A.C.v) + at) = o;
}

int launch_rope_append(const KvCache& C, const KvBatch& B, const void* const (&src)[3], const int64_t (&tok)[3],
                       const int64_t (&head)[3], int sdt, int T, int hq, const double* turns, int rot, int interleaved,
                       float attn_factor, const float* q_norm, const float* k_norm, float eps, uint16_t* q_out,
                       hipStream_t st) {
    if (T == 0) return PGMOE_OK;
    AppendArgs A{C, B, {src[0], src[1], src[2]}, {tok[0], tok[1], tok[2]}, {head[0], head[1], head[2]}, sdt, T, hq, rot,
                 interleaved, turns, attn_factor, eps, {q_norm, k_norm}, q_out};
    const int rpb = kAppendThreads / (C.dim / 8);
    const dim3 grid(T, div_up(hq + 2 * C.heads, rpb)), block(kAppendThreads);
#define APPEND(D)                                                                   \
    do {                                                                            \
        if (C.bf16)                                                                 \
            PG_LAUNCH((rope_append_kernel<D, true>), grid, block, 0, st, A);        \
        else                                                                        \
            PG_LAUNCH((rope_append_kernel<D, false>), grid, block, 0, st, A);       \
    } while (0)
    if (C.dim == 64)
        APPEND(64);
    else if (C.dim == 128)
        APPEND(128);
    else
        APPEND(256);
#undef APPEND
    return check_launch("rope_append");
}

}  // namespace pgmoe
