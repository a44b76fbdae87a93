// Attention of a batch over a paged KV cache whose first keys are shared by every sequence.
//
// The simplest right form: one wave per (query, head) walks the keys with the running maximum and sum of
// the softmax; each lane holds D / 64 columns, a score is a sum over the wave.
#include "kv.h"
#include "launch.h"

namespace pgmoe {

struct AttendArgs {
    KvCache C;
    KvBatch B;
    const uint16_t* q;
    int64_t q_tok, q_head;
    int T, hq;
    float scale;
    uint16_t* out;
    float* lse;
};

template <int D, bool BF16>
__global__ __launch_bounds__(64) void attend_simple_kernel(const AttendArgs A) {
    constexpr int N = D / 64;
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int kvh = h / (A.hq / A.C.heads);
    int b = t, lo = t, hi = t + 1;
    if (A.B.q_start) {
        int n = 0;
        for (int i = lane; i < A.B.seqs; i += 64) n += A.B.q_start[i] <= t;
        b = (int)group_sum<64>((float)n) - 1;
        if (b < 0) return;
        seq_tokens(A.B, b, A.T, lo, hi);
    }
    if (b >= A.B.seqs || t < lo || t >= hi) return;
    int len = A.B.lens[b];
    len = len < 0 ? 0 : len;
    const int cap = A.B.max_pages << A.C.page_shift;
    int64_t seen = (int64_t)len - (hi - t) + 1;
    const bool beyond = seen > cap;
    const int own = seen < 0 ? 0 : seen > cap ? cap : (int)seen;
    const uint16_t* qp = A.q + (int64_t)t * A.q_tok + (int64_t)h * A.q_head;
    float q[N], o[N], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = from16<BF16>(qp[lane + 64 * i]) * A.scale, o[i] = 0.0f;
    const int ps = 1 << A.C.page_shift;
    for (int j = 0; j < A.B.prefix + own; ++j) {
        const int jj = j < A.B.prefix ? j : j - A.B.prefix;
        const int page = j < A.B.prefix ? A.B.prefix_pages[jj >> A.C.page_shift]
                                        : A.B.table[(int64_t)b * A.B.table_stride + (jj >> A.C.page_shift)];
        float s = 0.0f, v[N];
        if (page >= 0 && page < A.C.n_pages) {
            const int64_t at = (int64_t)page * A.C.page_stride + (int64_t)kvh * A.C.head_stride +
                               (int64_t)(jj & (ps - 1)) * A.C.row_stride;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                s = __builtin_fmaf(q[i], from16<BF16>(A.C.k[at + lane + 64 * i]), s);
                v[i] = from16<BF16>(A.C.v[at + lane + 64 * i]);
            }
        } else {
            s = NAN;
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = NAN;
        }
        s = group_sum<64>(s);
        const float mn = fmaxf(m, s);
        const float c = m == -INFINITY ? 0.0f : expf(m - mn), p = expf(s - mn);
        l = l * c + p;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = o[i] * c + p * v[i];
        m = mn;
    }
    const bool empty = A.B.prefix + own == 0;
    if (beyond) l = NAN;
#pragma unroll
    for (int i = 0; i < N; ++i)
        A.out[((int64_t)t * A.hq + h) * D + lane + 64 * i] = empty ? 0 : to16<BF16>(o[i] / l);
    if (A.lse && lane == 0) A.lse[(int64_t)t * A.hq + h] = empty ? -INFINITY : m + logf(l);
}

size_t attend_ws_bytes(const KvCache& C, const KvBatch& B, int T, int hq) { return 0; }

int launch_attend(const KvCache& C, const KvBatch& B, const uint16_t* q, int64_t q_tok, int64_t q_head, int T, int hq,
                  float scale, uint16_t* out, float* lse, void* ws, hipStream_t st) {
    if (T == 0) return PGMOE_OK;
    AttendArgs A{C, B, q, q_tok, q_head, T, hq, scale, out, lse};
    const dim3 grid(T, hq), block(64);
#define ATT(D)                                                                   \
    do {                                                                         \
        if (C.bf16)                                                              \
            PG_LAUNCH((attend_simple_kernel<D, true>), grid, block, 0, st, A);   \
        else                                                                     \
            PG_LAUNCH((attend_simple_kernel<D, false>), grid, block, 0, st, A);  \
    } while (0)
    if (C.dim == 64)
        ATT(64);
    else if (C.dim == 128)
        ATT(128);
    else
        ATT(256);
#undef ATT
    return check_launch("attend");
}

}  // namespace pgmoe
