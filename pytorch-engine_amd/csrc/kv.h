// Paged KV cache and batch descriptions shared by append.hip and attend.hip (validated in api.hip).
#pragma once

#include "common.h"

namespace pgmoe {

typedef __bf16 bf16_t;

struct KvCache {
    uint16_t* k;  // 16-bit elements (fp16 or bf16)
    uint16_t* v;
    int64_t page_stride, head_stride, row_stride;  // elements
    int n_pages, page_shift, heads, dim;
    int bf16;
};
struct KvBatch {
    const int32_t* table;
    const int32_t* lens;
    const int32_t* q_start;
    const int32_t* prefix_pages;
    int64_t table_stride;
    int seqs, max_pages, prefix;
};
constexpr int kMaxSeqs = 4096;

// fp32 -> 16 bits, to nearest even.
template <bool BF16>
__device__ __forceinline__ uint16_t to16(float f) {
    if constexpr (BF16)
        return __builtin_bit_cast(uint16_t, (bf16_t)f);
    else
        return __builtin_bit_cast(uint16_t, (half_t)f);
}
template <bool BF16>
__device__ __forceinline__ float from16(uint16_t b) {
    if constexpr (BF16)
        return __builtin_bit_cast(float, (uint32_t)b << 16);
    else
        return h2f(b);
}

// Rows [lo, hi) of the call's tokens that sequence b holds, kept inside [0, T) whatever q_start holds.
__device__ __forceinline__ void seq_tokens(const KvBatch& B, int b, int T, int& lo, int& hi) {
    if (!B.q_start) {
        lo = b;
        hi = b + 1 < T ? b + 1 : T;
        if (lo > hi) lo = hi;
        return;
    }
    lo = B.q_start[b];
    hi = B.q_start[b + 1];
    lo = lo < 0 ? 0 : lo > T ? T : lo;
    hi = hi < lo ? lo : hi > T ? T : hi;
}

int launch_rope_append(const KvCache& C, const KvBatch& B, const void* const (&src)[3], const int64_t (&tok)[3],
                       const int64_t (&head)[3], int sdt, int T, int hq, const double* turns, int rot, int interleaved,
                       float attn_factor, const float* q_norm, const float* k_norm, float eps, uint16_t* q_out,
                       hipStream_t st);
size_t attend_ws_bytes(const KvCache& C, const KvBatch& B, int T, int hq);
int launch_attend(const KvCache& C, const KvBatch& B, const uint16_t* q, int64_t q_tok, int64_t q_head, int T, int hq,
                  float scale, uint16_t* out, float* lse, void* ws, hipStream_t st);

}  // namespace pgmoe
