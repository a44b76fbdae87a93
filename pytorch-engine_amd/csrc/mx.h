// Microscaled blocks (mx.hip, mx_linear.hip): 32 values along a row share a power of two.
#pragma once

#include "kv.h"

namespace pgmoe {

struct MxRows {  // validated in api.hip
    uint8_t* codes;
    uint8_t* scales;
    int64_t code_stride, scale_stride;  // bytes
    int rows, cols;
    int e2m1;
};
struct MxFloats {
    const void* p;
    int64_t stride;  // elements
    int dt;
};

int launch_mx_quantize(const MxFloats& x, const MxRows& y, hipStream_t st);
int launch_mx_dequantize(const MxRows& x, void* out, int odt, hipStream_t st);
int launch_mx_act_mul(const MxFloats& gate, const MxFloats& up, int act, const MxRows& y, hipStream_t st);
int launch_add_rmsnorm_mx(const void* x, int xdt, const void* delta, int ddt, const float* w, float eps, float* h_out,
                          const MxRows& y, hipStream_t st);
// The packed weights of a product: bytes, and their making from blocks of rows.
int64_t mx_packed_bytes(int64_t rows, int64_t cols);
int launch_mx_pack(const MxRows& w, uint8_t* dst, hipStream_t st);
struct MxLinear {
    const uint8_t* w;  // packed
    int N, K, M;
    MxRows x;          // activations in blocks
    const float* bias;
    void* out;
    int odt;
    bool wide;  // no product of a sum is cut above 2^-24 of its neighbours
};
constexpr int kMxFewRows = 16;  // up to so many rows are read against weights in registers
// Values of them become blocks inside the product where a workgroup keeps its rows; longer ones would become them again for
// every 16 outputs (1 x 12288 x 4096 16.1 us; in a launch of their own before, as more rows' are, 11).  Every workgroup makes all the
// blocks, so more rows gain less; us inside / in a launch before, in a captured graph, fp16 values to 8 bits, K = 4096:
//   outputs    1 row      8 rows     12 rows    16 rows
//   4096       4.5/7.0    6.7/7.5    8.1/8.1    9.1/8.5
//   12288      7.8/9.7    9.3/10.8   11.3/11.4  13.3/12.4
//   24576      12.1/14.1  13.2/15.2  15.9/16.2  17.5/17.2
// From 13 rows on the launch before is up to 0.9 us less; outside a graph it costs as much on the host.
inline bool mx_values_inside(int64_t rows, int64_t cols) { return rows <= kMxFewRows && cols <= 4096; }
int launch_mx_linear(const MxLinear& L, hipStream_t st);
// L.x: where the blocks of more rows go.
int launch_mx_linear_values(const MxLinear& L, const MxFloats& F, hipStream_t st);

// ---------------------------------------------------------------- blocks in registers
constexpr int kMxExpE4M3 = 8, kMxExpE2M1 = 2;  // exponents of the formats' largest powers of two

// Rows of one launch are numbered chunk by chunk, below 2^31 of them; n / d for such n.
struct FastDiv {
    uint32_t d, m, s;
    void set(uint32_t by) {
        d = by;
        uint32_t l = 0;
        while ((1ull << l) < by) ++l;
        m = (uint32_t)(((1ull << (31 + l)) + by - 1) / by);
        s = 31 + l;
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * m) >> s); }
};

// The codes of N values of a lane, N * LPB = 32 in the LPB lanes of a block (aligned lanes, all of the wave
// active), and the block's scale byte.  The scale is taken from the exponent bits of the largest magnitude, so
// scaling is exact; a block with an infinity or NaN gets byte 255 (NaN) and codes 0.
template <bool E2M1, int N>
__device__ __forceinline__ void mx_encode(float (&v)[N], uint32_t (&code)[E2M1 ? (N + 7) / 8 : N / 4], int& scale) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
    if constexpr (N <= 16) m = max(m, xor_lane_u<1>(m));
    if constexpr (N <= 8) m = max(m, xor_lane_u<2>(m));
    if constexpr (N <= 4) m = max(m, xor_lane_u<4>(m));
    const bool bad = m >= 0x7f800000u;
    const int e = max((int)(m >> 23) - (E2M1 ? kMxExpE2M1 : kMxExpE4M3), 0);
    if (__builtin_expect(bad, 0)) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0.0f;
    }
    scale = bad ? 255 : e;
    const float by = __builtin_bit_cast(float, (uint32_t)e << 23);  // 2^E as the conversions take it, 0 for 2^-127
    if constexpr (E2M1) {  // to nearest even, saturating
#pragma unroll
        for (int w = 0; w < (N + 7) / 8; ++w) {
            uint32_t c = 0;
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * w], v[8 * w + 1], by, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * w + 2], v[8 * w + 3], by, 1);
            if constexpr (N >= 8) {
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * w + 4], v[8 * w + 5], by, 2);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * w + 6], v[8 * w + 7], by, 3);
            }
            code[w] = c;
        }
    } else {  // to nearest even; past 464 2^E the conversion gives NaN, so the values are held to 448 2^E before it
        const float top = ldexpf(448.0f, e - 127);
        typedef short short2v __attribute__((ext_vector_type(2)));
        auto at = [&](int i) { return __builtin_amdgcn_fmed3f(v[i], -top, top); };
#pragma unroll
        for (int w = 0; w < N / 4; ++w) {
            short2v c = {0, 0};
            c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, at(4 * w), at(4 * w + 1), by, false);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, at(4 * w + 2), at(4 * w + 3), by, true);
            code[w] = __builtin_bit_cast(uint32_t, c);
        }
    }
}

}  // namespace pgmoe
