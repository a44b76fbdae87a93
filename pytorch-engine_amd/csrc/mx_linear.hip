// y[m][n] = sum_k x[m][k] w[n][k] (+ bias[n]): activations in 8- or 4-bit blocks, weights in 4-bit blocks.
//
// One v_mfma_scale_f32_16x16x128_f8f6f4 forms 16 weight rows x 16 activation rows over 128 inputs and multiplies each
// block of 32 by both its powers of two on the way, in fp32.  Lane l = 16 g + r of it holds, of row r,
//   4 bits: inputs 32 g .. 32 g + 31 (16 bytes);  8 bits: inputs 16 g .. + 15 and 64 + 16 g .. + 15;
//   the scale of block g;
// and of the result activation row r, weight rows 4 g .. 4 g + 3.
//
// With 4-bit activations the instruction's sums are exact to fp32.  With 8-bit ones it cuts the products of 8 neighbouring
// inputs below 2^-13 of the largest of them (2^10 + 2^-4 gives 2^10) before it adds them up: 1.6e-5 of the outputs'
// 2-norm at 500 x 4096 x 4096, far below what a 16-bit output keeps, and above an fp32 one.  fp32 outputs of 8-bit
// activations therefore take the bf16 instruction (16x16x32, cut at 2^-24): code times power of two is exact in bf16, and
// v_cvt_scalef32_pk_bf16_fp4 / _fp8 makes two of them at once.  Lane l then holds inputs 32 g .. 32 g + 31 of both, eight to
// each of four instructions.
//
// Packed weights: (16 rows x 128 inputs) tiles of 1 KB, lane l's 16 bytes at 16 l, K / 128 steps rounded up to a multiple
// of 4 a row group; behind all of them the scales, 256 bytes for 16 rows x 512 inputs: lane l's four bytes at 4 l,
// one a step.  Inputs past K have code 0 and scale 1 there, and activations past K are read from the same row's valid
// blocks: they count nothing, and their row is NaN anyway where one of them is.
// Reference: the W4A16 product of GGUFQuantLinear (pygguf_engine/quant_kernels.py:1165-1293), whose weights are integers
// with fp16 scales and whose activations stay fp16.
#include "launch.h"
#include "mx.h"

namespace pgmoe {

typedef int intx8 __attribute__((ext_vector_type(8)));

__host__ __device__ inline int mx_groups(int N) { return (N + 15) >> 4; }
__host__ __device__ inline int mx_quads(int K) { return (K + 511) >> 9; }  // units of four steps

int64_t mx_packed_bytes(int64_t rows, int64_t cols) { return ((rows + 15) / 16) * ((cols + 511) / 512) * (4096 + 256); }

// ---------------------------------------------------------------- packing (at load)
__global__ __launch_bounds__(256) void mx_pack_kernel(MxRows w, uint8_t* __restrict__ dst, int64_t lanes) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // (row group, quad, lane)
    if (i >= lanes) return;
    const int Q = mx_quads(w.cols), blocks = w.cols >> 5;
    const int lane = (int)(i & 63), r = lane & 15, g = lane >> 4;
    const int64_t gq = i >> 6;
    const int64_t row = (gq / Q) * 16 + r;
    const int q = (int)(gq % Q);
    uint32_t scale = 0;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int b = 16 * q + 4 * s + g;
        const bool in = row < w.rows && b < blocks;
        uint4 c = make_uint4(0, 0, 0, 0);
        if (in) c = *(const uint4*)(w.codes + row * w.code_stride + 16 * (int64_t)b);
        scale |= (in ? (uint32_t)w.scales[row * w.scale_stride + b] : 127u) << (8 * s);
        *(uint4*)(dst + (gq * 4 + s) * 1024 + lane * 16) = c;
    }
    *(uint32_t*)(dst + (lanes >> 6) * 4096 + gq * 256 + lane * 4) = scale;
}

int launch_mx_pack(const MxRows& w, uint8_t* dst, hipStream_t st) {
    const int64_t lanes = (int64_t)mx_groups(w.rows) * mx_quads(w.cols) * 64;
    PG_LAUNCH(mx_pack_kernel, dim3(div_up(lanes, 256)), dim3(256), 0, st, w, dst, lanes);
    return check_launch("mx_pack");
}

// ---------------------------------------------------------------- pieces of a product
enum MxMode { kS4, kS8, kB8 };  // scaled instruction on 4- or 8-bit activations; bf16 instruction on 8-bit ones

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A lane's activations at step s of its row (kept inside the row).
template <MxMode MODE>
__device__ __forceinline__ intx8 x_frag(const uint8_t* row, int s, int g, int K) {
    const int k = 128 * s + (MODE == kS8 ? 16 : 32) * g;
    const int64_t at = k < K ? k : 0, next = MODE == kB8 ? at + 16 : k + 64 < K ? k + 64 : 0;
    const int4 a = *(const int4*)(row + (MODE == kS4 ? at >> 1 : at));
    intx8 f = {a.x, a.y, a.z, a.w, 0, 0, 0, 0};
    if constexpr (MODE != kS4) {
        const int4 b = *(const int4*)(row + next);
        f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    }
    return f;
}

// 2^(b - 127) as the conversions take it: 0 for 2^-127, 255 for NaN.
__device__ __forceinline__ float scale_of(uint32_t b) { return __builtin_bit_cast(float, b << 23); }

__device__ __forceinline__ bf16x8 bf16_of_e2m1(uint32_t w, float s) {
    struct { bf16x2 v[4]; } o;
    o.v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0);
    o.v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1);
    o.v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2);
    o.v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
    return __builtin_bit_cast(bf16x8, o);
}
__device__ __forceinline__ bf16x8 bf16_of_e4m3(uint32_t lo, uint32_t hi, float s) {
    struct { bf16x2 v[4]; } o;
    o.v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false);
    o.v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
    o.v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false);
    o.v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
    return __builtin_bit_cast(bf16x8, o);
}

// acc[b][t] += w[b] . x[t] over one step of 128 inputs; ws[b]'s byte S and xs[t]'s lowest are the scales.
template <MxMode MODE, int S, int NB, int MT>
__device__ __forceinline__ void mx_step(const int4 (&w)[NB], const int (&ws)[NB], const intx8 (&x)[MT], const int (&xs)[MT],
                                        floatx4 (&acc)[NB][MT]) {
    if constexpr (MODE == kB8) {
        float wf[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) wf[b] = scale_of(((uint32_t)ws[b] >> (8 * S)) & 255u);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bf16x8 v[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b)
                v[b] = bf16_of_e2m1((uint32_t)(j == 0 ? w[b].x : j == 1 ? w[b].y : j == 2 ? w[b].z : w[b].w), wf[b]);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const bf16x8 u = bf16_of_e4m3((uint32_t)x[t][2 * j], (uint32_t)x[t][2 * j + 1], scale_of((uint32_t)xs[t]));
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[b], u, acc[b][t], 0, 0, 0);
            }
        }
    } else {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const intx8 a = {w[b].x, w[b].y, w[b].z, w[b].w, 0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < MT; ++t)
                acc[b][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, x[t], acc[b][t], 4, MODE == kS4 ? 4 : 0, S, ws[b],
                                                                             0, xs[t]);
        }
    }
}

// Outputs n .. n + 3 of row m.
__device__ __forceinline__ void put4(const MxLinear& L, int m, int n, float4 v) {
    float f[4] = {v.x, v.y, v.z, v.w};
    if (L.bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] += n + i < L.N ? L.bias[n + i] : 0.0f;
    }
    const int64_t at = (int64_t)m * L.N + n;
    const bool whole = n + 4 <= L.N && (L.N & 3) == 0;
    if (L.odt == PGMOE_DT_F32) {
        float* o = (float*)L.out + at;
        if (whole) {
            *(float4*)o = make_float4(f[0], f[1], f[2], f[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < L.N) o[i] = f[i];
        }
    } else {
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = L.odt == PGMOE_DT_F16 ? to16<false>(f[i]) : to16<true>(f[i]);
        uint16_t* o = (uint16_t*)L.out + at;
        if (whole) {
            *(uint2*)o = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < L.N) o[i] = (uint16_t)h[i];
        }
    }
}

// ---------------------------------------------------------------- few rows
// A workgroup forms NB row groups of weights for 16 MT activation rows; its W waves take every W-th quad of steps,
// weights and activations straight to registers, and their sums meet in LDS in wave order.
template <MxMode MODE, int MT, int NB, int W>
__global__ __launch_bounds__(64 * W) void mx_thin_kernel(const MxLinear L) {
    __shared__ float4 part[W][NB * MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int G = mx_groups(L.N), Q = mx_quads(L.K), blocks = L.K >> 5;
    const int across = div_up(G, NB);
    const int g0 = (blockIdx.x % across) * NB, m0 = (blockIdx.x / across) * (16 * MT);
    const uint8_t* xr[MT];
    const uint8_t* xsr[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = min(m0 + 16 * t + r, L.M - 1);
        xr[t] = L.x.codes + m * L.x.code_stride;
        xsr[t] = L.x.scales + m * L.x.scale_stride;
    }
    floatx4 acc[NB][MT];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[b][t] = floatx4{0, 0, 0, 0};
    const uint8_t* scales = L.w + (int64_t)G * Q * 4096;
    for (int q = wave; q < Q; q += W) {
        int4 w[4][NB];
        int ws[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int64_t at = (int64_t)min(g0 + b, G - 1) * Q + q;
            ws[b] = *(const int*)(scales + at * 256 + lane * 4);
#pragma unroll
            for (int s = 0; s < 4; ++s) w[s][b] = *(const int4*)(L.w + at * 4096 + s * 1024 + lane * 16);
        }
        auto step = [&](auto sc) {
            constexpr int s = decltype(sc)::value;
            intx8 x[MT];
            int xs[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                x[t] = x_frag<MODE>(xr[t], 4 * q + s, g, L.K);
                xs[t] = xsr[t][min(16 * q + 4 * s + g, blocks - 1)];
            }
            mx_step<MODE, s>(w[s], ws, x, xs, acc);
        };
        step(std::integral_constant<int, 0>());
        step(std::integral_constant<int, 1>());
        step(std::integral_constant<int, 2>());
        step(std::integral_constant<int, 3>());
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < MT; ++t) part[wave][b * MT + t][lane] = make_float4(acc[b][t][0], acc[b][t][1], acc[b][t][2], acc[b][t][3]);
    __syncthreads();
    for (int i = threadIdx.x; i < NB * MT * 64; i += 64 * W) {
        const int bt = i >> 6, l = i & 63;
        float4 v = part[0][bt][l];
#pragma unroll
        for (int k = 1; k < W; ++k) {
            const float4 p = part[k][bt][l];
            v = make_float4(v.x + p.x, v.y + p.y, v.z + p.z, v.w + p.w);
        }
        const int m = m0 + 16 * (bt % MT) + (l & 15), n = 16 * (g0 + bt / MT) + 4 * (l >> 4);
        if (m < L.M && n < L.N) put4(L, m, n, v);
    }
}

template <MxMode MODE>
static int thin_launch(const MxLinear& L, hipStream_t st) {
    const int G = mx_groups(L.N);
#define THIN(MT, NB, W) \
    PG_LAUNCH((mx_thin_kernel<MODE, MT, NB, W>), dim3(div_up(G, NB) * div_up(L.M, 16 * MT)), dim3(64 * W), 0, st, L)
    if (L.M <= 16)
        THIN(1, 2, 8);
    else if (L.M <= 32)
        THIN(2, 2, 8);
    else
        THIN(4, 2, 8);
#undef THIN
    return check_launch("mx_thin");
}

int launch_mx_linear(const MxLinear& L, hipStream_t st) {
    if (L.x.e2m1) return thin_launch<kS4>(L, st);
    return thin_launch<kB8>(L, st);
}

}  // namespace pgmoe
