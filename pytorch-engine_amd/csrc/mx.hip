// Rows to microscaled blocks and back: mx_quantize, the gated activation and the norm with blocks as output.
//
// Block of 32 along a row: E = max(-127, floor(log2 max|x|) - e), e = 8 (e4m3) or 2 (e2m1), held as the byte
// E + 127; codes x / 2^E to the nearest, ties to even, at most 448 or 6 in size.  x / 2^E is exact, so the codes are
// those of the definition whatever the order of the maximum.
// Reference: nothing of this form; the norm is exec_fused_add_rmsnorm (pygguf_engine/quant_kernels.py:1552-1597), the
// activation exec_fused_act_mul_rowscale (:1423-1475), whose output is fp16 with one scale a row.
//
// HBM-bound: values are read once, 16 bytes a lane, codes and scale bytes written once.
#include "launch.h"
#include "mx.h"

namespace pgmoe {

constexpr int kMxThreads = 256;

template <int DT>
struct Chunk {  // what one lane loads at once
    static constexpr int N = DT == PGMOE_DT_F32 ? 4 : 8;
};
template <int DT>
__device__ __forceinline__ void widen(const uint4& u, float (&v)[Chunk<DT>::N]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == PGMOE_DT_F32) {
            v[i] = __builtin_bit_cast(float, w[i]);
        } else if constexpr (DT == PGMOE_DT_F16) {
            v[2 * i] = lo_half(w[i]);
            v[2 * i + 1] = hi_half(w[i]);
        } else {
            v[2 * i] = __builtin_bit_cast(float, w[i] << 16);
            v[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
        }
    }
}

// Codes and scale byte of chunk c of a row (N values a chunk).
template <bool E2M1, int N>
__device__ __forceinline__ void put_codes(const MxRows& y, int64_t row, int c, const uint32_t (&code)[E2M1 ? (N + 7) / 8 : N / 4],
                                          int scale) {
    uint8_t* p = y.codes + row * y.code_stride + (int64_t)c * (E2M1 ? N / 2 : N);
    if constexpr (E2M1 && N == 4)
        *(uint16_t*)p = (uint16_t)code[0];
    else if constexpr ((E2M1 && N == 8) || (!E2M1 && N == 4))
        *(uint32_t*)p = code[0];
    else
        *(uint2*)p = make_uint2(code[0], code[1]);
    constexpr int LPB = 32 / N;
    if (c % LPB == 0) y.scales[row * y.scale_stride + c / LPB] = (uint8_t)scale;
}

// silu(g) = g / (1 + 2^-z) with z = log2(e) g, gelu(g) the same with z = 2 log2(e) sqrt(2 / pi) (g + 0.044715 g^3): no
// difference of near values for negative g.  The hardware's power of two and reciprocal are good to 2^-23 each, where codes
// hold 4 bits; what rounding z = g slope leaves out (|z| 2^-24 of the value) is put back to first order.
constexpr float kFarGate = 120.0f;  // |z| past it: 2^-z nears the end of fp32's range
constexpr float kLn2 = 0.69314718f;
template <int ACT>
struct Gate {
    static constexpr float kSlope = ACT ? 2.30220819813f : 1.44269504089f;   // z / g at 0, as fp32
    static constexpr float kRest = ACT ? 1.29484e-8f : 1.92596e-8f;          // and what is left
    float slope, z;
    __device__ __forceinline__ explicit Gate(float g) {
        slope = ACT ? __builtin_fmaf(0.102943239579f, g * g, kSlope) : kSlope;
        z = g * slope;
    }
    // z - from, to more bits than z has
    __device__ __forceinline__ float beyond(float g, float from) const {
        return __builtin_fmaf(g, kRest, __builtin_fmaf(g, slope, -from));
    }
    __device__ __forceinline__ float act(float g) const {
        float t = __builtin_amdgcn_exp2f(-z);
        t = __builtin_fmaf(-kLn2 * t, beyond(g, z), t);
        return g * __builtin_amdgcn_rcpf(1.0f + t);
    }
};
// act(g) u for z past kFarGate, where 1 + 2^-z is 1 to fp32, or 2^-z: g u, or g u 2^z, the power in parts so that none of them
// leaves the range before the product does (g = -100 is worth 7e-4 beside u = 2e38).
template <int ACT>
__device__ __forceinline__ float gated_far(float g, const Gate<ACT>& a, float u) {
    if (a.z > 0) return g * u;
    const bool gone = a.z < -400.0f;  // of any u
    const float n = gone ? -400.0f : rintf(a.z), f = gone ? 0.0f : a.beyond(g, n);
    return g * ldexpf(__builtin_amdgcn_exp2f(f), -120) * ldexpf(u, (int)n + 120);
}

// ACT < 0: the blocks of x; 0: of silu(x) u; 1: of gelu(x) u (tanh form).  A chunk a thread: with four (their loads on the way
// at once) 4096 x 12288 fp16 took as long, 28.8 us for 28.1 (5.4 TB/s) and 48.1 for 45.8 gated (41 to 42 alone, 6.1 TB/s), 64 x 4096
// 3.3 for 2.7.  Far gates are looked for once a chunk, by the largest |z|: a flag a gate cost silu 3 us of 41.
template <int DT, bool E2M1, int ACT>
__global__ __launch_bounds__(kMxThreads) void mx_rows_kernel(const void* __restrict__ x, int64_t xs, const void* __restrict__ u,
                                                            int64_t us, FastDiv cpr, uint32_t chunks, MxRows y) {
    constexpr int N = Chunk<DT>::N;
    constexpr int B = DT == PGMOE_DT_F32 ? 4 : 2;
    const uint32_t own = blockIdx.x * (uint32_t)kMxThreads + threadIdx.x;
    const uint32_t n = min(own, chunks - 1);  // lanes past the end repeat the last chunk: whole waves meet in mx_encode
    const uint32_t row = cpr.div(n), col = n - row * cpr.d;
    const uint4 a = *(const uint4*)((const uint8_t*)x + ((int64_t)row * xs + (int64_t)col * N) * B);
    float v[N];
    if constexpr (ACT >= 0) {
        const uint4 b = *(const uint4*)((const uint8_t*)u + ((int64_t)row * us + (int64_t)col * N) * B);
        float w[N];
        widen<DT>(a, v);
        widen<DT>(b, w);
        float gu[N], most = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const Gate<ACT> gate(v[i]);
            most = fmaxf(most, fabsf(gate.z));
            gu[i] = gate.act(v[i]) * w[i];
        }
        if (__builtin_expect(most > kFarGate, 0)) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const Gate<ACT> gate(v[i]);
                if (fabsf(gate.z) > kFarGate) gu[i] = gated_far<ACT>(v[i], gate, w[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = gu[i];
    } else {
        widen<DT>(a, v);
    }
    uint32_t code[E2M1 ? (N + 7) / 8 : N / 4];
    int scale;
    mx_encode<E2M1, N>(v, code, scale);
    if (own < chunks) put_codes<E2M1, N>(y, row, (int)col, code, scale);
}

// 4096 x 4096 to fp16: 9.7 us (5.2 TB/s) from 8 bits, 8.9 (4.8) from 4; 12288 x 4096 of 4 bits to fp32 36.5 (6.2).
template <bool E2M1>
__global__ __launch_bounds__(kMxThreads) void mx_dequantize_kernel(MxRows x, FastDiv cpr, uint32_t chunks, void* __restrict__ out,
                                                                  int odt) {
    const uint32_t n = blockIdx.x * (uint32_t)kMxThreads + threadIdx.x;
    if (n >= chunks) return;
    const int64_t row = cpr.div(n);
    const int c = (int)(n - (uint32_t)row * cpr.d);  // chunk of 8 values
    const int e = x.scales[row * x.scale_stride + c / 4];
    const uint8_t* p = x.codes + row * x.code_stride + (int64_t)c * (E2M1 ? 4 : 8);
    float v[8];
    if constexpr (E2M1) {
        const uint32_t w = *(const uint32_t*)p;
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
        const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
        v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = d[0], v[5] = d[1], v[6] = f[0], v[7] = f[1];
    } else {
        const uint2 w = *(const uint2*)p;
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, true);
        const auto d = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, false), f = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, true);
        v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = d[0], v[5] = d[1], v[6] = f[0], v[7] = f[1];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e == 255 ? __builtin_nanf("") : ldexpf(v[i], e - 127);
    const int64_t at = row * x.cols + 8 * (int64_t)c;
    if (odt == PGMOE_DT_F32) {
        float4* o = (float4*)((float*)out + at);
        o[0] = make_float4(v[0], v[1], v[2], v[3]);
        o[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = odt == PGMOE_DT_F16 ? (uint32_t)to16<false>(v[2 * i]) | (uint32_t)to16<false>(v[2 * i + 1]) << 16
                                       : (uint32_t)to16<true>(v[2 * i]) | (uint32_t)to16<true>(v[2 * i + 1]) << 16;
        *(uint4*)((uint16_t*)out + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ---------------------------------------------------------------- the norm
// h = x + delta, y = h * r * w, r = 1 / sqrt(sum(h^2) / D + eps), the rows of y to blocks in the same registers.  In 64 bits up
// to the codes, whatever the order of the sum: a code is then that of the formula, where roundings to fp32 put one of a million on
// the other side of a border, squares of no row pass the range, and the memory still bounds the time.  h_out is h, rounded once.
// A row takes T threads of a workgroup of max(T, 256); thread t owns the 4-value chunks t, t + T, ...: eight
// neighbouring lanes hold a block.  VPT > 0: the row stays in registers (D <= 4 T VPT), its loads all on the way before
// the first is used; VPT == 0: it is read twice.
struct Doubles {
    double v[4];
};
// group_sum in 64 bits: over G aligned lanes, each with the sum.
template <int G>
__device__ __forceinline__ double lanes_sum(double v) {
    if constexpr (G > 1) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        v += __builtin_bit_cast(double, (uint64_t)xor_lane_u<G / 2>((uint32_t)(b >> 32)) << 32 | xor_lane_u<G / 2>((uint32_t)b));
        return lanes_sum<G / 2>(v);
    }
    return v;
}
// d in fp32 for a further rounding to fewer bits: what does not fit sets the last bit (the other 29 of d's 52 are cut), so that
// no value moves onto a border between codes.
__device__ __forceinline__ float to_odd(double d) {
    uint64_t b = __builtin_bit_cast(uint64_t, d);
    if ((uint32_t)b & 0x1fffffffu) b = (b & ~(uint64_t)0x1fffffff) | 0x20000000u;
    return (float)__builtin_bit_cast(double, b);
}

template <int T, int VPT, bool E2M1>
__global__ __launch_bounds__(T < 256 ? 256 : T, T == 1024 ? 8 : 1) void add_rmsnorm_mx_kernel(const void* __restrict__ x, int xdt,
                                                                          const void* __restrict__ delta, int ddt,
                                                                          const float* __restrict__ w, float eps, double inv_cols,
                                                                          float* __restrict__ h_out, MxRows y) {
    constexpr int RPB = T < 256 ? 256 / T : 1, W = T / 64;  // rows a workgroup, waves a row
    __shared__ double wsum[W > 1 ? W : 1];
    const int t = threadIdx.x % T, n4 = y.cols >> 2;
    const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / T;
    if (row >= y.rows) return;  // whole waves; with one row a workgroup none
    const int64_t row4 = row * n4;
    auto load = [&](const void* p, int dt, int64_t i4) {
        if (dt == PGMOE_DT_F32) return ((const uint4*)p)[i4];
        const uint2 u = ((const uint2*)p)[i4];
        return make_uint4(u.x, u.y, 0, 0);
    };
    auto widen4 = [&](const uint4& u, int dt) {
        auto f = [](uint32_t v) { return __builtin_bit_cast(float, v); };
        if (dt == PGMOE_DT_F32) return make_float4(f(u.x), f(u.y), f(u.z), f(u.w));
        if (dt == PGMOE_DT_F16) return make_float4(lo_half(u.x), hi_half(u.x), lo_half(u.y), hi_half(u.y));
        return make_float4(f(u.x << 16), f(u.x & 0xffff0000u), f(u.y << 16), f(u.y & 0xffff0000u));
    };
    auto wide = [](float4 a) { return Doubles{{(double)a.x, (double)a.y, (double)a.z, (double)a.w}}; };
    auto add = [](Doubles a, Doubles b) { return Doubles{{a.v[0] + b.v[0], a.v[1] + b.v[1], a.v[2] + b.v[2], a.v[3] + b.v[3]}}; };
    auto squares = [](double acc, Doubles h) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = __builtin_fma(h.v[i], h.v[i], acc);
        return acc;
    };
    auto total = [&](double acc) {
        acc = lanes_sum<64>(acc);
        if constexpr (W > 1) {
            if ((threadIdx.x & 63) == 0) wsum[threadIdx.x >> 6] = acc;
            __syncthreads();
            acc = lanes_sum<W>(wsum[threadIdx.x % W]);
        }
        // the hardware's 1 / sqrt is good to 2^-24 or better, one step of Newton's to 2^-47; 0 and infinity stand
        const double m = __builtin_fma(acc, inv_cols, (double)eps), r = __builtin_amdgcn_rsq(m);
        return m > 0.0 && m < (double)__builtin_inff() ? __builtin_fma(0.5 * r, __builtin_fma(-m * r, r, 1.0), r) : r;
    };
    auto put_h = [&](int c, Doubles h) {
        if (h_out && c < n4) ((float4*)h_out)[row4 + c] = make_float4((float)h.v[0], (float)h.v[1], (float)h.v[2], (float)h.v[3]);
    };
    auto put = [&](int c, Doubles h, Doubles g, double r) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_odd((h.v[i] * r) * g.v[i]);
        uint32_t code[1];
        int scale;
        mx_encode<E2M1, 4>(v, code, scale);
        if (c < n4) put_codes<E2M1, 4>(y, row, c, code, scale);
    };
    if constexpr (VPT > 0) {
        auto at = [&](int j) { return min(t + T * j, n4 - 1); };  // chunks past the row repeat its last one
        uint4 xr[VPT], dr[VPT];
        constexpr bool LATE = T * VPT > 2048;  // weights asked for behind the sum: two workgroups a CU where a row takes most registers
        float4 g[VPT];
        if (xdt == PGMOE_DT_F32) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) xr[j] = load(x, PGMOE_DT_F32, row4 + at(j));
        } else {
#pragma unroll
            for (int j = 0; j < VPT; ++j) xr[j] = load(x, PGMOE_DT_F16, row4 + at(j));
        }
        if (delta) {
            if (ddt == PGMOE_DT_F32) {
#pragma unroll
                for (int j = 0; j < VPT; ++j) dr[j] = load(delta, PGMOE_DT_F32, row4 + at(j));
            } else {
#pragma unroll
                for (int j = 0; j < VPT; ++j) dr[j] = load(delta, PGMOE_DT_F16, row4 + at(j));
            }
        }
        if constexpr (!LATE) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) g[j] = ((const float4*)w)[at(j)];
        }
        __builtin_amdgcn_sched_barrier(0);
        auto h_of = [&](int j) {
            const Doubles h = wide(widen4(xr[j], xdt));
            return delta ? add(h, wide(widen4(dr[j], ddt))) : h;
        };
        double acc = 0.0;
        Doubles h[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            h[j] = h_of(j);
            if (t + T * j < n4) acc = squares(acc, h[j]);
        }
        const double r = total(acc);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int c = t + T * j;
            if constexpr (LATE) g[j] = ((const float4*)w)[at(j)];
            put_h(c, h[j]);
            put(c, h[j], wide(g[j]), r);
        }
    } else {
        auto h_at = [&](int c) {
            const Doubles h = wide(widen4(load(x, xdt, row4 + c), xdt));
            return delta ? add(h, wide(widen4(load(delta, ddt, row4 + c), ddt))) : h;
        };
        double acc = 0.0;
        for (int c = t; c < n4; c += T) acc = squares(acc, h_at(c));
        const double r = total(acc);
        for (int c0 = 0; c0 < n4; c0 += T) {  // every lane, as blocks meet across lanes
            const int c = c0 + t, k = min(c, n4 - 1);
            const Doubles h = h_at(k);
            put_h(c, h);
            put(c, h, wide(((const float4*)w)[k]), r);
        }
    }
}

// ---------------------------------------------------------------- launches
// One launch numbers fewer than 2^31 chunks: calls of more rows are cut into several.
template <class F>
static int by_rows(int64_t rows, int cpr, F launch) {
    const int64_t most = std::max<int64_t>(1, 0x7fffffff / cpr);
    for (int64_t r = 0; r < rows; r += most) {
        const int rc = launch(r, std::min(most, rows - r));
        if (rc) return rc;
    }
    return PGMOE_OK;
}

static MxRows rows_from(const MxRows& y, int64_t r, int64_t n) {
    MxRows z = y;
    z.codes += r * y.code_stride;
    z.scales += r * y.scale_stride;
    z.rows = (int)n;
    return z;
}

template <int DT, bool E2M1, int ACT>
static int rows_launch(const MxFloats& x, const MxFloats& u, const MxRows& y, hipStream_t st) {
    constexpr int N = Chunk<DT>::N, B = DT == PGMOE_DT_F32 ? 4 : 2;
    FastDiv cpr;
    cpr.set(y.cols / N);
    return by_rows(y.rows, y.cols / N, [&](int64_t r, int64_t n) {
        const uint32_t chunks = (uint32_t)(n * (y.cols / N));
        const void* xp = (const uint8_t*)x.p + r * x.stride * B;
        const void* up = u.p ? (const uint8_t*)u.p + r * u.stride * B : nullptr;
        const MxRows z = rows_from(y, r, n);
        PG_LAUNCH((mx_rows_kernel<DT, E2M1, ACT>), dim3(div_up(chunks, kMxThreads)), dim3(kMxThreads), 0, st, xp, x.stride, up,
                  u.stride, cpr, chunks, z);
        return check_launch("mx_rows");
    });
}

template <int ACT>
static int rows_by_type(const MxFloats& x, const MxFloats& u, const MxRows& y, hipStream_t st) {
#define ROWS(DT) return y.e2m1 ? rows_launch<DT, true, ACT>(x, u, y, st) : rows_launch<DT, false, ACT>(x, u, y, st)
    if (x.dt == PGMOE_DT_F32) ROWS(PGMOE_DT_F32);
    if (x.dt == PGMOE_DT_F16) ROWS(PGMOE_DT_F16);
    ROWS(PGMOE_DT_BF16);
#undef ROWS
}

int launch_mx_quantize(const MxFloats& x, const MxRows& y, hipStream_t st) {
    return rows_by_type<-1>(x, MxFloats{nullptr, 0, 0}, y, st);
}

int launch_mx_act_mul(const MxFloats& gate, const MxFloats& up, int act, const MxRows& y, hipStream_t st) {
    return act == PGMOE_ACT_SILU ? rows_by_type<0>(gate, up, y, st) : rows_by_type<1>(gate, up, y, st);
}

int launch_mx_dequantize(const MxRows& x, void* out, int odt, hipStream_t st) {
    FastDiv cpr;
    cpr.set(x.cols / 8);
    return by_rows(x.rows, x.cols / 8, [&](int64_t r, int64_t n) {
        const uint32_t chunks = (uint32_t)(n * (x.cols / 8));
        const MxRows z = rows_from(x, r, n);
        void* o = (uint8_t*)out + r * x.cols * (odt == PGMOE_DT_F32 ? 4 : 2);
        const dim3 grid(div_up(chunks, kMxThreads)), block(kMxThreads);
        if (x.e2m1)
            PG_LAUNCH((mx_dequantize_kernel<true>), grid, block, 0, st, z, cpr, chunks, o, odt);
        else
            PG_LAUNCH((mx_dequantize_kernel<false>), grid, block, 0, st, z, cpr, chunks, o, odt);
        return check_launch("mx_dequantize");
    });
}

// Rows of one launch: as many as 2^31 threads.
template <int T, int VPT>
static int norm_launch(const void* x, int xdt, const void* delta, int ddt, const float* w, float eps, float* h_out, const MxRows& y,
                       hipStream_t st) {
    constexpr int RPB = T < 256 ? 256 / T : 1;
    return by_rows(y.rows, T, [&](int64_t r, int64_t n) {
        const MxRows z = rows_from(y, r, n);
        const void* xp = (const uint8_t*)x + r * y.cols * (xdt == PGMOE_DT_F32 ? 4 : 2);
        const void* dp = delta ? (const uint8_t*)delta + r * y.cols * (ddt == PGMOE_DT_F32 ? 4 : 2) : nullptr;
        float* hp = h_out ? h_out + r * y.cols : nullptr;
        const dim3 grid(div_up(n, RPB)), block(T * RPB);
        const double inv = 1.0 / y.cols;
        if (y.e2m1)
            PG_LAUNCH((add_rmsnorm_mx_kernel<T, VPT, true>), grid, block, 0, st, xp, xdt, dp, ddt, w, eps, inv, hp, z);
        else
            PG_LAUNCH((add_rmsnorm_mx_kernel<T, VPT, false>), grid, block, 0, st, xp, xdt, dp, ddt, w, eps, inv, hp, z);
        return check_launch("add_rmsnorm_mx");
    });
}

int launch_add_rmsnorm_mx(const void* x, int xdt, const void* delta, int ddt, const float* w, float eps, float* h_out,
                          const MxRows& y, hipStream_t st) {
    const int n4 = y.cols >> 2;
    // 4 threads' work or less each while it fills workgroups of 256, more threads where a row is a CU's only one: 4096 columns,
    // fp32 and fp32, with 256 / 1024 threads: 1 row 4.3 / 3.4 us, 256 6.3 / 5.3, 700 10.0 / 9.5, 1024 12.0 / 12.6, 4003 38.0
    // (5.6 TB/s) / 42.9; 2048 columns, 1 row 3.0 / 3.1, 1024 7.9 / 9.3.  8192 columns in two chunks a thread or four of half the
    // threads: 1 row 4.5 / 5.0, 4003 both 81.5 (5.2 TB/s); 16384 in registers 156, read twice 205.  In fp32 they took 0.1 to 0.8 us
    // less up to 1024 rows, 1 to 2 % beyond.
#define NORM(T, V) return norm_launch<T, V>(x, xdt, delta, ddt, w, eps, h_out, y, st)
    if (n4 <= 64) NORM(64, 1);
    if (n4 <= 128) NORM(64, 2);
    if (n4 <= 256) NORM(256, 1);
    if (n4 <= 512) NORM(256, 2);
    if (n4 <= 1024 && y.rows > 768) NORM(256, 4);
    if (n4 <= 1024) NORM(1024, 1);
    if (n4 <= 2048) NORM(1024, 2);
    if (n4 <= 4096) NORM(1024, 4);
    NORM(1024, 0);
#undef NORM
}

}  // namespace pgmoe
