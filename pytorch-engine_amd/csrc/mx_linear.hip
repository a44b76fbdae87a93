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
// activations, callers that ask for fp32 sums, and up to 16 rows, where it costs nothing, therefore take the bf16 instruction
// (16x16x32, cut at 2^-24): code times power of two is exact in bf16, and v_cvt_scalef32_pk_bf16_fp4 / _fp8 makes two of them
// at once.  Lane l then holds inputs 32 g .. 32 g + 31 of both, eight to each of four instructions.
//
// Packed weights: (16 rows x 128 inputs) tiles of 1 KB, lane l's 16 bytes at 16 l, K / 128 steps rounded up to a multiple
// of 4 a row group; behind all of them the scales, 256 bytes for 16 rows x 512 inputs: lane l's four bytes at 4 l,
// one a step.  Inputs past K have code 0 and scale 1 there, and activations past K are read from the same row's valid
// blocks with scale 1: they count nothing, and their row is NaN anyway where a code of them is.
// Reference: the W4A16 product of GGUFQuantLinear (pygguf_engine/quant_kernels.py:1165-1293), whose weights are integers
// with fp16 scales and whose activations stay fp16.
#include "launch.h"
#include "mx.h"

namespace pgmoe {

#define PG_INLINE __attribute__((always_inline))

constexpr int kCUs = 256;
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

template <MxMode MODE>
struct XFrag {  // a lane's activations of one step
    int4 a, b;
    __device__ __forceinline__ intx8 operand() const { return intx8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}; }
    __device__ __forceinline__ uint32_t word(int i) const {
        return (uint32_t)(i == 0 ? a.x : i == 1 ? a.y : i == 2 ? a.z : i == 3 ? a.w : i == 4 ? b.x : i == 5 ? b.y : i == 6 ? b.z : b.w);
    }
};
template <>
struct XFrag<kS4> {
    int4 a;
    __device__ __forceinline__ intx8 operand() const { return intx8{a.x, a.y, a.z, a.w, 0, 0, 0, 0}; }
};

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

// The weights of one step as the instructions take them; byte S of ws[b] is their scale.
template <MxMode MODE, int NB>
struct WOps {
    int4 w[NB];
    template <int S>
    __device__ __forceinline__ void set(const int4 (&from)[NB], const int (&)[NB]) {
#pragma unroll
        for (int b = 0; b < NB; ++b) w[b] = from[b];
    }
};
template <int NB>
struct WOps<kB8, NB> {
    bf16x8 v[4][NB];
    template <int S>
    __device__ __forceinline__ void set(const int4 (&from)[NB], const int (&ws)[NB]) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float sw = scale_of(((uint32_t)ws[b] >> (8 * S)) & 255u);
            v[0][b] = bf16_of_e2m1((uint32_t)from[b].x, sw);
            v[1][b] = bf16_of_e2m1((uint32_t)from[b].y, sw);
            v[2][b] = bf16_of_e2m1((uint32_t)from[b].z, sw);
            v[3][b] = bf16_of_e2m1((uint32_t)from[b].w, sw);
        }
    }
};
// acc[b][t] += w[b] . f over one step of 128 inputs; byte S of ws[b] and byte SX of xs are the scales.
template <MxMode MODE, int S, int SX, int NB, int MT>
__device__ __forceinline__ void mx_products(const WOps<MODE, NB>& w, const int (&ws)[NB], int xs, const XFrag<MODE>& f, int t,
                                            floatx4 (&acc)[NB][MT]) {
    if constexpr (MODE == kB8) {
        const float sx = scale_of(((uint32_t)xs >> (8 * SX)) & 255u);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bf16x8 u = bf16_of_e4m3(f.word(2 * j), f.word(2 * j + 1), sx);
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[j][b], u, acc[b][t], 0, 0, 0);
        }
    } else {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const intx8 a = {w.w[b].x, w.w[b].y, w.w[b].z, w.w[b].w, 0, 0, 0, 0};
            acc[b][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, f.operand(), acc[b][t], 4, MODE == kS4 ? 4 : 0, S, ws[b],
                                                                         SX, xs);
        }
    }
}

// Rows of outputs begin at any value, as N is any, and stores of several values take any place (2452 x 288 x 14951 to fp32: 51 us,
// value by value 94; 3024 x 192 x 8131 to fp16 31 and 52; rows at multiples of 16 bytes as before).
// Outputs n .. n + 3 of a row, with their bias; and as 16-bit values.
__device__ __forceinline__ void add_bias(const MxLinear& L, int n, float (&f)[4]) {
    if (L.bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] += n + i < L.N ? L.bias[n + i] : 0.0f;
    }
}
__device__ __forceinline__ uint2 halves(const MxLinear& L, const float (&f)[4]) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = L.odt == PGMOE_DT_F16 ? to16<false>(f[i]) : to16<true>(f[i]);
    return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}
// Outputs n .. n + 3 of row m; WHOLE: all of them are the row's; BITS: 16 where every output of the kernel's has them, 0: either.
template <bool WHOLE, int BITS>
__device__ __forceinline__ void put4(const MxLinear& L, int m, int n, float4 v) {
    float f[4] = {v.x, v.y, v.z, v.w};
    add_bias(L, n, f);
    const int64_t at = (int64_t)m * L.N + n;
    if (BITS == 0 && L.odt == PGMOE_DT_F32) {
        float* o = (float*)L.out + at;
        if (WHOLE || n + 4 <= L.N) {
            __builtin_memcpy(o, f, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (n + i < L.N) o[i] = f[i];
        }
    } else {
        const uint2 h = halves(L, f);
        uint16_t* o = (uint16_t*)L.out + at;
        if (WHOLE || n + 4 <= L.N) {
            __builtin_memcpy(o, &h, 8);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (n + i < L.N) o[i] = (uint16_t)((i < 2 ? h.x : h.y) >> (16 * (i & 1)));
        }
    }
}
// 16-bit outputs of row m of two fragments, n .. n + 15 and n + 16 .. n + 31, of a lane 16 g + r the four at 4 g: after the two
// exchanges it has the eight at 8 g, and a row's 64 bytes go out at once (4096 x 24576 x 4096: 317 us, as 32 bytes 327; 4 bits 230
// and 242).  Stores past the caches made these products 4 % faster and what reads them slower (an FFN of 4096 rows 487 -> 505
// us), so they are ordinary ones.  All lanes take part; all of the outputs are the row's.
__device__ __forceinline__ void put_pair(const MxLinear& L, int m, int n, int g, floatx4 v0, floatx4 v1) {
    float f0[4] = {v0[0], v0[1], v0[2], v0[3]}, f1[4] = {v1[0], v1[1], v1[2], v1[3]};
    add_bias(L, n + 4 * g, f0);
    add_bias(L, n + 16 + 4 * g, f1);
    const uint2 h0 = halves(L, f0), h1 = halves(L, f1);
    auto x = __builtin_amdgcn_permlane32_swap(h0.x, h1.x, false, false);
    auto y = __builtin_amdgcn_permlane32_swap(h0.y, h1.y, false, false);
    x = __builtin_amdgcn_permlane16_swap(x[0], x[1], false, false);
    y = __builtin_amdgcn_permlane16_swap(y[0], y[1], false, false);
    const uint4 h = make_uint4(x[0], y[0], x[1], y[1]);
    if (m < L.M) __builtin_memcpy((uint16_t*)L.out + (int64_t)m * L.N + n + 8 * g, &h, 16);
}

// ---------------------------------------------------------------- up to 16 rows
// A workgroup forms NB times 16 outputs of all rows at a time; its W waves take every W-th quad of steps, weights and activations
// straight to registers, and their sums meet in LDS in wave order.  ONE: a quad is all that a wave has (K <= 512 W): the
// rows stay in registers, and the workgroup goes on to its next 16 outputs, whose weights are asked for during these products
// (rows kept so: 2048 x 151936 35 for 44 us).  They are waited for at the turn's end, before the sums meet: `w = next` is a copy of
// registers there.  Other waves of the CU fill that wait, or nothing does.
// Bound by the weights' arrival and, where they are few, by the latencies of one load, one sum and the launch: us for 1 / 16
// rows of fp16 values to 8 bits, inputs x outputs, weights from memory but for the head's: 4096 x 4096 4.4 / 9.1, 4096 x 24576 12.1
// (4.4 TB/s) / 17.5, 2048 x 151936 27 / 30, 12288 x 4096 10.6 / 15.3 (2.6 of it the blocks' own launch).
// SRC: the rows come in blocks (-1), or (ONE) as values of a PGMOE_DT_* that become blocks here, in LDS, eight values a lane, a
// wave its quad of every row: as much work as there are values.
template <int SRC>
struct ThinX {  // eight values of a row
    static constexpr int N = SRC == PGMOE_DT_F32 ? 2 : 1;
    uint4 v[N];
    __device__ __forceinline__ void load(const uint8_t* row, int chunk) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = ((const uint4*)(row + (int64_t)chunk * (16 * N)))[i];
    }
    __device__ __forceinline__ void widen(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (SRC == PGMOE_DT_F32) {
                    f[4 * i + k] = __builtin_bit_cast(float, w[k]);
                } else if constexpr (SRC == PGMOE_DT_F16) {
                    f[2 * k] = lo_half(w[k]);
                    f[2 * k + 1] = hi_half(w[k]);
                } else {
                    f[2 * k] = __builtin_bit_cast(float, w[k] << 16);
                    f[2 * k + 1] = __builtin_bit_cast(float, w[k] & 0xffff0000u);
                }
            }
        }
    }
};

template <MxMode MODE, int SRC, int W, bool ONE, int NB>
__global__ __launch_bounds__(64 * W, 4 / NB) void mx_thin_kernel(const MxLinear L, const MxFloats F) {
    static_assert(ONE || SRC < 0, "longer rows come in blocks");
    constexpr int ROW = MODE == kS4 ? 256 : 512, WAVE = kMxFewRows * (ROW + 16);  // a quad of a row's codes; of all rows, with scales
    constexpr int SUMS = 2 * W * NB * 1024;
    __shared__ __attribute__((aligned(16))) uint8_t smem[SRC < 0 || SUMS > W * WAVE ? SUMS : W * WAVE];
    auto part = (float4(*)[W][NB][64])smem;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int G = mx_groups(L.N), Q = mx_quads(L.K), last = (L.K >> 5) - 1, waves = min(W, Q);
    const int m = min(r, L.M - 1);  // rows past the last repeat it, blocks past the row's last too: their weights are 0
    const uint8_t* xr = L.x.codes + m * L.x.code_stride;
    const uint8_t* xsr = L.x.scales + m * L.x.scale_stride;
    const uint8_t* scales = L.w + (int64_t)G * Q * 4096;
    struct Weights {
        int4 w[4][NB];
        int s[NB];
    };
    auto load_w = [&](Weights& to, int gb, int q) PG_INLINE {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int64_t at = (int64_t)min(gb * NB + b, G - 1) * Q + min(q, Q - 1);
#pragma unroll
            for (int s = 0; s < 4; ++s) to.w[s][b] = *(const int4*)(L.w + at * 4096 + s * 1024 + lane * 16);
            to.s[b] = *(const int*)(scales + at * 256 + lane * 4);
        }
    };
    struct Rows {
        XFrag<MODE> f[4];
        int s[4];
    };
    auto load_x = [&](Rows& to, int q) PG_INLINE {
        auto block = [&](int s) PG_INLINE { return min(16 * q + 4 * s + g, last); };
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            to.f[s].a = *(const int4*)(xr + (int64_t)block(s) * (MODE == kS4 ? 16 : 32));
            if constexpr (MODE != kS4) to.f[s].b = *(const int4*)(xr + (int64_t)block(s) * 32 + 16);
            to.s[s] = xsr[block(s)];
        }
    };
    // The wave's quad of all rows, as values, to blocks; 16-byte chunk c of row i lies at c ^ i.
    auto encode_x = [&](Rows& to, int q, auto meanwhile) PG_INLINE {
        using X = ThinX<SRC < 0 ? PGMOE_DT_F16 : SRC>;
        constexpr int AHEAD = 8 / X::N;  // rows of values in registers
        X raw[AHEAD];
        uint8_t* own = smem + wave * WAVE;
        const int chunk = min(64 * q + lane, 4 * last + 3);  // past the row's last eight: them again
        auto load_rows = [&](int i0) PG_INLINE {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
                if (i0 + k < L.M) raw[k].load((const uint8_t*)F.p + (i0 + k) * F.stride * (SRC == PGMOE_DT_F32 ? 4 : 2), chunk);
        };
        load_rows(0);
        meanwhile();
        for (int i0 = 0; i0 < L.M; i0 += AHEAD) {
            if (i0) load_rows(i0);
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                if (i0 + k < L.M) {
                    const int i = i0 + k;
                    float v[8];
                    raw[k].widen(v);
                    uint32_t c[MODE == kS4 ? 1 : 2];
                    int scale;
                    mx_encode<MODE == kS4, 8>(v, c, scale);
                    if constexpr (MODE == kS4)
                        *(uint32_t*)(own + i * ROW + 16 * ((lane >> 2) ^ i) + 4 * (lane & 3)) = c[0];
                    else
                        *(uint2*)(own + i * ROW + 16 * ((lane >> 1) ^ i) + 8 * (lane & 1)) = make_uint2(c[0], c[1]);
                    if ((lane & 3) == 0) own[kMxFewRows * ROW + i * 16 + (lane >> 2)] = (uint8_t)scale;
                }
            }
        }
        // Lanes read what others of the wave wrote: its accesses to LDS run in their order, which the compiler has to keep.
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int b = 4 * s + g;
            if constexpr (MODE == kS4) {
                to.f[s].a = *(const int4*)(own + m * ROW + 16 * (b ^ m));
            } else {
                to.f[s].a = *(const int4*)(own + m * ROW + 16 * ((2 * b) ^ m));
                to.f[s].b = *(const int4*)(own + m * ROW + 16 * ((2 * b + 1) ^ m));
            }
            to.s[s] = own[kMxFewRows * ROW + m * 16 + b];
        }
    };
    auto products = [&](const Weights& w, const Rows& x, int q, floatx4 (&acc)[NB][1]) PG_INLINE {
        auto step = [&](auto sc) PG_INLINE {
            constexpr int s = decltype(sc)::value;
            WOps<MODE, NB> ops;
            ops.template set<s>(w.w[s], w.s);
            // 1 past the row, where the weights' 0 is to meet no infinity (chosen here, so that no load waits for it)
            const int xs = 16 * q + 4 * s + g <= last ? x.s[s] : 127;
            mx_products<MODE, s, 0>(ops, w.s, xs, x.f[s], 0, acc);
        };
        step(std::integral_constant<int, 0>());
        step(std::integral_constant<int, 1>());
        step(std::integral_constant<int, 2>());
        step(std::integral_constant<int, 3>());
    };
    Weights w;
    Rows x;
    if (wave < waves) {
        if constexpr (SRC >= 0) {
            encode_x(x, wave, [&]() PG_INLINE { load_w(w, blockIdx.x, wave); });
        } else {
            if constexpr (ONE || NB > 1) load_x(x, wave);
            load_w(w, blockIdx.x, wave);
        }
    }
    if constexpr (SRC >= 0) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the sums go to the same places
    int turn = 0;
    for (int gb = blockIdx.x; gb * NB < G; gb += gridDim.x, ++turn) {
        if (wave < waves) {
            floatx4 acc[NB][1];
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b][0] = floatx4{0, 0, 0, 0};
            if constexpr (ONE) {
                Weights next;
                load_w(next, gb + gridDim.x, wave);
                products(w, x, wave, acc);
                w = next;
            } else {
#pragma unroll 1
                // The next quad's weights, or the next outputs' first, are asked for during these products: where NB is 1 behind
                // most of them, and each step's rows right before their use, so that a quad shows a latency or two.
                for (int q = wave; q < Q; q += W) {
                    Weights next;
                    Rows then;
                    const bool more = q + W < Q;
                    if constexpr (NB > 1) load_x(then, more ? q + W : wave);
                    load_w(next, more ? gb : gb + gridDim.x, more ? q + W : wave);
                    if constexpr (NB == 1) load_x(x, q);
                    products(w, x, q, acc);
                    w = next;
                    if constexpr (NB > 1) x = then;
                }
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
                part[turn & 1][wave][b][lane] = make_float4(acc[b][0][0], acc[b][0][1], acc[b][0][2], acc[b][0][3]);
        }
        // (not for loads and stores, though the copy above has waited for the loads; a buffer is written again behind the next
        // barrier, which its reader passes too)
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (wave != (turn * NB + b) % W) continue;
            float4 v = part[turn & 1][0][b][lane];
            for (int k = 1; k < waves; ++k) {
                const float4 p = part[turn & 1][k][b][lane];
                v = make_float4(v.x + p.x, v.y + p.y, v.z + p.z, v.w + p.w);
            }
            const int n = 16 * (gb * NB + b) + 4 * g;
            if (r < L.M && n < L.N) put4<false, 0>(L, r, n, v);
        }
    }
}

// Workgroups: as many as stay on the card at once where each goes on to further outputs.  Four waves where K has no more
// quads (8 rows of 2048 inputs, 151936 outputs: 60 us with eight waves, half of them idle).  Longer rows: two groups of outputs at
// a time, on rows that are read once for both, with the next quad's on their way, where that leaves a workgroup to every CU
// (8 bits, 1 / 16 rows, 28672 x 8192 23.8 / 33 us for 28.7 / 50 one by one; 12288 x 4096 9.1 / 14.5 for 7.5 / 12.5).
template <MxMode MODE, int SRC>
static int thin_launch(const MxLinear& L, const MxFloats& F, hipStream_t st) {
    const int G = mx_groups(L.N), Q = mx_quads(L.K);
    if (Q <= 4)
        PG_LAUNCH((mx_thin_kernel<MODE, SRC, 4, true, 1>), dim3(std::min(G, 4 * kCUs)), dim3(256), 0, st, L, F);
    else if (Q <= 8)
        PG_LAUNCH((mx_thin_kernel<MODE, SRC, 8, true, 1>), dim3(std::min(G, 2 * kCUs)), dim3(512), 0, st, L, F);
    else if constexpr (SRC < 0) {
        if (G < 2 * kCUs)
            PG_LAUNCH((mx_thin_kernel<MODE, SRC, 8, false, 1>), dim3(G), dim3(512), 0, st, L, F);
        else
            PG_LAUNCH((mx_thin_kernel<MODE, SRC, 4, false, 2>), dim3(std::min((G + 1) / 2, 2 * kCUs)), dim3(256), 0, st, L, F);
    }
    return check_launch("mx_thin");
}

// ---------------------------------------------------------------- many rows
// A workgroup forms BM x BN outputs in WM x WN waves of 16 MT x 16 NT.  Activations and weights come through a ring of
// RING stages in LDS (128 bytes an activation row: 128 inputs in 8 bits, 256 in 4), copied straight from memory RING - 1
// stages ahead, so that a chain of stages runs at the rate of the products and not at a memory latency each.  At the top of stage
// s a wave waits until its copies of stage s have landed (EARLY: of s + 1), and the barrier makes all waves' visible; EARLY,
// the first fragments of s + 1 are then read under the last products of s.  Chunk c (16 bytes) of activation row r lies at
// c ^ (r / 2 & 7): the 16 rows of a fragment fall on different banks, but for the bf16 form's, whose chunks 2 g and 2 g + 1 meet
// (1.05 M conflict cycles at 500 x 4096 x 4096; a turn without them took the same time).  Weights lie as they are packed.
// Scales of 512 inputs come with the first of their stages: 16 bytes an activation row, which become a word a lane and row, a
// byte a step.
//
// WK parts of a workgroup, WM x WN waves and a ring each, share out the quads of the inputs, and their sums meet in LDS in
// the parts' order.  They are for few tiles: a CU then has more waves to hide a wait with and more copies under way, and smaller
// tiles spread the weights over more CUs (a CU takes in some 28 bytes a ns from memory, 110 from its L2).  77 x 4096 x 4096, 8
// bits: 96 tiles of 32 x 128 10.2 us, 192 of 32 x 64 in two parts 7.9; fp32 15.6, in four parts 9.3; 4 bits 8.3, in four 6.6.
//
// What bounds it: many rows the instruction, whose rate the power budget sets (random codes in registers alone: 4.0 PFLOP/s
// with 8-bit activations, 7.2 with 4-bit; 4096 x 24576 x 4096 runs at 2.6 and 3.6, 4096 x 4096 x 12288 at 2.7 and 4.4); fp32
// outputs the conversions beside the products (96 and 32 instructions a stage of a 64 x 128 tile: 1.3 of 2.0 PFLOP/s); few rows
// the weights' way to the CUs and the launch.
// Copies of 1 KB from memory to LDS, lane l's 16 bytes at base + off to lds + 16 l, each STEP behind the one before.  By
// hand, so that the compiler counts no loads and adds no waits; a copy reads m0 one wait state after its write.
#define PG_COPY(off, base) "s_nop 0\n\tglobal_load_lds_dwordx4 " off ", " base "\n\t"
template <int STEP>
__device__ __forceinline__ void copy_lds(uint32_t lds, const uint8_t* b0, uint32_t o0) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\t" PG_COPY("%2", "%3") "s_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(o0), "s"(b0)
                 : "memory");
}
template <int STEP>
__device__ __forceinline__ void copy_lds(uint32_t lds, const uint8_t* b0, uint32_t o0, const uint8_t* b1, uint32_t o1) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\t" PG_COPY("%2", "%3") "s_add_u32 m0, m0, %6\n\t" PG_COPY("%4", "%5")
                 "s_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(o0), "s"(b0), "v"(o1), "s"(b1), "n"(STEP)
                 : "memory", "scc");
}
template <int STEP>
__device__ __forceinline__ void copy_lds(uint32_t lds, const uint8_t* b0, uint32_t o0, const uint8_t* b1, uint32_t o1, const uint8_t* b2,
                                         uint32_t o2, const uint8_t* b3, uint32_t o3) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\t" PG_COPY("%2", "%3") "s_add_u32 m0, m0, %10\n\t" PG_COPY("%4", "%5")
                 "s_add_u32 m0, m0, %10\n\t" PG_COPY("%6", "%7") "s_add_u32 m0, m0, %10\n\t" PG_COPY("%8", "%9") "s_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(o0), "s"(b0), "v"(o1), "s"(b1), "v"(o2), "s"(b2), "v"(o3), "s"(b3), "n"(STEP)
                 : "memory", "scc");
}
#undef PG_COPY
// N of them, base(j) and off(j).
template <int STEP, int N, int J = 0, class B, class O>
__device__ __forceinline__ void copies_lds(uint32_t lds, B base, O off) {
    if constexpr (N - J >= 4) {
        copy_lds<STEP>(lds + J * STEP, base(J), off(J), base(J + 1), off(J + 1), base(J + 2), off(J + 2), base(J + 3), off(J + 3));
        copies_lds<STEP, N, J + 4>(lds, base, off);
    } else if constexpr (N - J >= 2) {
        copy_lds<STEP>(lds + J * STEP, base(J), off(J), base(J + 1), off(J + 1));
        copies_lds<STEP, N, J + 2>(lds, base, off);
    } else if constexpr (N - J == 1) {
        copy_lds<STEP>(lds + J * STEP, base(J), off(J));
    }
}
// All but the last N of this wave's copies have landed and its reads of LDS are done; then every wave's.
template <int N>
__device__ __forceinline__ void stage_ready() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <MxMode MODE, int MT, int NT, int WM, int WN, int WK, int RING, bool EARLY>
struct MxTile {
    static constexpr int BM = 16 * MT * WM, BN = 16 * NT * WN, NW = WM * WN;
    static constexpr int SPS = MODE == kS4 ? 2 : 1;            // steps a stage
    static constexpr int SPQ = 4 / SPS;                        // stages a quad
    static constexpr int XB = BM * 128, WB = BN / 16 * SPS * 1024, STAGE = XB + WB;
    static constexpr int XC = BM / 8 / NW, WC = WB / 1024 / NW;  // copies of a stage a wave
    static constexpr int SROWS = BM < 64 ? 64 : BM, SCOLS = BN < 64 ? 64 : BN;
    static constexpr int SPARTS = SROWS / 64 + SCOLS / 64, SC = (SPARTS + NW - 1) / NW;  // copies of scales: in all, a wave
    static constexpr int SB = (SROWS + SCOLS) * 16;
    static constexpr int NS = (RING - 1) / SPQ + 1;            // quads whose scales are held
    static constexpr int PART = RING * STAGE + NS * SB, LDS = WK * PART;
    static_assert(LDS >= (WK - 1) * BM * BN * 4, "sums of the other parts");
    static_assert(XC * 8 * NW == BM && WC * NW * 1024 == WB, "copies of a stage over the waves");
    // fragments read ahead: a step's, where registers hold two steps of them
    static constexpr bool WHOLE = EARLY && MT * NT <= 8;
    static constexpr int AHEAD = WHOLE ? MT : 1;
    static_assert(RING >= (EARLY ? 3 : 2), "stages under way");
    static_assert(LDS <= 160 * 1024, "LDS of a CU");
    // copies of a wave that may be under way at the top of stage s = J of a quad: those behind stage s + EARLY
    static constexpr int under_way(int j) {
        int n = 0;
        for (int k = EARLY ? 2 : 1; k <= RING - 2; ++k) n += XC + WC + ((j + k) % SPQ == 0 ? SC : 0);
        return n;
    }
    static_assert(under_way(0) <= 63, "the counter's range");
};

// Tile of a workgroup.  Workgroups go to the 8 XCDs in turn: each XCD takes one run of the tiles, in bands of 8
// row tiles at most, so that what it works on at a time shares rows and weights in its L2.
__device__ __forceinline__ void mx_tile_of(int id, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int n = tiles_m * tiles_n, per = n >> 3, rest = n & 7, x = id & 7;
    id = x * per + min(x, rest) + (id >> 3);
    const int band = id / (8 * tiles_n), in = id - band * 8 * tiles_n, high = min(8, tiles_m - 8 * band);
    tm = 8 * band + in % high;
    tn = in / high;
}

template <MxMode MODE, int MT, int NT, int WM, int WN, int WK, int RING, bool EARLY, int OCC>
__global__ __launch_bounds__(64 * WM * WN * WK, OCC) void mx_gemm_kernel(const MxLinear L, const int tiles_m, const int tiles_n) {
    using T = MxTile<MODE, MT, NT, WM, WN, WK, RING, EARLY>;
    __shared__ __attribute__((aligned(1024))) uint8_t all[T::LDS];
    const int lane = threadIdx.x & 63, own = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int part = own / T::NW, wave = own % T::NW;
    uint8_t* smem = all + part * T::PART;
    int tm, tn;
    mx_tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * T::BM, g0 = tn * (T::BN / 16);
    const int wm = wave % WM, wn = wave / WM;
    const int G = mx_groups(L.N), Q = mx_quads(L.K), blocks = L.K >> 5, stages = Q * T::SPQ;
    const int each = (Q + WK - 1) / WK, first = part * each, end = min(first + each, Q);  // quads of a part
    const uint32_t row_bytes = MODE == kS4 ? L.K >> 1 : L.K;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)smem;

    // Copies: rows past the last repeat it, groups past the last too, inputs past the row its last ones (their weights are
    // 0), stages behind the last the last one's (nothing reads them).
    const uint8_t* xb = L.x.codes + (int64_t)m0 * L.x.code_stride;
    const uint8_t* sb = L.x.scales + (int64_t)m0 * L.x.scale_stride;
    const uint32_t stride = (uint32_t)L.x.code_stride;
    const int rows = min(L.M - m0, T::BM) - 1;
    uint32_t x_off[T::XC];
#pragma unroll
    for (int j = 0; j < T::XC; ++j) x_off[j] = (uint32_t)min((wave + T::NW * j) * 8 + (lane >> 3), rows) * stride;
    const uint32_t chunk = 16u * (uint32_t)((lane ^ ((wave * 8 + (lane >> 3)) >> 1)) & 7);
    const uint8_t* wb[T::WC];  // copy j of the weights: this group and step of a stage
#pragma unroll
    for (int j = 0; j < T::WC; ++j) {
        const int c = wave + T::NW * j;
        wb[j] = L.w + ((int64_t)min(g0 + c / T::SPS, G - 1) * (4 * Q) + c % T::SPS) * 1024;
    }
    auto copy_stage = [&](int s, int slot) PG_INLINE {
        const uint32_t to = lds0 + (uint32_t)(slot * T::STAGE + wave * 1024);
        const uint32_t x_at = min(128u * (uint32_t)s + chunk, row_bytes - 16u);
        const uint32_t w_at = (uint32_t)(s * (T::SPS * 1024) + lane * 16);
        copies_lds<T::NW * 1024, T::XC>(to, [&](int) PG_INLINE { return xb; }, [&](int j) PG_INLINE { return x_off[j] + x_at; });
        copies_lds<T::NW * 1024, T::WC>(to + T::XB, [&](int j) PG_INLINE { return wb[j]; }, [&](int) PG_INLINE { return w_at; });
    };
    const uint8_t* wsb = L.w + ((int64_t)G * Q * 4096 + (int64_t)g0 * Q * 256);
    auto copy_scales = [&](int q) PG_INLINE {
        const uint32_t to = lds0 + RING * T::STAGE + (uint32_t)(q % T::NS) * T::SB;
        q = min(q, Q - 1);
#pragma unroll
        for (int j = 0; j < T::SC; ++j) {
            const int p = (wave + T::NW * j) % T::SPARTS;  // several waves may copy the same
            const bool x = p < T::SROWS / 64;
            const int c = x ? p : p - T::SROWS / 64;
            const uint32_t x_at = (uint32_t)min(c * 64 + lane, rows) * (uint32_t)L.x.scale_stride + 16u * (uint32_t)q;
            const uint32_t w_at = (uint32_t)min(c * 4 + (lane >> 4), G - 1 - g0) * (uint32_t)(Q * 256) + (uint32_t)(q * 256 + (lane & 15) * 16);
            copy_lds<0>(to + p * 1024, x ? sb : wsb, x ? x_at : w_at);
        }
    };

    floatx4 acc[NT][MT];
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[b][t] = floatx4{0, 0, 0, 0};
    int4 w[2][NT];
    int ws[NT], xs[MT];
    constexpr int GR = MT / T::AHEAD;  // groups of fragments a step
    XFrag<MODE> f[2][T::AHEAD];
    // this lane's places: weights, and the chunks of its activation rows (4 bits: of the stage's two steps)
    const int w_lane = lane * 16 + T::XB + wn * NT * T::SPS * 1024;
    const int x_row = (wm * MT * 16 + r) * 128, c0 = MODE == kB8 ? 2 * g : g, c1 = MODE == kB8 ? c0 + 1 : c0 + 4;
    const int x_lane[2] = {x_row + 16 * (c0 ^ (r >> 1)), x_row + 16 * (c1 ^ (r >> 1))};
    auto get_w = [&](int4 (&to)[NT], int base, int u) PG_INLINE {
        const uint8_t* from = smem + (w_lane + base);
#pragma unroll
        for (int b = 0; b < NT; ++b) to[b] = *(const int4*)(from + (b * T::SPS + u) * 1024);
    };
    auto get_x = [&](int base, int u, int t) PG_INLINE {
        XFrag<MODE> v;
        v.a = *(const int4*)(smem + (x_lane[MODE == kS4 ? u : 0] + base) + t * 2048);
        if constexpr (MODE != kS4) v.b = *(const int4*)(smem + (x_lane[1] + base) + t * 2048);
        return v;
    };
    const uint32_t pick = (uint32_t)(g | (4 + g) << 8);
    uint4 sv[MT];
    int wsv[NT];
    auto read_scales = [&](int q) PG_INLINE {
        const uint8_t* from = smem + RING * T::STAGE + (q % T::NS) * T::SB;
#pragma unroll
        for (int b = 0; b < NT; ++b) wsv[b] = *(const int*)(from + T::SROWS * 16 + (wn * NT + b) * 256 + lane * 4);
#pragma unroll
        for (int t = 0; t < MT; ++t) sv[t] = *(const uint4*)(from + ((wm * MT + t) * 16 + r) * 16);
    };
    auto set_scales = [&](int q) PG_INLINE {
#pragma unroll
        for (int b = 0; b < NT; ++b) ws[b] = wsv[b];
        // blocks past the row's last: 1, whatever lies there
        const int have = min(max((blocks - 16 * q - g + 3) >> 2, 0), 4);
        const uint32_t keep = have == 4 ? 0xffffffffu : (1u << (8 * have)) - 1u;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const uint32_t a = __builtin_amdgcn_perm(sv[t].y, sv[t].x, pick), b = __builtin_amdgcn_perm(sv[t].w, sv[t].z, pick);
            xs[t] = (int)((__builtin_amdgcn_perm(b, a, 0x05040100u) & keep) | (0x7f7f7f7fu & ~keep));
        }
    };
    // Step S of a quad, its weights and first AHEAD fragments in registers: the products of a group of fragments run while the
    // next group, or the next step's first and its weights, are read.  x(t), t past MT: the next step's.
    auto step = [&](auto sc, auto follows, int w_base, int w_u, auto x) PG_INLINE {
        constexpr int S = decltype(sc)::value;
        constexpr bool NEXT = decltype(follows)::value;  // the next step can be read already
        if constexpr (NEXT) get_w(w[(S + 1) & 1], w_base, w_u);
        WOps<MODE, NT> ops;
        ops.template set<S>(w[S & 1], ws);
#pragma unroll
        for (int i = 0; i < GR; ++i) {
            const int p = (S * GR + i) & 1;
#pragma unroll
            for (int k = 0; k < T::AHEAD; ++k)
                if (NEXT || i + 1 < GR) f[p ^ 1][k] = x((i + 1) * T::AHEAD + k);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < T::AHEAD; ++k) mx_products<MODE, S, S>(ops, ws, xs[i * T::AHEAD + k], f[p][k], i * T::AHEAD + k, acc);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    copy_scales(first);
#pragma unroll
    for (int s = 0; s < RING - 1; ++s) {
        if (s && s % T::SPQ == 0) copy_scales(first + s / T::SPQ);
        copy_stage(min(first * T::SPQ + s, stages - 1), s);
    }
    int slot = 0;
    if constexpr (EARLY) {
        stage_ready<T::under_way(T::SPQ - 1)>();  // stage 0, as at the top of the stage before it
#pragma unroll
        for (int k = 0; k < T::AHEAD; ++k) f[0][k] = get_x(0, 0, k);
        get_w(w[0], 0, 0);
    }
    if constexpr (T::WHOLE) read_scales(first);
    // stage J of quad q
    auto stage = [&](auto jc, int q) PG_INLINE {
        constexpr int J = decltype(jc)::value;
        const int s = q * T::SPQ + J, here = slot * T::STAGE;
        const int over = slot == 0 ? RING - 1 : slot - 1, after = slot == RING - 1 ? 0 : slot + 1, then = after * T::STAGE;
        stage_ready<T::under_way(J)>();
        if constexpr ((J + RING - 1) % T::SPQ == 0) copy_scales((s + RING - 1) / T::SPQ);
        copy_stage(min(s + RING - 1, stages - 1), over);
        if constexpr (J == 0) {
            if constexpr (!T::WHOLE) read_scales(q);
            set_scales(q);
        }
        if constexpr (T::WHOLE && J == T::SPQ - 1) read_scales(q + 1);  // theirs came with the next stage's
        constexpr int S = J * T::SPS;
        if constexpr (!EARLY) {
            get_w(w[S & 1], here, 0);
#pragma unroll
            for (int k = 0; k < T::AHEAD; ++k) f[(S * GR) & 1][k] = get_x(here, 0, k);
        }
        using Next = std::integral_constant<bool, EARLY>;
        if constexpr (T::SPS == 2) {
            step(std::integral_constant<int, S>(), std::true_type(), here, 1,
                 [&](int t) PG_INLINE { return t < MT ? get_x(here, 0, t) : get_x(here, 1, t - MT); });
            step(std::integral_constant<int, S + 1>(), Next(), then, 0,
                 [&](int t) PG_INLINE { return t < MT ? get_x(here, 1, t) : get_x(then, 0, t - MT); });
        } else {
            step(std::integral_constant<int, S>(), Next(), then, 0,
                 [&](int t) PG_INLINE { return t < MT ? get_x(here, 0, t) : get_x(then, 0, t - MT); });
        }
        slot = after;
    };
    for (int q = first; q < end; ++q) {
        stage(std::integral_constant<int, 0>(), q);
        stage(std::integral_constant<int, 1>(), q);
        if constexpr (T::SPQ == 4) {
            stage(std::integral_constant<int, 2>(), q);
            stage(std::integral_constant<int, 3>(), q);
        }
    }
    if constexpr (WK > 1)
        for (int n = (each - max(end - first, 0)) * T::SPQ; n > 0; --n) asm volatile("s_barrier" ::: "memory");  // a part with fewer
    stage_ready<0>();  // copies that nothing reads, before the LDS is another workgroup's
    if constexpr (WK > 1) {  // the parts' sums, in their order
        float4* sums = (float4*)all + wave * 64 + lane;
        auto at = [&](int p, int b, int t) PG_INLINE { return (((p - 1) * NT + b) * MT + t) * T::NW * 64; };
        if (part > 0) {
#pragma unroll
            for (int b = 0; b < NT; ++b)
#pragma unroll
                for (int t = 0; t < MT; ++t) sums[at(part, b, t)] = make_float4(acc[b][t][0], acc[b][t][1], acc[b][t][2], acc[b][t][3]);
        }
        __syncthreads();
        if (part > 0) return;
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int p = 1; p < WK; ++p) {
                    const float4 v = sums[at(p, b, t)];
                    acc[b][t] += floatx4{v.x, v.y, v.z, v.w};
                }
    }
    constexpr int BITS = MODE == kS8 ? 16 : 0;
    auto each_of = [&](auto put) PG_INLINE {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int b = 0; b < NT; ++b) put(t, b, m0 + (wm * MT + t) * 16 + r, (g0 + wn * NT + b) * 16);
    };
    if (16 * g0 + T::BN <= L.N) {  // no row ends in this tile
        if constexpr (NT % 2 == 0) {
            if (BITS == 16 || L.odt != PGMOE_DT_F32) {
                each_of([&](int t, int b, int m, int n) PG_INLINE {
                    if (b % 2 == 0) put_pair(L, m, n, g, acc[b][t], acc[b + 1][t]);
                });
                return;
            }
        }
        each_of([&](int t, int b, int m, int n) PG_INLINE {
            if (m < L.M) put4<true, BITS>(L, m, n + 4 * g, make_float4(acc[b][t][0], acc[b][t][1], acc[b][t][2], acc[b][t][3]));
        });
        return;
    }
    each_of([&](int t, int b, int m, int n) PG_INLINE {
        if (m < L.M && n + 4 * g < L.N) put4<false, BITS>(L, m, n + 4 * g, make_float4(acc[b][t][0], acc[b][t][1], acc[b][t][2], acc[b][t][3]));
    });
}

template <MxMode MODE, int MT, int NT, int WM, int WN, int WK, int RING, bool EARLY, int OCC>
static int gemm_launch(const MxLinear& L, hipStream_t st) {
    using T = MxTile<MODE, MT, NT, WM, WN, WK, RING, EARLY>;
    const int tm = div_up(L.M, T::BM), tn = div_up(L.N, T::BN);
    PG_LAUNCH((mx_gemm_kernel<MODE, MT, NT, WM, WN, WK, RING, EARLY, OCC>), dim3(tm * tn), dim3(64 * T::NW * WK), 0, st, L, tm, tn);
    return check_launch("mx_gemm");
}

// Which tile: the one whose fit a + b ceil(tiles / CUs) to the times measured is least.  The rule does not know K: it was fitted at
// K = 4096 and not measured at others, where a tile whose parts share out the quads gains less (up to 512 inputs one part works).
// us at K = 4096 for n tiles a CU, n = 1 / 2 / 4:
//   8 bits  128 x 256 33 / 52 / 100, 128 x 128 22 / 35 / 63, 64 x 128 14 / 22 / 39, 32 x 128 11 / 14 / 26, 32 x 64 8.2 / 11 / 19
//   4 bits  256 x 256 41 / 77, 128 x 128 17 / 27 / 47, 64 x 64 9.5 / 12.7 / 22, 32 x 128 11.8 / 13 / 24, 32 x 64 7.4 / 13 / 24
//   fp32    64 x 256 35 / 58 / 115, 64 x 128 21 / 34 / 62, 32 x 128 14 / 22 / 40, 32 x 64 9.8 / 14 / 25
// The choice against the best of them, 8 bits, outputs x 4096: 128 rows, 4096: 8.2 (others 10.6 / 13 / 20 / 33); 500: 14.5 (14.1
// to 33); 1024: 22.7 (22.2 to 34); 4096: 56.5 (57 to 122); fp32 500: 21.9 (21.2 to 35).
struct MxCost {
    int bm, bn;
    float a, b;
};
template <int TILES>
static int pick_tile(const MxCost (&c)[TILES], int M, int N) {
    int best = TILES - 1;
    float least = 0.0f;
    for (int i = TILES - 1; i >= 0; --i) {
        const int64_t tiles = (int64_t)div_up(M, c[i].bm) * div_up(N, c[i].bn);
        const float t = c[i].a + c[i].b * (float)((tiles + kCUs - 1) / kCUs);
        if (i == TILES - 1 || t < least) best = i, least = t;
    }
    return best;
}

static int linear_s8(const MxLinear& L, hipStream_t st) {
    static constexpr MxCost cost[] = {{128, 256, 9.6f, 23.4f}, {128, 128, 8.0f, 13.8f}, {64, 128, 6.0f, 8.1f}, {32, 128, 5.5f, 5.1f}, {32, 64, 4.8f, 3.5f}};
    switch (pick_tile(cost, L.M, L.N)) {
        case 0: return gemm_launch<kS8, 4, 8, 2, 2, 1, 2, false, 2>(L, st);
        case 1: return gemm_launch<kS8, 4, 4, 2, 2, 1, 3, false, 2>(L, st);
        case 2: return gemm_launch<kS8, 4, 2, 1, 4, 1, 4, true, 2>(L, st);
        case 3: return gemm_launch<kS8, 2, 2, 1, 4, 1, 4, true, 2>(L, st);
        default: return gemm_launch<kS8, 2, 2, 1, 2, 2, 4, true, 2>(L, st);
    }
}
static int linear_s4(const MxLinear& L, hipStream_t st) {
    static constexpr MxCost cost[] = {{256, 256, 5.0f, 35.8f}, {128, 128, 6.5f, 9.9f}, {64, 64, 5.5f, 3.9f}, {32, 128, 6.5f, 4.5f}, {32, 64, 2.2f, 5.4f}};
    switch (pick_tile(cost, L.M, L.N)) {
        case 0: return gemm_launch<kS4, 8, 4, 2, 4, 1, 2, false, 2>(L, st);
        case 1: return gemm_launch<kS4, 4, 4, 2, 2, 1, 2, false, 2>(L, st);
        case 2: return gemm_launch<kS4, 4, 1, 1, 4, 2, 2, false, 2>(L, st);
        case 3: return gemm_launch<kS4, 2, 2, 1, 4, 1, 3, true, 2>(L, st);
        default: return gemm_launch<kS4, 2, 1, 1, 4, 4, 2, false, 4>(L, st);
    }
}
static int linear_b8(const MxLinear& L, hipStream_t st) {
    static constexpr MxCost cost[] = {{64, 256, 10.0f, 24.5f}, {64, 128, 7.0f, 13.5f}, {32, 128, 5.5f, 8.3f}, {32, 64, 5.0f, 4.9f}};
    switch (pick_tile(cost, L.M, L.N)) {
        case 0: return gemm_launch<kB8, 4, 4, 1, 4, 1, 2, false, 2>(L, st);
        case 1: return gemm_launch<kB8, 4, 2, 1, 4, 2, 2, false, 2>(L, st);
        case 2: return gemm_launch<kB8, 2, 2, 1, 4, 2, 2, false, 2>(L, st);
        default: return gemm_launch<kB8, 2, 2, 1, 2, 4, 2, false, 4>(L, st);
    }
}

// Up to 16 rows are read against weights that go straight to registers (17 of 12288 x 4096: 12.0 us in two such tiles, 8.6 in
// tiles of 32 rows; 16: 8.7).  There the bf16 instruction costs nothing, as the weights' arrival bounds both.
int launch_mx_linear(const MxLinear& L, hipStream_t st) {
    if (L.M <= kMxFewRows) return L.x.e2m1 ? thin_launch<kS4, -1>(L, MxFloats{}, st) : thin_launch<kB8, -1>(L, MxFloats{}, st);
    if (L.x.e2m1) return linear_s4(L, st);
    return L.odt == PGMOE_DT_F32 || L.wide ? linear_b8(L, st) : linear_s8(L, st);
}

int launch_mx_linear_values(const MxLinear& L, const MxFloats& F, hipStream_t st) {
    if (mx_values_inside(L.M, L.K)) {
#define VALUES(DT) return L.x.e2m1 ? thin_launch<kS4, DT>(L, F, st) : thin_launch<kB8, DT>(L, F, st)
        if (F.dt == PGMOE_DT_F32) VALUES(PGMOE_DT_F32);
        if (F.dt == PGMOE_DT_F16) VALUES(PGMOE_DT_F16);
        VALUES(PGMOE_DT_BF16);
#undef VALUES
    }
    const int rc = launch_mx_quantize(F, L.x, st);
    return rc ? rc : launch_mx_linear(L, st);
}

}  // namespace pgmoe
