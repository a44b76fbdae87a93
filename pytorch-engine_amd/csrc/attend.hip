// Attention of a batch over a paged KV cache whose first keys are shared by every sequence.
//
// For query row (token t, head h) with visible keys j (the shared prefix, then the sequence's own up to the
// query): o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale (q . k_j - max)), in one pass over the keys with the
// running maximum and sum (exp2 of scores scaled by scale * log2 e in fp32).
//
// Rows that read the same keys are computed together: the rows of a sequence's tokens and of the query heads
// that share a KV head, and on the prefix the rows of every sequence.  A segment is such a set of rows on one
// KV head: up to 32 rows (split: one wave's) or a tile of 128 (shared: 32 a wave, the four waves share each
// tile of keys).  Every wave takes an equal run of the tiles of all split segments in order, then every
// workgroup one of the shared segments', found on the device from lens and q_start, so nothing about the
// lengths is known to or kept by the host.  A segment that several runs share leaves unnormalised partial
// rows and their (max, sum), merged in slot order by combine_rows_kernel.
//
// The products run on 32x32x16 MFMA, scores transposed: S^T = K Q^T has a query row per lane column, so the
// maximum and sum of a row are sums over a lane's registers and one swap of wave halves, and the rounded
// probabilities are already the B operand of O^T = V^T P^T (whose k index may be permuted as long as V's
// rows are too).  K and V go from memory to LDS without registers, rows swizzled over the banks for the 16-byte
// reads of K and the transposing 8-byte reads of V (of the prompts' LDS cycles a third are conflicts all the same).
//
// What bounds it (whole calls): a few rows a chain of latencies, lens to pages to keys to partial rows, and the
// second launch (one sequence of 5003 keys: 12 + 5 us); long caches of few rows HBM (32 sequences of up to
// 16000 keys, 8 KV heads of 128: 212 us, 5.4 TB/s); prompts and long prefixes reading K and V again for every row
// tile as much as the matrix units: the row tiles of a KV head are dealt over all XCDs, each with an L2 of its own, and
// stand at different keys.  Six prompts behind 4097 keys, 394 us, 790 TFLOP/s (414 on a slower card): 2.04 GB come from
// behind the L2s, of 2.54 GB that tiles ask for and 0.03 that are there, 5.2 TB/s, while MFMA is busy 39 % of the
// cycles; 256 rows behind 16000 shared keys, 125 us: 0.63 GB, for 0.19.  Giving half the waves a
// higher priority, or the products alone, moves it by 1 to 2 % at most.  Heads of 256: the same 32
// sequences on 4 KV heads 228 us, a prompt of 1024 behind 4096 keys 137 us, 565 TFLOP/s on one wave a SIMD.
//
// Masked keys: a tile with a key that some row does not see takes the checked path: scores of masked keys
// become -inf, and V values that are not finite reach only the rows that see them.  Rows past the last
// visible key are read as copies of it.
#include <atomic>

#include "kv.h"
#include "launch.h"

namespace pgmoe {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kValu = 0x2, kSalu = 0x4, kMfma = 0x8, kDs = 0x100;  // instruction classes of the sched_ barriers
constexpr int kSplitKeys = 32, kSharedKeys = 64;  // keys of a tile, by kind of segment
constexpr int kSplitRows = 32, kSharedRows = 128;
constexpr int kAlone = 16;  // row tiles that a lane sums by itself
// Tiles of a wave's run at least: one sequence of 5003 keys takes 16.4 us at 1 and 2 (and half the partial
// rows at 2), 16.7 at 4.
constexpr int kSplitLeast = 2;
// What a segment costs beside its tiles, in tiles.  64 rows of one token behind 8192 shared keys: 40.8 us;
// split heads of 1 and 6 42.4 and 42.2, shared ones of 2 and 10 43.7 and 41.8.
constexpr int kSplitHead = 3, kSharedHead = 5;

struct AttendArgs {
    KvCache C;
    KvBatch B;
    const uint16_t* q;
    int64_t q_tok, q_head;
    int T, hq, group;
    uint32_t by_group;  // ceil(2^32 / group): x / group = (x * by_group) >> 32 while x * group < 2^32
    float c;            // scale * log2(e)
    uint16_t* out;
    float* lse;
    // partial rows [prefix, if there is one, then own][slot][T * hq][dim], their (max in log2 units, sum), and
    // the slots a row has
    float* part;
    float2* ml;
    int* slots;
    int nslot, own;  // slots of a region; where the own keys' begin
};

template <int D>
struct Geo {
    static constexpr int RB = 2 * D;            // bytes of a row
    static constexpr int CPB = D / 32;          // 1 KB copies of 16 rows
    static constexpr int RPC = 16 / CPB;        // rows of a copy
    static constexpr int LPR = 64 / RPC;        // lanes of a row in a copy
    static constexpr int KM = D == 64 ? 7 : 15;  // K: 16-byte chunk c of row r lies at c ^ (r & KM)
    static constexpr int LDS = 512 * D;         // both kinds of segment
    static constexpr int OCC = D == 256 ? 1 : 2;  // waves a SIMD
    // V: 32-byte pair p of row r lies at p ^ vswz(r)
    __device__ static constexpr int vswz(int r) { return D == 64 ? (r >> 1) & 3 : r & 7; }
};

// 1 KB from memory to LDS, lane l's 16 bytes to lds + 16 l; waited for with vm_wait (copies are not in the
// compiler's own count of loads, which only makes its waits longer).  A copy reads m0 one wait state after a
// scalar write of it at the earliest: s_nop, as nothing looks into inline assembly for it.
__device__ __forceinline__ void copy_lds(const void* base, uint32_t off, uint32_t lds) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(off), "s"(base), "s"(lds)
                 : "memory");
}
// Four of them from rows that follow each other without gaps: the instruction's offset moves both addresses.
__device__ __forceinline__ void copy_lds4(const void* base, uint32_t o0, uint32_t o1, uint32_t o2, uint32_t o3,
                                          uint32_t lds) {
    uint32_t keep;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %6\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %5\n\t"
        "global_load_lds_dwordx4 %2, %5 offset:1024\n\t"
        "global_load_lds_dwordx4 %3, %5 offset:2048\n\t"
        "global_load_lds_dwordx4 %4, %5 offset:3072\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(keep)
        : "v"(o0), "v"(o1), "v"(o2), "v"(o3), "s"(base), "s"(lds)
        : "memory");
}
__device__ __forceinline__ void copy_lds2(const void* base, uint32_t o0, uint32_t o1, uint32_t lds) {
    uint32_t keep;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %4\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %3\n\t"
        "global_load_lds_dwordx4 %2, %3 offset:1024\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(keep)
        : "v"(o0), "v"(o1), "s"(base), "s"(lds)
        : "memory");
}
template <int N>
__device__ __forceinline__ void vm_wait() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void lds_wait() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uni64(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)uni((int)v) | (uint64_t)(uint32_t)uni((int)(v >> 32)) << 32);
}
// A scalar load: the index is the wave's, and nothing in this kernel writes page tables.
__device__ __forceinline__ int sload(const int32_t* p, int64_t i) {
    return ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)p)[i];
}

__device__ __forceinline__ int group_of(const AttendArgs& A, int x) {  // x / group
    return A.group == 1 ? x : (int)__umulhi((uint32_t)x, A.by_group);
}

// One sequence's rows and keys.
struct Seq {
    int lo, n, len, cap, rows;
    // keys that its token i sees: at most cap; `far` if lens says more
    __device__ __forceinline__ int seen(int i, bool* far = nullptr) const {
        const int64_t v = (int64_t)len - n + i + 1;
        if (far) *far = v > cap;
        return v < 0 ? 0 : v > cap ? cap : (int)v;
    }
    __device__ __forceinline__ int last_token(const AttendArgs& A, int tile) const {
        const int r = kSharedRows * (tile + 1);
        return r < rows ? group_of(A, r - 1) : n - 1;
    }
    __device__ __forceinline__ bool split() const { return rows <= kSplitRows; }
    __device__ __forceinline__ int tiles(const AttendArgs& A, int tile) const {  // of row tile `tile`; one at least
        const int k = split() ? (seen(n - 1) + kSplitKeys - 1) / kSplitKeys
                              : (seen(last_token(A, tile)) + kSharedKeys - 1) / kSharedKeys;
        return k < 1 ? 1 : k;
    }
};
__device__ __forceinline__ Seq load_seq(const AttendArgs& A, int b) {
    Seq s;
    int hi;
    seq_tokens(A.B, b, A.T, s.lo, hi);
    s.n = hi - s.lo;
    s.len = A.B.lens[b];
    s.len = s.len < 0 ? 0 : s.len;
    s.cap = A.B.max_pages << A.C.page_shift;
    s.rows = s.n * A.group;
    return s;
}
__device__ __forceinline__ int row_tiles(int rows) {
    return rows <= kSplitRows ? (rows > 0) : (rows + kSharedRows - 1) / kSharedRows;
}

// Tiles [j0, j1) of one segment: what a wave (split) or a workgroup (shared) computes at a time.
struct Work {
    int prefix, lo, rows, row0, kvh, b, keys, j0, j1, slot, nslots;
    int pre;          // tiles of the prefix before the own keys'
    int len, n, cap;  // own keys: Seq's
    int left;         // of the run behind this work
    __device__ __forceinline__ void scalar() {  // every lane holds the same: into scalar registers
        prefix = uni(prefix), lo = uni(lo), rows = uni(rows), row0 = uni(row0), kvh = uni(kvh), b = uni(b);
        keys = uni(keys), j0 = uni(j0), j1 = uni(j1), slot = uni(slot), nslots = uni(nslots);
        len = uni(len), n = uni(n), cap = uni(cap), left = uni(left), pre = uni(pre);
    }
};

// The prefix's segments of one kind and the sequences' of that kind lie one behind the other on an axis of
// tiles, each with kHead tiles' room before its first for what a segment costs by itself.  s_base holds
// where each thread's sequences begin.
template <bool SPLIT>
struct Axis {
    static constexpr int kHead = SPLIT ? kSplitHead : kSharedHead;
    int ptiles, psegs, run, total;
    int pre;  // the prefix's tiles where every row tile takes them before its own keys

    // The cost of one KV head of this lane's sequence (`in`: it has one).  A wave sums the row tiles of a long
    // prompt together.
    __device__ __forceinline__ int cost(const AttendArgs& A, const Seq& s, bool in, int lane) const {
        const int rt = in && s.split() == SPLIT ? row_tiles(s.rows) : 0;
        int c = 0;
        if constexpr (SPLIT) {
            if (rt) c = s.tiles(A, 0) + kHead;
        } else {
            if (rt <= kAlone)
                for (int t = 0; t < rt; ++t) c += s.tiles(A, t) + pre + kHead;
            for (uint64_t big = __ballot(rt > kAlone); big; big &= big - 1) {
                const int who = __builtin_ctzll(big);
                Seq m;
                m.n = __builtin_amdgcn_readlane(s.n, who), m.len = __builtin_amdgcn_readlane(s.len, who);
                m.rows = __builtin_amdgcn_readlane(s.rows, who), m.cap = s.cap;
                const int all = row_tiles(m.rows);
                int sum = 0;
                for (int t = lane; t < all; t += 64) sum += m.tiles(A, t) + pre + kHead;
                for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
                if (lane == who) c = sum;
            }
        }
        return c;
    }
    __device__ __forceinline__ Work fill(int start, int n, int at, int end, int who) const {
        Work W;
        const int first = at - start - kHead;  // a run may begin or end in the head
        W.j0 = first < 0 ? 0 : first;
        const int stop = end - start - kHead;
        W.j1 = stop < n ? stop : n;
        const int w0 = (start + kHead) / run;
        W.slot = who - w0;
        W.nslots = (start + kHead + n - 1) / run - w0 + 1;
        W.left = end - (start + kHead + n);
        return W;
    }
    // The work that begins at `at` of the run that ends at `end`, found by one wave.
    __device__ __forceinline__ Work find(const AttendArgs& A, const int* s_base, const int (*s_seq)[3], int per, int Tq,
                                         int at, int end, int who, int lane) const {
        const int pall = psegs * (ptiles + kHead);
        if (at < pall) {
            const int seg = at / (ptiles + kHead);
            Work W = fill(seg * (ptiles + kHead), ptiles, at, end, who);
            const int rows = Tq * A.group, prt = row_tiles(rows);
            W.prefix = 1, W.lo = 0, W.rows = rows, W.kvh = seg / prt, W.row0 = (seg - W.kvh * prt) * kSharedRows, W.b = 0;
            W.keys = A.B.prefix, W.len = 0, W.n = 0, W.cap = 0, W.pre = 0;
            return W;
        }
        // the thread, then among its sequences, then the row tile: the last that begins at or before `at`
        int i = 0;
#pragma unroll
        for (int g = 0; g < kThreads / 64; ++g) i += __popcll(__ballot(s_base[64 * g + lane] <= at));
        i -= 1;
        int from = uni(s_base[i]);
        i *= per;
        Seq s;
        int c = 0;
        if (per == 1) {
            s.lo = s_seq[i][0], s.n = s_seq[i][1], s.len = s_seq[i][2];
            s.cap = A.B.max_pages << A.C.page_shift, s.rows = s.n * A.group;
            c = uni(cost(A, s, lane == 0, lane));
        } else {
            const bool in = lane < per && i + lane < A.B.seqs;
            Seq m = load_seq(A, in ? i + lane : A.B.seqs - 1);
            const int mc = cost(A, m, in, lane) * A.C.heads;
            int inc = mc;
            for (int d = 1; d < 16; d <<= 1) {
                const int o = __shfl_up(inc, d);
                if (lane >= d) inc += o;
            }
            // lanes that hold nothing end where their neighbour does
            const int k = __popcll(__ballot(in && from + inc <= at));
            from += uni(__shfl(inc - mc, k));
            i += k;
            s = load_seq(A, i);
            c = uni(__shfl(mc, k)) / A.C.heads;
        }
        s.lo = uni(s.lo), s.n = uni(s.n), s.len = uni(s.len), s.rows = uni(s.rows);
        c = uni(c);
        const int kvh = (at - from) / c;
        from += kvh * c;
        int t = 0;
        if (!SPLIT) {
            const int rt = row_tiles(s.rows);
            for (;; t += 64) {
                int inc = t + lane < rt ? s.tiles(A, t + lane) + pre + kHead : 0;
                for (int d = 1; d < 64; d <<= 1) {
                    const int o = __shfl_up(inc, d);
                    if (lane >= d) inc += o;
                }
                const int k = __popcll(__ballot(t + lane < rt && from + inc <= at));
                if (k < 64 && t + k < rt) {
                    if (k) from += uni(__shfl(inc, k - 1));
                    t += k;
                    break;
                }
                from += uni(__shfl(inc, 63));
            }
        }
        Work W = fill(from, s.tiles(A, t) + pre, at, end, who);
        W.pre = pre, W.prefix = 0, W.lo = s.lo, W.rows = s.rows, W.row0 = t * kSharedRows, W.kvh = kvh, W.b = i;
        W.keys = s.seen(SPLIT ? s.n - 1 : s.last_token(A, t));
        W.len = s.len, W.n = s.n, W.cap = s.cap;
        return W;
    }
};

// The products and softmax of one wave's 32 rows, N2 groups of 32 keys at a time.
template <int D, bool BF16>
struct Core {
    using G = Geo<D>;
    static constexpr int NK = D / 16, ND = D / 32;
    u16x8 q[NK];
    f32x16 o[ND];
    float m, l, c;  // reference maximum (raw score), sum over this lane's keys times 2^kUp, scale * log2(e)
    bool far;       // a row is out of step: see grow
    int lane, n, h;
    uint32_t koff, voff[ND];  // LDS byte offsets of this lane's reads

    __device__ __forceinline__ static f32x16 mfma(u16x8 a, u16x8 b, f32x16 acc) {
        if constexpr (BF16)
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                           acc, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), acc,
                                                          0, 0, 0);
    }
    // Queries in ordinary registers, arrived before the loops.  256-wide heads take more than 256 registers: the
    // sums lie in accumulation registers throughout, and are moved only where they are rescaled.
    __device__ __forceinline__ void hold() {
#pragma unroll
        for (int i = 0; i < NK; ++i) asm volatile("" : "+v"(q[i]));
        hold_sums();
    }
    __device__ __forceinline__ void hold_sums() {
        if constexpr (D == 256) {
#pragma unroll
            for (int i = 0; i < ND; ++i) asm volatile("" : "+a"(o[i]));
        }
    }
    __device__ __forceinline__ static float swap32(float v) { return xor_lane<32>(v); }

    __device__ __forceinline__ void begin(int lane_) {
        lane = lane_, n = lane & 31, h = lane >> 5;
        m = -INFINITY, l = 0.0f, far = false;
#pragma unroll
        for (int i = 0; i < ND; ++i) o[i] = f32x16{};
        koff = n * G::RB + ((h ^ (n & G::KM)) << 4);
        // transposing read: 16 lanes take 4 rows of 16 columns, lane 4 r + i the row r and columns 4 i ..;
        // each ends with its column of the 4 rows
        const int r = 4 * h + ((lane & 15) >> 2);
#pragma unroll
        for (int d = 0; d < ND; ++d)
            voff[d] = r * G::RB + (((2 * d + ((lane >> 4) & 1)) ^ G::vswz(r)) << 5) + ((lane & 3) << 3);
    }
    __device__ __forceinline__ static int key_of(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }
    // S^T of N2 * 32 keys: s[g][i] is key 32 g + key_of(i, h) of this lane's row
    template <int N2>
    __device__ __forceinline__ void score_products(const uint8_t* K, f32x16 (&s)[N2]) {
#pragma unroll
        for (int g = 0; g < N2; ++g) s[g] = f32x16{};
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int g = 0; g < N2; ++g)
                s[g] = mfma(*(const u16x8*)(K + g * 32 * G::RB + (koff ^ (uint32_t)(i << 5))), q[i], s[g]);
    }
    template <int N2>
    __device__ __forceinline__ void scores(const uint8_t* K, f32x16 (&s)[N2]) {
        score_products<N2>(K, s);
        // four reads ahead of the products that take them
        __builtin_amdgcn_sched_group_barrier(kDs, 4, 0);
#pragma unroll
        for (int i = 0; i < N2 * NK - 4; ++i) {
            __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kDs, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kMfma, 4, 0);
    }
    // left: visible keys of this lane's row from the group's first on; bad: bit b: block b of 16 keys has no page
    __device__ __forceinline__ void mask(f32x16& s, int left, int bad) {
        left -= 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if ((bad >> (i >> 3)) & 1) s[i] = NAN;
            if (key_of(i, 0) >= left) s[i] = -INFINITY;
        }
    }
    // The reference m follows the running maximum only when that has grown by 2^8, and the rescaling of o (64
    // products a lane) all but vanishes: p = 2^(c (s - m) + kUp) is 2^(8 + kUp) at most.
    template <int N2>
    __device__ __forceinline__ void grow(const f32x16 (&s)[N2]) {
        float mx = s[0][0];
#pragma unroll
        for (int g = 0; g < N2; ++g)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[g][i]);
        mx = fmaxf(mx, swap32(mx));
        if (__builtin_expect(__any((mx - m) * c > 8.0f), 0)) {
            const float mn = fmaxf(m, mx);
            const float f = __builtin_amdgcn_exp2f((m - (mn == -INFINITY ? 0.0f : mn)) * c);
            l *= f;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
            m = mn;
            far = far || __any(out_of_step());
            hold_sums();
        }
    }
    // weigh forms c (s - m) as fma(s, c, -round(m c)), which is off by half a step of m c: the same factor of all of a
    // row's p, until that takes them out of fp16's range.  A row with |m c| above 2^23, of which a step is 1, is out of
    // step: the run is computed again on checked tiles, with s - m in such rows.  (s - m at once, where the maximum
    // grows, kept the scores from staying where the matrix units put them: heads of 256, 4 prompts of 100 to
    // 900 tokens 74 us, 69 so, 67 without either.)
    __device__ __forceinline__ bool out_of_step() const { return fabsf(m * c) > 8388608.0f && fabsf(m * c) < INFINITY; }
    // p = 2^(c (s - m) + kUp) rounded, l += sum p.  The product with V takes 16-bit probabilities (that is what the
    // matrix units multiply at full rate; each is off by half a step of the cache's type, as V itself is), the
    // sum l takes them as they are.  fp16 holds them from 2^-14 on: moved up by kUp, they keep their precision down
    // to 2^-21 of the reference, and those that vanish, below 2^-32 of it, add up to 2^-12 where 2^20 keys
    // are (without kUp 2^17 keys of 2^-26 each were 2^-9 of l and nothing of o).  bf16 holds any.
    static constexpr float kUp = BF16 ? 0.0f : 7.0f;
    template <int N2>
    __device__ __forceinline__ void weigh(const f32x16 (&s)[N2], u16x8 (&p)[2 * N2], bool again = false) {
        float mc = (m == -INFINITY ? 0.0f : m * c) - kUp, r = 0.0f;
        if (again && out_of_step()) mc = -kUp, r = m;
        float sum = 0.0f;  // the tile's by itself, so that light keys are not lost one by one beside l
#pragma unroll
        for (int g = 0; g < N2; ++g)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(again ? s[g][i] - r : s[g][i], c, -mc));
                sum = i + g ? sum + e : e;
                p[2 * g + (i >> 3)][i & 7] = to16<BF16>(e);
            }
        l += sum;
    }
    __device__ __forceinline__ u16x8 vfrag(const uint8_t* V, int st, int d) const {
        typedef __attribute__((address_space(3))) s16x4* lp;
        const uint8_t* at = V + voff[d] + st * 16 * G::RB;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)at);
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(at + 8 * G::RB));
        u16x8 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = (uint16_t)a[i], r[4 + i] = (uint16_t)b[i];
        return r;
    }
    template <int N2>
    __device__ __forceinline__ void values(const uint8_t* V, const u16x8 (&p)[2 * N2]) {
        // four reads ahead of the products, in this order; only arithmetic may move between them
        constexpr int AHEAD = 4, ALL = 2 * N2 * ND;
        u16x8 f[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) f[i] = vfrag(V, i / ND, i % ND);
#pragma unroll
        for (int i = 0; i < ALL; ++i) {
            __builtin_amdgcn_sched_barrier(kValu | kSalu);
            o[i % ND] = mfma(f[i % AHEAD], p[i / ND], o[i % ND]);
            if (i + AHEAD < ALL) f[i % AHEAD] = vfrag(V, (i + AHEAD) / ND, (i + AHEAD) % ND);
        }
    }
    __device__ __forceinline__ static bool odd(uint16_t v) {  // infinite or NaN
        constexpr uint16_t e = BF16 ? 0x7f80 : 0x7c00;
        return (v & e) == e;
    }
    // Whether one of 32 keys' values is infinite or NaN: an exponent of all ones plus one carries into bit 15.
    __device__ __forceinline__ bool any_odd(const uint8_t* V) const {
        constexpr uint32_t e = BF16 ? 0x7f807f80u : 0x7c007c00u, one = BF16 ? 0x00800080u : 0x04000400u;
        uint32_t t = 0;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {  // the wave's 64 lanes cover the 32 rows, 1 KB a step
            const uint4 v = *(const uint4*)(V + i * 1024 + lane * 16);
            t |= ((v.x & e) + one) | ((v.y & e) + one) | ((v.z & e) + one) | ((v.w & e) + one);
        }
        return __any((t & 0x80008000u) != 0);
    }
    // values() of 32 keys of which some are not finite, and not seen by every row: those are left out, then
    // added key by key to the rows that see them (0 * inf of a masked key would be NaN)
    __device__ __forceinline__ void values_odd(const uint8_t* V, const u16x8 (&p)[2], int left) {
        uint32_t keys = 0;
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                u16x8 v = vfrag(V, st, d);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (odd(v[i])) {
                        keys |= 1u << (16 * st + key_of(i, 0));
                        v[i] = 0;
                    }
                o[d] = mfma(v, p[st], o[d]);
            }
        keys <<= 4 * h;
        keys |= xor_lane_u<1>(keys);
        keys |= xor_lane_u<2>(keys);
        keys |= xor_lane_u<4>(keys);
        keys |= xor_lane_u<8>(keys);
        keys |= xor_lane_u<16>(keys);
        keys |= xor_lane_u<32>(keys);
        for (uint32_t rest = uni((int)keys); rest; rest &= rest - 1) {
            const int k = __builtin_ctz(rest);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                f32x16 a{};
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    u16x8 v = vfrag(V, st, d);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (!odd(v[i]) || 16 * st + key_of(i, 0) != k - 4 * h) v[i] = 0;
                    a = mfma(v, p[st], a);
                }
                if (k < left) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] += a[i];
                }
            }
        }
    }
    // 32 keys with masks; again: the second time of a run that had a row out of step
    __device__ __forceinline__ void checked(const uint8_t* K, const uint8_t* V, int left, int bad, bool again) {
        f32x16 s[1];
        u16x8 p[2];
        scores<1>(K, s);
        mask(s[0], left, bad);
        grow<1>(s);
        if (__builtin_expect(again, 0))
            weigh<1>(s, p, true);
        else
            weigh<1>(s, p);
        if (__builtin_expect(any_odd(V), 0)) {
            values_odd(V, p, left);
            hold_sums();
        } else {
            values<1>(V, p);
        }
    }
};

// Where the block of 16 keys from kb on (a multiple of 16) lies: element offset of its first row in k and v,
// and how many of its rows hold keys (all behind the last key: none; it then stands on the last key's block).
struct Block {
    int64_t at;
    int have, first;  // rows [0, have) are keys; the block's key 0 is row `first` of the rows at `at`
};
__device__ __forceinline__ Block find_block(const AttendArgs& A, const int32_t* pages, int kvh, int kb, int keys) {
    const int last = keys - 1;
    const int ke = kb > last ? last & ~15 : kb;
    int page = sload(pages, ke >> A.C.page_shift);
    if (page < 0 || page >= A.C.n_pages) page = 0;
    Block b;
    b.at = (int64_t)page * A.C.page_stride + (int64_t)kvh * A.C.head_stride +
           (int64_t)(ke & ((1 << A.C.page_shift) - 1)) * A.C.row_stride;
    b.have = keys - ke, b.first = kb - ke;
    return b;
}
// Copies a block's 16 rows of K or V into LDS; rows past the last key are copies of it.
template <int D, bool V>
__device__ __forceinline__ void copy_block(const AttendArgs& A, const uint16_t* cache, const Block& b, int lane, uint32_t lds) {
    using G = Geo<D>;
    const uint16_t* base = cache + b.at;
    const uint32_t rs = (uint32_t)A.C.row_stride * 2;
    asm volatile("" : "+v"(lane));  // offsets made here, not held (or spilled) across the loop
    const int lr = lane / G::LPR, cs = lane % G::LPR;
    auto chunk = [&](int i) {  // the 16-byte chunk that lane's place of copy i holds
        const int r = i * G::RPC + lr;
        return (uint32_t)(V ? cs ^ (2 * G::vswz(r)) : cs ^ (r & G::KM)) << 4;
    };
    if (b.have >= 16 && A.C.row_stride == D) {
        const uint32_t row = (uint32_t)lr * (2 * D);
        if constexpr (G::CPB == 2) {
            copy_lds2(base, row + chunk(0), row + chunk(1), lds);
        } else {
#pragma unroll
            for (int i = 0; i < G::CPB; i += 4)
                copy_lds4(base + i * 512, row + chunk(i), row + chunk(i + 1), row + chunk(i + 2), row + chunk(i + 3),
                          lds + i * 1024);
        }
    } else {
#pragma unroll
        for (int i = 0; i < G::CPB; ++i) {
            const int r = i * G::RPC + lr + b.first;
            copy_lds(base, (uint32_t)(r < b.have ? r : b.have - 1) * rs + chunk(i), lds + i * 1024);
        }
    }
}
// Bit b: the block of 16 keys from key + 16 b on has no page (keys past the last one count as it).
__device__ __forceinline__ int bad_blocks(const AttendArgs& A, const int32_t* pages, int key, int keys, int blocks) {
    int bad = 0;
    for (int i = 0; i < blocks; ++i) {
        const int k = key + 16 * i < keys ? key + 16 * i : keys - 1;
        const int page = sload(pages, k >> A.C.page_shift);
        bad |= (page < 0 || page >= A.C.n_pages) << i;
    }
    return bad;
}

// Four consecutive columns of a finished or partial row.
template <int D, bool BF16>
__device__ __forceinline__ void put4(const AttendArgs& A, const Work& W, bool direct, int64_t row, int d, float4 v,
                                     float inv) {
    if (direct) {
        const uint32_t a = to16<BF16>(v.x * inv) | (uint32_t)to16<BF16>(v.y * inv) << 16;
        const uint32_t b = to16<BF16>(v.z * inv) | (uint32_t)to16<BF16>(v.w * inv) << 16;
        *(uint2*)(A.out + row * D + d) = make_uint2(a, b);
    } else {
        const int64_t R = (int64_t)A.T * A.hq;
        *(float4*)(A.part + (((W.prefix ? 0 : A.own) + W.slot) * R + row) * D + d) = v;
    }
}
// The row's statistics: lse of a finished row, (max, sum) of a partial one; slot 0 says how many there are.
__device__ __forceinline__ void put_row(const AttendArgs& A, const Work& W, bool direct, int64_t row, float m, float l,
                                        bool empty) {
    if (direct) {
        if (A.lse) A.lse[row] = empty ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
    } else {
        const int64_t R = (int64_t)A.T * A.hq;
        A.ml[((W.prefix ? 0 : A.own) + W.slot) * R + row] = make_float2(m, l);
    }
    if (W.slot == 0) {
        A.slots[(W.prefix ? 0 : (int64_t)A.T * A.hq) + row] = empty ? 0 : W.nslots;
        if (W.pre) A.slots[row] = 0;
    }
}

// A wave's rows of one piece of work.
template <int D, bool BF16>
struct Rows {
    int tok, head, seen;
    int64_t orow;
    bool valid, far;
    __device__ __forceinline__ Rows(const AttendArgs& A, const Work& W, int row) {
        valid = row < W.rows;
        const int rc = valid ? row : W.rows - 1;
        tok = group_of(A, rc);
        head = W.kvh * A.group + rc - tok * A.group;
        orow = (int64_t)(W.lo + tok) * A.hq + head;
        far = false;
        seen = W.keys;
        if (!W.prefix) {
            Seq s;
            s.len = W.len, s.n = W.n, s.cap = W.cap;
            seen = s.seen(tok, &far);
        }
    }
    __device__ __forceinline__ void load_q(const AttendArgs& A, const Work& W, Core<D, BF16>& core) const {
        const uint16_t* qp = A.q + (int64_t)(W.lo + tok) * A.q_tok + (int64_t)head * A.q_head + 8 * core.h;
#pragma unroll
        for (int i = 0; i < Core<D, BF16>::NK; ++i) core.q[i] = *(const u16x8*)(qp + 16 * i);
    }
    __device__ __forceinline__ void store(const AttendArgs& A, const Work& W, const Core<D, BF16>& core) const {
        const bool direct = !W.prefix && (!A.B.prefix || W.pre) && W.nslots == 1;
        float l = core.l + core.swap32(core.l);
        if (far) l = NAN;
        const bool empty = !W.prefix && !A.B.prefix && seen == 0;
        const float inv = empty ? 0.0f : 1.0f / l;
        if (!valid) return;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                put4<D, BF16>(A, W, direct, orow, d * 32 + 8 * i + 4 * core.h,
                              make_float4(core.o[d][4 * i], core.o[d][4 * i + 1], core.o[d][4 * i + 2],
                                          core.o[d][4 * i + 3]),
                              inv);
        if (core.h == 0) put_row(A, W, direct, orow, core.m * A.c - core.kUp, l, empty);
    }
};

// Where the tiles from j0 on need no checks any more, up to j1: every key on a page, and of the `least` that
// every row sees.
__device__ __forceinline__ int plain_tiles(const AttendArgs& A, const int32_t* pages, int j0, int j1, int tile, int keys,
                                           int least, int lane) {
    bool ok = true;
    const int k0 = j0 * tile, k1 = j1 * tile < keys ? j1 * tile : keys;
    for (int i = (k0 >> A.C.page_shift) + lane; (int64_t)i << A.C.page_shift < k1; i += 64) {
        const int page = pages[i];
        ok = ok && page >= 0 && page < A.C.n_pages;
    }
    const int jf = __all(ok) ? least / tile : 0;
    return uni(jf < j0 ? j0 : jf < j1 ? jf : j1);
}

template <int D, bool BF16>
__global__ __launch_bounds__(kThreads, Geo<D>::OCC) void attend_kernel(const AttendArgs A) {
    using G = Geo<D>;
    using K = Core<D, BF16>;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[G::LDS];
    __shared__ int s_base[2][kThreads];
    __shared__ int s_seq[kThreads][3];
    __shared__ int s_red[4][6];
    __shared__ int s_far[4];
    const int tid = threadIdx.x, lane = tid & 63, wv = uni(tid >> 6);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)smem;

    // ---- the two axes: split segments are dealt to waves, shared ones to workgroups
    Axis<true> ax0;
    Axis<false> ax1;
    ax0.pre = ax1.pre = 0;
    const int per = (A.B.seqs + kThreads - 1) / kThreads;
    int mine[5] = {0, 0, 0, 0, 0};  // split and shared cost, shared row tiles; the longest segment of each kind
    bool down = false;              // q_start decreases
    for (int i = 0; i < per; ++i) {
        const int b = tid * per + i;
        const bool in = b < A.B.seqs;
        const Seq s = load_seq(A, in ? b : A.B.seqs - 1);
        if (in && A.B.q_start) down = down || A.B.q_start[b + 1] < A.B.q_start[b];
        if (per == 1) s_seq[tid][0] = s.lo, s_seq[tid][1] = s.n, s_seq[tid][2] = s.len;
        mine[0] += ax0.cost(A, s, in, lane) * A.C.heads;
        mine[1] += ax1.cost(A, s, in, lane) * A.C.heads;
        if (in && s.rows) {
            const int k = s.tiles(A, row_tiles(s.rows) - 1), kind = s.split() ? 3 : 4;
            mine[kind] = k > mine[kind] ? k : mine[kind];
            if (!s.split()) mine[2] += row_tiles(s.rows) * A.C.heads;
        }
    }
    int inc[3] = {mine[0], mine[1], mine[2]};
    for (int d = 1; d < 64; d <<= 1) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const int o = __shfl_up(inc[k], d);
            if (lane >= d) inc[k] += o;
        }
#pragma unroll
        for (int k = 3; k < 5; ++k) {
            const int x = __shfl_xor(mine[k], d);
            mine[k] = x > mine[k] ? x : mine[k];
        }
    }
    down = __any(down);
    if (lane == 63) {
#pragma unroll
        for (int k = 0; k < 3; ++k) s_red[wv][k] = inc[k];
        s_red[wv][3] = mine[3], s_red[wv][4] = mine[4], s_red[wv][5] = down;
    }
    __syncthreads();
    // Sequences of a q_start that decreases hold more rows together than the call, and the axis could leave 32 bits:
    // nothing is computed.
    if (uni(s_red[0][5] | s_red[1][5] | s_red[2][5] | s_red[3][5])) return;
    int before[3] = {inc[0] - mine[0], inc[1] - mine[1], inc[2] - mine[2]}, own[3] = {0, 0, 0}, most[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            if (i < wv) before[k] += s_red[i][k];
            own[k] += s_red[i][k];
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) most[k] = s_red[i][3 + k] > most[k] ? s_red[i][3 + k] : most[k];
    }
    int Tq = A.T;
    if (A.B.q_start) {
        const int e = A.B.q_start[A.B.seqs];
        Tq = uni(e < 0 ? 0 : e < Tq ? e : Tq);
    }
    int nsplit;
    {
        int prows = A.B.prefix ? Tq * A.group : 0;
        const bool sp = prows <= kSplitRows;
        const int tile = sp ? kSplitKeys : kSharedKeys, pt = (A.B.prefix + tile - 1) / tile;
        // Prompts: where every sequence fills row tiles of its own, the prefix has as few readers when each
        // row tile goes through it on the way to its own keys, and a row's parts are fewer (six prompts of
        // 200 to 1201 tokens on a prefix of 4097 keys: 444 -> 409 us).  Up to 1.25 times the prefix's row tiles: 64 sequences
        // of 16, 13, 11, 8 and 5 tokens (8 query heads on each of 4 KV heads) behind 4096 keys, 1, 1.23, 1.45, 2 and 3.2
        // times, take 106, 103, 94, 78 and 77 us this way and 120, 102, 91, 72 and 54 apart.
        if (prows && !own[0] && own[2] * 8 <= (row_tiles(prows) * A.C.heads) * 10) {
            ax1.pre = pt;
            prows = 0;
            own[1] += own[2] * pt, before[1] += before[2] * pt, most[1] += pt;
        }
        const int segs = row_tiles(prows) * A.C.heads;
        ax0.ptiles = ax1.ptiles = pt;
        ax0.psegs = sp ? segs : 0;
        ax1.psegs = sp ? 0 : segs;
        if (segs && pt > most[sp ? 0 : 1]) most[sp ? 0 : 1] = pt;
        const int p0 = ax0.psegs * (pt + kSplitHead), p1 = ax1.psegs * (pt + kSharedHead);
        s_base[0][tid] = p0 + before[0];
        s_base[1][tid] = p1 + before[1];
        ax0.total = uni(p0 + own[0]);
        ax1.total = uni(p1 + own[1]);
        // the workgroups by the time that the two kinds take, each kind spread evenly over the grid: the one
        // streams the cache while the other multiplies.  A shared tile counts as 3 split ones: 128 us for 256
        // rows of one token behind 16000 shared keys, against 138 at 1.5, 127 at 2, 130 at 4, 143 at 1; for 64
        // behind 8192 39.5 against 42.9, 40.9, 39.5, 45
        const float c0 = ax0.total, c1 = 3.0f * ax1.total;
        int g0 = (int)((float)gridDim.x * c0 / (c0 + c1 + 1.0f) + 0.5f);
        if (ax0.total && g0 < 1) g0 = 1;
        if (ax1.total && g0 > (int)gridDim.x - 1) g0 = gridDim.x - 1;
        if (!ax1.total) g0 = gridDim.x;
        nsplit = uni(g0);
        // equal runs, long enough that no segment meets more than nslot of them
        const int w0 = (g0 ? g0 : 1) * 4, w1 = (int)gridDim.x - g0 > 0 ? gridDim.x - g0 : 1;
        const int l0 = (most[0] + A.nslot - 3) / (A.nslot - 2), l1 = (most[1] + A.nslot - 3) / (A.nslot - 2);
        ax0.run = (ax0.total + w0 - 1) / w0;
        ax1.run = (ax1.total + w1 - 1) / w1;
        ax0.run = ax0.run > l0 ? ax0.run : l0;
        ax1.run = ax1.run > l1 ? ax1.run : l1;
        ax0.run = uni(ax0.run > kSplitLeast ? ax0.run : kSplitLeast);
        ax1.run = uni(ax1.run > 1 ? ax1.run : 1);
    }
    __syncthreads();

    const int before_me = (int)((int64_t)blockIdx.x * nsplit / gridDim.x);  // workgroups for split segments
    if ((int)((int64_t)(blockIdx.x + 1) * nsplit / gridDim.x) > before_me) {
        // ---- split segments: each wave by itself; the next tile's K is on its way while this one's V is used,
        // and the other way round
        const uint32_t kb = lds0 + wv * 128 * D, vb = kb + 64 * D;
        const uint8_t *kp = smem + wv * 128 * D, *vp = kp + 64 * D;
        const int who = wv * nsplit + before_me;  // neighbouring runs on other CUs
        int at = ax0.total / ax0.run < who ? ax0.total : who * ax0.run;
        const int end = at + ax0.run < ax0.total ? at + ax0.run : ax0.total;
        while (at < end) {
            Work W = ax0.find(A, s_base[0], s_seq, per, Tq, at, end, who, lane);
            W.scalar();
            at = end - W.left;
            if (W.j0 >= W.j1) continue;
            const int32_t* pages = W.prefix ? A.B.prefix_pages : A.B.table + (int64_t)W.b * A.B.table_stride;
            Block b0, b1;
            auto bring_k = [&](int key) {  // and where the same keys' values are
                b0 = find_block(A, pages, W.kvh, key, W.keys);
                b1 = find_block(A, pages, W.kvh, key + 16, W.keys);
                copy_block<D, false>(A, A.C.k, b0, lane, kb);
                copy_block<D, false>(A, A.C.k, b1, lane, kb + 32 * D);
            };
            auto bring_v = [&]() {
                copy_block<D, true>(A, A.C.v, b0, lane, vb);
                copy_block<D, true>(A, A.C.v, b1, lane, vb + 32 * D);
            };
            const int stop = W.j1 * kSplitKeys < W.keys ? W.j1 * kSplitKeys : W.keys;
            K core;
            core.c = A.c;
            const Rows<D, BF16> R(A, W, lane & 31);
            bool again = false;
            do {
                int key = W.j0 * kSplitKeys;
                core.begin(lane);
                R.load_q(A, W, core);
                if (key < stop) bring_k(key), bring_v();
                const int jf = again ? W.j0 : plain_tiles(A, pages, W.j0, W.j1, kSplitKeys, W.keys, uni(R.seen), lane);
                core.hold();  // arrived before the loops
                for (int j = W.j0; j < jf; ++j) {
                    core.hold_sums();
                    const int next = key + kSplitKeys;
                    f32x16 s[1];
                    u16x8 p[2];
                    vm_wait<D / 16>();
                    core.template scores<1>(kp, s);
                    lds_wait();
                    if (next < stop) bring_k(next);
                    core.template grow<1>(s);
                    core.template weigh<1>(s, p);
                    if (next < stop)
                        vm_wait<D / 16>();
                    else
                        vm_wait<0>();
                    core.template values<1>(vp, p);
                    lds_wait();
                    if (next < stop) bring_v();
                    key = next;
                }
                for (; key < stop; key += kSplitKeys) {
                    vm_wait<0>();
                    core.hold_sums();
                    core.checked(kp, vp, R.seen - key, bad_blocks(A, pages, key, W.keys, 2), again);
                    lds_wait();
                    if (key + kSplitKeys < stop) bring_k(key + kSplitKeys), bring_v();
                }
                again = !again && core.far;
            } while (__builtin_expect(again, 0));
            R.store(A, W, core);
        }
    } else {
        // ---- shared segments: the four waves take 32 rows each and every tile together, in two buffers of K and V
        const int who = blockIdx.x - before_me;
        int at = ax1.total / ax1.run < who ? ax1.total : who * ax1.run;
        const int end = at + ax1.run < ax1.total ? at + ax1.run : ax1.total;
        while (at < end) {
            Work W = ax1.find(A, s_base[1], s_seq, per, Tq, at, end, who, lane);
            W.scalar();
            at = end - W.left;
            if (W.j0 >= W.j1) continue;
            const int32_t* pages = W.prefix ? A.B.prefix_pages : A.B.table + (int64_t)W.b * A.B.table_stride;
            const bool works = 32 * wv < W.rows - W.row0;
            auto bring = [&](int j) {
                const uint32_t buf = lds0 + (j & 1) * 256 * D + wv * 32 * D;
                const bool p = j < W.pre;
                const Block b = find_block(A, p ? A.B.prefix_pages : pages, W.kvh,
                                           (p ? j : j - W.pre) * kSharedKeys + 16 * wv, p ? A.B.prefix : W.keys);
                copy_block<D, false>(A, A.C.k, b, lane, buf);
                copy_block<D, true>(A, A.C.v, b, lane, buf + 128 * D);
            };
            // a segment without own keys still has a tile for them, which is skipped
            const int last = W.keys > 0 ? W.j1 : W.pre < W.j1 ? W.pre : W.j1;
            const int stop = last > W.j0 ? last : W.j0;
            K core;
            core.c = A.c;
            const Rows<D, BF16> R(A, W, W.row0 + 32 * wv + (lane & 31));
            bool again = false;
            do {
                core.begin(lane);
                R.load_q(A, W, core);
                lds_barrier();  // every wave is done with the last segment's buffers
                if (W.j0 < stop) bring(W.j0);
                int j = W.j0;
#pragma unroll 1
                for (int part = 0; part < 2; ++part) {  // the prefix's tiles, which every row sees, then the own keys'
                    const int from = part ? W.pre : 0, to = part || stop < W.pre ? stop : W.pre;
                    if (j >= to) continue;
                    const int32_t* where = part ? pages : A.B.prefix_pages;
                    const int keys = part ? W.keys : A.B.prefix;
                    const int seen = part ? R.seen : keys;
                    const int seen1 = __builtin_amdgcn_readlane(seen, 31);  // the wave's last row sees most
                    int least = keys;
                    if (part && !W.prefix) {  // the first row of the whole tile sees least
                        Seq s;
                        s.len = W.len, s.n = W.n, s.cap = W.cap;
                        least = s.seen(group_of(A, W.row0));
                    }
                    const int jf =
                        again ? j : from + plain_tiles(A, where, j - from, to - from, kSharedKeys, keys, least, lane);
                    core.hold();  // arrived before the loops
                    for (; j < jf; ++j) {
                        vm_wait<0>();
                        lds_barrier();
                        if (j + 1 < stop) bring(j + 1);
                        const uint8_t* buf = smem + (j & 1) * 256 * D;
                        if (works) {
                            core.hold_sums();
                            f32x16 s[2];
                            u16x8 p[4];
                            core.template scores<2>(buf, s);
                            core.template grow<2>(s);
                            core.template weigh<2>(s, p);
                            core.template values<2>(buf + 128 * D, p);
                        }
                    }
                    for (; j < to; ++j) {
                        vm_wait<0>();
                        lds_barrier();
                        if (j + 1 < stop) bring(j + 1);
                        const uint8_t* buf = smem + (j & 1) * 256 * D;
#pragma unroll 1
                        for (int half = 0; half < 2 && works; ++half) {
                            const int key = (j - from) * kSharedKeys + 32 * half;
                            if (key >= seen1) break;
                            core.hold_sums();
                            core.checked(buf + half * 64 * D, buf + 128 * D + half * 64 * D, seen - key,
                                         bad_blocks(A, where, key, keys, 2), again);
                        }
                    }
                }
                if (again) break;
                if (lane == 0) s_far[wv] = core.far;  // the waves share the tiles
                lds_barrier();
                again = uni(s_far[0] | s_far[1] | s_far[2] | s_far[3]);
            } while (__builtin_expect(again, 0));
            R.store(A, W, core);
        }
    }
}

// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over a row's slots: GROUPS groups of D / 4 threads take
// every GROUPS-th slot each, then meet in group order.
template <int D, bool BF16, int GROUPS>
__global__ __launch_bounds__(kThreads) void combine_rows_kernel(const AttendArgs A) {
    constexpr int LPR = D / 4;                       // threads of a group, 4 columns each
    constexpr int RPB = kThreads / (LPR * GROUPS);   // rows of a workgroup
    __shared__ float4 s_o[kThreads];
    const int tid = threadIdx.x;
    const int g = (tid / LPR) % GROUPS, c = tid % LPR;
    const int64_t R = (int64_t)A.T * A.hq;
    const int64_t row = (int64_t)blockIdx.x * RPB + tid / (LPR * GROUPS);
    int ns = 0, np = 0;
    bool live = row < R && row < (int64_t)(A.B.q_start ? A.B.q_start[A.B.seqs] : A.B.seqs) * A.hq;
    if (live) {
        ns = A.slots[R + row];
        np = A.B.prefix ? A.slots[row] : 0;
        live = np || ns != 1;  // else written by the only run that had it
        ns = ns < 0 ? 0 : ns > A.nslot ? A.nslot : ns;
        np = np < 0 ? 0 : np > A.nslot ? A.nslot : np;
    }
    const bool empty = !A.B.prefix && ns == 0;
    const int all = live ? np + ns : 0;
    auto place = [&](int s) { return (s < np ? s : A.own + s - np) * R + row; };
    float mx = -INFINITY;
    for (int s = c; s < all; s += LPR) mx = fmaxf(mx, A.ml[place(s)].x);
    for (int d = LPR < 64 ? LPR / 2 : 32; d; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
    const float ref = mx == -INFINITY ? 0.0f : mx;
    float4 o = make_float4(0, 0, 0, 0);
    float sum = 0.0f;
#pragma unroll 4
    for (int s = g; s < all; s += GROUPS) {
        const int64_t at = place(s);
        const float2 ml = A.ml[at];
        const float4 p = *(const float4*)(A.part + at * D + 4 * c);
        const float f = __builtin_amdgcn_exp2f(ml.x - ref);
        sum += f * ml.y;
        o.x += f * p.x, o.y += f * p.y, o.z += f * p.z, o.w += f * p.w;
    }
    if constexpr (GROUPS > 1) {
        __shared__ float s_l[kThreads];
        s_o[tid] = o;
        s_l[tid] = sum;
        __syncthreads();
        if (g == 0)
#pragma unroll
            for (int i = 1; i < GROUPS; ++i) {
                const float4 p = s_o[tid + i * LPR];
                o.x += p.x, o.y += p.y, o.z += p.z, o.w += p.w;
                sum += s_l[tid + i * LPR];
            }
    }
    if (!live || g) return;
    const float inv = empty ? 0.0f : 1.0f / sum;
    const uint32_t a = to16<BF16>(o.x * inv) | (uint32_t)to16<BF16>(o.y * inv) << 16;
    const uint32_t b = to16<BF16>(o.z * inv) | (uint32_t)to16<BF16>(o.w * inv) << 16;
    *(uint2*)(A.out + row * D + 4 * c) = make_uint2(a, b);
    if (A.lse && c == 0) A.lse[row] = empty ? -INFINITY : (mx + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
}

static int attend_slots(int64_t rows, int D) {
    // Slots of every row, in each region: 130 (a long sequence alone on the chip), fewer where a region would pass 256
    // MiB, 4 at least, which passes it from 65536 rows of 256 on (8192 tokens of 32 heads of 128: 522 MiB, 1042 behind
    // a prefix).  A segment is cut into nslot - 2 runs at most: beside a prompt of 2048 tokens one sequence of
    // 100000 keys runs on few waves (689 us the call; 79 and 87 each in a call of its own).
    int64_t n = ((int64_t)256 << 20) / (rows * D * 4);
    return (int)(n < 4 ? 4 : n > 130 ? 130 : n);
}
struct AttendWs {
    int64_t ml, slots, total;
    int nslot;
};
static AttendWs attend_ws(const KvCache& C, const KvBatch& B, int T, int hq) {
    const int64_t R = (int64_t)T * hq;
    AttendWs w;
    w.nslot = attend_slots(R, C.dim);
    const int regions = B.prefix ? 2 : 1;
    w.ml = R * w.nslot * regions * C.dim * 4;
    w.slots = w.ml + R * w.nslot * regions * 8;
    w.total = (w.slots + R * 2 * 4 + 255) / 256 * 256;
    return w;
}
size_t attend_ws_bytes(const KvCache& C, const KvBatch& B, int T, int hq) { return attend_ws(C, B, T, hq).total; }

static int cu_count() {
    static std::atomic<int> cached[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    int n = cached[dev].load(std::memory_order_relaxed);
    if (!n) {
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
        cached[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

int launch_attend(const KvCache& C, const KvBatch& B, const uint16_t* q, int64_t q_tok, int64_t q_head, int T, int hq,
                  float scale, uint16_t* out, float* lse, void* ws, hipStream_t st) {
    if (T == 0) return PGMOE_OK;
    const AttendWs w = attend_ws(C, B, T, hq);
    uint8_t* b = (uint8_t*)ws;
    const int group = hq / C.heads;
    const AttendArgs A{C,   B,         q,   q_tok, q_head, T, hq, group, (uint32_t)(0x100000000ull / group + (group > 1)),
                       scale * 1.4426950408889634f, out, lse, (float*)b, (float2*)(b + w.ml), (int*)(b + w.slots), w.nslot, B.prefix ? w.nslot : 0};
    const int64_t R = (int64_t)T * hq;
    const dim3 block(kThreads);
    // Few rows have many slots each: 1024 / D groups a row, one row a workgroup; many have few.  One sequence of
    // 5003 keys (32 rows) 16.4 us, 25.3 with one group a row; 200 sequences of 1 to 60 keys (6400 rows) 17.1 with
    // one, 20.6 with eight.
    const bool few = R <= 2048;
#define COMBINE(D, BF)                                                                                           \
    do {                                                                                                         \
        if (few)                                                                                                 \
            PG_LAUNCH((combine_rows_kernel<D, BF, 1024 / D>), dim3((unsigned)R), block, 0, st, A);               \
        else                                                                                                     \
            PG_LAUNCH((combine_rows_kernel<D, BF, 1>), dim3((unsigned)((R * D + 1023) / 1024)), block, 0, st, A); \
    } while (0)
#define ATT(D)                                                               \
    do {                                                                     \
        const dim3 grid(cu_count() * Geo<D>::OCC);                           \
        if (C.bf16) {                                                        \
            PG_LAUNCH((attend_kernel<D, true>), grid, block, 0, st, A);      \
            COMBINE(D, true);                                                \
        } else {                                                             \
            PG_LAUNCH((attend_kernel<D, false>), grid, block, 0, st, A);     \
            COMBINE(D, false);                                               \
        }                                                                    \
    } while (0)
    if (C.dim == 64)
        ATT(64);
    else if (C.dim == 128)
        ATT(128);
    else
        ATT(256);
#undef ATT
#undef COMBINE
    return check_launch("attend");
}

}  // namespace pgmoe
