// fp8.cu -- e4m3 quantisation with a float32 scale per block of 128, and the product
//
//   y[m, n] = sum_j xs[m, j] ws[n / 128, j]  sum_{k in block j} xq[m, k] wq[n, k]
//
// on the tensor cores.  The scales differ from K block to K block, so the inner sums cannot stay in
// one accumulator: each 128-wide block is one short product (four tcgen05.mma of K = 32) into one of
// two tensor-memory accumulators, and the epilogue warps read it back, scale it and add it in
// float32 registers while the tensor core fills the other.  One warp moves tiles by TMA (128-byte
// swizzle; the tensor map's extents fill ragged edges with zeros, which are zeros in e4m3), one
// issues the products, one copies the scales.  What bounds it is the epilogue: a K block's 128 x 256
// sums take some 1000 cycles to read, scale and add, against 540 for the products (8192^3: 508 us,
// 2.2 PFLOP/s).
//
// The operand with 128 rows a tile (the tensor core's M) is x for many tokens and w for few: then a
// tile is 128 weight rows by all the tokens (16 to 64), the weights stream once, and K is split over
// a cluster of up to 8 CTAs whose partial sums meet in shared memory in a fixed order (so it is for few
// tiles of many tokens and a long K).  64 x 32000 x 768:
// 11.6 us, against 4.4 for its bytes: latency of set-up, six K blocks and the stores.
#include <cooperative_groups.h>

#include <type_traits>

#include "fp8.cuh"

#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace pma {

namespace {

using namespace tc;

// -------------------------------------------------------------------------------- quantisation
// e4m3 of 448 x / amax, nearest even, where float32 x has the product and the quotient rounded to float32
// first, as the same expression in any float32 arithmetic has (an x within 2 ulp of half-way between two
// e4m3 values on the block's scale may go to either); for bf16 x that is the nearest to the exact quotient.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
//
// float32: the division is only made where it can matter: x (448 / amax) is within 3 ulp of the quotient,
// which rounds to the same e4m3 value unless it lies that close to the middle of two (or is below 2^-6,
// where e4m3's spacing is fixed).
// bf16: never made. x and amax have 8 significant bits X and A, a middle t has 5, T: a quotient 7 X / A 2^n
// that is not t differs from it by 1 / (7 * 255) or 1 / (31 * 255) of its size or more, over 2^-13. So
// v = x (448 / amax), rounded to 16 bits, is t where the quotient is and on the quotient's side of t where
// it is not. The rounding: with d = 256 v, d - (d - v) is a multiple of d's last place (or half of it), and
// so is t.
struct Quant {
    float amax, pre, fast;
    bool plain;  // a block without NaN, infinities and huge values
    // amax of 0 (or below 2^-100) counts as 2^-100; a block of huge values is divided by 2^20 first,
    // so that 448 x stays finite
    __device__ __forceinline__ explicit Quant(float a) : amax(fmaxf(a, 7.888609052210118e-31f)), pre(448.0f),
          plain(a < 1e30f) {
        if (amax > 1e35f) {
            pre *= 9.5367431640625e-07f;
            amax *= 9.5367431640625e-07f;
        }
        fast = __fmul_rn(pre, __frcp_rn(amax));
    }
    __device__ __forceinline__ float exact(float x) const { return __fdiv_rn(x * pre, amax); }
    static __device__ __forceinline__ float scale(float a) {
        return a == a ? fmaxf(a, 7.888609052210118e-31f) / 448.0f : a;
    }
};

// NaN is kept: a block that holds one gets a NaN scale
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Eight consecutive elements of a row, zero past K.
template <typename T> struct Eight;
template <> struct Eight<float> {
    float v[8];
    __device__ __forceinline__ void load(const float *row, int k, int K, bool vec) {
        if (vec && k + 8 <= K) {
            const float4 a = load4(row + k), b = load4(row + k + 4);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
            v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = k + i < K ? row[k + i] : 0.f;
        }
    }
    __device__ __forceinline__ float at(int i) const { return v[i]; }
    __device__ __forceinline__ float amax() const {
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = max_nan(a, fabsf(v[i]));
        return a;
    }
};
template <> struct Eight<__nv_bfloat16> {
    uint32_t v[4];
    __device__ __forceinline__ void load(const __nv_bfloat16 *row, int k, int K, bool vec) {
        if (vec && k + 8 <= K) {
            const uint4 a = __ldg(reinterpret_cast<const uint4 *>(row + k));
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        } else {
            const unsigned short *r = reinterpret_cast<const unsigned short *>(row);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = (k + 2 * i < K ? r[k + 2 * i] : 0u) | (k + 2 * i + 1 < K ? (uint32_t)r[k + 2 * i + 1] : 0u) << 16;
        }
    }
    __device__ __forceinline__ float at(int i) const {
        return __uint_as_float(i & 1 ? v[i / 2] & 0xffff0000u : v[i / 2] << 16);
    }
    __device__ __forceinline__ float amax() const {  // two at a time, exact in bf16
        uint32_t a = v[0] & 0x7fff7fffu;
#pragma unroll
        for (int i = 1; i < 4; ++i) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(v[i] & 0x7fff7fffu));
        return max_nan(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
    }
};
__device__ __forceinline__ void store8(uint8_t *row, int k, int K, uint2 v) {
    if (k + 8 <= K) {
        *reinterpret_cast<uint2 *>(row + k) = v;  // rows start on 16 bytes, k is a multiple of 8
    } else {
        for (int i = 0; i < 8 && k + i < K; ++i) row[k + i] = (uint8_t)((i < 4 ? v.x : v.y) >> (8 * (i & 3)));
    }
}
template <typename E> __device__ __forceinline__ uint2 quant8(const E &x, const Quant &q) {
    float v[8], small = INFINITY;
    uint32_t off = 0xffffffffu;  // distance of the 20 bits below e4m3's significand from their middle, + 4
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = __fmul_rn(x.at(i), q.fast);
        off = min(off, __float_as_uint(v[i]) - 0x7fffcu & 0xfffffu);
        small = fminf(small, fabsf(v[i]));
    }
    if (off <= 8u || !(small >= 0.015625f)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = q.exact(x.at(i));
    }
    return make_uint2(e4m3x2(v[0], v[1]) | e4m3x2(v[2], v[3]) << 16, e4m3x2(v[4], v[5]) | e4m3x2(v[6], v[7]) << 16);
}

__device__ __forceinline__ uint2 quant8(const Eight<__nv_bfloat16> &x, const Quant &q) {
    float v[8];
    if (q.plain) {
        const float2 f256 = make_float2(q.fast * 256.0f, q.fast * 256.0f), neg = make_float2(-q.fast, -q.fast);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 e = make_float2(x.at(i), x.at(i + 1));
            const float2 d = __fmul2_rn(e, f256), c = __ffma2_rn(e, neg, d);
            const float2 r = __ffma2_rn(c, make_float2(-1.0f, -1.0f), d);
            v[i] = r.x, v[i + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = q.exact(x.at(i));
    }
    return make_uint2(e4m3x2(v[0], v[1]) | e4m3x2(v[2], v[3]) << 16, e4m3x2(v[4], v[5]) | e4m3x2(v[6], v[7]) << 16);
}

// Lets the product that follows in the stream start: it waits for this grid before it reads q.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// 8192 x 8192: bf16 in 38 us, 5.3 TB/s; float32 in 51 us, 6.5 TB/s, the rate of a copy. 16 lanes a
// block and 8 elements a lane, with twice the shuffles and work per block: 47 and 64. bf16 with float32's
// checks 61, with a division an element 71.
// 8 lanes a block of 128, two pieces of 8 elements each; a lane group takes GROUPS neighbouring blocks of a
// row (its loads in flight together).
template <typename T, int GROUPS>
__global__ void __launch_bounds__(256) quantize_rows(const T *__restrict__ x, int64_t xs, uint32_t items, int K,
                                                    uint32_t per_row, bool vec, uint8_t *__restrict__ q, int64_t qs,
                                                    float *__restrict__ scale, int64_t si, int64_t sj) {
    launch_dependents();
    const uint32_t g = blockIdx.x * 32u + (threadIdx.x >> 3);
    const bool on = g < items;
    const uint32_t m = on ? g / per_row : 0, j0 = on ? (g - m * per_row) * GROUPS : 0;
    const int k0 = (int)j0 * FP8_BLOCK + (threadIdx.x & 7) * 8;
    x += (int64_t)m * xs;
    q += (int64_t)m * qs;
    Eight<T> v[2 * GROUPS];
#pragma unroll
    for (int i = 0; i < 2 * GROUPS; ++i) v[i].load(x, on ? k0 + i * (FP8_BLOCK / 2) : K, K, vec);
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        float a = max_nan(v[2 * i].amax(), v[2 * i + 1].amax());
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
        const int k = k0 + i * FP8_BLOCK;
        if (on && (int)(j0 + i) * FP8_BLOCK < K) {
            const Quant qu(a);
            store8(q, k, K, quant8(v[2 * i], qu));
            store8(q, k + FP8_BLOCK / 2, K, quant8(v[2 * i + 1], qu));
            if ((threadIdx.x & 7) == 0) scale[(int64_t)m * si + (int64_t)(j0 + i) * sj] = Quant::scale(a);
        }
    }
}

// One CTA a 128 x 128 block of weights: 256 threads, 16 lanes a row.
template <typename T>
__global__ void __launch_bounds__(256) quantize_blocks(const T *__restrict__ w, int64_t ws, int N, int K, int blocks,
                                                      bool vec, uint8_t *__restrict__ q, int64_t qs,
                                                      float *__restrict__ scale) {
    __shared__ float s[8];
    const int nb = blockIdx.x / blocks, j = blockIdx.x - nb * blocks;
    const int l = threadIdx.x & 15, r0 = threadIdx.x >> 4, k = j * FP8_BLOCK + l * 8;
    float a = 0.f;
    for (int r = r0; r < FP8_BLOCK; r += 16) {
        const int n = nb * FP8_BLOCK + r;
        if (n >= N) break;
        Eight<T> v;
        v.load(w + (int64_t)n * ws, k, K, vec);
        a = max_nan(a, v.amax());
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = a;
    __syncthreads();
    a = s[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) a = max_nan(a, s[i]);
    const Quant qu(a);
    for (int r = r0; r < FP8_BLOCK; r += 16) {
        const int n = nb * FP8_BLOCK + r;
        if (n >= N) break;
        Eight<T> v;
        v.load(w + (int64_t)n * ws, k, K, vec);  // from L1 or L2: the block was just read
        store8(q + (int64_t)n * qs, k, K, quant8(v, qu));
    }
    if (threadIdx.x == 0) scale[(int64_t)nb * blocks + j] = Quant::scale(a);
}

// ------------------------------------------------------------------------------------- product
// Instruction descriptor, kind::f8f6f4: e4m3 x e4m3 -> float32, both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N) {
    return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(acc)
        : "memory");
}
// The same over the CTAs of a pair: 256 rows of A, 128 of each CTA, and 256 of B, 128 of each; every
// CTA's tensor memory gets its 128 rows of the result.  Issued by the pair's first CTA.
__device__ __forceinline__ void mma_e4m3_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(acc)
        : "memory");
}
// arrives on the barrier at this place in both CTAs once the products so far are complete
__device__ __forceinline__ void commit_pair(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(su32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
// the address of this place in the pair's first CTA
__device__ __forceinline__ uint32_t in_first(const void *p) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(su32(p)));
    return r;
}
__device__ __forceinline__ void arrive_in_first(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(in_first(bar)) : "memory");
}
// into this CTA's shared memory, counted on a barrier of the pair's first CTA
__device__ __forceinline__ void tma_load2_pair(void *dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
        "[%2];" ::"r"(su32(dst)),
        "l"(map), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void tma_load2(void *dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            su32(dst)),
        "l"(map), "r"(su32(bar)), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void tmem_issue(uint32_t t, uint32_t (&r)[16]) { tmem_ld16_issue(t, r); }
__device__ __forceinline__ void tmem_issue(uint32_t t, uint32_t (&r)[32]) { tmem_ld32_issue(t, r); }
// The kernel before this one in the stream is complete and its writes are visible.
__device__ __forceinline__ void wait_for_x() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void copy4(float *dst, const float *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(su32(dst)), "l"(src) : "memory");
}
// arrives on `bar` when this thread's copies so far have landed
__device__ __forceinline__ void copies_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(su32(bar)) : "memory");
}
// two float32 products and sums at once
__device__ __forceinline__ void fma2(unsigned long long &acc, uint32_t lo, uint32_t hi, unsigned long long s) {
    unsigned long long d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(d), "l"(s));
}
__device__ __forceinline__ unsigned long long pair(float v) {
    unsigned long long d;
    asm("mov.b64 %0, {%1, %1};" : "=l"(d) : "f"(v));
    return d;
}
__device__ __forceinline__ float half_of(unsigned long long v, int i) {
    return __uint_as_float((uint32_t)(i ? v >> 32 : v));
}

constexpr int OUT_PITCH = 80;  // bytes between rows of 64: 16-byte accesses of 8 lanes hit all banks

// 32 rows of 64 bytes in shared memory to `rows` rows of `cols` elements at y (row stride ys).
template <typename T>
__device__ __forceinline__ void store_rows(const uint8_t *s, T *y, int64_t ys, int rows, int cols, int lane) {
    constexpr int PER = 64 / sizeof(T), E16 = 16 / sizeof(T);
    if (rows <= 0 || cols <= 0) return;
    if (cols == PER && reinterpret_cast<uintptr_t>(y) % 16 == 0 && ys % E16 == 0) {
        const int q = lane & 3;
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += 8) {
            const int r = r0 + (lane >> 2);
            if (r < rows)
                *reinterpret_cast<uint4 *>(y + r * ys + q * E16) = *reinterpret_cast<const uint4 *>(s + r * OUT_PITCH + q * 16);
        }
    } else {
        constexpr int RPI = 32 / PER;  // rows a store covers: 1 (bf16) or 2 (float32)
        const int c = lane % PER;
        if (c < cols)
            for (int r = lane / PER; r < rows; r += RPI)
                y[r * ys + c] = *reinterpret_cast<const T *>(s + r * OUT_PITCH + c * sizeof(T));
    }
}

// BN: rows of the second operand in a tile; FEW: w is the 128-row operand.  BN = 256 runs on pairs of
// CTAs: a tile of 256 x 256, each CTA with half of both operands in shared memory, which halves what it
// stages and reads for a product.
template <int BN, bool FEW> struct Cfg {
    static constexpr bool PAIR = BN == 256;
    static constexpr int ROWS = PAIR ? 256 : 128;      // of the first operand in a tile
    static constexpr int EPI = BN == 256 ? 8 : 4;      // epilogue warps: 128 lanes x COLS columns each group of 4
    static constexpr int COLS = BN == 256 ? 128 : BN;  // accumulator columns of a thread
    static constexpr int WARPS = BN == 256 ? 12 : 7;   // and TMA, products, scales
    static constexpr int SLOT = (BN > 128 ? BN : 128) + 4;  // floats: one K block's scales
    static constexpr int THREADS = WARPS * 32;
    static constexpr int A_BYTES = 128 * 128, B_BYTES = (PAIR ? BN / 2 : BN) * 128, STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = BN >= 128 ? 6 : 4;
    static constexpr int TCOLS = 2 * BN < 32 ? 32 : 2 * BN;
    // K split: partial sums [BN][128] float32 take the place of the tiles
    static constexpr int SMEM = STAGES * STAGE + 1024;
};

constexpr int SLOTS = 8;  // K blocks whose scales are on their way or in use

template <int STAGES> struct Bars {
    uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], sc_full[SLOTS], sc_empty[SLOTS], never;
    uint32_t tmem;
    CtlShared ctl;
};

template <int BN, bool FEW>
__global__ void __launch_bounds__(Cfg<BN, FEW>::THREADS, FEW ? 2 : 1)
    fp8_matmul_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                      const Fp8Params p) {
    using G = Cfg<BN, FEW>;
    extern __shared__ uint8_t raw[];
    __shared__ Bars<G::STAGES> sm;
    __shared__ __align__(16) float scales[SLOTS][G::SLOT];
    __shared__ __align__(16) uint8_t out_s[FEW ? 1 : G::EPI][FEW ? 16 : 32 * OUT_PITCH];
    uint8_t *tiles = smem_align1024(raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    Ctl ctl{&sm.ctl, nullptr};

    if (tid == 0) {
        for (int i = 0; i < G::STAGES; ++i) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.acc_full[i], 1);
            mbar_init(&sm.acc_empty[i], G::PAIR ? 2 * G::EPI : G::EPI);  // used in the pair's first CTA
        }
        for (int i = 0; i < SLOTS; ++i) {
            mbar_init(&sm.sc_full[i], 32);
            mbar_init(&sm.sc_empty[i], G::EPI);
        }
        mbar_init(&sm.never, 1);
        init_ctl(sm.ctl, p.fault);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        if constexpr (G::PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&sm.tmem)),
                         "r"(G::TCOLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&sm.tmem)),
                         "r"(G::TCOLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    if constexpr (G::PAIR)
        cg::this_cluster().sync();  // both CTAs' barriers are set up
    else
        __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    const int half = G::PAIR ? (int)cg::this_cluster().block_rank() : 0;
    bool skip = false;
    if (p.test_wait_ns) {  // test hook: a wait expires before any copy or product is issued
        if (tid == 0) expire_test_wait(&sm.never, ctl, p.test_wait_ns, 130);
        __syncthreads();
        skip = ctl.aborted();
    }

    // Tiles of this CTA: one, with a share of the K blocks, or every gridDim.x-th.
    int split = 0, splits = 1, first = blockIdx.x, step = gridDim.x;
    if (G::PAIR) {
        first = blockIdx.x / 2;
        step = gridDim.x / 2;
    }
    if (!G::PAIR) {
        const cg::cluster_group cl = cg::this_cluster();
        split = (int)cl.block_rank();
        splits = (int)cl.num_blocks();
        if (FEW || splits > 1) {
            first = blockIdx.x / splits;
            step = p.tiles_a * p.tiles_b;
        }
    }
    const int all = skip ? 0 : p.tiles_a * p.tiles_b;
    const int j0 = (int)((int64_t)p.blocks * split / splits), j1 = (int)((int64_t)p.blocks * (split + 1) / splits);
    // Tiles go down a band of 16 row tiles before they go right, so that the CTAs at work share
    // rows and columns in L2.
    auto tile_at = [&](int t, int &ia, int &ib) {
        const int band = t / (16 * p.tiles_b), h = min(16, p.tiles_a - band * 16), r = t - band * 16 * p.tiles_b;
        ib = r / h;
        ia = band * 16 + r - ib * h;
    };

    if (warp >= G::EPI) {
        // registers to the accumulators: 256 x 224 + 128 x 56 = 384 x 168
        if (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == G::EPI) {
            // ------------------------------------------------------------------ TMA
            if (lane == 0) {
                // Until the kernel before has written x, load weights only.
                auto load_w = [&](int s, int j, int ia, int ib) {
                    if constexpr (G::PAIR)
                        tma_load2_pair(tiles + s * G::STAGE + G::A_BYTES, &tb, in_first(&sm.full[s]), j * 128, ib * BN + half * 128);
                    else if (FEW)
                        tma_load2(tiles + s * G::STAGE, &ta, &sm.full[s], j * 128, ia * 128);
                    else
                        tma_load2(tiles + s * G::STAGE + G::A_BYTES, &tb, &sm.full[s], j * 128, ib * BN);
                };
                auto load_x = [&](int s, int j, int ia, int ib) {
                    if constexpr (G::PAIR)
                        tma_load2_pair(tiles + s * G::STAGE, &ta, in_first(&sm.full[s]), j * 128, ia * 256 + half * 128);
                    else if (FEW)
                        tma_load2(tiles + s * G::STAGE + G::A_BYTES, &tb, &sm.full[s], j * 128, ib * BN);
                    else
                        tma_load2(tiles + s * G::STAGE, &ta, &sm.full[s], j * 128, ia * 128);
                };
                uint32_t n = 0;
                bool ok = true;
                const int early = first < all ? min(G::STAGES, j1 - j0) : 0;
                int ia, ib;
                tile_at(first, ia, ib);
                auto expect = [&](int s) {
                    if (half == 0) mbar_expect_tx(&sm.full[s], G::PAIR ? 2 * G::STAGE : G::STAGE);
                };
                for (int i = 0; i < early; ++i) {
                    expect(i);
                    load_w(i, j0 + i, ia, ib);
                }
                wait_for_x();
                for (int t = first; ok && t < all; t += step) {
                    tile_at(t, ia, ib);
                    for (int j = j0; j < j1; ++j, ++n) {
                        const int s = n % G::STAGES;
                        if (n >= (uint32_t)early) {
                            if (!(ok = mbar_wait(&sm.empty[s], ((n / G::STAGES) & 1) ^ 1, ctl, 131))) break;
                            expect(s);
                            load_w(s, j, ia, ib);
                        }
                        load_x(s, j, ia, ib);
                    }
                }
                // never leave with copies in flight (a pair's are waited for by its first CTA, whose barriers
                // count them; the second leaves after it, and where it gave up, after a while)
                if (half && !ok)
                    for (const unsigned long long w0 = gtimer(); gtimer() - w0 < 10000000ull;) {
                    }
                for (uint32_t i = half ? n : n > G::STAGES ? n - G::STAGES : 0; i < n; ++i) {
                    const unsigned long long w0 = gtimer();
                    while (!mbar_try(&sm.full[i % G::STAGES], (i / G::STAGES) & 1) && gtimer() - w0 < WAIT_NS) {
                    }
                }
            }
        } else if (warp == G::EPI + 1) {
            // ------------------------------------------------------------------ products
            if (lane == 0 && half == 0) {
                constexpr uint32_t ID = idesc_e4m3(G::ROWS, BN);
                constexpr uint64_t HI = desc_hi(16, 1024, 2);  // K-major rows of 128 bytes, 128-byte swizzle
                const uint32_t base = su32(tiles) >> 4;
                uint32_t n = 0;
                bool ok = true;
                for (int t = first; ok && t < all; t += step)
                    for (int j = j0; j < j1; ++j, ++n) {
                        const int s = n % G::STAGES, a = n & 1;
                        if (!(ok = mbar_wait(&sm.acc_empty[a], ((n >> 1) & 1) ^ 1, ctl, 132))) break;
                        if (!(ok = mbar_wait(&sm.full[s], (n / G::STAGES) & 1, ctl, 133))) break;
                        tc_fence_after();
                        const uint64_t da = (uint64_t)(base + s * (G::STAGE >> 4)) | HI;
                        const uint64_t db = (uint64_t)(base + s * (G::STAGE >> 4) + (G::A_BYTES >> 4)) | HI;
    #pragma unroll
                        for (int k = 0; k < 4; ++k) {  // 32 of K: 32 bytes along the swizzled rows
                            if constexpr (G::PAIR)
                                mma_e4m3_pair(tmem + a * BN, da + 2 * k, db + 2 * k, ID, k > 0);
                            else
                                mma_e4m3(tmem + a * BN, da + 2 * k, db + 2 * k, ID, k > 0);
                        }
                        if constexpr (G::PAIR) {
                            commit_pair(&sm.empty[s]);
                            commit_pair(&sm.acc_full[a]);
                        } else {
                            commit(&sm.empty[s]);
                            commit(&sm.acc_full[a]);
                        }
                    }
                // every product issued is complete before tensor memory is freed
                for (uint32_t i = n > 2 ? n - 2 : 0; i < n; ++i) {
                    const unsigned long long w0 = gtimer();
                    while (!mbar_try(&sm.acc_full[i & 1], (i >> 1) & 1) && gtimer() - w0 < WAIT_NS) {
                    }
                }
            }
        } else if (warp == G::EPI + 2) {
            // ------------------------------------------------------------------ scales
            // of a K block: x's rows of the tile, then w's blocks
            constexpr int ROWS = FEW ? BN : 128;
            wait_for_x();
            uint32_t n = 0;
            bool ok = true;
            for (int t = first; ok && t < all; t += step) {
                int ia, ib;
                tile_at(t, ia, ib);
                const int m0 = FEW ? ib * BN : ia * G::ROWS + half * 128, n0 = FEW ? ia : ib * (BN / 128);
                for (int j = j0; j < j1; ++j, ++n) {
                    const int s = n % SLOTS;
                    if (!(ok = mbar_wait(&sm.sc_empty[s], ((n / SLOTS) & 1) ^ 1, ctl, 135))) break;
    #pragma unroll
                    for (int i = 0; i < (ROWS + 31) / 32; ++i) {
                        const int r = i * 32 + lane;
                        if (r < ROWS) copy4(&scales[s][r], p.x.scale + (int64_t)min(m0 + r, p.M - 1) * p.x.si + j * p.x.sj);
                    }
                    if (lane < (FEW ? 1 : BN / 128))
                        copy4(&scales[s][G::SLOT - 4 + lane],
                              p.w.scale + (int64_t)min(n0 + lane, (p.N - 1) / 128) * p.w.si + j * p.w.sj);
                    copies_arrive(&sm.sc_full[s]);
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    } else {
        if (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ------------------------------------------------------------------ sums, output
        const int row = (warp & 3) * 32 + lane, col0 = (warp >> 2) * G::COLS;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16) + col0;
        uint32_t n = 0;
        bool ok = true;
        for (int t = first; ok && t < all; t += step) {
            int ia, ib;
            tile_at(t, ia, ib);
            const int ra = ia * G::ROWS + half * 128 + row, cb = ib * BN + col0;  // this thread's row and first column
            unsigned long long acc[G::COLS / 2];
#pragma unroll
            for (int i = 0; i < G::COLS / 2; ++i) acc[i] = 0ull;
            // CH columns are read while the CH before them are scaled, across K blocks too: a read's
            // latency, not its bandwidth, is what it costs
            constexpr int CH = G::COLS == 128 ? 32 : 16, NC = G::COLS / CH;
            uint32_t d[2][CH];
            auto open = [&](uint32_t(&to)[CH]) {  // the next K block's products, its first columns on their way
                ok = mbar_wait(&sm.acc_full[n & 1], (n >> 1) & 1, ctl, 134);
                tc_fence_after();
                if (ok) tmem_issue(mine + (n & 1) * BN, to);
            };
            if (!FEW && j0 < j1) open(d[0]);
            for (int j = j0; ok && j < j1; ++j) {
                const int a = n & 1, sl = n % SLOTS;
                if (!(ok = mbar_wait(&sm.sc_full[sl], (n / SLOTS) & 1, ctl, 136))) break;
                const float *sx = scales[sl];
                const float s = FEW ? sx[G::SLOT - 4] : sx[row] * sx[G::SLOT - 4 + col0 / 128];
                const unsigned long long sp = pair(s);
                if (FEW) {  // not ahead: registers for two CTAs an SM matter more
                    open(d[0]);
                    if (!ok) break;
                }
                ++n;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    uint32_t(&v)[CH] = d[NC % 2 ? 0 : c & 1];
                    tmem_wait_ld_regs(v);
                    if (c + 1 < NC) {
                        tmem_issue(mine + a * BN + (c + 1) * CH, d[(c + 1) & 1]);
                    } else {  // all columns are in registers
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if constexpr (G::PAIR)
                                arrive_in_first(&sm.acc_empty[a]);
                            else
                                mbar_arrive(&sm.acc_empty[a]);
                        }
                        if (!FEW && j + 1 < j1) open(d[0]);
                    }
#pragma unroll
                    for (int i = 0; i < CH; i += 2) {
                        unsigned long long x2 = sp;
                        if (FEW) {
                            x2 = *reinterpret_cast<const unsigned long long *>(sx + c * CH + i);
                            asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x2) : "l"(sp));
                        }
                        fma2(acc[(c * CH + i) / 2], v[i], v[i + 1], x2);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.sc_empty[sl]);
            }
            if (!ok) break;
            if (!G::PAIR && splits > 1) {
                float *part = reinterpret_cast<float *>(tiles);
#pragma unroll
                for (int i = 0; i < G::COLS; ++i) part[i * 128 + row] = half_of(acc[i / 2], i & 1);
            } else if (FEW) {
                if (ra < p.N) {
#pragma unroll
                    for (int i = 0; i < G::COLS; ++i)
                        if (cb + i < p.M) {
                            const float v = half_of(acc[i / 2], i & 1);
                            const int64_t at = (int64_t)(cb + i) * p.ys + ra;
                            if (p.y_f32)
                                static_cast<float *>(p.y)[at] = v;
                            else
                                static_cast<__nv_bfloat16 *>(p.y)[at] = __float2bfloat16_rn(v);
                        }
                }
            } else if (!FEW) {
                // rows leave through shared memory, 64 bytes of each at a time, so that a store covers
                // whole sectors whatever y's row stride is
                uint8_t *mine_s = out_s[warp];
                const int rows = min(32, p.M - (ra - lane));
                if (p.y_f32) {
#pragma unroll
                    for (int c = 0; c < G::COLS; c += 16) {
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const unsigned long long lo = acc[(c + i) / 2], hi = acc[(c + i) / 2 + 1];
                            *reinterpret_cast<ulonglong2 *>(mine_s + lane * OUT_PITCH + i * 4) = make_ulonglong2(lo, hi);
                        }
                        __syncwarp();
                        store_rows<float>(mine_s, static_cast<float *>(p.y) + (int64_t)(ra - lane) * p.ys + cb + c, p.ys, rows,
                                          min(16, p.N - cb - c), lane);
                        __syncwarp();
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < G::COLS; c += 32) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint4 v;
                            uint32_t *e = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
                            for (int h = 0; h < 4; ++h)
                                e[h] = pack2(half_of(acc[(c + i) / 2 + h], 0), half_of(acc[(c + i) / 2 + h], 1));
                            *reinterpret_cast<uint4 *>(mine_s + lane * OUT_PITCH + i * 2) = v;
                        }
                        __syncwarp();
                        store_rows<__nv_bfloat16>(mine_s, static_cast<__nv_bfloat16 *>(p.y) + (int64_t)(ra - lane) * p.ys + cb + c,
                                                  p.ys, rows, min(32, p.N - cb - c), lane);
                        __syncwarp();
                    }
                }
            }
        }
    }
    if (!G::PAIR && splits > 1) {
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();  // every CTA's partial sums are in its shared memory
        if (!skip && !ctl.aborted() && tid < 128) {
            int ia, ib;
            tile_at(first, ia, ib);
            const int r = ia * 128 + tid;  // of the 128-row operand
            // this CTA's columns: neighbouring ones where a thread's row is a row of y
            const int each = BN / splits, c0 = FEW ? split : split * each, dc = FEW ? splits : 1;
            const int rows = FEW ? p.N : p.M, cols = FEW ? p.M : p.N;
            for (int n = 0; n < each; ++n) {
                const int i = c0 + n * dc, c = ib * BN + i;
                if (c >= cols || r >= rows) break;
                float v = 0.f;
                for (int q = 0; q < splits; ++q)
                    v += cl.map_shared_rank(reinterpret_cast<float *>(tiles), q)[i * 128 + tid];
                const int64_t at = FEW ? (int64_t)c * p.ys + r : (int64_t)r * p.ys + c;
                if (p.y_f32)
                    static_cast<float *>(p.y)[at] = v;
                else
                    static_cast<__nv_bfloat16 *>(p.y)[at] = __float2bfloat16_rn(v);
            }
        }
        cl.sync();
    }
    tc_fence_before();
    if constexpr (G::PAIR)
        cg::this_cluster().sync();  // nothing of the other CTA reaches this one's memory any more
    else
        __syncthreads();
    tc_fence_after();
    if (warp == 0) {
        if constexpr (G::PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::TCOLS) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::TCOLS) : "memory");
    }
    if (tid == 0) report_fault(sm.ctl.abort_flag, p.fault);
}

template <int BN, bool FEW> cudaError_t matmul_t(Fp8Params &p, int sms, bool after_quantize, cudaStream_t st) {
    using G = Cfg<BN, FEW>;
    const Fp8Rows &a = FEW ? p.w : p.x, &b = FEW ? p.x : p.w;
    const int ra = FEW ? p.N : p.M, rb = FEW ? p.M : p.N;
    CUtensorMap ta, tb;
    if (!make_map_2d_u8(&ta, a.q, ra, p.K, a.stride, 128) || !make_map_2d_u8(&tb, b.q, rb, p.K, b.stride, G::PAIR ? BN / 2 : BN))
        return cudaErrorInvalidValue;
    p.tiles_a = (ra + G::ROWS - 1) / G::ROWS;
    p.tiles_b = (rb + BN - 1) / BN;
    const int64_t tiles = (int64_t)p.tiles_a * p.tiles_b;
    if (tiles > 0x3fffffff) return cudaErrorInvalidValue;
    cudaError_t e = set_smem_once<fp8_matmul_kernel<BN, FEW>>(G::SMEM);
    if (e != cudaSuccess) return e;
    int splits = 1;
    // K over a cluster while SMs would idle and a CTA keeps two K blocks: 256 x 128 x 4928 25.0 -> 16.1 us with the
    // quantisation. Joining the shares costs a short K more than that saves: 1024^3 takes 28.8, on pairs of
    // CTAs without a split 10.4.
    if (!G::PAIR)
        while (splits < 8 && tiles * splits * 2 <= sms && p.blocks >= splits * 4) splits *= 2;
    cudaLaunchConfig_t cfg{};
    const int64_t pairs = tiles < sms / 2 ? tiles : sms / 2;
    cfg.gridDim = dim3((unsigned)(FEW || splits > 1 ? tiles * splits : G::PAIR ? 2 * pairs : (tiles < sms ? tiles : sms)));
    cfg.blockDim = dim3(G::THREADS);
    cfg.dynamicSmemBytes = G::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = G::PAIR ? 2 : (unsigned)splits;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = after_quantize ? 2 : 1;  // only after our own kernel, which says when it may start
    e = cudaLaunchKernelEx(&cfg, fp8_matmul_kernel<BN, FEW>, ta, tb, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

cudaError_t launch_fp8_quantize(const void *x, int64_t xs, int dtype, int M, int K, uint8_t *q, int64_t qs,
                                float *scale, int64_t si, int64_t sj, int sms, cudaStream_t st) {
    const int blocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
    // two blocks a lane group once that still fills the GPU
    const int groups = (int64_t)M * blocks >= (int64_t)sms * 128 * 4 && blocks > 1 ? 2 : 1;
    const uint32_t per_row = (uint32_t)((blocks + groups - 1) / groups);
    const int64_t items = (int64_t)M * per_row;
    if (items > 0xfffffff0ll) return cudaErrorInvalidValue;
    const unsigned grid = (unsigned)((items + 31) / 32);
    const int step = dtype == PMA_F32 ? 4 : 8;  // 16-byte rows for the vector loads (load4 of bf16 is 8 bytes)
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && xs % step == 0;
    auto run = [&](auto *p) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
        if (groups == 2)
            quantize_rows<T, 2><<<grid, 256, 0, st>>>(p, xs, (uint32_t)items, K, per_row, vec, q, qs, scale, si, sj);
        else
            quantize_rows<T, 1><<<grid, 256, 0, st>>>(p, xs, (uint32_t)items, K, per_row, vec, q, qs, scale, si, sj);
    };
    if (dtype == PMA_F32)
        run(static_cast<const float *>(x));
    else
        run(static_cast<const __nv_bfloat16 *>(x));
    return cudaGetLastError();
}

cudaError_t launch_fp8_quantize_weight(const void *w, int64_t ws, int dtype, int N, int K, uint8_t *q, int64_t qs,
                                       float *scale, cudaStream_t st) {
    const int blocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
    const int64_t grid = (int64_t)((N + FP8_BLOCK - 1) / FP8_BLOCK) * blocks;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    const int step = dtype == PMA_F32 ? 4 : 8;
    const bool vec = reinterpret_cast<uintptr_t>(w) % 16 == 0 && ws % step == 0;
    if (dtype == PMA_F32)
        quantize_blocks<float><<<(unsigned)grid, 256, 0, st>>>(static_cast<const float *>(w), ws, N, K, blocks, vec, q,
                                                              qs, scale);
    else
        quantize_blocks<__nv_bfloat16><<<(unsigned)grid, 256, 0, st>>>(static_cast<const __nv_bfloat16 *>(w), ws, N, K,
                                                                       blocks, vec, q, qs, scale);
    return cudaGetLastError();
}

cudaError_t launch_fp8_matmul(Fp8Params p, int sms, bool after_quantize, cudaStream_t st) {
    p.blocks = (p.K + FP8_BLOCK - 1) / FP8_BLOCK;
    if (p.M <= 16) return matmul_t<16, true>(p, sms, after_quantize, st);
    if (p.M <= 32) return matmul_t<32, true>(p, sms, after_quantize, st);
    if (p.M <= 64) return matmul_t<64, true>(p, sms, after_quantize, st);
    // 256 x 256 on pairs of CTAs where its rounds of tiles take less: a round takes some 1.45 times as long
    // as one of 128 x 128 tiles, of half the work an SM (8192^3: 14 in 511 us, 28 in 706; 4096 x 2304 x 768: 2 in
    // 15.9, 4 in 20.4; 2048 x 3000 x 1024: 2 in 18.4, 3 in 18.7; 777 x 1530 x 1000: 1 in 12.0, 1 in 10.4)
    const int64_t pairs = (int64_t)((p.M + 255) / 256) * ((p.N + 255) / 256);
    const int64_t singles = (int64_t)((p.M + 127) / 128) * ((p.N + 127) / 128);
    const int64_t slots = sms / 2;
    if (20 * ((singles + sms - 1) / sms) >= 29 * ((pairs + slots - 1) / slots))
        return matmul_t<256, false>(p, sms, after_quantize, st);
    return matmul_t<128, false>(p, sms, after_quantize, st);
}

}  // namespace pma
