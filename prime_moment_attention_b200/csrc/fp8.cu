// fp8.cu -- e4m3 quantisation with a float32 scale per block of 128, and the product
//
//   y[m, n] = sum_j xs[m, j] ws[n / 128, j]  sum_{k in block j} xq[m, k] wq[n, k]
//
// on the tensor cores.  The scales differ from K block to K block, so the inner sums cannot stay in
// one accumulator: each 128-wide block is one short product (four tcgen05.mma of K = 32) into one of
// two tensor-memory accumulators, and the epilogue warps read it back, scale it and add it in
// float32 registers while the tensor core fills the other.  One warp moves tiles by TMA (128-byte
// swizzle; the tensor map's extents fill ragged edges with zeros, which are zeros in e4m3), one
// issues the products.
//
// The operand with 128 rows a tile (the tensor core's M) is x for many tokens and w for few: then a
// tile is 128 weight rows by all the tokens (16 to 128), the weights stream once, and K is split over
// a cluster of up to 8 CTAs whose partial sums meet in shared memory in a fixed order.
#include <cooperative_groups.h>

#include "fp8.cuh"

#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace pma {

namespace {

using namespace tc;

// -------------------------------------------------------------------------------- quantisation
// e4m3 of x * 448 / amax, rounded once from the correctly rounded quotient: an x that lies half-way
// between two e4m3 values on the block's scale is exactly half-way after the division too.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
struct Quant {
    float amax, pre;
    // amax of 0 (or below 2^-100) counts as 2^-100; a block of huge values is divided by 2^20 first,
    // so that 448 x stays finite
    __device__ __forceinline__ explicit Quant(float a) : amax(fmaxf(a, 7.888609052210118e-31f)), pre(448.0f) {
        if (amax > 1e35f) {
            pre *= 9.5367431640625e-07f;
            amax *= 9.5367431640625e-07f;
        }
    }
    __device__ __forceinline__ float operator()(float x) const { return __fdiv_rn(x * pre, amax); }
    static __device__ __forceinline__ float scale(float a) { return fmaxf(a, 7.888609052210118e-31f) / 448.0f; }
};

// NaN is kept: a block that holds one gets a NaN scale
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Eight consecutive elements of a row, zero past K.
template <typename T>
__device__ __forceinline__ void load8(const T *row, int k, int K, bool vec, float (&x)[8]) {
    if (vec && k + 8 <= K) {
        const float4 a = load4(row + k), b = load4(row + k + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = k + i < K ? Elem<T>::to_f(row[k + i]) : 0.f;
    }
}
__device__ __forceinline__ void store8(uint8_t *row, int k, int K, uint2 v) {
    if (k + 8 <= K) {
        *reinterpret_cast<uint2 *>(row + k) = v;  // rows start on 16 bytes, k is a multiple of 8
    } else {
        for (int i = 0; i < 8 && k + i < K; ++i) row[k + i] = (uint8_t)((i < 4 ? v.x : v.y) >> (8 * (i & 3)));
    }
}
__device__ __forceinline__ float amax8(const float (&x)[8]) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max_nan(a, fabsf(x[i]));
    return a;
}
__device__ __forceinline__ uint2 quant8(const float (&x)[8], const Quant &q) {
    return make_uint2(e4m3x2(q(x[0]), q(x[1])) | e4m3x2(q(x[2]), q(x[3])) << 16,
                      e4m3x2(q(x[4]), q(x[5])) | e4m3x2(q(x[6]), q(x[7])) << 16);
}

// 16 lanes a block of 128; the grid covers rows x blocks.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows(const T *__restrict__ x, int64_t xs, int M, int K, int blocks,
                                                    bool vec, uint8_t *__restrict__ q, int64_t qs,
                                                    float *__restrict__ scale, int64_t si, int64_t sj) {
    const int64_t g = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 4;
    const int l = threadIdx.x & 15;
    const bool on = g < (int64_t)M * blocks;
    const int m = on ? (int)(g / blocks) : 0, j = on ? (int)(g - (int64_t)m * blocks) : 0;
    const int k = on ? j * FP8_BLOCK + l * 8 : K;
    float v[8];
    load8(x + (int64_t)m * xs, k, K, vec, v);
    float a = amax8(v);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
    if (!on) return;
    store8(q + (int64_t)m * qs, k, K, quant8(v, Quant(a)));
    if (l == 0) scale[m * si + j * sj] = a == a ? Quant::scale(a) : a;
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
        float v[8];
        load8(w + (int64_t)n * ws, k, K, vec, v);
        a = max_nan(a, amax8(v));
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
        float v[8];
        load8(w + (int64_t)n * ws, k, K, vec, v);  // from L1 or L2: the block was just read
        store8(q + (int64_t)n * qs, k, K, quant8(v, qu));
    }
    if (threadIdx.x == 0) scale[(int64_t)nb * blocks + j] = a == a ? Quant::scale(a) : a;
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
__device__ __forceinline__ void tma_load2(void *dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            su32(dst)),
        "l"(map), "r"(su32(bar)), "r"(c0), "r"(c1)
        : "memory");
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

// BN: rows of the second operand in a tile; FEW: w is the 128-row operand.
template <int BN, bool FEW> struct Cfg {
    static constexpr int EPI = BN == 256 ? 8 : 4;      // epilogue warps: 128 lanes x COLS columns each group of 4
    static constexpr int COLS = BN == 256 ? 128 : BN;  // accumulator columns of a thread
    static constexpr int WARPS = BN == 256 ? 12 : 6;
    static constexpr int THREADS = WARPS * 32;
    static constexpr int A_BYTES = 128 * 128, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 4;
    static constexpr int TCOLS = 2 * BN < 32 ? 32 : 2 * BN;
    // K split: partial sums [BN][128] float32 take the place of the tiles
    static constexpr int SMEM = STAGES * STAGE + 1024;
};

template <int STAGES> struct Bars {
    uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], never;
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
            mbar_init(&sm.acc_empty[i], G::EPI);
        }
        mbar_init(&sm.never, 1);
        init_ctl(sm.ctl, p.fault);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&sm.tmem)),
                     "r"(G::TCOLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    bool skip = false;
    if (p.test_wait_ns) {  // test hook: a wait expires before any copy or product is issued
        if (tid == 0) expire_test_wait(&sm.never, ctl, p.test_wait_ns, 130);
        __syncthreads();
        skip = ctl.aborted();
    }

    // Tiles of this CTA (FEW: one, with a share of the K blocks; else every gridDim.x-th).
    int split = 0, splits = 1, first = blockIdx.x, step = gridDim.x;
    if (FEW) {
        const cg::cluster_group cl = cg::this_cluster();
        split = (int)cl.block_rank();
        splits = (int)cl.num_blocks();
        first = blockIdx.x / splits;
        step = p.tiles_a * p.tiles_b;
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

    if (warp == G::EPI) {
        // ------------------------------------------------------------------ TMA
        if (lane == 0) {
            uint32_t n = 0;
            bool ok = true;
            for (int t = first; ok && t < all; t += step) {
                int ia, ib;
                tile_at(t, ia, ib);
                for (int j = j0; j < j1; ++j, ++n) {
                    const int s = n % G::STAGES;
                    if (!(ok = mbar_wait(&sm.empty[s], ((n / G::STAGES) & 1) ^ 1, ctl, 131))) break;
                    mbar_expect_tx(&sm.full[s], G::STAGE);
                    tma_load2(tiles + s * G::STAGE, &ta, &sm.full[s], j * 128, ia * 128);
                    tma_load2(tiles + s * G::STAGE + G::A_BYTES, &tb, &sm.full[s], j * 128, ib * BN);
                }
            }
            // never leave with copies in flight
            for (uint32_t i = n > G::STAGES ? n - G::STAGES : 0; i < n; ++i) {
                const unsigned long long w0 = gtimer();
                while (!mbar_try(&sm.full[i % G::STAGES], (i / G::STAGES) & 1) && gtimer() - w0 < WAIT_NS) {
                }
            }
        }
    } else if (warp == G::EPI + 1) {
        // ------------------------------------------------------------------ products
        if (lane == 0) {
            constexpr uint32_t ID = idesc_e4m3(128, BN);
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
                    for (int k = 0; k < 4; ++k)  // 32 of K: 32 bytes along the swizzled rows
                        mma_e4m3(tmem + a * BN, da + 2 * k, db + 2 * k, ID, k > 0);
                    commit(&sm.empty[s]);
                    commit(&sm.acc_full[a]);
                }
            // every product issued is complete before tensor memory is freed
            for (uint32_t i = n > 2 ? n - 2 : 0; i < n; ++i) {
                const unsigned long long w0 = gtimer();
                while (!mbar_try(&sm.acc_full[i & 1], (i >> 1) & 1) && gtimer() - w0 < WAIT_NS) {
                }
            }
        }
    } else if (warp < G::EPI) {
        // ------------------------------------------------------------------ scales, sums, output
        const int row = (warp & 3) * 32 + lane, col0 = (warp >> 2) * G::COLS;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16) + col0;
        uint32_t n = 0;
        bool ok = true;
        for (int t = first; ok && t < all; t += step) {
            int ia, ib;
            tile_at(t, ia, ib);
            const int ra = ia * 128 + row, cb = ib * BN + col0;  // this thread's row and first column
            // its scales: of the row (x) or of the tile (w), and of the columns
            const float *sa = FEW ? p.w.scale + (int64_t)ia * p.w.si
                                  : p.x.scale + (int64_t)min(ra, p.M - 1) * p.x.si;
            const int64_t saj = FEW ? p.w.sj : p.x.sj;
            const float *sb = FEW ? p.x.scale : p.w.scale + (int64_t)min(cb / 128, (p.N - 1) / 128) * p.w.si;
            const int64_t sbj = FEW ? p.x.sj : p.w.sj;
            unsigned long long acc[G::COLS / 2];
#pragma unroll
            for (int i = 0; i < G::COLS / 2; ++i) acc[i] = 0ull;
            float s0 = j0 < j1 ? __ldg(sa + j0 * saj) * (FEW ? 1.f : __ldg(sb + j0 * sbj)) : 0.f;
            for (int j = j0; j < j1; ++j, ++n) {
                const int a = n & 1;
                const float s = s0;
                if (j + 1 < j1) s0 = __ldg(sa + (j + 1) * saj) * (FEW ? 1.f : __ldg(sb + (j + 1) * sbj));
                if (!(ok = mbar_wait(&sm.acc_full[a], (n >> 1) & 1, ctl, 134))) break;
                tc_fence_after();
                constexpr int CH = G::COLS < 32 ? 16 : 32;
#pragma unroll
                for (int c = 0; c < G::COLS; c += CH) {
                    uint32_t d[CH];
                    if constexpr (CH == 32)
                        tmem_ld32_issue(mine + a * BN + c, d);
                    else
                        tmem_ld16_issue(mine + a * BN + c, d);
                    tmem_wait_ld_regs(d);
                    if (c + CH == G::COLS) {  // all columns are in registers
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sm.acc_empty[a]);
                    }
                    if (FEW) {
#pragma unroll
                        for (int i = 0; i < CH; i += 2) {
                            const int m0 = cb + c + i, m1 = m0 + 1;
                            const float x0 = __ldg(sb + (int64_t)min(m0, p.M - 1) * p.x.si + j * sbj);
                            const float x1 = __ldg(sb + (int64_t)min(m1, p.M - 1) * p.x.si + j * sbj);
                            unsigned long long sc;
                            asm("mov.b64 %0, {%1, %2};" : "=l"(sc) : "f"(s * x0), "f"(s * x1));
                            fma2(acc[(c + i) / 2], d[i], d[i + 1], sc);
                        }
                    } else {
                        const unsigned long long sc = pair(s);
#pragma unroll
                        for (int i = 0; i < CH; i += 2) fma2(acc[(c + i) / 2], d[i], d[i + 1], sc);
                    }
                }
            }
            if (!ok) break;
            if (FEW && splits > 1) {
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
            } else if (ra < p.M) {
                if (p.y_f32) {
                    float *o = static_cast<float *>(p.y) + (int64_t)ra * p.ys + cb;
                    if (cb + G::COLS <= p.N && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
                        for (int i = 0; i < G::COLS; i += 4)
                            *reinterpret_cast<float4 *>(o + i) =
                                make_float4(half_of(acc[i / 2], 0), half_of(acc[i / 2], 1), half_of(acc[i / 2 + 1], 0),
                                            half_of(acc[i / 2 + 1], 1));
                    } else {
#pragma unroll
                        for (int i = 0; i < G::COLS; ++i)
                            if (cb + i < p.N) o[i] = half_of(acc[i / 2], i & 1);
                    }
                } else {
                    __nv_bfloat16 *o = static_cast<__nv_bfloat16 *>(p.y) + (int64_t)ra * p.ys + cb;
                    if (cb + G::COLS <= p.N && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
                        for (int i = 0; i < G::COLS; i += 8) {
                            uint4 v;
                            uint32_t *e = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
                            for (int h = 0; h < 4; ++h)
                                e[h] = pack2(half_of(acc[i / 2 + h], 0), half_of(acc[i / 2 + h], 1));
                            *reinterpret_cast<uint4 *>(o + i) = v;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < G::COLS; ++i)
                            if (cb + i < p.N) o[i] = __float2bfloat16_rn(half_of(acc[i / 2], i & 1));
                    }
                }
            }
        }
    }
    if (FEW && splits > 1) {
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();  // every CTA's partial sums are in its shared memory
        if (!skip && !ctl.aborted() && tid < 128) {
            int ia, ib;
            tile_at(first, ia, ib);
            const int nrow = ia * 128 + tid;
            for (int i = split; i < BN; i += splits) {
                const int m = ib * BN + i;
                if (m >= p.M || nrow >= p.N) break;
                float v = 0.f;
                for (int r = 0; r < splits; ++r)
                    v += cl.map_shared_rank(reinterpret_cast<float *>(tiles), r)[i * 128 + tid];
                const int64_t at = (int64_t)m * p.ys + nrow;
                if (p.y_f32)
                    static_cast<float *>(p.y)[at] = v;
                else
                    static_cast<__nv_bfloat16 *>(p.y)[at] = __float2bfloat16_rn(v);
            }
        }
        cl.sync();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::TCOLS) : "memory");
    if (tid == 0) report_fault(sm.ctl.abort_flag, p.fault);
}

template <int BN, bool FEW> cudaError_t matmul_t(Fp8Params &p, int sms, cudaStream_t st) {
    using G = Cfg<BN, FEW>;
    const Fp8Rows &a = FEW ? p.w : p.x, &b = FEW ? p.x : p.w;
    const int ra = FEW ? p.N : p.M, rb = FEW ? p.M : p.N;
    CUtensorMap ta, tb;
    if (!make_map_2d_u8(&ta, a.q, ra, p.K, a.stride, 128) || !make_map_2d_u8(&tb, b.q, rb, p.K, b.stride, BN))
        return cudaErrorInvalidValue;
    p.tiles_a = (ra + 127) / 128;
    p.tiles_b = (rb + BN - 1) / BN;
    const int64_t tiles = (int64_t)p.tiles_a * p.tiles_b;
    if (tiles > 0x3fffffff) return cudaErrorInvalidValue;
    cudaError_t e = set_smem_once<fp8_matmul_kernel<BN, FEW>>(G::SMEM);
    if (e != cudaSuccess) return e;
    int splits = 1;
    if (FEW)  // K over a cluster while SMs would idle and a CTA keeps two K blocks
        while (splits < 8 && tiles * splits * 2 <= sms && p.blocks >= splits * 4) splits *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(FEW ? tiles * splits : (tiles < sms ? tiles : sms)));
    cfg.blockDim = dim3(G::THREADS);
    cfg.dynamicSmemBytes = G::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)splits;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, fp8_matmul_kernel<BN, FEW>, ta, tb, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

cudaError_t launch_fp8_quantize(const void *x, int64_t xs, int dtype, int M, int K, uint8_t *q, int64_t qs,
                                float *scale, int64_t si, int64_t sj, cudaStream_t st) {
    const int blocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
    const int64_t grid = ((int64_t)M * blocks * 16 + 255) / 256;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    const int step = dtype == PMA_F32 ? 4 : 8;  // 16-byte rows for the vector loads (load4 of bf16 is 8 bytes)
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && xs % step == 0;
    if (dtype == PMA_F32)
        quantize_rows<float><<<(unsigned)grid, 256, 0, st>>>(static_cast<const float *>(x), xs, M, K, blocks, vec, q, qs,
                                                            scale, si, sj);
    else
        quantize_rows<__nv_bfloat16><<<(unsigned)grid, 256, 0, st>>>(static_cast<const __nv_bfloat16 *>(x), xs, M, K,
                                                                     blocks, vec, q, qs, scale, si, sj);
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

cudaError_t launch_fp8_matmul(Fp8Params p, int sms, cudaStream_t st) {
    p.blocks = (p.K + FP8_BLOCK - 1) / FP8_BLOCK;
    if (p.M <= 16) return matmul_t<16, true>(p, sms, st);
    if (p.M <= 32) return matmul_t<32, true>(p, sms, st);
    if (p.M <= 64) return matmul_t<64, true>(p, sms, st);
    // 256 columns halve the re-reads of x, once that leaves a tile for every SM
    const int64_t wide = (int64_t)((p.M + 127) / 128) * ((p.N + 255) / 256);
    if (wide >= sms) return matmul_t<256, false>(p, sms, st);
    return matmul_t<128, false>(p, sms, st);
}

}  // namespace pma
