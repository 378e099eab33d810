// recurrence.cu -- a gated linear recurrence per channel, its gradient and its one-token step.
//
//   u_t = f_t + bias          a_t = sigmoid(u_t)        z_t = 1 - a_t = sigmoid(-u_t)
//   h_t = a_t h_{t-1} + z_t x_t
//   y_t = h_t                       or, with a gate,      y_t = h_t silu(gate_t)
//
// A nonzero reset_t replaces h_{t-1} by zero (a document starts at t).
//
// The time axis is split: a tile is 128 tokens of 32 (or 64) channels, its warps hold consecutive
// rows and its lanes the channels.  A run of tokens is an affine map of the state that enters it,
//   h -> h + (H - Q h),   Q = 1 - prod a_t,   H = its result from a zero state,
// kept as Q rather than as the product: for slow decays 1 - prod a_t is what matters and the
// product itself would round it away.  A token joins a run by Q <- Q + z (1 - Q), H <- a H + z x.
// Every input is read once: a tile holds its rows in registers, publishes its (Q, H) as one 64-bit
// word per channel, gathers the words of the tiles before it back to one that has published the
// state leaving it, and then writes its outputs.  Words start as all ones (a NaN that no result
// carries) and are written once, so a word is its own flag and no fence is needed.  A state is
// always the same chain of joins, tile after tile, however far back a tile looked: results do not
// depend on timing.  Tiles are handed out in the order of a counter, so a tile only waits for
// tiles that are already running; every wait is bounded.
//
// Backward, from the right, with the carry c_t = a_t g_t:
//   g_t = dy_t silu(gate_t) + c_{t+1},   dx = z g,   df = g (h_{t-1} - x) a z,
//   dgate = dy h silu'(gate),            dbias = sum df,            dh0 = c_0.
// A tile recomputes its states from the one that entered it, which the forward pass kept (one
// float32 state per channel and 128 tokens).  dbias is summed within a tile, then over the tiles
// in a fixed order by a second kernel.
#include "recurrence.cuh"

#include "tc_common.cuh"

namespace pma {
namespace {

constexpr uint32_t EMPTY = 0xffffffffu;
constexpr int FAULT_CODE = 120;

// 2^x and 1/x to about 2 ulp, subnormals flushed
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
constexpr float LOG2E = 1.4426950408889634f;

// exp(min(u, 87)), NaN kept: finite, so that exp(u) sigmoid(-u) is a sigmoid and not inf * 0
__device__ __forceinline__ float exp_sat(float u) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(u * LOG2E), "f"(126.0f));
    return ex2(r);
}
__device__ __forceinline__ float sigmoid_neg(float u) { return rcp(1.0f + exp_sat(u)); }
__device__ __forceinline__ float sigmoid(float u) { return rcp(1.0f + ex2(-u * LOG2E)); }

// One token.  This form is exact at both ends (z = 0 keeps h, z = 1 takes x); rounding 1 - z costs a
// slow decay half an ulp a row, over the few rows between two joins.
__device__ __forceinline__ float advance(float h, float z, float x) { return fmaf(1.f - z, h, z * x); }

// the state h after a run (Q, H); Q = 1 cuts it off, whatever it was
__device__ __forceinline__ float join(float h, float q, float hh) {
    return q == 1.0f ? hh : h + fmaf(-q, h, hh);
}

// V consecutive channels of one row as one load or store
template <typename T, int V> struct Pack;
template <> struct Pack<float, 1> {
    float r;
    static constexpr int bytes = 4;
    __device__ __forceinline__ void zero() { r = 0.f; }
    __device__ __forceinline__ void load(const float *p, int) { r = __ldg(p); }
    __device__ __forceinline__ float at(int) const { return r; }
    static __device__ __forceinline__ void store(float *p, const float (&v)[1], int) { *p = v[0]; }
};
template <> struct Pack<__nv_bfloat16, 1> {
    uint16_t r;
    __device__ __forceinline__ void zero() { r = 0; }
    __device__ __forceinline__ void load(const __nv_bfloat16 *p, int) {
        r = __ldg(reinterpret_cast<const unsigned short *>(p));
    }
    __device__ __forceinline__ float at(int) const { return __uint_as_float((uint32_t)r << 16); }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float (&v)[1], int) {
        *p = __float2bfloat16_rn(v[0]);
    }
};
template <> struct Pack<__nv_bfloat16, 2> {
    uint32_t r;
    __device__ __forceinline__ void zero() { r = 0; }
    __device__ __forceinline__ void load(const __nv_bfloat16 *p, int) {
        r = __ldg(reinterpret_cast<const unsigned int *>(p));
    }
    __device__ __forceinline__ float at(int i) const {
        return __uint_as_float(i ? r & 0xffff0000u : r << 16);
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float (&v)[2], int) {
        *reinterpret_cast<uint32_t *>(p) = tc::pack2(v[0], v[1]);
    }
};

__device__ __forceinline__ uint32_t word_of(float v) {
    const uint32_t u = __float_as_uint(v);
    return u == EMPTY ? 0x7fffffffu : u;
}
__device__ __forceinline__ void put32(uint32_t *p, float v) {
    asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(word_of(v)) : "memory");
}
__device__ __forceinline__ void put64(unsigned long long *p, float q, float h) {
    const unsigned long long v = ((unsigned long long)word_of(h) << 32) | word_of(q);
    asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t get32(const uint32_t *p) {
    uint32_t v;
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ unsigned long long get64(const unsigned long long *p) {
    unsigned long long v;
    asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
    return v;
}

// The run (Q, H) of a tile before this one, or the state leaving it as the run (1, state).
// `must_end`: wait for the state.
__device__ __forceinline__ float2 fetch(const ScanParams &p, int64_t at, bool must_end) {
    unsigned long long t0 = 0;
    for (uint32_t it = 1;; ++it) {
        const uint32_t s = get32(p.incl + at);
        if (s != EMPTY) return make_float2(1.0f, __uint_as_float(s));
        if (!must_end) {
            const unsigned long long a = get64(p.agg + at);
            if (a != ~0ull) return make_float2(__uint_as_float((uint32_t)a), __uint_as_float((uint32_t)(a >> 32)));
        }
        if ((it & 255) == 0) {
            const unsigned long long now = tc::gtimer();
            if (!t0) t0 = now;
            const bool gone = *reinterpret_cast<volatile int *>(p.counter + 1) != -1;
            if (gone || now - t0 > p.wait_ns) {
                *reinterpret_cast<volatile int *>(p.counter + 1) = FAULT_CODE;
                tc::report_fault(FAULT_CODE, p.fault);
                return make_float2(1.0f, __uint_as_float(0x7fffffffu));
            }
        }
    }
}

// Test hook: a wait that nothing ends runs out, and the launch gives up before any other work.
__device__ __forceinline__ bool test_expired(const ScanParams &p) {
    if (!p.test_wait_ns) return false;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        const unsigned long long t0 = tc::gtimer();
        while (tc::gtimer() - t0 <= p.test_wait_ns) {
        }
        tc::report_fault(FAULT_CODE, p.fault);
    }
    return true;
}

struct Tile {
    int chunk, b, c;      // chunk in walking order; c: this lane's first channel
    int64_t word0;        // index of (b, chunk 0, c) in the word arrays
};

template <int V>
__device__ __forceinline__ Tile tile_of(const ScanParams &p, int t, int lane) {
    const int cols = p.B * p.ctiles;
    Tile k;
    k.chunk = t / cols;
    const int col = t - k.chunk * cols;
    k.b = col / p.ctiles;
    k.c = ((col - k.b * p.ctiles) * 32 + lane) * V;
    k.word0 = (int64_t)k.b * p.chunks * p.C + k.c;
    return k;
}

// Publish this tile's run, gather the runs of the W tiles that precede it in walking order (the
// last of them as a state) and return the state that enters the tile; publish the one that leaves.
// `slot(i)`: word of the tile i steps earlier.  Called by all warps; s_run holds W x 32 V runs.
template <int V, int W, typename Slot, typename First>
__device__ __forceinline__ void chain(const ScanParams &p, const Tile &k, const float (&q)[V], const float (&h)[V],
                                      float (&in)[V], float2 (*s_run)[32 * V], float (*s_in), int warp, int lane,
                                      bool live, bool publish, Slot slot, First first) {
    if (k.chunk == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) in[v] = live ? first(v) : 0.f;
        if (publish && warp == 0 && live) {
#pragma unroll
            for (int v = 0; v < V; ++v) put32(p.incl + slot(0) + v, join(in[v], q[v], h[v]));
        }
        return;
    }
    if (warp == 0 && live) {
#pragma unroll
        for (int v = 0; v < V; ++v) put64(p.agg + slot(0) + v, q[v], h[v]);
    }
    const int reach = k.chunk < W ? k.chunk : W;
    if (warp < reach) {
        const bool end = warp == reach - 1;
#pragma unroll
        for (int v = 0; v < V; ++v)
            s_run[warp][lane * V + v] = live ? fetch(p, slot(warp + 1) + v, end) : make_float2(1.f, 0.f);
    }
    __syncthreads();
    if (warp == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float s = 0.f;
            for (int i = reach - 1; i >= 0; --i) {
                const float2 r = s_run[i][lane * V + v];
                s = join(s, r.x, r.y);
            }
            s_in[lane * V + v] = s;
            if (live && publish) put32(p.incl + slot(0) + v, join(s, q[v], h[v]));
        }
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) in[v] = s_in[lane * V + v];
}

__device__ __forceinline__ uint32_t reset_mask(const ScanParams &p, int b, int row0, int rows, int lane) {
    if (!p.reset) return 0;
    const int l = row0 + lane;
    const bool r = lane < rows && l < p.L && p.reset[(int64_t)b * p.L + l] != 0;
    return __ballot_sync(0xffffffffu, r);
}

// ------------------------------------------------------------------------------------- forward
template <typename T, int V, int W, int R, bool GATE>
__global__ void __launch_bounds__(W * 32, 512 / (W * 32)) scan_forward(const ScanParams p) {
    static_assert(W * R == SCAN_ROWS, "tile");
    __shared__ float2 s_run[W][32 * V];
    __shared__ float s_in[32 * V];
    __shared__ int s_tile;
    if (test_expired(p)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int t = blockIdx.x;
    if (p.chunks > 1) {
        if (threadIdx.x == 0) s_tile = atomicAdd(p.counter, 1) + 1;
        __syncthreads();
        t = s_tile;
    }
    const Tile k = tile_of<V>(p, t, lane);
    const bool live = k.c < p.C;
    const int l0 = k.chunk * SCAN_ROWS + warp * R;
    const int rows = live ? min(R, p.L - l0) : 0;

    Pack<T, V> x[R], f[R], o[GATE ? R : 1];
    {
        const T *xp = static_cast<const T *>(p.x.p) + k.b * p.x.sb + l0 * p.x.sl + k.c;
        const T *fp = static_cast<const T *>(p.f.p) + k.b * p.f.sb + l0 * p.f.sl + k.c;
        const T *op = GATE ? static_cast<const T *>(p.gate.p) + k.b * p.gate.sb + l0 * p.gate.sl + k.c : nullptr;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r < rows) {
                f[r].load(fp + r * p.f.sl, V);
                x[r].load(xp + r * p.x.sl, V);
                if (GATE) o[GATE ? r : 0].load(op + r * p.gate.sl, V);
            } else {
                f[r].zero();
                x[r].zero();
                if (GATE) o[GATE ? r : 0].zero();
            }
        }
    }
    const uint32_t cuts = reset_mask(p, k.b, l0, R, lane);
    float z[R][V], q[V], h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float bias = live && p.bias ? __ldg(p.bias + k.c + v) : 0.f;
        q[v] = h[v] = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            z[r][v] = r < rows ? sigmoid_neg(f[r].at(v) + bias) : 0.f;
            if (cuts >> r & 1) {
                q[v] = 1.f;
                h[v] = 0.f;
            }
            h[v] = advance(h[v], z[r][v], x[r].at(v));
            q[v] = fmaf(z[r][v], 1.f - q[v], q[v]);
        }
        s_run[warp][lane * V + v] = make_float2(q[v], h[v]);
    }
    __syncthreads();
    // this warp's place in the tile: the run before its rows, and the whole tile's
    float pq[V], ph[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float cq = 0.f, ch = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w == warp) {
                pq[v] = cq;
                ph[v] = ch;
            }
            const float2 r = s_run[w][lane * V + v];
            ch = join(ch, r.x, r.y);
            cq = r.x == 1.f ? 1.f : fmaf(r.x, 1.f - cq, cq);
        }
        q[v] = cq;
        h[v] = ch;
    }
    __syncthreads();
    float in[V];
    chain<V, W>(
        p, k, q, h, in, s_run, s_in, warp, lane, live, p.chunks > 1,
        [&](int i) { return k.word0 + (int64_t)(k.chunk - i) * p.C; },
        [&](int v) { return p.h0 ? p.h0[(int64_t)k.b * p.C + k.c + v] : 0.f; });
    if (p.h_last && warp == 0 && k.chunk == p.chunks - 1 && live) {
#pragma unroll
        for (int v = 0; v < V; ++v) p.h_last[(int64_t)k.b * p.C + k.c + v] = join(in[v], q[v], h[v]);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = join(in[v], pq[v], ph[v]);
    T *yp = static_cast<T *>(p.y.p) + k.b * p.y.sb + l0 * p.y.sl + k.c;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float y[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (cuts >> r & 1) h[v] = 0.f;
            h[v] = advance(h[v], z[r][v], x[r].at(v));
            y[v] = h[v];
            if (GATE) {
                const float g = o[GATE ? r : 0].at(v);
                y[v] *= g * sigmoid(g);
            }
        }
        if (r < rows) Pack<T, V>::store(yp + r * p.y.sl, y, V);
    }
}

// ------------------------------------------------------------------------------------ backward
template <typename T, int V, int W, int R, bool GATE>
__global__ void __launch_bounds__(W * 32, 1) scan_backward(const ScanParams p) {
    static_assert(W * R == SCAN_ROWS, "tile");
    __shared__ float2 s_fwd[W][32 * V], s_run[W][32 * V];
    __shared__ float s_in[32 * V];
    __shared__ int s_tile;
    if (test_expired(p)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int t = blockIdx.x;
    if (p.chunks > 1) {
        if (threadIdx.x == 0) s_tile = atomicAdd(p.counter, 1) + 1;
        __syncthreads();
        t = s_tile;
    }
    const Tile k = tile_of<V>(p, t, lane);
    const bool live = k.c < p.C;
    const int chunk = p.chunks - 1 - k.chunk;  // the last tokens first
    const int l0 = chunk * SCAN_ROWS + warp * R;
    const int rows = live ? min(R, p.L - l0) : 0;

    Pack<T, V> x[R], f[R], dy[R], o[GATE ? R : 1];
    {
        const T *xp = static_cast<const T *>(p.x.p) + k.b * p.x.sb + l0 * p.x.sl + k.c;
        const T *fp = static_cast<const T *>(p.f.p) + k.b * p.f.sb + l0 * p.f.sl + k.c;
        const T *dp = static_cast<const T *>(p.dy.p) + k.b * p.dy.sb + l0 * p.dy.sl + k.c;
        const T *op = GATE ? static_cast<const T *>(p.gate.p) + k.b * p.gate.sb + l0 * p.gate.sl + k.c : nullptr;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r < rows) {
                f[r].load(fp + r * p.f.sl, V);
                x[r].load(xp + r * p.x.sl, V);
                dy[r].load(dp + r * p.dy.sl, V);
                if (GATE) o[GATE ? r : 0].load(op + r * p.gate.sl, V);
            } else {
                f[r].zero();
                x[r].zero();
                dy[r].zero();
                if (GATE) o[GATE ? r : 0].zero();
            }
        }
    }
    float start[V];
#pragma unroll
    for (int v = 0; v < V; ++v)
        start[v] = !live       ? 0.f
                   : chunk > 0 ? __uint_as_float(p.states[k.word0 + (int64_t)(chunk - 1) * p.C + v])
                   : p.h0      ? p.h0[(int64_t)k.b * p.C + k.c + v]
                               : 0.f;
    const uint32_t cuts = reset_mask(p, k.b, l0, R, lane);
    float bias[V], z[R][V], sg[GATE ? R : 1][V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bias[v] = live && p.bias ? __ldg(p.bias + k.c + v) : 0.f;
        float q = 0.f, h = 0.f, c = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            z[r][v] = r < rows ? sigmoid_neg(f[r].at(v) + bias[v]) : 0.f;
            if (cuts >> r & 1) {
                q = 1.f;
                h = 0.f;
            }
            h = advance(h, z[r][v], x[r].at(v));
            q = fmaf(z[r][v], 1.f - q, q);
        }
#pragma unroll
        for (int r = R - 1; r >= 0; --r) {
            float s = dy[r].at(v);
            if (GATE) {
                const float g = o[GATE ? r : 0].at(v);
                sg[GATE ? r : 0][v] = sigmoid(g);
                s *= g * sg[GATE ? r : 0][v];
            }
            s += c;
            c = cuts >> r & 1 ? 0.f : fmaf(-z[r][v], s, s);
        }
        s_fwd[warp][lane * V + v] = make_float2(q, h);
        s_run[warp][lane * V + v] = make_float2(q, c);
    }
    __syncthreads();
    float q[V], g[V], sq[V], sc[V];  // the tile's run from the right; the run of the rows right of this warp's
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float cq = 0.f, cc = 0.f;
#pragma unroll
        for (int w = W - 1; w >= 0; --w) {
            if (w == warp) {
                sq[v] = cq;
                sc[v] = cc;
            }
            const float2 r = s_run[w][lane * V + v];
            cc = join(cc, r.x, r.y);
            cq = r.x == 1.f ? 1.f : fmaf(r.x, 1.f - cq, cq);
        }
        q[v] = cq;
        g[v] = cc;
        float h = start[v];
        for (int w = 0; w < warp; ++w) {
            const float2 r = s_fwd[w][lane * V + v];
            h = join(h, r.x, r.y);
        }
        start[v] = h;
    }
    __syncthreads();
    float in[V];
    chain<V, W>(
        p, k, q, g, in, s_run, s_in, warp, lane, live, p.chunks > 1,
        [&](int i) { return k.word0 + (int64_t)(k.chunk - i) * p.C; },
        [&](int v) { return p.dh_last ? p.dh_last[(int64_t)k.b * p.C + k.c + v] : 0.f; });
    if (p.dh0 && warp == 0 && chunk == 0 && live) {
#pragma unroll
        for (int v = 0; v < V; ++v) p.dh0[(int64_t)k.b * p.C + k.c + v] = join(in[v], q[v], g[v]);
    }
    float prev[R][V], c[V], db[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        c[v] = join(in[v], sq[v], sc[v]);
        db[v] = 0.f;
        float h = start[v];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (cuts >> r & 1) h = 0.f;
            prev[r][v] = h;
            h = advance(h, z[r][v], x[r].at(v));
        }
    }
    T *dxp = static_cast<T *>(p.dx.p) + k.b * p.dx.sb + l0 * p.dx.sl + k.c;
    T *dfp = static_cast<T *>(p.df.p) + k.b * p.df.sb + l0 * p.df.sl + k.c;
    T *dop = GATE ? static_cast<T *>(p.dgate.p) + k.b * p.dgate.sb + l0 * p.dgate.sl + k.c : nullptr;
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
        float dx[V], df[V], dg[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float zz = z[r][v], hp = prev[r][v], dd = dy[r].at(v);
            float s = dd;
            if (GATE) {
                const float o_ = o[GATE ? r : 0].at(v), sig = sg[GATE ? r : 0][v];
                s *= o_ * sig;
                // silu'(o) = sigmoid(o) (1 + o (1 - sigmoid(o)))
                dg[v] = dd * advance(hp, zz, x[r].at(v)) * (sig * fmaf(o_, 1.f - sig, 1.f));
            }
            s += c[v];
            dx[v] = zz * s;
            // a = exp(u) sigmoid(-u): 1 - z would lose a small a
            const float a = exp_sat(f[r].at(v) + bias[v]) * zz;
            df[v] = dx[v] * (hp - x[r].at(v)) * a;
            if (r < rows) db[v] += df[v];
            c[v] = cuts >> r & 1 ? 0.f : fmaf(-zz, s, s);
        }
        if (r < rows) {
            Pack<T, V>::store(dxp + r * p.dx.sl, dx, V);
            Pack<T, V>::store(dfp + r * p.df.sl, df, V);
            if (GATE) Pack<T, V>::store(dop + r * p.dgate.sl, dg, V);
        }
    }
    if (p.dbias_part) {
        // s_fwd is free: every warp read it before the last barrier
#pragma unroll
        for (int v = 0; v < V; ++v) s_fwd[warp][lane * V + v].x = db[v];
        __syncthreads();
        if (warp == 0 && live) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float s = 0.f;
                for (int w = 0; w < W; ++w) s += s_fwd[w][lane * V + v].x;
                p.dbias_part[((int64_t)k.b * p.chunks + chunk) * p.C + k.c + v] = s;
            }
        }
    }
}

// dbias[c] = sum of the tiles' partial sums, in a fixed order: 32 channels a block, 16 warps
// stride the rows.
__global__ void __launch_bounds__(512) scan_bias_sum(const float *part, int64_t rows, int C, float *dbias) {
    __shared__ float s[16][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane;
    float a = 0.f;
    if (c < C)
        for (int64_t r = warp; r < rows; r += 16) a += part[r * C + c];
    s[warp][lane] = a;
    __syncthreads();
    if (warp == 0 && c < C) {
        float t = 0.f;
        for (int w = 0; w < 16; ++w) t += s[w][lane];
        dbias[c] = t;
    }
}

// --------------------------------------------------------------------------------- one token
template <typename T, int V>
__global__ void __launch_bounds__(128) scan_step(const ScanStepParams p) {
    const int per = (p.C + V - 1) / V;
    const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (i >= (int64_t)p.N * per) return;
    const int n = (int)(i / per), c = (int)(i - (int64_t)n * per) * V;
    int64_t row = n;
    bool held = true;  // a row outside the pool keeps no state: its output is zero
    if (p.rows) {
        row = p.rows[n];
        held = row >= 0 && row < p.pool_rows;
    }
    Pack<T, V> x, f, o;
    x.load(static_cast<const T *>(p.x.p) + n * p.x.sb + c, V);
    f.load(static_cast<const T *>(p.f.p) + n * p.f.sb + c, V);
    if (p.gate.p) o.load(static_cast<const T *>(p.gate.p) + n * p.gate.sb + c, V);
    float y[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        y[v] = 0.f;
        if (held) {
            float h = p.h_in[row * p.C + c + v];
            const float z = sigmoid_neg(f.at(v) + (p.bias ? __ldg(p.bias + c + v) : 0.f));
            h = advance(h, z, x.at(v));
            p.h_out[row * p.C + c + v] = h;
            y[v] = p.gate.p ? h * (o.at(v) * sigmoid(o.at(v))) : h;
        }
    }
    Pack<T, V>::store(static_cast<T *>(p.y.p) + n * p.y.sb + c, y, V);
}

// bf16 pairs need an even channel count and even strides on 4-byte boundaries; one channel a lane
// otherwise (half the bytes a warp moves per row: 64 instead of 128).
bool pairs(const Blc &t) {
    return !t.p || (reinterpret_cast<uintptr_t>(t.p) % 4 == 0 && t.sb % 2 == 0 && t.sl % 2 == 0);
}

template <typename T, int V>
cudaError_t forward_t(ScanParams &p, cudaStream_t st) {
    p.ctiles = (p.C + 32 * V - 1) / (32 * V);
    const int64_t tiles = (int64_t)p.chunks * p.B * p.ctiles;
    if (tiles > 0x7fffffff) return cudaErrorInvalidValue;
    if (p.gate.p)
        scan_forward<T, V, 8, 16, true><<<(unsigned)tiles, 256, 0, st>>>(p);
    else
        scan_forward<T, V, 8, 16, false><<<(unsigned)tiles, 256, 0, st>>>(p);
    return cudaGetLastError();
}

template <typename T, int V>
cudaError_t backward_t(ScanParams &p, cudaStream_t st) {
    p.ctiles = (p.C + 32 * V - 1) / (32 * V);
    const int64_t tiles = (int64_t)p.chunks * p.B * p.ctiles;
    if (tiles > 0x7fffffff) return cudaErrorInvalidValue;
    if (p.gate.p)
        scan_backward<T, V, 16, 8, true><<<(unsigned)tiles, 512, 0, st>>>(p);
    else
        scan_backward<T, V, 16, 8, false><<<(unsigned)tiles, 512, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_gated_scan(ScanParams p, int dtype, cudaStream_t st) {
    if (dtype == PMA_F32) return forward_t<float, 1>(p, st);
    if (p.C % 2 == 0 && pairs(p.x) && pairs(p.f) && pairs(p.gate) && pairs(p.y))
        return forward_t<__nv_bfloat16, 2>(p, st);
    return forward_t<__nv_bfloat16, 1>(p, st);
}

cudaError_t launch_gated_scan_backward(ScanParams p, int dtype, float *dbias, cudaStream_t st) {
    cudaError_t e;
    if (dtype == PMA_F32)
        e = backward_t<float, 1>(p, st);
    else if (p.C % 2 == 0 && pairs(p.x) && pairs(p.f) && pairs(p.gate) && pairs(p.dy) && pairs(p.dx) && pairs(p.df) &&
             pairs(p.dgate))
        e = backward_t<__nv_bfloat16, 2>(p, st);
    else
        e = backward_t<__nv_bfloat16, 1>(p, st);
    if (e != cudaSuccess || !dbias) return e;
    scan_bias_sum<<<(p.C + 31) / 32, 512, 0, st>>>(p.dbias_part, (int64_t)p.B * p.chunks, p.C, dbias);
    return cudaGetLastError();
}

cudaError_t launch_gated_scan_step(const ScanStepParams &p, int dtype, cudaStream_t st) {
    const bool two = dtype == PMA_BF16 && p.C % 2 == 0 && pairs(p.x) && pairs(p.f) && pairs(p.gate) && pairs(p.y);
    const int64_t items = (int64_t)p.N * (two ? p.C / 2 : p.C);
    const int64_t blocks = (items + 127) / 128;
    if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
    if (dtype == PMA_F32)
        scan_step<float, 1><<<(unsigned)blocks, 128, 0, st>>>(p);
    else if (two)
        scan_step<__nv_bfloat16, 2><<<(unsigned)blocks, 128, 0, st>>>(p);
    else
        scan_step<__nv_bfloat16, 1><<<(unsigned)blocks, 128, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace pma
