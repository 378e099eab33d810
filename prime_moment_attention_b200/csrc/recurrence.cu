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
//   h -> P h + H = h + (H - Q h),   P = prod a_t,   Q = 1 - P,   H = its result from a zero state,
// kept as Q where P > 1/2 and as P elsewhere: for slow decays 1 - prod a_t is what matters and the
// product would round it away; of a state that the run forgets only P h is left, and h + (H - Q h)
// would keep an ulp of h.  A token joins a run by Q <- Q + z P, P <- a P, H <- a H + z x.
// Every input is read once: a tile holds its rows in registers, publishes its run as one 64-bit
// word per channel, gathers the words of the tiles before it back to one that has published the
// state leaving it, and then writes its outputs.  Words start as all ones (a NaN that no result
// carries) and are written once, so a word is its own flag and no fence is needed.  A state is
// always the same chain of joins, tile after tile, whether a tile found the state that leaves a
// neighbour or joined the neighbour's run itself: results do not depend on timing.  A state that is
// not finite stays so up to a reset.  Tiles are handed out in the order of a counter, so a tile only
// waits for tiles that are already running; every wait is bounded.
//
// Backward, from the right, with the carry c_t = a_t g_t:
//   g_t = dy_t silu(gate_t) + c_{t+1},   dx = z g,   df = g (h_{t-1} - x) a z,
//   dgate = dy h silu'(gate),            dbias = sum df,            dh0 = c_0.
// A tile recomputes its states from the one that entered it, which the forward pass kept (one
// float32 state per channel and 128 tokens).  dbias is summed within a tile, then over the tiles
// in a fixed order by a second kernel.
#include "recurrence.cuh"

#include <cooperative_groups.h>

#include "tc_common.cuh"

namespace cg = cooperative_groups;

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

// 2^min(x, 126), NaN kept: finite, so that exp(u) sigmoid(-u) is a sigmoid and not inf * 0
__device__ __forceinline__ float ex2_sat(float x) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(126.0f));
    return ex2(r);
}

// V float32 values of a lane (its channels): pairs go through the two-wide float32 instructions,
// which halve the arithmetic a channel costs.
template <int V> struct Vf;
template <> struct Vf<1> {
    float v;
    static __device__ __forceinline__ Vf all(float a) { return {a}; }
    __device__ __forceinline__ float at(int) const { return v; }
};
template <> struct Vf<2> {
    unsigned long long v;
    static __device__ __forceinline__ Vf of(float a, float b) {
        Vf r;
        asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
        return r;
    }
    static __device__ __forceinline__ Vf all(float a) { return of(a, a); }
    __device__ __forceinline__ float at(int i) const {
        float a, b;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
        return i ? b : a;
    }
};
// The values f(0) .. f(V - 1)
template <int V, typename F> __device__ __forceinline__ Vf<V> gather(F f) {
    if constexpr (V == 1)
        return {f(0)};
    else
        return Vf<2>::of(f(0), f(1));
}

__device__ __forceinline__ Vf<1> fma(Vf<1> a, Vf<1> b, Vf<1> c) { return {fmaf(a.v, b.v, c.v)}; }
__device__ __forceinline__ Vf<1> mul(Vf<1> a, Vf<1> b) { return {a.v * b.v}; }
__device__ __forceinline__ Vf<1> add(Vf<1> a, Vf<1> b) { return {a.v + b.v}; }
__device__ __forceinline__ Vf<2> fma(Vf<2> a, Vf<2> b, Vf<2> c) {
    Vf<2> r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ Vf<2> mul(Vf<2> a, Vf<2> b) {
    Vf<2> r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Vf<2> add(Vf<2> a, Vf<2> b) {
    Vf<2> r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
template <int V, typename F> __device__ __forceinline__ Vf<V> each(Vf<V> a, F f) {
    if constexpr (V == 1)
        return {f(a.v)};
    else
        return Vf<2>::of(f(a.at(0)), f(a.at(1)));
}

// sigmoid(-u) for u in units of log 2; sigmoid(g)
template <int V> __device__ __forceinline__ Vf<V> sigmoid_neg2(Vf<V> u) {
    return each(add(each(u, ex2_sat), Vf<V>::all(1.f)), rcp);
}
template <int V> __device__ __forceinline__ Vf<V> sigmoid(Vf<V> g) {
    return each(add(each(mul(g, Vf<V>::all(-LOG2E)), ex2), Vf<V>::all(1.f)), rcp);
}

// One token.  This form is exact at both ends (z = 0 keeps h, z = 1 takes x); rounding 1 - z costs a
// slow decay half an ulp a row, over the few rows between two joins.
template <int V> __device__ __forceinline__ Vf<V> advance(Vf<V> h, Vf<V> z, Vf<V> x) {
    return fma(fma(z, Vf<V>::all(-1.f), Vf<V>::all(1.f)), h, mul(z, x));
}

// A run of tokens: H, and in n what it leaves of the state that enters: P > 0 where it is at most 1/2,
// else -Q (0: an empty run); DROP where the state is dropped whatever it was, NaN and infinities
// included (a reset, or a state handed on as a run).
constexpr float DROP = -1.f;
template <int V> struct Run {
    Vf<V> n, h;
};
// The state after a run.  CUT: the run may drop it; the result of other runs is the same with and without.
template <bool CUT, int V> __device__ __forceinline__ Vf<V> join(Vf<V> h, const Run<V> &r) {
    const Vf<V> t = fma(r.n, h, r.h), o = add(h, t);
    return gather<V>([&](int v) {
        const float n = r.n.at(v), some = n > 0.f ? t.at(v) : o.at(v);
        return CUT && n == DROP ? r.h.at(v) : some;
    });
}
// P > 0 or -Q <= 0.  A product that underflows is no drop: 2^-149 of what is not finite is not finite either.
template <int V> __device__ __forceinline__ Run<V> coded(Vf<V> p, Vf<V> q, Vf<V> h) {
    return {gather<V>([&](int v) { return p.at(v) <= 0.5f ? fmaxf(p.at(v), __uint_as_float(1u)) : -q.at(v); }), h};
}
// A run inside a tile: P to twice the precision, p + e, so that its joins are products and sums alone.
// Resets are the same for all channels: a part that has one replaces what it joins (the callers' business).
template <int V> struct Part {
    Vf<V> p, e, h;
};
template <int V> __device__ __forceinline__ Vf<V> minus(Vf<V> a, Vf<V> b) { return fma(b, Vf<V>::all(-1.f), a); }
template <int V> __device__ __forceinline__ Part<V> part_of(Vf<V> p, Vf<V> q, Vf<V> h) {
    const Vf<V> one = Vf<V>::all(1.f), hi = minus(one, q), lo = minus(minus(one, hi), q);
    return {gather<V>([&](int v) { return p.at(v) <= 0.5f ? p.at(v) : hi.at(v); }),
            gather<V>([&](int v) { return p.at(v) <= 0.5f ? 0.f : lo.at(v); }), h};
}
template <int V> __device__ __forceinline__ Part<V> no_part() {
    return {Vf<V>::all(1.f), Vf<V>::all(0.f), Vf<V>::all(0.f)};
}
template <int V> __device__ __forceinline__ Vf<V> join_part(Vf<V> h, const Part<V> &b) { return fma(b.p, h, fma(b.e, h, b.h)); }
template <int V> __device__ __forceinline__ Part<V> join_part(const Part<V> &a, const Part<V> &b) {
    const Vf<V> p = mul(a.p, b.p), r = fma(a.p, b.p, mul(p, Vf<V>::all(-1.f)));
    return {p, fma(a.p, b.e, fma(a.e, b.p, r)), join_part(a.h, b)};
}
template <int V> __device__ __forceinline__ Run<V> run_of(const Part<V> &a, bool dropped) {
    const Vf<V> q = minus(minus(Vf<V>::all(1.f), a.p), a.e);
    Run<V> r = coded(add(a.p, a.e), each(q, [](float v) { return fmaxf(v, 0.f); }), a.h);
    if (dropped) r.n = Vf<V>::all(DROP);
    return r;
}

// The parts of a tile that have a reset, as a mask
template <int W> __device__ __forceinline__ uint32_t which_cut(const bool (&cut)[W], int lane) {
    return __ballot_sync(0xffffffffu, lane < W && cut[lane & (W - 1)]);
}

// V consecutive channels of one row as one load or store
template <typename T, int V> struct Pack;
template <> struct Pack<float, 1> {
    float r;
    __device__ __forceinline__ void load(const float *p) { r = __ldg(p); }
    __device__ __forceinline__ Vf<1> f() const { return {r}; }
    static __device__ __forceinline__ void store(float *p, Vf<1> v) { *p = v.v; }
};
template <> struct Pack<__nv_bfloat16, 1> {
    uint16_t r;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { r = __ldg(reinterpret_cast<const unsigned short *>(p)); }
    __device__ __forceinline__ Vf<1> f() const { return {__uint_as_float((uint32_t)r << 16)}; }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, Vf<1> v) { *p = __float2bfloat16_rn(v.v); }
};
template <> struct Pack<__nv_bfloat16, 2> {
    uint32_t r;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { r = __ldg(reinterpret_cast<const unsigned int *>(p)); }
    __device__ __forceinline__ Vf<2> f() const {
        return Vf<2>::of(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, Vf<2> v) {
        *reinterpret_cast<uint32_t *>(p) = tc::pack2(v.at(0), v.at(1));
    }
};

// The rows stay packed in registers between two passes: without this the compiler keeps the unpacked
// float32 values as well and spills.
__device__ __forceinline__ void keep_packed(float &) {}
__device__ __forceinline__ void keep_packed(uint16_t &r) { asm volatile("" : "+h"(r)); }
__device__ __forceinline__ void keep_packed(uint32_t &r) { asm volatile("" : "+r"(r)); }
template <typename P, int R> __device__ __forceinline__ void keep_packed(P (&d)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) keep_packed(d[r].r);
}

__device__ __forceinline__ uint32_t word_of(float v) {
    const uint32_t u = __float_as_uint(v);
    return u == EMPTY ? 0x7fffffffu : u;
}
// V neighbouring words in one access (V divides C, so they are aligned); each word is whole.
__device__ __forceinline__ void put(uint32_t *p, Vf<1> v) {
    asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(word_of(v.v)) : "memory");
}
__device__ __forceinline__ void put(uint32_t *p, Vf<2> v) {
    asm volatile("st.relaxed.gpu.global.v2.u32 [%0], {%1, %2};" ::"l"(p), "r"(word_of(v.at(0))), "r"(word_of(v.at(1)))
                 : "memory");
}
__device__ __forceinline__ unsigned long long word_of(float n, float h) {
    return ((unsigned long long)word_of(h) << 32) | word_of(n);
}
__device__ __forceinline__ void put(unsigned long long *p, const Run<1> &r) {
    asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(word_of(r.n.v, r.h.v)) : "memory");
}
__device__ __forceinline__ void put(unsigned long long *p, const Run<2> &r) {
    asm volatile("st.relaxed.gpu.global.v2.u64 [%0], {%1, %2};" ::"l"(p), "l"(word_of(r.n.at(0), r.h.at(0))),
                 "l"(word_of(r.n.at(1), r.h.at(1)))
                 : "memory");
}
__device__ __forceinline__ void get(const uint32_t *p, uint32_t (&v)[1]) {
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v[0]) : "l"(p) : "memory");
}
__device__ __forceinline__ void get(const uint32_t *p, uint32_t (&v)[2]) {
    asm volatile("ld.relaxed.gpu.global.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "l"(p) : "memory");
}
__device__ __forceinline__ void get(const unsigned long long *p, unsigned long long (&v)[1]) {
    asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v[0]) : "l"(p) : "memory");
}
__device__ __forceinline__ void get(const unsigned long long *p, unsigned long long (&v)[2]) {
    asm volatile("ld.relaxed.gpu.global.v2.u64 {%0, %1}, [%2];" : "=l"(v[0]), "=l"(v[1]) : "l"(p) : "memory");
}

// The runs of V channels of K earlier tiles, at[0 .. K - 1] in the word arrays, or the states leaving
// them as runs (DROP, state); wait for the state where `must_end`, and skip a negative position.
template <int V, int K>
__device__ __forceinline__ void fetch(const ScanParams &p, const int64_t (&at)[K], const bool (&must_end)[K],
                                      Run<V> (&out)[K]) {
    unsigned long long t0 = 0;
    float n[K][V], h[K][V];
    bool got[K][V];
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            got[i][v] = at[i] < 0;
            n[i][v] = h[i][v] = 0.f;
        }
    for (uint32_t it = 1;; ++it) {
        bool all = true;
        uint32_t s[K][V];
        unsigned long long a[K][V];
#pragma unroll
        for (int i = 0; i < K; ++i) {  // every load is in flight before the first is looked at
            bool have = true;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                have = have && got[i][v];
                s[i][v] = EMPTY;
                a[i][v] = ~0ull;
            }
            if (!have) {
                get(p.incl + at[i], s[i]);
                if (!must_end[i]) get(p.agg + at[i], a[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < K; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (got[i][v]) continue;
                if (s[i][v] != EMPTY) {
                    n[i][v] = DROP;
                    h[i][v] = __uint_as_float(s[i][v]);
                    got[i][v] = true;
                } else if (a[i][v] != ~0ull) {
                    n[i][v] = __uint_as_float((uint32_t)a[i][v]);
                    h[i][v] = __uint_as_float((uint32_t)(a[i][v] >> 32));
                    got[i][v] = true;
                }
                all = all && got[i][v];
            }
        if (all) break;
        if ((it & 255) == 0) {
            const unsigned long long now = tc::gtimer();
            if (!t0) t0 = now;
            const bool gone = *reinterpret_cast<volatile int *>(p.counter + 1) != -1;
            if (gone || now - t0 > p.wait_ns) {  // NaN states: the launch's results are void
                *reinterpret_cast<volatile int *>(p.counter + 1) = FAULT_CODE;
                tc::report_fault(FAULT_CODE, p.fault);
#pragma unroll
                for (int i = 0; i < K; ++i)
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        n[i][v] = DROP;
                        h[i][v] = __uint_as_float(0x7fffffffu);
                    }
                break;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < K; ++i) {
        out[i].n = gather<V>([&](int v) { return n[i][v]; });
        out[i].h = gather<V>([&](int v) { return h[i][v]; });
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

// How many tiles back a tile looks: each step of the chain of states covers as many tiles.
constexpr int LOOK = 16;

template <int V> struct Scratch {
    Run<V> run[LOOK][32];
    Vf<V> in[32];
};

// Publish this tile's run (warp 0 holds it), gather the runs of the LOOK tiles that precede it in
// walking order (the last of them as a state) and return the state that enters the tile; publish
// the one that leaves, which `last` receives (warp 0).  sync(): a barrier of the W warps.
template <bool CUT, int V, int W, typename Sync, typename First, typename Last>
__device__ __forceinline__ Vf<V> chain(const ScanParams &p, const Tile &k, const Run<V> &whole, Scratch<V> &sm,
                                       int warp, int lane, bool live, Sync sync, First first, Last last) {
    const int64_t slot = k.word0 + (int64_t)k.chunk * p.C;
    Vf<V> in = Vf<V>::all(0.f);
    if (k.chunk == 0) {
        if (live) in = gather<V>(first);
    } else {
        if (warp == 0 && live) put(p.agg + slot, whole);
        const int reach = k.chunk < LOOK ? k.chunk : LOOK;
        constexpr int K = LOOK / W < 2 ? 1 : 2;  // tiles a warp asks for at once
        for (int d0 = warp; d0 < LOOK; d0 += K * W) {
            int64_t at[K];
            bool end[K];
            Run<V> r[K];
#pragma unroll
            for (int i = 0; i < K; ++i) {
                const int d = d0 + i * W;
                at[i] = d < reach && live ? slot - (int64_t)(d + 1) * p.C : -1;  // else an empty run
                end[i] = d == reach - 1;
            }
            fetch<V, K>(p, at, end, r);
#pragma unroll
            for (int i = 0; i < K; ++i) sm.run[d0 + i * W][lane] = r[i];
        }
        sync();
        if (warp == 0) {
            Run<V> r[LOOK];
#pragma unroll
            for (int i = 0; i < LOOK; ++i) r[i] = sm.run[i][lane];
#pragma unroll
            for (int i = LOOK - 1; i >= 0; --i) in = join<true>(in, r[i]);
            sm.in[lane] = in;
        }
    }
    if (warp == 0 && live) {
        const Vf<V> out = join<CUT>(in, whole);
        if (p.chunks > 1) put(p.incl + slot, out);
        if (k.chunk == p.chunks - 1) last(out);
    }
    if (k.chunk) {
        sync();
        in = sm.in[lane];
    }
    return in;
}

// Every CTA of the cluster runs, so that its shared memory may be written: said at the kernel's start,
// waited for before the first access.
__device__ __forceinline__ void cluster_start() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_started() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// The same for a sequence of a few tiles, whose CTAs form a cluster (rank: the tile in walking order):
// each sends its run to the later ones, and there is nothing to wait for but the cluster's barrier.
template <bool CUT, int V, typename First, typename Last>
__device__ __forceinline__ Vf<V> chain_cluster(const ScanParams &p, const Tile &k, const Run<V> &whole, Scratch<V> &sm,
                                               int warp, int lane, bool live, First first, Last last) {
    const cg::cluster_group cl = cg::this_cluster();
    cluster_started();
    if (warp == 0)
        for (int r = k.chunk + 1; r < p.chunks; ++r) cl.map_shared_rank(&sm, r)->run[k.chunk][lane] = whole;
    cl.sync();
    Vf<V> in = Vf<V>::all(0.f);
    if (live) in = gather<V>(first);
    for (int i = 0; i < k.chunk; ++i) in = join<CUT>(in, sm.run[i][lane]);
    if (warp == 0 && live) {
        const Vf<V> out = join<CUT>(in, whole);
        if (p.incl) put(p.incl + k.word0 + (int64_t)k.chunk * p.C, out);
        if (k.chunk == p.chunks - 1) last(out);
    }
    return in;
}

__device__ __forceinline__ uint32_t reset_mask(const ScanParams &p, int b, int row0, int rows, int lane) {
    const int l = row0 + lane;
    const bool r = lane < rows && l < p.L && p.reset[(int64_t)b * p.L + l] != 0;
    return __ballot_sync(0xffffffffu, r);
}

// R rows of a lane's channels.  Rows past the end and channels past C are read again from the last
// ones: every address is valid and nothing has to be skipped.
template <typename T, int V, int R>
__device__ __forceinline__ void load_rows(Pack<T, V> (&d)[R], const Blc &t, int b, int l0, int L, int c) {
    const T *p = static_cast<const T *>(t.p) + b * t.sb + l0 * t.sl + c;
    if (l0 + R <= L) {
#pragma unroll
        for (int r = 0; r < R; ++r) d[r].load(p + r * t.sl);
    } else {
#pragma unroll
        for (int r = 0; r < R; ++r) d[r].load(p + (int64_t)min(r, L - 1 - l0) * t.sl);
    }
}

// ------------------------------------------------------------------------------------- forward
template <typename T, int V, int W, int R, bool GATE, bool CUT, bool CLUSTER>
__global__ void __launch_bounds__(W * 32, 512 / (W * 32)) scan_forward(const ScanParams p) {
    static_assert(W * R == SCAN_ROWS, "tile");
    __shared__ Scratch<V> sm;  // the other tiles' runs
    __shared__ Part<V> parts[W][32];
    __shared__ bool s_cut[W];
    __shared__ int s_tile;
    if (test_expired(p)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int t = blockIdx.x;
    if (CLUSTER) {
        cluster_start();
        t = (int)(blockIdx.x % p.chunks) * (p.B * p.ctiles) + (int)(blockIdx.x / p.chunks);
    } else if (p.chunks > 1) {
        if (threadIdx.x == 0) s_tile = atomicAdd(p.counter, 1) + 1;
        __syncthreads();
        t = s_tile;
    }
    const Tile k = tile_of<V>(p, t, lane);
    const bool live = k.c < p.C;
    const int l0 = k.chunk * SCAN_ROWS + warp * R, rows = min(R, p.L - l0), c = live ? k.c : p.C - V;

    Pack<T, V> x[R], f[R], o[GATE ? R : 1];
    load_rows<T, V, R>(f, p.f, k.b, l0, p.L, c);
    load_rows<T, V, R>(x, p.x, k.b, l0, p.L, c);
    if constexpr (GATE) load_rows<T, V, R>(o, p.gate, k.b, l0, p.L, c);
    const uint32_t cuts = CUT ? reset_mask(p, k.b, l0, R, lane) : 0;
    const Vf<V> bias = gather<V>([&](int v) { return p.bias ? __ldg(p.bias + c + v) * LOG2E : 0.f; });
    Vf<V> z[R];
#pragma unroll
    for (int r = 0; r < R; ++r) z[r] = sigmoid_neg2(fma(f[r].f(), Vf<V>::all(LOG2E), bias));
    if (rows < R) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r >= rows) z[r] = Vf<V>::all(0.f);
    }
    {
        Vf<V> q = Vf<V>::all(0.f), h = q, left = Vf<V>::all(1.f);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (CUT && (cuts >> r & 1)) h = Vf<V>::all(0.f);
            h = advance(h, z[r], x[r].f());
            q = fma(z[r], left, q);
            left = mul(left, fma(z[r], Vf<V>::all(-1.f), Vf<V>::all(1.f)));
        }
        parts[warp][lane] = part_of(left, q, h);
        if (CUT) s_cut[warp] = cuts != 0;
    }
    __syncthreads();
    // the run of the tile's rows before this warp's; warp 0, which has none, joins the whole tile
    Part<V> part = no_part<V>();
    const int upto = warp ? warp : W;
    const uint32_t cut = CUT ? which_cut<W>(s_cut, lane) & ((1u << upto) - 1u) : 0;
    for (int w = 0; w < upto; ++w) {
        part = join_part(part, parts[w][lane]);
        if (CUT && (cut >> w & 1)) part.h = parts[w][lane].h;
    }
    const Run<V> run = run_of(part, cut);
    const auto join_tiles = [&](auto first, auto last) {
        if constexpr (CLUSTER)
            return chain_cluster<CUT, V>(p, k, run, sm, warp, lane, live, first, last);
        else
            return chain<CUT, V, W>(p, k, run, sm, warp, lane, live, [] { __syncthreads(); }, first, last);
    };
    const Vf<V> in = join_tiles(
        [&](int v) { return p.h0 ? p.h0[(int64_t)k.b * p.C + k.c + v] : 0.f; },
        [&](Vf<V> out) {
            if (p.h_last) {
#pragma unroll
                for (int v = 0; v < V; ++v) p.h_last[(int64_t)k.b * p.C + k.c + v] = out.at(v);
            }
        });
    Vf<V> h = warp ? join<CUT>(in, run) : in;
    keep_packed(x);
    if constexpr (GATE) keep_packed(o);
    T *yp = static_cast<T *>(p.y.p) + k.b * p.y.sb + l0 * p.y.sl + c;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (CUT && (cuts >> r & 1)) h = Vf<V>::all(0.f);
        h = advance(h, z[r], x[r].f());
        Vf<V> y = h;
        if constexpr (GATE) {
            const Vf<V> g = o[r].f();
            y = mul(y, mul(g, sigmoid(g)));
        }
        if (live && r < rows) Pack<T, V>::store(yp + r * p.y.sl, y);
    }
}

// ------------------------------------------------------------------------------------ backward
template <typename T, int V, int W, int R, bool GATE, bool CUT, bool CLUSTER>
__global__ void __launch_bounds__(W * 32, 1) scan_backward(const ScanParams p) {
    static_assert(W * R == SCAN_ROWS, "tile");
    __shared__ Scratch<V> sm;  // the other tiles' runs
    __shared__ Part<V> parts[W][32];
    __shared__ Vf<V> carries[W][32];  // the parts' H in the carries' direction
    __shared__ bool s_cut[W];
    __shared__ int s_tile;
    if (test_expired(p)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int t = blockIdx.x;
    if (CLUSTER) {
        cluster_start();
        t = (int)(blockIdx.x % p.chunks) * (p.B * p.ctiles) + (int)(blockIdx.x / p.chunks);
    } else if (p.chunks > 1) {
        if (threadIdx.x == 0) s_tile = atomicAdd(p.counter, 1) + 1;
        __syncthreads();
        t = s_tile;
    }
    const Tile k = tile_of<V>(p, t, lane);
    const bool live = k.c < p.C;
    const int chunk = p.chunks - 1 - k.chunk;  // the last tokens first
    const int l0 = chunk * SCAN_ROWS + warp * R, rows = min(R, p.L - l0), c = live ? k.c : p.C - V;

    Pack<T, V> x[R], f[R], dy[R], o[GATE ? R : 1];
    load_rows<T, V, R>(f, p.f, k.b, l0, p.L, c);
    load_rows<T, V, R>(x, p.x, k.b, l0, p.L, c);
    load_rows<T, V, R>(dy, p.dy, k.b, l0, p.L, c);
    if constexpr (GATE) load_rows<T, V, R>(o, p.gate, k.b, l0, p.L, c);
    const Vf<V> bias = gather<V>([&](int v) { return p.bias ? __ldg(p.bias + c + v) * LOG2E : 0.f; });
    Vf<V> start = gather<V>([&](int v) {
        if (chunk > 0) return __uint_as_float(p.states[((int64_t)k.b * p.chunks + chunk - 1) * p.C + c + v]);
        return p.h0 ? p.h0[(int64_t)k.b * p.C + c + v] : 0.f;
    });
    const uint32_t cuts = CUT ? reset_mask(p, k.b, l0, R, lane) : 0;
    Vf<V> z[R], sg[GATE ? R : 1];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        z[r] = sigmoid_neg2(fma(f[r].f(), Vf<V>::all(LOG2E), bias));
        if constexpr (GATE) sg[r] = sigmoid(o[r].f());
    }
    // dL/dh_t through y_t; zero past the end, where z is zero too
    auto into = [&](int r) {
        Vf<V> s = dy[r].f();
        if constexpr (GATE) s = mul(s, mul(o[r].f(), sg[r]));
        if (r >= rows) s = Vf<V>::all(0.f);
        return s;
    };
    if (rows < R) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r >= rows) z[r] = Vf<V>::all(0.f);
    }
    // the carry a g of one token
    auto carry = [&](int r, Vf<V> g) {
        if (CUT && (cuts >> r & 1)) return Vf<V>::all(0.f);
        return fma(mul(z[r], Vf<V>::all(-1.f)), g, g);
    };
    {
        Vf<V> q = Vf<V>::all(0.f), h = q, cc = q, left = Vf<V>::all(1.f);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (CUT && (cuts >> r & 1)) h = Vf<V>::all(0.f);
            h = advance(h, z[r], x[r].f());
            q = fma(z[r], left, q);
            left = mul(left, fma(z[r], Vf<V>::all(-1.f), Vf<V>::all(1.f)));
        }
#pragma unroll
        for (int r = R - 1; r >= 0; --r) cc = carry(r, add(into(r), cc));
        keep_packed(x);
        keep_packed(f);
        keep_packed(dy);
        if constexpr (GATE) keep_packed(o);
        parts[warp][lane] = part_of(left, q, h);
        carries[warp][lane] = cc;
        if (CUT) s_cut[warp] = cuts != 0;
    }
    __syncthreads();
    // the carries of the rows right of this warp's; the last warp, which has none, joins the tile's
    Part<V> part = no_part<V>();
    uint32_t cut = CUT ? which_cut<W>(s_cut, lane) : 0;
    {
        const int mine = W - 1 - warp, upto = mine ? mine : W;
        for (int i = 0; i < upto; ++i) {
            const int w = W - 1 - i;
            part = join_part(part, Part<V>{parts[w][lane].p, parts[w][lane].e, carries[w][lane]});
            if (CUT && (cut >> w & 1)) part.h = carries[w][lane];
        }
        for (int w = 0; w < warp; ++w) start = CUT && (cut >> w & 1) ? parts[w][lane].h : join_part(start, parts[w][lane]);
        cut >>= W - upto;  // those that were joined
    }
    const Run<V> run = run_of(part, cut);
    __syncthreads();
    // in walking order the last warp is the first one
    const auto join_tiles = [&](auto first, auto last) {
        if constexpr (CLUSTER)
            return chain_cluster<CUT, V>(p, k, run, sm, W - 1 - warp, lane, live, first, last);
        else
            return chain<CUT, V, W>(p, k, run, sm, W - 1 - warp, lane, live, [] { __syncthreads(); }, first, last);
    };
    const Vf<V> in = join_tiles(
        [&](int v) { return p.dh_last ? p.dh_last[(int64_t)k.b * p.C + k.c + v] : 0.f; },
        [&](Vf<V> out) {
            if (p.dh0) {
#pragma unroll
                for (int v = 0; v < V; ++v) p.dh0[(int64_t)k.b * p.C + k.c + v] = out.at(v);
            }
        });
    Vf<V> cc = warp == W - 1 ? in : cut ? part.h : join_part(in, part), prev[R], db = Vf<V>::all(0.f);
    {
        Vf<V> h = start;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (CUT && (cuts >> r & 1)) h = Vf<V>::all(0.f);
            prev[r] = h;
            h = advance(h, z[r], x[r].f());
        }
        keep_packed(x);
    }
    T *dxp = static_cast<T *>(p.dx.p) + k.b * p.dx.sb + l0 * p.dx.sl + c;
    T *dfp = static_cast<T *>(p.df.p) + k.b * p.df.sb + l0 * p.df.sl + c;
    T *dop = GATE ? static_cast<T *>(p.dgate.p) + k.b * p.dgate.sb + l0 * p.dgate.sl + c : nullptr;
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
        const Vf<V> xr = x[r].f(), g = add(into(r), cc), dx = mul(z[r], g);
        cc = carry(r, g);
        // a = exp(u) sigmoid(-u): 1 - z would lose a small a
        const Vf<V> a = mul(each(fma(f[r].f(), Vf<V>::all(LOG2E), bias), ex2_sat), z[r]);
        const Vf<V> df = mul(mul(dx, a), fma(xr, Vf<V>::all(-1.f), prev[r]));
        if (r < rows) db = add(db, df);
        if (live && r < rows) {
            Pack<T, V>::store(dxp + r * p.dx.sl, dx);
            Pack<T, V>::store(dfp + r * p.df.sl, df);
            if constexpr (GATE) {
                // silu'(o) = sigmoid(o) (1 + o (1 - sigmoid(o)))
                const Vf<V> one = Vf<V>::all(1.f), rest = fma(sg[r], Vf<V>::all(-1.f), one);
                const Vf<V> slope = mul(sg[r], fma(o[r].f(), rest, one));
                Pack<T, V>::store(dop + r * p.dgate.sl, mul(mul(dy[r].f(), advance(prev[r], z[r], xr)), slope));
            }
        }
    }
    if (p.dbias_part) {
        carries[warp][lane] = db;  // free: every warp read it before the last barrier
        __syncthreads();
        if (warp == 0 && live) {
            Vf<V> s = Vf<V>::all(0.f);
            for (int w = 0; w < W; ++w) s = add(s, carries[w][lane]);
#pragma unroll
            for (int v = 0; v < V; ++v)
                p.dbias_part[((int64_t)k.b * p.chunks + chunk) * p.C + k.c + v] = s.at(v);
        }
    }
}

// ------------------------------------------------------------------ forward, tiles moved by TMA
// Rows of 128 bytes (64 bf16 or 32 float32 channels).  One CTA an SM keeps taking tiles: a thread
// takes a tile's number and starts its copies, one of three groups of four warps works on it (32 rows
// a thread), and another thread stores the outputs, which lie where x lay, and frees the stage.
// Against the kernel above there are no addresses to compute, x and the gate need no registers, and
// a tile is on its way while three are at work.
// 262144 tokens x 1024 channels, bf16, gated: 498 us, 4.3 TB/s (2.15 GB; the kernel above takes 760 on rows
// that TMA refuses).  No pipe is full (issue slots and special functions 46 %): what bounds it is the chain of
// states through the tiles.
struct ScanMaps {
    CUtensorMap x, f, gate, y;
};

template <typename T, bool GATE> struct FwdCfg {
    static constexpr int GROUPS = 3, W = 4, R = SCAN_ROWS / W, V = sizeof(T) == 2 ? 2 : 1;
    static constexpr int TILE = SCAN_ROWS * 128;
    // f is done with after a tile's first pass, x and the gate after its last
    static constexpr int FSTAGES = 3, STAGES = 4, STAGE = (GATE ? 2 : 1) * TILE;
    static constexpr int SMEM = FSTAGES * TILE + STAGES * STAGE + 128;
    static constexpr int THREADS = (GROUPS * W + 2) * 32;
};

__device__ __forceinline__ void tma_load3(void *dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            tc::su32(dst)),
        "l"(map), "r"(tc::su32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
__device__ __forceinline__ void tma_store3(const CUtensorMap *map, const void *src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
                 "r"(tc::su32(src)), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}

// The lane's word of a 128-byte row.
template <typename T> struct Word;
template <> struct Word<float> {
    static __device__ __forceinline__ Vf<1> get(const uint8_t *p) { return {*reinterpret_cast<const float *>(p)}; }
    static __device__ __forceinline__ void put(uint8_t *p, Vf<1> v) { *reinterpret_cast<float *>(p) = v.v; }
};
template <> struct Word<__nv_bfloat16> {
    static __device__ __forceinline__ Vf<2> get(const uint8_t *p) {
        const uint32_t r = *reinterpret_cast<const uint32_t *>(p);
        return Vf<2>::of(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
    }
    static __device__ __forceinline__ void put(uint8_t *p, Vf<2> v) {
        *reinterpret_cast<uint32_t *>(p) = tc::pack2(v.at(0), v.at(1));
    }
};

// Barriers of the stages, and the tiles in them (chunk -1: no more).  The FSTAGES stages of the first
// pass's input (FSTAGES 0: none apart) are freed by the workers.
template <int FSTAGES, int STAGES> struct Ring {
    uint64_t full[STAGES], done[STAGES], empty[STAGES], f_empty[FSTAGES ? FSTAGES : 1];
    Tile tile[STAGES];
    tc::CtlShared ctl;
    __device__ __forceinline__ void init(int consumers, int *fault) {
        for (int i = 0; i < STAGES; ++i) {
            tc::mbar_init(&full[i], 1);
            tc::mbar_init(&done[i], consumers);
            tc::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < FSTAGES; ++i) tc::mbar_init(&f_empty[i], consumers);
        tc::init_ctl(ctl, fault);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // One thread: take tiles in the counter's order and start their copies.
    template <int V, typename Copy>
    __device__ __forceinline__ void produce(const ScanParams &p, int tiles, int ends, const tc::Ctl &c, Copy copy) {
        uint32_t n = 0;
        for (;; ++n) {
            const int s = n % STAGES;
            if (!tc::mbar_wait(&empty[s], ((n / STAGES) & 1) ^ 1, c, FAULT_CODE + 1)) break;
            const int t = p.chunks > 1 ? atomicAdd(p.counter, 1) + 1 : (int)(blockIdx.x + n * gridDim.x);
            if (t >= tiles) {  // an end for every group; the workers wait for every copy before they see one
                tile[s].chunk = -1;
                tc::mbar_arrive(&full[s]);
                if (--ends == 0) return;
                continue;
            }
            int fs = 0;
            if constexpr (FSTAGES > 0) {
                fs = n % FSTAGES;
                if (!tc::mbar_wait(&f_empty[fs], ((n / FSTAGES) & 1) ^ 1, c, FAULT_CODE + 1)) break;
            }
            tile[s] = tile_of<V>(p, t, 0);
            copy(s, fs, tile[s]);
        }
        // gave up: do not leave with copies in flight
        for (uint32_t i = n > STAGES ? n - STAGES : 0; i < n; ++i) {
            const unsigned long long w0 = tc::gtimer();
            while (!tc::mbar_try(&full[i % STAGES], (i / STAGES) & 1) && tc::gtimer() - w0 < tc::WAIT_NS) {
            }
        }
    }
    // One thread: store finished tiles and free their stages.
    template <typename Store> __device__ __forceinline__ void retire(int ends, const tc::Ctl &c, Store store) {
        for (uint32_t n = 0;; ++n) {
            const int s = n % STAGES;
            if (!tc::mbar_wait(&done[s], (n / STAGES) & 1, c, FAULT_CODE + 2)) break;
            if (tile[s].chunk < 0) {
                if (--ends == 0) break;
            } else {
                store(s, tile[s]);
                tc::bulk_commit();
                tc::bulk_wait_read();
            }
            tc::mbar_arrive(&empty[s]);
        }
        tc::bulk_wait_all();
    }
};

template <typename T, bool GATE, bool CUT>
__global__ void __launch_bounds__(FwdCfg<T, GATE>::THREADS, 1)
    scan_forward_tma(const __grid_constant__ ScanMaps maps, const ScanParams p, int tiles) {
    using G = FwdCfg<T, GATE>;
    constexpr int W = G::W, R = G::R, V = G::V;
    extern __shared__ uint8_t raw[];
    uint8_t *smem = raw + ((128u - (tc::su32(raw) & 127u)) & 127u), *f_tiles = smem + G::STAGES * G::STAGE;
    __shared__ Scratch<V> scratch[G::GROUPS];
    __shared__ Part<V> s_parts[G::GROUPS][W][32];
    __shared__ bool s_cut[G::GROUPS][W];
    __shared__ Ring<G::FSTAGES, G::STAGES> ring;
    if (test_expired(p)) return;
    const int lane = threadIdx.x & 31, group = threadIdx.x / (W * 32), warp = (threadIdx.x >> 5) & (W - 1);
    if (threadIdx.x == 0) ring.init(W * 32, p.fault);
    __syncthreads();
    const tc::Ctl ctl{&ring.ctl, nullptr};

    if (group == G::GROUPS) {
        if (warp == 0 && lane == 0)
            ring.template produce<V>(p, tiles, G::GROUPS, ctl, [&](int s, int fs, const Tile &k) {
                uint8_t *d = smem + s * G::STAGE;
                tc::mbar_expect_tx(&ring.full[s], G::STAGE + G::TILE);
                tma_load3(f_tiles + fs * G::TILE, &maps.f, &ring.full[s], k.c, k.chunk * SCAN_ROWS, k.b);
                tma_load3(d, &maps.x, &ring.full[s], k.c, k.chunk * SCAN_ROWS, k.b);
                if (GATE) tma_load3(d + G::TILE, &maps.gate, &ring.full[s], k.c, k.chunk * SCAN_ROWS, k.b);
            });
        if (warp == 1 && lane == 0)
            ring.retire(G::GROUPS, ctl, [&](int s, const Tile &k) {
                tma_store3(&maps.y, smem + s * G::STAGE, k.c, k.chunk * SCAN_ROWS, k.b);
            });
    } else {
        Scratch<V> &sm = scratch[group];
        Part<V>(&parts)[W][32] = s_parts[group];
        auto sync = [&] { tc::named_bar(1 + group, W * 32); };
        for (uint32_t n = group;; n += G::GROUPS) {
            const int s = n % G::STAGES;
            if (!tc::mbar_wait(&ring.full[s], (n / G::STAGES) & 1, ctl, FAULT_CODE + 3)) break;
            Tile k = ring.tile[s];
            if (k.chunk < 0) {
                tc::mbar_arrive(&ring.done[s]);
                break;
            }
            k.c += lane * V;
            k.word0 += lane * V;
            const bool live = k.c < p.C;
            const int l0 = k.chunk * SCAN_ROWS + warp * R, rows = p.L - l0;
            uint8_t *xs = smem + s * G::STAGE + warp * R * 128 + lane * 4;
            const uint8_t *os = xs + G::TILE;
            const uint8_t *fs = f_tiles + (n % G::FSTAGES) * G::TILE + warp * R * 128 + lane * 4;
            const uint32_t cuts = CUT ? reset_mask(p, k.b, l0, R, lane) : 0;
            const Vf<V> bias = gather<V>([&](int v) { return live && p.bias ? __ldg(p.bias + k.c + v) * LOG2E : 0.f; });
            Vf<V> z[R];
#pragma unroll
            for (int r = 0; r < R; ++r) z[r] = sigmoid_neg2(fma(Word<T>::get(fs + r * 128), Vf<V>::all(LOG2E), bias));
            tc::mbar_arrive_after_reads(&ring.f_empty[n % G::FSTAGES]);
            if (rows < R) {
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (r >= rows) z[r] = Vf<V>::all(0.f);
            }
            {
                Vf<V> q = Vf<V>::all(0.f), h = q, left = Vf<V>::all(1.f);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (CUT && (cuts >> r & 1)) h = Vf<V>::all(0.f);
                    const Vf<V> a = fma(z[r], Vf<V>::all(-1.f), Vf<V>::all(1.f));
                    h = fma(a, h, mul(z[r], Word<T>::get(xs + r * 128)));
                    q = fma(z[r], left, q);
                    left = mul(left, a);
                }
                parts[warp][lane] = part_of(left, q, h);
                if (CUT) s_cut[group][warp] = cuts != 0;
            }
            sync();
            Part<V> part = no_part<V>();
            const int upto = warp ? warp : W;
            const uint32_t cut = CUT ? which_cut<W>(s_cut[group], lane) & ((1u << upto) - 1u) : 0;
#pragma unroll 1
            for (int w = 0; w < upto; ++w) {
                part = join_part(part, parts[w][lane]);
                if (CUT && (cut >> w & 1)) part.h = parts[w][lane].h;
            }
            const Run<V> run = run_of(part, cut);
            sync();
            const Vf<V> in = chain<CUT, V, W>(
                p, k, run, sm, warp, lane, live, sync,
                [&](int v) { return p.h0 ? p.h0[(int64_t)k.b * p.C + k.c + v] : 0.f; },
                [&](Vf<V> out) {
                    if (p.h_last) {
#pragma unroll
                        for (int v = 0; v < V; ++v) p.h_last[(int64_t)k.b * p.C + k.c + v] = out.at(v);
                    }
                });
            Vf<V> h = warp ? join<CUT>(in, run) : in;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (CUT && (cuts >> r & 1)) h = Vf<V>::all(0.f);
                h = advance(h, z[r], Word<T>::get(xs + r * 128));
                Vf<V> y = h;
                if constexpr (GATE) {
                    const Vf<V> g = Word<T>::get(os + r * 128);
                    y = mul(y, mul(g, sigmoid(g)));
                }
                Word<T>::put(xs + r * 128, y);  // rows past the end are not stored
            }
            tc::mbar_arrive_after_reads(&ring.done[s]);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) tc::report_fault(ring.ctl.abort_flag, p.fault);
}

// ------------------------------------------------------------------ backward, tiles moved by TMA
// As the forward kernel, from the last tile to the first: x, f, dy and the gate in, and the gradients
// out where x, f and the gate lay.  A thread keeps, of its 16 rows, the runs before every fourth one; z,
// the states and the gate's sigmoid are computed again, four rows at a time, which costs less than the
// registers that would hold them.  8 x 4096 tokens x 768 channels, bf16, gated: 99 us, 3.6 TB/s, issue
// slots 54 % (the kernel above: 189 us).
struct ScanBackMaps {
    CUtensorMap x, f, gate, dy, dx, df, dgate;
};

template <typename T, bool GATE> struct BwdCfg {
    static constexpr int GROUPS = 2, W = 8, R = SCAN_ROWS / W, V = sizeof(T) == 2 ? 2 : 1;
    static constexpr int TILE = SCAN_ROWS * 128, STAGE = (GATE ? 4 : 3) * TILE;
    static constexpr int STAGES = GATE ? 3 : 4, SMEM = STAGES * STAGE + 128;
    static constexpr int THREADS = (GROUPS * W + 2) * 32;
};

template <typename T, bool GATE, bool CUT>
__global__ void __launch_bounds__(BwdCfg<T, GATE>::THREADS, 1)
    scan_backward_tma(const __grid_constant__ ScanBackMaps maps, const ScanParams p, int tiles) {
    using G = BwdCfg<T, GATE>;
    constexpr int W = G::W, R = G::R, V = G::V;
    extern __shared__ uint8_t raw[];
    uint8_t *smem = raw + ((128u - (tc::su32(raw) & 127u)) & 127u);
    __shared__ Scratch<V> scratch[G::GROUPS];
    __shared__ Part<V> s_parts[G::GROUPS][W][32];
    __shared__ Vf<V> s_carries[G::GROUPS][W][32];  // the parts' H in the carries' direction
    __shared__ bool s_cut[G::GROUPS][W];
    __shared__ Ring<0, G::STAGES> ring;
    if (test_expired(p)) return;
    const int lane = threadIdx.x & 31, group = threadIdx.x / (W * 32), warp = (threadIdx.x >> 5) & (W - 1);
    if (threadIdx.x == 0) ring.init(W * 32, p.fault);
    __syncthreads();
    const tc::Ctl ctl{&ring.ctl, nullptr};

    if (group == G::GROUPS) {
        if (warp == 0 && lane == 0)
            ring.template produce<V>(p, tiles, G::GROUPS, ctl, [&](int s, int, const Tile &k) {
                uint8_t *d = smem + s * G::STAGE;
                const int l = (p.chunks - 1 - k.chunk) * SCAN_ROWS;
                tc::mbar_expect_tx(&ring.full[s], G::STAGE);
                tma_load3(d + G::TILE, &maps.f, &ring.full[s], k.c, l, k.b);
                tma_load3(d, &maps.x, &ring.full[s], k.c, l, k.b);
                tma_load3(d + 2 * G::TILE, &maps.dy, &ring.full[s], k.c, l, k.b);
                if (GATE) tma_load3(d + 3 * G::TILE, &maps.gate, &ring.full[s], k.c, l, k.b);
            });
        if (warp == 1 && lane == 0)
            ring.retire(G::GROUPS, ctl, [&](int s, const Tile &k) {
                const uint8_t *d = smem + s * G::STAGE;
                const int l = (p.chunks - 1 - k.chunk) * SCAN_ROWS;
                tma_store3(&maps.dx, d, k.c, l, k.b);
                tma_store3(&maps.df, d + G::TILE, k.c, l, k.b);
                if (GATE) tma_store3(&maps.dgate, d + 3 * G::TILE, k.c, l, k.b);
            });
    } else {
        Scratch<V> &sm = scratch[group];
        Part<V>(&parts)[W][32] = s_parts[group];
        Vf<V>(&carries)[W][32] = s_carries[group];
        auto sync = [&] { tc::named_bar(1 + group, W * 32); };
        const Vf<V> one = Vf<V>::all(1.f), neg = Vf<V>::all(-1.f), none = Vf<V>::all(0.f);
        for (uint32_t n = group;; n += G::GROUPS) {
            const int s = n % G::STAGES;
            if (!tc::mbar_wait(&ring.full[s], (n / G::STAGES) & 1, ctl, FAULT_CODE + 3)) break;
            Tile k = ring.tile[s];
            if (k.chunk < 0) {
                tc::mbar_arrive(&ring.done[s]);
                break;
            }
            k.c += lane * V;
            k.word0 += lane * V;
            const bool live = k.c < p.C;
            const int chunk = p.chunks - 1 - k.chunk, l0 = chunk * SCAN_ROWS + warp * R, rows = p.L - l0;
            uint8_t *xs = smem + s * G::STAGE + warp * R * 128 + lane * 4, *fs = xs + G::TILE, *os = xs + 3 * G::TILE;
            const uint8_t *ds = xs + 2 * G::TILE;
            const uint32_t cuts = CUT ? reset_mask(p, k.b, l0, R, lane) : 0;
            const Vf<V> bias = gather<V>([&](int v) { return live && p.bias ? __ldg(p.bias + k.c + v) * LOG2E : 0.f; });
            Vf<V> start = gather<V>([&](int v) {
                if (!live) return 0.f;
                if (chunk > 0) return __uint_as_float(p.states[k.word0 + (int64_t)(chunk - 1) * p.C + v]);
                return p.h0 ? p.h0[(int64_t)k.b * p.C + k.c + v] : 0.f;
            });
            // 2^u of a row, with z of rows past the end zero
            auto power = [&](int r) { return each(fma(Word<T>::get(fs + r * 128), Vf<V>::all(LOG2E), bias), ex2_sat); };
            auto z_of = [&](int r, Vf<V> e) { return r < rows ? each(add(e, one), rcp) : none; };
            // dL/dh_t through y_t; past the end dy was filled with zeros
            auto into = [&](int r) {
                Vf<V> v = Word<T>::get(ds + r * 128);
                if constexpr (GATE) {
                    const Vf<V> o = Word<T>::get(os + r * 128);
                    v = mul(v, mul(o, sigmoid(o)));
                }
                return v;
            };
            auto carry = [&](int r, Vf<V> z, Vf<V> g) {  // a g of one token
                if (CUT && (cuts >> r & 1)) return none;
                return fma(mul(z, neg), g, g);
            };
            Run<V> every[R / 4];  // the run of the rows before every fourth one
            {
                Vf<V> q = none, h = none, left = one, cc = none, z[R];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (r % 4 == 0) every[r / 4] = coded(left, q, h);
                    z[r] = z_of(r, power(r));
                    if (CUT && (cuts >> r & 1)) h = none;
                    const Vf<V> a = fma(z[r], neg, one);
                    h = fma(a, h, mul(z[r], Word<T>::get(xs + r * 128)));
                    q = fma(z[r], left, q);
                    left = mul(left, a);
                }
#pragma unroll
                for (int r = R - 1; r >= 0; --r) cc = carry(r, z[r], add(into(r), cc));
                parts[warp][lane] = part_of(left, q, h);
                carries[warp][lane] = cc;
                if (CUT) s_cut[group][warp] = cuts != 0;
            }
            sync();
            // the carries of the rows right of this warp's; the last warp, which has none, joins the tile's
            Part<V> part = no_part<V>();
            const int mine = W - 1 - warp, upto = mine ? mine : W;
            auto carried = [&](int w) { return Part<V>{parts[w][lane].p, parts[w][lane].e, carries[w][lane]}; };
            uint32_t cut = CUT ? which_cut<W>(s_cut[group], lane) : 0;
            {
#pragma unroll 1
                for (int i = 0; i < upto; ++i) {
                    part = join_part(part, carried(W - 1 - i));
                    if (CUT && (cut >> (W - 1 - i) & 1)) part.h = carries[W - 1 - i][lane];
                }
#pragma unroll 1
                for (int w = 0; w < warp; ++w) start = CUT && (cut >> w & 1) ? parts[w][lane].h : join_part(start, parts[w][lane]);
                cut >>= W - upto;  // those that were joined to `part`
            }
            const Run<V> run = run_of(part, cut);
            sync();
            // in walking order the last warp is the first one
            const Vf<V> in = chain<CUT, V, W>(
                p, k, run, sm, W - 1 - warp, lane, live, sync,
                [&](int v) { return p.dh_last ? p.dh_last[(int64_t)k.b * p.C + k.c + v] : 0.f; },
                [&](Vf<V> out) {
                    if (p.dh0) {
#pragma unroll
                        for (int v = 0; v < V; ++v) p.dh0[(int64_t)k.b * p.C + k.c + v] = out.at(v);
                    }
                });
            Vf<V> cc = warp == W - 1 ? in : cut ? part.h : join_part(in, part), db = none;
#pragma unroll
            for (int r0 = R - 4; r0 >= 0; r0 -= 4) {
                Vf<V> prev[4], z[4], e[4], h = start;
                if (r0) h = CUT && (cuts & ((1u << r0) - 1u)) ? every[r0 / 4].h : join<false>(start, every[r0 / 4]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[i] = power(r0 + i);
                    z[i] = z_of(r0 + i, e[i]);
                    if (CUT && (cuts >> (r0 + i) & 1)) h = none;
                    prev[i] = h;
                    if (i < 3) h = advance(h, z[i], Word<T>::get(xs + (r0 + i) * 128));
                }
#pragma unroll
                for (int i = 3; i >= 0; --i) {
                    const int r = r0 + i;
                    const Vf<V> x = Word<T>::get(xs + r * 128), dy = Word<T>::get(ds + r * 128);
                    Vf<V> g = dy;
                    if constexpr (GATE) {
                        const Vf<V> o = Word<T>::get(os + r * 128), sg = sigmoid(o);
                        g = mul(dy, mul(o, sg));
                        // silu'(o) = sigmoid(o) (1 + o (1 - sigmoid(o)))
                        const Vf<V> slope = mul(sg, fma(o, fma(sg, neg, one), one));
                        Word<T>::put(os + r * 128, mul(mul(dy, advance(prev[i], z[i], x)), slope));
                    }
                    g = add(g, cc);
                    const Vf<V> dx = mul(z[i], g);
                    cc = carry(r, z[i], g);
                    // a = exp(u) sigmoid(-u): 1 - z would lose a small a
                    const Vf<V> df = mul(mul(dx, mul(e[i], z[i])), fma(x, neg, prev[i]));
                    db = add(db, df);
                    Word<T>::put(xs + r * 128, dx);
                    Word<T>::put(fs + r * 128, df);
                }
            }
            tc::mbar_arrive_after_reads(&ring.done[s]);
            if (p.dbias_part) {
                // the look-back's place: it is read before the chain's last barrier, and next written
                // after two of the next tile's
                sm.run[warp][lane].h = db;
                sync();
                if (warp == 0 && live) {
                    Vf<V> t = none;
#pragma unroll
                    for (int w = 0; w < W; ++w) t = add(t, sm.run[w][lane].h);
#pragma unroll
                    for (int v = 0; v < V; ++v)
                        p.dbias_part[((int64_t)k.b * p.chunks + chunk) * p.C + k.c + v] = t.at(v);
                }
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) tc::report_fault(ring.ctl.abort_flag, p.fault);
}

// (a few us; its reads are 1/128 of the backward pass's)
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
// One pass over x, f, gate and the state.  64 x 768: 1.9 us, a launch's time.
template <typename T, int V>
__global__ void __launch_bounds__(128) scan_step(const ScanStepParams p) {
    const int per = p.C / V;
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
    x.load(static_cast<const T *>(p.x.p) + n * p.x.sb + c);
    f.load(static_cast<const T *>(p.f.p) + n * p.f.sb + c);
    if (p.gate.p) o.load(static_cast<const T *>(p.gate.p) + n * p.gate.sb + c);
    Vf<V> y = Vf<V>::all(0.f);
    if (held) {
        const Vf<V> bias = gather<V>([&](int v) { return p.bias ? __ldg(p.bias + c + v) * LOG2E : 0.f; });
        Vf<V> h = gather<V>([&](int v) { return p.h_in[row * p.C + c + v]; });
        h = advance(h, sigmoid_neg2(fma(f.f(), Vf<V>::all(LOG2E), bias)), x.f());
#pragma unroll
        for (int v = 0; v < V; ++v) p.h_out[row * p.C + c + v] = h.at(v);
        y = p.gate.p ? mul(h, mul(o.f(), sigmoid(o.f()))) : h;
    }
    Pack<T, V>::store(static_cast<T *>(p.y.p) + n * p.y.sb + c, y);
}

// bf16 pairs need an even channel count and even strides on 4-byte boundaries; one channel a lane
// otherwise (half the bytes a warp moves per row: 64 instead of 128).
bool pairs(const Blc &t) {
    return !t.p || (reinterpret_cast<uintptr_t>(t.p) % 4 == 0 && t.sb % 2 == 0 && t.sl % 2 == 0);
}

template <auto Kernel> cudaError_t launch_cluster(const ScanParams &p, int tiles, int threads, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)tiles);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)p.chunks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, Kernel, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

// TMA rows: 16-byte starts and strides, and strides that are not 0 (a broadcast axis).
bool boxes(const Blc &t, int B, int L, int es) {
    return !t.p || (reinterpret_cast<uintptr_t>(t.p) % 16 == 0 && (L == 1 || (t.sl > 0 && t.sl * es % 16 == 0)) &&
                    (B == 1 || (t.sb > 0 && t.sb * es % 16 == 0)));
}

template <typename T, bool GATE, bool CUT> cudaError_t forward_tma_v(const ScanMaps &maps, const ScanParams &p, int tiles, int grid, cudaStream_t st) {
    using G = FwdCfg<T, GATE>;
    cudaError_t e = set_smem_once<scan_forward_tma<T, GATE, CUT>>(G::SMEM);
    if (e != cudaSuccess) return e;
    scan_forward_tma<T, GATE, CUT><<<grid, G::THREADS, G::SMEM, st>>>(maps, p, tiles);
    return cudaGetLastError();
}

template <typename T> cudaError_t forward_tma(ScanParams p, int sms, cudaStream_t st) {
    constexpr int V = sizeof(T) == 2 ? 2 : 1;
    p.ctiles = (p.C + 32 * V - 1) / (32 * V);
    const int64_t tiles = (int64_t)p.chunks * p.B * p.ctiles;
    if (tiles > 0x3fffffff) return cudaErrorInvalidValue;
    ScanMaps m;
    if (!tc::make_blc_map(&m.x, p.x.p, p.x.sb, p.x.sl, p.B, p.L, p.C, sizeof(T), SCAN_ROWS) ||
        !tc::make_blc_map(&m.f, p.f.p, p.f.sb, p.f.sl, p.B, p.L, p.C, sizeof(T), SCAN_ROWS) ||
        !tc::make_blc_map(&m.y, p.y.p, p.y.sb, p.y.sl, p.B, p.L, p.C, sizeof(T), SCAN_ROWS))
        return cudaErrorInvalidValue;
    if (p.gate.p && !tc::make_blc_map(&m.gate, p.gate.p, p.gate.sb, p.gate.sl, p.B, p.L, p.C, sizeof(T), SCAN_ROWS))
        return cudaErrorInvalidValue;
    const int grid = (int)(tiles < sms ? tiles : sms);
    if (p.gate.p)
        return p.reset ? forward_tma_v<T, true, true>(m, p, (int)tiles, grid, st)
                       : forward_tma_v<T, true, false>(m, p, (int)tiles, grid, st);
    return p.reset ? forward_tma_v<T, false, true>(m, p, (int)tiles, grid, st)
                   : forward_tma_v<T, false, false>(m, p, (int)tiles, grid, st);
}

template <typename T, bool GATE, bool CUT>
cudaError_t backward_tma_v(const ScanBackMaps &maps, const ScanParams &p, int tiles, int grid, cudaStream_t st) {
    using G = BwdCfg<T, GATE>;
    cudaError_t e = set_smem_once<scan_backward_tma<T, GATE, CUT>>(G::SMEM);
    if (e != cudaSuccess) return e;
    scan_backward_tma<T, GATE, CUT><<<grid, G::THREADS, G::SMEM, st>>>(maps, p, tiles);
    return cudaGetLastError();
}

template <typename T> cudaError_t backward_tma(ScanParams p, int sms, cudaStream_t st) {
    constexpr int V = sizeof(T) == 2 ? 2 : 1;
    p.ctiles = (p.C + 32 * V - 1) / (32 * V);
    const int64_t tiles = (int64_t)p.chunks * p.B * p.ctiles;
    if (tiles > 0x3fffffff) return cudaErrorInvalidValue;
    ScanBackMaps m;
    const Blc *from[7] = {&p.x, &p.f, &p.gate, &p.dy, &p.dx, &p.df, &p.dgate};
    CUtensorMap *to[7] = {&m.x, &m.f, &m.gate, &m.dy, &m.dx, &m.df, &m.dgate};
    for (int i = 0; i < 7; ++i)
        if (from[i]->p && !tc::make_blc_map(to[i], from[i]->p, from[i]->sb, from[i]->sl, p.B, p.L, p.C, sizeof(T), SCAN_ROWS))
            return cudaErrorInvalidValue;
    const int grid = (int)(tiles < sms ? tiles : sms);
    if (p.gate.p)
        return p.reset ? backward_tma_v<T, true, true>(m, p, (int)tiles, grid, st)
                       : backward_tma_v<T, true, false>(m, p, (int)tiles, grid, st);
    return p.reset ? backward_tma_v<T, false, true>(m, p, (int)tiles, grid, st)
                   : backward_tma_v<T, false, false>(m, p, (int)tiles, grid, st);
}

template <typename T, int V, bool GATE, bool CUT> cudaError_t forward_v(const ScanParams &p, int tiles, bool cluster, cudaStream_t st) {
    if (cluster) return launch_cluster<scan_forward<T, V, 8, 16, GATE, CUT, true>>(p, tiles, 256, st);
    scan_forward<T, V, 8, 16, GATE, CUT, false><<<(unsigned)tiles, 256, 0, st>>>(p);
    return cudaGetLastError();
}

template <typename T, int V> cudaError_t forward_t(ScanParams p, bool cluster, cudaStream_t st) {
    p.ctiles = (p.C + 32 * V - 1) / (32 * V);
    const int64_t tiles = (int64_t)p.chunks * p.B * p.ctiles;
    if (tiles > 0x7fffffff) return cudaErrorInvalidValue;
    if (p.gate.p)
        return p.reset ? forward_v<T, V, true, true>(p, (int)tiles, cluster, st) : forward_v<T, V, true, false>(p, (int)tiles, cluster, st);
    return p.reset ? forward_v<T, V, false, true>(p, (int)tiles, cluster, st) : forward_v<T, V, false, false>(p, (int)tiles, cluster, st);
}

template <typename T, int V, bool GATE, bool CUT> cudaError_t backward_v(const ScanParams &p, int tiles, bool cluster, cudaStream_t st) {
    if (cluster) return launch_cluster<scan_backward<T, V, 16, 8, GATE, CUT, true>>(p, tiles, 512, st);
    scan_backward<T, V, 16, 8, GATE, CUT, false><<<(unsigned)tiles, 512, 0, st>>>(p);
    return cudaGetLastError();
}

template <typename T, int V> cudaError_t backward_t(ScanParams p, bool cluster, cudaStream_t st) {
    p.ctiles = (p.C + 32 * V - 1) / (32 * V);
    const int64_t tiles = (int64_t)p.chunks * p.B * p.ctiles;
    if (tiles > 0x7fffffff) return cudaErrorInvalidValue;
    if (p.gate.p)
        return p.reset ? backward_v<T, V, true, true>(p, (int)tiles, cluster, st) : backward_v<T, V, true, false>(p, (int)tiles, cluster, st);
    return p.reset ? backward_v<T, V, false, true>(p, (int)tiles, cluster, st) : backward_v<T, V, false, false>(p, (int)tiles, cluster, st);
}

}  // namespace

// Sequences of 2 to 8 tiles while the tiles fit the GPU at once: a cluster a sequence, in one launch and
// without words to set up (301 tokens of 768 channels: 5.9 against 9.1 us).  More tiles: TMA.
bool scan_by_cluster(int B, int L, int C, int dtype, int sms) {
    const int chunks = scan_chunks(L);
    const int64_t cols = (int64_t)B * ((C + 31) / 32);  // at most, whatever the vector width
    return chunks > 1 && chunks <= 8 && chunks * cols <= (dtype == PMA_F32 ? 2 : 4) * (int64_t)sms;
}

cudaError_t launch_gated_scan(ScanParams p, int dtype, int sms, cudaStream_t st) {
    const int es = dtype == PMA_F32 ? 4 : 2;
    const bool cluster = scan_by_cluster(p.B, p.L, p.C, dtype, sms);
    if (!cluster && tc::tensor_maps_available() && p.C * es % 4 == 0 && boxes(p.x, p.B, p.L, es) &&
        boxes(p.f, p.B, p.L, es) && boxes(p.gate, p.B, p.L, es) && boxes(p.y, p.B, p.L, es))
        return dtype == PMA_F32 ? forward_tma<float>(p, sms, st) : forward_tma<__nv_bfloat16>(p, sms, st);
    if (dtype == PMA_F32) return forward_t<float, 1>(p, cluster, st);
    if (p.C % 2 == 0 && pairs(p.x) && pairs(p.f) && pairs(p.gate) && pairs(p.y))
        return forward_t<__nv_bfloat16, 2>(p, cluster, st);
    return forward_t<__nv_bfloat16, 1>(p, cluster, st);
}

cudaError_t launch_gated_scan_backward(ScanParams p, int dtype, float *dbias, int sms, cudaStream_t st) {
    cudaError_t e;
    const int es = dtype == PMA_F32 ? 4 : 2;
    const bool cluster = scan_by_cluster(p.B, p.L, p.C, dtype, sms);
    bool tma = !cluster && tc::tensor_maps_available() && p.C * es % 4 == 0;
    bool two = dtype == PMA_BF16 && p.C % 2 == 0;
    for (const Blc *t : {&p.x, &p.f, &p.gate, &p.dy, &p.dx, &p.df, &p.dgate}) {
        tma = tma && boxes(*t, p.B, p.L, es);
        two = two && pairs(*t);
    }
    if (tma)
        e = dtype == PMA_F32 ? backward_tma<float>(p, sms, st) : backward_tma<__nv_bfloat16>(p, sms, st);
    else if (dtype == PMA_F32)
        e = backward_t<float, 1>(p, cluster, st);
    else
        e = two ? backward_t<__nv_bfloat16, 2>(p, cluster, st) : backward_t<__nv_bfloat16, 1>(p, cluster, st);
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
