// sampling.cu -- one token per row of logits: temperature, top-k, top-p, min-p, and the inverse
// transform of one given uniform number.
//
//   z_i = (x_i - max x) / T        w_i = round(exp(z_i) 2^32), a whole number
//   order the tokens by (x descending, index ascending); a filter keeps a prefix of that order:
//     top-k   the first k
//     top-p   rank r while the weight of the ranks before it is below p times the top-k's weight
//     min-p   exp(z) >= min_p
//   token = the first kept i, by index, whose cumulated kept weight exceeds u times their total
//   logprob = z_token - log(sum of all w / 2^32)
//
// Weights are whole numbers so that every sum is exact: no result depends on the order of an
// addition, on atomics or on how a row is split, and two rows with the same logits and u get the
// same token in any batch.  (A token below 2^-33 of the most likely one has weight 0.)
//
// A cluster of 1 to 8 CTAs holds one row in shared memory, read from HBM once.  Nothing is
// sorted.  A cut of the order is a logit and how many of its equals are kept; it is found by
// histograms: first over z (512 bins), then, inside the bin that holds the cut, over the logits'
// ordered bits until a bin is one value.  Only tokens that can be near a cut enter a histogram:
//     top-k   with G >= k disjoint groups of tokens, the smallest of the groups' maxima is at most
//             the k-th largest logit (the groups are fixed lanes, so this comes with the maximum)
//     top-p   the tokens below z weigh less than V exp(z): those with V exp(z) <= (1 - p) W are cut;
//             the weight below two values of z is measured with W itself
// The kept weights are then summed by ranges of consecutive tokens, one a warp; the warp whose
// range holds the goal walks it.  Where the candidates of a row are few, the cluster's first CTA goes on
// with them alone.
//
// 256 x 131072 bf16 take 61 us without filters, 106 with top-p 0.95 (a language model's rows), of 10.3 that
// the bytes need.  No pipe is full: the 25 instructions a logit for its weight are 23 us of issue; the rest is the
// other passes over the row, the phases' barriers and a last wave of CTAs that is half empty.  A small
// batch is bound by the latency of its phases: a row of 32000 with top-k 50 takes 14.4 us.
#include <cooperative_groups.h>

#include "sampling.cuh"

namespace cg = cooperative_groups;

namespace pma {
namespace {

constexpr int NW = 16;       // warps of a CTA
constexpr int NB = NW * 32;  // histogram bins: one a thread
constexpr int LIST = 192;    // candidates a warp keeps
constexpr int FEW = 32;      // and how many of them one CTA may take over
constexpr int MAXC = 8;      // CTAs of a cluster
constexpr float ZMIN = -23.0f;  // exp(-23) 2^32 < 1/2: weight 0 below
constexpr float ZCUT0 = -4.5f, ZCUT1 = -9.0f;  // where the tail's weight is measured
constexpr unsigned long long ONE = 1ull << 32;

struct Found {
    int bin;                       // -1: the goal lies past the last bin
    uint32_t count;                // tokens before the bin
    unsigned long long weight;     // their weight
};

// A thread's bin of the row's histogram (its CTA's slice of it), and what lies before it in the slice.
struct Bin {
    uint32_t count, before;
    unsigned long long weight, before_weight;
};

struct Shared {
    uint32_t cnt[NB], lo[NB], hi[NB];  // this CTA's histogram (weights as two 32-bit halves)
    // written by the CTAs of the cluster, one slot each
    float x_max[MAXC], x_bound[MAXC];
    unsigned long long x_sum[MAXC], x_below[2][MAXC];
    uint32_t x_klo[MAXC], x_khi[MAXC];
    uint32_t x_cnt[MAXC];
    unsigned long long x_w[MAXC];
    Found found;
    int listed[MAXC * NW];             // length of every warp's list (-1: it does not fit)
    uint16_t list_at[NW][LIST];        // where the listed logits lie in their warp's range
    uint16_t few_at[MAXC * NW][FEW];   // the row's candidates, where they are few: FEW places a warp
    // per warp
    float w_max[NW], w_bound[NW];
    unsigned long long w_sum[NW];
    uint32_t b_cnt[NW];                // block scans
    unsigned long long b_w[NW], b_w2[NW];
    uint32_t w_klo[NW], w_khi[NW];
    unsigned long long f_gt[MAXC * NW];  // weight of the tokens before the cut in every warp's range
    uint32_t f_eq[MAXC * NW];            // tokens equal to it
    int owner;                         // warp of this CTA that holds the goal, or -1
    unsigned long long goal;           // goal left when its range starts
    uint32_t eq_left;                  // equals that may still be kept there
};

// A vector of VEC logits as loaded, and the largest of it without unpacking (NaN loses).
template <typename T> struct Row;
template <> struct Row<float> {
    static constexpr int VEC = 4;
    using Raw = float4;
    static __device__ __forceinline__ void get(const Raw &v, float (&x)[4]) { x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w; }
    static __device__ __forceinline__ Raw max(const Raw &a, const Raw &b) {
        return make_float4(fmaxf(a.x, b.x), fmaxf(a.y, b.y), fmaxf(a.z, b.z), fmaxf(a.w, b.w));
    }
    static __device__ __forceinline__ float max(const Raw &v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
    static __device__ __forceinline__ Raw none() { return make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); }
    static __device__ __forceinline__ float lowest() { return -INFINITY; }
    static __device__ __forceinline__ float one(float x) { return x; }
};
template <> struct Row<__nv_bfloat16> {
    static constexpr int VEC = 8;
    using Raw = uint4;
    static __device__ __forceinline__ void get(const Raw &v, float (&x)[8]) {
        const uint32_t a[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(a[i] << 16);
            x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ Raw max(const Raw &a, const Raw &b) {
        return make_uint4(max2(a.x, b.x), max2(a.y, b.y), max2(a.z, b.z), max2(a.w, b.w));
    }
    static __device__ __forceinline__ float max(const Raw &v) {
        const uint32_t m = max2(max2(v.x, v.y), max2(v.z, v.w));
        return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    }
    static __device__ __forceinline__ Raw none() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
    static __device__ __forceinline__ __nv_bfloat16 lowest() { return __ushort_as_bfloat16(0xff80); }
    static __device__ __forceinline__ float one(__nv_bfloat16 x) { return __bfloat162float(x); }
};

// Bits of x in an order that matches <, with -0 as +0.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __uint_as_float(k ^ ((k >> 31) - 1u | 0x80000000u));
}

// Keys: the ordered bits that a logit of this type can have.
template <typename T> __device__ __forceinline__ uint32_t key_of(float x) {
    return sizeof(T) == 2 ? ordered(x) >> 16 : ordered(x);
}
template <typename T> __device__ __forceinline__ float logit_of(uint32_t k) {
    // of a negative logit the ordered bits below bf16's are ones
    return unordered(sizeof(T) == 2 ? k << 16 | (k >> 15 ? 0u : 0xffffu) : k);
}

// z and weights of one row
struct Scale {
    float top, inv;
    bool inf_top;  // the largest logit is +inf: its equals share the row
    __device__ __forceinline__ float z(float x) const {
        if (inf_top) return x == top ? 0.f : -INFINITY;
        return __fmul_rn(__fsub_rn(x, top), inv);
    }
};
// round(e 2^32) for e in [0, 1]; the conversion saturates only at e = 1
__device__ __forceinline__ uint32_t weight32(float e) { return __float2uint_rn(__fmul_rn(e, 4294967296.0f)); }
__device__ __forceinline__ unsigned long long weight(float e) {
    const uint32_t w = weight32(e);
    return w == 0xffffffffu ? ONE : w;
}

__device__ __forceinline__ void add32(unsigned long long &a, uint32_t w) {
    asm("mad.wide.u32 %0, %1, 1, %0;" : "+l"(a) : "r"(w));
}

template <typename T> __device__ __forceinline__ T warp_add(T v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <typename T> __device__ __forceinline__ T warp_before(T v, int lane) {  // exclusive prefix sum
    T s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
    }
    return s - v;
}

// One row's CTA.
template <typename T> struct Sampler {
    static constexpr int VEC = Row<T>::VEC;
    Shared &s;
    const T *seg;       // NW * range tokens
    T *list;            // [NW][list_stride] this CTA's candidates, by index
    cg::cluster_group cl;
    int nc, rank, warp, lane, range;
    int listed;      // logits in this warp's list; -1: none made, or they do not fit
    float list_low;  // it holds those from here on
    int list_stride;
    uint32_t slice_count;  // this CTA's slice of the last merged histogram
    unsigned long long slice_weight;

    template <typename F> __device__ __forceinline__ void each(F f) const {
        const T *w = seg + warp * range;
        for (int i = lane * VEC; i < range; i += 32 * VEC) {
            float x[VEC];
            Row<T>::get(*reinterpret_cast<const typename Row<T>::Raw *>(w + i), x);
#pragma unroll
            for (int v = 0; v < VEC; ++v) f(x[v]);
        }
    }
    // Every logit through f, and those that are at least `low` (not -inf) into this warp's list:
    // what follows goes by the list, a candidate a lane, instead of through vectors with one in them.
    template <bool ALL, typename F> __device__ __forceinline__ void list_from(float low, T *few, F f) {
        const T *w = seg + warp * range;
        int n = 0;
        for (int i0 = 0; i0 < range; i0 += 32 * VEC) {
            const int i = i0 + lane * VEC;
            const typename Row<T>::Raw raw =
                i < range ? *reinterpret_cast<const typename Row<T>::Raw *>(w + i) : Row<T>::none();
            float x[VEC];
            if (ALL) {
                Row<T>::get(raw, x);
#pragma unroll
                for (int v = 0; v < VEC; ++v) f(x[v]);
            }
            if (n <= LIST && __any_sync(0xffffffffu, Row<T>::max(raw) >= low)) {
                if (!ALL) Row<T>::get(raw, x);
                // lanes hold neighbouring vectors: a candidate's place is behind those of the lanes before
                int at = n, all = 0;
                const uint32_t before = (1u << lane) - 1u;
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const uint32_t who = __ballot_sync(0xffffffffu, x[v] >= low);
                    at += __popc(who & before);
                    all += __popc(who);
                }
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    if (x[v] >= low && at < LIST) {
                        list[warp * LIST + at] = (T)x[v];
                        s.list_at[warp][at++] = (uint16_t)(i + v);
                    }
                n += all;
            }
        }
        __syncwarp();
        listed = n <= LIST ? n : -1;
        list_low = low;
        // to the first CTA of the cluster, should all lists be this short
        if (n <= FEW) {
            const int q = rank * NW + warp;
            Shared *o = cl.map_shared_rank(&s, 0);
            T *x = cl.map_shared_rank(few, 0);
            x[q * FEW + lane] = lane < n ? list[warp * LIST + lane] : Row<T>::lowest();
            if (lane < n) o->few_at[q][lane] = s.list_at[warp][lane];
        }
        if (lane < nc) cl.map_shared_rank(&s, lane)->listed[rank * NW + warp] = listed;
    }
    // A barrier of the row's CTAs.
    __device__ __forceinline__ void sync() const {
        if (nc == 1)
            __syncthreads();
        else
            cl.sync();
    }
    // The logits that are at least `low` and not masked, from the list where it has them all.
    template <typename F> __device__ __forceinline__ void each_from(float low, F f) const {
        if (listed >= 0 && low >= list_low) {
            const T *w = list + warp * list_stride;
#pragma unroll 1
            for (int i = lane; i < listed; i += 32) {
                const float x = Row<T>::one(w[i]);
                if (x >= low && x > -INFINITY) f(x);
            }
            return;
        }
        const T *w = seg + warp * range;
        for (int i = lane * VEC; i < range; i += 32 * VEC) {
            const typename Row<T>::Raw raw = *reinterpret_cast<const typename Row<T>::Raw *>(w + i);
            if (Row<T>::max(raw) >= low) {
                float x[VEC];
                Row<T>::get(raw, x);
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    if (x[v] >= low && x[v] > -INFINITY) f(x[v]);
            }
        }
    }

    __device__ __forceinline__ void clear() {
        for (int i = threadIdx.x; i < NB; i += NW * 32) s.cnt[i] = s.lo[i] = s.hi[i] = 0;
        __syncthreads();
    }
    __device__ __forceinline__ void count(int bin, uint32_t w32) {
        atomicAdd(&s.cnt[bin], 1u);
        if (w32) {
            const uint32_t old = atomicAdd(&s.lo[bin], w32);
            // 2^32 is held as 2^32 - 1 by the conversion: the one left over goes to the carry
            uint32_t up = old + w32 < old;
            if (w32 == 0xffffffffu) {
                const uint32_t o2 = atomicAdd(&s.lo[bin], 1u);
                up += o2 == 0xffffffffu;
            }
            if (up) atomicAdd(&s.hi[bin], up);
        }
    }
    // Sum the CTAs' histograms: this CTA takes the slice [rank, rank + 1) * NB / nc of the bins, a bin a
    // thread, and everybody gets the slices' totals.
    __device__ __forceinline__ Bin merge() {
        sync();
        const int per = NB / nc, t = threadIdx.x;
        Bin m{0, 0, 0, 0};
        if (t < per) {
            for (int r = 0; r < nc; ++r) {
                const Shared *o = cl.map_shared_rank(&s, r);
                const int at = rank * per + t;
                m.count += o->cnt[at];
                m.weight += ((unsigned long long)o->hi[at] << 32) + o->lo[at];
            }
        }
        m.before = warp_before(m.count, lane);
        m.before_weight = warp_before(m.weight, lane);
        if (lane == 31) {
            s.b_cnt[warp] = m.before + m.count;
            s.b_w[warp] = m.before_weight + m.weight;
        }
        __syncthreads();
        uint32_t c = 0;
        unsigned long long w = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            if (i == warp) {
                m.before += c;
                m.before_weight += w;
            }
            c += s.b_cnt[i];
            w += s.b_w[i];
        }
        totals(c, w);
        slice_count = c;
        slice_weight = w;
        return m;
    }
    __device__ __forceinline__ void totals(uint32_t c, unsigned long long w) {
        if (warp == 0 && lane < nc) {
            Shared *o = cl.map_shared_rank(&s, lane);
            o->x_cnt[rank] = c;
            o->x_w[rank] = w;
        }
        sync();
    }
    // The bin in which the tokens reach past `by_rank` tokens (or past the weight `goal`), given what
    // comes before the first bin.
    __device__ __forceinline__ Found find(const Bin &m, bool by_count, uint32_t by_rank, double goal, uint32_t c0,
                                          unsigned long long w0) {
        int owner = -1;
        uint32_t c = c0;
        unsigned long long w = w0;
        for (int r = 0; r < nc; ++r) {
            const uint32_t c2 = c + s.x_cnt[r];
            const unsigned long long w2 = w + s.x_w[r];
            if (by_count ? c2 > by_rank : !((double)w2 < goal)) {
                owner = r;
                break;
            }
            c = c2;
            w = w2;
        }
        if (owner == rank && (int)threadIdx.x < NB / nc) {
            c += m.before;
            w += m.before_weight;
            const bool here = by_count ? c <= by_rank && c + m.count > by_rank
                                       : m.count && (w == 0 || (double)w < goal) && !((double)(w + m.weight) < goal);
            if (here) {
                const Found f{(int)(rank * (NB / nc) + threadIdx.x), c, w};
                for (int r = 0; r < nc; ++r) cl.map_shared_rank(&s, r)->found = f;
            }
        }
        sync();
        return owner < 0 ? Found{-1, c, w} : s.found;
    }
};

struct Cut {
    uint32_t key;    // of the last kept logit; 0: keep all
    uint32_t keep;   // how many of its equals are kept
    unsigned long long before;  // weight before it
};

template <typename T>
__global__ void __launch_bounds__(NW * 32, 2) sample_kernel(const SampleParams p) {
    constexpr int VEC = Row<T>::VEC;
    extern __shared__ __align__(16) unsigned char raw[];
    Shared &s = *reinterpret_cast<Shared *>(raw);
    T *few = reinterpret_cast<T *>(raw + (sizeof(Shared) + 15) / 16 * 16), *list = few + MAXC * NW * FEW;
    T *seg = p.lists ? list + NW * LIST : few;
    const cg::cluster_group cl = cg::this_cluster();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA runs
    int nc = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int b = blockIdx.x / nc, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int range = p.range;
    Sampler<T> S{s, seg, list, cl, nc, rank, warp, lane, range, -1, 0.f, LIST, 0, 0};

    // ---- the row into shared memory, its maximum, and the top-k bound
    const int first = (rank * NW + warp) * range;  // this warp's tokens of the row
    const T *row = static_cast<const T *>(p.logits) + (int64_t)b * p.stride;
    const int n = max(0, min(range, p.V - first));
    float mx = -INFINITY;
    {
        T *w = seg + warp * range;
        const T *src = row + first;
        using Raw = typename Row<T>::Raw;
        if (reinterpret_cast<uintptr_t>(row) % 16 == 0) {  // ranges are whole vectors
            const int whole = n / VEC * VEC;
            Raw top = Row<T>::none();
#pragma unroll 4
            for (int i = lane * VEC; i < whole; i += 32 * VEC) {
                const Raw v = __ldcs(reinterpret_cast<const Raw *>(src + i));
                *reinterpret_cast<Raw *>(w + i) = v;
                top = Row<T>::max(top, v);
            }
            mx = Row<T>::max(top);
            for (int i = whole + lane; i < n; i += 32) {
                w[i] = src[i];
                mx = fmaxf(mx, Row<T>::one(src[i]));
            }
        } else {
            for (int i = lane; i < n; i += 32) {
                const T v = src[i];
                w[i] = v;
                mx = fmaxf(mx, Row<T>::one(v));
            }
        }
        for (int i = n + lane; i < range; i += 32) w[i] = Row<T>::lowest();
        __syncwarp();
    }
    const float temp = p.temperature.at(b);
    const bool greedy = !(temp > 0.f);
    const float top_p = p.top_p.at(b), min_p = p.min_p.at(b);
    int top_k = p.top_k.at(b);
    if (top_k <= 0 || top_k >= p.V) top_k = 0;
    // lanes of a group: as many as leave top_k groups
    int group = 32;
    while (group > 1 && nc * NW * 32 / group < top_k) group >>= 1;
    const bool bounded = top_k > 0 && nc * NW * 32 / group >= top_k;
    {
        float bound = mx;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, bound, o), m2 = __shfl_xor_sync(0xffffffffu, mx, o);
            bound = o < group ? fmaxf(bound, other) : fminf(bound, other);
            mx = fmaxf(mx, m2);
        }
        if (lane == 0) {
            s.w_max[warp] = mx;
            s.w_bound[warp] = bound;
        }
    }
    __syncthreads();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // all of them do: their memory may be written
    if (warp == 0) {
        mx = s.w_max[lane & (NW - 1)];
        float bound = s.w_bound[lane & (NW - 1)];
#pragma unroll
        for (int o = 1; o < NW; o <<= 1) {
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            bound = fminf(bound, __shfl_xor_sync(0xffffffffu, bound, o));
        }
        if (lane < nc) {
            Shared *o = cl.map_shared_rank(&s, lane);
            o->x_max[rank] = mx;
            o->x_bound[rank] = bound;
        }
    }
    cl.sync();
    float bound = INFINITY;
    mx = -INFINITY;
    for (int r = 0; r < nc; ++r) {
        mx = fmaxf(mx, s.x_max[r]);
        bound = fminf(bound, s.x_bound[r]);
    }
    if (mx == -INFINITY) {  // every token is masked (the same in every CTA of the cluster)
        if (rank == 0 && threadIdx.x == 0) {
            p.token[b] = -1;
            if (p.logprob) p.logprob[b] = -INFINITY;
        }
        return;
    }
    const Scale sc{mx, greedy ? 1.f : fminf(__frcp_rn(temp), 3.402823466e38f), mx == INFINITY};

    // ---- the weight of all tokens, and with top-k the list of those above its bound
    const bool only_first = greedy || !(top_p > 0.f) || !(min_p <= 1.f);
    const bool by_k = !only_first && top_k > 0, by_p = !only_first && top_p < 1.f;
    float low = by_k && bounded ? bound : -INFINITY;  // tokens below it are behind every cut
    float fine = 0.f;                                  // bins per unit of z
    auto set_bins = [&] {
        // farther tokens share the last bin
        fine = (float)NB / fminf(fmaxf(-sc.z(low), 1e-6f), -ZMIN);
    };
    auto bin_of = [&](float z) { return (int)fminf(-z * fine, (float)(NB - 1)); };
    unsigned long long total = 0;
    {
        uint32_t ones = 0;
        unsigned long long below[2] = {0, 0};
        auto add = [&](float x) {
            const uint32_t w = weight32(expf(sc.z(x)));  // NaN converts to 0
            add32(total, w);
            ones += w == 0xffffffffu;
        };
        if (low > -INFINITY && p.lists) {
            S.template list_from<true>(low, few, add);
        } else if (by_p && !by_k) {
            // also the weight below two values of z, for a bound on the nucleus
            S.each([&](float x) {
                const float z = sc.z(x);
                const uint32_t w = weight32(expf(z));
                ones += w == 0xffffffffu;
                if (z >= ZCUT0)
                    add32(total, w);
                else if (z >= ZCUT1)
                    add32(below[0], w);
                else
                    add32(below[1], w);
            });
            below[0] = warp_add(below[0] + below[1]);
            below[1] = warp_add(below[1]);
            if (lane == 0) {
                s.b_w[warp] = below[0];
                s.b_w2[warp] = below[1];
            }
        } else {
            S.each(add);
        }
        total = warp_add(total + ones) + below[0];
        if (lane == 0) s.w_sum[warp] = total;
        __syncthreads();
        if (warp == 0) {
            total = warp_add(lane < NW ? s.w_sum[lane] : 0ull);
            if (by_p && !by_k) {
                below[0] = warp_add(lane < NW ? s.b_w[lane] : 0ull);
                below[1] = warp_add(lane < NW ? s.b_w2[lane] : 0ull);
            }
            if (lane < nc) {
                Shared *o = cl.map_shared_rank(&s, lane);
                o->x_sum[rank] = total;
                o->x_below[0][rank] = below[0];
                o->x_below[1][rank] = below[1];
            }
        }
    }
    auto all_weight = [&] {  // after a cluster barrier
        unsigned long long t = 0;
        for (int r = 0; r < nc; ++r) t += s.x_sum[r];
        return t;
    };

    bool alone = false;  // only the candidates are left, in one CTA
    int row_ranges = 0;
    unsigned long long all_of_row = 0;

    // ---- the cut
    Cut cut{0, 0xffffffffu, 0};  // keeps every token
    if (only_first) {
        cut = Cut{key_of<T>(mx), 1, 0};
    } else if (by_k || by_p) {
        unsigned long long wk = 0;  // weight of the top-k tokens
        if (!by_k) {
            cl.sync();
            wk = all_weight();
            // weights are rounded up by at most 1/2 each; the margin covers the logarithm's error
            const float room = (1.f - top_p) * (float)wk * (1.f / 4294967296.f) / (float)p.V - 1.f / 8589934592.f;
            float zl = room > 0.f ? logf(room) - 0.02f : ZMIN;
            // or where the weight above is known to hold the nucleus
            unsigned long long tail[2] = {0, 0};
            for (int r = 0; r < nc; ++r) {
                tail[0] += s.x_below[0][r];
                tail[1] += s.x_below[1][r];
            }
            const double goal = (double)top_p * (double)wk;
            if (!((double)(wk - tail[1]) < goal)) zl = fmaxf(zl, ZCUT1 - 0.02f);
            if (!((double)(wk - tail[0]) < goal)) zl = fmaxf(zl, ZCUT0 - 0.02f);
            if (zl > ZMIN && !sc.inf_top) low = mx + zl / sc.inv - 4e-7f * fabsf(mx);
            if (low > -INFINITY && p.lists) S.template list_from<false>(low, few, [](float) {});
        }
        if (low > -INFINITY && p.lists) {
            cl.sync();
            if (by_k) wk = all_weight();
            int most = 0, least = 0;
            for (int i = lane; i < nc * NW; i += 32) {
                most = max(most, s.listed[i]);
                least = min(least, s.listed[i]);
            }
            most = __reduce_max_sync(0xffffffffu, most);
            least = __reduce_min_sync(0xffffffffu, least);
            if (least == 0 && most <= FEW) {
                // The first CTA goes on alone, with the candidates as its segment: its own barriers
                // cost a fraction of a cluster's.
                if (rank != 0) return;
                all_of_row = all_weight();
                row_ranges = nc * NW;
                S.seg = seg = few;
                S.nc = nc = 1;
                S.range = range = row_ranges * FEW / NW;
                S.list = few;
                S.list_stride = S.listed = range;
                S.list_low = -INFINITY;
                alone = true;
            }
        }
        set_bins();
        S.clear();
        S.each_from(low, [&](float x) {
            const float z = sc.z(x);
            S.count(bin_of(z), weight32(expf(z)));
        });
        const Bin over_z = S.merge();
        const uint32_t z_count = S.slice_count;
        const unsigned long long z_weight = S.slice_weight;

        // Narrow the bin that holds the goal down to one logit.
        auto narrow = [&](bool by_count, uint32_t by_rank, double goal, Found f) {
            uint32_t klo = 0xffffffffu, khi = 0;
            S.each_from(low, [&](float x) {
                if (bin_of(sc.z(x)) == f.bin) {
                    const uint32_t k = key_of<T>(x);
                    klo = min(klo, k);
                    khi = max(khi, k);
                }
            });
            klo = __reduce_min_sync(0xffffffffu, klo);
            khi = __reduce_max_sync(0xffffffffu, khi);
            if (lane == 0) {
                s.w_klo[warp] = klo;
                s.w_khi[warp] = khi;
            }
            __syncthreads();
            if (warp == 0) {
                klo = __reduce_min_sync(0xffffffffu, s.w_klo[lane & (NW - 1)]);
                khi = __reduce_max_sync(0xffffffffu, s.w_khi[lane & (NW - 1)]);
                if (lane < nc) {
                    Shared *o = cl.map_shared_rank(&s, lane);
                    o->x_klo[rank] = klo;
                    o->x_khi[rank] = khi;
                }
            }
            S.sync();
            klo = 0xffffffffu;
            khi = 0;
            for (int r = 0; r < nc; ++r) {
                klo = min(klo, s.x_klo[r]);
                khi = max(khi, s.x_khi[r]);
            }
            for (int level = 0; level < 4 && klo < khi; ++level) {  // 9 of 32 bits each
                int shift = 0;
                while ((khi - klo) >> shift >= NB) ++shift;
                S.clear();
                S.each_from(logit_of<T>(klo), [&](float x) {
                    const uint32_t k = key_of<T>(x);
                    if (k <= khi) S.count((int)((khi - k) >> shift), weight32(expf(sc.z(x))));
                });
                const Bin over_bits = S.merge();
                f = S.find(over_bits, by_count, by_rank, goal, f.count, f.weight);
                if (f.bin < 0) break;  // not reached: the goal lies in this range
                khi -= (uint32_t)f.bin << shift;
                const uint32_t width = (1u << shift) - 1;
                if (khi - klo > width) klo = khi - width;
            }
            Cut c;
            c.key = khi;
            c.before = f.weight;
            if (by_count) {
                c.keep = by_rank + 1 - f.count;
            } else {
                // the largest m with before + (m - 1) w < goal
                const unsigned long long w = weight(expf(sc.z(logit_of<T>(khi))));
                if (w == 0) {
                    c.keep = 0xffffffffu;
                } else {
                    const double m = ceil((goal - (double)f.weight) / (double)w);
                    uint32_t k = (uint32_t)fmin(fmax(m, 1.0), (double)p.V);
                    // the quotient may be off by its rounding
                    if (k > 1 && !((double)(f.weight + (unsigned long long)(k - 1) * w) < goal)) --k;
                    if ((double)(f.weight + (unsigned long long)k * w) < goal) ++k;
                    c.keep = k;
                }
            }
            return c;
        };

        if (by_k) {
            const Found f = S.find(over_z, true, (uint32_t)top_k - 1, 0.0, 0, 0);
            if (!alone) wk = all_weight();
            if (f.bin >= 0) {
                cut = narrow(true, (uint32_t)top_k - 1, 0.0, f);
                wk = cut.before + cut.keep * weight(expf(sc.z(logit_of<T>(cut.key))));
            }
        }
        if (by_p) {
            const double goal = (double)top_p * (double)wk;
            if (by_k) S.totals(z_count, z_weight);  // the slices' totals over z again
            const Found f = S.find(over_z, false, 0, goal, 0, 0);
            if (f.bin >= 0) {
                const Cut c = narrow(false, 0, goal, f);
                if (c.key > cut.key || (c.key == cut.key && c.keep < cut.keep)) cut = c;
            }
        }
    }

    // ---- kept weight by ranges of consecutive tokens
    const float xcut = cut.key == 0 ? -INFINITY : logit_of<T>(cut.key);
    const float need = only_first ? 0.f : min_p;
    {
        unsigned long long gt = 0;
        uint32_t eq = 0;
        if (cut.key == 0 && !(need > 0.f) && !alone) {
            gt = s.w_sum[warp];  // every token
        } else {
            // tokens that min-p lets through are above its logarithm
            float from = xcut;
            if (need > 0.f && !sc.inf_top) from = fmaxf(from, mx + (logf(need) - 0.01f) / sc.inv - 4e-7f * fabsf(mx));
            S.each_from(from, [&](float x) {
                const float e = expf(sc.z(x));
                if (!(e < need)) {
                    if (x > xcut)
                        gt += weight(e);
                    else
                        ++eq;
                }
            });
            gt = warp_add(gt);
            eq = warp_add(eq);
        }
        if (lane < nc) {  // to every CTA: nobody reads another's memory after the barrier
            Shared *o = cl.map_shared_rank(&s, lane);
            o->f_gt[rank * NW + warp] = gt;
            o->f_eq[rank * NW + warp] = eq;
        }
    }
    S.sync();
    total = alone ? all_of_row : all_weight();
    const float ecut = expf(sc.z(xcut));
    const unsigned long long wcut = cut.key == 0 ? 0 : weight(ecut);
    if (warp == 0) {
        // every CTA goes through all ranges: 4 lanes' worth of 32 at most
        uint32_t eqs[MAXC * NW / 32];
        unsigned long long gts[MAXC * NW / 32];
        const int ranges = nc * NW, each_lane = (ranges + 31) / 32;
        uint32_t le = 0;
#pragma unroll
        for (int i = 0; i < MAXC * NW / 32; ++i) {
            const int r = lane * each_lane + i;
            const bool on = i < each_lane && r < ranges;
            eqs[i] = on ? s.f_eq[r] : 0;
            gts[i] = on ? s.f_gt[r] : 0;
            le += eqs[i];
        }
        uint32_t seen = warp_before(le, lane);
        unsigned long long sum = 0;
        uint32_t left[MAXC * NW / 32];
#pragma unroll
        for (int i = 0; i < MAXC * NW / 32; ++i) {
            left[i] = cut.keep > seen ? cut.keep - seen : 0;
            seen += eqs[i];
            gts[i] += (unsigned long long)min(left[i], eqs[i]) * wcut;
            sum += gts[i];
        }
        unsigned long long at = warp_before(sum, lane);
        const unsigned long long all = warp_add(sum);
        // `all` is at least the most likely token's 2^32
        const double t = (double)p.u[b] * (double)all;
        unsigned long long goal = t > 0.0 ? (t < (double)all ? (unsigned long long)t : all - 1) : 0;
        if (goal > all - 1) goal = all - 1;
        if (lane == 0) s.owner = -1;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < MAXC * NW / 32; ++i) {
            const int r = lane * each_lane + i;
            if (gts[i] && goal >= at && goal - at < gts[i] && r / NW == rank) {
                s.owner = r % NW;
                s.goal = goal - at;
                s.eq_left = left[i];
            }
            at += gts[i];
        }
    }
    __syncthreads();
    if (s.owner == warp) {
        unsigned long long at = 0;
        const unsigned long long goal = s.goal;
        uint32_t left = s.eq_left;
        const T *w = seg + warp * range;
        for (int i0 = 0; i0 < range; i0 += 32 * VEC) {
            const int i = i0 + lane * VEC;
            float x[VEC], z[VEC];
            unsigned long long wt[VEC], sum = 0;
            uint32_t eqn = 0;
            if (i < range) {
                Row<T>::get(*reinterpret_cast<const typename Row<T>::Raw *>(w + i), x);
            } else {
#pragma unroll
                for (int v = 0; v < VEC; ++v) x[v] = -INFINITY;
            }
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                wt[v] = 0;
                z[v] = sc.z(x[v]);
                if (x[v] >= xcut && x[v] > -INFINITY) {
                    const float e = expf(z[v]);
                    if (!(e < need)) {
                        wt[v] = weight(e);
                        eqn += x[v] == xcut;
                    }
                }
            }
            uint32_t before = warp_before(eqn, lane);
            const uint32_t eq_all = warp_add(eqn);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                if (x[v] == xcut && wt[v]) {
                    if (before >= left) wt[v] = 0;
                    ++before;
                }
                sum += wt[v];
            }
            left = left > eq_all ? left - eq_all : 0;
            unsigned long long c = at + warp_before(sum, lane);
            if (goal >= c && goal - c < sum) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    if (goal >= c && goal - c < wt[v]) {
                        const int q = (warp * range + i + v) / FEW;  // alone: the warp it came from
                        p.token[b] = alone ? q * p.range + s.few_at[q][(i + v) % FEW] : first + i + v;
                        if (p.logprob) p.logprob[b] = z[v] - logf((float)total * (1.f / 4294967296.f));
                    }
                    c += wt[v];
                }
            }
            at += warp_add(sum);
            if (at > goal) break;
        }
    }
}

}  // namespace

cudaError_t launch_sample(SampleParams p, int dtype, int sms, cudaStream_t st) {
    const int vec = dtype == PMA_F32 ? 4 : 8, esize = dtype == PMA_F32 ? 4 : 2;
    // CTAs of a row: enough that a segment is at most 64 KB (bf16) or 48 KB (two CTAs fit an SM), more while
    // the batch leaves SMs without one and a warp keeps a vector a lane.
    int nc = 1;
    while (nc < MAXC && ((int64_t)p.V * esize > (int64_t)nc * (esize == 4 ? 49152 : 65536) ||
                         ((int64_t)p.B * nc < sms && p.V >= nc * 2 * NW * 32 * vec)))
        nc *= 2;
    p.range = ((p.V + nc * NW - 1) / (nc * NW) + vec - 1) / vec * vec;
    int smem = (int)((sizeof(Shared) + 15) / 16 * 16) + NW * p.range * esize;
    const int lists = (MAXC * NW * FEW + NW * LIST) * esize;
    // lists where they do not cost the second CTA of an SM
    p.lists = smem + lists <= (smem <= 112 * 1024 ? 112 : 227) * 1024;
    if (p.lists) smem += lists;
    cudaError_t e;
    constexpr int most = 227 * 1024;
    if (dtype == PMA_F32)
        e = set_smem_once<sample_kernel<float>>(most);
    else
        e = set_smem_once<sample_kernel<__nv_bfloat16>>(most);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(p.B * nc));
    cfg.blockDim = dim3(NW * 32);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)nc;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = dtype == PMA_F32 ? cudaLaunchKernelEx(&cfg, sample_kernel<float>, p)
                         : cudaLaunchKernelEx(&cfg, sample_kernel<__nv_bfloat16>, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace pma
