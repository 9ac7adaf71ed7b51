// The next token of each row of logits, from given random numbers: temperature, top-k, top-p, min-p.
//
//   weight     w_i = exp((l_i - max l) / T), held as the whole number mass_i = round(2^40 w_i)   (masked: l = -inf or NaN, mass 0)
//   order      larger logits first, among equal ones the lower index
//   top-k      K = the first k entries of that order
//   top-p      P = the shortest prefix of K whose mass is at least p times K's
//   min-p      M = the entries with w_i >= m, a prefix as well
//   token      the first entry of the order whose running mass, its own included, exceeds u times the mass of P and M's intersection
//
// Sums are over whole numbers, so they do not depend on their order, and the same row gives the same token on any grid.  What has
// to be found is always "the first entry of the order whose running count or mass exceeds t"; three of them at most, each
// target known from the one before (the intersection of two prefixes has the smaller of their masses).
//
// Bounded by HBM: the logits are read once.  A cluster of up to eight CTAs holds a row in its shared memory.  A histogram over 1024
// equal intervals of max - l, as far as weights are not 0 (28.5 T), in counts and masses says which interval holds an entry that is
// sought; the entries of that interval alone are collected, sorted and summed.  Where an interval has more entries
// than the list, a histogram over the range of their (value, index) takes its place, as often as it takes.
// Weights take eleven fp64 instructions an entry (a table of 256 steps of 2^(1/256) and a polynomial of degree four, below
// 1e-15); rows with a small k take them for the entries of the list only.
#include <cuda_fp16.h>
#include <float.h>
#include <math.h>

#include "common.cuh"

namespace {

typedef unsigned long long u64;

constexpr int SM_THREADS = 512;
constexpr int SM_WARPS = SM_THREADS / 32;
constexpr int SM_BINS = 1024;
constexpr int SM_LIST = 1024;        // entries that are sorted, most
constexpr int SM_CLUSTER = 8;
constexpr int SM_MAX_DATA = 45056;   // logits that a CTA can hold
constexpr double SM_MASS = 1099511627776.0;   // 2^40

struct SampleParams {
    int *token;
    float *prob;
    const void *logits;
    long long row_stride;
    int vocab, ctas, idx_bits;
    int cap;                 // logits of a CTA's share, at most
    const float *u;
    float temperature, top_p, min_p;
    int top_k;
    const float *temperatures, *top_ps, *min_ps;
    const int *top_ks;
};

// What the first CTA tells the others (whole words, so that it can be copied as such).
struct Window {
    int kind;                // entries of: 0: intervals b0 .. b1 of the histogram over max - l, and c0 .. c1; 1: lo .. hi as well
    int b0, b1, c0, c1;
    int count;               // entries in it
    u64 lo, hi;
    u64 base_count, base_mass;   // of the entries in front of it
};
constexpr int W_EVERYTHING = SM_LIST + 1;   // count of the window that says: more than a list

struct alignas(16) Shared {
    uint2 mass[SM_BINS];         // this CTA's histogram: masses in two words, counts
    unsigned cnt[SM_BINS];
    // first CTA: running counts and masses over the first histogram's intervals
    unsigned run_cnt[SM_BINS];
    u64 run_mass[SM_BINS];
    // a list's entries of this CTA, and of all (first CTA); running masses of the sorted list; a later histogram's running sums
    u64 mine[SM_LIST], all[SM_LIST];
    double table[256];
    u64 scan[SM_WARPS];
    unsigned scan_cnt[SM_WARPS];
    u64 slot_a[SM_CLUSTER], slot_b[SM_CLUSTER];        // a word of each CTA
    float warp_a[SM_WARPS], warp_b[SM_WARPS];
    Window w[2];                 // the one in force and the next: a CTA may still look at one while the first CTA writes the other
    u64 low, high;
    int found[4];                // what was found, in turns: the answer before last is free
    unsigned n_mine, n_all, at_all;
};

__device__ __forceinline__ void cluster_sync() {   // (by whole warps)
    __syncwarp();
    mx::cluster_sync();
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void st_cluster(uint32_t addr, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory"); }
__device__ __forceinline__ uint32_t ld_cluster32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ u64 ld_cluster64(uint32_t addr) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t add_cluster(uint32_t addr, uint32_t v) {
    uint32_t old;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
    return old;
}

template <typename T> __device__ __forceinline__ float logit(T v);
template <> __device__ __forceinline__ float logit(float v) { return v; }
template <> __device__ __forceinline__ float logit(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float logit(__nv_bfloat16 v) { return __bfloat162float(v); }

// as it is kept: NaN is masked, infinity the largest number
__device__ __forceinline__ float kept_logit(float l) { return l == l ? fminf(l, FLT_MAX) : -INFINITY; }

// whole numbers in the order of the floats, and back
__device__ __forceinline__ uint32_t order_key(float l) {
    const uint32_t b = __float_as_uint(l);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_float(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k); }

// 2^(j / 256), j of a table, times the polynomial of 2^r for |r| <= 1/512; at most 42 octaves below 1, exactly 1 for l = m
__device__ __forceinline__ double weight(float l, double m, double log2e_t, const double *table) {
    const double x = ((double)l - m) * log2e_t;
    const double magic = 6755399441055744.0;   // 1.5 * 2^52: the sum's last bits are the rounded whole number
    const double t = fma(x, 256.0, magic);
    const int n = __double2loint(t);
    const double r = fma(t - magic, -0.00390625, x);
    // ln 2^i / i!
    double p = fma(r, 9.618129107628477e-3, 5.550410866482158e-2);
    p = fma(r, p, 2.402265069591007e-1);
    p = fma(r, p, 6.931471805599453e-1);
    p = fma(r, p, 1.0);
    p *= table[n & 255];
    return __hiloint2double(__double2hiint(p) + ((n >> 8) << 20), __double2loint(p));
}
__device__ __forceinline__ u64 to_mass(double w) {   // (ties cannot be: no weight but 1 is a binary fraction)
    return (u64)__double_as_longlong(fma(w, SM_MASS, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
}

// interval of max - l; SM_BINS: no weight, or masked (an infinite difference, or NaN where the scale is 0).  Monotone in l: a
// difference, a product and a sum, each rounded.
__device__ __forceinline__ unsigned interval(float l, float m, float scale) {
    return __float_as_uint(fminf((m - l) * scale, (float)SM_BINS) + 8388608.0f) & 0x7FFFFFu;
}

// running sums of n counts and masses (n <= 2 * SM_THREADS), two a thread, in place; counts may be null
__device__ __forceinline__ void running_sums(unsigned *cnt, u64 *mass, int n, Shared &S) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = 2 * threadIdx.x;
    const u64 m0 = i < n ? mass[i] : 0, m1 = i + 1 < n ? mass[i + 1] : 0;
    const unsigned c0 = cnt && i < n ? cnt[i] : 0, c1 = cnt && i + 1 < n ? cnt[i + 1] : 0;
    u64 m = m0 + m1;
    unsigned c = c0 + c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 mu = __shfl_up_sync(0xFFFFFFFFu, m, o);
        const unsigned cu = __shfl_up_sync(0xFFFFFFFFu, c, o);
        if (lane >= o) m += mu, c += cu;
    }
    if (lane == 31) S.scan[warp] = m, S.scan_cnt[warp] = c;
    __syncthreads();
    // (the sums of the warps in front: a lane takes one, then all are added)
    u64 before = lane < warp ? S.scan[lane] : 0;
    unsigned cb = lane < warp ? S.scan_cnt[lane] : 0;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
        cb += __shfl_xor_sync(0xFFFFFFFFu, cb, o);
    }
    m += __shfl_sync(0xFFFFFFFFu, before, 0), c += __shfl_sync(0xFFFFFFFFu, cb, 0);
    if (i < n) {
        mass[i] = m - m1;
        if (cnt) cnt[i] = c - c1;
    }
    if (i + 1 < n) {
        mass[i + 1] = m;
        if (cnt) cnt[i + 1] = c;
    }
    __syncthreads();
}

// first index whose running sum exceeds t (there is one)
template <typename R>
__device__ __forceinline__ int first_over(const R *run, int n, u64 t, int *found) {
    for (int i = threadIdx.x; i < n; i += SM_THREADS)
        if ((u64)run[i] > t && (i == 0 || (u64)run[i - 1] <= t)) *found = i;
    __syncthreads();
    return *found;
}

// Sorts n <= E * SM_THREADS entries of v, largest first, by the bitonic network: a thread has E of them, SM_THREADS apart; strides
// below 32 go through the warp, larger ones through v and `other` in turns.  Warps without entries stay out of it.
template <int E>
__device__ __forceinline__ void sort_entries(u64 *v, u64 *other, int n) {
    const int tid = threadIdx.x;
    int threads = 32;
    while (threads < n && threads < SM_THREADS) threads <<= 1;
    u64 e[E];
    if (tid < threads) {
#pragma unroll
        for (int h = 0; h < E; ++h) e[h] = tid + h * SM_THREADS < n ? v[tid + h * SM_THREADS] : 0;
        u64 *buf = other, *next = v;
        for (int k = 2; k < 2 * n; k <<= 1) {
            int j = k >> 1;
            if (E == 2 && j == SM_THREADS) {
                const u64 a = max(e[0], e[E - 1]);
                e[E - 1] = min(e[0], e[E - 1]), e[0] = a;
                j >>= 1;
            }
            for (; j >= 32; j >>= 1) {
#pragma unroll
                for (int h = 0; h < E; ++h) buf[tid + h * SM_THREADS] = e[h];
                asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
#pragma unroll
                for (int h = 0; h < E; ++h) {
                    const int i = tid + h * SM_THREADS;
                    const u64 o = buf[i ^ j];
                    e[h] = ((i & j) == 0) == ((i & k) == 0) ? max(e[h], o) : min(e[h], o);   // this place of the pair gets the larger one
                }
                u64 *const b = buf;
                buf = next, next = b;
            }
            for (; j > 0; j >>= 1)
#pragma unroll
                for (int h = 0; h < E; ++h) {
                    const int i = tid + h * SM_THREADS;
                    const u64 o = __shfl_xor_sync(0xFFFFFFFFu, e[h], j);
                    e[h] = ((i & j) == 0) == ((i & k) == 0) ? max(e[h], o) : min(e[h], o);
                }
        }
    }
    __syncthreads();   // (the last exchange has been read)
    if (tid < threads)
#pragma unroll
        for (int h = 0; h < E; ++h)
            if (tid + h * SM_THREADS < n) v[tid + h * SM_THREADS] = e[h];
    __syncthreads();
}
__device__ __forceinline__ void sort_down(u64 *v, u64 *other, int n) {
    static_assert(SM_LIST == 2 * SM_THREADS, "two entries a thread");
    if (n <= SM_THREADS) sort_entries<1>(v, other, n);
    else sort_entries<2>(v, other, n);
}

template <typename T>
__global__ void __launch_bounds__(SM_THREADS) sample_kernel(const SampleParams P) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared &S = *(Shared *)smem;
    float *data = (float *)(smem + sizeof(Shared));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int C = P.ctas, row = blockIdx.x / C, rank = blockIdx.x - row * C;
    const bool first_cta = rank == 0;
    mx::pdl_trigger();
    __syncwarp();
    mx::cluster_arrive_relaxed();   // waited for before the first store to another CTA's memory
    if (tid < 256) S.table[tid] = exp2((double)tid / 256.0);
    mx::pdl_wait();

    float T_ = P.temperatures ? P.temperatures[row] : P.temperature;
    int k = P.top_ks ? P.top_ks[row] : P.top_k;
    const float p = P.top_ps ? P.top_ps[row] : P.top_p, min_p = P.min_ps ? P.min_ps[row] : P.min_p;
    float u = P.u[row];
    u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;

    // ---- this CTA's share of the row: whole 16-byte pieces ----
    constexpr int VE = 16 / (int)sizeof(T);
    const T *src = (const T *)P.logits + (long long)row * P.row_stride;
    const int shift = (int)(((uintptr_t)src / sizeof(T)) % VE);   // elements between the last 16-byte boundary and the row
    const int pieces = (P.vocab + shift + VE - 1) / VE;
    const int v0 = (int)((long long)pieces * rank / C), v1 = (int)((long long)pieces * (rank + 1) / C);
    const int n = (v1 - v0) * VE, idx0 = v0 * VE - shift;         // data[i] is logit idx0 + i
    float hi = -INFINITY, lo = INFINITY;
    constexpr int LOADS = 4;   // in flight
    for (int v = tid; v < v1 - v0; v += LOADS * SM_THREADS) {
        uint4 raw[LOADS];
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
            const int at = idx0 + (v + l * SM_THREADS) * VE;
            if (v + l * SM_THREADS < v1 - v0 && at >= 0 && at + VE <= P.vocab) raw[l] = *(const uint4 *)(src + at);
        }
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
            const int w = v + l * SM_THREADS, at = idx0 + w * VE;
            if (w >= v1 - v0) break;
            const T *e = (const T *)&raw[l];
            float f[VE];
            if (at >= 0 && at + VE <= P.vocab) {
#pragma unroll
                for (int i = 0; i < VE; ++i) f[i] = kept_logit(logit(e[i]));
            } else {
#pragma unroll
                for (int i = 0; i < VE; ++i) f[i] = at + i >= 0 && at + i < P.vocab ? kept_logit(logit(src[at + i])) : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < VE; i += 4) *(float4 *)(data + w * VE + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                hi = fmaxf(hi, f[i]);
                lo = fminf(lo, f[i] == -INFINITY ? INFINITY : f[i]);
            }
        }
    }
    hi = mx::warp_max(hi), lo = mx::warp_min(lo);
    if (lane == 0) S.warp_a[warp] = hi, S.warp_b[warp] = lo;
    __syncthreads();
    mx::cluster_wait();
    if (warp == 0) {
        hi = mx::warp_max(S.warp_a[lane % SM_WARPS]), lo = mx::warp_min(S.warp_b[lane % SM_WARPS]);
        if (lane < C) st_cluster(mx::cluster_map(mx::smem_u32(&S.slot_a[rank]), lane), (u64)__float_as_uint(hi) << 32 | __float_as_uint(lo));
    }
    cluster_sync();
    float m = -INFINITY, least = INFINITY;
    for (int c = 0; c < C; ++c) m = fmaxf(m, __uint_as_float((uint32_t)(S.slot_a[c] >> 32))), least = fminf(least, __uint_as_float((uint32_t)S.slot_a[c]));
    if (m == -INFINITY) {   // nothing is left to choose from
        if (first_cta && tid == 0) {
            P.token[row] = -1;
            if (P.prob) P.prob[row] = 0.0f;
        }
        return;
    }
    // ---- the most likely one alone ----
    if (!(T_ > 0.0f) || k == 1 || p <= 0.0f) {
        if (tid == 0) S.n_mine = 0xFFFFFFFFu;
        __syncthreads();
        unsigned best = 0xFFFFFFFFu;
        for (int i = tid; i < n; i += SM_THREADS)
            if (data[i] == m) best = min(best, (unsigned)(idx0 + i));
        if (best != 0xFFFFFFFFu) atomicMin(&S.n_mine, best);
        __syncthreads();
        if (tid == 0) st_cluster(mx::cluster_map(mx::smem_u32(&S.slot_b[rank]), 0), (u64)S.n_mine);
        cluster_sync();
        if (first_cta && tid == 0) {
            u64 b = 0xFFFFFFFFu;
            for (int c = 0; c < C; ++c) b = min(b, S.slot_b[c]);
            P.token[row] = (int)b;
            if (P.prob) P.prob[row] = 1.0f;
        }
        return;
    }
    T_ = fminf(T_, 1e30f);   // (28.7 T stays finite)
    if (k <= 0 || k >= P.vocab) k = 0;
    const double log2e_t = 1.4426950408889634 / (double)T_, m64 = (double)m;
    // intervals over what has weight (2^-41 and more: 28.42 T) and what there is
    const float range = fminf(28.7f * T_, m - least);
    const float scale = range > 0.0f ? fminf((float)(SM_BINS - 1) / range, FLT_MAX) : 0.0f;
    const float floor_l = fmaxf(m - 28.75f * T_, -FLT_MAX);   // no weight here and below (at most 41.5 octaves below 1)
    const double min_w = min_p > 0.0f ? (double)fminf(min_p, 1.0f) : 0.0;

    auto entry = [&](int i) {   // (-0 is 0)
        return (u64)order_key(data[i] + 0.0f) << P.idx_bits | (((1u << P.idx_bits) - 1) - (unsigned)(idx0 + i));
    };
    auto entry_logit = [&](u64 e) { return key_float((uint32_t)(e >> P.idx_bits)); };
    auto add_to = [&](unsigned b, u64 mass) {   // a 64-bit sum by two words
        const unsigned l = (unsigned)mass, old = atomicAdd(&S.mass[b].x, l);
        const unsigned h = (unsigned)(mass >> 32) + (old + l < old);
        if (h) atomicAdd(&S.mass[b].y, h);
    };
    auto clear = [&]() {
        for (int b = tid; b < SM_BINS; b += SM_THREADS) S.cnt[b] = 0, S.mass[b] = make_uint2(0, 0);
        __syncthreads();
    };
    int turn = 0;
    auto answer = [&]() { return &S.found[turn++ & 3]; };
    // the CTAs' histograms, added up by shares of the intervals into the first CTA's arrays, there as running sums
    auto merge = [&](unsigned *to_cnt, u64 *to_mass) {
        cluster_sync();
        const int b0 = SM_BINS / C * rank;
        for (int b = b0 + tid; b < b0 + SM_BINS / C; b += SM_THREADS) {
            unsigned c = 0;
            u64 ms = 0;
#pragma unroll 8
            for (int r = 0; r < C; ++r) {
                c += ld_cluster32(mx::cluster_map(mx::smem_u32(&S.cnt[b]), r));
                ms += ld_cluster64(mx::cluster_map(mx::smem_u32(&S.mass[b]), r));
            }
            st_cluster(mx::cluster_map(mx::smem_u32(&to_cnt[b]), 0), c);
            st_cluster(mx::cluster_map(mx::smem_u32(&to_mass[b]), 0), ms);
        }
        cluster_sync();
        if (first_cta) running_sums(to_cnt, to_mass, SM_BINS, S);
    };
    // first CTA, by warp 0, of whose lane 0 this is the next window: it goes to all; then it is the one in force
    int wp = 0;
    auto tell = [&](const Window &next) {
        if (first_cta && warp == 0) {
            constexpr int W = sizeof(Window) / 4;
            if (lane == 0) S.w[wp ^ 1] = next, S.n_all = 0;
            __syncwarp();
            for (int i = lane; i < (C - 1) * W; i += 32) {
                uint32_t *word = (uint32_t *)&S.w[wp ^ 1] + i % W;
                st_cluster(mx::cluster_map(mx::smem_u32(word), 1 + i / W), *word);
            }
        }
        cluster_sync();
        wp ^= 1;
    };
    // f(i) for every logit of this CTA that lies in the window
    auto for_window = [&](auto f) {
        const Window w = S.w[wp];
        const unsigned b0 = w.b0, span_b = w.b1 - w.b0, c0 = w.c0, span_c = w.c1 - w.c0;
        for (int i = tid * 4; i < n; i += SM_THREADS * 4) {
            const float4 l4 = *(const float4 *)(data + i);
            const float l[4] = {l4.x, l4.y, l4.z, l4.w};
            unsigned in = 0;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const unsigned b = interval(l[v], m, scale);
                bool is = b - b0 <= span_b || b - c0 <= span_c;
                if (w.kind == 1 && is) {
                    const u64 e = entry(i + v);
                    is = e >= w.lo && e <= w.hi;
                }
                in |= (unsigned)is << v;
            }
            for (; in; in &= in - 1) f(i + __ffs(in) - 1);
        }
    };
    // the window's entries, sorted, and their running masses (first CTA: S.all, S.mine); at most SM_LIST
    auto collect = [&]() {
        if (tid == 0) S.n_mine = 0;
        __syncthreads();
        for_window([&](int i) {
            const unsigned at = atomicAdd(&S.n_mine, 1u);
            if (at < SM_LIST) S.mine[at] = entry(i);
        });
        __syncthreads();
        // into the first CTA's list, behind what others have put there; nobody looks at this CTA's memory any more
        const unsigned c = min(S.n_mine, (unsigned)SM_LIST);
        if (c) {
            if (tid == 0) S.at_all = add_cluster(mx::cluster_map(mx::smem_u32(&S.n_all), 0), c);
            __syncthreads();
            const unsigned base = S.at_all;
            for (unsigned i = tid; i < c; i += SM_THREADS)
                if (base + i < SM_LIST) st_cluster(mx::cluster_map(mx::smem_u32(&S.all[base + i]), 0), S.mine[i]);
        }
        cluster_sync();
        int total = 0;
        if (first_cta) {
            total = (int)min(S.n_all, (unsigned)SM_LIST);
            sort_down(S.all, S.mine, total);
            for (int i = tid; i < total; i += SM_THREADS) S.mine[i] = to_mass(weight(entry_logit(S.all[i]), m64, log2e_t, S.table));
            __syncthreads();
            running_sums(nullptr, S.mine, total, S);
        }
        return total;
    };
    // first entry of the order whose running count (by_mass: mass) exceeds t; in the first CTA: its number in the sorted list,
    // the window and S.mine say what lies in front of it
    auto search = [&](u64 t, bool by_mass) {
        Window next{};
        if (first_cta) {
            const int b = by_mass ? first_over(S.run_mass, SM_BINS, t, answer()) : first_over(S.run_cnt, SM_BINS, t, answer());
            next.b0 = next.b1 = next.c0 = next.c1 = b;
            if (b) next.base_count = S.run_cnt[b - 1], next.base_mass = S.run_mass[b - 1];
            next.count = (int)(S.run_cnt[b] - (unsigned)next.base_count);
        }
        tell(next);
        while (S.w[wp].count > SM_LIST) {
            // the range of the window's entries
            u64 e_lo = ~0ull, e_hi = 0;
            for_window([&](int i) {
                const u64 e = entry(i);
                e_lo = min(e_lo, e), e_hi = max(e_hi, e);
            });
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                e_lo = min(e_lo, __shfl_xor_sync(0xFFFFFFFFu, e_lo, o));
                e_hi = max(e_hi, __shfl_xor_sync(0xFFFFFFFFu, e_hi, o));
            }
            if (tid == 0) S.low = ~0ull, S.high = 0;
            clear();
            if (lane == 0) atomicMin(&S.low, e_lo), atomicMax(&S.high, e_hi);
            __syncthreads();
            if (tid < C) {
                st_cluster(mx::cluster_map(mx::smem_u32(&S.slot_a[rank]), tid), S.low);
                st_cluster(mx::cluster_map(mx::smem_u32(&S.slot_b[rank]), tid), S.high);
            }
            cluster_sync();
            for (int c = 0; c < C; ++c) e_lo = min(e_lo, S.slot_a[c]), e_hi = max(e_hi, S.slot_b[c]);
            int shr = 0;
            while ((e_hi - e_lo) >> shr >= SM_BINS) ++shr;
            for_window([&](int i) {
                const unsigned b = (unsigned)((e_hi - entry(i)) >> shr);
                atomicAdd(&S.cnt[b], 1u);
                add_to(b, to_mass(weight(data[i], m64, log2e_t, S.table)));
            });
            unsigned *c_run = (unsigned *)S.all;   // (no list is in use)
            merge(c_run, S.mine);
            if (first_cta) {
                next = S.w[wp];
                const u64 left = t - (by_mass ? next.base_mass : next.base_count);
                const int b = by_mass ? first_over(S.mine, SM_BINS, left, answer()) : first_over(c_run, SM_BINS, left, answer());
                const u64 c_before = b ? c_run[b - 1] : 0;
                next.kind = 1;
                next.hi = e_hi - ((u64)b << shr);
                next.lo = next.hi - e_lo < (1ull << shr) ? e_lo : next.hi - ((1ull << shr) - 1);
                next.count = (int)(c_run[b] - c_before);
                next.base_count += c_before, next.base_mass += b ? S.mine[b - 1] : 0;
            }
            tell(next);
        }
        const int total = collect();
        if (!first_cta) return 0;
        return by_mass ? first_over(S.mine, total, t - S.w[wp].base_mass, answer()) : (int)(t - S.w[wp].base_count);
    };
    auto share = [&](double of, u64 total) { return (u64)fmin(of * (double)total, (double)total); };   // (cut off, not rounded)

    bool with_mass = k == 0 || k > SM_LIST / 2;
    u64 z = 0, z_min = 0;   // first CTA: mass of K, then of what is kept; of M
    for (;;) {
        // ---- histogram over max - l ----
        clear();
        u64 sum_min = 0;
        for (int i = tid * 4; i < n; i += SM_THREADS * 4) {
            const float4 l4 = *(const float4 *)(data + i);
            const float l[4] = {l4.x, l4.y, l4.z, l4.w};
            if (with_mass) {
                double w[4];
#pragma unroll
                for (int v = 0; v < 4; ++v) w[v] = weight(fmaxf(l[v], floor_l), m64, log2e_t, S.table);
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const unsigned b = interval(l[v], m, scale);
                    const u64 mass = to_mass(w[v]);
                    if (b >= SM_BINS) continue;
                    atomicAdd(&S.cnt[b], 1u);
                    add_to(b, mass);
                    if (min_w > 0.0 && w[v] >= min_w) sum_min += mass;
                }
            } else {
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const unsigned b = interval(l[v], m, scale);
                    if (b < SM_BINS) atomicAdd(&S.cnt[b], 1u);
                }
            }
        }
        if (with_mass && min_w > 0.0) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum_min += __shfl_xor_sync(0xFFFFFFFFu, sum_min, o);
            if (lane == 0) S.scan[warp] = sum_min;
            __syncthreads();
            if (tid == 0) {
                for (int w = 1; w < SM_WARPS; ++w) sum_min += S.scan[w];
                st_cluster(mx::cluster_map(mx::smem_u32(&S.slot_b[rank]), 0), sum_min);
            }
        }
        merge(S.run_cnt, S.run_mass);
        // ---- what is to be looked at: all that can be kept, if that is a list; else (k = 0) the interval where P ends and those where
        // the token then can be, if they are; else more than that ----
        Window next{};
        if (first_cta) {
            const unsigned there = S.run_cnt[SM_BINS - 1];
            z = z_min = S.run_mass[SM_BINS - 1];
            int b = SM_BINS - 1;
            if (k) b = first_over(S.run_cnt, SM_BINS, (u64)min((unsigned)k, there) - 1, answer());
            else if (p < 1.0f) b = first_over(S.run_mass, SM_BINS, (u64)ceil((double)p * (double)z) - 1, answer());
            if (with_mass && min_w > 0.0) {
                z_min = 0;
                for (int c = 0; c < C; ++c) z_min += S.slot_b[c];
            }
            next.b1 = next.c1 = b, next.count = (int)S.run_cnt[b];
            if (next.count > SM_LIST && k == 0) {
                // the kept mass lies between these, and u's share of it too
                const u64 z0 = min(z_min, p < 1.0f ? (b ? S.run_mass[b - 1] : 0) : z), z1 = min(z_min, p < 1.0f ? S.run_mass[b] : z);
                next.c0 = first_over(S.run_mass, SM_BINS, z0 ? min(share((double)u, z0), z0 - 1) : 0, answer());
                next.c1 = first_over(S.run_mass, SM_BINS, min(share((double)u, z1), z1 - 1), answer());
                if (p < 1.0f) {
                    if (next.c1 >= b) next.c1 = b;
                    next.b0 = next.b1 = b;
                    if (next.c1 == b) next.b0 = next.c0;   // (next to each other: one range)
                } else next.b0 = next.c0, next.b1 = next.c1;
                const unsigned in_b = S.run_cnt[next.b1] - (next.b0 ? S.run_cnt[next.b0 - 1] : 0);
                const unsigned in_c = S.run_cnt[next.c1] - (next.c0 ? S.run_cnt[next.c0 - 1] : 0);
                next.count = (int)(next.c1 == next.b1 ? in_b : in_b + in_c);
            }
            if (next.count > SM_LIST) next.count = W_EVERYTHING;
        }
        tell(next);
        if (S.w[wp].count <= SM_LIST || with_mass) break;
        with_mass = true;   // (many equal logits, or many close to the k-th)
    }
    int at;
    if (S.w[wp].count <= SM_LIST) {
        const int total = collect();
        if (!first_cta) return;
        // the list's running masses are those of the whole order less what lies in front of its ranges: of c (or b, if it is one
        // range), and between c and b
        const Window w = S.w[wp];
        const bool one = w.c1 == w.b1;
        const u64 front = w.c0 ? S.run_mass[w.c0 - 1] : 0;
        u64 between = 0;
        if (!one) {
            const u64 in_c = S.mine[S.run_cnt[w.c1] - (w.c0 ? S.run_cnt[w.c0 - 1] : 0) - 1];
            between = S.run_mass[w.b0 - 1] - front - in_c;
        }
        if (k) z = S.mine[min(k, total) - 1];
        u64 keep = z;
        if (p < 1.0f) keep = front + between + S.mine[first_over(S.mine, total, (u64)ceil((double)p * (double)z) - 1 - front - between, answer())];
        if (min_w > 0.0) {
            if (with_mass) keep = min(keep, z_min);
            else {   // the last entry of M among the list's; M beyond the list keeps all that P keeps
                if (tid == 0) S.low = 0;
                __syncthreads();
                for (int i = tid; i < total; i += SM_THREADS)
                    if (weight(entry_logit(S.all[i]), m64, log2e_t, S.table) >= min_w) atomicMax(&S.low, S.mine[i]);
                __syncthreads();
                keep = min(keep, S.low);
            }
        }
        z = keep;
        const u64 t = min(share((double)u, z), z - 1) - front;
        // (behind c: in b)
        at = first_over(S.mine, total, one || t < S.mine[S.run_cnt[w.c1] - (w.c0 ? S.run_cnt[w.c0 - 1] : 0) - 1] ? t : t - between, answer());
    } else {
        if (k) {
            const int i = search(first_cta ? (u64)min((unsigned)k, S.run_cnt[SM_BINS - 1]) - 1 : 0, false);
            if (first_cta) z = S.w[wp].base_mass + S.mine[i];
        }
        if (p < 1.0f) {
            const int i = search(first_cta ? (u64)ceil((double)p * (double)z) - 1 : 0, true);
            if (first_cta) z = S.w[wp].base_mass + S.mine[i];
        }
        if (first_cta) z = min(z, z_min);
        at = search(first_cta ? min(share((double)u, z), z - 1) : 0, true);
        if (!first_cta) return;
    }
    if (tid == 0) {
        const u64 e = S.all[at];
        P.token[row] = (int)(((1u << P.idx_bits) - 1) - (unsigned)(e & ((1ull << P.idx_bits) - 1)));
        if (P.prob) P.prob[row] = (float)((double)(S.mine[at] - (at ? S.mine[at - 1] : 0)) / (double)z);
    }
}

template <typename T>
int launch_sample(mx230_handle *h, cudaStream_t st, SampleParams P, int n_rows) {
    constexpr int VE = 16 / (int)sizeof(T);
    const int pieces = P.vocab / VE + 2;
    // Smallest cluster whose CTAs can hold the row; more CTAs while SMs have none and each still has a few thousand logits.
    int c = 1;
    auto share_of = [&](int n) { return ((pieces + n - 1) / n + 1) * VE; };
    while (c < SM_CLUSTER && share_of(c) > SM_MAX_DATA) c *= 2;
    while (c < SM_CLUSTER && (long long)n_rows * c < 2ll * h->sm_count && P.vocab / c > 4096) c *= 2;
    P.ctas = c, P.cap = share_of(c);
    const size_t sm = sizeof(Shared) + (size_t)P.cap * sizeof(float);
    MX_SMEM_ATTR_ONCE(h->device, sample_kernel<T>, 227 * 1024);
    MX_LAUNCH(h, st, MX230_K_SAMPLE, mx_launch(sample_kernel<T>, dim3((unsigned)(n_rows * c)), SM_THREADS, sm, st, c, true, P));
    return MX230_OK;
}

}  // namespace

extern "C" int mx230_sample(mx230_handle *h, void *stream, int *token, float *prob, const void *logits, int dtype, int n_rows,
                            int vocab, long long row_stride, const float *u, float temperature, const float *temperatures,
                            int top_k, const int *top_ks, float top_p, const float *top_ps, float min_p, const float *min_ps) {
    MX_REQUIRE(h, MX230_ERR_INVALID_ARG, "sample: null handle");
    MX_REQUIRE(dtype == MX230_F32 || dtype == MX230_F16 || dtype == MX230_BF16, MX230_ERR_INVALID_ARG, "sample: element type %d", dtype);
    MX_REQUIRE(n_rows >= 0 && vocab > 0, MX230_ERR_INVALID_ARG, "sample: %d rows of %d logits", n_rows, vocab);
    MX_REQUIRE(vocab <= SM_CLUSTER * (SM_MAX_DATA - 32), MX230_ERR_UNSUPPORTED, "sample: %d logits a row (at most %d)", vocab,
               SM_CLUSTER * (SM_MAX_DATA - 32));
    MX_REQUIRE(n_rows <= (1 << 27), MX230_ERR_UNSUPPORTED, "sample: %d rows", n_rows);
    if (n_rows == 0) return MX230_OK;
    MX_REQUIRE(token && logits && u, MX230_ERR_INVALID_ARG, "sample: null argument");
    MX_REQUIRE(row_stride >= 0, MX230_ERR_INVALID_ARG, "sample: row stride %lld", row_stride);
    const size_t size = dtype == MX230_F32 ? 4 : 2;
    MX_REQUIRE((uintptr_t)logits % size == 0 &&
                   (((uintptr_t)token | (uintptr_t)prob | (uintptr_t)u | (uintptr_t)temperatures | (uintptr_t)top_ks | (uintptr_t)top_ps |
                     (uintptr_t)min_ps) & 3) == 0, MX230_ERR_INVALID_ARG, "sample: misaligned pointer");
    SampleParams P{};
    P.token = token, P.prob = prob, P.logits = logits, P.row_stride = row_stride, P.vocab = vocab, P.u = u;
    P.temperature = temperature, P.top_k = top_k, P.top_p = top_p, P.min_p = min_p;
    P.temperatures = temperatures, P.top_ks = top_ks, P.top_ps = top_ps, P.min_ps = min_ps;
    while ((1 << P.idx_bits) < vocab) ++P.idx_bits;
    if (P.idx_bits == 0) P.idx_bits = 1;
    mx230_device_guard guard(h->device);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == MX230_F32) return launch_sample<float>(h, st, P, n_rows);
    if (dtype == MX230_F16) return launch_sample<__half>(h, st, P, n_rows);
    return launch_sample<__nv_bfloat16>(h, st, P, n_rows);
}
