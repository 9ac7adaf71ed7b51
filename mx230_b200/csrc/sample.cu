// The next token of each row of logits, from given random numbers: temperature, top-k, top-p, min-p.
//
//   weight     w_i = exp((l_i - max l) / T), held as the whole number mass_i = round(2^40 w_i)   (masked: l = -inf or NaN, mass 0)
//   order      larger logits first, among equal ones the lower index
//   top-k      K = the first k entries of that order
//   top-p      P = the shortest prefix of K whose mass is at least p times K's
//   min-p      M = the entries with w_i >= m, a prefix as well
//   kept       what is in P and in M
//   token      the first kept entry, by index, with which the sum over those so far exceeds u times the sum over all
//
// Sums are over whole numbers, so they do not depend on their order, and the same row gives the same token on any grid.  K and P end
// with "the first entry of the order whose running count or mass exceeds t"; then what is kept is known, and the token is the
// first one by index whose running mass exceeds t.
//
// The logits have to be read once, 4 or 2 bytes each; what bounds the kernel is latency: for many rows what a weight takes, a chain
// of fp64, and barriers (64 rows of 128000 in fp32 with top-p 0.95: 67 us, 5 of them HBM's; half of the cycles issue), for a few rows the
// cluster's barriers (one row of 32000: 10 us).
// A cluster of one to eight CTAs takes a row, each a part of the vocabulary that follows the one before.  A histogram over 2048 equal
// intervals of max - l, as far as weights are not 0 (28.7 T), in counts (top-k) or masses says in which interval K or P ends.  If all
// down to there is one list, its entries are collected, sorted and summed, and what is kept of them is sorted again by index.  Else the
// interval's entries are, and the last one that is kept goes to all CTAs.  (Where the interval is more than a list, a histogram over the
// range of its (value, index) takes its place, as often as it takes.)  They add up what is kept by pieces of the row of 128 logits or
// more, so the piece that holds the token is known, and is looked at again.  Without top-k and top-p that is all there is to do.
// A weight takes fifteen fp64 instructions; rows with a small k take them for the entries of the list only.
#include <cuda_fp16.h>
#include <float.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"

namespace {

typedef unsigned long long u64;

constexpr int SM_THREADS = 512;
constexpr int SM_WARPS = SM_THREADS / 32;
constexpr int SM_BINS = 2048;
constexpr int SM_LIST = 1024;        // entries that are sorted, most
constexpr int SM_CLUSTER = 8;
constexpr int SM_MAX = 1 << 22;      // logits of a row: their masses stay below 2^63
constexpr double SM_MASS = 1099511627776.0;   // 2^40
typedef std::integral_constant<int, 0> First;    // passes over the logits
typedef std::integral_constant<int, 1> Weigh;
typedef std::integral_constant<int, 2> Look;
constexpr size_t SM_ALL = 224 * 1024, SM_HALF = 112 * 1024;   // shared memory of a CTA that has an SM to itself, that shares it

struct Coefficients {
    double magic, two52, c[9];
};
const Coefficients POWER_OF_TWO = {
    6755399441055744.0,   // 1.5 * 2^52: the last bits of a sum with it are the rounded whole number
    4503599627370496.0,   // 2^52
    {1.0203121063391729e-07, 1.3255224878668817e-06, 1.525268684626772e-05, 0.00015403455852453838, 0.0013333558179043112,
     0.009618129159402558, 0.055504108664760424, 0.2402265069581299, 0.6931471805599453}};
struct SampleParams {
    int *token;
    float *prob;
    const void *logits;
    long long row_stride;
    int vocab, ctas, idx_bits;
    const float *u;
    float temperature, top_p, min_p;
    int top_k;
    const float *temperatures, *top_ps, *min_ps;
    const int *top_ks;
    Coefficients power;
};

// What the first CTA tells the others (whole words, so that it can be copied as such).
struct Window {
    int kind;                // entries of: 0: intervals b0 .. b1 of the histogram over max - l; 1: and of lo .. hi as well
    int b0, b1;
    int count;               // entries in it
    u64 lo, hi;
    u64 base_count, base_mass;   // of the entries in front of it
};

struct alignas(16) Shared {
    // this CTA's histogram: counts, masses in two words; what has no weight is counted behind them, by lanes
    unsigned cnt[SM_BINS + 32], lo[SM_BINS + 32], hi[SM_BINS + 32];
    // first CTA: running counts and masses over the first histogram's intervals
    unsigned run_cnt[SM_BINS];
    u64 run_mass[SM_BINS];
    // a list's entries of this CTA, and of all (first CTA); running masses of the sorted list; a later histogram's running sums
    u64 mine[SM_LIST], all[SM_LIST];
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
__device__ __forceinline__ uint32_t add_cluster(uint32_t addr, uint32_t v) {
    uint32_t old;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
    return old;
}

template <typename T> __device__ __forceinline__ float logit(T v);
template <> __device__ __forceinline__ float logit(float v) { return v; }
template <> __device__ __forceinline__ float logit(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float logit(__nv_bfloat16 v) { return __bfloat162float(v); }

// a row's first or last piece of 16 bytes, masked where it is outside the row
template <typename T>
__device__ __noinline__ uint4 ragged_piece(const T *src, int at, int vocab) {
    constexpr int VE = 16 / (int)sizeof(T);
    const T masked = (T)-INFINITY;
    uint32_t word[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        T v[VE / 4];
#pragma unroll
        for (int c = 0; c < VE / 4; ++c) {
            const int x = at + i * (VE / 4) + c;
            v[c] = x >= 0 && x < vocab ? src[x] : masked;
        }
        word[i] = *(const uint32_t *)v;
    }
    return make_uint4(word[0], word[1], word[2], word[3]);
}

// whole numbers in the order of the floats, and back
__device__ __forceinline__ uint32_t order_key(float l) {
    const uint32_t b = __float_as_uint(l);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_float(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k); }

// Weight of a logit d <= 0 above the largest, e^(d / T) = 2^n 2^r: 2^n, and 2^r for |r| <= 1/2 by a polynomial of degree nine that
// is 1 at 0 and meets 2^r at the Chebyshev nodes (3.7e-14 of it elsewhere).  fp64 throughout: a table of powers in shared memory, in
// place of five of the steps, was read by 32 lanes at random, and that and the histogram's sums took what its banks give.  The
// coefficients come with the launch's parameters, from where an instruction takes them as an operand; as literals they were
// moved into registers again and again.
struct Weight {
    int n;
    double p;
};
__device__ __forceinline__ Weight weight_of(double d, double log2e_t, const Coefficients &k) {
    const double t = fma(d, log2e_t, k.magic), r = fma(d, log2e_t, k.magic - t);
    double p = fma(r, k.c[0], k.c[1]);
#pragma unroll
    for (int i = 2; i < 9; ++i) p = fma(r, p, k.c[i]);
    return {__double2loint(t), fma(r, p, 1.0)};
}
__device__ __forceinline__ double weight(double d, double log2e_t, const Coefficients &k) {
    const Weight w = weight_of(d, log2e_t, k);
    return w.p * __hiloint2double((1023 + w.n) * (1 << 20), 0);
}
// as a whole number of 2^-40: added to 2^52, it is the last bits of the sum (ties cannot be: no weight but 1 is a binary fraction)
__device__ __forceinline__ u64 mass_of(double d, double log2e_t, const Coefficients &k) {
    const Weight w = weight_of(d, log2e_t, k);
    return (u64)__double_as_longlong(fma(w.p, __hiloint2double((1023 + 40 + w.n) * (1 << 20), 0), k.two52)) & 0xFFFFFFFFFFFFFull;
}
__device__ __forceinline__ float finite(float l) {   // infinity is the largest number; NaN stays
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(l), "f"(FLT_MAX));
    return r;
}

// Interval of max - l, as the float 2^23 + interval: a difference, and a product and a sum rounded once, so it is monotone in l.
// (Masked logits are not among those that have one.)
constexpr float SM_INTERVAL = 8388608.0f;
__device__ __forceinline__ float interval(float l, float m, float scale) { return fmaf(m - l, scale, SM_INTERVAL); }

// running sums of n counts and masses (n <= PER * SM_THREADS), PER a thread, in place; either may be null
template <int PER>
__device__ __forceinline__ void running_sums(unsigned *cnt, u64 *mass, int n, Shared &S) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i0 = PER * threadIdx.x;
    u64 ms[PER], m = 0;
    unsigned cs[PER], c = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        m += mass && i0 + i < n ? mass[i0 + i] : 0, c += cnt && i0 + i < n ? cnt[i0 + i] : 0;
        ms[i] = m, cs[i] = c;
    }
    const u64 own_m = m;
    const unsigned own_c = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        if (mass) {
            const u64 mu = __shfl_up_sync(0xFFFFFFFFu, m, o);
            if (lane >= o) m += mu;
        }
        if (cnt) {
            const unsigned cu = __shfl_up_sync(0xFFFFFFFFu, c, o);
            if (lane >= o) c += cu;
        }
    }
    if (lane == 31) S.scan[warp] = m, S.scan_cnt[warp] = c;
    __syncthreads();
    // (the sums of the warps in front: a lane takes one, then all are added)
    u64 before = lane < warp ? S.scan[lane] : 0;
    unsigned cb = lane < warp ? S.scan_cnt[lane] : 0;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
        if (mass) before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
        if (cnt) cb += __shfl_xor_sync(0xFFFFFFFFu, cb, o);
    }
    before = __shfl_sync(0xFFFFFFFFu, before, 0) + m - own_m, cb = __shfl_sync(0xFFFFFFFFu, cb, 0) + c - own_c;
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (i0 + i < n) {
            if (mass) mass[i0 + i] = before + ms[i];
            if (cnt) cnt[i0 + i] = cb + cs[i];
        }
    __syncthreads();
}

// first index whose running sum exceeds t (there is one; whatever is found, it is an index)
template <typename R>
__device__ __forceinline__ int first_over(const R *run, int n, u64 t, int *found) {
    for (int i = threadIdx.x; i < n; i += SM_THREADS)
        if ((u64)run[i] > t && (i == 0 || (u64)run[i - 1] <= t)) *found = i;
    __syncthreads();
    return max(0, min(*found, n - 1));
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
    if (n <= SM_THREADS / 4) {   // few: an entry's place is the number of larger ones (no two are equal), counted by four lanes
        const int i = min((int)threadIdx.x >> 2, max(n - 1, 0));
        const u64 e = v[i];
        int place = 0;
#pragma unroll 4
        for (int o = threadIdx.x & 3; o < n; o += 4) place += v[o] > e;
        place += __shfl_xor_sync(0xFFFFFFFFu, place, 1);
        place += __shfl_xor_sync(0xFFFFFFFFu, place, 2);
        __syncthreads();
        if (threadIdx.x < 4 * n && (threadIdx.x & 3) == 0) v[place] = e;
        __syncthreads();
    } else if (n <= SM_THREADS) sort_entries<1>(v, other, n);
    else sort_entries<2>(v, other, n);
}

// KEEP: a CTA's share of the row stays in its shared memory; else it is read again where it is needed again.
template <typename T, bool KEEP>
__global__ void __launch_bounds__(SM_THREADS, 2) sample_kernel(const SampleParams P) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared &S = *(Shared *)smem;
    float *data = (float *)(smem + sizeof(Shared));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int C = P.ctas, row = blockIdx.x / C, rank = blockIdx.x - row * C;
    const bool first_cta = rank == 0;
    mx::pdl_trigger();
    __syncwarp();
    mx::cluster_arrive_relaxed();   // waited for before the first store to another CTA's memory
    auto clear_histogram = [&]() {   // (its three arrays follow one another)
        for (int i = tid; i < (int)(3 * sizeof(S.cnt) / 16); i += SM_THREADS) ((uint4 *)S.cnt)[i] = make_uint4(0, 0, 0, 0);
    };
    clear_histogram();
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
    // f(i, l) for four logits of this CTA at a time, l[0] being logit idx0 + i; in the first pass they are put in shared memory (KEEP)
    float m = -INFINITY, least = INFINITY;   // the row's largest and smallest (unmasked) logit
    auto for_logits = [&](auto f, auto pass) {
        constexpr bool first = pass.value == 0;
        if (KEEP && !first) {
            for (int i = tid * 4; i < n; i += SM_THREADS * 4) {
                const float4 l4 = *(const float4 *)(data + i);
                const float l[4] = {l4.x, l4.y, l4.z, l4.w};
                f(i, l);
            }
            return;
        }
        constexpr int LOADS = pass.value == 1 ? 1 : 4;   // in flight (weights take their time, and registers)
        for (int v = tid; v < v1 - v0; v += LOADS * SM_THREADS) {
            uint4 raw[LOADS];
#pragma unroll
            for (int q = 0; q < LOADS; ++q) {
                const int w = v + q * SM_THREADS, at = idx0 + w * VE;
                if (w >= v1 - v0) break;
                if (at >= 0 && at + VE <= P.vocab) raw[q] = *(const uint4 *)(src + at);
                else raw[q] = ragged_piece(src, at, P.vocab);
            }
#pragma unroll
            for (int q = 0; q < LOADS; ++q) {
                const int w = v + q * SM_THREADS;
                if (w >= v1 - v0) break;
                const T *e = (const T *)&raw[q];
#pragma unroll
                for (int i = 0; i < VE; i += 4) {
                    const float l[4] = {logit(e[i]), logit(e[i + 1]), logit(e[i + 2]), logit(e[i + 3])};
                    if (KEEP) *(float4 *)(data + w * VE + i) = make_float4(l[0], l[1], l[2], l[3]);
                    f(w * VE + i, l);
                }
            }
        }
    };
    // (infinity is the largest number; NaN is passed over)
    float hi = -INFINITY, lo = INFINITY;
    for_logits([&](int, const float (&l)[4]) {
#pragma unroll
        for (int c = 0; c < 4; ++c) hi = fmaxf(hi, l[c]), lo = fminf(lo, l[c] == -INFINITY ? INFINITY : l[c]);
    }, First());
    hi = fminf(hi, FLT_MAX), lo = fminf(lo, FLT_MAX);
    hi = mx::warp_max(hi), lo = mx::warp_min(lo);
    if (lane == 0) S.warp_a[warp] = hi, S.warp_b[warp] = lo;
    __syncthreads();
    mx::cluster_wait();
    if (warp == 0) {
        hi = mx::warp_max(S.warp_a[lane % SM_WARPS]), lo = mx::warp_min(S.warp_b[lane % SM_WARPS]);
        if (lane < C) st_cluster(mx::cluster_map(mx::smem_u32(&S.slot_a[rank]), lane), (u64)__float_as_uint(hi) << 32 | __float_as_uint(lo));
    }
    cluster_sync();
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
        for_logits([&](int i, const float (&l)[4]) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (finite(l[c]) == m) best = min(best, (unsigned)(idx0 + i + c));
        }, Look());
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
    const bool cut_p = p < 1.0f;
    const double log2e_t = 1.4426950408889634 / (double)T_, m64 = (double)m;
    // intervals over what has weight (2^-41 and more: 28.42 T) and what there is
    const float range = fminf(28.7f * T_, m - least);
    const float scale = range > 0.0f ? fminf((float)(SM_BINS - 1) / range, FLT_MAX) : 0.0f;
    // The least logit with an interval, 28.7 T below the largest or one step of the floats from there, where they are that far apart.
    // (The intervals' number alone would not do: where T is subnormal, or nearly, they reach farther, and weights out of what mass_of takes.)
    float lowest = fmaxf(least, m - 28.7f * T_);
    if (interval(lowest, m, scale) >= SM_INTERVAL + SM_BINS) lowest = nextafterf(lowest, INFINITY);

    auto entry = [&](int i, float l) {   // (-0 is 0)
        return (u64)order_key(l + 0.0f) << P.idx_bits | (((1u << P.idx_bits) - 1) - (unsigned)(idx0 + i));
    };
    auto entry_logit = [&](u64 e) { return key_float((uint32_t)(e >> P.idx_bits)); };
    bool with_mass = cut_p && (k == 0 || k > SM_LIST / 2);   // (a small k: only its entries' weights are asked for)
    const bool with_count = k != 0;
    auto mass = [&](float l) { return mass_of((double)l - m64, log2e_t, P.power); };
    auto add_to = [&](unsigned b, u64 mass) {   // a 64-bit sum by two words
        const unsigned l = (unsigned)mass, old = atomicAdd(&S.lo[b], l);
        const unsigned h = (unsigned)(mass >> 32) + (old + l < old);
        if (h) atomicAdd(&S.hi[b], h);
    };
    auto clear = [&]() {
        clear_histogram();
        __syncthreads();
    };
    int turn = 0;
    auto answer = [&]() { return &S.found[turn++ & 3]; };
    // the CTAs' histograms, added up by shares of the intervals into the first CTA's arrays, there as running sums
    auto merge = [&](unsigned *to_cnt, u64 *to_mass, bool counted, bool weighed, auto bins) {
        cluster_sync();
        const int b0 = bins.value / C * rank;
        for (int b = b0 + tid; b < b0 + bins.value / C; b += SM_THREADS) {
            unsigned c = 0;
            u64 ms = 0;
            if (counted)
#pragma unroll 8
                for (int r = 0; r < C; ++r) c += ld_cluster32(mx::cluster_map(mx::smem_u32(&S.cnt[b]), r));
            if (weighed)
#pragma unroll 8
                for (int r = 0; r < C; ++r)
                    ms += (u64)ld_cluster32(mx::cluster_map(mx::smem_u32(&S.hi[b]), r)) << 32 | ld_cluster32(mx::cluster_map(mx::smem_u32(&S.lo[b]), r));
            if (!counted) {
                // at most so many have this mass: none has less than the interval's end (the masses are whole; below 1: any number)
                const double least_mass = floor(weight(fmax(-(b + 0.51) / (double)scale, -28.75 * (double)T_), log2e_t, P.power) * (SM_MASS * (1 - 1e-6)) - 0.5);
                c = least_mass >= 1.0 ? (unsigned)fmin((double)ms / least_mass + 1.0, SM_LIST + 1.0) : SM_LIST + 1;
            }
            st_cluster(mx::cluster_map(mx::smem_u32(&to_cnt[b]), 0), c);
            if (weighed) st_cluster(mx::cluster_map(mx::smem_u32(&to_mass[b]), 0), ms);
        }
        cluster_sync();
        if (first_cta) running_sums<bins.value / SM_THREADS>(to_cnt, weighed ? to_mass : nullptr, bins.value, S);
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
    // f(i, l) for every logit of this CTA that lies in the window
    auto for_window = [&](auto f) {
        const Window w = S.w[wp];
        const bool exact = w.kind == 1;
        // logits of intervals b0 .. b1 lie between these, by more than the interval's own rounding
        const bool flat = !(scale > 0.0f);
        const float hi = flat || w.b0 == 0 ? INFINITY : m - ((float)w.b0 - 0.6f) / scale + 1e-6f * (fabsf(m) + (float)w.b0 / scale);
        const float lo = fmaxf(lowest, flat ? -INFINITY : m - ((float)w.b1 + 0.6f) / scale - 1e-6f * (fabsf(m) + (float)w.b1 / scale));
        for_logits([&](int i, const float (&l)[4]) {
            bool in[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) in[v] = l[v] >= lo & l[v] <= hi;
            if (in[0] | in[1] | in[2] | in[3])
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    if (in[v]) {
                        const float x = finite(l[v]), b = interval(x, m, scale) - SM_INTERVAL;
                        if (!(b >= w.b0 && b <= w.b1)) continue;
                        if (exact) {
                            const u64 e = entry(i + v, x);
                            if (e < w.lo || e > w.hi) continue;
                        }
                        f(i + v, x);
                    }
        }, Look());
    };
    // running masses of the n entries of S.all, of which `logit_of` gives the logit, into S.mine
    auto running_masses = [&](int n, auto logit_of) {
        for (int i = tid; i < n; i += SM_THREADS) S.mine[i] = mass(logit_of(S.all[i]));
        __syncthreads();
        running_sums<SM_LIST / SM_THREADS>(nullptr, S.mine, n, S);
    };
    // the window's entries, sorted, and their running masses (first CTA: S.all, S.mine); at most SM_LIST
    auto collect = [&](bool masses) {
        if (tid == 0) S.n_mine = 0;
        __syncthreads();
        for_window([&](int i, float l) {
            const unsigned at = atomicAdd(&S.n_mine, 1u);
            if (at < SM_LIST) S.mine[at] = entry(i, l);
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
            if (masses) running_masses(total, entry_logit);
        }
        return total;
    };
    // first entry of the order whose running count (by_mass: mass) exceeds t; in the first CTA: its number in the sorted list,
    // the window and S.mine say what lies in front of it
    auto search = [&](u64 t, bool by_mass) {
        Window next{};
        if (first_cta) {
            const int b = by_mass ? first_over(S.run_mass, SM_BINS, t, answer()) : first_over(S.run_cnt, SM_BINS, t, answer());
            next.b0 = next.b1 = b;
            if (b) next.base_count = S.run_cnt[b - 1], next.base_mass = S.run_mass[b - 1];
            next.count = (int)(S.run_cnt[b] - (unsigned)next.base_count);
        }
        tell(next);
        while (S.w[wp].count > SM_LIST) {
            // the range of the window's entries
            u64 e_lo = ~0ull, e_hi = 0;
            for_window([&](int i, float l) {
                const u64 e = entry(i, l);
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
            while ((e_hi - e_lo) >> shr >= SM_LIST) ++shr;
            for_window([&](int i, float l) {
                const unsigned b = (unsigned)((e_hi - entry(i, l)) >> shr);
                atomicAdd(&S.cnt[b], 1u);
                add_to(b, mass(l));
            });
            unsigned *c_run = (unsigned *)S.all;   // (no list is in use)
            merge(c_run, S.mine, true, true, std::integral_constant<int, SM_LIST>());
            if (first_cta) {
                next = S.w[wp];
                const u64 left = t - (by_mass ? next.base_mass : next.base_count);
                const int b = by_mass ? first_over(S.mine, SM_LIST, left, answer()) : first_over(c_run, SM_LIST, left, answer());
                const u64 c_before = b ? c_run[b - 1] : 0;
                next.kind = 1;
                next.hi = e_hi - ((u64)b << shr);
                next.lo = next.hi - e_lo < (1ull << shr) ? e_lo : next.hi - ((1ull << shr) - 1);
                next.count = (int)(c_run[b] - c_before);
                next.base_count += c_before, next.base_mass += b ? S.mine[b - 1] : 0;
            }
            tell(next);
        }
        const int total = collect(cut_p);
        if (!first_cta) return 0;
        return by_mass ? first_over(S.mine, total, t - S.w[wp].base_mass, answer()) : (int)(t - S.w[wp].base_count);
    };
    auto histogram = [&](auto counts, auto masses) {
        // (byte address of an interval's sum from its float; what has no weight goes behind the intervals)
        const uint32_t at0 = mx::smem_u32(S.cnt) - 4u * __float_as_uint(SM_INTERVAL), none = mx::smem_u32(&S.cnt[SM_BINS + lane]);
        constexpr uint32_t TO_LO = sizeof(S.cnt), TO_HI = 2 * sizeof(S.cnt);
        for_logits([&](int, const float (&raw)[4]) {
            uint32_t at[4];
            float l[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                l[v] = finite(raw[v]);
                at[v] = l[v] >= lowest ? at0 + 4u * __float_as_uint(interval(l[v], m, scale)) : none;
                if constexpr (decltype(counts)::value) asm volatile("red.shared.add.u32 [%0], 1;" ::"r"(at[v]) : "memory");
            }
            if constexpr (decltype(masses)::value) {
                u64 ms[4];
                unsigned old[4];
#pragma unroll
                for (int v = 0; v < 4; ++v) ms[v] = mass(l[v]);
                // (the four sums' low words together, then what is carried)
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    asm volatile("atom.shared.add.u32 %0, [%1], %2;" : "=r"(old[v]) : "r"(at[v] + TO_LO), "r"((unsigned)ms[v]) : "memory");
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const unsigned h = (unsigned)(ms[v] >> 32) + (old[v] + (unsigned)ms[v] < old[v]);
                    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p red.shared.add.u32 [%0], %1;\n\t}" ::"r"(at[v] + TO_HI), "r"(h)
                                 : "memory");
                }
            }
        }, Weigh());
    };
    auto share = [&](u64 total) { return min((u64)((double)u * (double)total), total - 1); };   // u's part of it (cut off, not rounded)
    // M: w >= min_w, in doubt only close to the logit for which it is equal
    const double min_w = min_p > 0.0f ? (double)fminf(min_p, 1.0f) : 0.0;
    auto in_m = [&](float l) { return weight((double)l - m64, log2e_t, P.power) >= min_w; };
    auto done = [&](int token, u64 mass, u64 of) {
        P.token[row] = token;
        if (P.prob) P.prob[row] = (float)((double)mass / (double)of);
    };

    // ---- the last entry of K and P: it is known, with all in front of it, from a list; or as the least entry that is kept ----
    u64 least_kept = 0;
    if (k || cut_p) {
        u64 z = 0;   // first CTA: mass of K
        for (bool again = false;; again = true) {
            if (again) clear();
            if (!with_mass) histogram(std::true_type(), std::false_type());
            else if (with_count) histogram(std::true_type(), std::true_type());
            else histogram(std::false_type(), std::true_type());
            merge(S.run_cnt, S.run_mass, with_count, with_mass, std::integral_constant<int, SM_BINS>());
            Window next{};
            if (first_cta) {
                if (with_mass) z = S.run_mass[SM_BINS - 1];   // (k = 0)
                next.b1 = k ? first_over(S.run_cnt, SM_BINS, (u64)min((unsigned)k, S.run_cnt[SM_BINS - 1]) - 1, answer())
                            : first_over(S.run_mass, SM_BINS, (u64)ceil((double)p * (double)z) - 1, answer());
                next.count = min((int)S.run_cnt[next.b1], SM_LIST + 1);
            }
            tell(next);
            if (S.w[wp].count <= SM_LIST || with_mass || !cut_p) break;
            with_mass = true;   // (many equal logits, or many close to the k-th)
        }
        if (S.w[wp].count <= SM_LIST) {   // all that can be kept is a list
            int n = collect(cut_p);
            if (!first_cta) return;
            if (k) n = min(k, n);
            if (cut_p) n = first_over(S.mine, n, (u64)ceil((double)p * (double)(k ? S.mine[n - 1] : z)) - 1, answer()) + 1;
            if (min_w > 0.0) {
                int in = 0;
                for (int i = tid; i < SM_LIST; i += SM_THREADS) in += __syncthreads_count(i < n && in_m(entry_logit(S.all[i])));
                n = in;
            }
            // what is kept, by index
            for (int i = tid; i < n; i += SM_THREADS) {
                const u64 e = S.all[i];
                S.all[i] = (e & ((1ull << P.idx_bits) - 1)) << 32 | e >> P.idx_bits;
            }
            __syncthreads();
            sort_down(S.all, S.mine, n);
            running_masses(n, [&](u64 e) { return key_float((uint32_t)e); });
            z = S.mine[n - 1];
            const int at = first_over(S.mine, n, share(z), answer());
            if (tid == 0) done((int)(((1u << P.idx_bits) - 1) - (unsigned)(S.all[at] >> 32)), S.mine[at] - (at ? S.mine[at - 1] : 0), z);
            return;
        }
        if (k) {
            const int i = search(first_cta ? (u64)min((unsigned)k, S.run_cnt[SM_BINS - 1]) - 1 : 0, false);
            if (first_cta) least_kept = S.all[i], z = cut_p ? S.w[wp].base_mass + S.mine[i] : 0;
        }
        if (cut_p) {
            const int i = search(first_cta ? (u64)ceil((double)p * (double)z) - 1 : 0, true);
            if (first_cta) least_kept = S.all[i];
        }
        if (first_cta && tid < C) st_cluster(mx::cluster_map(mx::smem_u32(&S.low), tid), least_kept);
        cluster_sync();
        least_kept = S.low;
        clear();
    }
    // ---- masses of what is kept, by pieces of the row that follow one another (a CTA's share is one of them): where u's part of them
    // is passed ----
    const float m_at = min_w > 0.0 ? m + logf((float)min_w) * T_ : -FLT_MAX, m_slack = 1e-5f * (fabsf(m) + fabsf(m_at) + T_) + FLT_MIN;
    float cut = entry_logit(least_kept);
    int cut_idx = (int)(((1u << P.idx_bits) - 1) - (unsigned)(least_kept & ((1ull << P.idx_bits) - 1)));
    if (least_kept == 0) cut = lowest, cut_idx = P.vocab;   // (what is below has no weight)
    const float from = min_w > 0.0 ? fmaxf(cut, m_at - m_slack) : cut, sure = min_w > 0.0 ? m_at + m_slack : -FLT_MAX;
    auto kept_mass = [&](int i, float raw) -> u64 {
        if (!(raw >= from)) return 0;
        const float l = finite(raw);
        if ((l == cut && idx0 + i > cut_idx) || (l < sure && !in_m(l))) return 0;
        return mass(l);
    };
    constexpr int UNIT = KEEP ? 128 : 32 * VE;   // logits that a warp takes at a time
    int piece = KEEP || VE == 4 ? 7 : 8;         // of 2^piece logits
    while ((n - 1) >> piece >= SM_BINS) ++piece;
    const int n_pieces = ((n - 1) >> piece) + 1;
    for (int i0 = warp * UNIT; i0 < n; i0 += SM_WARPS * UNIT) {   // (whole warps)
        u64 sum = 0;
        if constexpr (KEEP) {
            const int i = i0 + 4 * lane;
            if (i < n) {
                const float4 l = *(const float4 *)(data + i);
                sum = kept_mass(i, l.x) + kept_mass(i + 1, l.y) + kept_mass(i + 2, l.z) + kept_mass(i + 3, l.w);
            }
        } else {
            const int i = i0 + VE * lane, at = idx0 + i;
            if (i < n) {
                const uint4 raw = at >= 0 && at + VE <= P.vocab ? *(const uint4 *)(src + at) : ragged_piece(src, at, P.vocab);
                const T *e = (const T *)&raw;
#pragma unroll
                for (int c = 0; c < VE; ++c) sum += kept_mass(i + c, logit(e[c]));
            }
        }
        if (!__any_sync(0xFFFFFFFFu, sum != 0)) continue;
        // (at most eight masses a lane, 2^43: in two parts whose sums have 32 bits)
        const unsigned a = __reduce_add_sync(0xFFFFFFFFu, (unsigned)sum & 0xFFFFFF), b = __reduce_add_sync(0xFFFFFFFFu, (unsigned)(sum >> 24));
        if (lane == 0) add_to(i0 >> piece, ((u64)b << 24) + a);
    }
    __syncthreads();
    for (int b = tid; b < n_pieces; b += SM_THREADS) S.run_mass[b] = (u64)S.hi[b] << 32 | S.lo[b];
    __syncthreads();
    running_sums<SM_BINS / SM_THREADS>(nullptr, S.run_mass, n_pieces, S);
    const u64 own = S.run_mass[n_pieces - 1];
    if (tid < C) st_cluster(mx::cluster_map(mx::smem_u32(&S.slot_b[rank]), tid), own);
    cluster_sync();
    u64 z = 0, before = 0;
    for (int c = 0; c < C; ++c) {
        if (c == rank) before = z;
        z += S.slot_b[c];
    }
    u64 t = share(z);
    if (t < before || t - before >= own) return;
    t -= before;
    const int b = first_over(S.run_mass, n_pieces, t, answer());
    t -= b ? S.run_mass[b - 1] : 0;
    const int end = min(n, (b + 1) << piece);
    for (int i0 = b << piece; i0 < end; i0 += SM_THREADS) {
        const int i = i0 + tid, at = idx0 + i;
        u64 own_mass = 0;
        if (i < end && at >= 0 && at < P.vocab) own_mass = kept_mass(i, KEEP ? data[i] : logit(src[at]));
        S.mine[tid] = own_mass;
        __syncthreads();
        running_sums<1>(nullptr, S.mine, SM_THREADS, S);
        const u64 all = S.mine[SM_THREADS - 1];
        if (all > t) {
            if (S.mine[tid] > t && S.mine[tid] - own_mass <= t) done(at, own_mass, z);
            return;
        }
        t -= all;
        __syncthreads();
    }
}

template <typename T>
int launch_sample(mx230_handle *h, cudaStream_t st, SampleParams P, int n_rows) {
    constexpr int VE = 16 / (int)sizeof(T);
    const int pieces = P.vocab / VE + 2;
    // CTAs of a row, each with a few thousand logits, by whether their clusters then all run at once.  us with one / two / four / eight,
    // in fp32 but for 50257 (bf16), "own" with settings of each row's own:
    //   eight, which leave room for half as many CTAs as there are SMs: 128000, top-p: 9 rows 137, 80, 41, 28; 16 rows 139, 81, 41, 55;
    //   four, where two would not keep the row: 128000, top-p: 32 rows 143, 90, 43, 46; 70 rows 166, 108, 68, 112; 74 rows 144, 86, 111, 118.
    //     Short rows only where four keep it too: 50257, top-p: 33 rows 57, 35, 25, 35; 38 rows 57, 34, 37, 51; top-k 18, 14, 16, 24;
    //   two, two of them an SM: 148 rows of 50257, top-p 61, 57, 97; 147 rows of it, top-k 25, 22, 42; 148 rows of 128000, top-p 150, 116, 171.
    //     Up to half as many again, since rows take unequal time: 200 rows of 50257, own, 82, 60, 74; top-p 86, 92, 109; 200 rows of 128000, top-p 210,
    //     188, 196.  But not short rows of which a few entries are asked for, all alike: 200 rows of 50257, top-k 29, 40, 48.  (Where each row
    //     has its own k they are taken to be unequal: the host does not see them.)
    const bool few = P.top_ks == nullptr && P.top_k > 0 && P.top_k <= SM_LIST / 2;
    const bool short_row = P.vocab <= 65536;
    auto fits = [&](int to) {
        const long long all = (long long)n_rows * to, sms = h->sm_count;
        if (to == 8) return all * 2 <= sms;
        if (to == 4) return all * 10 <= (short_row ? 9 : 19) * sms;   // (clusters of four find no place on a tenth of the SMs)
        return all <= 2 * sms || (all <= 3 * sms && !(few && short_row));
    };
    int c = 1;
    while (c < SM_CLUSTER && P.vocab / c > 4096 && fits(2 * c)) c *= 2;
    const int share = ((pieces + c - 1) / c + 1) * VE;
    P.ctas = c;
    P.power = POWER_OF_TWO;
    const dim3 grid((unsigned)(n_rows * c));
    // The row stays in shared memory where its CTAs all have their places with that (top-p: 33 rows of 128000, four CTAs each: 43 us, read
    // again 63; 34 rows, which have not, 83 and 64; 64 rows 85 and 67; 64 rows of 50257, two each: 35 and 53).
    const size_t kept = sizeof(Shared) + (size_t)share * sizeof(float);
    MX_SMEM_ATTR_ONCE(h->device, (sample_kernel<T, true>), SM_ALL);
    MX_SMEM_ATTR_ONCE(h->device, (sample_kernel<T, false>), sizeof(Shared));
    if ((kept <= SM_HALF && (long long)n_rows * c <= 2ll * h->sm_count) || (kept <= SM_ALL && (long long)n_rows * c * 10 <= (c > 2 ? 9ll : 10ll) * h->sm_count)) MX_LAUNCH(h, st, MX230_K_SAMPLE, mx_launch(sample_kernel<T, true>, grid, SM_THREADS, kept, st, c, true, P));
    else MX_LAUNCH(h, st, MX230_K_SAMPLE, mx_launch(sample_kernel<T, false>, grid, SM_THREADS, sizeof(Shared), st, c, true, P));
    return MX230_OK;
}

}  // namespace

extern "C" int mx230_sample(mx230_handle *h, void *stream, int *token, float *prob, const void *logits, int dtype, int n_rows,
                            int vocab, long long row_stride, const float *u, float temperature, const float *temperatures,
                            int top_k, const int *top_ks, float top_p, const float *top_ps, float min_p, const float *min_ps) {
    MX_REQUIRE(h, MX230_ERR_INVALID_ARG, "sample: null handle");
    MX_REQUIRE(dtype == MX230_F32 || dtype == MX230_F16 || dtype == MX230_BF16, MX230_ERR_INVALID_ARG, "sample: element type %d", dtype);
    MX_REQUIRE(n_rows >= 0 && vocab > 0, MX230_ERR_INVALID_ARG, "sample: %d rows of %d logits", n_rows, vocab);
    MX_REQUIRE(vocab <= SM_MAX, MX230_ERR_UNSUPPORTED, "sample: %d logits a row (at most %d)", vocab, SM_MAX);
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
