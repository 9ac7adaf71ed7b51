// Products of a few rows with a matrix of 4-bit weights (the projections of a decode step, beside mx230_gemv and mx230_gemv_int8):
//   y[r][o] = sum_i x[r][i] s[g][o] (q[i][o] - z[g][o]) + bias[o] + add[r][o],   g = i / group
//
// Bounded by HBM on the weights: half a byte each, read once, and 4 bytes of scale and zero point per group.  At that rate an SM
// takes 46 weights a cycle, so a weight may cost about two instructions of a lane; multiply-adds on CUDA cores, with the
// conversion from 4 bits in front, would take more for a single row and that many times more for several.  Hence warp-level
// tensor-core tiles (m16n8k16) with the weights as A: 16 outputs x 16 inputs.  Four bits at places 0 to 3 or 4 to 7 of an fp16 are the
// number q 2^-24 or q 2^-20 (a subnormal), so a pair of weights costs an "and", a quarter of a shift and one rounded-once multiply-add
// that makes it (q - z) 2^-10, exactly: a zero point so has no rounding of its own, and what a weight of 0 meets does not count
// however large it is.  (Sums of x q and of x apart save the multiply-add, but what is left of their difference goes by
// sum |x| (q + z): with one x of 10^4 among 4096 whose own weight is 0, 9e-5 of the result.)  The rows are the eight columns of B, two
// columns a row:
//   x 2^e = hi + lo, both fp16, e such that the largest of the 64 values of a tile lies in [2^14, 2^15):
// |x 2^e - hi - lo| <= 2^-23 |x 2^e|, an ulp of fp32 (but for values 2^-17 times the tile's largest and less, which keep an
// absolute error of 2^-39 of that).  Products are then exact in fp32; sums are fp32, per tile of 64 inputs (32, if groups are of
// 32).  The row's total gets s 2^(10 - e) times the tile's sum.  Infinite x are
// infinite in hi and 0 in lo, so sums are infinite or NaN as those of x itself.
//
// About 84 instructions a warp and tile at one to four rows.  4096 x 14336, one row: 11.5 us where HBM would need 4.7, bounded by latency
// (seventeen warps an SM, each scheduler issues in 0.45 of its cycles); 4096 x 128000, four rows: 67 to 71 where it would need 42 (0.61).
//
// Layout, made once by mx230_pack_int4: tiles of 16 outputs x 64 inputs, 512 bytes, of which lane (g = lane / 4, j = lane % 4) has 16:
// words [row g: inputs 8j .. 8j+7][row g: inputs 32 + 8j ..][row g + 8: 8j ..][row g + 8: 32 + 8j ..], input 2p of eight at bits
// 4p, input 2p + 1 at bits 16 + 4p.  (Which input a k index of the MMA stands for is free, as long as A and B agree.)  Tiles of an
// output row follow one another along the inputs; behind all tiles, per (16 outputs, group), 16 words (s, -z 2^-10) of fp16.
//
// Weights come by bulk copies, a lane's for a CTA of sixteen warps, into a ring of stages (some output tiles, up to 32 tiles of their
// inputs each: 16 KB in a row and their (s, z)).  Loads to registers, two to four tiles ahead, kept too few bytes on their way with
// the warps that fit beside them (16 of them read 5.6 TB/s with nothing else to do, 32 read 6.1), and took four instructions a
// tile; a ring by cp.async of every lane took as many; bulk copies by the warp, of a KB, were bound by their number.
//
// Order of the sums: the inputs are cut over the CTAs of a cluster and there by turns over sixteen warps (a tile each), by n_in and n_out
// alone; a warp sums in index order, then the warps' and the CTAs' sums are added pairwise.  So a row has the same bits whatever
// rows are computed with it.
#include <cuda_fp16.h>

#include "common.cuh"
#include "pieces.h"

namespace {

constexpr int W4_K = 64;          // inputs of a tile
constexpr int W4_N = 16;          // outputs of a tile
constexpr int W4_WARPS = 16;         // that compute
constexpr int W4_THREADS = W4_WARPS * 32, W4_PRODUCER = 32;
constexpr int W4_CLUSTER = 8;     // most CTAs whose sums are added through shared memory
constexpr int W4_K_CTA = 64;      // tiles of the inputs of a CTA, up to eight CTAs; then twice that
constexpr int W4_STAGES = 6;      // most
constexpr int W4_SMEM = 222 * 1024;

struct Int4Params {
    float *y;
    const float *x;
    const uint4 *codes;      // [n_tiles][k_tiles][32]
    const uint32_t *sz;      // [n_tiles][groups][16]
    const float *bias, *add;
    int n_rows, n_in, n_out, group, groups;
    int n_tiles, k_tiles;
    int ctas_k;              // CTAs of a cluster, each with a part of the inputs
    int n_groups, n_clusters;   // of output tiles that a cluster computes at a time; clusters, each with every n_clusters-th of them
    int stages, stage_k;     // of the ring; tiles of the inputs in one
    int k_cta;               // tiles of the inputs of a CTA, at most
    uint32_t group_magic;    // 2^32 over the tiles of a group of inputs, rounded up; 0: one
    int x_vec;               // rows are 16-byte aligned
    int *status;             // where a wait that ran out is recorded
    int test_drop_tile;      // test hook: stage from which on CTA 0's producer requests nothing; -1 = off
    long long x_stride, y_stride, add_stride;
};

// (s, -z 2^-10) and codes of one output tile and input tile; padding: s = 0
__global__ void pack_int4_kernel(uint4 *codes_out, uint32_t *sz_out, const uint8_t *codes, const __half *scales, const uint8_t *zeros,
                                 int n_in, int n_out, int group, int n_tiles, int k_tiles, int groups) {
    const long long n_codes = (long long)n_tiles * k_tiles * 32, n_sz = (long long)n_tiles * groups * 16;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n_codes + n_sz; i += (long long)gridDim.x * blockDim.x) {
        if (i < n_codes) {
            const int lane = (int)(i & 31), g = lane >> 2, j = lane & 3;
            const long long t = i >> 5;
            const int nt = (int)(t / k_tiles), kt = (int)(t - (long long)nt * k_tiles);
            uint32_t w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int o = nt * W4_N + g + (q >> 1) * 8, k0 = kt * W4_K + (q & 1) * 32 + 8 * j;
                uint32_t v = 0;
                for (int e = 0; e < 8; ++e)
                    if (o < n_out && k0 + e < n_in) v |= (uint32_t)(codes[(size_t)(k0 + e) * n_out + o] & 15) << (4 * (e >> 1) + 16 * (e & 1));
                w[q] = v;
            }
            codes_out[i] = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            const long long s = i - n_codes;
            const long long t = s >> 4;
            const int nt = (int)(t / groups), gr = (int)(t - (long long)nt * groups), o = nt * W4_N + (int)(s & 15);
            __half sc = __float2half(0.0f), z = __float2half(8.0f);
            if (o < n_out) {
                sc = scales[(size_t)gr * n_out + o];
                if (zeros) z = __float2half((float)zeros[(size_t)gr * n_out + o]);   // (0 to 255: exact, and so is -z 2^-10)
            }
            sz_out[s] = (uint32_t)__half_as_ushort(sc) | (uint32_t)__half_as_ushort(__float2half(-0x1p-10f * __half2float(z))) << 16;
        }
    }
}

__device__ __forceinline__ uint32_t h2_u(__half2 v) { return *(uint32_t *)&v; }
__device__ __forceinline__ __half2 u_h2(uint32_t v) { return *(__half2 *)&v; }

// eight codes -> four pairs (inputs 2p, 2p + 1) of (q - z) 2^-10; nz: -z 2^-10, twice
__device__ __forceinline__ void pairs8(uint32_t w, __half2 nz, uint32_t (&a)[4]) {
    const __half2 low = __half2half2(__ushort_as_half(0x7400)), high = __half2half2(__ushort_as_half(0x6400));   // 2^14, 2^10
    const uint32_t v = w >> 8;
    a[0] = h2_u(__hfma2(u_h2(w & 0x000F000Fu), low, nz)), a[1] = h2_u(__hfma2(u_h2(w & 0x00F000F0u), high, nz));
    a[2] = h2_u(__hfma2(u_h2(v & 0x000F000Fu), low, nz)), a[3] = h2_u(__hfma2(u_h2(v & 0x00F000F0u), high, nz));
}

// c = a b + c, or a b
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// pairwise sum of n (a power of two, at most 16) values `step` apart
__device__ __forceinline__ float tree_sum(const float *p, int n, int step) {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = i < n ? p[i * step] : 0.0f;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1)
        if (n > o)
#pragma unroll
            for (int i = 0; i < 16; i += 2 * o) v[i] += v[i + o];
    return v[0];
}

// NT: column tiles of four rows.  T: output tiles of a warp.  G32: groups of 32 inputs (else a multiple of 64).
// Shared memory: ring [stages][T][stage_k x 512 of codes, stage_k x 64 (groups of 32: 128) of (s, z)]; sums [2][16 warps][T * NT * 64];
// in clusters, this CTA's share of everybody's sums [2][C][T * NT * 64 / C]; per (tile, row) 2^-e; 32
// bytes of zeros; rows [k_cta][NT][lanes][8 words].
template <int NT, int T, bool G32>
struct Int4Form {
    static constexpr int SUMS = T * NT * 64;                // floats of a warp
    static constexpr int TILE = 512 + (G32 ? 128 : 64);     // bytes of a tile in a stage
};

template <int NT, int T, bool G32>
__global__ void __launch_bounds__(W4_THREADS + W4_PRODUCER, 1) gemv_int4_kernel(const Int4Params P) {
    using S = Int4Form<NT, T, G32>;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(8) unsigned long long full[W4_STAGES], empty[W4_STAGES];
    __shared__ int aborted;
    __shared__ volatile int stop_grp, stop_k;               // first stage that the producer, having given up, does not request
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j = lane & 3;
    constexpr int KW = W4_WARPS;                            // warps along the inputs, by turns
    const int C = P.ctas_k;
    const int rank = blockIdx.x % C, grp0 = blockIdx.x / C;
    const int row0 = blockIdx.y * (4 * NT), rows = min(4 * NT, P.n_rows - row0);
    const int rt = NT == 1 ? rows : 4;                      // rows of a column tile that are there at all
    const int x_lanes = 8 * rt;
    const int share = S::SUMS / C;                          // of the CTA's sums, those that it finishes
    const int stage_bytes = T * P.stage_k * S::TILE;
    float *sums = (float *)(smem + P.stages * stage_bytes); // [2][16][SUMS]
    float *parts = sums + 2 * W4_WARPS * S::SUMS;           // [2][C][share]
    float *xrow = parts + (C > 1 ? 2 * S::SUMS : 0);        // [k_cta][NT * 4]
    uint4 *zeros = (uint4 *)(xrow + P.k_cta * NT * 4);      // 32 bytes
    uint4 *xf = zeros + 2;                                  // [k_cta][NT][x_lanes][2]
    // this CTA's inputs
    const int k0 = (int)((long long)P.k_tiles * rank / C), k1 = (int)((long long)P.k_tiles * (rank + 1) / C);
    // group of a tile: by a product with 2^32 / per_group, exact for the 1024 tiles there can be (0: every tile is one)
    auto sz_group = [&](int kt) { return G32 ? 2 * kt : P.group_magic ? (int)__umulhi((uint32_t)kt, P.group_magic) : kt; };

    mx::pdl_trigger();
    if (C > 1) mx::cluster_arrive_relaxed();   // waited for before the first store to another CTA's memory
    if (tid < 2) zeros[tid] = make_uint4(0, 0, 0, 0);
    if (tid == 0) {
        aborted = 0, stop_grp = 0x7FFFFFFF;
        for (int i = 0; i < P.stages; ++i) mx::mbar_init(mx::smem_u32(&full[i]), 1), mx::mbar_init(mx::smem_u32(&empty[i]), W4_WARPS);
        mx::mbar_fence_init();
    }
    __syncthreads();
    mx::pdl_wait();

    if (warp == W4_WARPS) {
        // ---- producer: the tiles of every group, stage by stage (lane 0).  In clusters the warp counts in the barrier at every group's
        // end: it arrives once the group's stages are requested, and waits for the barrier only before it arrives at the next one ----
        int stage = 0, parity = 1, count = 0;
        bool on = true;
        for (int grp = grp0; grp < P.n_groups; grp += P.n_clusters) {
            if (lane == 0 && on)
                for (int k = k0; k < k1; k += P.stage_k) {
                    if ((count == P.test_drop_tile && blockIdx.x == 0 && blockIdx.y == 0) ||
                        !mx::mbar_wait(mx::smem_u32(&empty[stage]), parity, &aborted, P.status)) {
                        on = false;   // (what was requested is waited for by those who read it)
                        stop_k = k;
                        __threadfence_block();
                        stop_grp = grp;
                        break;
                    }
                    ++count;
                    const int n = min(P.stage_k, k1 - k), here = min(T, P.n_tiles - grp * T);
                    const int g_first = sz_group(k), g_last = G32 ? min(2 * (k + n), P.groups) : sz_group(k + n - 1) + 1;
                    const uint32_t bar = mx::smem_u32(&full[stage]), sz_bytes = (uint32_t)(g_last - g_first) * 64;
                    uint32_t dst = mx::smem_u32(smem + stage * stage_bytes);
                    mx::mbar_expect_tx(bar, here * (n * 512 + sz_bytes));
                    for (int t = 0; t < here; ++t, dst += P.stage_k * S::TILE) {
                        const size_t nt = (size_t)grp * T + t;
                        mx::bulk_load(dst, P.codes + (nt * P.k_tiles + k) * 32, n * 512, bar);
                        mx::bulk_load(dst + P.stage_k * 512, P.sz + (nt * P.groups + g_first) * 16, sz_bytes, bar);
                    }
                    if (++stage == P.stages) stage = 0, parity ^= 1;
                }
            __syncwarp();
            if (C > 1) {
                mx::cluster_wait();
                mx::cluster_arrive_release();
            }
        }
        if (C > 1) mx::cluster_wait();
        return;
    }
    auto sync = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(W4_THREADS) : "memory"); };

    // ---- rows: scaled, split, in the order of B's fragments.  A thread takes the 16 inputs (8j .. , 32 + 8j ..) of a (tile, row); the
    // four of a row follow one another ----
    {
        const int rr = NT == 1 ? rt : 4 * NT, n_x = (k1 - k0) * rr * 4;
        for (int i0 = tid & ~31; i0 < n_x; i0 += W4_THREADS) {   // (whole warps, for the shuffles)
            const int i = min(i0 + lane, n_x - 1);
            const int jj = i & 3, q = (i >> 2) / rr, r = (i >> 2) - q * rr, kt = k0 + q;
            const bool in = i0 + lane < n_x && r < rows;
            float v[16];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const int k = kt * W4_K + hf * 32 + 8 * jj;
                const float *src = P.x + (long long)(row0 + r) * P.x_stride + k;
                if (in && P.x_vec && k + 8 <= P.n_in) {
                    *(float4 *)&v[8 * hf] = *(const float4 *)src, *(float4 *)&v[8 * hf + 4] = *(const float4 *)(src + 4);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[8 * hf + e] = in && k + e < P.n_in ? src[e] : 0.0f;
                }
            }
            float amax = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(v[e]));
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
            const bool infinite = amax == INFINITY;
            if (infinite) {   // the largest finite one, of the row's four lanes, which are all here; infinite ones go in as they are
                amax = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; ++e) amax = fmaxf(amax, isinf(v[e]) ? 0.0f : fabsf(v[e]));
                amax = fmaxf(amax, __shfl_xor_sync(0xFu << (lane & 28), amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xFu << (lane & 28), amax, 2));
            }
            // e = 14 - exponent of amax; 2^e and 2^-e by their bits
            const int eb = max((int)(__float_as_uint(amax) >> 23), 15);
            const float up = __uint_as_float((uint32_t)(268 - eb) << 23), down = __uint_as_float((uint32_t)(eb - 14) << 23);
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] *= up;
            if (i0 + lane >= n_x) continue;
            if (jj == 0) xrow[q * (NT * 4) + r] = down;
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float a = v[2 * e], b = v[2 * e + 1];
                const __half2 h = __floats2half2_rn(a, b);
                const float2 back = __half22float2(h);
                float low_a = a - back.x, low_b = b - back.y;
                if (infinite) low_a = isinf(a) ? 0.0f : low_a, low_b = isinf(b) ? 0.0f : low_b;
                hi[e] = h2_u(h), lo[e] = h2_u(__floats2half2_rn(low_a, low_b));
            }
            // lanes of columns 2 (r % 4) and 2 (r % 4) + 1; pairs 0 .. 3 of each half of the tile: MMA steps 2 hf, 2 hf + 1
            uint4 *dst = xf + ((size_t)(q * NT + (r >> 2)) * x_lanes + (r & 3) * 8 + jj) * 2;
            dst[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]), dst[1] = make_uint4(hi[4], hi[5], hi[6], hi[7]);
            dst[8] = make_uint4(lo[0], lo[1], lo[2], lo[3]), dst[9] = make_uint4(lo[4], lo[5], lo[6], lo[7]);
        }
    }
    sync();
    if (C > 1) mx::cluster_wait();
    const bool has_x = lane < x_lanes;                        // columns of rows that are not there: zeros
    const int x_n = has_x ? x_lanes * 2 : 0, x_step = KW * NT * x_n, tile_bytes = P.stage_k * S::TILE;
    int stage = 0, parity = 0, buf = 0;
    bool late = false;
    for (int grp = grp0; grp < P.n_groups; grp += P.n_clusters) {
        float total[T][NT][2];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) total[t][n][0] = total[t][n][1] = 0.0f;
        const uint4 *xp = has_x ? xf + ((size_t)warp * NT * x_lanes + lane) * 2 : zeros;
        const float *rp = xrow + warp * (NT * 4) + (NT == 1 ? min(j, rt - 1) : j);   // the row that this lane has
        for (int k = k0; k < k1; k += P.stage_k) {
            const uint32_t bar = mx::smem_u32(&full[stage]);
            if (!mx::mbar_wait(bar, parity, &aborted, P.status)) {
                // (its copies, if they are requested, still land here: it goes on once they have, and its sums do not count)
                for (const long long since = clock64(); !mx::mbar_try_wait(bar, parity) && clock64() - since < mx::LANDING_CYCLES;)
                    if (stop_grp < grp || (stop_grp == grp && stop_k <= k)) break;
                late = true;
            }
            const unsigned char *base = smem + stage * stage_bytes;
            const int end = min(k1, k + P.stage_k), g_first = sz_group(k);
            for (int kt = k + warp; kt < end; kt += KW) {
                const unsigned char *at = base + (kt - k) * 512;
                const uint32_t *sz = (const uint32_t *)(base + P.stage_k * 512) + (sz_group(kt) - g_first) * 16 + g;
                uint4 b[NT][2];
                float back[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    b[n][0] = xp[n * x_n], b[n][1] = xp[n * x_n + 1];
                    back[n] = rp[n * 4];
                }
                xp += x_step, rp += KW * NT * 4;
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const uint4 w = *(const uint4 *)(at + t * tile_bytes + lane * 16);
                    float acc[NT][4];
                    float s0, s1;   // scales of the lane's two outputs
                    __half2 z0, z1;
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        if (G32 || hf == 0) {
                            // (a second group of 32 that is not there belongs to inputs that are not there either: s = z = 0)
                            const bool there = !G32 || hf == 0 || 2 * kt + 1 < P.groups;
                            const uint32_t *z = sz + t * (tile_bytes / 4) + (G32 ? hf * 16 : 0);
                            const __half2 w0 = u_h2(there ? z[0] : 0), w1 = u_h2(there ? z[8] : 0);
                            s0 = __low2float(w0), s1 = __low2float(w1), z0 = __high2half2(w0), z1 = __high2half2(w1);
                        }
                        uint32_t a0[4], a1[4];
                        pairs8(hf ? w.y : w.x, z0, a0);
                        pairs8(hf ? w.w : w.z, z1, a1);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (G32 || hf == 0) mma_f16_first(acc[n], a0[0], a1[0], a0[1], a1[1], b[n][hf].x, b[n][hf].y);
                            else mma_f16(acc[n], a0[0], a1[0], a0[1], a1[1], b[n][hf].x, b[n][hf].y);
                            mma_f16(acc[n], a0[2], a1[2], a0[3], a1[3], b[n][hf].z, b[n][hf].w);
                        }
                        if (G32 || hf == 1)
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                total[t][n][0] = fmaf(s0, (acc[n][0] + acc[n][1]) * back[n], total[t][n][0]);
                                total[t][n][1] = fmaf(s1, (acc[n][2] + acc[n][3]) * back[n], total[t][n][1]);
                            }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mx::mbar_arrive(mx::smem_u32(&empty[stage]));
            if (++stage == P.stages) stage = 0, parity ^= 1;
        }
        // ---- slices of the CTA, then of the cluster, pairwise; each CTA of it finishes a share ----
        float *mine = sums + buf * W4_WARPS * S::SUMS;
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) mine[warp * S::SUMS + ((t * NT + n) * 2 + e) * 32 + lane] = late ? NAN : total[t][n][e];
        sync();
        float *theirs = parts + buf * S::SUMS;
        if (C > 1) {
            for (int i = tid; i < S::SUMS; i += W4_THREADS) {
                const float v = tree_sum(mine + i, KW, S::SUMS);
                const int to = i / share;
                const uint32_t dst = mx::cluster_map(mx::smem_u32(theirs + rank * share + i - to * share), to);
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(v) : "memory");
            }
            mx::cluster_sync();
        }
        for (int i = rank * share + tid; i < (rank + 1) * share; i += W4_THREADS) {
            const int l = i & 31, hf = (i >> 5) & 1, n = (i >> 6) % NT, t = (i >> 6) / NT;
            float v = C > 1 ? tree_sum(theirs + i - rank * share, C, share) : tree_sum(mine + i, KW, S::SUMS);
            const int o = (grp * T + t) * W4_N + (l >> 2) + 8 * hf, r = n * 4 + (l & 3);
            if (o < P.n_out && r < rows) {
                v *= 0x1p10f;   // (sums of (q - z) 2^-10)
                float out = P.bias ? v + P.bias[o] : v;
                if (P.add) out = P.add[(long long)(row0 + r) * P.add_stride + o] + out;
                P.y[(long long)(row0 + r) * P.y_stride + o] = out;
            }
        }
        // (the sums of the group before last are read by nobody any more: its barrier is behind all of them)
        buf ^= 1;
    }
}

// Clusters of C CTAs that the device holds at once, each of which fills an SM (asked once per size, of any form of the kernel).
int clusters_held(mx230_handle *h, int C, int *held) {
    static int fit[64][4];
    const int size = C == 2 ? 1 : C == 4 ? 2 : 3;
    *held = h->sm_count;
    if (C == 1) return MX230_OK;
    if (h->device >= 64 || fit[h->device][size] == 0) {
        MX_SMEM_ATTR_ONCE(h->device, (gemv_int4_kernel<1, 1, false>), W4_SMEM);
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute at;
        cfg.gridDim = dim3(C), cfg.blockDim = dim3(W4_THREADS + W4_PRODUCER), cfg.dynamicSmemBytes = W4_SMEM, cfg.attrs = &at, cfg.numAttrs = 1;
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = C, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
        MX_CHECK_CUDA(cudaOccupancyMaxActiveClusters(held, gemv_int4_kernel<1, 1, false>, &cfg));
        if (*held < 1) *held = 1;
        if (h->device < 64) fit[h->device][size] = *held;
    } else *held = fit[h->device][size];
    return MX230_OK;
}

// What comes before the ring in shared memory: rows and sums.
size_t fixed_bytes(const Int4Params &P, int x_tile, int sums) {
    return (size_t)2 * (W4_WARPS + (P.ctas_k > 1 ? 1 : 0)) * sums * 4 + 32 + (size_t)P.k_cta * x_tile;
}

template <int NT, int T, bool G32>
int launch_int4(mx230_handle *h, cudaStream_t st, Int4Params P, int x_tile, int held) {
    using S = Int4Form<NT, T, G32>;
    P.n_groups = (P.n_tiles + T - 1) / T;
    // Shared memory: rows and sums, and what is left for stages, of four tiles a warp where three of them fit, or two, or one (a whole
    // number of turns; 4096 x 128000, one row: four take a tenth less than two).
    const size_t fixed = fixed_bytes(P, x_tile, S::SUMS);
    P.stage_k = 4 * W4_WARPS;
    while (P.stage_k > W4_WARPS && fixed + (size_t)(P.stage_k == 2 * W4_WARPS ? 2 : 3) * T * P.stage_k * S::TILE > W4_SMEM) P.stage_k /= 2;
    if (P.stage_k > P.k_cta) P.stage_k = P.k_cta;
    const size_t stage = (size_t)T * P.stage_k * S::TILE;
    MX_REQUIRE(fixed + 2 * stage <= W4_SMEM, MX230_ERR_UNSUPPORTED, "gemv_int4: %d inputs a CTA and two stages do not fit shared memory", P.k_cta * W4_K);
    P.stages = (int)((W4_SMEM - fixed) / stage);
    if (P.stages > W4_STAGES) P.stages = W4_STAGES;
    const size_t sm = fixed + P.stages * stage;
    MX_SMEM_ATTR_ONCE(h->device, (gemv_int4_kernel<NT, T, G32>), W4_SMEM);
    P.n_clusters = held < P.n_groups ? held : P.n_groups;
    const dim3 grid((unsigned)(P.n_clusters * P.ctas_k), (unsigned)((P.n_rows + 4 * NT - 1) / (4 * NT)));
    MX_LAUNCH(h, st, MX230_K_GEMV_INT4, mx_launch(gemv_int4_kernel<NT, T, G32>, grid, W4_THREADS + W4_PRODUCER, sm, st, P.ctas_k, true, P));
    return MX230_OK;
}

int check_shape(const char *who, int n_in, int n_out, int group) {
    MX_REQUIRE(n_in > 0 && n_out > 0, MX230_ERR_INVALID_ARG, "%s: n_in %d, n_out %d", who, n_in, n_out);
    MX_REQUIRE(group == 32 || (group > 0 && group % 64 == 0), MX230_ERR_UNSUPPORTED, "%s: groups of %d inputs (32, or a multiple of 64)", who, group);
    return MX230_OK;
}

size_t codes_bytes(int n_in, int n_out) {
    return (size_t)((n_out + (long long)W4_N - 1) / W4_N) * (size_t)((n_in + (long long)W4_K - 1) / W4_K) * 512;
}

}  // namespace

extern "C" size_t mx230_int4_bytes(int n_in, int n_out, int group) {
    if (n_in <= 0 || n_out <= 0 || group <= 0) return 0;
    return codes_bytes(n_in, n_out) + (size_t)((n_out + (long long)W4_N - 1) / W4_N) * (size_t)((n_in + (long long)group - 1) / group) * 64;
}

extern "C" int mx230_pack_int4(mx230_handle *h, void *stream, void *packed, const uint8_t *codes, const void *scales,
                               const uint8_t *zeros, int n_in, int n_out, int group) {
    MX_REQUIRE(h && packed && codes && scales, MX230_ERR_INVALID_ARG, "pack_int4: null argument");
    int rc = check_shape("pack_int4", n_in, n_out, group);
    if (rc) return rc;
    MX_REQUIRE(((uintptr_t)packed & 15) == 0 && ((uintptr_t)scales & 1) == 0, MX230_ERR_INVALID_ARG, "pack_int4: misaligned pointer");
    mx230_device_guard guard(h->device);
    cudaStream_t st = (cudaStream_t)stream;
    const int n_tiles = (int)((n_out + (long long)W4_N - 1) / W4_N), k_tiles = (int)((n_in + (long long)W4_K - 1) / W4_K);
    const int groups = (int)((n_in + (long long)group - 1) / group);
    const long long work = (long long)n_tiles * k_tiles * 32 + (long long)n_tiles * groups * 16;
    const long long blocks = (work + 255) / 256, most = 64ll * h->sm_count;
    MX_LAUNCH(h, st, MX230_K_PACK_INT4, (pack_int4_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, st>>>(
        (uint4 *)packed, (uint32_t *)((char *)packed + codes_bytes(n_in, n_out)), codes, (const __half *)scales, zeros, n_in, n_out, group,
        n_tiles, k_tiles, groups)));
    return MX230_OK;
}

extern "C" int mx230_gemv_int4(mx230_handle *h, void *stream, float *y, const float *x, const void *packed, const float *bias,
                               const float *add, int n_rows, int n_in, int n_out, int group, long long x_stride,
                               long long y_stride, long long add_stride) {
    MX_REQUIRE(h, MX230_ERR_INVALID_ARG, "gemv_int4: null handle");
    int rc = check_shape("gemv_int4", n_in, n_out, group);
    if (rc) return rc;
    MX_REQUIRE(n_rows >= 0, MX230_ERR_INVALID_ARG, "gemv_int4: %d rows", n_rows);
    if (n_rows == 0) return MX230_OK;
    MX_REQUIRE(y && x && packed, MX230_ERR_INVALID_ARG, "gemv_int4: null argument");
    MX_REQUIRE(n_rows < 2 || (x_stride >= 0 && y_stride >= n_out && (add == nullptr || add_stride >= 0)), MX230_ERR_INVALID_ARG,
               "gemv_int4: rows of y share memory, or a stride is negative (x %lld, y %lld, add %lld)", x_stride, y_stride, add_stride);
    MX_REQUIRE(((uintptr_t)packed & 15) == 0 && (((uintptr_t)x | (uintptr_t)y | (uintptr_t)bias | (uintptr_t)add) & 3) == 0, MX230_ERR_INVALID_ARG,
               "gemv_int4: misaligned pointer");
    MX_REQUIRE(add != y || n_rows < 2 || add_stride == y_stride, MX230_ERR_INVALID_ARG, "gemv_int4: add is y, with another stride");
    MX_REQUIRE(n_rows <= 65535 * 4, MX230_ERR_UNSUPPORTED, "gemv_int4: %d rows", n_rows);
    MX_REQUIRE(n_in <= 2 * W4_K_CTA * W4_CLUSTER * W4_K, MX230_ERR_UNSUPPORTED, "gemv_int4: n_in %d (at most %d)", n_in, 2 * W4_K_CTA * W4_CLUSTER * W4_K);
    auto rows_of = [&](const void *at, int n, long long stride) {
        return Pieces{at, (size_t)n * 4, 1, 0, n_rows, n_rows < 2 ? 0 : (long long)((unsigned long long)stride * 4)};
    };
    const Pieces out = rows_of(y, n_out, y_stride);
    MX_REQUIRE(!pieces_overlap(out, rows_of(x, n_in, x_stride)), MX230_ERR_INVALID_ARG, "gemv_int4: y shares memory with x, which other blocks still read");
    MX_REQUIRE(bias == nullptr || !pieces_overlap(out, {bias, (size_t)n_out * 4, 1, 0, 1, 0}), MX230_ERR_INVALID_ARG, "gemv_int4: y shares memory with the bias");
    MX_REQUIRE(add == nullptr || add == y || !pieces_overlap(out, rows_of(add, n_out, add_stride)), MX230_ERR_INVALID_ARG,
               "gemv_int4: add shares memory with y, but is not y");
    MX_REQUIRE(!pieces_overlap(out, {packed, mx230_int4_bytes(n_in, n_out, group), 1, 0, 1, 0}), MX230_ERR_INVALID_ARG, "gemv_int4: y shares memory with the weights");
    Int4Params P{};
    P.y = y, P.x = x, P.bias = bias, P.add = add;
    P.codes = (const uint4 *)packed, P.sz = (const uint32_t *)((const char *)packed + codes_bytes(n_in, n_out));
    P.n_rows = n_rows, P.n_in = n_in, P.n_out = n_out, P.group = group;
    P.groups = (int)((n_in + (long long)group - 1) / group);
    P.n_tiles = (int)((n_out + (long long)W4_N - 1) / W4_N), P.k_tiles = (int)((n_in + (long long)W4_K - 1) / W4_K);
    P.x_stride = x_stride, P.y_stride = y_stride, P.add_stride = add_stride;
    P.x_vec = ((uintptr_t)x & 15) == 0 && (n_rows < 2 || x_stride % 4 == 0);
    P.status = h->status_dev, P.test_drop_tile = h->test_drop_tile;
    const unsigned long long per_group = group == 32 ? 1 : group / W4_K;
    P.group_magic = per_group == 1 ? 0 : (uint32_t)(((1ull << 32) + per_group - 1) / per_group);
    // Inputs over CTAs so that a CTA's rows fit its shared memory, and where there are few output tiles.  This fixes the order of the sums.
    P.ctas_k = 1;
    while (P.ctas_k < W4_CLUSTER && (P.k_tiles > W4_K_CTA * P.ctas_k || (P.k_tiles >= 64 * P.ctas_k && (long long)P.n_tiles * P.ctas_k < h->sm_count))) P.ctas_k *= 2;
    P.k_cta = (P.k_tiles + P.ctas_k - 1) / P.ctas_k;
    // Rows of a pass: eight, or four where eight do not fit.
    const int nt = n_rows <= 4 || P.k_cta > W4_K_CTA ? 1 : 2, x_tile = nt * (32 * (nt == 1 ? 8 * (n_rows < 4 ? n_rows : 4) : 32) + 16);
    mx230_device_guard guard(h->device);
    int held;
    rc = clusters_held(h, P.ctas_k, &held);
    if (rc) return rc;
    const bool g32 = group == 32;
    // Output tiles of a warp, which share what is read of the rows.  Up to two rows: one, two or four, whichever needs least time, taken as
    // rounds of the clusters times 3, 5 or 9; three and four rows: one or two.  One row, us with one / two / four: 896 x 1152 2.2, 2.4, 3.0;
    // 4096 x 4096 5.2, 5.0, 6.3; 4096 x 14336 11.9, 11.7, 11.8; 14336 x 4096 17.5, 13.8, 12.2; 4096 x 128000 75, 65, 62 (four rows 78, 67, 73;
    // 14336 x 4096 18.4, 14.5, 14.0).  Eight rows: two where there is a round of them and three stages fit beside the rows (14336 x 4096
    // 26.4, 20.0; 4096 x 14336 19.3, 18.7; in groups of 32, where two stages would, 20.5, 21.5).
    int t = 1;
    if (nt == 1) {
        const int cost[3] = {30, 50, 89};
        long long best = 0;
        for (int i = 0; i < (n_rows < 3 ? 3 : 2); ++i) {
            const long long groups = (P.n_tiles + (1 << i) - 1) >> i, time = (groups + held - 1) / held * cost[i];
            if (i == 0 || time < best) best = time, t = 1 << i;
        }
    } else if (P.n_tiles > held) {
        const size_t stage = (size_t)2 * W4_WARPS * (g32 ? Int4Form<2, 2, true>::TILE : Int4Form<2, 2, false>::TILE);
        if (fixed_bytes(P, x_tile, Int4Form<2, 2, false>::SUMS) + 3 * stage <= W4_SMEM) t = 2;
    }
    cudaStream_t st = (cudaStream_t)stream;
    if (nt == 1) {
        if (t == 4) return g32 ? launch_int4<1, 4, true>(h, st, P, x_tile, held) : launch_int4<1, 4, false>(h, st, P, x_tile, held);
        if (t == 2) return g32 ? launch_int4<1, 2, true>(h, st, P, x_tile, held) : launch_int4<1, 2, false>(h, st, P, x_tile, held);
        return g32 ? launch_int4<1, 1, true>(h, st, P, x_tile, held) : launch_int4<1, 1, false>(h, st, P, x_tile, held);
    }
    if (t == 2) return g32 ? launch_int4<2, 2, true>(h, st, P, x_tile, held) : launch_int4<2, 2, false>(h, st, P, x_tile, held);
    return g32 ? launch_int4<2, 1, true>(h, st, P, x_tile, held) : launch_int4<2, 1, false>(h, st, P, x_tile, held);
}
