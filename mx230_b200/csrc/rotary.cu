// Rotary positions of one part of a program's heads, in the forms that mx230_rope* (the reference's: whole heads of fp32, pairs
// half a head apart, one base) does not have: pairs half the rotated part apart or next to each other, a part of the head, angles
// stretched for contexts longer than the trained one, fp32 / fp16 / bf16, any strides, and the way back for a gradient.
//
//   pair i of row r:  a' = (a cos - b sin) f,  b' = (a sin + b cos) f,   angle = pos[r] * freq[i]   (inverse: -angle)
//
// The inverse is the transposed matrix, so it carries a gradient back through the forward call.
//
// Angles: a frequency is held as a whole number of 2^-64 turns per position.  pos * turns modulo 2^64 is then the exact remainder
// of the angle modulo a turn, for any position and with one integer product; what is rounded is the remainder, to 2^-27 turns at
// an eighth of a turn.  (fp32 products pos * freq are off by 0.03 rad at position 10^6.)
//
// Bounded by HBM: every element is read once and written once.  A block takes a few rows: the angles of all their pairs go into
// shared memory, once for all heads (a head of its own would have 25 instructions of angle per element of 16 bits), then each
// thread moves 16-byte pieces with the same pairs of many heads.  16384 rows of 40 heads of 128, bf16: 64 us, 0.81 of the measured copy;
// 1900 of 36 heads of 64, fp32: 8.3, 0.65; one head a row leaves the angles to be the work (32768 rows of 128, fp32: 14 us, 0.36).
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "pieces.h"

namespace {

constexpr int RT_THREADS = 256;
constexpr int RT_PAIRS = 2048;    // angles in shared memory, most
constexpr int RT_UNROLL = 2;      // heads whose loads a thread has in flight

struct RotaryParams {
    void *out;
    const void *x;
    const int *pos;              // per row, or null: pos0 + row
    int pos0;
    const uint64_t *turns;       // [half]
    float factor;
    int n_rows, n_head, head_dim, half, inverse;
    int rows_per_block, heads_per_block;
    int units, slots;            // pieces of a head; heads that a block moves at a time
    long long x_row, x_head, out_row, out_head;   // in elements
};

// N elements of T, loaded and stored together, and as floats (16-bit ones by twos)
template <typename T, int N>
struct alignas(sizeof(T) * N) Piece {
    T v[N];
};
template <int N>
__device__ __forceinline__ void unpack(const Piece<float, N> &p, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = p.v[i];
}
template <int N>
__device__ __forceinline__ void pack(Piece<float, N> &p, const float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) p.v[i] = f[i];
}
template <int N>
__device__ __forceinline__ void unpack(const Piece<__half, N> &p, float (&f)[N]) {
    if constexpr (N == 1) f[0] = __half2float(p.v[0]);
    else
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 t = __half22float2(*(const __half2 *)&p.v[i]);
            f[i] = t.x, f[i + 1] = t.y;
        }
}
template <int N>
__device__ __forceinline__ void pack(Piece<__half, N> &p, const float (&f)[N]) {
    if constexpr (N == 1) p.v[0] = __float2half_rn(f[0]);
    else
#pragma unroll
        for (int i = 0; i < N; i += 2) *(__half2 *)&p.v[i] = __floats2half2_rn(f[i], f[i + 1]);
}
template <int N>
__device__ __forceinline__ void unpack(const Piece<__nv_bfloat16, N> &p, float (&f)[N]) {
    if constexpr (N == 1) f[0] = __bfloat162float(p.v[0]);
    else
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint32_t w = *(const uint32_t *)&p.v[i];
            f[i] = __uint_as_float(w << 16), f[i + 1] = __uint_as_float(w & 0xFFFF0000u);
        }
}
template <int N>
__device__ __forceinline__ void pack(Piece<__nv_bfloat16, N> &p, const float (&f)[N]) {
    if constexpr (N == 1) p.v[0] = __float2bfloat16_rn(f[0]);
    else
#pragma unroll
        for (int i = 0; i < N; i += 2) *(uint32_t *)&p.v[i] = mx::pack_bf16(f[i], f[i + 1]);
}

// cos and sin of `t` * 2^-64 turns: the nearest quarter turn is taken off as an integer, so that what is left has 27 bits behind
// the point as a float, and put back by exchanging and negating.
__device__ __forceinline__ float2 turn_cos_sin(uint64_t t) {
    const uint32_t hi = (uint32_t)(t >> 32), q = (hi + 0x20000000u) >> 30;
    float s, c;
    sincospif((float)(int)(hi - (q << 30)) * 0x1p-31f, &s, &c);
    if (q & 1) {
        const float k = c;
        c = -s, s = k;
    }
    return (q & 2) ? make_float2(-c, -s) : make_float2(c, s);
}

// N: elements of a piece.  Pairs half apart: unit u < half / N is a piece of the lower and the matching one of the upper half, units
// behind are pieces of what is not rotated.  INTER: unit u is a piece of the head; N == 1 stands for pairs (and single elements of
// the rest) by themselves, in either layout.  IN_PLACE: what is not rotated stays as it is.
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(RT_THREADS, 4) rotary_kernel(const RotaryParams P) {
    // the angles of a row lie so that lanes with pieces next to each other read words next to each other: the first two pairs of
    // every piece, then the next two (16 rows of words apart they were read four at a time: 84 us for the interleaved case of 64)
    __shared__ __align__(16) float2 cs[RT_PAIRS];
    constexpr int PAIRS = INTER ? (N > 1 ? N / 2 : 1) : N;     // of a piece
    const int pieces = (P.half + PAIRS - 1) / PAIRS, row_cs = pieces * PAIRS;
    auto place = [&](int p) { return PAIRS == 1 ? p : (p % PAIRS / 2 * pieces + p / PAIRS) * 2 + (p & 1); };
    mx::pdl_trigger();
    mx::pdl_wait();
    const int half = P.half, tid = threadIdx.x;
    const int r0 = blockIdx.x * P.rows_per_block, nr = min(P.rows_per_block, P.n_rows - r0);
    const int h0 = blockIdx.y * P.heads_per_block, nh = min(P.heads_per_block, P.n_head - h0);
    for (int i = tid; i < nr * half; i += RT_THREADS) {
        const int r = i / half, p = i - r * half;
        const long long pos = P.pos ? (long long)P.pos[r0 + r] : (long long)P.pos0 + r0 + r;
        float2 a = turn_cos_sin((uint64_t)pos * P.turns[p]);
        a.x *= P.factor, a.y *= P.inverse ? -P.factor : P.factor;
        cs[r * row_cs + place(p)] = a;
    }
    __syncthreads();
    const T *x = (const T *)P.x;
    T *out = (T *)P.out;
    constexpr bool SINGLE = N == 1;
    const int rot_units = SINGLE || !INTER ? half / N : 0;
    const int slot = tid / P.units;
    if (slot >= P.slots) return;
    for (int u = tid - slot * P.units; u < P.units; u += RT_THREADS) {   // (more than one only where a head has more units than threads)
        // first and second piece of the unit within the head
        const bool rot = INTER && !SINGLE ? true : u < rot_units;
        const int d0 = !rot ? 2 * half + (u - rot_units) * N : SINGLE ? (INTER ? 2 * u : u) : u * N;
        const int d1 = !rot || (INTER && !SINGLE) ? d0 : SINGLE && INTER ? d0 + 1 : d0 + half;
        const bool two = d1 != d0;
        if (!rot && x == out) continue;
        if (INTER && !SINGLE && x == out && d0 >= 2 * half) continue;
        // items (row, head) of this slot: slot, slot + slots, ...
        int r = slot / nh, h = slot - r * nh;
        const int dr = P.slots / nh, dh = P.slots - dr * nh;
        const T *src = x + (long long)(r0 + r) * P.x_row + (long long)(h0 + h) * P.x_head;
        T *dst = out + (long long)(r0 + r) * P.out_row + (long long)(h0 + h) * P.out_head;
        const long long src_step = dr * P.x_row + dh * P.x_head, dst_step = dr * P.out_row + dh * P.out_head;
        const long long src_wrap = src_step + P.x_row - nh * P.x_head, dst_wrap = dst_step + P.out_row - nh * P.out_head;
        while (r < nr) {
            Piece<T, N> a[RT_UNROLL], b[RT_UNROLL];
            T *to[RT_UNROLL];
            int ri[RT_UNROLL];
#pragma unroll
            for (int k = 0; k < RT_UNROLL; ++k) {
                ri[k] = r, to[k] = dst;
                if (r < nr) {
                    a[k] = *(const Piece<T, N> *)(src + d0);
                    if (two) b[k] = *(const Piece<T, N> *)(src + d1);
                }
                r += dr, h += dh;
                const bool wrap = h >= nh;
                if (wrap) h -= nh, ++r;
                src += wrap ? src_wrap : src_step, dst += wrap ? dst_wrap : dst_step;
            }
#pragma unroll
            for (int k = 0; k < RT_UNROLL; ++k) {
                if (ri[k] >= nr) break;
                const float2 *c = cs + ri[k] * row_cs;
                float2 t[PAIRS];
                if constexpr (PAIRS == 1) {
                    if (rot) t[0] = c[INTER && !SINGLE ? min(u, half - 1) : u];
                } else if (rot) {
                    const int v = min(u, pieces - 1);   // (behind the rotated part: not used)
#pragma unroll
                    for (int q = 0; q < PAIRS; q += 2) {
                        const float4 two_pairs = *(const float4 *)(c + (q / 2 * pieces + v) * 2);
                        t[q] = make_float2(two_pairs.x, two_pairs.y), t[q + 1] = make_float2(two_pairs.z, two_pairs.w);
                    }
                }
                float f[N];
                unpack(a[k], f);
                if constexpr (INTER && !SINGLE) {
#pragma unroll
                    for (int e = 0; e + 1 < N; e += 2)
                        if ((d0 + e) >> 1 < half) mx::rope_pair(f[e], f[e + 1], t[e / 2].x, t[e / 2].y);
                    pack(a[k], f);
                } else if (rot) {
                    float g[N];
                    unpack(b[k], g);
#pragma unroll
                    for (int e = 0; e < N; ++e) mx::rope_pair(f[e], g[e], t[e].x, t[e].y);
                    pack(a[k], f), pack(b[k], g);
                }
                *(Piece<T, N> *)(to[k] + d0) = a[k];
                if (two) *(Piece<T, N> *)(to[k] + d1) = b[k];
            }
        }
    }
}

template <typename T, int N>
int launch_n(mx230_handle *h, cudaStream_t st, const RotaryParams &P, dim3 grid, bool inter) {
    if (inter) MX_LAUNCH(h, st, MX230_K_ROTARY, mx_launch(rotary_kernel<T, N, true>, grid, RT_THREADS, 0, st, 1, true, P));
    else MX_LAUNCH(h, st, MX230_K_ROTARY, mx_launch(rotary_kernel<T, N, false>, grid, RT_THREADS, 0, st, 1, true, P));
    return MX230_OK;
}

template <typename T>
int launch_t(mx230_handle *h, cudaStream_t st, RotaryParams P, bool inter) {
    // Elements of a piece: the largest power of two, up to 16 bytes, that divides every offset a piece can start at.
    const int tail = P.head_dim - 2 * P.half;
    unsigned long long any = (unsigned long long)(uintptr_t)P.x / sizeof(T) | (uintptr_t)P.out / sizeof(T);
    if (P.n_rows > 1) any |= (unsigned long long)P.x_row | (unsigned long long)P.out_row;
    if (P.n_head > 1) any |= (unsigned long long)P.x_head | (unsigned long long)P.out_head;
    any |= inter ? (unsigned long long)P.head_dim : (unsigned long long)P.half | (unsigned long long)tail;
    int n = 16 / (int)sizeof(T);
    while (n > 1 && (any & (unsigned)(n - 1))) n >>= 1;
    P.units = n == 1 ? P.half + tail : inter ? P.head_dim / n : (P.half + tail) / n;
    P.slots = P.units >= RT_THREADS ? 1 : RT_THREADS / P.units;
    // Rows and heads of a block: enough for every thread to have its heads in flight twice, unless that left SMs without a block.
    P.heads_per_block = P.n_head;
    auto parts = [](long long n, long long of) { return (n + of - 1) / of; };   // (of numbers up to the largest int)
    int rows = (int)parts(2 * RT_UNROLL * P.slots, P.n_head);
    const int fill = (int)parts(P.n_rows, 2 * h->sm_count);
    if (rows > fill) rows = fill;
    const int pairs = n == 1 ? 1 : inter ? n / 2 : n, row_cs = (P.half + pairs - 1) / pairs * pairs;
    if (rows > RT_PAIRS / row_cs) rows = RT_PAIRS / row_cs;
    if (rows < 1) rows = 1;
    P.rows_per_block = rows;
    // few rows: the heads of a row over several blocks
    while (P.heads_per_block > P.slots && parts(P.n_rows, rows) * parts(P.n_head, P.heads_per_block) < 2 * h->sm_count)
        P.heads_per_block = (int)parts(P.heads_per_block, 2);
    const dim3 grid((unsigned)parts(P.n_rows, rows), (unsigned)parts(P.n_head, P.heads_per_block));
    MX_REQUIRE(grid.y <= 65535, MX230_ERR_UNSUPPORTED, "rotary: %d heads", P.n_head);
    if constexpr (sizeof(T) == 2)
        if (n == 8) return launch_n<T, 8>(h, st, P, grid, inter);
    if (n == 4) return launch_n<T, 4>(h, st, P, grid, inter);
    if (n == 2) return launch_n<T, 2>(h, st, P, grid, inter);
    return launch_n<T, 1>(h, st, P, grid, inter);
}

}  // namespace

extern "C" int mx230_rotary_table(uint64_t *turns_host, float *factor_host, int rot_dim, double theta, int scaling, double factor,
                                  double low, double high, int length) {
    MX_REQUIRE(turns_host && factor_host, MX230_ERR_INVALID_ARG, "rotary_table: null output");
    MX_REQUIRE(rot_dim > 0 && rot_dim % 2 == 0, MX230_ERR_INVALID_ARG, "rotary_table: rotated part of %d values", rot_dim);
    MX_REQUIRE(theta > 0.0 && isfinite(theta), MX230_ERR_INVALID_ARG, "rotary_table: base %g", theta);
    MX_REQUIRE(scaling >= MX230_ROTARY_PLAIN && scaling <= MX230_ROTARY_YARN, MX230_ERR_INVALID_ARG, "rotary_table: scaling %d", scaling);
    MX_REQUIRE(scaling == MX230_ROTARY_PLAIN || (factor > 0.0 && isfinite(factor)), MX230_ERR_INVALID_ARG, "rotary_table: scaling factor %g", factor);
    const double tau = 6.283185307179586476925286766559;
    if (scaling == MX230_ROTARY_WAVELENGTH)
        MX_REQUIRE(length > 0 && low > 0.0 && high > low && isfinite(high), MX230_ERR_INVALID_ARG,
                   "rotary_table: trained length %d, %g to %g turns over it", length, low, high);
    if (scaling == MX230_ROTARY_YARN)
        MX_REQUIRE(length > 0 && low > 0.0 && high > low && isfinite(high) && theta != 1.0, MX230_ERR_INVALID_ARG,
                   "rotary_table: trained length %d, slow %g, fast %g turns over it, base %g", length, low, high, theta);
    const int half = rot_dim / 2;
    if (scaling == MX230_ROTARY_NTK && rot_dim > 2) theta *= pow(factor, rot_dim / (rot_dim - 2.0));
    double first = 0.0, last = 0.0;
    if (scaling == MX230_ROTARY_YARN) {
        // pairs that make `high` and `low` turns over the trained length
        first = floor(rot_dim * log(length / (high * tau)) / (2.0 * log(theta)));
        last = ceil(rot_dim * log(length / (low * tau)) / (2.0 * log(theta)));
        first = fmax(first, 0.0), last = fmin(last, rot_dim - 1.0);
    }
    *factor_host = scaling == MX230_ROTARY_YARN && factor > 1.0 ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
    for (int i = 0; i < half; ++i) {
        double f = pow(theta, -2.0 * i / rot_dim);
        if (scaling == MX230_ROTARY_LINEAR) f /= factor;
        if (scaling == MX230_ROTARY_WAVELENGTH) {
            const double part = fmin(1.0, fmax(0.0, (length * f / tau - low) / (high - low)));
            f = part * f + (1.0 - part) * f / factor;
        }
        if (scaling == MX230_ROTARY_YARN) {
            const double part = fmin(1.0, fmax(0.0, (i - first) / fmax(last - first, 1e-3)));
            f = part * f / factor + (1.0 - part) * f;
        }
        long double t = (long double)f / 6.283185307179586476925286766559005768L;
        t -= floorl(t);
        const long double u = roundl(ldexpl(t, 64));
        turns_host[i] = u >= 18446744073709551616.0L ? 0 : (uint64_t)u;
    }
    return MX230_OK;
}

extern "C" int mx230_rotary(mx230_handle *h, void *stream, void *out, const void *x, int dtype, const int *pos, int pos0,
                            const uint64_t *turns, float factor, int n_rows, int n_head, int head_dim, int rot_dim,
                            int interleaved, int inverse, long long x_row, long long x_head, long long out_row,
                            long long out_head) {
    MX_REQUIRE(h, MX230_ERR_INVALID_ARG, "rotary: null handle");
    MX_REQUIRE(dtype == MX230_F32 || dtype == MX230_F16 || dtype == MX230_BF16, MX230_ERR_INVALID_ARG, "rotary: element type %d", dtype);
    MX_REQUIRE(n_rows >= 0 && n_head >= 0, MX230_ERR_INVALID_ARG, "rotary: %d rows of %d heads", n_rows, n_head);
    MX_REQUIRE(head_dim > 0 && rot_dim > 0 && rot_dim % 2 == 0 && rot_dim <= head_dim, MX230_ERR_INVALID_ARG,
               "rotary: %d of %d values rotated (an even number, at most the head)", rot_dim, head_dim);
    MX_REQUIRE(rot_dim / 2 <= RT_PAIRS, MX230_ERR_UNSUPPORTED, "rotary: %d values rotated (at most %d)", rot_dim, 2 * RT_PAIRS);
    if (n_rows == 0 || n_head == 0) return MX230_OK;
    MX_REQUIRE(out && x && turns, MX230_ERR_INVALID_ARG, "rotary: null argument");
    MX_REQUIRE(x_row >= 0 && x_head >= 0 && out_row >= 0 && out_head >= 0, MX230_ERR_INVALID_ARG, "rotary: negative stride");
    // the outputs lie apart: the smaller stride spans a head, the larger one all that lies under it
    const bool heads_inside = n_rows < 2 || (n_head >= 2 && out_head <= out_row);
    {
        const long long in_s = heads_inside ? out_head : out_row, out_s = heads_inside ? out_row : out_head;
        const int in_n = heads_inside ? n_head : n_rows, out_n = heads_inside ? n_rows : n_head;
        MX_REQUIRE((in_n < 2 || in_s >= head_dim) && (out_n < 2 || out_s >= (in_n < 2 ? 0 : in_s * (in_n - 1)) + head_dim), MX230_ERR_INVALID_ARG,
                   "rotary: rows or heads of the output share memory (strides %lld and %lld)", out_row, out_head);
    }
    MX_REQUIRE(x != out || ((n_rows < 2 || x_row == out_row) && (n_head < 2 || x_head == out_head)), MX230_ERR_INVALID_ARG,
               "rotary: in place, but x and out have different strides");
    const size_t size = dtype == MX230_F32 ? 4 : 2;
    MX_REQUIRE(((uintptr_t)x | (uintptr_t)out) % size == 0 && (uintptr_t)turns % 8 == 0 && (uintptr_t)pos % 4 == 0, MX230_ERR_INVALID_ARG,
               "rotary: misaligned pointer");
    if (x != out) {
        auto heads_of = [&](const void *at, long long row, long long head) {
            row = (long long)((unsigned long long)row * size), head = (long long)((unsigned long long)head * size);
            return heads_inside ? Pieces{at, head_dim * size, n_head, head, n_rows, row} : Pieces{at, head_dim * size, n_rows, row, n_head, head};
        };
        MX_REQUIRE(!pieces_overlap(heads_of(out, out_row, out_head), heads_of(x, x_row, x_head)), MX230_ERR_INVALID_ARG,
                   "rotary: out shares memory with x, which other blocks still read, but is not x");
    }
    RotaryParams P{};
    P.out = out, P.x = x, P.pos = pos, P.pos0 = pos0, P.turns = turns, P.factor = factor;
    P.n_rows = n_rows, P.n_head = n_head, P.head_dim = head_dim, P.half = rot_dim / 2, P.inverse = inverse ? 1 : 0;
    P.x_row = x_row, P.x_head = x_head, P.out_row = out_row, P.out_head = out_head;
    mx230_device_guard guard(h->device);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == MX230_F32) return launch_t<float>(h, st, P, interleaved != 0);
    if (dtype == MX230_F16) return launch_t<__half>(h, st, P, interleaved != 0);
    return launch_t<__nv_bfloat16>(h, st, P, interleaved != 0);
}
