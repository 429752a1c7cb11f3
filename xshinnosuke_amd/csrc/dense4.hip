// Products of rows with weights held in 4 bits, a float16 scale for each group of inputs and output.
//
//   y[m][n] = sum_g scale[g][n] sum_{k in g} x[m][k] c[k][n]  (+ bias[n]),   c a whole number in -8 .. 7
//
// The weights lie as the matrix instructions want them: a lane's 16 bytes of a chunk of 128 inputs are its operand of four
// 16 x 16 x 32 multiplications, and a wave's load of them is 1 KB in a row.  The inner sums run on the matrix cores
// with c as it is: as float16, in which it is exact, or as an 8-bit number times sixteen.  float32 rows are split into two float16 values
// after they have been scaled by a power of two that takes the row's largest value below 2^15: off by 2^-22 of the value at
// most, and where a part is too small for float16 by 2^-28 of the row's largest value; float32 sums of such products are as far off.
// Rows of 8-bit numbers give whole sums, exact in 32 bits.
#include "xsmi_internal.h"
#include <math.h>

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef f4 f4u __attribute__((aligned(4)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef int i2 __attribute__((ext_vector_type(2)));
typedef i2 i2u __attribute__((aligned(1)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// Eight weights as float16, in the order 0 4 1 5 2 6 3 7: with the sign turned into an offset a code's four bits are the low
// bits of the float16 1024 + c + 8, or, four places up, of 64 + c + 8; taking 1032 or 72 off is exact.
__device__ __forceinline__ h8 weights_f16(uint32_t w) {
    uint32_t low = 0x000f000fu, high = 0x00f000f0u, at10 = 0x64006400u, at6 = 0x54005400u;
    asm("" : "+s"(low), "+s"(high), "+v"(at10), "+v"(at6));      // registers: an instruction takes one constant or scalar
    const uint32_t u = w ^ 0x88888888u, v = u >> 8;
    const h2 far = {(_Float16)1032.f, (_Float16)1032.f}, near = {(_Float16)72.f, (_Float16)72.f};
    const h2 a = __builtin_bit_cast(h2, (u & low) | at10) - far;
    const h2 b = __builtin_bit_cast(h2, (u & high) | at6) - near;
    const h2 c = __builtin_bit_cast(h2, (v & low) | at10) - far;
    const h2 d = __builtin_bit_cast(h2, (v & high) | at6) - near;
    return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Eight weights times sixteen as bytes, in the order 0 2 4 6 1 3 5 7.
__device__ __forceinline__ u2 weights_i8(uint32_t w) { return u2{(w << 4) & 0xf0f0f0f0u, w & 0xf0f0f0f0u}; }

// Eight values of a row, already scaled, as the two float16 parts of each, in the order of weights_f16.  An infinity or NaN
// has no second part.
__device__ __forceinline__ void split8(const float *x, h8 &hi, h8 &lo) {
    constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float v = x[order[e]];
        hi[e] = (_Float16)v;
        const float rest = v - (float)hi[e];
        lo[e] = (_Float16)(fabsf(v) < INFINITY ? rest : 0.f);
    }
}

__device__ __forceinline__ u2 order_i8(i2 x) {       // eight bytes in the order of weights_i8
    return u2{__builtin_amdgcn_perm((uint32_t)x.y, (uint32_t)x.x, 0x06040200u), __builtin_amdgcn_perm((uint32_t)x.y, (uint32_t)x.x, 0x07050301u)};
}

// The power of two that takes values up to `most` (its bits) below 2^15, and the one that takes them back.
__device__ __forceinline__ float scale_up(uint32_t most) {
    const int e = (int)(most >> 23);
    return __uint_as_float((uint32_t)min(268 - e, 254) << 23);
}
__device__ __forceinline__ float scale_down(uint32_t most) {
    const int e = (int)(most >> 23);
    return ldexpf(1.f, max(e - 141, -127));
}
__device__ __forceinline__ uint32_t size_bits(float v) {     // of a finite value; 0 of one that is not
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}

__device__ __forceinline__ void load8(const float *x, int k, int K, float *v) {
    if (k + 8 <= K) {
        const f4 a = *reinterpret_cast<const f4u *>(x + k), b = *reinterpret_cast<const f4u *>(x + k + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k + e < K ? x[k + e] : 0.f;
}
__device__ __forceinline__ i2 load8(const int8_t *x, int k, int K) {
    if (k + 8 <= K) return *reinterpret_cast<const i2u *>(x + k);
    uint32_t r[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (k + e < K) r[e >> 2] |= (uint32_t)(uint8_t)x[k + e] << (8 * (e & 3));
    return i2{(int)r[0], (int)r[1]};
}

struct Dense {
    const void *x;
    const float *x_scale;                            // of 8-bit rows
    const uint8_t *codes;
    const _Float16 *scales;
    const float *bias;
    float *y;
    int M, K, N, chunks, cols;                       // chunks of 128 inputs, outputs up to a multiple of 16
};

// ---- few rows ----------------------------------------------------------------------------------------------------
// All products are of 8-bit numbers here: weights times sixteen take three operations for eight of them, a quarter of what
// float16 takes, and one row leaves that as the bound beside memory.  A float32 row becomes four rows of 8-bit digits: scaled by a
// power of two to whole numbers below 2^30 and written in base 256 with signed digits, its sums are exact within a group and the
// rows off by 2^-31 of the largest value at most.
//
// A workgroup of eight waves has 16 NT outputs and splits their inputs over its waves, chunk by chunk.  Each wave lays the rows'
// part of its own PF chunks of a window out in its own stretch of LDS, by powers of two of its own, so that the waves meet
// only where their sums are added at the end.  The loads of the next window are under way while one is multiplied.
constexpr int WAVES = 8;

// Eight whole numbers as four octets of digits, lowest first, in the order of weights_i8.
__device__ __forceinline__ void digits8(const int *x, u2 *to) {
    uint32_t y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = ((uint32_t)x[e] + 0x00808080u) ^ 0x00808080u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {                    // numbers 0 2 4 6, then 1 3 5 7
        const uint32_t a = __builtin_amdgcn_perm(y[2 + h], y[h], 0x05010400u), b = __builtin_amdgcn_perm(y[6 + h], y[4 + h], 0x05010400u);
        const uint32_t c = __builtin_amdgcn_perm(y[2 + h], y[h], 0x07030602u), d = __builtin_amdgcn_perm(y[6 + h], y[4 + h], 0x07030602u);
        to[0][h] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        to[1][h] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        to[2][h] = __builtin_amdgcn_perm(d, c, 0x05040100u);
        to[3][h] = __builtin_amdgcn_perm(d, c, 0x07060302u);
    }
}

// DIGITS 1: int8 rows, 4: float32 rows; CT tiles of 16 columns (a row and digit each), of which RPT octets a thread lays out.
// Columns without a row repeat the last one: a column's sums are its own.  LOOP: there is more than one window.
// One row, 8192 x 8192, groups of 128: 9.5 us, 3.6 TB/s, a chain of loads, digits, sums and their join; what a wave does between loads is
// longer than the loads.  SIDE: where rows are so few that all groups of a chunk find columns side by side, each column meets zeros outside of its group, and
// a chunk's sums are scaled once and not once for each group (one row, 8192 x 16384, groups of 32: 20.0 us, one by one 28.7; 8-bit: 17.0 and 26.1).
template <int G, int DIGITS, int CT, int NT, int PF, int RPT, bool LOOP, bool SIDE>
__global__ void __launch_bounds__(WAVES * 64, 2) dense4_few_kernel(Dense a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int unusual[16];
    constexpr int GROUPS = 128 / G, SCALES = SIDE ? 1 : GROUPS;      // of a chunk, and those whose scales a lane needs
    constexpr bool F32 = DIGITS == 4;
    static_assert(!SIDE || (CT == 1 && GROUPS > 1), "groups side by side share one tile of columns");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, col = lane & 15;
    const int M = a.M, R = M * DIGITS, own = SIDE ? min(col / R, GROUPS - 1) : 0;      // the group of this lane's column
    const int tiles = a.cols / 16, t0 = blockIdx.x * NT;
    if (F32 && threadIdx.x < 16) unusual[threadIdx.x] = 0;
    if (F32) __syncthreads();
    // A row's part of a window, 16 PF octets, is laid out by `share` lanes (float32: one row of a lane's own, so that the
    // lanes of a row find its largest value together; int8: octets as they come).
    const int width = !F32 || M <= 1 ? 1 : M <= 2 ? 2 : M <= 4 ? 4 : M <= 8 ? 8 : 16, share = 64 / width, m = lane / share;
    char *const mine = lds + wave * (PF * 128 * R);
    const int first = wave, chunks = a.chunks;       // this wave's chunks: wave, wave + WAVES, ...
    float xf[F32 ? RPT : 1][8];
    i2 xi[F32 ? 1 : RPT];
    u4 w[NT][PF];
    h4 s[NT][PF][SCALES];
    // the octet of this thread's i-th in a window: row, chunk of the window, octet of the chunk
    auto place = [&](int i, int &r, int &k, int &o) {
        if (F32) {
            const int p = lane % share + i * share;
            r = m, k = p >> 4, o = p & 15;
            return r < M && p < 16 * PF;
        }
        const int p = lane + i * 64;
        r = p / (16 * PF), k = (p >> 4) % PF, o = p & 15;
        return r < M;
    };
    auto load = [&](int c0) {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            int r, k, o;
            const bool live = place(i, r, k, o);
            const int c = c0 + k * WAVES;
            if (F32) {
                if (live && c < chunks) load8(static_cast<const float *>(a.x) + (uint64_t)r * a.K, c * 128 + o * 8, a.K, xf[i]);
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e) xf[i][e] = 0.f;
            } else {
                xi[i] = i2{0, 0};
                if (live && c < chunks) xi[i] = load8(static_cast<const int8_t *>(a.x) + (uint64_t)r * a.K, c * 128 + o * 8, a.K);
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int tile = min(t0 + t, tiles - 1);
            const u4 *const codes = reinterpret_cast<const u4 *>(a.codes) + (uint64_t)tile * chunks * 64 + lane;
#pragma unroll
            for (int i = 0; i < PF; ++i) {
                const int c = min(c0 + i * WAVES, chunks - 1);       // a repeated chunk meets rows of zeros
                w[t][i] = codes[(uint64_t)c * 64];
#pragma unroll
                for (int g = 0; g < SCALES; ++g) s[t][i][g] = *reinterpret_cast<const h4 *>(a.scales + (uint64_t)(c * GROUPS + own + g) * a.cols + tile * 16 + 4 * q);
            }
        }
    };
    f4 acc[NT][CT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < CT; ++u) acc[t][u] = f4{0.f, 0.f, 0.f, 0.f};
    if (first < chunks) load(first);
    for (int c0 = first; c0 < chunks; c0 += LOOP ? WAVES * PF : chunks) {
        int exponent = 0;
        if (F32) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < RPT; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(xf[i][e]) & 0x7fffffffu);
            if (top >= 0x7f800000u) {                // infinities and NaN are left to the end
                top = 0;
#pragma unroll
                for (int i = 0; i < RPT; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (!(fabsf(xf[i][e]) < INFINITY)) xf[i][e] = 0.f;
                        top = max(top, __float_as_uint(xf[i][e]) & 0x7fffffffu);
                    }
                unusual[m] = 1;
            }
            for (int o = share / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
            exponent = (int)(top >> 23) - 156;       // values are below 2^(exponent + 30)
        }
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            int r, k, o;
            if (place(i, r, k, o)) {
                // 16 bytes of a lane's operand hold octets o and o + 4 of eight
                u2 *const to = reinterpret_cast<u2 *>(mine) + (((k * 2 + (o >> 3)) * 4 + (o & 3)) * R + r * DIGITS) * 2 + (o >> 2 & 1);
                if (F32) {
                    int n[8];
                    u2 d[4];
#pragma unroll
                    for (int e = 0; e < 8; ++e) n[e] = __float2int_rn(ldexpf(xf[i][e], -exponent));
                    digits8(n, d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) to[2 * e] = d[e];
                } else
                    to[0] = order_i8(xi[i]);
            }
        }
        u4 wc[NT][PF];
        h4 sc[NT][PF][SCALES];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < PF; ++i) {
                wc[t][i] = w[t][i];
#pragma unroll
                for (int g = 0; g < SCALES; ++g) sc[t][i][g] = s[t][i][g];
            }
        if (LOOP && c0 + WAVES * PF < chunks) load(c0 + WAVES * PF);
        asm volatile("" ::: "memory");               // a wave's LDS operations stay in order
        f4 sum[NT][CT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < CT; ++u) sum[t][u] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < PF; ++i) {
#pragma unroll
            for (int u = 0; u < CT; ++u) {
                const int row = min(u * 16 + col - own * R, R - 1);
                i4 x[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    x[j] = reinterpret_cast<const i4 *>(mine)[((i * 2 + j) * 4 + q) * R + row];
                    if (SIDE) {                      // inputs 64 j and on, of which the second half may be of another group
                        const int lo = own == 2 * j * 32 / G ? -1 : 0, hi = own == (2 * j + 1) * 32 / G ? -1 : 0;
                        x[j].x &= lo, x[j].y &= lo, x[j].z &= hi, x[j].w &= hi;
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    i4 d = {0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const u2 lo = weights_i8(wc[t][i][2 * j]), hi = weights_i8(wc[t][i][2 * j + 1]);
                        if (G == 32 && !SIDE) {
                            const i4 zero = {0, 0, 0, 0};
                            const i4 e = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, lo), __builtin_bit_cast(long, i2{x[j].x, x[j].y}), zero, 0, 0, 0);
                            const i4 f = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, hi), __builtin_bit_cast(long, i2{x[j].z, x[j].w}), zero, 0, 0, 0);
#pragma unroll
                            for (int v = 0; v < 4; ++v) {
                                sum[t][u][v] += (float)sc[t][i][2 * j % SCALES][v] * (float)e[v];
                                sum[t][u][v] += (float)sc[t][i][(2 * j + 1) % SCALES][v] * (float)f[v];
                            }
                        } else {
                            d = __builtin_amdgcn_mfma_i32_16x16x64_i8(i4{(int)lo.x, (int)lo.y, (int)hi.x, (int)hi.y}, x[j], d, 0, 0, 0);
                            if ((G == 64 && !SIDE) || j == 1) {
#pragma unroll
                                for (int v = 0; v < 4; ++v) sum[t][u][v] += (float)sc[t][i][j % SCALES][v] * (float)d[v];
                                d = i4{0, 0, 0, 0};
                            }
                        }
                    }
                }
            }
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int u = 0; u < CT; ++u) {
            // a column's digit, the sixteen in its weights, and its row's power of two in this wave and window
            const int row = min(u * 16 + col - own * R, R - 1);
            const int e = F32 ? __shfl(exponent, row / 4 * share) + 8 * (row & 3) - 4 : -4;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[t][u][v] += ldexpf(sum[t][u][v], e);
        }
    }
    __syncthreads();
    float *const part = reinterpret_cast<float *>(lds);      // [wave][tile of outputs][column][output]
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < CT; ++u) *reinterpret_cast<f4 *>(part + (((wave * NT + t) * CT + u) * 16 + col) * 16 + 4 * q) = acc[t][u];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * NT * M; i += WAVES * 64) {
        const int r = i / (16 * NT), t = i / 16 % NT, n = (t0 + t) * 16 + (i & 15);
        if (n >= a.N) continue;
        float y = 0.f;
        for (int k = 0; k < WAVES; ++k)
#pragma unroll
            for (int e = DIGITS - 1; e >= 0; --e)
                for (int g = 0; g < (SIDE ? GROUPS : 1); ++g) y += part[((k * NT + t) * CT * 16 + g * R + r * DIGITS + e) * 16 + (i & 15)];
        if (!F32) y *= a.x_scale[r];
        if (F32 && unusual[r]) {                     // what is not finite decides; one thread goes through the row
            const float *const x = static_cast<const float *>(a.x) + (uint64_t)r * a.K;
            for (int k = 0; k < a.K; ++k)
                if (!(fabsf(x[k]) < INFINITY)) {
                    const int in = k & 127;
                    const uint8_t b = a.codes[(((uint64_t)(n >> 4) * chunks + (k >> 7)) * 64 + 16 * (in % 32 / 8) + (n & 15)) * 16 + 4 * (in / 32) + in % 8 / 2];
                    y += x[k] * ((float)((int)((k & 1 ? b >> 4 : b & 15) ^ 8) - 8) * (float)a.scales[(uint64_t)(k / G) * a.cols + n]);
                }
        }
        a.y[(uint64_t)r * a.N + n] = a.bias ? y + a.bias[n] : y;
    }
}

// ---- many rows ---------------------------------------------------------------------------------------------------
// The rows are laid out first as the matrix instructions read them, for each 64 rows and chunk of 128 inputs in one piece:
// float32 [step of 32 inputs][tile of 16 rows][part][lane], a lane's octet of one row as float16; int8 [64 inputs][tile][lane][octets o and o + 4].
// One workgroup a row (200 x 4096: 7.3 us, 3.8 without its stores).  Rows behind the last one are not written: a column's sums are its own.
constexpr int BLOCK_ROWS = 64;
constexpr uint32_t piece_bytes(bool int8) { return int8 ? 64 * 128 : 64 * 128 * 4; }
constexpr int many_stages(bool int8) { return int8 ? 4 : 2; }
constexpr uint32_t many_stage_bytes(bool int8) { return 2 * piece_bytes(int8) + (int8 ? 2 * (8 + 1) * 1024 : 0); }       // rows of two chunks; their codes and scales
constexpr uint32_t many_lds_bytes(bool int8) { return many_stages(int8) * many_stage_bytes(int8); }

template <bool INT8>
__global__ void __launch_bounds__(256) dense4_rows_kernel(Dense a, char *operand, float *back) {
    __shared__ uint32_t most[4];
    const int m = blockIdx.x, octets = a.chunks * 16, in = m & 63;
    char *const block = operand + (uint64_t)(m >> 6) * a.chunks * piece_bytes(INT8);
    if (INT8) {
        const int8_t *const x = static_cast<const int8_t *>(a.x) + (uint64_t)m * a.K;
        for (int o = threadIdx.x; o < octets; o += 256) {
            const int k = o & 15;
            u2 *const to = reinterpret_cast<u2 *>(block + (uint64_t)(o >> 4) * piece_bytes(true)) + (((k >> 3) * 4 + (in >> 4)) * 64 + (k & 3) * 16 + (in & 15)) * 2 + (k >> 2 & 1);
            *to = order_i8(load8(x, o * 8, a.K));
        }
        return;
    }
    const float *const x = static_cast<const float *>(a.x) + (uint64_t)m * a.K;
    uint32_t top = 0;
    for (int o = threadIdx.x; o < octets; o += 256) {
        float v[8];
        load8(x, o * 8, a.K, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, size_bits(v[e]));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(most[0], most[1]), max(most[2], most[3]));
    if (threadIdx.x == 0) back[m] = scale_down(top);
    const float up = scale_up(top);
    for (int o = threadIdx.x; o < octets; o += 256) {
        float v[8];
        load8(x, o * 8, a.K, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= up;
        h8 hi, lo;
        split8(v, hi, lo);
        const int k = o & 15;
        h8 *const to = reinterpret_cast<h8 *>(block + (uint64_t)(o >> 4) * piece_bytes(false)) + ((k >> 2) * 4 + (in >> 4)) * 128 + (k & 3) * 16 + (in & 15);
        to[0] = hi;
        to[64] = lo;
    }
}

// A workgroup of eight waves has 128 outputs and 64 rows, a wave 32 of the outputs, all the rows and every other chunk of
// inputs.  The rows of two chunks are loaded straight into a stage in LDS while those of another stage are multiplied, and a step's operands
// are read from there while the step before it is multiplied: one workgroup a compute unit has nobody else to hide a wait behind.
// Each weight is turned into float16 by one wave only, for 64 rows: where two waves do it for 32 rows each, that takes
// the vector unit as long as the multiplications take the matrix unit.  float32 rows fill the LDS with two stages, and a wave loads its codes
// and scales into registers; 8-bit rows, which are multiplied faster than a load comes back, leave room for four stages with
// codes and scales.  200 rows, 4096 x 8192, groups of 128: 36.8 us, 730 TFLOP/s of two-part multiplications; 8-bit rows 20 us.  A
// pair of chunks takes 1.85 us, of which the matrix unit is busy for 0.96; without its loads 1.6, without its barrier 1.6, without
// reading the rows 1.7: nothing alone bounds it.
template <int G, bool INT8>
__global__ void __launch_bounds__(512, 2) dense4_many_kernel(Dense a, const char *operand, const float *back, float *part, int each) {
    constexpr uint32_t ROWS = piece_bytes(INT8), STAGE = many_stage_bytes(INT8);
    constexpr int STAGES = many_stages(INT8), LOADS = 2 * ROWS / 8192 + (INT8 ? 4 : 0);      // of a wave for a stage, straight into LDS
    constexpr int GROUPS = 128 / G, NT = 2, MT = 4;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, col = lane & 15;
    const int tiles = a.cols / 16, t0 = blockIdx.x * 8, n_wave = (wave & 3) * NT, half = wave >> 2;
    const int p0 = blockIdx.z * each, pairs = min((a.chunks + 1) / 2, p0 + each);      // this workgroup's pairs of chunks
    const char *const block = operand + (uint64_t)blockIdx.y * a.chunks * ROWS;
    const uint8_t *const own_codes = a.codes + (uint64_t)min(t0 + wave, tiles - 1) * a.chunks * 1024;
    const uint32_t lds0 = (uint32_t)(uintptr_t)&lds[0];
    // scales: 16 lanes for the 256 bytes of a group's 128 outputs; what lies behind the row of scales reads as zero
    const uint32_t row_bytes = (uint32_t)min(256, (a.cols - t0 * 16) * 2), in_row = (uint32_t)col * 16;
    auto issue = [&](int p, int at_stage) {          // what lies behind the last chunk reads as zero
        const uint32_t to = lds0 + (uint32_t)at_stage * STAGE;
        const int left = min(2, a.chunks - 2 * p);
        const xsmi::xsmi_int32x4 rows = xsmi::make_rsrc(block + (uint64_t)(2 * p) * ROWS, (uint32_t)left * ROWS);
#pragma unroll
        for (uint32_t i = 0; i < 2 * ROWS / 8192; ++i) xsmi::load_lds_b128(rows, to + (i * 8 + wave) * 1024, lane * 16, (i * 8 + wave) * 1024);
        if (INT8) {
            const xsmi::xsmi_int32x4 codes = xsmi::make_rsrc(own_codes + (uint64_t)(2 * p) * 1024, (uint32_t)left * 1024);
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                xsmi::load_lds_b128(codes, to + 2 * ROWS + (i * 8 + wave) * 1024, lane * 16, i * 1024);
                // group (lane >> 4) of the chunk; the same by every wave, so that all have as many loads under way
                const xsmi::xsmi_int32x4 scales = xsmi::make_rsrc(a.scales + (uint64_t)min(2 * p + (int)i, a.chunks - 1) * GROUPS * a.cols + t0 * 16,
                                                                  (uint32_t)(GROUPS - 1) * a.cols * 2 + row_bytes);
                xsmi::load_lds_b128(scales, to + 2 * ROWS + 16384 + i * 1024, q < GROUPS && in_row < row_bytes ? (uint32_t)q * a.cols * 2 + in_row : 0x80000000u, 0);
            }
        }
    };
    struct Weights {
        u4 w[NT];
        h4 s[NT][GROUPS];
    };
    auto load_weights = [&](int p, Weights &r) {
        const int c = min(2 * p + half, a.chunks - 1);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int tile = min(t0 + n_wave + t, tiles - 1);
            r.w[t] = reinterpret_cast<const u4 *>(a.codes)[((uint64_t)tile * a.chunks + c) * 64 + lane];
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) r.s[t][g] = *reinterpret_cast<const h4 *>(a.scales + (uint64_t)(c * GROUPS + g) * a.cols + tile * 16 + 4 * q);
        }
    };
    auto read_weights = [&](const char *stage, Weights &r) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            r.w[t] = reinterpret_cast<const u4 *>(stage + 2 * ROWS)[(half * 8 + n_wave + t) * 64 + lane];
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) r.s[t][g] = *reinterpret_cast<const h4 *>(stage + 2 * ROWS + 16384 + half * 1024 + g * 256 + (n_wave + t) * 32 + q * 8);
        }
    };
    struct Rows {
        u4 x[INT8 ? 1 : 2][MT];
    };
    auto read_rows = [&](const char *stage, int step, Rows &r) {
#pragma unroll
        for (int u = 0; u < MT; ++u)
#pragma unroll
            for (int p = 0; p < (INT8 ? 1 : 2); ++p)
                r.x[p][u] = reinterpret_cast<const u4 *>(stage + half * ROWS)[((step * 4 + u) * (INT8 ? 1 : 2) + p) * 64 + lane];
    };
    f4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[t][u] = f4{0.f, 0.f, 0.f, 0.f};
    f4 d[NT][MT];
    // One step's multiplications, with the next step's weights and rows made ready between them: a multiplication takes the matrix unit
    // four times as long as it takes to issue, and the two waves of a SIMD go through their steps together.
    auto multiply_f16 = [&](const Weights &r, const h8 *w, const Rows &x, int step, h8 *w_next, const char *stage, Rows &x_next) {
        if (step < 3) read_rows(stage, step + 1, x_next);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);               // the wave that multiplies goes before the one that makes ready: 39.8 -> 39.2 us
        if (step < 3) {
#pragma unroll
            for (int t = 0; t < NT; ++t) w_next[t] = weights_f16(r.w[t][step + 1]);
        }
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int u = 0; u < MT; ++u)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const f4 from = p == 0 && step % (G / 32) == 0 ? f4{0.f, 0.f, 0.f, 0.f} : d[t][u];
                    d[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[t], __builtin_bit_cast(h8, x.x[INT8 ? 0 : p][u]), from, 0, 0, 0);
                }
        if (step < 3) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);       // multiplication
                __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);       // vector
            }
        }
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        if ((step + 1) % (G / 32) == 0) {
#pragma unroll
            for (int u = 0; u < MT; ++u)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int v = 0; v < 4; ++v) acc[t][u][v] += (float)r.s[t][step / (G / 32)][v] * d[t][u][v];
        }
    };
    i4 n[NT][MT];
    auto multiply_i8 = [&](const Weights &r, const Rows &x, int step) {      // steps of 64 inputs
        const i4 zero = {0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const u2 lo = weights_i8(r.w[t][2 * step]), hi = weights_i8(r.w[t][2 * step + 1]);
#pragma unroll
            for (int u = 0; u < MT; ++u) {
                const u4 b = x.x[0][u];
                if (G == 32) {
                    const i4 e = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, lo), __builtin_bit_cast(long, u2{b.x, b.y}), zero, 0, 0, 0);
                    const i4 f = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, hi), __builtin_bit_cast(long, u2{b.z, b.w}), zero, 0, 0, 0);
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        acc[t][u][v] += (float)r.s[t][2 * step % GROUPS][v] * (float)e[v];
                        acc[t][u][v] += (float)r.s[t][(2 * step + 1) % GROUPS][v] * (float)f[v];
                    }
                } else {
                    n[t][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(i4{(int)lo.x, (int)lo.y, (int)hi.x, (int)hi.y}, __builtin_bit_cast(i4, b),
                                                                    G == 64 || step == 0 ? zero : n[t][u], 0, 0, 0);
                    if (G == 64 || step == 1) {
#pragma unroll
                        for (int v = 0; v < 4; ++v) acc[t][u][v] += (float)r.s[t][step % GROUPS][v] * (float)n[t][u][v];
                    }
                }
            }
        }
    };
    Weights w, next;
#pragma unroll
    for (int p = 0; p < STAGES - 1; ++p)
        if (p0 + p < pairs) issue(p0 + p, p);
    if (!INT8) load_weights(p0, w);
    int stage = 0;
    for (int p = p0; p < pairs; ++p) {
        // This wave's loads of the stage have arrived (no more than the later stages' are under way) and, behind the barrier,
        // everybody's have; and everybody has read the stage before it, which is loaded anew.
        if (INT8 && p + STAGES - 1 <= pairs) xsmi::wait_vmcnt<LOADS *(STAGES - 2)>(); else xsmi::wait_vmcnt<0>();
        xsmi::block_barrier();
        const char *const from = lds + (uint32_t)stage * STAGE;
        const bool live = 2 * p + half < a.chunks;
        auto ahead = [&] {
            if (p + STAGES - 1 < pairs) issue(p + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
        };
        Rows x, y;
        if (INT8) {
            ahead();
            read_weights(from, w);
            if (live) {
                read_rows(from, 0, x);
                read_rows(from, 1, y);
                multiply_i8(w, x, 0);
                multiply_i8(w, y, 1);
            }
        } else {
            h8 v0[NT], v1[NT];
            if (live) {
                read_rows(from, 0, x);
#pragma unroll
                for (int t = 0; t < NT; ++t) v0[t] = weights_f16(w.w[t][0]);
                multiply_f16(w, v0, x, 0, v1, from, y);
            }
            ahead();                                 // behind the first multiplications: issuing the loads takes as long as a step
            load_weights(p + 1, next);
            if (live) {
                multiply_f16(w, v1, y, 1, v0, from, x);
                multiply_f16(w, v0, x, 2, v1, from, y);
                multiply_f16(w, v1, y, 3, v0, from, x);
            }
        }
        if (!INT8) w = next;
        xsmi::wait_lgkmcnt0();                       // read, before the barrier that lets the stage go
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    // the halves' sums: those of the second through LDS to the waves of the first
    __syncthreads();
    f4 *const other = reinterpret_cast<f4 *>(lds) + ((wave & 3) * NT * MT) * 64 + lane;
    if (half) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < MT; ++u) other[(t * MT + u) * 64] = acc[t][u];
    }
    __syncthreads();
    if (half) return;
#pragma unroll
    for (int u = 0; u < MT; ++u) {
        const int m = blockIdx.y * BLOCK_ROWS + u * 16 + col;
        if (m >= a.M) continue;
        if (part) {                                  // one of several workgroups for these results: the sums as they are
#pragma unroll
            for (int t = 0; t < NT; ++t)
                if ((t0 + n_wave + t) * 16 < a.cols)
                    *reinterpret_cast<f4 *>(part + ((uint64_t)blockIdx.z * a.M + m) * a.cols + (t0 + n_wave + t) * 16 + 4 * q) = acc[t][u] + other[(t * MT + u) * 64];
            continue;
        }
        const float f = INT8 ? a.x_scale[m] * 0.0625f : back[m];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int n = (t0 + n_wave + t) * 16 + 4 * q;
            f4 y = (acc[t][u] + other[(t * MT + u) * 64]) * f;
            float *const to = a.y + (uint64_t)m * a.N + n;
            if (n + 4 <= a.N) {
                if (a.bias) y += *reinterpret_cast<const f4u *>(a.bias + n);
                *reinterpret_cast<f4u *>(to) = y;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < a.N) to[e] = a.bias ? y[e] + a.bias[n + e] : y[e];
            }
        }
    }
}

// The sums of a result's workgroups, in order of their inputs (64 x 4096 of 8: 4.7 us, most of it the launch).
template <bool INT8>
__global__ void __launch_bounds__(256) dense4_join_kernel(Dense a, const float *__restrict__ part, const float *__restrict__ back, int splits) {
    const int m = blockIdx.y, n = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (n >= a.N) return;
    f4 y = {0.f, 0.f, 0.f, 0.f};
    for (int z = 0; z < splits; ++z) y += *reinterpret_cast<const f4 *>(part + ((uint64_t)z * a.M + m) * a.cols + n);
    y *= INT8 ? a.x_scale[m] * 0.0625f : back[m];
    float *const to = a.y + (uint64_t)m * a.N + n;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < a.N) to[e] = a.bias ? y[e] + a.bias[n + e] : y[e];
}

// ---- the weights -------------------------------------------------------------------------------------------------
// One workgroup for a tile's 1 KB of a chunk, one thread for eight inputs of an output: a group's value of largest magnitude becomes -8,
// whatever its sign, and the others go to the nearest number.  8192 x 8192: 95 us, 3.2 TB/s (976 where every thread went through its
// group by itself).
__device__ __forceinline__ float farther(float a, float b) {         // the first of equals; a NaN stays
    return a != a || fabsf(b) <= fabsf(a) ? a : b;
}
__global__ void __launch_bounds__(256) quantize4_kernel(const float *__restrict__ w, uint8_t *codes, _Float16 *scales, int K, int N, int group, int chunks, int cols) {
    __shared__ float far[16][17];                    // [octet of inputs][output]
    const int c = (int)(blockIdx.x % (uint32_t)chunks), t = (int)(blockIdx.x / (uint32_t)chunks);
    const int in = threadIdx.x & 15, o = threadIdx.x >> 4, n = t * 16 + in, k0 = c * 128 + o * 8;
    float v[8], most = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = n < N && k0 + e < K ? w[(uint64_t)(k0 + e) * N + n] : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = farther(most, v[e]);
    far[o][in] = most;
    __syncthreads();
    const int octets = group / 8, first = o / octets * octets;
    float extreme = 0.f;
    for (int i = first; i < first + octets; ++i) extreme = farther(extreme, far[i][in]);
    const _Float16 s = (_Float16)(extreme / -8.f);
    const float sf = (float)s;
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float r = sf == 0.f || v[e] == 0.f ? 0.f : fminf(fmaxf(rintf(v[e] / sf), -8.f), 7.f);
        word |= ((uint32_t)(int)r & 15u) << (4 * e);
    }
    // octet o is step o / 4 of lanes 16 (o % 4) and on
    reinterpret_cast<uint32_t *>(codes)[((uint64_t)blockIdx.x * 64 + 16 * (o & 3) + in) * 4 + (o >> 2)] = word;
    if (o == first) scales[(uint64_t)((k0 - c * 128) / group + c * (128 / group)) * cols + n] = s;
}

// One workgroup for four tiles of a chunk, a wave for each, a lane for the 32 inputs of an output that lie together.
// 8192 x 8192: 70 us, 4.3 TB/s (a thread for each weight: 158).
__global__ void __launch_bounds__(256) dequantize4_kernel(const uint8_t *__restrict__ codes, const _Float16 *__restrict__ scales, float *w, int K, int N, int group,
                                                          int chunks, int cols) {
    const int c = (int)(blockIdx.x % (uint32_t)chunks), t = (int)(blockIdx.x / (uint32_t)chunks) * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, n = t * 16 + (lane & 15);
    if (n >= N) return;
    const u4 x = reinterpret_cast<const u4 *>(codes)[((uint64_t)t * chunks + c) * 64 + lane];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k0 = c * 128 + 32 * j + 8 * (lane >> 4);
        const float s = (float)scales[(uint64_t)(c * (128 / group) + 32 * j / group) * cols + n];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k0 + e < K) w[(uint64_t)(k0 + e) * N + n] = (float)((int)((x[j] >> (4 * e) & 15u) ^ 8u) - 8) * s;
    }
}

inline int up(int v, int to) { return (v + to - 1) / to * to; }

// 2^24 inputs or outputs: launches and offsets inside a chunk count in 32 bits.
inline bool sizes_ok(int K, int N) { return K >= 1 && N >= 1 && K <= (1 << 24) && N <= (1 << 24); }

int check_weights(const char *who, int K, int N, int group) {
    XSMI_CHECK_ARG(sizes_ok(K, N), "%s: %d inputs, %d outputs", who, K, N);
    XSMI_CHECK_ARG(group == 32 || group == 64 || group == 128, "%s: groups of %d inputs, expected 32, 64 or 128", who, group);
    return XSMI_OK;
}

// Many rows: where the results make fewer workgroups than there are compute units, the inputs are split among several, of two pairs of
// chunks at least, and their sums joined by a launch of its own (64 rows, 4096 x 4096: 34 us on 32 workgroups, 20 on 256).
struct Split {
    int splits, pairs;                               // pairs of chunks of each
};
inline Split split_of(int M, int K, int N) {
    const int64_t groups = (int64_t)((up(N, 16) + 127) / 128) * ((M + 63) / 64);
    const int pairs = (up(K, 128) / 128 + 1) / 2;
    int splits = groups >= 256 ? 1 : (int)(256 / groups);
    if (splits > pairs / 2) splits = pairs / 2;
    if (splits > 16) splits = 16;
    if (splits < 1) splits = 1;
    const int each = (pairs + splits - 1) / splits;
    return Split{(pairs + each - 1) / each, each};
}

// More tiles of outputs than compute units: two a workgroup, for which the rows are laid out once (2 rows, 5000 x 4096: 7.6 us by one
// tile, 7.9 by two; 5000 x 5000: 12.8 and 8.0; 43 rows of 8 bits, groups of 32, 4096 x 4096: 9.7 and 12.7; 5000 x 7001: 26.1 and 18.3).
constexpr int WIDE = 4096;

// Few rows: those whose digits fit two tiles of columns, and up to four tiles where a wave goes through less than eight windows: each
// takes some 3 us then, and the many rows' kernels 12 us and more in all (16 rows, 8192 x 2048: 25.6 us as few, 19.9 as
// many; 12 rows, 4096 x 4096: 12.7 and 16; 43 rows of 8 bits, 5000 x 7001: 18.3 and 20.4).  Three tiles of 8-bit rows with one tile of
// outputs a workgroup take less for a window (43, 8192 x 4096: 14.2 as few, 18.0 as many; 16384 x 4096: 25.4 and 22.4).
inline bool few(size_t M, int K, int N, bool int8) {
    if (M <= (int8 ? 32u : 8u)) return true;
    const int windows = (up(K, 128) / 128 + WAVES - 1) / WAVES, rounds = (up(N, 32) / 32 + 255) / 256;
    return M <= (int8 ? 64u : 16u) && (int64_t)windows * rounds < (int8 && M <= 48 && N <= WIDE ? 12 : 8);
}

// ROWS: the most that there may be.
template <int G, int DIGITS, int ROWS, int NT, int PF, bool LOOP, bool SIDE = false>
int launch_few(const Dense &a) {
    constexpr int CT = (ROWS * DIGITS + 15) / 16, LAID = DIGITS == 4 && ROWS == 12 ? 16 : ROWS, RPT = PF * LAID < 4 ? 1 : PF * LAID / 4;
    const size_t rows = (size_t)WAVES * PF * 128 * a.M * DIGITS, sums = (size_t)WAVES * NT * CT * 1024, bytes = rows > sums ? rows : sums;
    hipLaunchKernelGGL((dense4_few_kernel<G, DIGITS, CT, NT, PF, RPT, LOOP, SIDE>), dim3((a.cols / 16 + NT - 1) / NT), dim3(WAVES * 64), bytes, xsmi::stream(), a);
    XSMI_LAUNCH_CHECK("dense4_few_kernel");
    return XSMI_OK;
}

// Rows of one tile of columns.
template <int G, int DIGITS, int ROWS, bool SIDE>
int launch_tile(const Dense &a, int each) {
    if (each <= 1) return launch_few<G, DIGITS, ROWS, 1, 1, false, SIDE>(a);
    if (each <= 2) return launch_few<G, DIGITS, ROWS, 1, 2, false, SIDE>(a);
    // (one window of two tiles is worth its registers where the scales of 32 inputs do not take twice as many more: 2 rows, 4096 x 16384,
    // groups of 64: 12.0 us by one tile, 9.4 by two; 3000 x 12000, groups of 32: 10.8 and 13.3)
    if (each <= 4 && a.cols > WIDE && (SIDE || G != 32)) return launch_few<G, DIGITS, ROWS, 2, 4, false, SIDE>(a);
    if (each <= 4) return launch_few<G, DIGITS, ROWS, 1, 4, false, SIDE>(a);
    // (one row of long inputs: the vector unit bounds groups of 32, and two tiles save it the rows' layout; 16384 x 8192: 23.0 us by one tile,
    // 19.1 by two; groups of 128: 16.6 and 17.9)
    if (ROWS == 1 && G == 32 && each >= 8 && a.cols > WIDE) return launch_few<G, DIGITS, 1, 2, 2, true, SIDE>(a);
    if (ROWS == 1) return each <= 8 ? launch_few<G, DIGITS, 1, 1, 8, false, SIDE>(a) : launch_few<G, DIGITS, 1, 1, 4, true, SIDE>(a);
    if (a.cols > WIDE) return launch_few<G, DIGITS, ROWS, 2, 2, true, SIDE>(a);
    return launch_few<G, DIGITS, ROWS, 1, 4, true, SIDE>(a);
}

// Rows of several tiles of columns.
template <int G, int DIGITS, int ROWS, int PF>
int launch_wide(const Dense &a) {
    return a.cols > WIDE ? launch_few<G, DIGITS, ROWS, 2, PF, true>(a) : launch_few<G, DIGITS, ROWS, 1, PF, true>(a);
}

// One window where a wave's chunks fit one, and 64 KB of LDS.
template <int G, int DIGITS>
int launch_few(const Dense &a) {
    constexpr int FULL = 16 / DIGITS;                // rows of a tile of columns
    constexpr int APART = FULL * G / 128;            // and those whose groups find columns side by side
    const int R = a.M * DIGITS, each = (a.chunks + WAVES - 1) / WAVES;
    if (a.M == 1) return launch_tile<G, DIGITS, 1, G != 128>(a, each);
    if constexpr (G != 128 && APART > 1) {
        if (a.M <= APART) return launch_tile<G, DIGITS, APART, true>(a, each);
    }
    if (R <= 16) return launch_tile<G, DIGITS, FULL, false>(a, each);
    if (R <= 32) return launch_wide<G, DIGITS, 2 * FULL, 2>(a);
    // (three tiles of float32 rows are up to twelve, which lay out as sixteen)
    if (R <= 48) return launch_wide<G, DIGITS, 3 * FULL, 1>(a);
    return launch_wide<G, DIGITS, 4 * FULL, 1>(a);
}

template <int G, bool INT8>
int launch(const Dense &a, void *ws) {
    if (few(a.M, a.K, a.N, INT8)) return launch_few<G, INT8 ? 1 : 4>(a);
    const Split split = split_of(a.M, a.K, a.N);
    float *const back = (float *)ws;
    char *const operand = (char *)ws + up(a.M, BLOCK_ROWS) * 4;
    float *const part = split.splits > 1 ? (float *)(operand + (size_t)up(a.M, BLOCK_ROWS) * a.chunks * 128 * (INT8 ? 1 : 4)) : nullptr;
    hipLaunchKernelGGL(dense4_rows_kernel<INT8>, dim3(a.M), dim3(256), 0, xsmi::stream(), a, operand, back);
    XSMI_LAUNCH_CHECK("dense4_rows_kernel");
    hipLaunchKernelGGL((dense4_many_kernel<G, INT8>), dim3((a.cols + 127) / 128, (a.M + BLOCK_ROWS - 1) / BLOCK_ROWS, split.splits), dim3(512), many_lds_bytes(INT8),
                       xsmi::stream(), a, (const char *)operand, (const float *)back, part, split.pairs);
    XSMI_LAUNCH_CHECK("dense4_many_kernel");
    if (part) {
        hipLaunchKernelGGL(dense4_join_kernel<INT8>, dim3((a.cols + 1023) / 1024, a.M), dim3(256), 0, xsmi::stream(), a, (const float *)part, (const float *)back, split.splits);
        XSMI_LAUNCH_CHECK("dense4_join_kernel");
    }
    return XSMI_OK;
}

}  // namespace

extern "C" {

size_t xsmi_dense_4bit_code_bytes(int K, int N) {
    if (!sizes_ok(K, N)) return 0;
    return (size_t)up(K, 128) * up(N, 16) / 2;
}

size_t xsmi_dense_4bit_scale_count(int K, int N, int group) {
    if (!sizes_ok(K, N) || (group != 32 && group != 64 && group != 128)) return 0;
    return (size_t)(up(K, 128) / group) * up(N, 16);
}

size_t xsmi_dense_4bit_workspace_bytes(size_t M, int K, int N, int x_bits) {
    if (!sizes_ok(K, N) || (x_bits != 8 && x_bits != 32) || M >= (1u << 21) || few(M, K, N, x_bits == 8)) return 0;
    const int splits = split_of((int)M, K, N).splits;
    return (size_t)up((int)M, BLOCK_ROWS) * (4 + (size_t)up(K, 128) * (x_bits == 8 ? 1 : 4)) + (splits > 1 ? (size_t)splits * M * up(N, 16) * 4 : 0);
}

int xsmi_quantize_4bit(const float *w, int K, int N, int group, uint8_t *codes, void *scales) {
    XSMI_REQUIRE_INIT();
    if (int rc = check_weights("xsmi_quantize_4bit", K, N, group)) return rc;
    XSMI_CHECK_ARG(w && codes && scales, "xsmi_quantize_4bit: null pointer");
    XSMI_CHECK_ARG(((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 7) == 0, "xsmi_quantize_4bit: unaligned codes or scales");
    const int chunks = up(K, 128) / 128, cols = up(N, 16);
    const uint64_t groups = (uint64_t)(cols / 16) * chunks;
    XSMI_CHECK_ARG(groups < (1u << 24), "xsmi_quantize_4bit: %d x %d weights", K, N);
    hipLaunchKernelGGL(quantize4_kernel, dim3((uint32_t)groups), dim3(256), 0, xsmi::stream(), w, codes, (_Float16 *)scales, K, N, group, chunks, cols);
    XSMI_LAUNCH_CHECK("quantize4_kernel");
    return XSMI_OK;
}

int xsmi_dequantize_4bit(const uint8_t *codes, const void *scales, int K, int N, int group, float *w) {
    XSMI_REQUIRE_INIT();
    if (int rc = check_weights("xsmi_dequantize_4bit", K, N, group)) return rc;
    XSMI_CHECK_ARG(w && codes && scales, "xsmi_dequantize_4bit: null pointer");
    const int chunks = up(K, 128) / 128;
    const uint64_t groups = (uint64_t)((up(N, 16) / 16 + 3) / 4) * chunks;
    XSMI_CHECK_ARG(groups < (1u << 24), "xsmi_dequantize_4bit: %d x %d weights", K, N);
    hipLaunchKernelGGL(dequantize4_kernel, dim3((uint32_t)groups), dim3(256), 0, xsmi::stream(), codes, (const _Float16 *)scales, w, K, N, group, chunks, up(N, 16));
    XSMI_LAUNCH_CHECK("dequantize4_kernel");
    return XSMI_OK;
}

int xsmi_dense_4bit(const void *x, const float *x_scale, const uint8_t *codes, const void *scales, const float *bias, float *y, size_t M, int K, int N, int group,
                    void *ws, size_t ws_bytes) {
    XSMI_REQUIRE_INIT();
    if (int rc = check_weights("xsmi_dense_4bit", K, N, group)) return rc;
    if (M == 0) return XSMI_OK;
    XSMI_CHECK_ARG(x && codes && scales && y, "xsmi_dense_4bit: null pointer");
    XSMI_CHECK_ARG(M < (1u << 21), "xsmi_dense_4bit: %zu rows", M);      // 64 rows of a workgroup in one direction of the launch, one in another
    XSMI_CHECK_ARG(((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 7) == 0 && ((uintptr_t)ws & 15) == 0, "xsmi_dense_4bit: unaligned codes, scales or workspace");
    const bool int8 = x_scale != nullptr;
    const size_t want = xsmi_dense_4bit_workspace_bytes(M, K, N, int8 ? 8 : 32);
    XSMI_CHECK_ARG(ws_bytes >= want && (ws || !want), "xsmi_dense_4bit: workspace of %zu bytes, needs %zu", ws_bytes, want);
    const Dense a = {x, x_scale, codes, (const _Float16 *)scales, bias, y, (int)M, K, N, up(K, 128) / 128, up(N, 16)};
    if (int8) return group == 32 ? launch<32, true>(a, ws) : group == 64 ? launch<64, true>(a, ws) : launch<128, true>(a, ws);
    return group == 32 ? launch<32, false>(a, ws) : group == 64 ? launch<64, false>(a, ws) : launch<128, false>(a, ws);
}

}  // extern "C"
