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
    const uint32_t u = w ^ 0x88888888u, v = u >> 8;
    const h2 far = {(_Float16)1032.f, (_Float16)1032.f}, near = {(_Float16)72.f, (_Float16)72.f};
    const h2 a = __builtin_bit_cast(h2, (u & 0x000f000fu) | 0x64006400u) - far;
    const h2 b = __builtin_bit_cast(h2, (u & 0x00f000f0u) | 0x54005400u) - near;
    const h2 c = __builtin_bit_cast(h2, (v & 0x000f000fu) | 0x64006400u) - far;
    const h2 d = __builtin_bit_cast(h2, (v & 0x00f000f0u) | 0x54005400u) - near;
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
// A workgroup of W waves has 16 outputs and splits their inputs over its waves, chunk by chunk; the rows go through LDS, in
// windows of W PF chunks, and the waves' sums are added at the end.  A float32 row takes two of the 16 columns of a multiplication, one for
// each part (columns 0 to 7 the first parts, 8 to 15 the second), an 8-bit row one.  Columns without a row repeat the last
// one: a column's sums are its own.  A window's loads are all under way before the first of them is needed: the rows' first, for
// loads come back in order, then a wave's PF kilobytes of codes and their scales.
template <int G, bool INT8, int W, int PF>
__global__ void __launch_bounds__(W * 64) dense4_few_kernel(Dense a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ uint32_t most[W];
    constexpr int GROUPS = 128 / G;                  // of a chunk
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, col = lane & 15;
    const int n0 = blockIdx.x * 16, M = a.M;
    const u4 *const codes = reinterpret_cast<const u4 *>(a.codes) + (uint64_t)blockIdx.x * a.chunks * 64 + lane;
    const _Float16 *const scales = a.scales + n0 + 4 * q;
    const int row = INT8 ? min(col, M - 1) : min(col & 7, M - 1);
    // float32 rows: W / width waves for each of up to `width` rows; a thread has up to MINE octets of one
    constexpr int MINE = 4;
    static_assert(INT8 || W == 8, "128 PF octets a row: 4 of each thread for PF 8, 4, 2 and width 2, 4, 8");
    const int width = M <= 1 ? 1 : M <= 2 ? 2 : M <= 4 ? 4 : 8, waves = W / width, m = wave / waves, mine = (wave % waves) * 64 + lane;
    f4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int first = 0; first < a.chunks; first += W * PF) {
        const int here = min(W * PF, a.chunks - first), octets = here * 16;
        float v[MINE][8];
        if (!INT8) {
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                const int o = mine + i * waves * 64;
                if (m < M && o < octets) load8(static_cast<const float *>(a.x) + (uint64_t)m * a.K, first * 128 + o * 8, a.K, v[i]);
            }
        } else {
            u2 *const to = reinterpret_cast<u2 *>(lds);
            for (int r = 0; r < M; ++r)
                for (int o = threadIdx.x; o < octets; o += W * 64)
                    to[o * M + r] = order_i8(load8(static_cast<const int8_t *>(a.x) + (uint64_t)r * a.K, first * 128 + o * 8, a.K));
        }
        u4 w[PF];
        h4 s[PF][GROUPS];
#pragma unroll
        for (int i = 0; i < PF; ++i) {
            const int c = first + min(wave + W * i, here - 1);
            w[i] = codes[(uint64_t)c * 64];
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) s[i][g] = *reinterpret_cast<const h4 *>(scales + (uint64_t)(c * GROUPS + g) * a.cols);
        }
        float back = 1.f;
        if (!INT8) {
            h8 *const to = reinterpret_cast<h8 *>(lds);
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < MINE; ++i)
                if (m < M && mine + i * waves * 64 < octets)
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = max(top, size_bits(v[i][e]));
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
            if (lane == 0) most[wave] = top;
            __syncthreads();
            uint32_t other = 0;
            for (int k = 0; k < waves; ++k) {
                top = max(top, most[m * waves + k]);
                other = max(other, most[row * waves + k]);
            }
            back = scale_down(other);
            const float up = scale_up(top);
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                const int o = mine + i * waves * 64;
                if (m < M && o < octets) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[i][e] *= up;
                    h8 hi, lo;
                    split8(v[i], hi, lo);
                    to[(2 * o) * M + m] = hi;
                    to[(2 * o + 1) * M + m] = lo;
                }
            }
        }
        __syncthreads();
        f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < PF; ++i) {
            const int c = wave + W * i;
            if (c < here) {
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    if (INT8) {
                        i4 d = {0, 0, 0, 0};
                        const u2 *const from = reinterpret_cast<const u2 *>(lds);
                        if (G == 32) {
                            const u2 wa = weights_i8(w[i][g]), xb = from[(c * 16 + g * 4 + q) * M + row];
                            d = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, wa), __builtin_bit_cast(long, xb), d, 0, 0, 0);
                        } else {
#pragma unroll
                            for (int j = g * (G / 32); j < (g + 1) * (G / 32); j += 2) {
                                const u2 w0 = weights_i8(w[i][j]), w1 = weights_i8(w[i][j + 1]);
                                const u2 x0 = from[(c * 16 + j * 4 + q) * M + row], x1 = from[(c * 16 + j * 4 + 4 + q) * M + row];
                                d = __builtin_amdgcn_mfma_i32_16x16x64_i8(i4{(int)w0.x, (int)w0.y, (int)w1.x, (int)w1.y},
                                                                          i4{(int)x0.x, (int)x0.y, (int)x1.x, (int)x1.y}, d, 0, 0, 0);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) sum[e] += (float)s[i][g][e] * (float)d[e];
                    } else {
                        f4 d = {0.f, 0.f, 0.f, 0.f};
                        const h8 *const from = reinterpret_cast<const h8 *>(lds);
#pragma unroll
                        for (int j = g * (G / 32); j < (g + 1) * (G / 32); ++j)
                            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(weights_f16(w[i][j]), from[(2 * (c * 16 + j * 4 + q) + (col >> 3)) * M + row], d, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; ++e) sum[e] += (float)s[i][g][e] * d[e];
                    }
                }
            }
        }
        acc += sum * back;                           // a window has its own power of two
        __syncthreads();
    }
    float *const part = reinterpret_cast<float *>(lds);      // [wave][column][output]
    *reinterpret_cast<f4 *>(part + wave * 256 + col * 16 + 4 * q) = acc;
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * M; i += W * 64) {
        const int r = i >> 4, n = n0 + (i & 15);
        float y = 0.f;
        for (int k = 0; k < W; ++k) {
            y += part[k * 256 + i];
            if (!INT8) y += part[k * 256 + i + 128];
        }
        if (INT8) y *= a.x_scale[r] * 0.0625f;
        if (n < a.N) a.y[(uint64_t)r * a.N + n] = a.bias ? y + a.bias[n] : y;
    }
}

// ---- many rows ---------------------------------------------------------------------------------------------------
// The rows laid out first as the matrix instructions read them: [32 inputs][16 rows][part][lane], a lane's octet of one row.
// One workgroup a row.  Rows behind the last one are not written: a column's sums are its own.
template <bool INT8>
__global__ void __launch_bounds__(256) dense4_rows_kernel(Dense a, void *operand, float *back, int tiles) {
    __shared__ uint32_t most[4];
    const int m = blockIdx.x, octets = a.chunks * 16;
    if (INT8) {
        u2 *const to = static_cast<u2 *>(operand);
        for (int o = threadIdx.x; o < octets; o += 256)
            to[((uint64_t)(o >> 2) * tiles + (m >> 4)) * 64 + (o & 3) * 16 + (m & 15)] = order_i8(load8(static_cast<const int8_t *>(a.x) + (uint64_t)m * a.K, o * 8, a.K));
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
    h8 *const to = static_cast<h8 *>(operand);
    for (int o = threadIdx.x; o < octets; o += 256) {
        float v[8];
        load8(x, o * 8, a.K, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= up;
        h8 hi, lo;
        split8(v, hi, lo);
        const uint64_t at = (((uint64_t)(o >> 2) * tiles + (m >> 4)) * 2) * 64 + (o & 3) * 16 + (m & 15);
        to[at] = hi;
        to[at + 64] = lo;
    }
}

// A wave has 16 outputs and MT tiles of 16 rows, a workgroup four waves of the same rows.
template <int G, bool INT8, int MT>
__global__ void __launch_bounds__(256) dense4_many_kernel(Dense a, const void *operand, const float *back, int tiles) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, col = lane & 15;
    const int tile = blockIdx.x * 4 + wave, n0 = tile * 16, t0 = blockIdx.y * MT;
    if (n0 >= a.cols) return;
    const u4 *const codes = reinterpret_cast<const u4 *>(a.codes) + (uint64_t)tile * a.chunks * 64 + lane;
    const _Float16 *const scales = a.scales + n0 + 4 * q;
    f4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f4{0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < a.chunks; ++c) {
        const u4 w = codes[(uint64_t)c * 64];
#pragma unroll
        for (int g = 0; g < 128 / G; ++g) {
            const h4 s = *reinterpret_cast<const h4 *>(scales + (uint64_t)(c * (128 / G) + g) * a.cols);
            if (INT8) {
                const u2 *const from = static_cast<const u2 *>(operand) + lane;
                i4 d[MT];
#pragma unroll
                for (int t = 0; t < MT; ++t) d[t] = i4{0, 0, 0, 0};
#pragma unroll
                for (int j = g * (G / 32); j < (g + 1) * (G / 32); ++j) {
                    const long wa = __builtin_bit_cast(long, weights_i8(w[j]));
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        const u2 x = from[((uint64_t)(c * 4 + j) * tiles + min(t0 + t, tiles - 1)) * 64];
                        d[t] = __builtin_amdgcn_mfma_i32_16x16x32_i8(wa, __builtin_bit_cast(long, x), d[t], 0, 0, 0);
                    }
                }
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[t][e] += (float)s[e] * (float)d[t][e];
            } else {
                const h8 *const from = static_cast<const h8 *>(operand) + lane;
                f4 d[MT];
#pragma unroll
                for (int t = 0; t < MT; ++t) d[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = g * (G / 32); j < (g + 1) * (G / 32); ++j) {
                    const h8 wa = weights_f16(w[j]);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        const h8 *const x = from + ((uint64_t)(c * 4 + j) * tiles + min(t0 + t, tiles - 1)) * 128;
                        d[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wa, x[0], d[t], 0, 0, 0);
                        d[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wa, x[64], d[t], 0, 0, 0);
                    }
                }
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[t][e] += (float)s[e] * d[t][e];
            }
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = (t0 + t) * 16 + col;
        if (m >= a.M) continue;
        const float f = INT8 ? a.x_scale[m] * 0.0625f : back[m];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int n = n0 + 4 * q + e;
            if (n < a.N) a.y[(uint64_t)m * a.N + n] = acc[t][e] * f + (a.bias ? a.bias[n] : 0.f);
        }
    }
}

// ---- the weights -------------------------------------------------------------------------------------------------
// One thread for a lane's eight inputs of a step, one output: a group's value of largest magnitude becomes -8, whatever its
// sign, and the others go to the nearest number.  The value is looked for by every thread of its group again.
__global__ void __launch_bounds__(256) quantize4_kernel(const float *__restrict__ w, uint8_t *codes, _Float16 *scales, int K, int N, int group, int chunks, int cols) {
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x, total = (uint64_t)(cols / 16) * chunks * 256;
    if (i >= total) return;
    const int j = (int)(i & 3), lane = (int)(i >> 2) & 63;
    const uint64_t tc = i >> 8;
    const int c = (int)(tc % (uint64_t)chunks), t = (int)(tc / (uint64_t)chunks);
    const int n = t * 16 + (lane & 15), k0 = c * 128 + j * 32 + (lane >> 4) * 8, g = k0 / group;
    float extreme = 0.f;
    if (n < N)
        for (int k = g * group; k < min(K, (g + 1) * group); ++k) {
            const float v = w[(uint64_t)k * N + n];
            if (!(fabsf(v) <= fabsf(extreme))) extreme = v;          // the first of equals; a NaN stays
            if (extreme != extreme) break;
        }
    const _Float16 s = (_Float16)(extreme / -8.f);
    const float sf = (float)s;
    uint32_t word = 0;
    for (int e = 0; e < 8; ++e) {
        const int k = k0 + e;
        const float v = n < N && k < K ? w[(uint64_t)k * N + n] : 0.f;
        const float r = sf == 0.f || v == 0.f ? 0.f : fminf(fmaxf(rintf(v / sf), -8.f), 7.f);
        word |= ((uint32_t)(int)r & 15u) << (4 * e);
    }
    reinterpret_cast<uint32_t *>(codes)[(tc * 64 + lane) * 4 + j] = word;
    if (k0 % group == 0) scales[(uint64_t)g * cols + n] = s;
}

__global__ void __launch_bounds__(256) dequantize4_kernel(const uint8_t *__restrict__ codes, const _Float16 *__restrict__ scales, float *w, int K, int N, int group,
                                                          int chunks, int cols) {
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (uint64_t)K * N) return;
    const int k = (int)(i / (uint64_t)N), n = (int)(i - (uint64_t)k * N), r = k & 127;
    const uint64_t tile = (uint64_t)(n >> 4) * chunks + (k >> 7);
    const uint8_t b = codes[(tile * 64 + 16 * (r % 32 / 8) + (n & 15)) * 16 + 4 * (r / 32) + r % 8 / 2];
    const int c = (int)((k & 1 ? b >> 4 : b & 15) ^ 8) - 8;
    w[i] = (float)c * (float)scales[(uint64_t)(k / group) * cols + n];
}

constexpr int ROW_TILES = 4;                         // of 16 rows: of a workgroup of dense4_many_kernel
inline int up(int v, int to) { return (v + to - 1) / to * to; }

int check_weights(const char *who, int K, int N, int group) {
    XSMI_CHECK_ARG(K >= 1 && N >= 1 && K <= (1 << 30) && N <= (1 << 30), "%s: %d inputs, %d outputs", who, K, N);
    XSMI_CHECK_ARG(group == 32 || group == 64 || group == 128, "%s: groups of %d inputs, expected 32, 64 or 128", who, group);
    return XSMI_OK;
}

// Few rows: those that fit the columns of one multiplication.
inline bool few(size_t M, bool int8) { return M <= (int8 ? 16u : 8u); }

template <int G, bool INT8, int PF>
int launch_few(const Dense &a) {
    constexpr int W = 8;
    const int window = a.chunks < W * PF ? a.chunks : W * PF;
    const size_t rows = (size_t)window * 128 * a.M * (INT8 ? 1 : 4), sums = W * 1024, bytes = rows > sums ? rows : sums;
    hipLaunchKernelGGL((dense4_few_kernel<G, INT8, W, PF>), dim3(a.cols / 16), dim3(W * 64), bytes, xsmi::stream(), a);
    XSMI_LAUNCH_CHECK("dense4_few_kernel");
    return XSMI_OK;
}

template <int G, bool INT8>
int launch(const Dense &a, void *ws) {
    if (few(a.M, INT8)) {
        const int rows = INT8 ? (a.M + 3) / 4 : a.M;         // windows of 64 KB at most
        return rows <= 2 ? launch_few<G, INT8, 8>(a) : rows <= 4 ? launch_few<G, INT8, 4>(a) : launch_few<G, INT8, 2>(a);
    }
    const int tiles = up(a.M, 16) / 16;
    float *const back = (float *)ws;
    void *const operand = (char *)ws + up(a.M, 64) * 4;
    hipLaunchKernelGGL(dense4_rows_kernel<INT8>, dim3(a.M), dim3(256), 0, xsmi::stream(), a, operand, back, tiles);
    XSMI_LAUNCH_CHECK("dense4_rows_kernel");
    hipLaunchKernelGGL((dense4_many_kernel<G, INT8, ROW_TILES>), dim3((a.cols / 16 + 3) / 4, (tiles + ROW_TILES - 1) / ROW_TILES), dim3(256), 0, xsmi::stream(), a,
                       (const void *)operand, (const float *)back, tiles);
    XSMI_LAUNCH_CHECK("dense4_many_kernel");
    return XSMI_OK;
}

}  // namespace

extern "C" {

size_t xsmi_dense_4bit_code_bytes(int K, int N) {
    if (K < 1 || N < 1 || K > (1 << 30) || N > (1 << 30)) return 0;
    return (size_t)up(K, 128) * up(N, 16) / 2;
}

size_t xsmi_dense_4bit_scale_count(int K, int N, int group) {
    if (K < 1 || N < 1 || K > (1 << 30) || N > (1 << 30) || (group != 32 && group != 64 && group != 128)) return 0;
    return (size_t)(up(K, 128) / group) * up(N, 16);
}

size_t xsmi_dense_4bit_workspace_bytes(size_t M, int K, int N, int x_bits) {
    if (K < 1 || N < 1 || K > (1 << 30) || N > (1 << 30) || (x_bits != 8 && x_bits != 32) || M >= (1u << 21) || few(M, x_bits == 8)) return 0;
    return (size_t)up((int)M, 64) * 4 + (size_t)up((int)M, 16) * up(K, 128) * (x_bits == 8 ? 1 : 4);
}

int xsmi_quantize_4bit(const float *w, int K, int N, int group, uint8_t *codes, void *scales) {
    XSMI_REQUIRE_INIT();
    if (int rc = check_weights("xsmi_quantize_4bit", K, N, group)) return rc;
    XSMI_CHECK_ARG(w && codes && scales, "xsmi_quantize_4bit: null pointer");
    XSMI_CHECK_ARG(((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 7) == 0, "xsmi_quantize_4bit: unaligned codes or scales");
    const int chunks = up(K, 128) / 128, cols = up(N, 16);
    const uint64_t groups = (uint64_t)(cols / 16) * chunks;
    XSMI_CHECK_ARG(groups < (1ull << 31), "xsmi_quantize_4bit: %d x %d weights", K, N);
    hipLaunchKernelGGL(quantize4_kernel, dim3((uint32_t)groups), dim3(256), 0, xsmi::stream(), w, codes, (_Float16 *)scales, K, N, group, chunks, cols);
    XSMI_LAUNCH_CHECK("quantize4_kernel");
    return XSMI_OK;
}

int xsmi_dequantize_4bit(const uint8_t *codes, const void *scales, int K, int N, int group, float *w) {
    XSMI_REQUIRE_INIT();
    if (int rc = check_weights("xsmi_dequantize_4bit", K, N, group)) return rc;
    XSMI_CHECK_ARG(w && codes && scales, "xsmi_dequantize_4bit: null pointer");
    const uint64_t groups = ((uint64_t)K * N + 255) / 256;
    XSMI_CHECK_ARG(groups < (1ull << 31), "xsmi_dequantize_4bit: %d x %d weights", K, N);
    hipLaunchKernelGGL(dequantize4_kernel, dim3((uint32_t)groups), dim3(256), 0, xsmi::stream(), codes, (const _Float16 *)scales, w, K, N, group, up(K, 128) / 128, up(N, 16));
    XSMI_LAUNCH_CHECK("dequantize4_kernel");
    return XSMI_OK;
}

int xsmi_dense_4bit(const void *x, const float *x_scale, const uint8_t *codes, const void *scales, const float *bias, float *y, size_t M, int K, int N, int group,
                    void *ws, size_t ws_bytes) {
    XSMI_REQUIRE_INIT();
    if (int rc = check_weights("xsmi_dense_4bit", K, N, group)) return rc;
    if (M == 0) return XSMI_OK;
    XSMI_CHECK_ARG(x && codes && scales && y, "xsmi_dense_4bit: null pointer");
    XSMI_CHECK_ARG(M < (1u << 21), "xsmi_dense_4bit: %zu rows", M);
    XSMI_CHECK_ARG(((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 7) == 0 && ((uintptr_t)ws & 15) == 0, "xsmi_dense_4bit: unaligned codes, scales or workspace");
    const bool int8 = x_scale != nullptr;
    const size_t want = xsmi_dense_4bit_workspace_bytes(M, K, N, int8 ? 8 : 32);
    XSMI_CHECK_ARG(ws_bytes >= want && (ws || !want), "xsmi_dense_4bit: workspace of %zu bytes, needs %zu", ws_bytes, want);
    const Dense a = {x, x_scale, codes, (const _Float16 *)scales, bias, y, (int)M, K, N, up(K, 128) / 128, up(N, 16)};
    if (int8) return group == 32 ? launch<32, true>(a, ws) : group == 64 ? launch<64, true>(a, ws) : launch<128, true>(a, ws);
    return group == 32 ? launch<32, false>(a, ws) : group == 64 ? launch<64, false>(a, ws) : launch<128, false>(a, ws);
}

}  // extern "C"
