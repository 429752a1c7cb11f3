// Root-mean-square normalisation of rows, with the residual's addition in front of it, forward and backward, and with an
// output in 8 bits.
//
//   s = x + residual        r = 1 / sqrt(mean_j s_j^2 + eps)        y_j = gamma_j s_j r
//   backward, with a_j = gamma_j dy_j and xhat_j = s_j r:
//     ds_j += r (a_j - xhat_j mean_i(a_i xhat_i))                   dgamma_j = sum_rows dy_j xhat_j
//
// All of it is bound by memory: a row is read once, kept in registers while its sum is formed, and written once.
#include "xsmi_internal.h"
#include <math.h>

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef f4 f4u __attribute__((aligned(4)));              // rows of an odd length start at any element

// The sum over the T threads that share a row, in every one of them; T is a power of two, at least one wave's share of a row.
template <int T, typename V>
__device__ __forceinline__ V row_sum(V v, V *sm) {
#pragma unroll
    for (int o = (T < 64 ? T : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if (T > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
        __syncthreads();
        const int first = threadIdx.x / T * (T / 64);
        v = sm[first];
#pragma unroll
        for (int w = 1; w < T / 64; ++w) v += sm[first + w];
    }
    return v;
}

// The sum of one value and the largest of another, likewise.
template <int T>
__device__ __forceinline__ void row_sum_max(double &sum, double &most, double2 *sm) {
#pragma unroll
    for (int o = (T < 64 ? T : 64) / 2; o > 0; o >>= 1) {
        sum += __shfl_xor(sum, o);
        most = fmax(most, __shfl_xor(most, o));
    }
    if (T > 64) {
        if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = make_double2(sum, most);
        __syncthreads();
        const int first = threadIdx.x / T * (T / 64);
        sum = sm[first].x;
        most = sm[first].y;
#pragma unroll
        for (int w = 1; w < T / 64; ++w) {
            sum += sm[first + w].x;
            most = fmax(most, sm[first + w].y);
        }
    }
}

// STREAM: past the caches' replacement, for operands that are larger than they are.
template <bool STREAM = false>
__device__ __forceinline__ f4 load4(const float *p, int j, int cols) {
    if (j + 4 <= cols) return STREAM ? __builtin_nontemporal_load(reinterpret_cast<const f4u *>(p + j)) : *reinterpret_cast<const f4u *>(p + j);
    f4 r = {0.f, 0.f, 0.f, 0.f};
    if (j < cols) r.x = p[j];
    if (j + 1 < cols) r.y = p[j + 1];
    if (j + 2 < cols) r.z = p[j + 2];
    return r;
}

template <bool STREAM = false>
__device__ __forceinline__ void store4(float *p, int j, int cols, f4 v) {
    if (j + 4 <= cols) {
        if (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<f4u *>(p + j));
        else *reinterpret_cast<f4u *>(p + j) = v;
        return;
    }
    if (j < cols) p[j] = v.x;
    if (j + 1 < cols) p[j + 1] = v.y;
    if (j + 2 < cols) p[j + 2] = v.z;
}

struct Forward {
    const float *x, *residual, *gamma;
    float *sum, *y, *rstd;
    int8_t *q;
    float *scale;
    uint64_t rows;
    int cols;
    float eps;
};

// T threads a row, NT threads a workgroup, V vectors of four a thread: rows of up to 4 T V elements stay in registers.
// 16384 x 4096 with a residual: 174 us, 6.2 TB/s; 32 x 512: 2.9 us, a chain of load, sum across the workgroup and store.
template <int T, int NT, int V, bool STREAM>
__global__ void __launch_bounds__(NT) rms_fwd_kernel(Forward a) {
    __shared__ float sm[NT / 64];
    const uint64_t row = (uint64_t)blockIdx.x * (NT / T) + threadIdx.x / T;
    const int t = threadIdx.x % T, cols = a.cols;
    const bool live = row < a.rows;
    const uint64_t at = row * (uint64_t)cols;
    f4 s[V];
    float sq = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int j = 4 * (v * T + t);
        s[v] = f4{0.f, 0.f, 0.f, 0.f};
        if (live && j < cols) {
            s[v] = load4<STREAM>(a.x + at, j, cols);
            if (a.residual) s[v] += load4<STREAM>(a.residual + at, j, cols);
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 4; ++e) sq += s[v][e] * s[v][e];
    sq = row_sum<T>(sq, sm);
    const float r = 1.f / sqrtf(sq / (float)cols + a.eps);
    if (!live) return;
    if (t == 0 && a.rstd) a.rstd[row] = r;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int j = 4 * (v * T + t);
        if (j < cols) {
            if (a.sum) store4<STREAM>(a.sum + at, j, cols, s[v]);
            store4<STREAM>(a.y + at, j, cols, s[v] * r * load4(a.gamma, j, cols));
        }
    }
}

// Longer rows: a workgroup reads its row twice (512 x 65536 with a residual: 125 us, 81 for the bytes).
template <int NT>
__global__ void __launch_bounds__(NT) rms_fwd_long_kernel(Forward a) {
    __shared__ float sm[NT / 64];
    const uint64_t row = blockIdx.x, at = row * (uint64_t)a.cols;
    const int cols = a.cols;
    float sq = 0.f;
    for (int j = 4 * threadIdx.x; j < cols; j += 4 * NT) {
        f4 s = load4(a.x + at, j, cols);
        if (a.residual) {
            s += load4(a.residual + at, j, cols);
            store4(a.sum + at, j, cols, s);
        }
        sq += (s.x * s.x + s.y * s.y) + (s.z * s.z + s.w * s.w);
    }
    sq = row_sum<NT>(sq, sm);
    const float r = 1.f / sqrtf(sq / (float)cols + a.eps);
    if (threadIdx.x == 0 && a.rstd) a.rstd[row] = r;
    const float *s = a.residual ? a.sum + at : a.x + at;     // a thread reads what it has written itself
    for (int j = 4 * threadIdx.x; j < cols; j += 4 * NT) store4(a.y + at, j, cols, load4(s, j, cols) * r * load4(a.gamma, j, cols));
}

// Four numbers of 8 bits, to the nearest, ties to even.
__device__ __forceinline__ void store_q(int8_t *p, int j, int cols, const double *y, double inverse) {
    int q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = (int)rint(y[e] * inverse);
    if (j + 4 <= cols && ((uintptr_t)(p + j) & 3) == 0) {
        *reinterpret_cast<uint32_t *>(p + j) = (q[0] & 255) | (q[1] & 255) << 8 | (q[2] & 255) << 16 | (uint32_t)q[3] << 24;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (j + e < cols) p[j + e] = (int8_t)q[e];
}

// The output in 8 bits: q_j = round(127 y_j / max |y|), scale = max |y| / 127.  The root is common to a row's y, so the numbers are those of
// z_j = gamma_j s_j, and the sum and the largest value are found together.  In 64 bits, which run at the rate of 32 here and
// are not what bounds this: a number next to a border falls on the side that the exact value is on, whatever the order
// of the sums.  16384 x 4096 with a residual: 137 us, 6.4 TB/s; one row of 4096: 4.9 us.  A row of zeros has the numbers 0 and the scale 0, one with a NaN or an infinity the numbers 0 and the scale NaN.
struct Steps {
    bool bad;
    double inverse;
};
__device__ __forceinline__ Steps steps_of(const Forward &a, double sq, double most, uint64_t row, bool writes) {
    const bool bad = !(most < INFINITY);
    if (writes) a.scale[row] = bad ? NAN : most == 0.0 ? 0.f : (float)(most / sqrt(sq / (double)a.cols + (double)a.eps) / 127.0);
    return Steps{bad, bad || most == 0.0 ? 0.0 : 127.0 / most};
}

template <int T, int NT, int V, bool STREAM>
__global__ void __launch_bounds__(NT) rms_fwd_int8_kernel(Forward a) {
    __shared__ double2 sm[NT / 64];
    const uint64_t row = (uint64_t)blockIdx.x * (NT / T) + threadIdx.x / T;
    const int t = threadIdx.x % T, cols = a.cols;
    const bool live = row < a.rows;
    const uint64_t at = row * (uint64_t)cols;
    f4 s[V], g[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int j = 4 * (v * T + t);
        s[v] = g[v] = f4{0.f, 0.f, 0.f, 0.f};
        if (live && j < cols) {
            s[v] = load4<STREAM>(a.x + at, j, cols);
            g[v] = load4(a.gamma, j, cols);
            if (a.residual) s[v] += load4<STREAM>(a.residual + at, j, cols);
        }
    }
    double sq = 0.0, most = 0.0;
    bool nan = false;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int j = 4 * (v * T + t);
        if (a.sum && live && j < cols) store4<STREAM>(a.sum + at, j, cols, s[v]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double z = (double)s[v][e] * (double)g[v][e];
            sq += (double)s[v][e] * (double)s[v][e];
            nan |= z != z;
            most = fmax(most, fabs(z));
        }
    }
    most = nan ? INFINITY : most;
    row_sum_max<T>(sq, most, sm);
    if (!live) return;
    const Steps step = steps_of(a, sq, most, row, t == 0);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int j = 4 * (v * T + t);
        if (j < cols) {
            double z[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = step.bad ? 0.0 : (double)s[v][e] * (double)g[v][e];
            store_q(a.q + at, j, cols, z, step.inverse);
        }
    }
}

template <int NT>
__global__ void __launch_bounds__(NT) rms_fwd_int8_long_kernel(Forward a) {
    __shared__ double2 sm[NT / 64];
    const uint64_t row = blockIdx.x, at = row * (uint64_t)a.cols;
    const int cols = a.cols;
    double sq = 0.0, most = 0.0;
    bool nan = false;
    for (int j = 4 * threadIdx.x; j < cols; j += 4 * NT) {
        f4 s = load4(a.x + at, j, cols);
        const f4 g = load4(a.gamma, j, cols);
        if (a.residual) {
            s += load4(a.residual + at, j, cols);
            store4(a.sum + at, j, cols, s);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double z = (double)s[e] * (double)g[e];
            sq += (double)s[e] * (double)s[e];
            nan |= z != z;
            most = fmax(most, fabs(z));
        }
    }
    most = nan ? INFINITY : most;
    row_sum_max<NT>(sq, most, sm);
    const Steps step = steps_of(a, sq, most, row, threadIdx.x == 0);
    const float *from = a.residual ? a.sum + at : a.x + at;
    for (int j = 4 * threadIdx.x; j < cols; j += 4 * NT) {
        const f4 s = load4(from, j, cols), g = load4(a.gamma, j, cols);
        double z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = step.bad ? 0.0 : (double)s[e] * (double)g[e];
        store_q(a.q + at, j, cols, z, step.inverse);
    }
}

struct Backward {
    const float *dy, *s, *rstd, *gamma, *ds;
    float *dx1, *dx2, *part;
    int acc1, acc2;
    uint64_t rows;
    int cols;
    float *dgamma;                                   // written by workgroups behind the first `groups`, or NULL
    int acc_gamma, groups;
};

// dgamma of 32 columns: eight threads of four columns for each of NT / 8 stretches of rows.
template <int NT>
__device__ __forceinline__ void rms_columns(const Backward &a, int block) {
    __shared__ f4 sm[NT / 8][8];
    const int t = threadIdx.x & 7, j = block * 32 + 4 * t, w = threadIdx.x >> 3, cols = a.cols;
    f4 s = {0.f, 0.f, 0.f, 0.f};
    if (j < cols) {
#pragma unroll 2
        for (uint64_t i = w; i < a.rows; i += NT / 8) s += load4(a.dy + i * cols, j, cols) * (load4(a.s + i * cols, j, cols) * a.rstd[i]);
    }
    sm[w][t] = s;
    __syncthreads();
    for (int n = NT / 16; n >= 1; n >>= 1) {
        if (w < n) sm[w][t] += sm[w + n][t];
        __syncthreads();
    }
    if (w == 0 && j < cols) store4(a.dgamma, j, cols, a.acc_gamma ? sm[0][t] + load4(a.dgamma, j, cols) : sm[0][t]);
}

// T threads a row; a workgroup takes every (NT / T gridDim)-th lot of rows, and adds the terms of dgamma of the columns
// that a thread owns in its registers; those of a workgroup go to its row of part at the end.  All that a row needs is loaded before its sum is
// formed.  16384 x 4096 with ds and two gradients: 224 us, 6.0 TB/s, and 5 for the sums of part.  Rows that a workgroup has side by
// side share its row of part: with one for each of them 65536 x 33 took 62 us instead of 16, for the one workgroup that adds 16384.
template <int T, int NT, int V, bool STREAM>
__global__ void __launch_bounds__(NT) rms_bwd_kernel(Backward a) {
    __shared__ float sm[NT / 64];
    if (a.dgamma && (int)blockIdx.x >= a.groups) {
        rms_columns<NT>(a, (int)blockIdx.x - a.groups);
        return;
    }
    const int t = threadIdx.x % T, cols = a.cols;
    const float inv = 1.f / (float)cols;
    f4 dg[V], gm[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int j = 4 * (v * T + t);
        dg[v] = f4{0.f, 0.f, 0.f, 0.f};
        gm[v] = j < cols ? load4(a.gamma, j, cols) : dg[v];
    }
    for (uint64_t first = (uint64_t)blockIdx.x * (NT / T); first < a.rows; first += (uint64_t)a.groups * (NT / T)) {
        const uint64_t row = first + threadIdx.x / T, at = row * (uint64_t)cols;
        const bool live = row < a.rows;
        f4 s[V], d[V], g[V];
        float c = 0.f;
        const float r = live ? a.rstd[row] : 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int j = 4 * (v * T + t);
            s[v] = d[v] = g[v] = f4{0.f, 0.f, 0.f, 0.f};
            if (live && j < cols) {
                s[v] = load4<STREAM>(a.s + at, j, cols);
                d[v] = load4<STREAM>(a.dy + at, j, cols);
                if (a.ds) g[v] = load4<STREAM>(a.ds + at, j, cols);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            s[v] *= r;
            dg[v] += d[v] * s[v];
            d[v] *= gm[v];
#pragma unroll
            for (int e = 0; e < 4; ++e) c += d[v][e] * s[v][e];
        }
        c = row_sum<T>(c, sm) * inv;
        if (live && a.dx1) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int j = 4 * (v * T + t);
                if (j < cols) {
                    g[v] += (d[v] - s[v] * c) * r;
                    store4<STREAM>(a.dx1 + at, j, cols, a.acc1 ? g[v] + load4(a.dx1 + at, j, cols) : g[v]);
                    if (a.dx2) store4<STREAM>(a.dx2 + at, j, cols, a.acc2 ? g[v] + load4(a.dx2 + at, j, cols) : g[v]);
                }
            }
        }
    }
    if (a.part) {
        if (T < NT) {                                // the rows that were worked on side by side
            constexpr int W = NT / 64, L = T < 64 ? T : 64;
            __shared__ f4 beside[W][V][L];
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int o = 32; o >= T; o >>= 1)
#pragma unroll
                    for (int e = 0; e < 4; ++e) dg[v][e] += __shfl_xor(dg[v][e], o);
            if ((threadIdx.x & 63) < L)
#pragma unroll
                for (int v = 0; v < V; ++v) beside[threadIdx.x >> 6][v][t] = dg[v];
            __syncthreads();
            if (threadIdx.x >= T) return;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int w = 1; w < W; ++w) dg[v] += beside[w][v][t];
        }
        float *part = a.part + (uint64_t)blockIdx.x * cols;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int j = 4 * (v * T + t);
            if (j < cols) store4(part, j, cols, dg[v]);
        }
    }
}

// Longer rows, read twice; the terms of dgamma are added in memory, in this workgroup's own row of part (512 x 65536: 185 us, 81 for
// the bytes without part).
template <int NT>
__global__ void __launch_bounds__(NT) rms_bwd_long_kernel(Backward a) {
    __shared__ float sm[NT / 64];
    const int cols = a.cols;
    float *part = a.part ? a.part + (uint64_t)blockIdx.x * cols : nullptr;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint64_t at = row * (uint64_t)cols;
        const float r = a.rstd[row];
        float c = 0.f;
        for (int j = 4 * threadIdx.x; j < cols; j += 4 * NT) {
            const f4 s = load4(a.s + at, j, cols) * r, d = load4(a.dy + at, j, cols), x = d * s;
            if (part) store4(part, j, cols, row == blockIdx.x ? x : load4(part, j, cols) + x);
            const f4 w = x * load4(a.gamma, j, cols);
            c += (w.x + w.y) + (w.z + w.w);
        }
        c = row_sum<NT>(c, sm) / (float)cols;
        if (a.dx1)
            for (int j = 4 * threadIdx.x; j < cols; j += 4 * NT) {
                const f4 s = load4(a.s + at, j, cols) * r;
                f4 g = (load4(a.dy + at, j, cols) * load4(a.gamma, j, cols) - s * c) * r;
                if (a.ds) g += load4(a.ds + at, j, cols);
                store4(a.dx1 + at, j, cols, a.acc1 ? g + load4(a.dx1 + at, j, cols) : g);
                if (a.dx2) store4(a.dx2 + at, j, cols, a.acc2 ? g + load4(a.dx2 + at, j, cols) : g);
            }
    }
}

// dgamma[j] = (accumulate ? dgamma[j] : 0) + sum over the rows of part: 32 columns a workgroup, eight threads of four columns for each
// of 128 stretches of rows (512 rows of 4096: 5.0 us, most of it the launch and the joining).
__global__ void __launch_bounds__(1024) rms_dgamma_kernel(const float *__restrict__ part, int rows, int cols, float *dgamma, int accumulate) {
    __shared__ f4 sm[128][8];
    const int t = threadIdx.x & 7, j = blockIdx.x * 32 + 4 * t, w = threadIdx.x >> 3;
    f4 s = {0.f, 0.f, 0.f, 0.f};
    if (j < cols) {
#pragma unroll 4
        for (int i = w; i < rows; i += 128) s += load4(part + (uint64_t)i * cols, j, cols);
    }
    sm[w][t] = s;
    __syncthreads();
    for (int n = 64; n >= 8; n >>= 1) {              // the stretches by halves, the last eight one after the other
        if (w < n) sm[w][t] += sm[w + n][t];
        __syncthreads();
    }
    if (w == 0 && j < cols) {
        f4 r = sm[0][t];
#pragma unroll
        for (int i = 1; i < 8; ++i) r += sm[i][t];
        if (accumulate) r += load4(dgamma, j, cols);
        store4(dgamma, j, cols, r);
    }
}

constexpr uint64_t MAX_ROWS = 1ull << 31;

constexpr size_t LAUNCH_ROWS = 1u << 21;             // of one launch: its threads count in 32 bits
Forward lot(Forward a, size_t first) {
    const uint64_t at = first * (uint64_t)a.cols;
    a.x += at;
    a.rows = a.rows - first < LAUNCH_ROWS ? a.rows - first : LAUNCH_ROWS;
    if (a.residual) a.residual += at, a.sum += at;
    if (a.y) a.y += at;
    if (a.rstd) a.rstd += first;
    if (a.q) a.q += at, a.scale += first;
    return a;
}

// Many rows go by a wave each up to 1024 columns, without a barrier (65536 x 257, backward: 80 us, by workgroups of 256 threads 123), and
// in 8 bits by narrower workgroups above (16384 x 4096: 137 us, by 1024 threads 252; 13000 x 5000: 158 and 246); few rows go by as
// many threads as they have use for (200 x 1000, backward: 3.8 us, by waves 4.2).  The forward of more than 512 columns goes by
// waves only where the operands stay in the caches (2048 x 600: 6.9 us, by workgroups 9.1; 65536 x 600: 123 and 113).
constexpr uint64_t WAVE_ROWS = 512;
inline bool by_waves(uint64_t rows) { return rows >= WAVE_ROWS; }

// Workgroups of the backward, each with a row of part.
int backward_groups(uint64_t rows, int cols) {
    const int need = (cols + 3) / 4, side = need <= 16 ? 16 : need <= 64 || (need <= 256 && by_waves(rows)) ? 4 : 1;       // rows side by side
    const uint64_t lots = (rows + side - 1) / side;
    // as many workgroups as fill the card, and at least two lots of rows each where there are more than two a compute unit
    const uint64_t most = need > 1024 ? 256 : 1024, few = most / 2, two = (lots + 1) / 2;
    return (int)(lots <= few ? lots : two <= few ? few : two < most ? two : most);
}

// Few rows: dgamma by workgroups of its own, which read dy and s again beside the ones of the rows, in one launch and without a
// workspace (32 x 512: 3.1 us, against 3.4 and 3.0).
inline bool columns_apart(size_t rows, int cols) { return rows <= 1024 && cols <= 16384 && rows * (size_t)cols <= (1u << 18); }

int check(const char *who, size_t rows, int cols, float eps) {
    XSMI_CHECK_ARG(cols >= 1 && cols <= (1 << 30), "%s: %d columns", who, cols);
    XSMI_CHECK_ARG(rows < MAX_ROWS, "%s: %zu rows", who, rows);
    XSMI_CHECK_ARG(eps >= 0, "%s: epsilon %g", who, (double)eps);
    return XSMI_OK;
}

// Operands past the last-level cache (256 MB) are streamed: 16384 rows of 4096, backward 252 us without, 226 with; where they
// fit, the next kernel finds them there.
inline bool streams(size_t rows, int cols, int operands) { return (double)rows * cols * operands * 4 > 256e6; }

#define LAUNCH(kernel, grid, threads, args) hipLaunchKernelGGL(kernel, dim3((uint32_t)(grid)), dim3(threads), 0, xsmi::stream(), args)

#define LAUNCH_TWO(kernel, T, NT, V, grid, args)                          \
    do {                                                                 \
        if (stream) LAUNCH((kernel<T, NT, V, true>), grid, NT, args);    \
        else LAUNCH((kernel<T, NT, V, false>), grid, NT, args);          \
    } while (0)

}  // namespace

extern "C" {

int xsmi_rms_norm_fwd(const float *x, const float *residual, const float *gamma, float *sum, float *y, float *rstd, size_t rows, int cols,
                      float eps) {
    XSMI_REQUIRE_INIT();
    if (int rc = check("xsmi_rms_norm_fwd", rows, cols, eps)) return rc;
    if (rows == 0) return XSMI_OK;
    XSMI_CHECK_ARG(x && gamma && y && (residual == nullptr) == (sum == nullptr), "xsmi_rms_norm_fwd: null pointer (a residual comes with a sum)");
    const bool stream = streams(rows, cols, residual ? 4 : 2);
    const int need = (cols + 3) / 4;
    for (size_t first = 0; first < rows; first += LAUNCH_ROWS) {
        const Forward a = lot({x, residual, gamma, sum, y, rstd, nullptr, nullptr, rows, cols, eps}, first);
        const size_t n = a.rows;
        if (need <= 16) LAUNCH_TWO(rms_fwd_kernel, 16, 256, 1, (n + 15) / 16, a);
        else if (need <= 64) LAUNCH_TWO(rms_fwd_kernel, 64, 256, 1, (n + 3) / 4, a);
        else if (need <= 128 && by_waves(n)) LAUNCH_TWO(rms_fwd_kernel, 64, 256, 2, (n + 3) / 4, a);
        else if (need <= 256 && by_waves(n) && !stream) LAUNCH((rms_fwd_kernel<64, 256, 4, false>), (n + 3) / 4, 256, a);
        else if (need <= 256) LAUNCH_TWO(rms_fwd_kernel, 256, 256, 1, n, a);
        else if (need <= 1024) LAUNCH_TWO(rms_fwd_kernel, 512, 512, 2, n, a);
        else if (need <= 4096) LAUNCH_TWO(rms_fwd_kernel, 1024, 1024, 4, n, a);
        else LAUNCH((rms_fwd_long_kernel<1024>), n, 1024, a);
        XSMI_LAUNCH_CHECK("rms_fwd_kernel");
    }
    return XSMI_OK;
}

int xsmi_rms_norm_int8(const float *x, const float *residual, const float *gamma, float *sum, int8_t *q, float *scale, size_t rows, int cols,
                       float eps) {
    XSMI_REQUIRE_INIT();
    if (int rc = check("xsmi_rms_norm_int8", rows, cols, eps)) return rc;
    if (rows == 0) return XSMI_OK;
    XSMI_CHECK_ARG(x && gamma && q && scale && (residual == nullptr) == (sum == nullptr), "xsmi_rms_norm_int8: null pointer (a residual comes with a sum)");
    const bool stream = streams(rows, cols, residual ? 3 : 1);
    const int need = (cols + 3) / 4;
    for (size_t first = 0; first < rows; first += LAUNCH_ROWS) {
        const Forward a = lot({x, residual, gamma, sum, nullptr, nullptr, q, scale, rows, cols, eps}, first);
        const size_t n = a.rows;
        if (need <= 16) LAUNCH_TWO(rms_fwd_int8_kernel, 16, 256, 1, (n + 15) / 16, a);
        else if (need <= 64) LAUNCH_TWO(rms_fwd_int8_kernel, 64, 256, 1, (n + 3) / 4, a);
        else if (need <= 128 && by_waves(n)) LAUNCH_TWO(rms_fwd_int8_kernel, 64, 256, 2, (n + 3) / 4, a);
        else if (need <= 256 && by_waves(n)) LAUNCH_TWO(rms_fwd_int8_kernel, 64, 256, 4, (n + 3) / 4, a);
        else if (need <= 256) LAUNCH((rms_fwd_int8_kernel<256, 256, 1, false>), n, 256, a);
        else if (need <= 1024 && by_waves(n)) LAUNCH_TWO(rms_fwd_int8_kernel, 256, 256, 4, n, a);
        else if (need <= 1024) LAUNCH((rms_fwd_int8_kernel<1024, 1024, 1, false>), n, 1024, a);
        else if (need <= 2048 && by_waves(n)) LAUNCH_TWO(rms_fwd_int8_kernel, 512, 512, 4, n, a);
        else if (need <= 4096) LAUNCH_TWO(rms_fwd_int8_kernel, 1024, 1024, 4, n, a);
        else LAUNCH((rms_fwd_int8_long_kernel<1024>), n, 1024, a);
        XSMI_LAUNCH_CHECK("rms_fwd_int8_kernel");
    }
    return XSMI_OK;
}

size_t xsmi_rms_norm_workspace_bytes(size_t rows, int cols) {
    if (rows == 0 || rows >= MAX_ROWS || cols < 1 || cols > (1 << 30) || columns_apart(rows, cols)) return 0;
    return (size_t)backward_groups(rows, cols) * (size_t)cols * sizeof(float);
}

int xsmi_rms_norm_bwd(const float *dy, const float *s, const float *rstd, const float *gamma, const float *ds, float *dx1, float beta1,
                      float *dx2, float beta2, float *dgamma, float beta_gamma, size_t rows, int cols, void *ws, size_t ws_bytes) {
    XSMI_REQUIRE_INIT();
    if (int rc = check("xsmi_rms_norm_bwd", rows, cols, 0.f)) return rc;
    XSMI_CHECK_ARG((beta1 == 0.f || beta1 == 1.f) && (beta2 == 0.f || beta2 == 1.f) && (beta_gamma == 0.f || beta_gamma == 1.f),
                   "xsmi_rms_norm_bwd: beta is 0 or 1");
    XSMI_CHECK_ARG(!dx2 || (dx1 && dx1 != dx2), "xsmi_rms_norm_bwd: a second gradient comes beside the first, in memory of its own");
    if (rows == 0) return dgamma && beta_gamma == 0.f ? xsmi_fill(dgamma, 0.f, (size_t)cols) : XSMI_OK;
    XSMI_CHECK_ARG(dy && s && rstd && gamma, "xsmi_rms_norm_bwd: null pointer");
    const size_t want = dgamma ? xsmi_rms_norm_workspace_bytes(rows, cols) : 0;
    XSMI_CHECK_ARG(ws_bytes >= want && (ws || !want) && ((uintptr_t)ws & 15) == 0, "xsmi_rms_norm_bwd: workspace of %zu bytes, needs %zu", ws_bytes, want);
    if (!dx1 && !dgamma) return XSMI_OK;
    const int groups = backward_groups(rows, cols);
    const bool apart = dgamma && columns_apart(rows, cols);
    const Backward a = {dy, s, rstd, gamma, ds, dx1, dx2, dgamma && !apart ? (float *)ws : nullptr, beta1 != 0.f, beta2 != 0.f, rows, cols,
                        apart ? dgamma : nullptr, beta_gamma != 0.f, groups};
    const int grid = groups + (apart ? (cols + 31) / 32 : 0);
    const bool stream = streams(rows, cols, 3 + (ds != nullptr) + (dx2 != nullptr));
    const int need = (cols + 3) / 4;
    if (need <= 16) LAUNCH_TWO(rms_bwd_kernel, 16, 256, 1, grid, a);
    else if (need <= 64) LAUNCH_TWO(rms_bwd_kernel, 64, 256, 1, grid, a);
    else if (need <= 128 && by_waves(rows)) LAUNCH_TWO(rms_bwd_kernel, 64, 256, 2, grid, a);
    else if (need <= 256 && by_waves(rows)) LAUNCH_TWO(rms_bwd_kernel, 64, 256, 4, grid, a);
    else if (need <= 256) LAUNCH((rms_bwd_kernel<256, 256, 1, false>), grid, 256, a);
    else if (need <= 1024) LAUNCH_TWO(rms_bwd_kernel, 1024, 1024, 1, grid, a);
    else if (need <= 4096) LAUNCH_TWO(rms_bwd_kernel, 1024, 1024, 4, grid, a);
    else LAUNCH((rms_bwd_long_kernel<1024>), groups, 1024, a);
    XSMI_LAUNCH_CHECK("rms_bwd_kernel");
    if (dgamma && !apart) {
        hipLaunchKernelGGL(rms_dgamma_kernel, dim3((cols + 31) / 32), dim3(1024), 0, xsmi::stream(), (const float *)ws, groups, cols, dgamma,
                           beta_gamma != 0.f);
        XSMI_LAUNCH_CHECK("rms_dgamma_kernel");
    }
    return XSMI_OK;
}

}  // extern "C"
