// AdamW over many tensors in one launch, with moments in 32 or in 8 bits.
//
//   m' = beta1 m + (1 - beta1) g        v' = beta2 v + (1 - beta2) g^2
//   p' = p (1 - lr decay) - lr m' / (1 - beta1^t) / (sqrt(v' / (1 - beta2^t)) + eps)
//
// The number of steps taken lives in device memory and a one-thread launch in front of the step moves it: a recorded
// step that is replayed goes on counting.
//
// Moments in 8 bits.  Blocks of 256 elements share the exponent byte E of their largest value; a code keeps a float's
// exponent, counted from E - D, and the three leading bits of its fraction: code k > 0 is the float whose bits are
// (k - 1 + 8 (E - D)) << 20, and 0 is zero.  The first moment has a sign and seven bits (D = 14), the second eight bits
// (D = 30).  The scale of a block is a power of two, so a block whose largest value changes keeps its other values
// where they are: nothing is rounded again that has not moved.  Rounding is stochastic.  To the nearest code it would
// lose every change below half a step, 3 to 6 % of the value, and the second moment moves by 0.1 % of its distance to
// g^2 in a step: it would never decay.  The noise is a hash of the element's position, the step and a seed, so a step
// gives the same bits however it is launched.  The parameters are updated from the moments before they are rounded.
#include "xsmi_internal.h"
#include <math.h>

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef f4 f4u __attribute__((aligned(4)));              // parameters and gradients may start at any element
constexpr int MAX_TENSORS = 96;                          // of one launch: its arguments stay below 4 KB
constexpr int BLOCK = 256;                               // elements that share an exponent
constexpr uint64_t MAX_GROUPS = (1u << 24) - 1;          // workgroups of 256 threads in a launch

// What a step needs beside its tensors, moved by the launch in front of it (device memory of the caller).
struct StepState {
    uint64_t steps;      // taken so far
    float rate, root;    // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)
    uint32_t key, unused;
};
static_assert(sizeof(StepState) == XSMI_ADAMW_STATE_BYTES, "the header's size of the step state");

struct Tensors {
    float *p[MAX_TENSORS];
    const float *g[MAX_TENSORS];
    uint64_t start[MAX_TENSORS], n[MAX_TENSORS];
    uint32_t first[MAX_TENSORS];                         // workgroup that a tensor starts with
    int count;
};

struct Factors {
    float keep, b1, c1, b2, c2, eps;                     // 1 - lr decay, beta1, 1 - beta1, beta2, 1 - beta2, eps
};

struct Moments8 {
    uint8_t *m, *v, *me, *ve;
};

constexpr uint32_t STRIDE = 0x9E3779B1u;                 // fraction of the golden ratio, odd
__host__ __device__ __forceinline__ uint32_t mix(uint32_t h) {
    h ^= h >> 16;
    h *= 0x6A09E667u;                                    // fraction of the root of 2
    h ^= h >> 15;
    h *= 0xBB67AE85u;                                    // fraction of the root of 3
    return h ^ (h >> 16);
}

__device__ double power(double b, uint64_t t) {
    double r = 1.0;
    for (; t; t >>= 1, b *= b)
        if (t & 1) r *= b;
    return r;
}

// 2.3 us, a launch and two divisions in 64 bits.
__global__ void adamw_tick_kernel(StepState *s, double lr, double beta1, double beta2, uint32_t seed) {
    const uint64_t t = s->steps + 1;
    s->steps = t;
    s->rate = (float)(lr / (1.0 - power(beta1, t)));
    s->root = (float)(1.0 / sqrt(1.0 - power(beta2, t)));
    s->key = mix(seed + (uint32_t)t * STRIDE);
}

// Each product and sum of the moments is rounded by itself: the 8-bit codes are defined by these values.  Root and reciprocal
// are the hardware's, off by 2^-23; the root takes a value below 2^-126 for zero, so that much is added to it: where epsilon is 0 a
// parameter without gradients stays, and epsilon is all that counts where it is above 2^-60.
__device__ __forceinline__ void update(float &p, float g, float &m, float &v, const Factors &f, float rate, float root) {
    {
#pragma clang fp contract(off)
        m = m * f.b1 + g * f.c1;
        v = v * f.b2 + g * f.c2 * g;
    }
    p = p * f.keep - m * rate * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v + 0x1p-126f) * root + f.eps);
}

// The tensor of this workgroup (the last one whose first workgroup is not behind it).
__device__ __forceinline__ int tensor_of(const Tensors &t, uint32_t group) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= group) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// STREAM: past the caches' replacement, where a step's operands are larger than the caches.
template <bool STREAM>
__device__ __forceinline__ f4 load4(const float *p) {    // from any element on
    return STREAM ? __builtin_nontemporal_load(reinterpret_cast<const f4u *>(p)) : *reinterpret_cast<const f4u *>(p);
}
template <bool STREAM>
__device__ __forceinline__ void store4(float *p, f4 v) {
    if (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<f4u *>(p));
    else *reinterpret_cast<f4u *>(p) = v;
}
template <bool STREAM, typename T>
__device__ __forceinline__ T load(const T *p) {
    return STREAM ? __builtin_nontemporal_load(p) : *p;
}
template <bool STREAM, typename T>
__device__ __forceinline__ void store(T *p, T v) {
    if (STREAM) __builtin_nontemporal_store(v, p);
    else *p = v;
}

template <bool STREAM>
__device__ __forceinline__ f4 load4(const float *p, uint64_t i, uint64_t n) {
    if (i + 4 <= n) return load4<STREAM>(p + i);
    f4 r = {0.f, 0.f, 0.f, 0.f};
    if (i < n) r.x = p[i];
    if (i + 1 < n) r.y = p[i + 1];
    if (i + 2 < n) r.z = p[i + 2];
    return r;
}

template <bool STREAM>
__device__ __forceinline__ void store4(float *p, uint64_t i, uint64_t n, f4 v) {
    if (i + 4 <= n) {
        store4<STREAM>(p + i, v);
        return;
    }
    if (i < n) p[i] = v.x;
    if (i + 1 < n) p[i + 1] = v.y;
    if (i + 2 < n) p[i + 2] = v.z;
}

// 256 threads, four elements each of one tensor: more of them a thread gains nothing (ResNet-18, 11.7 million elements, from the caches: 57.5 us;
// eight a thread 58.2, sixteen 60.3).  Streamed, from memory: 57 us, 5.7 TB/s; not streamed 62.  The moments are padded to whole blocks of 256 elements, of which those behind the tensor stay
// zero: zero gradients of zero moments.
template <bool STREAM>
__global__ void __launch_bounds__(256) adamw_kernel(Tensors t, float *__restrict__ m, float *__restrict__ v, Factors f,
                                                    const StepState *__restrict__ s) {
    const int k = tensor_of(t, blockIdx.x);
    const uint64_t n = t.n[k], i = (uint64_t)(blockIdx.x - t.first[k]) * 1024u + 4u * threadIdx.x;
    if (i >= n) return;
    float *const p = t.p[k];
    f4 *const mp = reinterpret_cast<f4 *>(m + t.start[k] + i), *const vp = reinterpret_cast<f4 *>(v + t.start[k] + i);
    const float rate = s->rate, root = s->root;
    f4 pp = load4<STREAM>(p, i, n), mm = load<STREAM>(mp), vv = load<STREAM>(vp);
    const f4 gg = load4<STREAM>(t.g[k], i, n);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float pe = pp[e], me = mm[e], ve = vv[e];
        update(pe, gg[e], me, ve, f, rate, root);
        pp[e] = pe, mm[e] = me, vv[e] = ve;
    }
    store4<STREAM>(p, i, n, pp);
    store<STREAM>(mp, mm);
    store<STREAM>(vp, vv);
}

__device__ __forceinline__ float decode_bits(uint32_t k, int lowest) {       // lowest = 8 (E - D) - 1
    return __uint_as_float(k ? (uint32_t)((int)k + lowest) << 20 : 0u);
}

// Whether a value below the smallest code becomes that code instead of zero; unit is 2^-16 of the smallest code.
__device__ __forceinline__ uint32_t reaches(uint32_t bits, uint32_t noise, float unit) {
    return __uint_as_float(bits) > ((float)noise + 0.5f) * unit ? 1u : 0u;
}

// The largest value of a wave, in a scalar register: by rows of 16 lanes, then across rows.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#define STEP(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, false))
    STEP(0x111, 0xf);                                    // from one, two, four and eight lanes below
    STEP(0x112, 0xf);
    STEP(0x114, 0xf);
    STEP(0x118, 0xf);
    STEP(0x142, 0xa);                                    // a row's last lane to the row above
    STEP(0x143, 0xc);                                    // lane 31 to the upper half
#undef STEP
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

constexpr int DEPTH_M = 14, DEPTH_V = 30, LEAST_M = 48, LEAST_V = 64, BAD = 255;

// One wave of four elements a lane for each block of 256.  What bounds it beside memory is the vector unit: some 70 operations
// an element, of which the hash takes 16 and the choice between the smallest code and zero would take another twelve: a wave makes it
// only where one of its values lies that low.  134 million elements: 336 us, 6.4 TB/s; ResNet-18: 37 us, 5.1 TB/s.
template <bool FULL, bool STREAM>
__device__ __forceinline__ void adamw8_block(float *p, const float *g, uint64_t block, uint64_t n, uint64_t start, const Moments8 &q, const Factors &f,
                                             float rate, float root, uint32_t key, int lane) {
    const uint64_t i = block + 4u * lane, place = start + block, b = place / BLOCK;
    f4 pp, gg;
    if (FULL) {
        pp = load4<STREAM>(p + i);
        gg = load4<STREAM>(g + i);
    } else {
        pp = load4<STREAM>(p, i, n);
        gg = load4<STREAM>(g, i, n);
    }
    uint32_t *const mp = reinterpret_cast<uint32_t *>(q.m + place) + lane, *const vp = reinterpret_cast<uint32_t *>(q.v + place) + lane;
    uint32_t mq = load<STREAM>(mp), vq = load<STREAM>(vp);
    int em = __builtin_amdgcn_readfirstlane((int)q.me[b]), ev = __builtin_amdgcn_readfirstlane((int)q.ve[b]);
    float mm[4], vv[4];
    const int lm = 8 * (em - DEPTH_M) - 1, lv = 8 * (ev - DEPTH_V) - 1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        mm[e] = copysignf(decode_bits(mq >> (8 * e) & 127u, lm), __uint_as_float(mq << (24 - 8 * e)));
        vv[e] = decode_bits(vq >> (8 * e) & 255u, lv);
    }
    if (em == BAD) mm[0] = mm[1] = mm[2] = mm[3] = NAN;
    if (ev == BAD) vv[0] = vv[1] = vv[2] = vv[3] = NAN;
    uint32_t mb[4], vb[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float pe = pp[e];
        update(pe, gg[e], mm[e], vv[e], f, rate, root);
        pp[e] = pe;
        mb[e] = __float_as_uint(mm[e]) & 0x7fffffffu;
        vb[e] = __float_as_uint(vv[e]) & 0x7fffffffu;
    }
    if (FULL) store4<STREAM>(p + i, pp);
    else store4<STREAM>(p, i, n, pp);
    em = max((int)(wave_max(max(max(mb[0], mb[1]), max(mb[2], mb[3]))) >> 23), LEAST_M);
    ev = max((int)(wave_max(max(max(vb[0], vb[1]), max(vb[2], vb[3]))) >> 23), LEAST_V);
    const int lm2 = 8 * (em - DEPTH_M) - 1, lv2 = 8 * (ev - DEPTH_V) - 1;
    const uint32_t floor_m = (uint32_t)(em - DEPTH_M) << 23, floor_v = (uint32_t)(ev - DEPTH_V) << 23;
    const uint32_t first = (uint32_t)place * STRIDE + (uint32_t)(place >> 32) * 0x510E527Fu + key + 4u * (uint32_t)lane * STRIDE;
    uint32_t h[4], mk[4], vk[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        h[e] = mix(first + (uint32_t)e * STRIDE);
        mk[e] = ((mb[e] + ((h[e] << 4 & 0xffff0u) | 8u)) >> 20) - (uint32_t)lm2;
        vk[e] = ((vb[e] + ((h[e] >> 12 & 0xffff0u) | 8u)) >> 20) - (uint32_t)lv2;
    }
    const bool low = min(min(mb[0], mb[1]), min(mb[2], mb[3])) < floor_m || min(min(vb[0], vb[1]), min(vb[2], vb[3])) < floor_v;
    if (__builtin_amdgcn_ballot_w64(low)) {
        const float um = __uint_as_float(floor_m - (16u << 23)), uv = __uint_as_float(floor_v - (16u << 23));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (mb[e] < floor_m) mk[e] = reaches(mb[e], h[e] & 0xffffu, um);
            if (vb[e] < floor_v) vk[e] = reaches(vb[e], h[e] >> 16, uv);
        }
    }
    mq = vq = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        mq |= (mk[e] | (__float_as_uint(mm[e]) >> 24 & 128u)) << (8 * e);
        vq |= vk[e] << (8 * e);
    }
    // A value of 2^127 and more, an infinity or NaN: the whole block reads as NaN from now on.
    if (em >= 254) em = BAD, mq = 0;
    if (ev >= 254) ev = BAD, vq = 0;
    store<STREAM>(mp, mq);
    store<STREAM>(vp, vq);
    if (lane == 0) q.me[b] = (uint8_t)em, q.ve[b] = (uint8_t)ev;
}

template <bool STREAM>
__global__ void __launch_bounds__(256) adamw8_kernel(Tensors t, Moments8 q, Factors f, const StepState *__restrict__ s) {
    const int k = tensor_of(t, blockIdx.x);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t n = t.n[k], block = (uint64_t)(blockIdx.x - t.first[k]) * 1024u + 256u * wave;
    if (block >= n) return;                              // the same for the whole wave
    if (block + BLOCK <= n) adamw8_block<true, STREAM>(t.p[k], t.g[k], block, n, t.start[k], q, f, s->rate, s->root, s->key, lane);
    else adamw8_block<false, STREAM>(t.p[k], t.g[k], block, n, t.start[k], q, f, s->rate, s->root, s->key, lane);
}

// The values that 8-bit moments stand for, four of each a thread (134 million: 219 us, 6.1 TB/s).
template <bool STREAM>
__global__ void __launch_bounds__(256) adamw_moments_kernel(Moments8 q, float *__restrict__ m, float *__restrict__ v, uint64_t n) {
    const uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    const uint32_t mq = load<STREAM>(reinterpret_cast<const uint32_t *>(q.m + i)), vq = load<STREAM>(reinterpret_cast<const uint32_t *>(q.v + i));
    const int em = q.me[i / BLOCK], ev = q.ve[i / BLOCK];
    f4 mm, vv;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t mk = mq >> (8 * e) & 255u, vk = vq >> (8 * e) & 255u;
        mm[e] = em == BAD ? NAN : copysignf(decode_bits(mk & 127u, 8 * (em - DEPTH_M) - 1), __uint_as_float(mk << 24));
        vv[e] = ev == BAD ? NAN : decode_bits(vk, 8 * (ev - DEPTH_V) - 1);
    }
    store<STREAM>(reinterpret_cast<f4 *>(m + i), mm);
    store<STREAM>(reinterpret_cast<f4 *>(v + i), vv);
}

}  // namespace

extern "C" {

int xsmi_adamw_step(int count, float *const *ps, const float *const *gs, const size_t *starts, const size_t *ns, void *m, void *v,
                    uint8_t *m_exp, uint8_t *v_exp, size_t moments, int state_bits, double lr, double beta1, double beta2, double eps,
                    double weight_decay, uint32_t seed, void *state) {
    XSMI_REQUIRE_INIT();
    XSMI_CHECK_ARG(count >= 0 && (count == 0 || (ps && gs && starts && ns)), "xsmi_adamw_step: bad argument");
    XSMI_CHECK_ARG(state_bits == 32 || state_bits == 8, "xsmi_adamw_step: moments in 32 or 8 bits, not %d", state_bits);
    XSMI_CHECK_ARG(m && v && state && (state_bits == 32 || (m_exp && v_exp)), "xsmi_adamw_step: null pointer");
    XSMI_CHECK_ARG((((uintptr_t)m | (uintptr_t)v) & 15) == 0 && ((uintptr_t)state & 7) == 0, "xsmi_adamw_step: the moments are not aligned to 16 bytes");
    XSMI_CHECK_ARG(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "xsmi_adamw_step: betas %g and %g, expected 0 <= beta < 1", beta1, beta2);
    XSMI_CHECK_ARG(lr >= 0 && eps >= 0 && weight_decay >= 0, "xsmi_adamw_step: negative rate, epsilon or decay");
    for (int i = 0; i < count; ++i) {
        XSMI_CHECK_ARG(ps[i] && gs[i], "xsmi_adamw_step: null pointer in tensor %d", i);
        XSMI_CHECK_ARG(starts[i] % BLOCK == 0 && starts[i] <= moments && ns[i] <= moments - starts[i],
                       "xsmi_adamw_step: tensor %d has its moments at %zu of %zu", i, starts[i], moments);
        XSMI_CHECK_ARG(ns[i] < 1024ull * MAX_GROUPS, "xsmi_adamw_step: tensor %d has %zu elements", i, ns[i]);
    }
    XSMI_CHECK_ARG(moments % BLOCK == 0, "xsmi_adamw_step: room for %zu moments, expected a multiple of %d", moments, BLOCK);
    hipLaunchKernelGGL(adamw_tick_kernel, dim3(1), dim3(1), 0, xsmi::stream(), (StepState *)state, lr, beta1, beta2, seed);
    XSMI_LAUNCH_CHECK("adamw_tick_kernel");
    const Factors f = {(float)(1.0 - lr * weight_decay), (float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps};
    const Moments8 q = {(uint8_t *)m, (uint8_t *)v, m_exp, v_exp};
    // What is read: past half of the last-level cache (256 MB) it is streamed, for a forward and a backward have the cache before it comes
    // again (ResNet-18, 187 MB: 66.5 us without and 58.0 with, after other operands; 51.7 and 56.4 if nothing ran in between).
    double bytes = 0;
    for (int i = 0; i < count; ++i) bytes += (double)ns[i] * (state_bits == 32 ? 16 : 10);
    const bool stream = bytes > 128e6;
    for (int done = 0; done < count;) {
        Tensors t;
        uint64_t groups = 0;
        int k = 0;
        for (; done < count && k < MAX_TENSORS; ++done) {
            if (ns[done] == 0) continue;
            const uint64_t more = (ns[done] + 1023u) / 1024u;
            if (groups + more > MAX_GROUPS) break;
            t.p[k] = ps[done], t.g[k] = gs[done], t.start[k] = starts[done], t.n[k] = ns[done];
            t.first[k++] = (uint32_t)groups;
            groups += more;
        }
        t.count = k;
        if (k == 0) break;                               // nothing but empty tensors was left
#define LAUNCH(kernel, ...) hipLaunchKernelGGL((kernel), dim3((uint32_t)groups), dim3(256), 0, xsmi::stream(), t, __VA_ARGS__, f, (const StepState *)state)
        if (state_bits == 32) {
            if (stream) LAUNCH((adamw_kernel<true>), (float *)m, (float *)v);
            else LAUNCH((adamw_kernel<false>), (float *)m, (float *)v);
        } else {
            if (stream) LAUNCH((adamw8_kernel<true>), q);
            else LAUNCH((adamw8_kernel<false>), q);
        }
#undef LAUNCH
        XSMI_LAUNCH_CHECK("adamw_kernel");
    }
    return XSMI_OK;
}

int xsmi_adamw_moments(const uint8_t *m8, const uint8_t *v8, const uint8_t *m_exp, const uint8_t *v_exp, float *m, float *v, size_t moments) {
    XSMI_REQUIRE_INIT();
    if (moments == 0) return XSMI_OK;
    XSMI_CHECK_ARG(m8 && v8 && m_exp && v_exp && m && v, "xsmi_adamw_moments: null pointer");
    XSMI_CHECK_ARG(moments % BLOCK == 0, "xsmi_adamw_moments: %zu moments, expected a multiple of %d", moments, BLOCK);
    XSMI_CHECK_ARG((((uintptr_t)m | (uintptr_t)v) & 15) == 0 && (((uintptr_t)m8 | (uintptr_t)v8) & 3) == 0, "xsmi_adamw_moments: unaligned moments");
    const uint64_t groups = (moments + 1023) / 1024;
    XSMI_CHECK_ARG(groups <= MAX_GROUPS, "xsmi_adamw_moments: %zu moments", moments);
    const Moments8 q = {(uint8_t *)m8, (uint8_t *)v8, (uint8_t *)m_exp, (uint8_t *)v_exp};
    if ((double)moments * 10 > 256e6) hipLaunchKernelGGL(adamw_moments_kernel<true>, dim3((uint32_t)groups), dim3(256), 0, xsmi::stream(), q, m, v, (uint64_t)moments);
    else hipLaunchKernelGGL(adamw_moments_kernel<false>, dim3((uint32_t)groups), dim3(256), 0, xsmi::stream(), q, m, v, (uint64_t)moments);
    XSMI_LAUNCH_CHECK("adamw_moments_kernel");
    return XSMI_OK;
}

}  // extern "C"
