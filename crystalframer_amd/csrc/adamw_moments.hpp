// AdamW over many tensors of several types with moments in 32 or in 8 bits, and the common norm of the gradients that it
// clips by.  The rule, the 8-bit formats and the hash are written down in crystalframer_hip.h.
//
// Bound by HBM: per float32 parameter 16 bytes (8 bits) or 28 (32 bits), in 16 bits 10 or 22, against some 60 or 20 vector
// instructions.  151 M float32 parameters: the update 432 us in 8 bits (5.6 TB/s), 740 in 32 (5.7), the gradients' norm 90 (6.7),
// the values of 8-bit moments 300 (5.0); 25 M bfloat16: 54 us in 8 bits (4.6 TB/s, the instructions nearly as long), 103 in 32 (5.4).
// 952 000 float32 in 65 tensors: 7 us, and 2 to 3 for the launch before.
//
// The tensors' addresses travel in the kernel arguments.  What all elements share (the step's bias corrections, its hash
// key, the clipping factor) is made by a launch of one workgroup before, which also advances the step.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "element_types.hpp"

namespace cfh {

constexpr int MOMENT_BLOCK = 64;          // elements that share a scale
constexpr int PARAM_MAX_JOBS = 88;        // tensors per launch (kernel arguments: 4 KB)
constexpr int ADAMW_CHUNK = 2048;         // elements per workgroup of 256 threads
constexpr uint32_t MAX_CHUNKS = 0xffffff;     // workgroups of a launch: a grid counts its threads in 32 bits
constexpr int ADAMW_FEW = 1024;           // the same where there are not enough of those to go round
constexpr int64_t CACHED_BYTES = 256LL << 20;      // that the last cache holds
constexpr int GRAD_NORM_CHUNK = 8192;     // elements per turn of a workgroup of 256 threads: eight (four) loads under way per lane
constexpr int GRAD_NORM_FEW = 2048;       // the same where there are not enough of those to go round
constexpr int GRAD_NORM_BLOCKS = 2048;    // workgroups per launch at most

struct ParamJob {
    void* p;
    const void* g;
    uint64_t first;       // element of the flat moments
    uint32_t n;
    uint32_t chunk0;      // first chunk of this tensor
    int32_t dtype;
    int32_t reserved0;
};
struct ParamJobs {
    ParamJob job[PARAM_MAX_JOBS];
    int32_t njobs;
    uint32_t chunks;
};
struct Moments {
    void* m;
    void* v;
    uint8_t* m_scale;
    uint8_t* v_scale;
};
// The step's share of the update, in device memory.
struct AdamWStep {
    float step_size, inv_sqrt_bc2, decay, clip;
    uint32_t key;
};
struct AdamWRates {
    double beta1, beta2;
    float eps;
};

// The job with job[k].chunk0 <= chunk < job[k + 1].chunk0: every lane looks at one or two of them, a round trip to memory instead of
// one for every halving.
__device__ __forceinline__ const ParamJob& job_of(const ParamJobs& T, uint32_t chunk) {
    static_assert(PARAM_MAX_JOBS <= 128);
    const int lane = (int)threadIdx.x & 63;
    const bool a = lane < T.njobs && T.job[min(lane, PARAM_MAX_JOBS - 1)].chunk0 <= chunk;
    const bool b = lane + 64 < T.njobs && T.job[min(lane + 64, PARAM_MAX_JOBS - 1)].chunk0 <= chunk;
    return T.job[__popcll(__builtin_amdgcn_ballot_w64(a)) + __popcll(__builtin_amdgcn_ballot_w64(b)) - 1];
}

__device__ __forceinline__ double block_sum(double x) {
    __shared__ double part[4];
    for (int d = 32; d > 0; d /= 2) x += __shfl_xor(x, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    return part[0] + part[1] + part[2] + part[3];
}

struct GradClip {
    const double* sums;
    int count;
    double max_norm;
    float* norm;              // NULL: no clipping
};

// One workgroup: the norm by all its threads, what depends on the number of the step by one of another wavefront meanwhile.
__global__ __launch_bounds__(256) void adamw_begin_kernel(AdamWStep* out, unsigned long long* step, double lr, double beta1, double beta2,
                                                          double wd, const GradClip C) {
    if (threadIdx.x == 64) {
        const unsigned long long t = *step + 1ULL;
        *step = t;
        // 1 - beta^t by expm1: for beta close to 1 and the first steps the difference cancels
        const double bc1 = -expm1((double)t * log(beta1)), bc2 = -expm1((double)t * log(beta2));
        out->step_size = (float)(lr / bc1);
        out->inv_sqrt_bc2 = (float)(1.0 / sqrt(bc2));
        out->decay = (float)(1.0 - lr * wd);
        uint32_t k = (uint32_t)t * 0x6A09E667u;
        k = (k ^ (k >> 15)) * 0x9E3779B1u;
        out->key = k ^ (k >> 16);
    }
    float factor = 1.0f;
    if (C.norm) {
        double s = 0.0;
        for (int i = threadIdx.x; i < C.count; i += 256) s += C.sums[i];
        s = sqrt(block_sum(s));
        const double c = C.max_norm / (s + 1e-6);
        factor = c >= 1.0 ? 1.0f : (float)c;
        if (threadIdx.x == 0) *C.norm = (float)s;
    }
    if (threadIdx.x == 0) out->clip = factor;
}

// of element * 0x9E3779B1 + key
__device__ __forceinline__ uint32_t moment_hash(uint32_t x) {
    x = (x ^ (x >> 16)) * 0xBB67AE85u;
    return x ^ (x >> 15);
}

// How a chunk is gone through.  WHOLE: all its elements are there; else a lane may find fewer, or none.  STREAM: past the caches.
// EXACT: see adamw_update.
template <bool WHOLE_, bool STREAM_, bool EXACT_ = false>
struct Way {
    static constexpr bool WHOLE = WHOLE_, STREAM = STREAM_, EXACT = EXACT_;
};
// The hardware's root and reciprocal: each within one unit of the last place of what is a thousandth of the parameter.  The root takes
// what is below 2^-126 for zero: beside an eps of 2^-38 that is no difference (2^-63), beside a smaller one whole functions
// are called (WAY::EXACT).
template <typename WAY, typename T, typename M, int E>
__device__ __forceinline__ void adamw_update(T (&p)[E], const M (&m)[E], const M (&v)[E], const AdamWStep& S, float eps) {
    if constexpr (WAY::EXACT) {
#pragma unroll
        for (int j = 0; j < E; j++)
            p[j] = from_float<T>(to_float(p[j]) * S.decay - S.step_size * ((float)m[j] / (sqrtf((float)v[j]) * S.inv_sqrt_bc2 + eps)));
        return;
    }
#pragma unroll
    for (int j = 0; j < E; j++) {
        const float root = __builtin_amdgcn_sqrtf((float)v[j]) * S.inv_sqrt_bc2 + eps;
        p[j] = from_float<T>(to_float(p[j]) * S.decay - S.step_size * ((float)m[j] * __builtin_amdgcn_rcpf(root)));
    }
}

// An 8-bit code without its sign is a double's exponent and mantissa cut to three bits: its bits, moved under the high word's
// exponent field, are the value times 2^bias, denormals included, and back it is one shift.  bias: 1016 (exp_avg, e4m3: the
// smallest normal value 2^-6 has exponent field 1) and 993 (exp_avg_sq: 2^-29).
constexpr int M_BIAS = 1016, V_BIAS = 993, M_TOP = 7, V_TOP = 0;
constexpr uint32_t HIGH_INF = 0x7ff00000u, HIGH_2_128 = 0x47f00000u;      // high words: no number from here on; 2^128

__device__ __forceinline__ uint32_t high_word(double x) { return (uint32_t)__double2hiint(x); }
// The value of byte j of a word of codes; with the sign in its top bit for exp_avg.
__device__ __forceinline__ double m_value(uint32_t word, int j, int scale) {
    const int high = (((int)(word << (24 - 8 * j)) >> 24) << 17) & (int)0x80FE0000u;
    return ldexp(__hiloint2double(high, 0), scale);
}
__device__ __forceinline__ double v_value(uint32_t word, int j, int scale) {
    return ldexp(__hiloint2double((int)((word >> 8 * j & 255u) << 17), 0), scale);
}
// floor(x / step + (2 k + 1) / 2^17) as a code; x >= 0, odd = 2 k + 1 in 17 bits
__device__ __forceinline__ uint32_t code_of(double x, int scale, uint32_t odd) { return (high_word(ldexp(x, scale)) + odd) >> 17; }
// Whether a word of codes holds one that is no number (exp_avg) or more than 32 bits hold (exp_avg_sq).
__device__ __forceinline__ bool m_odd(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }
__device__ __forceinline__ bool v_odd(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & w & 0x80808080u) != 0; }

// The scale byte of a block whose largest magnitude has this high word (0: none): the largest then lies in [2^top, 2^(top + 1)).
__device__ __forceinline__ int scale_byte(uint32_t high, int top) {
    const int e = (int)(high >> 20) - 1023 - top;
    return high == 0 ? 0 : min(max(e, -127), 127) + 127;
}

// b x + y, every product and the sum rounded by itself: sums of codes and of gradients of few bits lie on powers of two,
// the borders of a block's scale, more often than by chance, and a fused product would come out on the other side of them.
__device__ __forceinline__ double moment_mix(double b, double x, double y) {
#pragma clang fp contract(off)
    return b * x + y;
}

// Largest over the LANES (8 or 16) neighbouring lanes of a block.
template <int LANES>
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
    auto other = [&](auto ctrl) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, false); };
    x = max(x, other(std::integral_constant<int, 0xB1>()));       // quad_perm [1,0,3,2], [2,3,0,1], half_mirror, mirror
    x = max(x, other(std::integral_constant<int, 0x4E>()));
    x = max(x, other(std::integral_constant<int, 0x141>()));
    if constexpr (LANES == 16) x = max(x, other(std::integral_constant<int, 0x140>()));
    return x;
}

// Words of a lane's 4 to 32 bytes at an address of ALIGN bytes, for accesses past the caches.
template <int BYTES, int ALIGN>
struct Words;
#define CFH_WORDS(bytes, alignment) \
    template <> struct Words<bytes, alignment> { typedef uint32_t type __attribute__((ext_vector_type(bytes / 4), aligned(alignment))); };
CFH_WORDS(16, 4)
CFH_WORDS(16, 2)
CFH_WORDS(32, 4)
CFH_WORDS(8, 1)
CFH_WORDS(8, 2)
#undef CFH_WORDS
template <> struct Words<4, 1> { typedef uint32_t type __attribute__((aligned(1))); };

// `E` elements of a tensor from `i` on, of which a lane takes care: a block of 64 lies in 64 / E lanes.
template <typename WAY, typename T, int E>
__device__ __forceinline__ void load_elements(T (&o)[E], const T* from, uint32_t i, uint32_t n) {
    if (WAY::WHOLE || i + E <= n) {
        if constexpr (WAY::STREAM) {
            using V = typename Words<sizeof(o), alignof(T)>::type;
            const V x = __builtin_nontemporal_load(reinterpret_cast<const V*>(from + i));
            __builtin_memcpy(o, &x, sizeof(o));
        } else __builtin_memcpy(o, from + i, sizeof(o));
    } else {
#pragma unroll
        for (int j = 0; j < E; j++) o[j] = i + j < n ? from[i + j] : T{};
    }
}
template <typename WAY, typename T, int E>
__device__ __forceinline__ void store_elements(T* to, const T (&o)[E], uint32_t i, uint32_t n) {
    if (WAY::WHOLE || i + E <= n) {
        if constexpr (WAY::STREAM) {
            using V = typename Words<sizeof(o), alignof(T)>::type;
            V x;
            __builtin_memcpy(&x, o, sizeof(o));
            __builtin_nontemporal_store(x, reinterpret_cast<V*>(to + i));
        } else __builtin_memcpy(to + i, o, sizeof(o));
    } else {
#pragma unroll
        for (int j = 0; j < E; j++)
            if (i + j < n) to[i + j] = o[j];
    }
}
// E codes as words
template <typename WAY, int E>
__device__ __forceinline__ void load_codes(uint32_t (&w)[E / 4], const uint8_t* from, uint32_t i, uint32_t n) {
    uint8_t c[E];
    load_elements<WAY>(c, from, i, n);
    __builtin_memcpy(w, c, E);
}
template <typename WAY, int E>
__device__ __forceinline__ void store_codes(uint8_t* to, const uint32_t (&w)[E / 4], uint32_t i, uint32_t n) {
    uint8_t c[E];
    __builtin_memcpy(c, w, E);
    store_elements<WAY>(to, c, i, n);
}

template <typename WAY, typename T, int E>
__device__ __forceinline__ void moments32(const ParamJob& J, uint32_t i, const T (&g)[E], T (&p)[E], const Moments& W, const AdamWStep& S,
                                          const AdamWRates& R) {
    float* const pm = reinterpret_cast<float*>(W.m) + J.first;
    float* const pv = reinterpret_cast<float*>(W.v) + J.first;
    const float b1 = (float)R.beta1, a1 = (float)(1.0 - R.beta1), b2 = (float)R.beta2, a2 = (float)(1.0 - R.beta2);
    float m[E], v[E];
    load_elements<WAY>(m, pm, i, J.n);
    load_elements<WAY>(v, pv, i, J.n);
#pragma unroll
    for (int j = 0; j < E; j++) {
        const float c = to_float(g[j]) * S.clip;
        m[j] = b1 * m[j] + a1 * c;
        v[j] = b2 * v[j] + a2 * c * c;
    }
    adamw_update<WAY>(p, m, v, S, R.eps);
    store_elements<WAY>(pm, m, i, J.n);
    store_elements<WAY>(pv, v, i, J.n);
}

// Some 60 vector instructions per element, which the 16 bytes of a float32 parameter hide and the 10 of one in 16 bits nearly do;
// what 32 bits do not hold is looked for in words of four codes and in the largest of a lane, and dealt with on a path of its own.
template <typename WAY, typename T, int E>
__device__ __forceinline__ void moments8(const ParamJob& J, uint32_t i, const T (&g)[E], T (&p)[E], const Moments& W, const AdamWStep& S,
                                         const AdamWRates& R) {
    uint8_t* const pm = reinterpret_cast<uint8_t*>(W.m) + J.first;
    uint8_t* const pv = reinterpret_cast<uint8_t*>(W.v) + J.first;
    uint8_t* const ps = W.m_scale + J.first / MOMENT_BLOCK;
    uint8_t* const pt = W.v_scale + J.first / MOMENT_BLOCK;
    uint32_t cm[E / 4], cv[E / 4];
    load_codes<WAY, E>(cm, pm, i, J.n);
    load_codes<WAY, E>(cv, pv, i, J.n);
    const bool some = WAY::WHOLE || i < J.n;
    const int sm0 = some ? M_BIAS - 127 + (int)ps[i / MOMENT_BLOCK] : 0, sv0 = some ? V_BIAS - 127 + (int)pt[i / MOMENT_BLOCK] : 0;
    const double a1 = 1.0 - R.beta1, a2 = 1.0 - R.beta2;
    double m[E], v[E];
    bool odd = false;
#pragma unroll
    for (int k = 0; k < E / 4; k++) odd = odd || m_odd(cm[k]) || v_odd(cv[k]);
#pragma unroll
    for (int j = 0; j < E; j++) {
        m[j] = m_value(cm[j / 4], j % 4, sm0);
        v[j] = v_value(cv[j / 4], j % 4, sv0);
    }
    if (__any(odd)) {
#pragma unroll
        for (int j = 0; j < E; j++) {
            if ((cm[j / 4] >> 8 * (j % 4) & 127u) == 127u) m[j] = __longlong_as_double(0x7ff8000000000000LL);
            if ((cv[j / 4] >> 8 * (j % 4) & 255u) == 255u) v[j] = __longlong_as_double(0x7ff0000000000000LL);
        }
    }
    uint32_t hm = 0, hv = 0;
#pragma unroll
    for (int j = 0; j < E; j++) {
        const double c = (double)to_float(g[j]) * (double)S.clip;
        m[j] = moment_mix(R.beta1, m[j], a1 * c);
        v[j] = moment_mix(R.beta2, v[j], a2 * c * c);
        hm = max(hm, high_word(m[j]) & 0x7fffffffu);
        hv = max(hv, high_word(v[j]));
    }
    odd = __any(hm >= HIGH_INF || hv >= HIGH_2_128);
    if (odd) {            // what 32 bits do not hold stays out of the scale
        hm = hv = 0;
#pragma unroll
        for (int j = 0; j < E; j++) {
            const uint32_t a = high_word(m[j]) & 0x7fffffffu, b = high_word(v[j]);
            hm = a < HIGH_INF ? max(hm, a) : hm;
            hv = b < HIGH_2_128 ? max(hv, b) : hv;
        }
    }
    const int sm = scale_byte(block_max<MOMENT_BLOCK / E>(hm), M_TOP), sv = scale_byte(block_max<MOMENT_BLOCK / E>(hv), V_TOP);
    const uint32_t x0 = ((uint32_t)J.first + i) * 0x9E3779B1u + S.key;
#pragma unroll
    for (int k = 0; k < E / 4; k++) cm[k] = cv[k] = 0;
#pragma unroll
    for (int j = 0; j < E; j++) {
        const uint32_t h = moment_hash(x0 + (uint32_t)j * 0x9E3779B1u);
        uint32_t a = code_of(fabs(m[j]), -(M_BIAS - 127 + sm), (h << 1 & 0x1ffffu) | 1u);
        uint32_t b = code_of(v[j], -(V_BIAS - 127 + sv), h >> 15 | 1u);
        b = max(b, min(high_word(v[j]), 1u));          // (no double that comes up here is below 2^-1022)
        if (odd) {
            if ((high_word(m[j]) & 0x7fffffffu) >= HIGH_INF) a = 127u;
            if (high_word(v[j]) >= HIGH_2_128) b = 255u;
        }
        cm[j / 4] |= ((high_word(m[j]) >> 24 & 128u) | a) << 8 * (j % 4);
        cv[j / 4] |= b << 8 * (j % 4);
    }
    adamw_update<WAY>(p, m, v, S, R.eps);
    store_codes<WAY, E>(pm, cm, i, J.n);
    store_codes<WAY, E>(pv, cv, i, J.n);
    if (some && i % MOMENT_BLOCK == 0) {
        ps[i / MOMENT_BLOCK] = (uint8_t)sm;
        pt[i / MOMENT_BLOCK] = (uint8_t)sv;
    }
}

template <typename T, int BITS, int CHUNK, typename WAY>
__device__ __forceinline__ void adamw_chunk(const ParamJob& J, uint32_t base, const Moments& W, const AdamWStep* step, const AdamWRates& R) {
    constexpr int E = 16 / (int)sizeof(T) < CHUNK / 256 ? 16 / (int)sizeof(T) : CHUNK / 256;
    T* const pp = reinterpret_cast<T*>(J.p);
    const AdamWStep S = *step;
    for (int k = 0; k < CHUNK / (256 * E); k++) {
        const uint32_t i = base + ((uint32_t)k * 256 + threadIdx.x) * E;
        T g[E], p[E];
        load_elements<WAY>(g, reinterpret_cast<const T*>(J.g), i, J.n);
        load_elements<WAY>(p, pp, i, J.n);
        if constexpr (BITS == 32) moments32<WAY>(J, i, g, p, W, S, R);
        else moments8<WAY>(J, i, g, p, W, S, R);
        store_elements<WAY>(pp, p, i, J.n);
    }
}

// STREAM: tensors and moments that the last cache does not hold from one step to the next go past it (151 M float32 parameters, 8 bits
// 430 -> 420 us, 32 bits 764 -> 746); smaller ones stay for who reads them next (25 M bfloat16: the values of the moments 48 -> 36).
template <int BITS, int CHUNK, bool STREAM, bool EXACT>
__global__ __launch_bounds__(256) void adamw_moments_kernel(const ParamJobs T, const Moments W, const AdamWStep* step,
                                                            const AdamWRates R) {
    const ParamJob& J = job_of(T, blockIdx.x);
    const uint32_t base = (blockIdx.x - J.chunk0) * CHUNK;
    auto run = [&](auto t) {
        using E = decltype(t);
        if (base + CHUNK <= J.n) adamw_chunk<E, BITS, CHUNK, Way<true, STREAM, EXACT>>(J, base, W, step, R);
        else adamw_chunk<E, BITS, CHUNK, Way<false, STREAM, EXACT>>(J, base, W, step, R);
    };
    if (J.dtype == TYPE_F32) run(float());
    else if (J.dtype == TYPE_BF16) run(bf16());
    else run(f16());
}

// Four elements from `at` on of one of the moments (blockIdx.y) per lane, nothing of it left in the caches: bound by HBM's writes.  In 32 bits the
// codes' bits, moved under a float's exponent field, are the values times 2^-120 and 2^-97.
constexpr int VALUES_CHUNK = 256 * 4;
__global__ __launch_bounds__(256) void moment_values_kernel(const Moments W, uint64_t at, uint64_t size, float* m, float* v) {
    typedef float f4 __attribute__((ext_vector_type(4)));
    const bool first = blockIdx.y == 0;
    const uint64_t e = at + (uint64_t)blockIdx.x * VALUES_CHUNK + threadIdx.x * 4;
    if (e >= size) return;
    const uint8_t* const codes = reinterpret_cast<const uint8_t*>(first ? W.m : W.v) + e;
    float* const out = (first ? m : v) + e;
    const uint32_t n = size - e < 4 ? (uint32_t)(size - e) : 4u;
    uint32_t w[1];
    if (n == 4) w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(codes));
    else load_codes<Way<false, false>, 4>(w, codes, 0, n);
    const int scale = (first ? 120 - 127 : 97 - 127) + (int)(first ? W.m_scale : W.v_scale)[e / MOMENT_BLOCK];
    const uint32_t field = first ? 127u : 255u, none = first ? 0x7fc00000u : 0x7f800000u, sign = first ? 0x80000000u : 0u;
    float a[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t c = w[0] >> 8 * j & field;
        const uint32_t bits = c == field ? none : (uint32_t)__float_as_int(ldexpf(__int_as_float((int)(c << 20)), scale));
        a[j] = __int_as_float((int)(bits | (w[0] << (24 - 8 * j) & sign)));
    }
    if (n == 4 && ((uintptr_t)out & 15) == 0) __builtin_nontemporal_store(f4{a[0], a[1], a[2], a[3]}, reinterpret_cast<f4*>(out));
    else store_elements<Way<false, false>>(out, a, 0, n);
}

// ------------------------------------------------------------------------------------------------- norm of the gradients

template <typename T, int CHUNK, bool STREAM>
__device__ __forceinline__ double square_sum(const ParamJob& J, uint32_t base) {
    constexpr int E = 16 / (int)sizeof(T), TURNS = CHUNK / (256 * E);
    T g[TURNS][E];
#pragma unroll
    for (int k = 0; k < TURNS; k++)
        load_elements<Way<false, STREAM>>(g[k], reinterpret_cast<const T*>(J.g), base + (k * 256 + threadIdx.x) * E, J.n);
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < TURNS; k++)
#pragma unroll
        for (int j = 0; j < E; j++) {
            const double x = (double)to_float(g[k][j]);
            s = fma(x, x, s);
        }
    return s;
}

// STREAM: gradients that the last cache does not hold until the update reads them again go past it; 134 M float32 gradients, norm and
// update 511 -> 460 us, 34 M (128 MiB) 120 -> 121, 34 M bfloat16 87 -> 91.
template <int CHUNK, bool STREAM>
__global__ __launch_bounds__(256) void grad_square_kernel(const ParamJobs T, double* partial) {
    double s = 0.0;
    for (uint32_t c = blockIdx.x; c < T.chunks; c += gridDim.x) {
        const ParamJob& J = job_of(T, c);
        const uint32_t base = (c - J.chunk0) * CHUNK;
        s += J.dtype == TYPE_F32 ? square_sum<float, CHUNK, STREAM>(J, base)
             : J.dtype == TYPE_BF16 ? square_sum<bf16, CHUNK, STREAM>(J, base) : square_sum<f16, CHUNK, STREAM>(J, base);
    }
    s = block_sum(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

}  // namespace cfh
