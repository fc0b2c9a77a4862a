// AdamW over many tensors of several types with moments in 32 or in 8 bits, and the common norm of the gradients that it
// clips by.  The rule, the 8-bit formats and the hash are written down in crystalframer_hip.h.
//
// The tensors' addresses travel in the kernel arguments.  What all elements share (the step's bias corrections, its hash
// key, the clipping factor) is made by a launch of one wavefront before, which also advances the step.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "element_types.hpp"

namespace cfh {

constexpr int MOMENT_BLOCK = 64;          // elements that share a scale
constexpr int PARAM_MAX_JOBS = 88;        // tensors per launch (kernel arguments: 4 KB)
constexpr int ADAMW_CHUNK = 256;          // elements per workgroup of 256 threads
constexpr int GRAD_NORM_CHUNK = 4096;     // elements per turn of a workgroup of 256 threads
constexpr int GRAD_NORM_BLOCKS = 1024;    // workgroups per launch at most

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

__device__ __forceinline__ const ParamJob& job_of(const ParamJobs& T, uint32_t chunk) {
    int lo = 0, hi = T.njobs;            // job[lo].chunk0 <= chunk < job[hi].chunk0
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (T.job[mid].chunk0 <= chunk) lo = mid; else hi = mid;
    }
    return T.job[lo];
}

__global__ void adamw_begin_kernel(AdamWStep* out, unsigned long long* step, double lr, double beta1, double beta2, double wd,
                                   const float* clip) {
    const unsigned long long t = *step + 1ULL;
    *step = t;
    // 1 - beta^t by expm1: for beta close to 1 and the first steps the difference cancels
    const double bc1 = -expm1((double)t * log(beta1)), bc2 = -expm1((double)t * log(beta2));
    out->step_size = (float)(lr / bc1);
    out->inv_sqrt_bc2 = (float)(1.0 / sqrt(bc2));
    out->decay = (float)(1.0 - lr * wd);
    out->clip = clip ? clip[1] : 1.0f;
    uint32_t k = (uint32_t)t * 0x6A09E667u;
    k = (k ^ (k >> 15)) * 0x9E3779B1u;
    out->key = k ^ (k >> 16);
}

__device__ __forceinline__ uint32_t moment_hash(uint32_t element, uint32_t key) {
    uint32_t x = element * 0x9E3779B1u + key;
    x = (x ^ (x >> 16)) * 0xBB67AE85u;
    return x ^ (x >> 15);
}

__device__ __forceinline__ float adamw_update(float p, float m, float v, const AdamWStep& S, float eps) {
    return p * S.decay - S.step_size * (m / (sqrtf(v) * S.inv_sqrt_bc2 + eps));
}

// An 8-bit code without its sign is a double's exponent and mantissa cut to three bits: its bits, moved under the high word's
// exponent field, are the value times 2^bias, denormals included, and back it is one shift.  bias: 1016 (exp_avg, e4m3: the
// smallest normal value 2^-6 has exponent field 1) and 993 (exp_avg_sq: 2^-29).
constexpr int M_BIAS = 1016, V_BIAS = 993, M_TOP = 7, V_TOP = 0;

__device__ __forceinline__ double code_value(uint32_t code, int bias) {
    return ldexp(__hiloint2double((int)(code << 17), 0), bias);
}
// floor(x / step + (2 k + 1) / 2^17) as a code; x >= 0, k in 16 bits
__device__ __forceinline__ uint32_t code_of(double x, int bias, uint32_t k) {
    return ((uint32_t)__double2hiint(ldexp(x, -bias)) + 2u * k + 1u) >> 17;
}
__device__ __forceinline__ bool finite_double(double x) { return (__double2hiint(x) & 0x7ff00000) != 0x7ff00000; }

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

template <typename T, int BITS>
__device__ void adamw_chunk(const ParamJob& J, uint32_t base, const Moments& W, const AdamWStep& S, const AdamWRates& R) {
    const uint32_t i = base + threadIdx.x;
    const bool live = i < J.n;
    const uint64_t e = J.first + i;
    T* const p = reinterpret_cast<T*>(J.p) + i;
    const float g = live ? to_float(reinterpret_cast<const T*>(J.g)[i]) : 0.0f;
    if constexpr (BITS == 32) {
        if (!live) return;
        float* const pm = reinterpret_cast<float*>(W.m) + e;
        float* const pv = reinterpret_cast<float*>(W.v) + e;
        const float c = g * S.clip;
        const float m = (float)R.beta1 * *pm + (float)(1.0 - R.beta1) * c;
        const float v = (float)R.beta2 * *pv + (float)(1.0 - R.beta2) * c * c;
        *pm = m;
        *pv = v;
        *p = from_float<T>(adamw_update(to_float(*p), m, v, S, R.eps));
    } else {
        uint8_t* const pm = reinterpret_cast<uint8_t*>(W.m) + e;
        uint8_t* const pv = reinterpret_cast<uint8_t*>(W.v) + e;
        double m = 0.0, v = 0.0;
        if (live) {
            const uint32_t cm = *pm, cv = *pv;
            const double c = (double)g * (double)S.clip;
            m = code_value(cm & 127u, M_BIAS + (int)W.m_scale[e / MOMENT_BLOCK] - 127);
            if ((cm & 127u) == 127u) m = __longlong_as_double(0x7ff8000000000000LL);
            if (cm & 128u) m = -m;
            v = code_value(cv, V_BIAS + (int)W.v_scale[e / MOMENT_BLOCK] - 127);
            if (cv == 255u) v = __longlong_as_double(0x7ff0000000000000LL);
            m = moment_mix(R.beta1, m, (1.0 - R.beta1) * c);
            v = moment_mix(R.beta2, v, (1.0 - R.beta2) * c * c);
        }
        const bool fm = finite_double(m), fv = fabs(v) < 0x1p128;
        uint32_t hm = fm ? (uint32_t)__double2hiint(m) & 0x7fffffffu : 0u, hv = fv ? (uint32_t)__double2hiint(v) : 0u;
        for (int d = 1; d < 64; d *= 2) {
            hm = max(hm, (uint32_t)__shfl_xor((int)hm, d));
            hv = max(hv, (uint32_t)__shfl_xor((int)hv, d));
        }
        if (!live) return;
        const int sm = scale_byte(hm, M_TOP), sv = scale_byte(hv, V_TOP);
        const uint32_t h = moment_hash((uint32_t)e, S.key);
        uint32_t cm = fm ? code_of(fabs(m), M_BIAS + sm - 127, h & 0xffffu) : 127u;
        uint32_t cv = fv ? code_of(v, V_BIAS + sv - 127, h >> 16) : 255u;
        if (cv == 0u && v > 0.0) cv = 1u;
        *pm = (uint8_t)(cm | ((uint32_t)__double2hiint(m) >> 31 << 7));
        *pv = (uint8_t)cv;
        if (i % MOMENT_BLOCK == 0) {
            W.m_scale[e / MOMENT_BLOCK] = (uint8_t)sm;
            W.v_scale[e / MOMENT_BLOCK] = (uint8_t)sv;
        }
        *p = from_float<T>(adamw_update(to_float(*p), (float)m, (float)v, S, R.eps));
    }
}

template <int BITS>
__global__ __launch_bounds__(256) void adamw_moments_kernel(const ParamJobs T, const Moments W, const AdamWStep* step,
                                                            const AdamWRates R) {
    const ParamJob& J = job_of(T, blockIdx.x);
    const uint32_t base = (blockIdx.x - J.chunk0) * ADAMW_CHUNK;
    const AdamWStep S = *step;
    if (J.dtype == TYPE_F32) adamw_chunk<float, BITS>(J, base, W, S, R);
    else if (J.dtype == TYPE_BF16) adamw_chunk<bf16, BITS>(J, base, W, S, R);
    else adamw_chunk<f16, BITS>(J, base, W, S, R);
}

__global__ __launch_bounds__(256) void moment_values_kernel(const Moments W, uint64_t size, float* m, float* v) {
    const uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= size) return;
    const uint32_t cm = reinterpret_cast<const uint8_t*>(W.m)[e], cv = reinterpret_cast<const uint8_t*>(W.v)[e];
    const float a = (float)code_value(cm & 127u, M_BIAS + (int)W.m_scale[e / MOMENT_BLOCK] - 127);
    m[e] = copysignf((cm & 127u) == 127u ? __int_as_float(0x7fc00000) : a, cm & 128u ? -1.0f : 1.0f);
    v[e] = cv == 255u ? __int_as_float(0x7f800000) : (float)code_value(cv, V_BIAS + (int)W.v_scale[e / MOMENT_BLOCK] - 127);
}

// ------------------------------------------------------------------------------------------------- norm of the gradients
__device__ __forceinline__ double block_sum(double x) {
    __shared__ double part[4];
    for (int d = 32; d > 0; d /= 2) x += __shfl_xor(x, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    return part[0] + part[1] + part[2] + part[3];
}

template <typename T>
__device__ double square_sum(const ParamJob& J, uint32_t base) {
    const T* const g = reinterpret_cast<const T*>(J.g);
    double s = 0.0;
    for (uint32_t i = base + threadIdx.x; i < min(base + (uint32_t)GRAD_NORM_CHUNK, J.n); i += 256) {
        const double x = (double)to_float(g[i]);
        s = fma(x, x, s);
    }
    return s;
}

__global__ __launch_bounds__(256) void grad_norm_kernel(const ParamJobs T, double* partial) {
    double s = 0.0;
    for (uint32_t c = blockIdx.x; c < T.chunks; c += gridDim.x) {
        const ParamJob& J = job_of(T, c);
        const uint32_t base = (c - J.chunk0) * GRAD_NORM_CHUNK;
        s += J.dtype == TYPE_F32 ? square_sum<float>(J, base) : J.dtype == TYPE_BF16 ? square_sum<bf16>(J, base) : square_sum<f16>(J, base);
    }
    s = block_sum(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(256) void grad_norm_end_kernel(const double* partial, int count, double max_norm, float* out) {
    double s = 0.0;
    for (int i = threadIdx.x; i < count; i += 256) s += partial[i];
    s = sqrt(block_sum(s));
    if (threadIdx.x == 0) {
        const double c = max_norm / (s + 1e-6);
        out[0] = (float)s;
        out[1] = c >= 1.0 ? 1.0f : (float)c;
    }
}

}  // namespace cfh
