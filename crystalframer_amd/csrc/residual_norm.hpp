// Residual stream and block output joined and normed: h = s_x x + s_f gate N_b(f), y = N(h), and the backward pass
//     u = gy w;  dh = gh + r (u - [mean u] - xhat mean(u xhat))      ([.]: layer norm only; r: one over the deviation)
//     dx = s_x dh;  da = s_f gate dh;  dgate = sum s_f a dh;  df = N_b's backward of da;  dw = sum gy xhat;  db = sum gy
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "element_types.hpp"

namespace cfh {

constexpr int NORM_MAX_DIM = 16384;

struct ResidualNorm {
    const void *x, *f, *gate, *w, *b, *wf, *bf;
    int64_t rows, xs, fs, gate_span;      // gate_span: rows that share a row of the gate
    int32_t dim, norm, block_norm, w_float;
    float eps, block_eps, sx, sf;
    float in_scale;                       // of x where h is put together (1: x holds h)
};

__device__ __forceinline__ float block_sum4(float x, float* part) {
    for (int d = 32; d > 0; d /= 2) x += __shfl_xor(x, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    return part[0] + part[1] + part[2] + part[3];
}

template <typename T>
__device__ __forceinline__ float weight_at(const ResidualNorm& A, const void* w, int c, float none) {
    return !w ? none : A.w_float ? reinterpret_cast<const float*>(w)[c] : to_float(reinterpret_cast<const T*>(w)[c]);
}

template <typename T>
struct NormRow {
    const ResidualNorm& A;
    const T *x, *f, *gate;
    float mean_a = 0.0f, r_a = 1.0f, mean_h = 0.0f, r_h = 1.0f;
    __device__ NormRow(const ResidualNorm& A_, int64_t row) : A(A_) {
        x = reinterpret_cast<const T*>(A.x) + row * A.xs;
        f = A.f ? reinterpret_cast<const T*>(A.f) + row * A.fs : nullptr;
        gate = A.gate ? reinterpret_cast<const T*>(A.gate) + row / A.gate_span * A.dim : nullptr;
    }
    __device__ float ahat(int c) const { return (to_float(f[c]) - mean_a) * r_a; }
    __device__ float a(int c) const {
        if (!A.block_norm) return to_float(f[c]);
        return ahat(c) * weight_at<T>(A, A.wf, c, 1.0f) + weight_at<T>(A, A.bf, c, 0.0f);
    }
    __device__ float g(int c) const { return gate ? to_float(gate[c]) : 1.0f; }
    __device__ float h(int c) const {
        const float v = A.in_scale * to_float(x[c]);
        return f ? v + A.sf * (g(c) * a(c)) : v;
    }
    __device__ float hhat(int c) const { return (h(c) - mean_h) * r_h; }
};

template <typename T>
__global__ __launch_bounds__(256) void residual_norm_forward_kernel(const ResidualNorm A, T* h, T* y, float* stats) {
    __shared__ float part[4];
    const int64_t row = blockIdx.x;
    NormRow<T> R(A, row);
    const float inv = 1.0f / (float)A.dim;
    if (A.block_norm) {
        float s = 0.0f;
        if (A.block_norm == 1) {
            for (int c = threadIdx.x; c < A.dim; c += 256) s += to_float(R.f[c]);
            R.mean_a = block_sum4(s, part) * inv;
        }
        s = 0.0f;
        for (int c = threadIdx.x; c < A.dim; c += 256) { const float d = R.ahat(c); s = fmaf(d, d, s); }
        R.r_a = 1.0f / sqrtf(block_sum4(s, part) * inv + A.block_eps);
    }
    if (A.norm) {
        float s = 0.0f;
        if (A.norm == 1) {
            for (int c = threadIdx.x; c < A.dim; c += 256) s += R.h(c);
            R.mean_h = block_sum4(s, part) * inv;
        }
        s = 0.0f;
        for (int c = threadIdx.x; c < A.dim; c += 256) { const float d = R.hhat(c); s = fmaf(d, d, s); }
        R.r_h = 1.0f / sqrtf(block_sum4(s, part) * inv + A.eps);
    }
    for (int c = threadIdx.x; c < A.dim; c += 256) {
        if (h) h[row * A.dim + c] = from_float<T>(R.h(c));
        if (y) y[row * A.dim + c] = from_float<T>(R.hhat(c) * weight_at<T>(A, A.w, c, 1.0f) + weight_at<T>(A, A.b, c, 0.0f));
    }
    if (stats && threadIdx.x == 0) {
        stats[4 * row] = R.mean_a; stats[4 * row + 1] = R.r_a; stats[4 * row + 2] = R.mean_h; stats[4 * row + 3] = R.r_h;
    }
}

struct NormGrads {
    const float* stats;
    const void *gh, *gy;
    void *dx, *df, *dgate, *dw, *db, *dwf, *dbf;
    float* mid;              // (rows, 4): mean u, mean u xhat of N and of N_b
};

template <typename T>
struct NormGradRow : NormRow<T> {
    const T *gh, *gy;
    float u_h = 0.0f, ux_h = 0.0f, u_a = 0.0f, ux_a = 0.0f;
    __device__ NormGradRow(const ResidualNorm& A, const NormGrads& G, int64_t row) : NormRow<T>(A, row) {
        gh = G.gh ? reinterpret_cast<const T*>(G.gh) + row * A.dim : nullptr;
        gy = G.gy ? reinterpret_cast<const T*>(G.gy) + row * A.dim : nullptr;
        this->mean_a = G.stats[4 * row]; this->r_a = G.stats[4 * row + 1];
        this->mean_h = G.stats[4 * row + 2]; this->r_h = G.stats[4 * row + 3];
    }
    __device__ float uh(int c) const { return to_float(gy[c]) * weight_at<T>(this->A, this->A.w, c, 1.0f); }
    __device__ float dh(int c) const {
        float d = gh ? to_float(gh[c]) : 0.0f;
        if (gy) d += this->r_h * (uh(c) - u_h - this->hhat(c) * ux_h);
        return d;
    }
    __device__ float da(int c) const { return this->A.sf * this->g(c) * dh(c); }
    __device__ float ua(int c) const { return da(c) * weight_at<T>(this->A, this->A.wf, c, 1.0f); }
};

template <typename T>
__global__ __launch_bounds__(256) void residual_norm_row_grad_kernel(const ResidualNorm A, const NormGrads G) {
    __shared__ float part[4];
    const int64_t row = blockIdx.x;
    NormGradRow<T> R(A, G, row);
    const float inv = 1.0f / (float)A.dim;
    if (R.gy) {
        float s = 0.0f, t = 0.0f;
        for (int c = threadIdx.x; c < A.dim; c += 256) { const float u = R.uh(c); s += u; t = fmaf(u, R.hhat(c), t); }
        s = block_sum4(s, part) * inv;
        R.u_h = A.norm == 1 ? s : 0.0f;
        R.ux_h = block_sum4(t, part) * inv;
    }
    if (A.block_norm) {
        float s = 0.0f, t = 0.0f;
        for (int c = threadIdx.x; c < A.dim; c += 256) { const float u = R.ua(c); s += u; t = fmaf(u, R.ahat(c), t); }
        s = block_sum4(s, part) * inv;
        R.u_a = A.block_norm == 1 ? s : 0.0f;
        R.ux_a = block_sum4(t, part) * inv;
    }
    if (threadIdx.x == 0) {
        G.mid[4 * row] = R.u_h; G.mid[4 * row + 1] = R.ux_h; G.mid[4 * row + 2] = R.u_a; G.mid[4 * row + 3] = R.ux_a;
    }
    const int64_t o = row * A.dim;
    for (int c = threadIdx.x; c < A.dim; c += 256) {
        const float dh = R.dh(c);
        if (G.df) reinterpret_cast<T*>(G.df)[o + c] =
            from_float<T>(A.block_norm ? R.r_a * (R.ua(c) - R.u_a - R.ahat(c) * R.ux_a) : R.da(c));
        if (G.dgate && A.gate_span == 1) reinterpret_cast<T*>(G.dgate)[o + c] = from_float<T>(A.sf * R.a(c) * dh);
        if (G.dx) reinterpret_cast<T*>(G.dx)[o + c] = from_float<T>(A.sx * dh);
    }
}

// what: 0 dw, 1 db, 2 dwf, 3 dbf, 4 dgate of one row of the gate
template <typename T>
__device__ void column_grad(const ResidualNorm& A, const NormGrads& G, int what, int64_t row0, int64_t row1, void* out, int64_t o, bool f32) {
    __shared__ float part[4][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), lane = threadIdx.x >> 6;
    float s = 0.0f;
    if (c < A.dim)
        for (int64_t row = row0 + lane; row < row1; row += 4) {
            NormGradRow<T> R(A, G, row);
            R.u_h = G.mid[4 * row]; R.ux_h = G.mid[4 * row + 1];
            s += what == 0 ? to_float(R.gy[c]) * R.hhat(c) : what == 1 ? to_float(R.gy[c]) : what == 2 ? R.da(c) * R.ahat(c)
                 : what == 3 ? R.da(c) : A.sf * R.a(c) * R.dh(c);
        }
    part[lane][threadIdx.x & 63] = s;
    __syncthreads();
    if (lane == 0 && c < A.dim) {
        s = part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x];
        if (f32) reinterpret_cast<float*>(out)[o + c] = s;
        else reinterpret_cast<T*>(out)[o + c] = from_float<T>(s);
    }
    __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(256) void residual_norm_column_grad_kernel(const ResidualNorm A, const NormGrads G) {
    if (blockIdx.y > 0 || !G.dgate || A.gate_span == 1) {
        const int what = (int)blockIdx.y - 1;
        void* const out = what == 0 ? G.dw : what == 1 ? G.db : what == 2 ? G.dwf : G.dbf;
        if (what < 0 || !out) return;
        column_grad<T>(A, G, what, 0, G.gy || what > 1 ? A.rows : 0, out, 0, A.w_float);
    } else
        for (int64_t r = 0; r < A.rows; r += A.gate_span)
            column_grad<T>(A, G, 4, r, r + A.gate_span, G.dgate, r / A.gate_span * A.dim, false);
}

}  // namespace cfh
