// Residual stream and block output joined and normed: h = s_x x + s_f gate N_b(f), y = N(h), and the backward pass
//     u = gy w;  dh = gh + r (u - [mean u] - xhat mean(u xhat))      ([.]: layer norm only; r: one over the deviation)
//     dx = s_x dh;  da = s_f gate dh;  dgate = sum s_f a dh;  df = N_b's backward of da;  dw = sum gy xhat;  db = sum gy
//
// Both passes are bound by HBM: some 20 operations per element and way against 2 to 4 bytes for each of 3 to 7 arrays.  A row
// is held in the registers of a team of 16, 64, 256 or 1024 lanes, 16 bytes of each array per lane and turn, so that every
// array is read once and the statistics (mean first, then the squares of what is left) need no second pass over memory.
// Rows need not be aligned to more than their elements: gfx950 takes 16-byte accesses at any address.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "element_types.hpp"
#include "residual_norm_args.hpp"
#include "wave_reduce.hpp"

namespace cfh {

template <typename T>
struct Vec {
    static constexpr int N = 16 / (int)sizeof(T);
    T e[N];
};

// Sum over the LANES lanes of a team; every lane gets it.  Teams of more than a wavefront are whole workgroups; two halves of `part`
// in turn, so that one barrier per sum is enough.
template <int LANES>
struct TeamSum {
    float* part;
    int phase = 0;
    __device__ __forceinline__ explicit TeamSum(float* p) : part(p) {}
    static constexpr int WAVES = LANES > 64 ? LANES / 64 : 1;
    static constexpr int WORDS = LANES > 64 ? 4 * WAVES : 1;
    __device__ __forceinline__ void operator()(float& a, float& b) {
        if constexpr (LANES == 16) { a = row_sum(a); b = row_sum(b); return; }
        a = wave_sum(a);
        b = wave_sum(b);
        if constexpr (LANES > 64) {
            float* const p = part + phase * 2 * WAVES;
            phase ^= 1;
            if ((threadIdx.x & 63) == 0) { p[threadIdx.x >> 6] = a; p[WAVES + (threadIdx.x >> 6)] = b; }
            __syncthreads();
            a = 0.0f;
            b = 0.0f;
            for (int k = 0; k < WAVES; k++) { a += p[k]; b += p[WAVES + k]; }
        }
    }
    __device__ __forceinline__ float operator()(float a) {
        if constexpr (LANES == 16) return row_sum(a);
        a = wave_sum(a);
        if constexpr (LANES > 64) {
            float* const p = part + phase * 2 * WAVES;
            phase ^= 1;
            if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = a;
            __syncthreads();
            a = 0.0f;
            for (int k = 0; k < WAVES; k++) a += p[k];
        }
        return a;
    }
};

// A lane's part of a row: VPT pieces of 16 bytes, LANES * 16 bytes apart.
template <typename T, int LANES, int VPT>
struct Share {
    static constexpr int E = Vec<T>::N, N = VPT * E, CAP = LANES * N;
    struct Raw { Vec<T> v[VPT]; };
    int lane, dim;
    __device__ __forceinline__ int col(int k) const { return (k * LANES + lane) * E; }
    __device__ __forceinline__ bool live(int i) const { return col(i / E) + i % E < dim; }
    __device__ __forceinline__ void load(Raw& r, const T* row) const {
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            const int c = col(k);
            if (c + E <= dim) __builtin_memcpy(&r.v[k], row + c, 16);
            else {
#pragma unroll
                for (int j = 0; j < E; j++) r.v[k].e[j] = c + j < dim ? row[c + j] : (T)0.0f;
            }
        }
    }
    // weights: of the type of the rows or float32; `none` where there are none, 0 behind the last
    __device__ __forceinline__ void weights(float (&o)[N], const void* w, bool f32, float none) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int c = col(i / E) + i % E;
            o[i] = c >= dim ? 0.0f : !w ? none : f32 ? reinterpret_cast<const float*>(w)[c] : to_float(reinterpret_cast<const T*>(w)[c]);
        }
    }
    __device__ __forceinline__ void store(T* row, const float (&o)[N]) const {
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            const int c = col(k);
            Vec<T> v;
#pragma unroll
            for (int j = 0; j < E; j++) v.e[j] = from_float<T>(o[k * E + j]);
            if (c + E <= dim) __builtin_memcpy(row + c, &v, 16);
            else {
#pragma unroll
                for (int j = 0; j < E; j++)
                    if (c + j < dim) row[c + j] = v.e[j];
            }
        }
    }
    __device__ __forceinline__ static float at(const Raw& r, int i) { return to_float(r.v[i / E].e[i % E]); }
};

// Mean (layer norm; else 0) and one over the deviation of a team's row.
template <int LANES, typename S>
__device__ __forceinline__ void row_stats(const S& sh, const float (&v)[S::N], int kind, float eps, TeamSum<LANES>& sum, float& mean, float& r) {
    const float inv = 1.0f / (float)sh.dim;
    mean = 0.0f;
    float s = 0.0f;
    if (kind == 1) {
#pragma unroll
        for (int i = 0; i < S::N; i++) s += v[i];
        mean = sum(s) * inv;
    }
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < S::N; i++) {
        const float d = sh.live(i) ? v[i] - mean : 0.0f;
        s = fmaf(d, d, s);
    }
    r = 1.0f / sqrtf(sum(s) * inv + eps);
}

template <typename T, int LANES, int VPT, bool BN>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void residual_norm_forward_kernel(const ResidualNorm A, T* h_out, T* y_out,
                                                                                          float* stats) {
    using S = Share<T, LANES, VPT>;
    constexpr int N = S::N, TEAMS = LANES > 256 ? 1 : 256 / LANES;
    __shared__ float part[TeamSum<LANES>::WORDS];
    TeamSum<LANES> sum(part);
    const S sh{(int)threadIdx.x % LANES, A.dim};
    float w[N], b[N], wf[BN ? N : 1], bf[BN ? N : 1];
    if (y_out) {
        sh.weights(w, A.w, A.w_float, 1.0f);
        sh.weights(b, A.b, A.w_float, 0.0f);
    }
    if constexpr (BN) {
        sh.weights(wf, A.wf, A.w_float, 1.0f);
        sh.weights(bf, A.bf, A.w_float, 0.0f);
    }
    for (int64_t row = (int64_t)blockIdx.x * TEAMS + threadIdx.x / LANES; row < A.rows; row += (int64_t)gridDim.x * TEAMS) {
        typename S::Raw rx, rf, rg;
        sh.load(rx, reinterpret_cast<const T*>(A.x) + row * A.xs);
        if (A.f) sh.load(rf, reinterpret_cast<const T*>(A.f) + row * A.fs);
        if (A.gate) sh.load(rg, reinterpret_cast<const T*>(A.gate) + row / A.gate_span * A.dim);
        float h[N], st[4] = {0.0f, 1.0f, 0.0f, 1.0f};
        if (A.f) {
#pragma unroll
            for (int i = 0; i < N; i++) h[i] = S::at(rf, i);
            if constexpr (BN) {
                row_stats<LANES, S>(sh, h, A.block_norm, A.block_eps, sum, st[0], st[1]);
#pragma unroll
                for (int i = 0; i < N; i++) h[i] = fmaf((h[i] - st[0]) * st[1], wf[i], bf[i]);
            }
            if (A.gate) {
#pragma unroll
                for (int i = 0; i < N; i++) h[i] *= S::at(rg, i);
            }
#pragma unroll
            for (int i = 0; i < N; i++) h[i] = fmaf(A.sf, h[i], A.in_scale * S::at(rx, i));
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) h[i] = A.in_scale * S::at(rx, i);
        }
        if (h_out) sh.store(h_out + row * A.dim, h);
        if (A.norm) {
            row_stats<LANES, S>(sh, h, A.norm, A.eps, sum, st[2], st[3]);
            if (y_out) {
#pragma unroll
                for (int i = 0; i < N; i++) h[i] = fmaf((h[i] - st[2]) * st[3], w[i], b[i]);
                sh.store(y_out + row * A.dim, h);
            }
        }
        if (stats && sh.lane == 0) *reinterpret_cast<float4*>(stats + 4 * row) = make_float4(st[0], st[1], st[2], st[3]);
    }
}

// Sums over rows are kept per lane, for its columns, while a workgroup goes through its strips, then added over its teams and
// written down per workgroup (or strip, for the gate); a second launch adds these in a fixed order.
// GATE: 0 none, 1 a row for several rows (its gradient is a column sum), 2 one for each row.
template <typename T, int LANES, int VPT, bool BN, int GATE>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void residual_norm_backward_kernel(const ResidualNorm A, const NormGrads G) {
    using S = Share<T, LANES, VPT>;
    constexpr int N = S::N, TEAMS = LANES > 256 ? 1 : 256 / LANES;
    __shared__ float part[TeamSum<LANES>::WORDS];
    __shared__ float cols[TEAMS > 1 ? TEAMS * S::CAP : 1];
    TeamSum<LANES> sum(part);
    const int team = (int)threadIdx.x / LANES;
    const S sh{(int)threadIdx.x % LANES, A.dim};
    const T* const gh = reinterpret_cast<const T*>(G.gh);
    const T* const gy = reinterpret_cast<const T*>(G.gy);
    const float inv = 1.0f / (float)A.dim;
    float w[N], wf[BN ? N : 1], bf[BN ? N : 1], g[GATE ? N : 1];
    float dw[N], db[N], dwf[BN ? N : 1], dbf[BN ? N : 1], dg[GATE == 1 ? N : 1];
    sh.weights(w, A.w, A.w_float, 1.0f);
    if constexpr (BN) {
        sh.weights(wf, A.wf, A.w_float, 1.0f);
        sh.weights(bf, A.bf, A.w_float, 0.0f);
#pragma unroll
        for (int i = 0; i < N; i++) dwf[i] = dbf[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < N; i++) dw[i] = db[i] = 0.0f;

    // the workgroup's sum of a column each: to float32 `sums`, or (NULL) rounded to `out`
    auto flush = [&](const float (&acc)[N], float* sums, void* out, bool f32) {
        auto put = [&](int c, float v) {
            if (sums) sums[c] = v;
            else if (f32) reinterpret_cast<float*>(out)[c] = v;
            else reinterpret_cast<T*>(out)[c] = from_float<T>(v);
        };
        if (!sums && !out) return;
        if constexpr (TEAMS == 1) {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (sh.live(i)) put(sh.col(i / S::E) + i % S::E, acc[i]);
        } else {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; i++) cols[team * S::CAP + sh.col(i / S::E) + i % S::E] = acc[i];
            __syncthreads();
            for (int c = threadIdx.x; c < A.dim; c += 256) {
                float s = 0.0f;
                for (int t = 0; t < TEAMS; t++) s += cols[t * S::CAP + c];
                put(c, s);
            }
        }
    };

    const int64_t span = GATE == 1 ? A.gate_span : A.rows;
    for (int64_t strip = blockIdx.x; strip < G.strips; strip += gridDim.x) {
        const int64_t segment = strip / G.parts, sub = strip - segment * G.parts;
        const int64_t row0 = segment * span + span * sub / G.parts, row1 = segment * span + span * (sub + 1) / G.parts;
        if constexpr (GATE == 1) {
            typename S::Raw rg;
            sh.load(rg, reinterpret_cast<const T*>(A.gate) + segment * A.dim);
#pragma unroll
            for (int i = 0; i < N; i++) { g[i] = S::at(rg, i); dg[i] = 0.0f; }
        }
        for (int64_t row = row0 + team; row < row1; row += TEAMS) {
            typename S::Raw rx, rf, rg, rgh, rgy;
            sh.load(rx, reinterpret_cast<const T*>(A.x) + row * A.xs);
            if (A.f) sh.load(rf, reinterpret_cast<const T*>(A.f) + row * A.fs);
            if constexpr (GATE == 2) sh.load(rg, reinterpret_cast<const T*>(A.gate) + row * A.dim);
            if (gh) sh.load(rgh, gh + row * A.dim);
            if (gy) sh.load(rgy, gy + row * A.dim);
            const float4 st = *reinterpret_cast<const float4*>(G.stats + 4 * row);
            if constexpr (GATE == 2) {
#pragma unroll
                for (int i = 0; i < N; i++) g[i] = S::at(rg, i);
            }
            float a[BN || GATE ? N : 1], dh[N];
            if constexpr (BN || GATE) {
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const float f = S::at(rf, i);
                    a[i] = BN ? (f - st.x) * st.y : f;          // with a norm of the block: before its weight
                }
            }
            auto block_out = [&](int i) { return BN ? fmaf(a[i], wf[i], bf[i]) : a[i]; };
#pragma unroll
            for (int i = 0; i < N; i++) dh[i] = gh ? S::at(rgh, i) : 0.0f;
            if (gy) {
                float s = 0.0f, t = 0.0f, xhat[N];
#pragma unroll
                for (int i = 0; i < N; i++) {
                    float v = A.in_scale * S::at(rx, i);
                    if constexpr (BN || GATE) v = fmaf(A.sf, GATE ? g[i] * block_out(i) : block_out(i), v);
                    else if (A.f) v = fmaf(A.sf, S::at(rf, i), v);
                    xhat[i] = (v - st.z) * st.w;
                    const float e = S::at(rgy, i), u = e * w[i];
                    s += u;
                    t = fmaf(u, xhat[i], t);
                    dw[i] = fmaf(e, xhat[i], dw[i]);
                    db[i] += e;
                }
                sum(s, t);
                s = A.norm == 1 ? s * inv : 0.0f;
                t *= inv;
#pragma unroll
                for (int i = 0; i < N; i++) dh[i] = fmaf(st.w, S::at(rgy, i) * w[i] - s - xhat[i] * t, dh[i]);
            }
            float o[N];
            if (G.dx) {
#pragma unroll
                for (int i = 0; i < N; i++) o[i] = A.sx * dh[i];
                sh.store(reinterpret_cast<T*>(G.dx) + row * A.dim, o);
            }
            if constexpr (GATE == 1) {
#pragma unroll
                for (int i = 0; i < N; i++) dg[i] = fmaf(A.sf * block_out(i), dh[i], dg[i]);
            }
            if constexpr (GATE == 2) {
                if (G.dgate) {
#pragma unroll
                    for (int i = 0; i < N; i++) o[i] = A.sf * block_out(i) * dh[i];
                    sh.store(reinterpret_cast<T*>(G.dgate) + row * A.dim, o);
                }
            }
#pragma unroll
            for (int i = 0; i < N; i++) dh[i] *= GATE ? A.sf * g[i] : A.sf;
            if constexpr (BN) {
                float s = 0.0f, t = 0.0f;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const float u = dh[i] * wf[i];
                    s += u;
                    t = fmaf(u, a[i], t);
                    dwf[i] = fmaf(dh[i], a[i], dwf[i]);
                    dbf[i] += dh[i];
                }
                sum(s, t);
                s = A.block_norm == 1 ? s * inv : 0.0f;
                t *= inv;
#pragma unroll
                for (int i = 0; i < N; i++) dh[i] = st.y * (dh[i] * wf[i] - s - a[i] * t);
            }
            if (G.df) sh.store(reinterpret_cast<T*>(G.df) + row * A.dim, dh);
        }
        if constexpr (GATE == 1)
            flush(dg, G.gate_column ? G.gate_column + strip * A.dim : nullptr,
                  G.dgate ? reinterpret_cast<T*>(G.dgate) + segment * A.dim : nullptr, false);
    }
    auto column = [&](int k) { return G.column ? G.column + ((int64_t)k * gridDim.x + blockIdx.x) * A.dim : nullptr; };
    if (G.dw) flush(dw, column(0), G.dw, A.w_float);
    if (G.db) flush(db, column(1), G.db, A.w_float);
    if constexpr (BN) {
        if (G.dwf) flush(dwf, column(2), G.dwf, A.w_float);
        if (G.dbf) flush(dbf, column(3), G.dbf, A.w_float);
    }
}

// Adds the `count` rows of a column sum: blockIdx.y 0 to 3 dw, db, dwf, dbf (count: the workgroups of the launch before), 4 on: rows of
// the gate (count: parts).  16 columns per workgroup, 16 lanes for each.
template <typename T>
__global__ __launch_bounds__(256) void residual_norm_columns_kernel(const NormGrads G, int dim, int blocks, int w_float) {
    __shared__ float part[16][16];
    const int k = (int)blockIdx.y, c = (int)blockIdx.x * 16 + (threadIdx.x & 15), lane = threadIdx.x >> 4;
    void* const out = k == 0 ? G.dw : k == 1 ? G.db : k == 2 ? G.dwf : k == 3 ? G.dbf : G.dgate;
    if (!out) return;
    const int64_t count = k < 4 ? blocks : G.parts;
    const float* const src = k < 4 ? G.column + (int64_t)k * blocks * dim : G.gate_column + (int64_t)(k - 4) * G.parts * dim;
    float s = 0.0f;
    if (c < dim)
        for (int64_t r = lane; r < count; r += 16) s += src[r * dim + c];
    part[lane][threadIdx.x & 15] = s;
    __syncthreads();
    if (lane == 0 && c < dim) {
        s = 0.0f;
        for (int t = 0; t < 16; t++) s += part[t][threadIdx.x];
        const int64_t o = k < 4 ? c : (int64_t)(k - 4) * dim + c;
        if (k < 4 && w_float) reinterpret_cast<float*>(out)[o] = s;
        else reinterpret_cast<T*>(out)[o] = from_float<T>(s);
    }
}

// ------------------------------------------------------------------------------------------------- launches
// Lanes of a team and pieces of 16 bytes per lane: the smallest that hold a row, up to 64 bytes of each array per lane.  16 lanes
// for short rows, so that a wavefront is not half idle; a wavefront while its registers hold the row (sums without a barrier).
template <typename T, typename F>
void with_share(int64_t dim, F f) {
    constexpr int E = Vec<T>::N;
    if (dim <= 16 * E) f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
    else if (dim <= 16 * E * 2) f(std::integral_constant<int, 16>(), std::integral_constant<int, 2>());
    else if (dim <= 64 * E) f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    else if (dim <= 64 * E * 2) f(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    else if (dim <= 256 * E) f(std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
    else if (dim <= 256 * E * 2) f(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
    else if (dim <= 256 * E * 4) f(std::integral_constant<int, 256>(), std::integral_constant<int, 4>());
    else if (dim <= 1024 * E * 2) f(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
    else if constexpr (1024 * E * 2 < NORM_MAX_DIM) f(std::integral_constant<int, 1024>(), std::integral_constant<int, 4>());
}

template <typename T>
void residual_norm_forward(const ResidualNorm& A, T* h, T* y, float* stats, hipStream_t st) {
    with_share<T>(A.dim, [&](auto lanes, auto vpt) {
        constexpr int L = decltype(lanes)::value, V = decltype(vpt)::value, TEAMS = L > 256 ? 1 : 256 / L, THREADS = L > 256 ? L : 256;
        const int64_t blocks = (A.rows + TEAMS - 1) / TEAMS, most = (int64_t)NORM_CUS * 8;
        const dim3 grid((unsigned)(blocks < most ? blocks : most));
        if (A.block_norm) hipLaunchKernelGGL((residual_norm_forward_kernel<T, L, V, true>), grid, dim3(THREADS), 0, st, A, h, y, stats);
        else hipLaunchKernelGGL((residual_norm_forward_kernel<T, L, V, false>), grid, dim3(THREADS), 0, st, A, h, y, stats);
    });
}

template <typename T>
void residual_norm_backward(const ResidualNorm& A, NormGrads G, int64_t gate_rows, float* scratch, hipStream_t st) {
    const NormPlan P = norm_plan(A.rows, A.dim, Vec<T>::N, gate_rows);
    G.column = P.column_floats ? scratch : nullptr;
    G.gate_column = P.gate_floats ? scratch + P.column_floats : nullptr;
    G.strips = P.strips;
    G.parts = P.parts;
    int blocks = P.blocks;
    if (A.rows > 0) {
        with_share<T>(A.dim, [&](auto lanes, auto vpt) {
            constexpr int L = decltype(lanes)::value, V = decltype(vpt)::value, THREADS = L > 256 ? L : 256;
            auto launch = [&](auto bn, auto gate) {
                hipLaunchKernelGGL((residual_norm_backward_kernel<T, L, V, decltype(bn)::value, decltype(gate)::value>), dim3((unsigned)blocks),
                                   dim3(THREADS), 0, st, A, G);
            };
            auto gated = [&](auto bn) {
                if (gate_rows == 0) launch(bn, std::integral_constant<int, 0>());
                else if (P.gate_rows_shared) launch(bn, std::integral_constant<int, 1>());
                else launch(bn, std::integral_constant<int, 2>());
            };
            if (A.block_norm) gated(std::true_type());
            else gated(std::false_type());
        });
    } else {
        blocks = 0;         // sums over no rows
        G.parts = 0;
    }
    const bool columns = (G.column || A.rows == 0) && (G.dw || G.db || G.dwf || G.dbf);
    const bool gates = G.dgate && (G.gate_column || A.rows == 0);
    if (columns || gates) {
        if (!columns) G.dw = G.db = G.dwf = G.dbf = nullptr;
        const int64_t y = 4 + (gates ? (A.rows == 0 ? gate_rows : P.segments) : 0);
        hipLaunchKernelGGL(residual_norm_columns_kernel<T>, dim3((unsigned)((A.dim + 15) / 16), (unsigned)y), dim3(256), 0, st, G, A.dim, blocks,
                           A.w_float);
    }
}

}  // namespace cfh
