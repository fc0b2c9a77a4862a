// Residual stream and block output joined and normed: h = s_x x + s_f gate N_b(f), y = N(h), and the backward pass
//     u = gy w;  dh = gh + r (u - [mean u] - xhat mean(u xhat))      ([.]: layer norm only; r: one over the deviation)
//     dx = s_x dh;  da = s_f gate dh;  dgate = sum s_f a dh;  df = N_b's backward of da;  dw = sum gy xhat;  db = sum gy
//
// Both passes are bound by HBM: some 20 operations per element and way against 2 to 4 bytes for each of 3 to 7 arrays.  A row
// is held in the registers of a team of lanes, from an eighth of a wavefront to 16 of them, 16 bytes of each array per lane, so that every
// array is read once and the statistics (mean first, then the squares of what is left) need no second pass over memory.
// Measured (bytes of the arrays that are read and written): forward 4096 x 5120 bfloat16, one norm, 34 us (4.9 TB/s); 524288 x 64
// 46 (5.9); 16384 x 1024 float32 42 (6.4); 16384 x 4096 bfloat16 with both norms and a gate 115 (4.7).  Backward 524288 x 64 74
// (5.4 TB/s); 16384 x 4096 with both norms and a gate 180 and 10 for the columns (4.2); 8190 x 2048, gate per channel, 37 and 8.
// 2372 x 128 float32, which the caches hold: 3 us forward, 6 and 3 backward.
// Rows need not be aligned to more than their elements: gfx950 takes 16-byte accesses at any address.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "element_types.hpp"
#include "residual_norm_args.hpp"
#include "wave_reduce.hpp"

namespace cfh {

template <typename T, int E>
struct Vec {
    T e[E];
};

// Sum over the lanes of a team; every lane gets it.  LANES 8, 16, 32 or 64: a part of a wavefront, in DPP and lane swaps; 0: the whole
// workgroup, through two halves of `part` in turn, so that one barrier per sum is enough.
template <int LANES>
struct TeamSum {
    static constexpr int MOST = 16;                     // wavefronts of a workgroup
    static constexpr int WORDS = LANES == 0 ? 4 * MOST : 1;
    float* part;
    int phase = 0;
    __device__ __forceinline__ explicit TeamSum(float* p) : part(p) {}
    __device__ __forceinline__ static float lanes(float a) {
        if constexpr (LANES == 8) return half_row_sum(a);
        if constexpr (LANES == 16) return row_sum(a);
        if constexpr (LANES == 32) {
            float p, q;
            swap16(row_sum(a), p, q);
            return p + q;
        }
        return wave_sum(a);
    }
    __device__ __forceinline__ void operator()(float& a, float& b) {
        a = lanes(a);
        b = lanes(b);
        if constexpr (LANES == 0) {
            float* const p = part + phase * 2 * MOST;
            phase ^= 1;
            const int waves = (int)blockDim.x >> 6;
            if ((threadIdx.x & 63) == 0) { p[threadIdx.x >> 6] = a; p[MOST + (threadIdx.x >> 6)] = b; }
            __syncthreads();
            a = 0.0f;
            b = 0.0f;
            for (int k = 0; k < waves; k++) { a += p[k]; b += p[MOST + k]; }
        }
    }
    __device__ __forceinline__ float operator()(float a) {
        a = lanes(a);
        if constexpr (LANES == 0) {
            float* const p = part + phase * 2 * MOST;
            phase ^= 1;
            const int waves = (int)blockDim.x >> 6;
            if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = a;
            __syncthreads();
            a = 0.0f;
            for (int k = 0; k < waves; k++) a += p[k];
        }
        return a;
    }
};

// A lane's part of a row: VPT pieces of E elements (16 bytes; one element where a row is shorter than that), a team's width apart.  TAIL: the pieces of a team reach over
// the row's end; else they are the row, and nothing has to be looked at.
template <typename T, int E_, int LANES, int VPT, bool TAIL>
struct Share {
    static constexpr int E = E_, BYTES = E * (int)sizeof(T), N = VPT * E, CAP = LANES * N, TEAMS = LANES ? 256 / LANES : 1;
    struct Raw { Vec<T, E> v[VPT]; };
    int lane, dim, width;
    __device__ __forceinline__ explicit Share(int dim_) : dim(dim_) {
        width = LANES ? LANES : (int)blockDim.x;
        lane = LANES ? (int)threadIdx.x % (LANES ? LANES : 1) : (int)threadIdx.x;
    }
    __device__ __forceinline__ static int team() { return LANES ? (int)threadIdx.x / (LANES ? LANES : 1) : 0; }
    __device__ __forceinline__ int col(int k) const { return (k * width + lane) * E; }
    __device__ __forceinline__ bool live(int i) const { return !TAIL || col(i / E) + i % E < dim; }
    // What lies behind the row's end is not read.  TAIL: a piece that reaches over it, or lies behind it, is read from the row's last E
    // elements and moved into place by trim(), so that no load waits behind a branch.
    __device__ __forceinline__ void load(Raw& r, const T* row) const {
#pragma unroll
        for (int k = 0; k < VPT; k++) __builtin_memcpy(&r.v[k], row + (TAIL ? min(col(k), dim - E) : col(k)), BYTES);
    }
    __device__ __forceinline__ void trim(Raw& r) const {
        if constexpr (!TAIL) return;
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            const int over = col(k) + E - dim;
            if (over > 0) {
                if constexpr (E == 1) r.v[k].e[0] = (T)0.0f;
                else {
                    uint64_t w[2];
                    __builtin_memcpy(w, &r.v[k], 16);
                    const int bits = over * 8 * (int)sizeof(T);
                    if (bits >= 64) {
                        w[0] = bits >= 128 ? 0 : w[1] >> (bits - 64);
                        w[1] = 0;
                    } else {
                        w[0] = w[0] >> bits | w[1] << (64 - bits);
                        w[1] >>= bits;
                    }
                    __builtin_memcpy(&r.v[k], w, 16);
                }
            }
        }
    }
    // weights: of the type of the rows or float32; `none` where there are none, 0 behind the last
    __device__ __forceinline__ void weights(float (&o)[N], const void* w, bool f32, float none) const {
        if (!w) {
#pragma unroll
            for (int i = 0; i < N; i++) o[i] = live(i) ? none : 0.0f;
            return;
        }
        if (sizeof(T) < 4 && !f32) {
            Raw r;
            load(r, reinterpret_cast<const T*>(w));
            trim(r);
#pragma unroll
            for (int i = 0; i < N; i++) o[i] = at(r, i);
            return;
        }
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            if (!TAIL) {
                __builtin_memcpy(o + k * E, reinterpret_cast<const float*>(w) + col(k), E * sizeof(float));
                continue;
            }
            __builtin_memcpy(o + k * E, reinterpret_cast<const float*>(w) + min(col(k), dim - E), E * sizeof(float));
            const int over = col(k) + E - dim;
            if (over > 0) {
#pragma unroll
                for (int d = E / 2; d > 0; d /= 2)
#pragma unroll
                    for (int j = 0; j < E; j++) {
                        const float v = j + d < E ? o[k * E + (j + d) % E] : 0.0f;
                        o[k * E + j] = over & d ? v : o[k * E + j];
                    }
                if (over >= E) {
#pragma unroll
                    for (int j = 0; j < E; j++) o[k * E + j] = 0.0f;
                }
            }
        }
    }
    __device__ __forceinline__ void store(T* row, const float (&o)[N]) const {
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            const int c = col(k);
            Vec<T, E> v;
#pragma unroll
            for (int j = 0; j < E; j++) v.e[j] = from_float<T>(o[k * E + j]);
            if (!TAIL || c + E <= dim) __builtin_memcpy(row + c, &v, BYTES);
            else if (TAIL) {
#pragma unroll
                for (int j = 0; j < E; j++)
                    if (c + j < dim) row[c + j] = v.e[j];
            }
        }
    }
    __device__ __forceinline__ static float at(const Raw& r, int i) { return to_float(r.v[i / E].e[i % E]); }
};

// Mean (layer norm; else 0) and one over the deviation of a team's row.  CENTRE: there may be layer norms.
template <bool CENTRE, int LANES, typename S>
__device__ __forceinline__ void row_stats(const S& sh, const float (&v)[S::N], int kind, float eps, TeamSum<LANES>& sum, float& mean, float& r) {
    const float inv = 1.0f / (float)sh.dim;
    mean = 0.0f;
    float s = 0.0f;
    if constexpr (!CENTRE) {
#pragma unroll
        for (int i = 0; i < S::N; i++) s = fmaf(v[i], v[i], s);          // (behind the row's end it is zero)
    } else {
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
    }
    r = 1.0f / sqrtf(sum(s) * inv + eps);
}

// GENERAL: some norm is a layer norm or has a bias; else root-mean-square norms with weights alone.
template <typename T, int E, int LANES, int VPT, bool TAIL, bool BN, bool GENERAL>
__global__ __launch_bounds__(LANES ? 256 : 1024) void residual_norm_forward_kernel(const ResidualNorm A, T* h_out, T* y_out,
                                                                                          float* stats) {
    using S = Share<T, E, LANES, VPT, TAIL>;
    constexpr int N = S::N, TEAMS = S::TEAMS;
    __shared__ float part[TeamSum<LANES>::WORDS];
    TeamSum<LANES> sum(part);
    const S sh(A.dim);
    float w[N], b[GENERAL ? N : 1], wf[BN ? N : 1], bf[BN && GENERAL ? N : 1];
    if (y_out) sh.weights(w, A.w, A.w_float, 1.0f);
    if constexpr (GENERAL) {
        if (y_out) sh.weights(b, A.b, A.w_float, 0.0f);
    }
    if constexpr (BN) sh.weights(wf, A.wf, A.w_float, 1.0f);
    if constexpr (BN && GENERAL) sh.weights(bf, A.bf, A.w_float, 0.0f);
    // The next row is on its way through the sums of this one, where there are registers for it (32768 x 1024 bfloat16, both norms: 51.1 ->
    // 47.2 us; 4096 x 16384, four pieces per lane: 142 -> 186).
    constexpr bool AHEAD = VPT == 1;
    typename S::Raw rx, rf, rg, nx, nf;
    auto fetch = [&](int64_t r) {
        sh.load(nx, reinterpret_cast<const T*>(A.x) + r * A.xs);
        if (A.f) sh.load(nf, reinterpret_cast<const T*>(A.f) + r * A.fs);
    };
    const int64_t row0 = (int64_t)blockIdx.x * TEAMS + S::team(), stride = (int64_t)gridDim.x * TEAMS;
    if (AHEAD && row0 < A.rows) fetch(row0);
    for (int64_t row = row0; row < A.rows; row += stride) {
        if (!AHEAD) fetch(row);
        rx = nx;
        if (A.f) rf = nf;
        if (AHEAD && row + stride < A.rows) fetch(row + stride);
        if (A.gate) sh.load(rg, reinterpret_cast<const T*>(A.gate) + row / A.gate_span * A.dim);
        sh.trim(rx);
        if (A.f) sh.trim(rf);
        if (A.gate) sh.trim(rg);
        float h[N], st[4] = {0.0f, 1.0f, 0.0f, 1.0f};
        if (A.f) {
#pragma unroll
            for (int i = 0; i < N; i++) h[i] = S::at(rf, i);
            if constexpr (BN) {
                row_stats<GENERAL, LANES, S>(sh, h, A.block_norm, A.block_eps, sum, st[0], st[1]);
#pragma unroll
                for (int i = 0; i < N; i++) h[i] = GENERAL ? fmaf((h[i] - st[0]) * st[1], wf[i], bf[i]) : h[i] * st[1] * wf[i];
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
            row_stats<GENERAL, LANES, S>(sh, h, A.norm, A.eps, sum, st[2], st[3]);
            if (y_out) {
#pragma unroll
                for (int i = 0; i < N; i++) h[i] = GENERAL ? fmaf((h[i] - st[2]) * st[3], w[i], b[i]) : h[i] * st[3] * w[i];
                sh.store(y_out + row * A.dim, h);
            }
        }
        if (stats && sh.lane == 0) *reinterpret_cast<float4*>(stats + 4 * row) = make_float4(st[0], st[1], st[2], st[3]);
    }
}

// Normed values before the weights, (v - mean) r.  v r - mean r rounds the mean in units of the deviation, 2^-24 of their ratio: float32 is
// centred first, as in the forward pass.  Values in 16 bits are whole multiples of 2^-8 (2^-11) of their size, which bounds that ratio by
// about 2^8 (2^11) for rows that are not all but constant: a rounding of 2^-16 (2^-13) beside the values' own (a large constant row
// plus a small one has a larger ratio, but then the sum's own rounding is as large), and they take one operation instead
// of two where registers are short (8192 x 8192 bfloat16, layer norms on both sides: both passes 326 us, centred 358).
template <bool GENERAL, typename T>
struct Normed {
    static constexpr bool CENTRED = GENERAL && sizeof(T) == 4;
    float mean, r, off;
    __device__ __forceinline__ Normed(float mean_, float r_) : mean(mean_), r(r_), off(-mean_ * r_) {}
    __device__ __forceinline__ float scaled(float v) const { return !GENERAL || CENTRED ? v * r : fmaf(v, r, off); }
    __device__ __forceinline__ float operator()(float v) const { return scaled(CENTRED ? v - mean : v); }
    // of s v + rest: begun with the first term, less the mean in float32, ended by scaled()
    __device__ __forceinline__ float begin(float s, float v) const { return CENTRED ? fmaf(s, v, -mean) : s * v; }
};

// Sums over rows are kept per lane, for its columns, while a workgroup goes through its strips, then added over its teams and
// written down per workgroup (or strip, for the gate); a second launch adds these in a fixed order.
// GATE: 0 none, 1 a row for several rows (its gradient is a column sum), 2 one for each row.
// GENERAL as above, or the gradient of a bias is wanted.  SUMS: else the column sums are the column kernel's, and the rows' means are left to it.
template <typename T, int E, int LANES, int VPT, bool TAIL, bool BN, int GATE, bool GENERAL, bool SUMS>
__global__ __launch_bounds__(LANES ? 256 : 1024) void residual_norm_backward_kernel(const ResidualNorm A, const NormGrads G) {
    using S = Share<T, E, LANES, VPT, TAIL>;
    constexpr int N = S::N, TEAMS = S::TEAMS;
    __shared__ float part[TeamSum<LANES>::WORDS];
    __shared__ float cols[TEAMS > 1 ? TEAMS * S::CAP : 1];
    TeamSum<LANES> sum(part);
    const int team = S::team();
    const S sh(A.dim);
    const T* const gh = reinterpret_cast<const T*>(G.gh);
    const T* const gy = reinterpret_cast<const T*>(G.gy);
    const float inv = 1.0f / (float)A.dim;
    constexpr bool SUM_B = SUMS && GENERAL, SUM_WF = SUMS && BN, SUM_BF = SUMS && BN && GENERAL, SUM_G = SUMS && GATE == 1;
    float dw[SUMS ? N : 1], db[SUM_B ? N : 1], dwf[SUM_WF ? N : 1], dbf[SUM_BF ? N : 1], dg[SUM_G ? N : 1];
#pragma unroll
    for (int i = 0; i < N; i++) {
        if constexpr (SUMS) dw[i] = 0.0f;
        if constexpr (SUM_B) db[i] = 0.0f;
        if constexpr (SUM_WF) dwf[i] = 0.0f;
        if constexpr (SUM_BF) dbf[i] = 0.0f;
    }

    // The weights (w, wf, bf) of rows with a piece per lane are kept in LDS, in quads of a piece a team's width apart, so that lanes that
    // read together read what lies together.  (Longer rows have no room there and read them from the caches.)
    constexpr bool HELD = VPT == 1;
    constexpr int QUAD = E < 4 ? E : 4;
    extern __shared__ float held[];
    auto place = [&](int k, int i) { return (k * N + i / QUAD * QUAD) * sh.width + sh.lane * QUAD + i % QUAD; };
    auto weights = [&](int k, float (&o)[N], const void* from, float none) {
        if constexpr (HELD) {
#pragma unroll
            for (int i = 0; i < N; i++) o[i] = held[place(k, i)];
        } else sh.weights(o, from, A.w_float, none);
    };
    // the workgroup's sum of a column each: to float32 `sums`, or (NULL) rounded to `out`
    auto flush = [&](const float (&acc)[N], float* sums, void* out, bool f32) {
        auto put = [&](int c, float v) {
            if (sums) sums[c] = v;
            else if (f32) reinterpret_cast<float*>(out)[c] = v;
            else reinterpret_cast<T*>(out)[c] = from_float<T>(v);
        };
        if constexpr (TEAMS == 1) {
#pragma unroll
            for (int k = 0; k < VPT; k++) {
                const int c = sh.col(k);
                if (sums && (!TAIL || c + E <= A.dim)) {
                    __builtin_memcpy(sums + c, acc + k * E, E * sizeof(float));
                    continue;
                }
#pragma unroll
                for (int j = 0; j < E; j++)
                    if (sh.live(k * E + j)) put(c + j, acc[k * E + j]);
            }
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
        typename S::Raw rg, rx, rf, rgh, rgy;
        if constexpr (GATE == 1) {
            sh.load(rg, reinterpret_cast<const T*>(A.gate) + segment * A.dim);
            sh.trim(rg);
        }
        if constexpr (SUM_G) {
#pragma unroll
            for (int i = 0; i < N; i++) dg[i] = 0.0f;
        }
        // The next row's pieces are asked for as soon as this row's are done with, so that they are on their way through its sums.
        auto fetch_x = [&](int64_t r) { sh.load(rx, reinterpret_cast<const T*>(A.x) + r * A.xs); };
        auto fetch_f = [&](int64_t r) { sh.load(rf, reinterpret_cast<const T*>(A.f) + r * A.fs); };
        auto fetch_gate = [&](int64_t r) { sh.load(rg, reinterpret_cast<const T*>(A.gate) + r * A.dim); };
        if (row0 + team < row1) {
            const int64_t row = row0 + team;
            if (gy) { fetch_x(row); sh.load(rgy, gy + row * A.dim); }
            if (A.f) fetch_f(row);
            if constexpr (GATE == 2) fetch_gate(row);
            if (gh) sh.load(rgh, gh + row * A.dim);
        }
        // (behind the first row's fetch: the two wait together)
        if constexpr (HELD) {
            if (strip == blockIdx.x) {
                if (team == 0) {
                    float o[N];
                    auto hold = [&](int k, const void* from, float none) {
                        sh.weights(o, from, A.w_float, none);
#pragma unroll
                        for (int i = 0; i < N; i++) held[place(k, i)] = o[i];
                    };
                    hold(0, A.w, 1.0f);
                    if constexpr (BN) hold(1, A.wf, 1.0f);
                    if constexpr (BN && GENERAL) hold(2, A.bf, 0.0f);
                }
                __syncthreads();
            }
        }
        for (int64_t row = row0 + team; row < row1; row += TEAMS) {
            const int64_t next = row + TEAMS;
            const bool more = next < row1;
            const float4 st = *reinterpret_cast<const float4*>(G.stats + 4 * row);
            if (gy) { sh.trim(rx); sh.trim(rgy); }
            if (A.f) sh.trim(rf);
            if constexpr (GATE == 2) sh.trim(rg);
            if (gh) sh.trim(rgh);
            // What the rows' own values give is computed again where it is needed a second time, and the weights are read again for every
            // row: kept in registers, they would halve the wavefronts.
            float wf[BN ? N : 1], bf[BN && GENERAL ? N : 1];
            if constexpr (BN) weights(1, wf, A.wf, 1.0f);
            if constexpr (BN && GENERAL) weights(2, bf, A.bf, 0.0f);
            auto gate = [&](int i) { return GATE ? S::at(rg, i) : 1.0f; };
            const Normed<GENERAL, T> of_a(st.x, st.y), of_h(st.z, st.w);
            auto ahat = [&](int i) { return of_a(S::at(rf, i)); };
            auto block_out = [&](int i) {
                if constexpr (BN && GENERAL) return fmaf(ahat(i), wf[i], bf[i]);
                else if constexpr (BN) return ahat(i) * wf[i];
                else return S::at(rf, i);
            };
            float dh[N];
            float4 mid = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (gy) {
                float w[N], xhat[N], s = 0.0f, t = 0.0f;
                weights(0, w, A.w, 1.0f);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    float v = of_h.begin(A.in_scale, S::at(rx, i));
                    if (BN || GATE || A.f) v = fmaf(A.sf, GATE ? gate(i) * block_out(i) : block_out(i), v);
                    xhat[i] = of_h.scaled(v);
                    const float e = S::at(rgy, i);
                    if constexpr (SUMS) dw[i] = fmaf(e, xhat[i], dw[i]);
                    if constexpr (SUM_B) db[i] += e;
                    dh[i] = e * w[i];
                    if constexpr (GENERAL) s += dh[i];
                    t = fmaf(dh[i], xhat[i], t);
                }
                if (more) {
                    fetch_x(next);
                    sh.load(rgy, gy + next * A.dim);
                }
                if constexpr (GENERAL) {
                    sum(s, t);
                    s = A.norm == 1 ? s * inv : 0.0f;
                } else t = sum(t);
                t *= inv;
                mid.x = s;
                mid.y = t;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const float v = fmaf(-xhat[i], t, GENERAL ? dh[i] - s : dh[i]);
                    dh[i] = gh ? fmaf(st.w, v, S::at(rgh, i)) : st.w * v;
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) dh[i] = gh ? S::at(rgh, i) : 0.0f;
            }
            if (gh && more) sh.load(rgh, gh + next * A.dim);
            if (G.dx) {
                float o[N];
#pragma unroll
                for (int i = 0; i < N; i++) o[i] = A.sx * dh[i];
                sh.store(reinterpret_cast<T*>(G.dx) + row * A.dim, o);
            }
            if constexpr (SUM_G) {
#pragma unroll
                for (int i = 0; i < N; i++) dg[i] = fmaf(A.sf * block_out(i), dh[i], dg[i]);
            }
            if constexpr (GATE == 2) {
                if (G.dgate) {
                    float o[N];
#pragma unroll
                    for (int i = 0; i < N; i++) o[i] = A.sf * block_out(i) * dh[i];
                    sh.store(reinterpret_cast<T*>(G.dgate) + row * A.dim, o);
                }
            }
#pragma unroll
            for (int i = 0; i < N; i++) dh[i] *= GATE ? A.sf * gate(i) : A.sf;
            if constexpr (GATE == 2) {
                if (more) fetch_gate(next);
            }
            if constexpr (BN) {
                float s = 0.0f, t = 0.0f;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const float u = dh[i] * wf[i], v = ahat(i);
                    if constexpr (GENERAL) s += u;
                    t = fmaf(u, v, t);
                    if constexpr (SUM_WF) dwf[i] = fmaf(dh[i], v, dwf[i]);
                    if constexpr (SUM_BF) dbf[i] += dh[i];
                }
                if constexpr (GENERAL) {
                    sum(s, t);
                    s = A.block_norm == 1 ? s * inv : 0.0f;
                } else t = sum(t);
                t *= inv;
                mid.z = s;
                mid.w = t;
#pragma unroll
                for (int i = 0; i < N; i++) dh[i] = st.y * fmaf(dh[i], wf[i], fmaf(-ahat(i), t, -s));
            }
            if constexpr (!SUMS) {
                if (sh.lane == 0) *reinterpret_cast<float4*>(G.mid + 4 * row) = mid;
            }
            if (A.f && more) fetch_f(next);
            if (G.df) sh.store(reinterpret_cast<T*>(G.df) + row * A.dim, dh);
        }
        if constexpr (SUM_G) {
            if (G.dgate) flush(dg, G.gate_column ? G.gate_column + strip * A.dim : nullptr, reinterpret_cast<T*>(G.dgate) + segment * A.dim, false);
        }
    }
    auto column = [&](int k) { return G.column ? G.column + ((int64_t)k * gridDim.x + blockIdx.x) * A.dim : nullptr; };
    if constexpr (SUMS) {
        if (G.dw) flush(dw, column(0), G.dw, A.w_float);
    }
    if constexpr (SUM_B) {
        if (G.db) flush(db, column(1), G.db, A.w_float);
    }
    if constexpr (SUM_WF) {
        if (G.dwf) flush(dwf, column(2), G.dwf, A.w_float);
    }
    if constexpr (SUM_BF) {
        if (G.dbf) flush(dbf, column(3), G.dbf, A.w_float);
    }
}

// The column sums alone, with the rows' means known (4096 x 16384 bfloat16, layer norms on both sides, gate per element: the rows 336 us,
// the columns 132 for 0.7 GB, 5.1 TB/s): a lane goes down the rows of its strip with a piece of 16 bytes of each array, four
// wavefronts of a workgroup over the same columns.  Nothing is exchanged before the end.
template <typename T, bool TAIL, bool BN, int GATE, bool GENERAL>
__global__ __launch_bounds__(256) void residual_norm_column_kernel(const ResidualNorm A, const NormGrads G) {
    constexpr int E = 16 / (int)sizeof(T), N = E, WIDE = 64 * E;
    using S = Share<T, E, 64, 1, TAIL>;
    __shared__ float cols[4][WIDE];
    S sh(A.dim);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), c0 = (int)blockIdx.x * WIDE;
    sh.lane += (int)blockIdx.x * 64;
    const T* const gh = reinterpret_cast<const T*>(G.gh);
    const T* const gy = reinterpret_cast<const T*>(G.gy);
    float w[N], wf[BN ? N : 1], bf[BN && GENERAL ? N : 1];
    sh.weights(w, A.w, A.w_float, 1.0f);
    if constexpr (BN) sh.weights(wf, A.wf, A.w_float, 1.0f);
    if constexpr (BN && GENERAL) sh.weights(bf, A.bf, A.w_float, 0.0f);
    float dw[N], db[GENERAL ? N : 1], dwf[BN ? N : 1], dbf[BN && GENERAL ? N : 1], dg[GATE == 1 ? N : 1];
#pragma unroll
    for (int i = 0; i < N; i++) {
        dw[i] = 0.0f;
        if constexpr (GENERAL) db[i] = 0.0f;
        if constexpr (BN) dwf[i] = 0.0f;
        if constexpr (BN && GENERAL) dbf[i] = 0.0f;
    }
    auto flush = [&](const float (&acc)[N], float* sums, void* out, bool f32) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) cols[wave][sh.col(0) - c0 + i] = acc[i];
        __syncthreads();
        for (int c = threadIdx.x; c < min(WIDE, A.dim - c0); c += 256) {
            const float s = cols[0][c] + cols[1][c] + cols[2][c] + cols[3][c];
            if (sums) sums[c0 + c] = s;
            else if (f32) reinterpret_cast<float*>(out)[c0 + c] = s;
            else reinterpret_cast<T*>(out)[c0 + c] = from_float<T>(s);
        }
    };
    const int64_t span = GATE == 1 ? A.gate_span : A.rows;
    for (int64_t strip = blockIdx.y; strip < G.strips; strip += gridDim.y) {
        const int64_t segment = strip / G.parts, sub = strip - segment * G.parts;
        const int64_t row0 = segment * span + span * sub / G.parts, row1 = segment * span + span * (sub + 1) / G.parts;
        typename S::Raw rx, rf, rg, rgh, rgy;
        if constexpr (GATE == 1) {
            sh.load(rg, reinterpret_cast<const T*>(A.gate) + segment * A.dim);
            sh.trim(rg);
#pragma unroll
            for (int i = 0; i < N; i++) dg[i] = 0.0f;
        }
        for (int64_t row = row0 + wave; row < row1; row += 4) {
            if (gy) {
                sh.load(rx, reinterpret_cast<const T*>(A.x) + row * A.xs);
                sh.load(rgy, gy + row * A.dim);
            }
            if (A.f) sh.load(rf, reinterpret_cast<const T*>(A.f) + row * A.fs);
            if constexpr (GATE == 2) sh.load(rg, reinterpret_cast<const T*>(A.gate) + row * A.dim);
            if (gh) sh.load(rgh, gh + row * A.dim);
            const float4 st = *reinterpret_cast<const float4*>(G.stats + 4 * row);
            const float4 mid = *reinterpret_cast<const float4*>(G.mid + 4 * row);
            if (gy) { sh.trim(rx); sh.trim(rgy); }
            if (A.f) sh.trim(rf);
            if constexpr (GATE == 2) sh.trim(rg);
            if (gh) sh.trim(rgh);
            const Normed<GENERAL, T> of_a(st.x, st.y), of_h(st.z, st.w);
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float g = GATE ? S::at(rg, i) : 1.0f;
                float ahat = 0.0f, a = 0.0f;
                if (BN || GATE || A.f) {
                    ahat = !BN ? S::at(rf, i) : of_a(S::at(rf, i));
                    a = !BN ? ahat : GENERAL ? fmaf(ahat, wf[i], bf[i]) : ahat * wf[i];
                }
                float dh = gh ? S::at(rgh, i) : 0.0f;
                if (gy) {
                    const float xhat = of_h.scaled(fmaf(A.sf, GATE ? g * a : a, of_h.begin(A.in_scale, S::at(rx, i))));
                    const float e = S::at(rgy, i);
                    dw[i] = fmaf(e, xhat, dw[i]);
                    if constexpr (GENERAL) db[i] += e;
                    const float u = fmaf(-xhat, mid.y, GENERAL ? e * w[i] - mid.x : e * w[i]);
                    dh = fmaf(st.w, u, dh);
                }
                if constexpr (GATE == 1) dg[i] = fmaf(A.sf * a, dh, dg[i]);
                if constexpr (BN) {
                    const float da = dh * (GATE ? A.sf * g : A.sf);
                    dwf[i] = fmaf(da, ahat, dwf[i]);
                    if constexpr (GENERAL) dbf[i] += da;
                }
            }
        }
        if constexpr (GATE == 1) {
            if (G.dgate) flush(dg, G.gate_column ? G.gate_column + strip * A.dim : nullptr, reinterpret_cast<T*>(G.dgate) + segment * A.dim, false);
        }
    }
    auto column = [&](int k) { return G.column ? G.column + ((int64_t)k * gridDim.y + blockIdx.y) * A.dim : nullptr; };
    if (G.dw) flush(dw, column(0), G.dw, A.w_float);
    if constexpr (GENERAL) {
        if (G.db) flush(db, column(1), G.db, A.w_float);
    }
    if constexpr (BN) {
        if (G.dwf) flush(dwf, column(2), G.dwf, A.w_float);
    }
    if constexpr (BN && GENERAL) {
        if (G.dbf) flush(dbf, column(3), G.dbf, A.w_float);
    }
}

// Adds the `count` rows of a column sum: blockIdx.y 0 to 3 dw, db, dwf, dbf (count: the workgroups of the launch before), 4: the `gates`
// rows of the gate, a gridDim.z'th of them (count: parts).  16 columns per workgroup, eight loads under way per lane; 64 lanes for a column where the
// launch has few workgroups (1021 x 1001: 16 lanes 6.6 us, 64 lanes 4.9), 16 where it has many (16384 x 4096: 10.6, 16.8).
template <typename T>
__global__ __launch_bounds__(1024) void residual_norm_columns_kernel(const NormGrads G, int dim, int64_t blocks, int64_t gates, int w_float) {
    __shared__ float part[16][16];
    const int k = (int)blockIdx.y, c = (int)blockIdx.x * 16 + (threadIdx.x & 15), lane = threadIdx.x >> 4;
    void* const out = k == 0 ? G.dw : k == 1 ? G.db : k == 2 ? G.dwf : k == 3 ? G.dbf : G.dgate;
    if (!out) return;
    const int64_t count = k < 4 ? blocks : G.parts;
    const int lanes = (int)blockDim.x / 16;
    for (int64_t segment = blockIdx.z; segment < (k < 4 ? 1 : gates); segment += gridDim.z) {
        const float* const src = k < 4 ? G.column + (int64_t)k * blocks * dim : G.gate_column + segment * G.parts * dim;
        float s = 0.0f;
        if (c < dim)
            for (int64_t r0 = lane; r0 < count; r0 += 8 * lanes) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = r0 + lanes * j < count ? src[(r0 + lanes * j) * dim + c] : 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j++) s += v[j];
            }
        s = rows_sum(s);
        if ((threadIdx.x & 48) == 0) part[threadIdx.x >> 6][threadIdx.x & 15] = s;
        __syncthreads();
        if (lane == 0 && c < dim) {
            s = 0.0f;
            for (int t = 0; t < lanes / 4; t++) s += part[t][threadIdx.x];
            const int64_t o = k < 4 ? c : segment * dim + c;
            if (k < 4 && w_float) reinterpret_cast<float*>(out)[o] = s;
            else reinterpret_cast<T*>(out)[o] = from_float<T>(s);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------- launches
// f(elements of a piece, lanes of a team, pieces per lane, whether they reach over a row's end, threads of a workgroup): see norm_threads.
template <typename T, typename F>
void with_share(int64_t dim, F f) {
    constexpr int E = 16 / (int)sizeof(T);
    const int threads = norm_threads(dim, E);
    using std::integral_constant;
    auto share = [&](auto lanes, auto vpt) {
        const integral_constant<int, E> e;
        const int64_t whole = (int64_t)(decltype(lanes)::value ? decltype(lanes)::value : threads) * decltype(vpt)::value * E;
        if (dim == whole) f(e, lanes, vpt, std::false_type(), threads);
        else f(e, lanes, vpt, std::true_type(), threads);
    };
    if (dim < E) f(integral_constant<int, 1>(), integral_constant<int, 8>(), integral_constant<int, 1>(), std::true_type(), threads);
    else if (dim <= 8 * E) share(integral_constant<int, 8>(), integral_constant<int, 1>());
    else if (dim <= 16 * E) share(integral_constant<int, 16>(), integral_constant<int, 1>());
    else if (dim <= 32 * E) share(integral_constant<int, 32>(), integral_constant<int, 1>());
    else if (dim <= 64 * E) share(integral_constant<int, 64>(), integral_constant<int, 1>());
    else if (dim <= 1024 * E) share(integral_constant<int, 0>(), integral_constant<int, 1>());
    else if (dim <= 1024 * E * 2) share(integral_constant<int, 0>(), integral_constant<int, 2>());
    else if constexpr (1024 * E * 2 < NORM_MAX_DIM) share(integral_constant<int, 0>(), integral_constant<int, 4>());
}

template <typename T>
void residual_norm_forward(const ResidualNorm& A, T* h, T* y, float* stats, hipStream_t st) {
    with_share<T>(A.dim, [&](auto e, auto lanes, auto vpt, auto tail, int threads) {
        constexpr int E = decltype(e)::value, L = decltype(lanes)::value, V = decltype(vpt)::value, TEAMS = L ? 256 / L : 1;
        constexpr bool TAIL = decltype(tail)::value;
        const int64_t blocks = (A.rows + TEAMS - 1) / TEAMS, most = (int64_t)NORM_CUS * (2048 / threads);
        const dim3 grid((unsigned)(blocks < most ? blocks : most));
        auto launch = [&](auto bn, auto general) {
            hipLaunchKernelGGL((residual_norm_forward_kernel<T, E, L, V, TAIL, decltype(bn)::value, decltype(general)::value>), grid, dim3(threads), 0, st, A,
                               h, y, stats);
        };
        auto kind_of = [&](auto bn) {
            if (A.norm == 1 || A.block_norm == 1 || A.b || A.bf) launch(bn, std::true_type());
            else launch(bn, std::false_type());
        };
        if (A.block_norm) kind_of(std::true_type());
        else kind_of(std::false_type());
    });
}

// f(whether the block is normed, the kind of gate, general), as the kernels' parameters.
template <typename F>
void with_form(const ResidualNorm& A, const NormGrads& G, int64_t gate_rows, bool shared, F f) {
    using std::integral_constant;
    auto kind_of = [&](auto bn, auto gate) {
        if (A.norm == 1 || A.block_norm == 1 || A.b || A.bf || G.db || G.dbf) f(bn, gate, std::true_type());
        else f(bn, gate, std::false_type());
    };
    auto gated = [&](auto bn) {
        if (gate_rows == 0) kind_of(bn, integral_constant<int, 0>());
        else if (shared) kind_of(bn, integral_constant<int, 1>());
        else kind_of(bn, integral_constant<int, 2>());
    };
    if (A.block_norm) gated(std::true_type());
    else gated(std::false_type());
}

template <typename T>
void residual_norm_backward(const ResidualNorm& A, NormGrads G, int64_t gate_rows, float* scratch, hipStream_t st) {
    const NormPlan P = norm_plan(A.rows, A.dim, 16 / (int)sizeof(T), gate_rows, A.block_norm != 0,
                                 A.norm == 1 || A.block_norm == 1 || A.b || A.bf);
    const bool wanted = G.dw || G.db || G.dwf || G.dbf || (G.dgate && P.gate_rows_shared);
    G.column = P.column_floats ? scratch : nullptr;
    G.gate_column = P.gate_floats ? scratch + P.column_floats : nullptr;
    G.mid = P.mid_floats ? scratch + (P.column_floats + P.gate_floats + 3) / 4 * 4 : nullptr;
    int64_t blocks = P.column_blocks;
    if (A.rows > 0) {
        with_share<T>(A.dim, [&](auto e, auto lanes, auto vpt, auto tail, int threads) {
            constexpr int E = decltype(e)::value, L = decltype(lanes)::value, V = decltype(vpt)::value;
            constexpr bool TAIL = decltype(tail)::value;
            with_form(A, G, gate_rows, P.gate_rows_shared, [&](auto bn, auto gate, auto general) {
                constexpr bool BN = decltype(bn)::value, GENERAL = decltype(general)::value;
                constexpr int GATE = decltype(gate)::value;
                auto launch = [&](auto sums) {
                    const auto kernel = residual_norm_backward_kernel<T, E, L, V, TAIL, BN, GATE, GENERAL, decltype(sums)::value>;
                    constexpr int ARRAYS = V > 1 ? 0 : 1 + BN + (BN && GENERAL);
                    const size_t lds = sizeof(float) * ARRAYS * (L ? L : threads) * E;
                    // (beside up to 17 KB of the kernel's own; more than 64 KB has to be asked for)
                    if (lds > 40 * 1024) (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
                    NormGrads R = G;
                    R.strips = P.strips;
                    R.parts = P.parts;
                    hipLaunchKernelGGL(kernel, dim3((unsigned)P.blocks), dim3(threads), lds, st, A, R);
                };
                // (what norm_split can say for these parameters; GENERAL without a norm or bias that is: a bias' gradient alone is wanted)
                constexpr bool ALWAYS = V > 1, SOMETIMES = L == 0 && sizeof(T) == 2 && BN && GENERAL && GATE != 0;
                if constexpr (!ALWAYS) {
                    if (!P.split) launch(std::true_type());
                }
                if constexpr (ALWAYS || SOMETIMES) {
                    if (P.split) launch(std::false_type());
                    if (P.split && wanted) {
                        constexpr int WIDE = 64 * E;
                        const dim3 grid((unsigned)((A.dim + WIDE - 1) / WIDE), (unsigned)P.column_blocks);
                        NormGrads C = G;
                        C.strips = P.column_strips;
                        C.parts = P.column_parts;
                        if (A.dim % WIDE) hipLaunchKernelGGL((residual_norm_column_kernel<T, true, BN, GATE, GENERAL>), grid, dim3(256), 0, st, A, C);
                        else hipLaunchKernelGGL((residual_norm_column_kernel<T, false, BN, GATE, GENERAL>), grid, dim3(256), 0, st, A, C);
                    }
                }
            });
        });
        G.parts = P.split ? P.column_parts : P.parts;
    } else {
        blocks = 0;         // sums over no rows
        G.parts = 0;
    }
    const bool columns = (G.column || A.rows == 0) && (G.dw || G.db || G.dwf || G.dbf);
    const bool gates = G.dgate && (G.gate_column || A.rows == 0);
    if (columns || gates) {
        if (!columns) G.dw = G.db = G.dwf = G.dbf = nullptr;
        if (!gates) G.dgate = nullptr;
        const int64_t segments = !gates ? 1 : A.rows == 0 ? gate_rows : P.segments;
        const dim3 grid((unsigned)((A.dim + 15) / 16), 5, (unsigned)(segments < 64 ? segments : 64));
        const unsigned columns_threads = (int64_t)grid.x * (4 + grid.z) >= 2 * NORM_CUS ? 256 : 1024;
        hipLaunchKernelGGL(residual_norm_columns_kernel<T>, grid, dim3(columns_threads), 0, st, G, A.dim, blocks, segments, A.w_float);
    }
}

}  // namespace cfh
