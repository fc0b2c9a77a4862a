// C ABI of the operators around the layers' products (see include/crystalframer_hip.h): AdamW over tensors of several types with
// moments in 32 or 8 bits, the norm of the gradients, and the residual stream joined and normed.  Host side: argument
// checks and launches.  Nothing here allocates or synchronises.
#include "../../include/crystalframer_hip.h"

#include <hip/hip_runtime.h>

#include <cmath>

#include "adamw_moments.hpp"
#include "host_error.hpp"
#include "residual_norm_args.hpp"

namespace {

using cfh::fail;
using cfh::finish_launch;

constexpr int64_t MAX_ELEMENTS = 1LL << 40;      // of a tensor and of the flat moments
constexpr int64_t JOB_ELEMENTS = 1LL << 30;      // a longer tensor takes several entries of the launch's table

int check_jobs(const char* what, const cfh_param_job* jobs, int32_t njobs, bool update) {
    if (njobs < 0 || (njobs > 0 && !jobs)) return fail(CFH_EINVAL, "%s: jobs is NULL or njobs negative", what);
    for (int32_t j = 0; j < njobs; j++) {
        const cfh_param_job& J = jobs[j];
        if (J.n < 0 || J.n > MAX_ELEMENTS) return fail(CFH_EINVAL, "%s: job %d: n = %lld out of range", what, (int)j, (long long)J.n);
        if (J.dtype < CFH_FLOAT32 || J.dtype > CFH_FLOAT16) return fail(CFH_EINVAL, "%s: job %d: dtype %d", what, (int)j, (int)J.dtype);
        if (J.n > 0 && (!J.grad || (update && !J.param))) return fail(CFH_EINVAL, "%s: job %d: param and grad must not be NULL", what, (int)j);
        const uintptr_t mask = J.dtype == CFH_FLOAT32 ? 3 : 1;
        if (((uintptr_t)J.grad & mask) || (update && ((uintptr_t)J.param & mask)))
            return fail(CFH_EINVAL, "%s: job %d: an address is not one of an element", what, (int)j);
    }
    return CFH_OK;
}

// Calls launch(table) for tables of at most PARAM_MAX_JOBS entries, chunks of `chunk` elements numbered through each.
template <typename F>
void in_tables(const cfh_param_job* jobs, int32_t njobs, int64_t chunk, F launch) {
    cfh::ParamJobs T{};
    for (int32_t j = 0; j < njobs; j++)
        for (int64_t at = 0; at < jobs[j].n; at += JOB_ELEMENTS) {
            const int64_t n = jobs[j].n - at < JOB_ELEMENTS ? jobs[j].n - at : JOB_ELEMENTS, size = jobs[j].dtype == CFH_FLOAT32 ? 4 : 2;
            const int64_t chunks = (n + chunk - 1) / chunk;
            if (T.njobs == cfh::PARAM_MAX_JOBS || (int64_t)T.chunks + chunks > cfh::MAX_CHUNKS) {
                launch(T);
                T.njobs = 0;
                T.chunks = 0;
            }
            cfh::ParamJob& W = T.job[T.njobs++];
            W.p = jobs[j].param ? (char*)jobs[j].param + at * size : nullptr;
            W.g = (const char*)jobs[j].grad + at * size;
            W.first = (uint64_t)(jobs[j].first + at);
            W.n = (uint32_t)n;
            W.chunk0 = T.chunks;
            W.dtype = jobs[j].dtype;
            T.chunks += (uint32_t)chunks;
        }
    if (T.njobs > 0) launch(T);
}

int64_t elements(const cfh_param_job* jobs, int32_t njobs) {
    int64_t n = 0;
    for (int32_t j = 0; j < njobs; j++) n += jobs[j].n;
    return n;
}

// Elements that a workgroup of the norm takes at a time: the larger count once there are two such turns for each compute unit.
int64_t norm_chunk(const cfh_param_job* jobs, int32_t njobs) {
    return elements(jobs, njobs) < 512LL * cfh::GRAD_NORM_CHUNK ? cfh::GRAD_NORM_FEW : cfh::GRAD_NORM_CHUNK;
}

// Bytes of the tensors' elements.
int64_t tensor_bytes(const cfh_param_job* jobs, int32_t njobs) {
    int64_t bytes = 0;
    for (int32_t j = 0; j < njobs; j++) bytes += jobs[j].n * (jobs[j].dtype == CFH_FLOAT32 ? 4 : 2);
    return bytes;
}

int check_moments(const char* what, const cfh_moments* s) {
    if (!s) return fail(CFH_EINVAL, "%s: state must not be NULL", what);
    if (s->bits != 8 && s->bits != 32) return fail(CFH_EINVAL, "%s: moments in %d bits: 8 or 32", what, (int)s->bits);
    if (s->size < 0 || s->size > MAX_ELEMENTS) return fail(CFH_EINVAL, "%s: size = %lld out of range", what, (long long)s->size);
    if (s->size > 0 && (!s->exp_avg || !s->exp_avg_sq || (s->bits == 8 && (!s->exp_avg_scale || !s->exp_avg_sq_scale))))
        return fail(CFH_EINVAL, "%s: the moments and, in 8 bits, their scales must not be NULL", what);
    if (((uintptr_t)s->exp_avg | (uintptr_t)s->exp_avg_sq) & 15) return fail(CFH_EINVAL, "%s: the moments must be aligned to 16 bytes", what);
    return CFH_OK;
}

int check_norm(const cfh_residual_norm* a, bool backward) {
    if (!a || a->struct_size != (int32_t)sizeof(cfh_residual_norm)) return fail(CFH_EINVAL, "residual_norm: struct_size does not match");
    if (a->dtype < CFH_FLOAT32 || a->dtype > CFH_FLOAT16) return fail(CFH_EINVAL, "residual_norm: dtype %d", (int)a->dtype);
    if (a->weight_dtype != a->dtype && a->weight_dtype != CFH_FLOAT32)
        return fail(CFH_EINVAL, "residual_norm: weight_dtype %d is neither dtype nor float32", (int)a->weight_dtype);
    if (a->norm < 0 || a->norm > CFH_NORM_RMS || a->block_norm < 0 || a->block_norm > CFH_NORM_RMS)
        return fail(CFH_EINVAL, "residual_norm: norm %d, block_norm %d", (int)a->norm, (int)a->block_norm);
    if (a->rows < 0 || a->rows > 0x7fffffffLL) return fail(CFH_EINVAL, "residual_norm: rows = %lld out of range", (long long)a->rows);
    if (a->dim < 1 || a->dim > cfh::NORM_MAX_DIM)
        return fail(CFH_EINVAL, "residual_norm: dim = %lld: 1 to %d", (long long)a->dim, cfh::NORM_MAX_DIM);
    if (!(a->eps >= 0.0f) || !(a->block_eps >= 0.0f)) return fail(CFH_EINVAL, "residual_norm: eps must not be negative");
    if (a->gate_rows < 0 || (a->gate_rows > 0 && (a->rows % a->gate_rows || (!a->gate && a->rows > 0))) || (a->gate_rows == 0 && a->gate && a->rows > 0))
        return fail(CFH_EINVAL, "residual_norm: gate_rows = %lld does not go with gate and %lld rows", (long long)a->gate_rows, (long long)a->rows);
    if (a->x_stride < 0 || a->block_stride < 0) return fail(CFH_EINVAL, "residual_norm: strides must not be negative");
    if (a->rows > 0 && !a->x) return fail(CFH_EINVAL, "residual_norm: x must not be NULL");
    const bool block = a->block || (backward && a->joined);
    if (a->rows > 0 && !block && (a->gate || a->block_norm)) return fail(CFH_EINVAL, "residual_norm: gate and block_norm need a block");
    if (backward && a->joined && (a->gate || a->block_norm || a->block))
        return fail(CFH_EINVAL, "residual_norm: joined does not go with a gate, a block or its norm");
    return CFH_OK;
}

cfh::ResidualNorm device_args(const cfh_residual_norm* a) {
    cfh::ResidualNorm A{};
    A.x = a->x; A.f = a->block; A.gate = a->gate; A.w = a->weight; A.b = a->bias; A.wf = a->block_weight; A.bf = a->block_bias;
    A.rows = a->rows; A.xs = a->x_stride; A.fs = a->block_stride;
    A.gate_span = a->gate_rows > 0 ? a->rows / a->gate_rows : 0;
    A.dim = (int32_t)a->dim; A.norm = a->norm; A.block_norm = a->block_norm;
    A.w_float = a->weight_dtype == CFH_FLOAT32;
    A.eps = a->eps; A.block_eps = a->block_eps; A.sx = a->residual_scale; A.sf = a->block_scale;
    A.in_scale = a->residual_scale;
    return A;
}

template <typename F>
void with_type(int dtype, F f) {
    if (dtype == CFH_FLOAT32) f(float());
    else if (dtype == CFH_BFLOAT16) f(cfh::bf16());
    else f(cfh::f16());
}

}  // namespace

extern "C" {

int cfh_adamw_step_moments(const cfh_param_job* jobs, int32_t njobs, const cfh_moments* state, double lr, double beta1, double beta2,
                           double eps, double weight_decay, const cfh_grad_clip* clip, uint64_t* step_dev, float* scratch, void* stream) {
    int rc = check_jobs("adamw", jobs, njobs, true);
    if (rc || (rc = check_moments("adamw", state))) return rc;
    if (!step_dev || !scratch) return fail(CFH_EINVAL, "adamw: step_dev and scratch must not be NULL");
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0))
        return fail(CFH_EINVAL, "adamw: beta1 = %g, beta2 = %g must lie in [0, 1), eps = %g must not be negative", beta1, beta2, eps);
    for (int32_t j = 0; j < njobs; j++)
        if (jobs[j].first < 0 || jobs[j].first % cfh::MOMENT_BLOCK || jobs[j].first > state->size - jobs[j].n)
            return fail(CFH_EINVAL, "adamw: job %d: elements %lld ... of %lld moments (a multiple of %d)", (int)j, (long long)jobs[j].first,
                        (long long)state->size, cfh::MOMENT_BLOCK);
    if (clip && (!clip->norm || clip->count < 0 || (clip->count > 0 && !clip->sums) || !(clip->max_norm >= 0.0)))
        return fail(CFH_EINVAL, "adamw: clip: max_norm = %g must not be negative, sums and norm not NULL", clip->max_norm);
    hipStream_t st = (hipStream_t)stream;
    const cfh::Moments W{state->exp_avg, state->exp_avg_sq, state->exp_avg_scale, state->exp_avg_sq_scale};
    cfh::AdamWStep* const S = reinterpret_cast<cfh::AdamWStep*>(scratch);
    const cfh::AdamWRates R{beta1, beta2, (float)eps};
    const bool past = 2 * tensor_bytes(jobs, njobs) + state->size * (state->bits / 4) >= 2 * cfh::CACHED_BYTES;
    cfh::GradClip C{};
    if (clip) C = {clip->sums, clip->count, clip->max_norm, clip->norm};
    hipLaunchKernelGGL(cfh::adamw_begin_kernel, dim3(1), dim3(256), 0, st, S, reinterpret_cast<unsigned long long*>(step_dev), lr, beta1, beta2,
                       weight_decay, C);
    const bool exact = R.eps < 0x1p-38f, few = !exact && elements(jobs, njobs) < 512LL * cfh::ADAMW_CHUNK;
    in_tables(jobs, njobs, few ? cfh::ADAMW_FEW : cfh::ADAMW_CHUNK, [&](const cfh::ParamJobs& T) {
        using cfh::adamw_moments_kernel;
        auto form = [&](auto bits) {
            constexpr int BITS = decltype(bits)::value;
            return exact  ? adamw_moments_kernel<BITS, cfh::ADAMW_CHUNK, false, true>
                   : few  ? adamw_moments_kernel<BITS, cfh::ADAMW_FEW, false, false>
                   : past ? adamw_moments_kernel<BITS, cfh::ADAMW_CHUNK, true, false>
                          : adamw_moments_kernel<BITS, cfh::ADAMW_CHUNK, false, false>;
        };
        const auto kernel = state->bits == 8 ? form(std::integral_constant<int, 8>()) : form(std::integral_constant<int, 32>());
        hipLaunchKernelGGL(kernel, dim3(T.chunks), dim3(256), 0, st, T, W, S, R);
    });
    return finish_launch("adamw_step_moments");
}

int cfh_adamw_moments(const cfh_moments* state, float* exp_avg, float* exp_avg_sq, void* stream) {
    int rc = check_moments("adamw_moments", state);
    if (rc) return rc;
    if (state->bits != 8) return fail(CFH_EINVAL, "adamw_moments: moments in 32 bits stand for themselves");
    if (state->size == 0) return CFH_OK;
    if (!exp_avg || !exp_avg_sq) return fail(CFH_EINVAL, "adamw_moments: exp_avg and exp_avg_sq must not be NULL");
    const cfh::Moments W{state->exp_avg, state->exp_avg_sq, state->exp_avg_scale, state->exp_avg_sq_scale};
    for (int64_t at = 0, most = (int64_t)cfh::MAX_CHUNKS * cfh::VALUES_CHUNK; at < state->size; at += most) {
        const int64_t n = state->size - at < most ? state->size - at : most;
        hipLaunchKernelGGL(cfh::moment_values_kernel, dim3((unsigned)((n + cfh::VALUES_CHUNK - 1) / cfh::VALUES_CHUNK), 2), dim3(256), 0,
                           (hipStream_t)stream, W, (uint64_t)at, (uint64_t)state->size, exp_avg, exp_avg_sq);
    }
    return finish_launch("adamw_moments");
}

int32_t cfh_grad_square_sums_count(const cfh_param_job* jobs, int32_t njobs) {
    int rc = check_jobs("grad_square_sums", jobs, njobs, false);
    if (rc) return rc;
    int64_t n = 0;
    in_tables(jobs, njobs, norm_chunk(jobs, njobs), [&](const cfh::ParamJobs& T) { n += T.chunks < cfh::GRAD_NORM_BLOCKS ? T.chunks : cfh::GRAD_NORM_BLOCKS; });
    if (n > 0x7fffffff) return fail(CFH_EINVAL, "grad_square_sums: too many tensors");
    return (int32_t)n;
}

int cfh_grad_square_sums(const cfh_param_job* jobs, int32_t njobs, double* sums, int32_t count, void* stream) {
    const int32_t need = cfh_grad_square_sums_count(jobs, njobs);
    if (need < 0) return need;
    if (count != need || (need > 0 && !sums) || ((uintptr_t)sums & 7))
        return fail(CFH_EINVAL, "grad_square_sums: %d sums, aligned to 8 bytes, have to be there", (int)need);
    hipStream_t st = (hipStream_t)stream;
    const int64_t chunk = norm_chunk(jobs, njobs), bytes = tensor_bytes(jobs, njobs);
    in_tables(jobs, njobs, chunk, [&](const cfh::ParamJobs& T) {
        const int blocks = T.chunks < cfh::GRAD_NORM_BLOCKS ? (int)T.chunks : cfh::GRAD_NORM_BLOCKS;
        const auto kernel = chunk == cfh::GRAD_NORM_FEW ? cfh::grad_square_kernel<cfh::GRAD_NORM_FEW, false>
                            : bytes < cfh::CACHED_BYTES ? cfh::grad_square_kernel<cfh::GRAD_NORM_CHUNK, false>
                                                        : cfh::grad_square_kernel<cfh::GRAD_NORM_CHUNK, true>;
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, st, T, sums);
        sums += blocks;
    });
    return finish_launch("grad_square_sums");
}

int cfh_residual_norm_forward(const cfh_residual_norm* a, void* h, void* y, float* stats, void* stream) {
    int rc = check_norm(a, false);
    if (rc) return rc;
    if (a->joined) return fail(CFH_EINVAL, "residual_norm: joined is of the backward pass");
    if (y && a->norm == CFH_NORM_NONE) return fail(CFH_EINVAL, "residual_norm: y needs a norm");
    if (a->rows == 0 || (!h && !y && !stats)) return CFH_OK;
    const cfh::ResidualNorm A = device_args(a);
    with_type(a->dtype, [&](auto t) {
        using T = decltype(t);
        cfh::residual_norm_forward<T>(A, (T*)h, (T*)y, stats, (hipStream_t)stream);
    });
    return finish_launch("residual_norm_forward");
}

size_t cfh_residual_norm_backward_workspace_bytes(const cfh_residual_norm* a) {
    if (check_norm(a, true)) return 0;
    const cfh::NormPlan P = cfh::norm_plan(a->rows, a->dim, a->dtype == CFH_FLOAT32 ? 4 : 8, a->gate_rows, a->block_norm != 0,
                                           a->norm == CFH_NORM_LAYER || a->block_norm == CFH_NORM_LAYER || a->bias || a->block_bias);
    return (P.column_floats + P.gate_floats + P.mid_floats + 8) * sizeof(float);
}

int cfh_residual_norm_backward(const cfh_residual_norm* a, const float* stats, const void* gh, const void* gy, void* dx, void* dblock,
                               void* dgate, void* dweight, void* dbias, void* dblock_weight, void* dblock_bias, void* workspace,
                               size_t workspace_bytes, void* stream) {
    int rc = check_norm(a, true);
    if (rc) return rc;
    if (gy && a->norm == CFH_NORM_NONE) return fail(CFH_EINVAL, "residual_norm: gy needs a norm");
    if (a->rows > 0 && !stats) return fail(CFH_EINVAL, "residual_norm: stats must not be NULL");
    if ((dblock && !a->block && !a->joined) || (dgate && !a->gate_rows) || ((dblock_weight || dblock_bias) && !a->block_norm) ||
        ((dweight || dbias) && !a->norm))
        return fail(CFH_EINVAL, "residual_norm: a gradient of what is not there");
    if (dblock && dblock == dx && (a->gate || a->block_norm || a->residual_scale != a->block_scale))
        return fail(CFH_EINVAL, "residual_norm: dblock differs from dx");
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < cfh_residual_norm_backward_workspace_bytes(a))
        return fail(CFH_EWORKSPACE, "residual_norm: workspace of %zu bytes, aligned to 16, is missing",
                    cfh_residual_norm_backward_workspace_bytes(a));
    cfh::ResidualNorm A = device_args(a);
    if (a->joined) A.in_scale = 1.0f;
    cfh::NormGrads G{};
    G.stats = stats; G.gh = gh; G.gy = gy; G.dx = dx; G.df = dblock == dx ? nullptr : dblock; G.dgate = dgate;
    G.dw = dweight; G.db = dbias; G.dwf = dblock_weight; G.dbf = dblock_bias;
    with_type(a->dtype, [&](auto t) {
        cfh::residual_norm_backward<decltype(t)>(A, G, a->gate_rows, reinterpret_cast<float*>(workspace), (hipStream_t)stream);
    });
    return finish_launch("residual_norm_backward");
}

}  // extern "C"
