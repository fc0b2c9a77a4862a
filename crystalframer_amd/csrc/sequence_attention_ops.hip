// C ABI of attention between sequences (see include/crystalframer_hip.h): argument checks and launches.  Nothing here allocates or
// synchronises.
#include "../../include/crystalframer_hip.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "element_types.hpp"
#include "host_error.hpp"
#include "sequence_attention_args.hpp"

namespace {

using cfh::fail;
using cfh::finish_launch;

constexpr int64_t MAX_ROWS = 0x7fffff00LL;      // of a sequence, and of all packed ones
constexpr int64_t MAX_ALL = 1LL << 40;               // rows of a batch
constexpr int64_t MAX_THREADS = 0xffffff00LL;      // of a grid's first dimension

// Rows begin at multiples of 16 bytes, and a tile of them is less than 2^30 bytes.
int check_rows(const void* at, const int64_t* stride, int dtype) {
    const int64_t bytes = dtype == CFH_FLOAT32 ? 4 : 2;
    uint64_t all = (uint64_t)(uintptr_t)at;
    for (int n = 0; n < 3; n++) {
        if (stride[n] < 0 || stride[n] > INT64_MAX / 8) return fail(CFH_EINVAL, "attention: strides must not be negative");
        all |= (uint64_t)(stride[n] * bytes);
    }
    if (all & 15) return fail(CFH_EINVAL, "attention: an address or a stride is no multiple of 16 bytes");
    if (stride[1] * bytes >= 1 << 24) return fail(CFH_EINVAL, "attention: strides: rows %lld bytes apart: less than 2^24", (long long)(stride[1] * bytes));
    return CFH_OK;
}

int check_attention(const cfh_attention* a) {
    if (!a || a->struct_size != (int32_t)sizeof(cfh_attention)) return fail(CFH_EINVAL, "attention: struct_size does not match");
    if (a->dtype < CFH_FLOAT32 || a->dtype > CFH_FLOAT16) return fail(CFH_EINVAL, "attention: dtype %d", (int)a->dtype);
    if (a->dim < 1 || a->dim > CFH_ATTENTION_MAX_DIM)
        return fail(CFH_EINVAL, "attention: dim = %d: 1 to %d channels of a head", (int)a->dim, CFH_ATTENTION_MAX_DIM);
    if (a->heads < 1 || a->heads > 65535 || a->kv_heads < 1 || a->heads % a->kv_heads)
        return fail(CFH_EINVAL, "attention: heads = %d, kv_heads = %d: every key head serves as many of up to 65535 heads", (int)a->heads, (int)a->kv_heads);
    if (a->batch < 0 || a->query_rows < 0 || a->query_rows > MAX_ROWS || a->key_rows < 0 || a->key_rows > MAX_ROWS)
        return fail(CFH_EINVAL, "attention: batch = %d, query_rows = %lld, key_rows = %lld out of range", (int)a->batch, (long long)a->query_rows,
                    (long long)a->key_rows);
    if (!a->packed && a->batch > 0 && (a->query_rows * a->batch > MAX_ALL || a->key_rows * a->batch > MAX_ALL))
        return fail(CFH_EINVAL, "attention: %d sequences of %lld and %lld rows are too many", (int)a->batch, (long long)a->query_rows, (long long)a->key_rows);
    if (!(a->scale > 0.0f) || !(a->scale <= CFH_ATTENTION_MAX_SCALE)) return fail(CFH_EINVAL, "attention: scale = %g: positive, up to %g", a->scale, CFH_ATTENTION_MAX_SCALE);
    if (a->packed && (!a->query_starts || !a->key_starts)) return fail(CFH_EINVAL, "attention: packed sequences need query_starts and key_starts");
    if (a->packed && (a->query_sizes || a->key_sizes)) return fail(CFH_EINVAL, "attention: query_sizes and key_sizes are of sequences that are not packed");
    if (!a->packed && (a->query_starts || a->key_starts)) return fail(CFH_EINVAL, "attention: query_starts and key_starts are of packed sequences");
    const int64_t q_all = a->packed ? a->query_rows : a->query_rows * a->batch, k_all = a->packed ? a->key_rows : a->key_rows * a->batch;
    if ((q_all > 0 && !a->q) || (k_all > 0 && (!a->k || !a->v))) return fail(CFH_EINVAL, "attention: q, k and v must not be NULL");
    for (int rc : {check_rows(a->q, a->q_stride, a->dtype), check_rows(a->k, a->k_stride, a->dtype), check_rows(a->v, a->v_stride, a->dtype)})
        if (rc) return rc;
    if (a->table) {
        if (a->table_dtype != a->dtype && a->table_dtype != CFH_FLOAT32)
            return fail(CFH_EINVAL, "attention: table_dtype %d is neither dtype nor float32", (int)a->table_dtype);
        if (a->reach < 0 || a->reach > CFH_ATTENTION_MAX_REACH)
            return fail(CFH_EINVAL, "attention: reach = %d: 0 to %d", (int)a->reach, CFH_ATTENTION_MAX_REACH);
        if (a->buckets < 1 || a->buckets > 65535) return fail(CFH_EINVAL, "attention: buckets = %d: 1 to 65535", (int)a->buckets);
        if (!a->bucket_of) return fail(CFH_EINVAL, "attention: a table needs bucket_of");
    } else if (a->buckets || a->reach || a->bucket_of) {
        return fail(CFH_EINVAL, "attention: buckets, reach and bucket_of belong to a table");
    }
    if (a->table && !(a->scale >= 0x1p-64f && a->scale <= 0x1p64f)) return fail(CFH_EINVAL, "attention: scale = %g: from 2^-64 to 2^64 with a table", a->scale);
    return CFH_OK;
}

// A single row needs no stride to the next; the kernels need one, so that what they read behind it lies behind its buffer's end, too.
cfh::AttentionRows device_rows(const cfh_attention* a, const void* at, const int64_t* stride, int64_t rows) {
    const int each = a->dtype == CFH_FLOAT32 ? 4 : 8;
    return {at, stride[0], rows > 1 ? stride[1] : (a->dim + each - 1) / each * each, stride[2]};
}
cfh::SequenceAttention device_args(const cfh_attention* a) {
    cfh::SequenceAttention A{};
    A.q = device_rows(a, a->q, a->q_stride, a->query_rows);
    A.k = device_rows(a, a->k, a->k_stride, a->key_rows);
    A.v = device_rows(a, a->v, a->v_stride, a->key_rows);
    A.mask = a->key_mask;
    A.q_starts = a->query_starts; A.k_starts = a->key_starts; A.q_sizes = a->query_sizes; A.k_sizes = a->key_sizes;
    A.table = a->table; A.bucket_of = a->bucket_of;
    A.q_rows = a->query_rows; A.k_rows = a->key_rows;
    A.packed = a->packed; A.batch = a->batch; A.heads = a->heads; A.kv_heads = a->kv_heads; A.share = a->heads / a->kv_heads;
    A.dim = a->dim; A.buckets = a->buckets; A.reach = a->reach; A.causal = a->causal; A.last = a->queries_last;
    A.table_float = a->table_dtype == CFH_FLOAT32;
    A.float32 = a->dtype == CFH_FLOAT32;
    A.scale = a->scale;
    return A;
}
int padded_dim(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }
int64_t q_all(const cfh::SequenceAttention& A) { return (A.packed ? A.q_rows : A.q_rows * A.batch) * A.heads; }
int64_t k_all(const cfh::SequenceAttention& A) { return (A.packed ? A.k_rows : A.k_rows * A.batch) * A.kv_heads; }

// The launches' sizes; a row more than a grid holds is refused here.
int check_grids(const cfh::SequenceAttention& A, bool backward) {
    const cfh::AttentionPlan P = cfh::attention_plan(A);
    const cfh::AttentionGradPlan B = cfh::attention_grad_plan(A);
    const int64_t rows = A.packed ? A.q_rows : A.q_rows * A.batch;
    const bool fits = !backward ? P.slots <= MAX_THREADS / (P.few ? 64 * P.waves : 256) / (P.few ? 1 : A.heads) && (P.splits == 1 || rows <= MAX_THREADS / 64 / A.heads)
                                : B.q_slots <= MAX_THREADS / (64 * B.q_waves) / A.heads && B.k_slots <= MAX_THREADS / (64 * B.k_waves) / A.kv_heads;
    if (!fits) return fail(CFH_EINVAL, "attention: %lld rows and %lld keys of %d heads are more than a grid holds", (long long)rows, (long long)A.k_rows, (int)A.heads);
    return CFH_OK;
}
int check_workspace(const void* workspace, size_t have, size_t need) {
    if (need > 0 && (!workspace || ((uintptr_t)workspace & 15) || have < need))
        return fail(CFH_EWORKSPACE, "attention: workspace of %zu bytes, aligned to 16, is missing", need);
    return CFH_OK;
}
template <typename F>
void with_type(int dtype, F f) {
    if (dtype == CFH_FLOAT32) f(float());
    else if (dtype == CFH_BFLOAT16) f(cfh::bf16());
    else f(cfh::f16());
}

}  // namespace

extern "C" {

size_t cfh_attention_forward_workspace_bytes(const cfh_attention* a) {
    if (check_attention(a)) return 0;
    const cfh::SequenceAttention A = device_args(a);
    const cfh::AttentionPlan P = cfh::attention_plan(A);
    return P.splits > 1 ? (size_t)P.splits * q_all(A) * (padded_dim(A.dim) + 2) * sizeof(float) : 0;
}

int cfh_attention_forward(const cfh_attention* a, void* out, void* out_rest, float* stats, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_attention(a);
    if (rc) return rc;
    const cfh::SequenceAttention A = device_args(a);
    if (q_all(A) == 0) return CFH_OK;
    if (!out || (((uintptr_t)out | (uintptr_t)out_rest) & 15)) return fail(CFH_EINVAL, "attention: out must not be NULL, and aligned to 16 bytes, as out_rest");
    if (a->dtype == CFH_FLOAT32 && out_rest) return fail(CFH_EINVAL, "attention: out_rest is of 16-bit types");
    if ((rc = check_grids(A, false))) return rc;
    if ((rc = check_workspace(workspace, workspace_bytes, cfh_attention_forward_workspace_bytes(a)))) return rc;
    with_type(a->dtype, [&](auto t) {
        using T = decltype(t);
        cfh::sequence_attention_forward<T>(A, cfh::attention_plan(A), (T*)out, (T*)out_rest, stats, (float*)workspace, (hipStream_t)stream);
    });
    return finish_launch("attention_forward");
}

size_t cfh_attention_backward_workspace_bytes(const cfh_attention* a) {
    if (check_attention(a)) return 0;
    const cfh::SequenceAttention A = device_args(a);
    const cfh::AttentionGradPlan P = cfh::attention_grad_plan(A);
    size_t floats = (size_t)q_all(A) + 32;
    if (P.q_splits > 1) floats += (size_t)P.q_splits * q_all(A) * A.dim;
    if (P.k_splits > 1) floats += 2 * (size_t)P.k_splits * k_all(A) * A.dim;
    if (A.table) floats += (size_t)P.q_slots * P.q_splits * A.heads * A.buckets + (P.q_splits > 1 ? 3 * (size_t)P.q_splits * q_all(A) : 0);
    return floats * sizeof(float);
}

int cfh_attention_backward(const cfh_attention* a, const void* out, const void* out_rest, const float* stats, const void* gout, const int64_t gout_stride[3],
                           void* dq, void* dk, void* dv, void* dtable, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_attention(a);
    if (rc) return rc;
    const cfh::SequenceAttention A = device_args(a);
    if (dtable && !a->table) return fail(CFH_EINVAL, "attention: a gradient of a table that is not there");
    if (q_all(A) > 0 && (!out || !stats || !gout || !gout_stride || !dq)) return fail(CFH_EINVAL, "attention: out, stats, gout, its strides and dq must not be NULL");
    if (q_all(A) > 0 && !out_rest != (a->dtype == CFH_FLOAT32)) return fail(CFH_EINVAL, "attention: out_rest belongs to 16-bit types");
    if (k_all(A) > 0 && !dk != !dv) return fail(CFH_EINVAL, "attention: dk and dv go together");
    if (((uintptr_t)out | (uintptr_t)out_rest | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) return fail(CFH_EINVAL, "attention: out, dq, dk and dv must be aligned to 16 bytes");
    const int64_t none[3] = {0, 0, 0};
    const int64_t* const gs = gout_stride ? gout_stride : none;
    if ((rc = check_rows(gout, gs, a->dtype))) return rc;
    if ((rc = check_grids(A, true))) return rc;
    if ((rc = check_workspace(workspace, workspace_bytes, cfh_attention_backward_workspace_bytes(a)))) return rc;
    cfh::AttentionGrads G{};
    G.go = device_rows(a, gout, gs, a->query_rows);
    G.out = out; G.rest = out_rest; G.stats = stats; G.dq = dq; G.dk = dk; G.dv = dv;
    with_type(a->dtype, [&](auto t) {
        cfh::sequence_attention_backward<decltype(t)>(A, cfh::attention_grad_plan(A), G, dtable, (float*)workspace, (hipStream_t)stream);
    });
    return finish_launch("attention_backward");
}

}  // extern "C"
