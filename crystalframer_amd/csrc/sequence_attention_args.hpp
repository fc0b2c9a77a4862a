// What the kernels of attention between sequences are told, and which of them a call takes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cfh {

constexpr int ATTENTION_MAX_DIM = 128;
constexpr int ATTENTION_MAX_REACH = 1024;      // relative positions beyond this (either way) share a bucket
constexpr int ATTENTION_CUS = 256;
constexpr int ATTENTION_LDS = 160 * 1024;
// Beyond the reach by this much on either side biases are kept in LDS: a tile that is not beyond it as a whole needs no bounds.
constexpr int ATTENTION_MARGIN = 96;

// Element strides of (batch, position, head); channels lie next to one another, rows at multiples of 16 bytes.
struct AttentionRows {
    const void* at;
    int64_t batch, row, head;
};

struct SequenceAttention {
    AttentionRows q, k, v;
    const uint8_t* mask;               // per key: 0 = not there; packed (k_rows) or (batch, k_rows); NULL: all are
    const int64_t *q_starts, *k_starts, *q_sizes, *k_sizes;
    const void* table;                 // (buckets, heads)
    const int32_t* bucket_of;          // (2 reach + 1): of the relative positions -reach ... reach
    int64_t q_rows, k_rows;            // packed: of all sequences; else of one
    int32_t packed, batch, heads, kv_heads, share, dim, buckets, reach, causal, last, table_float, float32;
    float scale;
};

struct AttentionGrads {
    AttentionRows go;
    const void *out, *rest;            // (rows, heads, dim), as all that follows; rest: what rounding left of out, in 16 bits
    const float* stats;                // (rows, heads, 2): largest score, one over the sum
    float* rows;                       // (rows, heads): D, from the queries' kernel for the keys'
    void *dq, *dk, *dv;                // (dk, dv over kv_heads)
    float *dq_parts, *dk_parts, *dv_parts;      // of the splits, or NULL
    float* dtable;                     // (workgroups, buckets), or NULL
    float* row_parts;                  // (splits, rows, heads, 3): sum of ds, of P beyond the reach on either side; NULL: one split
};

// Tiles of the grid for rows of `tile`: packed sequence b begins at tile starts[b] / tile + b, which leaves every sequence as many as it
// needs without anyone adding up lengths.
inline int64_t tile_slots(int packed, int64_t rows, int batch, int tile) {
    return packed ? rows / tile + batch + 1 : (int64_t)batch * ((rows + tile - 1) / tile);
}
// Into how many parts an axis goes so that there are about `wanted` wavefronts, with at least `least` rows of the axis to each.
inline int split_count(int64_t wavefronts, int64_t wanted, int64_t rows, int64_t least) {
    const int64_t n = wavefronts > 0 ? wanted / wavefronts : 1, most = rows / least;
    return (int)(n < 1 || most < 1 ? 1 : n > most ? most : n);
}

// Wavefronts of few_kernel and of the backward kernels: what the 160 KB of LDS hold.
constexpr int few_waves(bool float32, int dim) { return float32 && dim > 64 ? 2 : 4; }
inline int64_t queries_lds(bool float32, int dim, int reach, bool table, int waves) {
    const int64_t pitch = dim <= 32 ? 32 : dim <= 64 ? 64 : 128, entries = 2 * (reach + ATTENTION_MARGIN) + 1;
    return 4 * 32 * pitch * (float32 ? 6 : 2) + 64 * 4 + (table ? (entries * (2 * waves + 1) + 2 * waves) * 4 : 0);
}

// Whether few_kernel keeps the biases of its heads in LDS (up to 8 KB); otherwise it reads what tiles within the reach take.
__host__ __device__ inline bool few_line(int heads, int reach) { return heads * (2 * (reach + ATTENTION_MARGIN) + 1) <= 2048; }

struct AttentionPlan {
    bool few, past;        // few_kernel, and keys and values past the caches
    int waves, splits;
    int64_t slots;
};
inline AttentionPlan attention_plan(const SequenceAttention& A) {
    AttentionPlan P{};
    const int64_t q_each = A.packed && A.batch > 0 ? A.q_rows / A.batch : A.q_rows, k_each = A.packed && A.batch > 0 ? A.k_rows / A.batch : A.k_rows;
    const int64_t whole = tile_slots(A.packed, A.q_rows, A.batch, 128);
    // few_kernel where its 32 columns hold a sequence's queries, and where tiles_kernel's workgroups of 128 queries would leave compute
    // units idle (us, few and tiles, workgroups of these: 4 x 512 queries, 2048 keys, 8 heads of 64, 128: 29, 39; 1024 x 1024, 8 heads of 128,
    // 64: 22, 28, twice that, 128: 29, 29; odd lengths in float32, all passes: 217, 226).
    P.few = q_each * (A.share < 32 ? A.share : 32) <= 32 || whole * A.heads < 192;
    P.splits = 1;
    P.slots = whole;
    P.waves = 4;
    if (!P.few) return P;
    const int at_once = A.share < 32 ? A.share : 32, groups = (A.share + at_once - 1) / at_once;
    P.slots = tile_slots(A.packed, A.q_rows, A.batch, 32 / at_once);
    // One wavefront where there are no keys for more (256 x 16 queries, up to 60 keys, all passes: 56 us, with four 83); but biases of a call that
    // leaves compute units idle are brought by all of them (37 tokens with a bias: 7.7 us, with one wavefront 10.7).
    const bool idle = P.slots * A.kv_heads * groups <= ATTENTION_CUS;
    P.waves = k_each <= 64 && !(A.table && idle) ? 1 : few_waves(A.float32, A.dim);
    const int64_t keys = A.packed ? A.k_rows : A.k_rows * A.batch;
    // One tile of queries for each key head reads keys and values once: bytes, which many wavefronts bring fastest (16 x 1 to 8192 keys of
    // 16 heads of 64: 80 us undivided, 71 with 32 wavefronts for each compute unit).  Several tiles read them from the caches: no more parts
    // than fill the SIMDs, since a part costs its sums' way through memory (4 x 512 queries, 2048 keys, 8 heads of 64: 29 us, four parts 40).
    const bool once = q_each * at_once <= 32 && groups == 1;
    P.past = once && keys * A.kv_heads * A.dim * (A.float32 ? 8 : 4) >= 1 << 27;
    P.splits = split_count(P.slots * A.kv_heads * groups * P.waves, (once ? 32 : 4) * ATTENTION_CUS, k_each, 64 * P.waves);
    return P;
}

struct AttentionGradPlan {
    int q_waves, q_splits, k_waves, k_splits;
    int64_t q_slots, k_slots;
};
inline AttentionGradPlan attention_grad_plan(const SequenceAttention& A) {
    AttentionGradPlan P{};
    const int64_t q_each = A.packed && A.batch > 0 ? A.q_rows / A.batch : A.q_rows, k_each = A.packed && A.batch > 0 ? A.k_rows / A.batch : A.k_rows;
    P.q_waves = q_each > 64 && queries_lds(A.float32, A.dim, A.reach, A.table != nullptr, 4) <= ATTENTION_LDS ? 4 : 1;
    P.k_waves = k_each > 64 ? 4 : 1;
    P.q_slots = tile_slots(A.packed, A.q_rows, A.batch, 32 * P.q_waves);
    P.k_slots = tile_slots(A.packed, A.k_rows, A.batch, 32 * P.k_waves);
    // (parts: odd lengths, 5 heads on 1 of 40 in float32, all passes 217 us, without 599; 6 heads on 3 of 80 in float16 62 and 81)
    P.q_splits = split_count(P.q_slots * A.heads * P.q_waves, 8 * ATTENTION_CUS, k_each, 128);
    P.k_splits = split_count(P.k_slots * A.kv_heads * P.k_waves, 8 * ATTENTION_CUS, q_each * A.share, 128);
    return P;
}

template <typename T>
void sequence_attention_forward(const SequenceAttention& A, const AttentionPlan& P, T* out, T* rest, float* stats, float* scratch, hipStream_t st);
template <typename T>
void sequence_attention_backward(const SequenceAttention& A, const AttentionGradPlan& P, AttentionGrads G, void* dtable, float* scratch, hipStream_t st);
}  // namespace cfh
