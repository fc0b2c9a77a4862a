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

// Wavefronts of few_kernel: as many as the 160 KB of LDS hold tiles for (a power of two; float32 of 128 channels: 48 KB each).
constexpr int few_waves(bool float32, int dim) { return float32 && dim > 64 ? 2 : 4; }
inline int64_t queries_lds(bool float32, int dim, int reach, bool table, int waves) {
    const int64_t pitch = dim <= 32 ? 32 : dim <= 64 ? 64 : 128, entries = 2 * (reach + ATTENTION_MARGIN) + 1;
    return 4 * 32 * pitch * (float32 ? 6 : 2) + 64 * 4 + (table ? (entries * (2 * waves + 1) + 2 * waves) * 4 : 0);
}

// Whether few_kernel keeps the biases of its heads in LDS (up to 8 KB); otherwise it reads what tiles within the reach take.  (us, read and
// kept: 6 x 500 tokens, 5 heads of 40 in float32, reach 77, 7 KB: 57, 50; 4 x 200, 8 heads of 64 in 16 bits, reach 128, 2 KB: 19.6, 17.8; but
// single tokens of 64 heads on 8 of 128 to 4096 positions, 14 KB, where fewer workgroups have room: 70, 94.)
__host__ __device__ inline bool few_line(int heads, int reach) { return heads * (2 * (reach + ATTENTION_MARGIN) + 1) <= 2048; }

// (Times at the rules: us a pass, those of wavefronts, parts, lines and caches replayed from captured graphs, some 8 us with each replay.)
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
    // A wavefront has two tiles of a part at least (us with a half, one, two, four, eight: one token to 2000 keys, 8 heads of 64: 20, 18, 17, 19, 27;
    // 4 to 4000, 32 heads on 8 of 128: 49, 39, 30, 29, 35).
    // Such keys and values go past the caches from 128 MB on, as the tensors have, filled or not: a model's call reads caches that other layers'
    // have been read after.  (us, through and past the caches, 16 heads of 64: of several caches in turn 96 MB 35, 32; 160 MB 47, 43; 256 MB
    // 63, 56; 640 MB 132, 116; one that the call before read 96 MB 30, 30; 160 MB 41, 43; 256 MB 53, 56; 352 MB 79, 73.  Of 512 MB an eighth
    // filled, in turn: 23.4, 24.9, a quarter: 40, 36.)
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
    // A workgroup has one wavefront where a sequence has no rows for more.  us of all passes with one and four, 128 sequences, 8 heads of 64:
    //   queries_kernel  bfloat16  33 tokens 44, 50;  48: 52, 55;  64: 60, 61;  65: 76, 76;  96: 89, 86      float32  33: 129, 122;  64: 136, 128;  96: 238, 176
    //                   with a bias  64: 126, 88;  100: 194, 123       256 x 16 queries of 16 channels, 30 keys, float32: 50, 57
    //   keys_kernel     bfloat16  30 tokens 38, 47;  48: 52, 60;  64: 60, 65;  65: 70, 75;  96: 85, 86      float32  30: 77, 97;  64: 136, 146;  96: 210, 175
    // (one bound for all; below it float32 and biases lose by it in queries_kernel).  Also where four have no room in LDS: float32 of more than
    // 64 channels with a reach beyond 809.
    P.q_waves = q_each > 64 && queries_lds(A.float32, A.dim, A.reach, A.table != nullptr, 4) <= ATTENTION_LDS ? 4 : 1;
    P.k_waves = k_each > 64 ? 4 : 1;
    P.q_slots = tile_slots(A.packed, A.q_rows, A.batch, 32 * P.q_waves);
    P.k_slots = tile_slots(A.packed, A.k_rows, A.batch, 32 * P.k_waves);
    // (parts: odd lengths, 5 heads on 1 of 40 in float32, all passes 217 us, without 599; 6 heads on 3 of 80 in float16 62 and 81.  At least
    // 128 rows of the other axis to each; with 64, 128, 256, 512: 6 x 500 tokens, 5 heads on 1 of 40 in float32 205, 206, 182, 183; 7 x 200 queries,
    // 350 keys, 6 heads on 3 of 80 in float16 60, 58, 68, 69; 1000 tokens, 8 heads of 64 63, 65, 63, 91; 2 x 300, 2000 keys, 4 heads of 128 97, 89, 80, 89.)
    P.q_splits = split_count(P.q_slots * A.heads * P.q_waves, 8 * ATTENTION_CUS, k_each, 128);
    P.k_splits = split_count(P.k_slots * A.kv_heads * P.k_waves, 8 * ATTENTION_CUS, q_each * A.share, 128);
    return P;
}

template <typename T>
void sequence_attention_forward(const SequenceAttention& A, const AttentionPlan& P, T* out, T* rest, float* stats, float* scratch, hipStream_t st);
template <typename T>
void sequence_attention_backward(const SequenceAttention& A, const AttentionGradPlan& P, AttentionGrads G, void* dtable, float* scratch, hipStream_t st);
}  // namespace cfh
