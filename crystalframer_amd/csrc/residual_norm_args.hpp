// What the residual norms' kernels are told, and how their backward pass is cut into strips.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cfh {

constexpr int NORM_MAX_DIM = 16384;

struct ResidualNorm {
    const void *x, *f, *gate, *w, *b, *wf, *bf;
    int64_t rows, xs, fs, gate_span;      // gate_span: rows that share a row of the gate
    int32_t dim, norm, block_norm, w_float;
    float eps, block_eps, sx, sf;
    float in_scale;                       // of x where h is put together (1: x holds h)
};

struct NormGrads {
    const float* stats;
    const void *gh, *gy;
    void *dx, *df, *dgate, *dw, *db, *dwf, *dbf;
    float* column;           // (4, gridDim.x, dim): sums of the workgroups, in the order dw, db, dwf, dbf; NULL: one workgroup, final
    float* gate_column;      // (strips, dim): sums of the strips; NULL: a strip is all that shares its row of the gate, final
    float* mid;              // (rows, 4): mean u and mean u xhat of N and of N_b, for the column kernel; NULL: column sums with the rows
    int64_t strips;
    int32_t parts;           // strips of the rows that share a row of the gate
};

constexpr int NORM_CUS = 256;

struct NormPlan {
    int teams, blocks, parts, column_blocks, column_parts;
    int64_t segments, strips, column_strips;
    bool gate_rows_shared, split;       // split: column sums in a kernel of their own: column_blocks workgroups to a group of columns
    size_t column_floats, gate_floats, mid_floats;
};

// Threads of a workgroup: for rows of up to 64 pieces of 16 bytes 256, in teams of 8, 16, 32 or 64 lanes with a piece each; else one team of as
// many wavefronts as there are 64 pieces in a row, up to 16, where lanes take two or four.  A piece per lane is what leaves the backward
// pass, with its column sums, registers for four wavefronts per SIMD (128) in float32 and, in 16 bits, for one norm of whole rows;
// 16-bit rows with both norms spill there: 20 bytes a lane for whole rows and root-mean-square norms with a shared gate, up to 276 for layer norms
// with a tail and a gate.  Several pieces per lane spill in most forms (up to 476 bytes in 16 bits, 676 in float32).
inline int norm_threads(int64_t dim, int elements) {
    const int64_t pieces = (dim + elements - 1) / elements;
    if (pieces <= 64) return 256;
    return pieces >= 1024 ? 1024 : (int)((pieces + 63) / 64 * 64);
}
inline int norm_teams(int64_t dim, int elements) {
    const int64_t pieces = (dim + elements - 1) / elements;
    return pieces <= 8 ? 32 : pieces <= 16 ? 16 : pieces <= 32 ? 8 : pieces <= 64 ? 4 : 1;
}

// Whether the backward pass makes its column sums in a kernel of its own, which reads the rows' arrays again but keeps no lane waiting for
// another: where one kernel has no registers for both.  These are rows of more than 1024 pieces (4096 x 16384 bfloat16, layer norms on
// both sides and a gate: 1365 us in one kernel, 424 in two; 4096 x 12288, one norm: 451, 194; 4096 x 8192 float32, gated: 371, 273), and
// rows in 16 bits, where a lane has eight columns, with both norms, biases and a gate (32768 x 1024: 221, 168; 8192 x 4096: 215, 176;
// without the gate 114, 129, and root-mean-square norms alone 104, 135: one kernel), from 2^20 elements on (both passes in a graph, float16,
// a gate per element: 4096 x 1001 77, 54; 1021 x 1001 38.6, 37.4; 256 x 4096 29.5, 29.7; 256 x 1001 24.5, 27.8; 64 x 4096 21.9, 25.9).
inline bool norm_split(int64_t rows, int64_t dim, int elements, int64_t gate_rows, bool block_norm, bool general) {
    return dim > 1024 * elements || (elements == 8 && dim > 64 * elements && rows * dim >= 1 << 20 && block_norm && general && gate_rows > 0);
}

// Strips of rows: as many as there are workgroups at once, but with two rows for each team of a workgroup where there are fewer, and
// none across two rows of the gate.
inline NormPlan norm_plan(int64_t rows, int64_t dim, int elements, int64_t gate_rows, bool block_norm, bool general) {
    NormPlan P{};
    P.teams = norm_teams(dim, elements);
    P.gate_rows_shared = gate_rows > 0 && gate_rows < rows;
    P.segments = P.gate_rows_shared ? gate_rows : 1;
    const int threads = norm_threads(dim, elements);
    const int64_t resident = 1024 / threads, target = NORM_CUS * (resident < 1 ? 1 : resident), span = rows / P.segments;
    auto in_parts = [&](int64_t strips, int64_t most) {
        strips = strips < 1 ? 1 : strips > most ? most : strips;
        int64_t parts = strips / P.segments;
        if (parts < 1) parts = 1;
        if (parts > span) parts = span > 0 ? span : 1;
        return (int)parts;
    };
    P.parts = in_parts(rows / (2 * P.teams), target);
    P.strips = P.segments * P.parts;
    P.blocks = (int)(P.strips < target ? P.strips : target);
    P.split = norm_split(rows, dim, elements, gate_rows, block_norm, general);
    P.column_strips = P.strips;
    P.column_parts = P.parts;
    P.column_blocks = P.blocks;
    if (P.split) {
        const int64_t groups = (dim + 64 * elements - 1) / (64 * elements);
        const int64_t most = 4 * NORM_CUS / groups;      // (at least 16: there are up to 64 groups)
        P.column_parts = in_parts(rows / 16, most);
        P.column_strips = P.segments * P.column_parts;
        P.column_blocks = (int)(P.column_strips < most ? P.column_strips : most);
        P.mid_floats = (size_t)rows * 4;
    }
    P.column_floats = P.column_blocks > 1 ? (size_t)4 * P.column_blocks * dim : 0;
    P.gate_floats = P.gate_rows_shared && P.column_parts > 1 ? (size_t)P.column_strips * dim : 0;
    return P;
}

template <typename T>
void residual_norm_forward(const ResidualNorm& A, T* h, T* y, float* stats, hipStream_t st);
template <typename T>
void residual_norm_backward(const ResidualNorm& A, NormGrads G, int64_t gate_rows, float* scratch, hipStream_t st);

}  // namespace cfh
