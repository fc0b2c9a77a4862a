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
    int64_t strips;
    int32_t parts;           // strips of the rows that share a row of the gate
};

constexpr int NORM_CUS = 256;

struct NormPlan {
    int teams, blocks, parts;
    int64_t segments, strips;
    bool gate_rows_shared;
    size_t column_floats, gate_floats;
};

// Threads of a workgroup: for rows of up to 64 pieces of 16 bytes 256, in teams of 16, 32 or 64 lanes with a piece each; else one team of as
// many wavefronts as there are 64 pieces in a row, up to 16, where lanes take two or four.  A piece per lane is what leaves the backward
// pass, with its column sums, registers for four wavefronts per SIMD.
inline int norm_threads(int64_t dim, int elements) {
    const int64_t pieces = (dim + elements - 1) / elements;
    if (pieces <= 64) return 256;
    return pieces >= 1024 ? 1024 : (int)((pieces + 63) / 64 * 64);
}
inline int norm_teams(int64_t dim, int elements) {
    const int64_t pieces = (dim + elements - 1) / elements;
    return pieces <= 16 ? 16 : pieces <= 32 ? 8 : pieces <= 64 ? 4 : 1;
}

// Strips of rows: as many as there are workgroups at once, but with two rows for each team of a workgroup where there are fewer, and
// none across two rows of the gate.
inline NormPlan norm_plan(int64_t rows, int64_t dim, int elements, int64_t gate_rows) {
    NormPlan P{};
    P.teams = norm_teams(dim, elements);
    P.gate_rows_shared = gate_rows > 0 && gate_rows < rows;
    P.segments = P.gate_rows_shared ? gate_rows : 1;
    const int64_t resident = 1024 / norm_threads(dim, elements), target = NORM_CUS * (resident < 1 ? 1 : resident), span = rows / P.segments;
    int64_t strips = rows / (2 * P.teams);
    strips = strips < 1 ? 1 : strips > target ? target : strips;
    int64_t parts = strips / P.segments;
    if (parts < 1) parts = 1;
    if (parts > span) parts = span > 0 ? span : 1;
    P.parts = (int)parts;
    P.strips = P.segments * parts;
    P.blocks = (int)(P.strips < target ? P.strips : target);
    P.column_floats = P.blocks > 1 ? (size_t)4 * P.blocks * dim : 0;
    P.gate_floats = P.gate_rows_shared && P.parts > 1 ? (size_t)P.strips * dim : 0;
    return P;
}

template <typename T>
void residual_norm_forward(const ResidualNorm& A, T* h, T* y, float* stats, hipStream_t st);
template <typename T>
void residual_norm_backward(const ResidualNorm& A, NormGrads G, int64_t gate_rows, float* scratch, hipStream_t st);

}  // namespace cfh
