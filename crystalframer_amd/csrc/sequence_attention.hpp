// Attention between the sequences of a batch and those of another, or the same, batch (cross_attention, relative_attention):
//
//   t_ij = scale q_i . k_j + table[bucket_of[j - i - shift]],   P_ij = exp(t_ij - m_i) / l_i,   o_i = sum_j P_ij v_j
//   D_i = do_i . o_i,   ds_ij = P_ij (do_i . v_j - D_i)
//   dv_j = sum_i P_ij do_i,   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dtable[b] = sum over bucket b of ds_ij
//
// All products are matrix instructions of 32 x 32 results, 16 terms deep.  A result has its column in the lane (l % 32) and 16 of its
// rows in the lane's registers: rows 8 (r / 4) + 4 (l / 32) + r % 4.  The scores are made transposed
// where sums over keys follow (rows: keys, columns: queries), and upright where sums over queries follow: either way the probabilities
// are, register by register, the right operand of the product that follows, whose terms may come in any order as long as the left
// operand has them in the same one.  That operand is the transpose of a tile in LDS (ds_read_b64_tr_b16).
// Statistics of a row, its largest score and its sum, then live in one lane (two: the halves of the wavefront share a column).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

#include "element_types.hpp"
#include "sequence_attention_args.hpp"
#include "wave_reduce.hpp"

namespace cfh {
namespace attention {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float NONE = -__builtin_inff();

// ---- operands: 8 terms per lane, 16 per step -------------------------------------------------------------------------------------
template <typename T> struct Operand;
template <> struct Operand<bf16> {
    typedef bf16 Eight __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 product(Eight a, Eight b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Operand<f16> {
    typedef f16 Eight __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 product(Eight a, Eight b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
// float32: three bfloat16 parts hold a value's 24 bits (each what the ones before leave, to the nearest), and six products of parts, from the
// small ones on, hold theirs to 2^-24 (m l and l m are left out): 192 cycles where float32's own instruction takes 512.  An infinity becomes NaN.
template <> struct Operand<float> {
    typedef Operand<bf16>::Eight Part;
    struct Eight { Part h, m, l; };
    static __device__ __forceinline__ f32x16 product(const Eight& a, const Eight& b, f32x16 c) {
        c = Operand<bf16>::product(a.l, b.h, c);
        c = Operand<bf16>::product(a.h, b.l, c);
        c = Operand<bf16>::product(a.m, b.m, c);
        c = Operand<bf16>::product(a.m, b.h, c);
        c = Operand<bf16>::product(a.h, b.m, c);
        return Operand<bf16>::product(a.h, b.h, c);
    }
    // The same with a sum of its own for what is small: an addition of a matrix instruction cuts what lies below its sum's last place, always
    // towards 0, and a row's ds then have a sum of one sign.  For do . v in the backward pass, whose errors a wide bucket of the table
    // adds up over all rows (10 buckets to distance 383, 551 positions, 96 channels: gradient off by 3.8e-6 -> 5e-7 of its size, at 1 % of the time).
    static __device__ __forceinline__ f32x16 product(const Eight& a, const Eight& b, f32x16 c, f32x16& small) {
        small = Operand<bf16>::product(a.l, b.h, small);
        small = Operand<bf16>::product(a.h, b.l, small);
        small = Operand<bf16>::product(a.m, b.m, small);
        small = Operand<bf16>::product(a.m, b.h, small);
        small = Operand<bf16>::product(a.h, b.m, small);
        return Operand<bf16>::product(a.h, b.h, c);
    }
};
template <typename T> using Eight = typename Operand<T>::Eight;

template <int N>
__device__ __forceinline__ void split(const float (&x)[N], bf16* h, bf16* m, bf16* l) {
#pragma unroll
    for (int n = 0; n < N; n++) {
        h[n] = from_float<bf16>(x[n]);
        const float y = x[n] - to_float(h[n]);
        m[n] = from_float<bf16>(y);
        l[n] = from_float<bf16>(y - to_float(m[n]));
    }
}
__device__ __forceinline__ Eight<float> in_parts(const float (&x)[8]) {
    bf16 h[8], m[8], l[8];
    split(x, h, m, l);
    Eight<float> y;
#pragma unroll
    for (int n = 0; n < 8; n++) y.h[n] = h[n], y.m[n] = m[n], y.l[n] = l[n];
    return y;
}
// Registers 8 s ... 8 s + 7 of a result, rounded to T (half a step each: 2^-8, 2^-11 of the value; float32 stays), as an operand of step s.
template <typename T>
__device__ __forceinline__ Eight<T> rounded(const f32x16& x, int s) {
    if constexpr (sizeof(T) == 4) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = x[8 * s + e];
        return in_parts(y);
    } else {
        Eight<T> y;
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = from_float<T>(x[8 * s + e]);
        return y;
    }
}
template <typename T>
__device__ __forceinline__ float value(const Eight<T>& x, int e) {
    if constexpr (sizeof(T) == 4) return to_float(x.h[e]) + (to_float(x.m[e]) + to_float(x.l[e]));
    else return to_float(x[e]);
}
// Row of register r of a result, without the lane's 4 (l / 32).
__device__ __forceinline__ constexpr int result_row(int r) { return 8 * (r / 4) + r % 4; }

// What float16's range takes: powers of a running row, which reach 2^8 (see Running), are lifted by 2^6 and probabilities by 2^15 before
// they are rounded, so that a term is lost only below 2^-31 of the row's largest, or 2^-40.  A gradient of scores has no bound: it is
// multiplied by a power of two for each column, which brings the column's largest so far to 2^14 (Scaled).
template <typename T> constexpr bool NARROW = std::is_same<T, f16>::value;
template <typename T> constexpr float POWER_LIFT = NARROW<T> ? 6.0f : 0.0f;
template <typename T> constexpr float P_LIFT = NARROW<T> ? 15.0f : 0.0f;

// ---- tiles in LDS: rows of DP channels in pieces of 16 bytes, whose places are exchanged by the row so that 16 rows of one piece, and
// the pieces of one transposed read, lie in different banks (conflicts counted: in up to 0.7 % of few_kernel's cycles, none elsewhere) ----
// A lane's address is made once per tile; what changes inside a tile is exclusive-ored into it or lies in the instruction's offset, which
// leaves registers to the sums.  Tiles begin at multiples of their rows' length.
typedef __attribute__((address_space(3))) char lds_char;
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(lds_char*)p; }
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at) { return *reinterpret_cast<__attribute__((address_space(3))) const V*>(at); }

// Channels of a row in LDS, for heads of up to DC (a multiple of 16).
constexpr int pitch(int dc) { return dc <= 32 ? 32 : dc <= 64 ? 64 : 128; }
template <typename T, int DP>
struct Tile {
    static constexpr int E = 16 / sizeof(T), PIECES = DP / E;           // in memory
    static constexpr int ROW = DP * 2, PLANES = sizeof(T) == 4 ? 3 : 1;  // in LDS: float32 as three tiles of parts
    static constexpr int bytes(int rows) { return rows * ROW * PLANES; }
    static __device__ __forceinline__ constexpr int mixed(int row) {
        if (DP == 128) return (row & 3) << 2 | (row >> 2 & 3);
        if (DP == 64) return (row >> 1 & 1) << 2 | (row >> 2 & 3);
        return row >> 2 & 3;
    }
    static __device__ __forceinline__ int place(int row, int piece) { return row * ROW + ((piece ^ mixed(row)) << 4); }
    // The lane's part of an address for rows() and columns().
    static __device__ __forceinline__ uint32_t rows_at(int lane) { return place(lane & 31, lane >> 5); }
    static __device__ __forceinline__ uint32_t columns_at(int lane) {
        return place(4 * (lane >> 5) + (lane & 15) / 4, 2 * (lane >> 4 & 1) + (lane & 3) / 2) + (lane & 1) * 8;
    }
    template <typename U>
    static __device__ __forceinline__ Eight<U> transposed(uint32_t at, int base, int d) {
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>((at ^ d << 6) + base * ROW));
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>((at ^ (d << 6 | 32)) + (base + 8) * ROW));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        return __builtin_bit_cast(Eight<U>, s16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]});
    }
    // Channels 16 step + 8 (l / 32) ... of row base + l % 32 of a tile of ROWS rows.
    template <int ROWS>
    static __device__ __forceinline__ Eight<T> rows(uint32_t at, int base, int step) {
        const uint32_t a = (at ^ step << 5) + base * ROW;
        if constexpr (sizeof(T) == 2) {
            return lds_read<Eight<T>>(a);
        } else {
            typedef Operand<float>::Part Part;
            return {lds_read<Part>(a), lds_read<Part>(a + ROWS * ROW), lds_read<Part>(a + 2 * ROWS * ROW)};
        }
    }
    // Channel 32 d + l % 32 of rows base + 8 (e / 4) + 4 (l / 32) + e % 4.
    template <int ROWS>
    static __device__ __forceinline__ Eight<T> columns(uint32_t at, int base, int d) {
        if constexpr (sizeof(T) == 2) return transposed<T>(at, base, d);
        else return {transposed<bf16>(at, base, d), transposed<bf16>(at, base + ROWS, d), transposed<bf16>(at, base + 2 * ROWS, d)};
    }
};

// ---- rows in memory ------------------------------------------------------------------------------------------------------------------
// Rows lie at multiples of 16 bytes, apart from one another, and are read as pieces of a buffer that ends behind the last row that is
// there: what is beyond comes back as 0, without a branch.  (A last piece that the row's channels do not fill is filled with zeros in memory.)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int BEYOND = 0x40000000;      // behind any buffer here
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* at, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(at), 0, bytes, 0x00027000);
}
// 16 bytes of a row from channel `from` on; channels that the row does not have are 0.
template <typename T>
__device__ __forceinline__ u32x4 elements_of(const T* row, int from, int dim) {
    constexpr int E = 16 / sizeof(T);
    T e[E];
#pragma unroll
    for (int n = 0; n < E; n++) e[n] = from + n < dim ? row[from + n] : T(0);
    u32x4 x;
    __builtin_memcpy(&x, e, 16);
    return x;
}
// Operands of all steps straight from memory: channels 16 step + 8 (l / 32) ... of the lane's row.  `whole`: of rows as above.
template <typename T, int DC>
__device__ __forceinline__ void row_operands(Eight<T> (&y)[DC / 16], const T* row, bool there, int dim, bool whole, int lane) {
    constexpr int E = 16 / sizeof(T), EACH = sizeof(T) / 2;
    u32x4 x[DC / 16 * EACH];
#pragma unroll
    for (int n = 0; n < DC / 16 * EACH; n++) x[n] = u32x4{0, 0, 0, 0};
    if (there) {
        const int first = 8 * (lane >> 5);
#pragma unroll
        for (int n = 0; n < DC / 16 * EACH; n++) {
            const int from = 16 * (n / EACH) + first + n % EACH * E;
            if (whole) {
                if (from < dim) x[n] = *reinterpret_cast<const u32x4*>(row + from);
            } else {
                x[n] = elements_of<T>(row, from, dim);
            }
        }
    }
    if constexpr (sizeof(T) == 2) {
        __builtin_memcpy(y, x, sizeof(x));
    } else {
#pragma unroll
        for (int c = 0; c < DC / 16; c++) {
            float e[8];
            __builtin_memcpy(e, x + 2 * c, 32);
            y[c] = in_parts(e);
        }
    }
}

// Waits for operands here.  (Left to their first use, in the loop, the wait would also be for the tile that was asked for last.)
template <typename T, int N>
__device__ __forceinline__ void settle(Eight<T> (&y)[N]) {
#pragma unroll
    for (int n = 0; n < N; n++) {
        if constexpr (sizeof(T) == 2) asm volatile("" : "+v"(y[n]));
        else asm volatile("" : "+v"(y[n].h), "+v"(y[n].m), "+v"(y[n].l));
    }
}

// Which of the next keys are there: a bit for each, of the mask's bytes on their way (lane l: key l), or of their number.
struct KeyBits {
    uint32_t byte = 0;
    int left = 0;
    __device__ __forceinline__ void load(const uint8_t* mask, int left_, int lane) {
        left = left_;
        if (mask) byte = __builtin_amdgcn_raw_buffer_load_b8(buffer(mask, left < 0 ? 0 : left), lane, 0, 0);
    }
    __device__ __forceinline__ uint64_t get(const uint8_t* mask) const {
        if (mask) return __ballot((byte & 255) != 0);
        return left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
    }
};

// ROWS rows on their way into a tile through the registers of THREADS lanes.  A row that is not there is 0 in LDS: what memory holds
// in its place, infinities and NaN among it, meets no product.
template <typename T, int DP, int ROWS, int THREADS, int HOW = 0>
struct Staged {
    using L = Tile<T, DP>;
    static constexpr int ALL = ROWS * L::PIECES, EACH = (ALL + THREADS - 1) / THREADS, EVERY = THREADS / L::PIECES;
    static_assert(THREADS % L::PIECES == 0, "a lane has one piece of several rows");
    u32x4 x[EACH];
    __device__ __forceinline__ void load(const T* first, int64_t stride, int there, int dim, int thread) {
        const int row = thread / L::PIECES, piece = thread % L::PIECES;
        const int rows = there < ROWS ? there : ROWS, step = (int)stride * (int)sizeof(T), last = (dim + L::E - 1) / L::E * 16;
        const auto from = buffer(first, rows <= 0 ? 0 : (rows - 1) * step + last);
        const int at = piece * 16 < last && row < ROWS ? row * step + piece * 16 : BEYOND;
#pragma unroll
        for (int n = 0; n < EACH; n++) x[n] = __builtin_amdgcn_raw_buffer_load_b128(from, at + n * EVERY * step, 0, HOW);
    }
    // rows whose bit is 0 are not there
    __device__ __forceinline__ void store(char* tile, int thread, uint64_t bits = ~0ull) const {
        const int row = thread / L::PIECES, piece = thread % L::PIECES;
        const bool whole = bits == ~0ull;
#pragma unroll
        for (int n = 0; n < EACH; n++) {
            const int r = row + n * EVERY;
            if (ALL % THREADS != 0 && r >= ROWS) continue;
            u32x4 y = x[n];
            if (!whole) y &= (uint32_t)((int64_t)(bits << (63 - (r & 63))) >> 63);      // all bits of the row's
            if constexpr (sizeof(T) == 2) {
                *reinterpret_cast<u32x4*>(tile + L::place(r, piece)) = y;
            } else {      // half a piece of each part
                typedef bf16 Four __attribute__((ext_vector_type(4)));
                float e[4];
                bf16 part[3][4];
                __builtin_memcpy(e, &y, 16);
                split(e, part[0], part[1], part[2]);
#pragma unroll
                for (int a = 0; a < 3; a++)
                    *reinterpret_cast<Four*>(tile + a * ROWS * L::ROW + L::place(r, piece / 2) + piece % 2 * 8) =
                        Four{part[a][0], part[a][1], part[a][2], part[a][3]};
            }
        }
    }
};

// Four neighbouring channels of a row (from: a multiple of 4).
template <typename T>
__device__ __forceinline__ void put_four(T* row, int from, int dim, f32x4 x) {
    if ((dim & 3) == 0) {
        if (from >= dim) return;
        typedef T Four __attribute__((ext_vector_type(4)));
        Four y;
#pragma unroll
        for (int n = 0; n < 4; n++) y[n] = from_float<T>(x[n]);
        *reinterpret_cast<Four*>(row + from) = y;
    } else {
#pragma unroll
        for (int n = 0; n < 4; n++)
            if (from + n < dim) row[from + n] = from_float<T>(x[n]);
    }
}

// The order of what stands before it in a block: operands are read from LDS `AHEAD` products before the one that takes them, which is
// longer than a read takes.  (Left alone, a read is followed by the wait for it.)  EACH reads to a product.
template <int PRODUCTS, int AHEAD, int EACH>
__device__ __forceinline__ void reads_ahead() {
    constexpr int first = AHEAD < PRODUCTS ? AHEAD : PRODUCTS;
    __builtin_amdgcn_sched_group_barrier(0x100, first * EACH, 0);
#pragma unroll
    for (int n = 0; n < PRODUCTS - first; n++) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, first, 0);
}

// An output and, for the backward pass, what its rounding to 16 bits left (rounded to them in turn): D, the sum of do . o, then has an
// error of 2^-16 of its terms (float16: 2^-22) instead of 2^-8 (2^-11), which a row's ds have in common and its sums over keys would keep.
template <typename T>
__device__ __forceinline__ void put_output(T* out, T* rest, int64_t row, int from, int dim, f32x4 x) {
    put_four<T>(out + row * dim, from, dim, x);
    if constexpr (sizeof(T) == 2) {
        if (rest) put_four<T>(rest + row * dim, from, dim, f32x4{x[0] - to_float(from_float<T>(x[0])), x[1] - to_float(from_float<T>(x[1])),
                                                                  x[2] - to_float(from_float<T>(x[2])), x[3] - to_float(from_float<T>(x[3]))});
    }
}

// ---- which rows a workgroup has --------------------------------------------------------------------------------------------------------
struct Span {
    int64_t first;      // row of the sequence's first position among all rows
    int64_t batch;      // index of the sequence in tensors with a batch dimension
    int there, rows;    // positions; rows to write (those that are no position get 0)
};
__device__ __forceinline__ int64_t between(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }

// Sequence b of a batch; packed sequence number `batch` is what lies behind the last one.
__device__ __forceinline__ Span span_of(const int64_t* starts, const int64_t* sizes, int64_t rows, int packed, int batch, int b) {
    Span s;
    if (packed) {
        const int64_t lo = b == 0 ? 0 : between(starts[b], 0, rows), hi = b == batch ? rows : between(starts[b + 1], lo, rows);
        s.first = lo;
        s.batch = 0;
        s.rows = (int)(hi - lo);
        s.there = b == batch ? 0 : s.rows;
    } else {
        s.first = (int64_t)b * rows;
        s.batch = b;
        s.rows = (int)rows;
        s.there = sizes ? (int)between(sizes[b], 0, rows) : (int)rows;
    }
    return s;
}
// Sequence and first row in it of slot w; false: none.
__device__ __forceinline__ bool find_slot(const int64_t* starts, int64_t rows, int packed, int batch, int tile, int64_t w, int lane, int& b, int& from) {
    if (!packed) {
        const int per = (int)((rows + tile - 1) / tile);
        b = (int)(w / per);
        from = (int)(w - (int64_t)b * per) * tile;
        return b < batch;
    }
    auto base = [&](int n) { return (n == 0 ? 0 : (int64_t)((uint32_t)between(starts[n], 0, rows) / (uint32_t)tile)) + n; };
    int lo = 0, n = batch + 1;      // the last of n from lo on whose first slot is not behind w
    while (n > 1) {
        const int step = (n + 63) / 64, probe = lane * step;
        const bool before = probe < n && base(lo + probe) <= w;
        const int count = __popcll(__ballot(before));
        const int skip = (count > 0 ? count - 1 : 0) * step;
        lo += skip;
        n = n - skip < step ? n - skip : step;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    b = lo;
    const int64_t at = (w - base(lo)) * (int64_t)tile;
    if (at < 0 || at > rows) return false;
    from = (int)at;
    return true;
}
// Head and slot of a workgroup (false: none).  Workgroups that follow one another on one of the 8 dies share what its cache holds: the
// tiles of a head.  Causal tiles differ in their work: a die takes its sequences' and heads' longest ones first.
__device__ __forceinline__ bool workgroup_item(int64_t id, int64_t slots, int heads, const SequenceAttention& A, bool last_first, int& head, int64_t& slot) {
    const int64_t count = slots * heads, pairs = (int64_t)A.batch * heads;
    if (A.causal && !A.packed && (pairs & 7) == 0) {
        const int64_t mine = pairs / 8, tiles = slots / A.batch, local = id >> 3, pair = (id & 7) * mine + local % mine;
        int64_t tile = local / mine;
        if (tile >= tiles) return false;
        if (last_first) tile = tiles - 1 - tile;
        head = (int)(pair / A.batch);
        slot = (pair - (int64_t)head * A.batch) * tiles + tile;
        return true;
    }
    const int64_t at = (id & 7) * ((count + 7) / 8) + (id >> 3);
    if (at >= count) return false;
    head = (int)(at / slots);
    slot = at - head * slots;
    return true;
}

template <typename T>
__device__ __forceinline__ const T* row_start(const AttentionRows& r, const Span& s, int packed, int head) {
    return static_cast<const T*>(r.at) + (packed ? s.first * r.row : s.batch * r.batch) + head * r.head;
}
// What to add to a query's position for the key's that is its own.  Causal: keys behind the last query's are seen by none, and not there.
__device__ __forceinline__ int shift_of(const SequenceAttention& A, const Span& q, Span& k) {
    const int shift = A.last ? k.there - q.there : 0;
    if (A.causal) k.there = max(0, min(k.there, q.there + shift));
    return shift;
}

// ---- scores ----------------------------------------------------------------------------------------------------------------------------
// A score t is what the product sums up to, q . k + bias / scale, and exp2((t - m) rate) its power.  The bias costs no instruction of its
// own that way: near ones are what the product's sum begins with, and one that is the same for a whole tile goes into m.  float32 takes
// the difference to the maximum before anything is rounded, 16-bit types in one instruction with the factor.
template <typename T>
struct Score {
    static constexpr bool WIDE = sizeof(T) == 4;
    float rate;
    __device__ __forceinline__ explicit Score(float scale) : rate(scale * LOG2E) {}
    // `shift` = -m rate
    __device__ __forceinline__ float power(float t, float m, float shift) const {
        return __builtin_amdgcn_exp2f(WIDE ? (t - m) * rate : __builtin_fmaf(t, rate, shift));
    }
};

// Biases of one head by relative position in LDS, from -reach - MARGIN to reach + MARGIN.
constexpr int MARGIN = ATTENTION_MARGIN;
// (No branch but the one on the table's type, which is the same for all: loads of several entries are on their way together.)
template <typename T>
__device__ __forceinline__ float table_entry(const SequenceAttention& A, int at, int head) {
    const int b = A.bucket_of[at];
    const bool real = (unsigned)b < (unsigned)A.buckets;
    const int64_t n = (int64_t)(real ? b : 0) * A.heads + head;
    const float x = A.table_float ? static_cast<const float*>(A.table)[n] : to_float(static_cast<const T*>(A.table)[n]);
    // (beyond 2^16, where a mask's lowest value would end a float32's range with 1 / scale, all are as far away; infinities stay)
    const float most = 65536.0f, size = fabsf(x);
    return real ? size > most && size < -NONE ? copysignf(most, x) : x : 0.0f;
}
__device__ __forceinline__ int clamped(int r, int reach) { return (r < -reach ? -reach : r > reach ? reach : r) + reach; }
template <typename T>
__device__ __forceinline__ void fill_line(const SequenceAttention& A, int head, float* line, int thread, int threads) {
    const float by = 1.0f / A.scale;
    for (int n = thread; n <= 2 * (A.reach + MARGIN); n += threads)
        line[n] = table_entry<T>(A, clamped(n - A.reach - MARGIN, A.reach), head) * by;
}

// A bias that is the same for a whole tile goes into the maximum, unless it is plus infinity or NaN: it would reach the keys of the tile
// that are not there, or that a row does not see, so that the scores begin with it as with a near one, and these keys' are dropped.
__device__ __forceinline__ bool far_in_scores(float far) { return !(far < -NONE); }
__device__ __forceinline__ bool any_far_in_scores(const float* line, int reach) {
    return __any(far_in_scores(line[0]) || far_in_scores(line[2 * (reach + MARGIN)]));
}

__device__ __forceinline__ float other_half_max(float x) { float a, b; swap32(x, a, b); return fmaxf(a, b); }
__device__ __forceinline__ float other_half_sum(float x) { float a, b; swap32(x, a, b); return a + b; }

// Running maximum, sum and weighted sum of one column.  The maximum that the powers are relative to follows the true one when that is
// more than 2^8 ahead: the sums are scaled anew in few tiles only, and no power is above 2^8.
template <int ND>
struct Running {
    float m = NONE, l = 0.0f;
    f32x16 o[ND];
    __device__ __forceinline__ Running() {
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
    }
    __device__ __forceinline__ void meet(float top, float rate) {
        const bool ahead = (top - m) * rate > 8.0f;      // (no for -inf against -inf)
        if (!__any(ahead)) return;
        const float by = ahead ? __builtin_amdgcn_exp2f((m - top) * rate) : 1.0f;
        m = ahead ? top : m;
        l *= by;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] *= by;
    }
    __device__ __forceinline__ float base() const { return m == NONE ? 0.0f : m; }
};

// Gradients of scores on their way into a product whose sums `sum` are per column (see NARROW).
template <typename T, int ND>
struct Scaled {
    float by = 1.0f;
    bool met = false;
    __device__ __forceinline__ void meet(f32x16& ds, f32x16* sum) {
        if (!NARROW<T>) return;
        float top = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; r++) top = fmaxf(top, fabsf(ds[r]));
        top = other_half_max(top);
        const bool ahead = top < __builtin_inff() && (met ? top * by >= 32768.0f : top > 0.0f);
        if (__any(ahead)) {
            const int e = (int)(__float_as_uint(top) >> 23);                                  // 2^(e - 127) <= top
            const int to = 2 * 127 + 14 - e;
            const float next = ahead ? __uint_as_float((uint32_t)(to > 253 ? 253 : to < 1 ? 1 : to) << 23) : by;
            const float change = met ? next / by : 1.0f;                                      // (nothing but 0 is there before)
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int r = 0; r < 16; r++) sum[d][r] *= change;
            by = next;
            met = met || ahead;
        }
#pragma unroll
        for (int r = 0; r < 16; r++) ds[r] *= by;
    }
    __device__ __forceinline__ float back() const { return NARROW<T> ? 1.0f / by : 1.0f; }
};

// Without the keys (rows) that are not there: `gone` holds 0 for one that is and all bits for others, in LDS.  (One instruction for a
// score, as an addition of minus infinity would be; but that leaves a bias of plus infinity or NaN a NaN.)
__device__ __forceinline__ void drop_keys(f32x16& s, uint32_t gone, int lane) {
    uint32_t none = __float_as_uint(NONE);
    asm("" : "+s"(none));                  // (with a known number the choice of bits becomes two instructions)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
        const u32x4 x = lds_read<u32x4>(gone + (result_row(r) + 4 * (lane >> 5)) * 4);
#pragma unroll
        for (int e = 0; e < 4; e++) s[r + e] = __uint_as_float((x[e] & none) | (~x[e] & __float_as_uint(s[r + e])));
    }
}
// Without the rows behind number `last` of the tile.
__device__ __forceinline__ void drop_behind(f32x16& s, int last, int lane) {
    const int mine = last - (lane >> 5) * 4;
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] = result_row(r) <= mine ? s[r] : NONE;
}
// For keys in columns: without the queries (rows) before number `first`.
__device__ __forceinline__ void drop_before(f32x16& s, int first, int lane) {
    const int mine = first - (lane >> 5) * 4;
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] = result_row(r) >= mine ? s[r] : NONE;
}
// Writes what drop_keys() reads, for COUNT keys.
template <int COUNT>
__device__ __forceinline__ void put_keys(uint32_t* at, uint64_t bits, int thread) {
    if (thread < COUNT) at[thread] = bits >> thread & 1 ? 0u : ~0u;
}
template <int COUNT>
__device__ __forceinline__ bool all_there(uint64_t bits) { return COUNT == 64 ? bits == ~0ull : (uint32_t)bits == ~0u; }

// ---- few queries: the keys in parts -----------------------------------------------------------------------------------------------------
// 32 columns are (query, head of one key head): single tokens of shared heads fill them together.  Every wavefront goes through keys of
// its own, in tiles of 32 that it alone puts into LDS and reads (no barrier in the loop), and the wavefronts' sums are joined at the end;
// so are, by combine_parts, those of `splits` workgroups.  Bound by the bytes of keys and values for single tokens; PAST: these go past the
// caches (see attention_plan).
__device__ __forceinline__ int heads_at_once(int share) { return share < 32 ? share : 32; }

template <typename T, int DP, int NW>
struct FewLds {
    static constexpr int TILE = Tile<T, DP>::bytes(32), SUM = 32 * (DP + 4) * 4;
    static constexpr int EACH = 2 * TILE > SUM ? 2 * TILE : SUM;
    alignas(512) char wave[NW][(EACH + 511) / 512 * 512];
    float m[NW][32], l[NW][32];
    uint32_t gone[NW][32];
};

template <typename T, int DC, int NW, bool BIAS, bool PAST>
__global__ __launch_bounds__(NW * 64, (sizeof(T) == 2 && NW == 4 ? 2 : 1)) void few_kernel(SequenceAttention A, T* out, T* rest, float* stats, float* part_o, float* part_ml, int splits) {
    constexpr int DP = pitch(DC), ND = (DC + 31) / 32, KEYS = 32;
    using L = Tile<T, DP>;
    __shared__ FewLds<T, DP, NW> S;
    // (an aligned attribute of the variable's own would take the place of the type's)
    static_assert(__alignof__(S) % L::ROW == 0 && sizeof(S.wave[0]) % L::ROW == 0 && L::bytes(32) % L::ROW == 0, "tiles begin at multiples of their rows' length");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int at_once = heads_at_once(A.share), groups = (A.share + at_once - 1) / at_once, tile = 32 / at_once;
    int b, i0;
    if (!find_slot(A.q_starts, A.q_rows, A.packed, A.batch, tile, blockIdx.x, lane, b, i0)) return;
    const Span q = span_of(A.q_starts, A.q_sizes, A.q_rows, A.packed, A.batch, b);
    if (i0 >= q.rows) return;
    Span k{0, 0, 0, 0};
    if (!A.packed || b < A.batch) k = span_of(A.k_starts, A.k_sizes, A.k_rows, A.packed, A.batch, b);
    const int kh = blockIdx.y / groups, h0 = kh * A.share + (blockIdx.y % groups) * at_once;
    const int column = lane & 31, i = i0 + column / at_once, h = h0 + column % at_once;
    const bool mine = column / at_once < tile && i < q.there && h < (kh + 1) * A.share;
    const int shift = shift_of(A, q, k);
    const Score<T> score(A.scale);

    // the tiles of this split that any of the queries sees
    const int i_last = min(i0 + tile, q.there) - 1;
    int seen = i0 < q.there ? k.there : 0;
    if (A.causal) seen = min(seen, i_last + shift + 1);
    const int tiles = seen > 0 ? (seen + 31) / 32 : 0;
    // (padded sequences: parts of one length, so that long ones take more workgroups, not longer ones)
    const int part = A.packed ? (tiles + splits - 1) / splits : (int)((A.k_rows + 32LL * splits - 1) / (32LL * splits));
    const int first = min(tiles, (int)blockIdx.z * part), end = min(tiles, first + part);

    Eight<T> qf[DC / 16];
    const T* const q_row = row_start<T>(A.q, q, A.packed, mine ? h : 0) + (mine ? i : 0) * A.q.row;
    row_operands<T, DC>(qf, q_row, mine, A.dim, true, lane);
    const T* const k_at = row_start<T>(A.k, k, A.packed, kh);
    const T* const v_at = row_start<T>(A.v, k, A.packed, kh);
    const uint8_t* const mask = A.mask ? A.mask + k.first : nullptr;
    const float by = 1.0f / A.scale;
    float far[2] = {0.0f, 0.0f};
    if (BIAS) {
        const int head = mine ? h : 0;
        far[0] = table_entry<T>(A, 0, head) * by;
        far[1] = table_entry<T>(A, 2 * A.reach, head) * by;
    }
    char* const kt = S.wave[wave];
    char* const vt = kt + FewLds<T, DP, NW>::TILE;
    const uint32_t kr = lds_address(kt) + L::rows_at(lane), vc = lds_address(vt) + L::columns_at(lane);
    Running<ND> sum;
    Staged<T, DP, 32, 64, PAST ? 2 : 0> kx, vx;
    KeyBits bits;
    auto fetch = [&](int n) {
        const int j0 = n * 32;
        bits.load(mask ? mask + j0 : nullptr, min(k.there - j0, 32), lane);
        kx.load(k_at + j0 * A.k.row, A.k.row, k.there - j0, A.dim, lane);
        vx.load(v_at + j0 * A.v.row, A.v.row, k.there - j0, A.dim, lane);
    };
    if (first + wave < end) fetch(first + wave);
    extern __shared__ float line[];        // (heads at once, entries) where few_line() says so
    const int entries = 2 * (A.reach + MARGIN) + 1;
    const bool lines = BIAS && few_line(at_once, A.reach);
    if (lines) {
        if (first < end && first * 32 - i_last - shift < A.reach && end * 32 - 1 - i0 - shift > -A.reach)
            for (int n = threadIdx.x; n < at_once * entries; n += NW * 64) {
                const int g = n / entries, head = h0 + g < (kh + 1) * A.share ? h0 + g : h0;
                line[n] = table_entry<T>(A, clamped(n - g * entries - A.reach - MARGIN, A.reach), head) * by;
            }
        __syncthreads();
    }
    settle<T>(qf);
    for (int n = first + wave; n < end; n += NW) {
        const int j0 = n * 32;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const uint32_t there = (uint32_t)bits.get(mask);
        const uint64_t rows = mask ? there | ~0xffffffffull : ~0ull;      // (rows behind the last are 0 already)
        if (!all_there<32>(there)) put_keys<32>(S.gone[wave], there, lane);
        kx.store(kt, lane, rows);
        vx.store(vt, lane, rows);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (n + NW < end) fetch(n + NW);
        f32x16 s;
        const int low = j0 - i_last - shift, high = j0 + 31 - i0 - shift;      // relative positions of the tile
        const bool near = BIAS && low < A.reach && high > -A.reach;
        if (near && lines) {
            const float* const at = line + column % at_once * entries + (j0 + 4 * half - i - shift + A.reach + MARGIN);
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = at[result_row(r)];
        } else if (near) {
            const int r0 = j0 + 4 * half - i - shift;
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = mine ? table_entry<T>(A, clamped(r0 + result_row(r), A.reach), h) * by : 0.0f;
        } else {
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = BIAS && far_in_scores(far[low >= A.reach]) ? far[low >= A.reach] : 0.0f;
        }
#pragma unroll
        for (int c = 0; c < DC / 16; c++) s = Operand<T>::product(L::template rows<KEYS>(kr, 0, c), qf[c], s);
        if (!all_there<32>(there)) drop_keys(s, lds_address(S.gone[wave]), lane);
        if (A.causal && high > 0) drop_behind(s, i + shift - j0, lane);
        const float flat = BIAS && !near && !far_in_scores(far[low >= A.reach]) ? far[low >= A.reach] : 0.0f;
        float top = s[0];
#pragma unroll
        for (int r = 1; r < 16; r++) top = fmaxf(top, s[r]);
        sum.meet(other_half_max(top) + flat, score.rate);
        const float m = sum.base() - flat, off = POWER_LIFT<T> - m * score.rate;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            s[r] = score.power(s[r], m, off);
            sum.l += s[r];
        }
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const Eight<T> p = rounded<T>(s, c);
#pragma unroll
            for (int d = 0; d < ND; d++) sum.o[d] = Operand<T>::product(L::template columns<KEYS>(vc, 16 * c, d), p, sum.o[d]);
        }
    }
    // the wavefronts' sums, side by side in LDS
    __syncthreads();
    sum.l = other_half_sum(sum.l);
    float* const mine_o = reinterpret_cast<float*>(S.wave[wave]);
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<f32x4*>(mine_o + column * (DP + 4) + 32 * d + result_row(r) + 4 * half) =
                f32x4{sum.o[d][r], sum.o[d][r + 1], sum.o[d][r + 2], sum.o[d][r + 3]};
    if (half == 0) {
        S.m[wave][column] = sum.m;
        S.l[wave][column] = sum.l;
    }
    __syncthreads();
    const int fours = (A.dim + 3) / 4;
    for (int n = threadIdx.x; n < 32 * fours; n += NW * 64) {
        const int c = n / fours, from = (n - c * fours) * 4, ci = i0 + c / at_once, ch = h0 + c % at_once;
        if (c / at_once >= tile || ci >= q.rows || ch >= (kh + 1) * A.share) continue;
        float m = NONE, l = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) m = fmaxf(m, S.m[w][c]);
        f32x4 o{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float by = S.m[w][c] == NONE ? 0.0f : __builtin_amdgcn_exp2f((S.m[w][c] - m) * score.rate);
            l += by * S.l[w][c];
            o += by * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(S.wave[w]) + c * (DP + 4) + from);
        }
        if (ci >= q.there) {
            m = NONE;
            l = 0.0f;
            o = f32x4{0, 0, 0, 0};
        }
        const int64_t row = (q.first + ci) * A.heads + ch;
        if (splits > 1) {
            const int64_t rows = (A.packed ? A.q_rows : A.q_rows * A.batch) * A.heads, at = blockIdx.z * rows + row;
            if (m != NONE) *reinterpret_cast<f32x4*>(part_o + at * DP + from) = o;
            if (from == 0) {
                part_ml[2 * at] = m;
                part_ml[2 * at + 1] = l;
            }
            continue;
        }
        const float inverse = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        put_output<T>(out, rest, row, from, A.dim, o * inverse);
        if (stats && from == 0) {
            stats[2 * row] = m == NONE ? -NONE : m;
            stats[2 * row + 1] = inverse * (NARROW<T> ? 0x1p6f : 1.0f);
        }
    }
}

// Joins the splits: 8 rows to a workgroup, 32 lanes to a row.  The lanes look at a part's statistics each, and then all at its sums.
template <typename T, int DC>
__global__ __launch_bounds__(256) void combine_parts(SequenceAttention A, const float* part_o, const float* part_ml, int splits, int64_t rows, T* out,
                                                     T* rest, float* stats) {
    constexpr int DP = pitch(DC);
    const int64_t row = blockIdx.x * 8LL + threadIdx.x / 32;
    const int lane = threadIdx.x & 31, from = lane * 4;
    if (row >= rows) return;
    const Score<T> score(A.scale);
    float m = NONE, l = 0.0f;
    f32x4 o{0, 0, 0, 0};
    for (int z0 = 0; z0 < splits; z0 += 32) {
        float mz = NONE, lz = 0.0f;
        if (z0 + lane < splits) {
            mz = part_ml[2 * ((z0 + lane) * rows + row)];
            lz = part_ml[2 * ((z0 + lane) * rows + row) + 1];
        }
        float top = mz;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 32));
        top = fmaxf(top, m);
        const float old = m == NONE ? 0.0f : __builtin_amdgcn_exp2f((m - top) * score.rate);
        const float by = mz == NONE ? 0.0f : __builtin_amdgcn_exp2f((mz - top) * score.rate);
        float sum = by * lz;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 32);
        l = l * old + sum;
        o *= old;
        m = top;
        const int here = splits - z0 < 32 ? splits - z0 : 32;
#pragma unroll 4
        for (int z = 0; z < here; z++) {
            const float w = __shfl(by, z, 32);
            if (w != 0.0f && from < DP) o += w * *reinterpret_cast<const f32x4*>(part_o + ((z0 + z) * rows + row) * DP + from);
        }
    }
    const float inverse = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    if (from < A.dim) put_output<T>(out, rest, row, from, A.dim, o * inverse);
    if (stats && lane == 0) {
        stats[2 * row] = m == NONE ? -NONE : m;
        stats[2 * row + 1] = inverse * (NARROW<T> ? 0x1p6f : 1.0f);
    }
}

// ---- many queries: tiles of keys shared by the wavefronts of a workgroup ------------------------------------------------------------------
template <typename T>
constexpr int keys_at_once() { return sizeof(T) == 2 ? 64 : 32; }

template <typename T, int DC, int NW, bool BIAS>
__global__ __launch_bounds__(NW * 64, (sizeof(T) == 2 ? 2 : 1)) void tiles_kernel(SequenceAttention A, T* out, T* rest, float* stats, int64_t slots) {
    constexpr int DP = pitch(DC), ND = (DC + 31) / 32;
    using L = Tile<T, DP>;
    constexpr int KEYS = keys_at_once<T>(), TILE = L::bytes(KEYS);
    extern __shared__ __attribute__((aligned(512))) char lds[];
    char* const tiles = lds;                    // two pairs of a tile of keys and one of values
    uint32_t* const keys = reinterpret_cast<uint32_t*>(lds + 4 * TILE);      // which are not there: two times KEYS
    float* const line = reinterpret_cast<float*>(keys + 2 * KEYS);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, column = lane & 31;
    int h;
    int64_t slot;
    if (!workgroup_item(blockIdx.x, slots, A.heads, A, true, h, slot)) return;
    const int kh = h / A.share;
    int b, from;
    if (!find_slot(A.q_starts, A.q_rows, A.packed, A.batch, NW * 32, slot, lane, b, from)) return;
    const Span q = span_of(A.q_starts, A.q_sizes, A.q_rows, A.packed, A.batch, b);
    if (from >= q.rows) return;
    Span k{0, 0, 0, 0};
    if (!A.packed || b < A.batch) k = span_of(A.k_starts, A.k_sizes, A.k_rows, A.packed, A.batch, b);
    const int i0 = from + wave * 32, i = i0 + column;
    const bool mine = i < q.there;
    const int shift = shift_of(A, q, k);
    const Score<T> score(A.scale);
    int seen = from < q.there ? k.there : 0;
    if (A.causal) seen = min(seen, min(from + NW * 32, q.there) + shift);
    const int count = seen > 0 ? (seen + KEYS - 1) / KEYS : 0;

    Eight<T> qf[DC / 16];
    const T* const q_row = row_start<T>(A.q, q, A.packed, h) + (mine ? i : 0) * A.q.row;
    row_operands<T, DC>(qf, q_row, mine, A.dim, true, lane);
    const T* const k_at = row_start<T>(A.k, k, A.packed, kh);
    const T* const v_at = row_start<T>(A.v, k, A.packed, kh);
    const uint8_t* const mask = A.mask ? A.mask + k.first : nullptr;
    Running<ND> sum;
    Staged<T, DP, KEYS, NW * 64> kx, vx;
    KeyBits bits;
    uint64_t there = 0;                         // keys of the tile in LDS
    auto fetch = [&](int n) {
        const int j0 = n * KEYS;
        bits.load(mask ? mask + j0 : nullptr, min(k.there - j0, KEYS), lane);
        kx.load(k_at + j0 * A.k.row, A.k.row, k.there - j0, A.dim, threadIdx.x);
        vx.load(v_at + j0 * A.v.row, A.v.row, k.there - j0, A.dim, threadIdx.x);
    };
    auto put = [&](int n) {
        there = bits.get(mask);
        const uint64_t rows = mask ? there | (KEYS < 64 ? ~0ull << (KEYS & 63) : 0ull) : ~0ull;      // (rows behind the last are 0 already)
        if (!all_there<KEYS>(there)) put_keys<KEYS>(keys + (n & 1) * KEYS, there, threadIdx.x);
        kx.store(tiles + (n & 1) * 2 * TILE, threadIdx.x, rows);
        vx.store(tiles + (n & 1) * 2 * TILE + TILE, threadIdx.x, rows);
    };
    if (count > 0) fetch(0);
    if (BIAS) fill_line<T>(A, h, line, threadIdx.x, NW * 64);
    if (count > 0) put(0);
    settle<T>(qf);
    __syncthreads();
    const bool odd = BIAS && any_far_in_scores(line, A.reach);
    for (int n = 0; n < count; n++) {
        const uint32_t tile = lds_address(tiles) + (n & 1) * 2 * TILE, kr = tile + L::rows_at(lane), vc = tile + TILE + L::columns_at(lane);
        if (n + 1 < count) fetch(n + 1);
        f32x16 s[KEYS / 32];
        const int j0 = n * KEYS, low = j0 - (i0 + 31) - shift, high = j0 + KEYS - 1 - i0 - shift;
        const bool near = BIAS && low < A.reach && high > -A.reach;
        auto products = [&] {
#pragma unroll
            for (int c = 0; c < DC / 16; c++)
#pragma unroll
                for (int u = 0; u < KEYS / 32; u++) s[u] = Operand<T>::product(L::template rows<KEYS>(kr, 32 * u, c), qf[c], s[u]);
            if (sizeof(T) == 2) reads_ahead<DC / 16 * KEYS / 32, 4, 1>();
        };
        const bool side = low >= A.reach, begin = near || (odd && far_in_scores(line[side ? 2 * (A.reach + MARGIN) : 0]));
        if (begin) {
            const float* const at = line + (near ? j0 + 4 * half - i - shift + A.reach + MARGIN : side ? 2 * A.reach + MARGIN : 0);
#pragma unroll
            for (int u = 0; u < KEYS / 32; u++)
#pragma unroll
                for (int r = 0; r < 16; r++) s[u][r] = at[32 * u + result_row(r)];
            products();
        } else {
#pragma unroll
            for (int u = 0; u < KEYS / 32; u++)
#pragma unroll
                for (int r = 0; r < 16; r++) s[u][r] = 0.0f;
            products();
        }
        const float flat = BIAS && !begin ? line[side ? 2 * (A.reach + MARGIN) : 0] : 0.0f;
        if (!all_there<KEYS>(there))
#pragma unroll
            for (int u = 0; u < KEYS / 32; u++) drop_keys(s[u], lds_address(keys + (n & 1) * KEYS + 32 * u), lane);
        if (A.causal && high > 0)
#pragma unroll
            for (int u = 0; u < KEYS / 32; u++) drop_behind(s[u], i + shift - j0 - 32 * u, lane);
        float top = NONE;
#pragma unroll
        for (int u = 0; u < KEYS / 32; u++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[u][r]);
        sum.meet(other_half_max(top) + flat, score.rate);
        const float m = sum.base() - flat, off = POWER_LIFT<T> - m * score.rate;
#pragma unroll
        for (int u = 0; u < KEYS / 32; u++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[u][r] = score.power(s[u][r], m, off);
                sum.l += s[u][r];
            }
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const Eight<T> p = rounded<T>(s[u], c);
#pragma unroll
                for (int d = 0; d < ND; d++) sum.o[d] = Operand<T>::product(L::template columns<KEYS>(vc, 32 * u + 16 * c, d), p, sum.o[d]);
            }
        }
        if (n + 1 < count) put(n + 1);
        __syncthreads();
    }
    if (i >= q.rows) return;
    const float l = other_half_sum(sum.l);
    const float inverse = mine && (l > 0.0f || l != l) ? 1.0f / l : 0.0f;
    const int64_t row = (q.first + i) * A.heads + h;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            f32x4 x{sum.o[d][r], sum.o[d][r + 1], sum.o[d][r + 2], sum.o[d][r + 3]};
            x *= inverse;
            put_output<T>(out, rest, row, 32 * d + result_row(r) + 4 * half, A.dim, mine ? x : f32x4{0, 0, 0, 0});
        }
    if (stats && half == 0) {
        stats[2 * row] = mine && sum.m != NONE ? sum.m : -NONE;
        stats[2 * row + 1] = inverse * (NARROW<T> ? 0x1p6f : 1.0f);
    }
}

// ---- backward: queries' side ---------------------------------------------------------------------------------------------------------------
// Probability of a stored row: exp2((t - m) rate) / l; 16 bits: with 1 / l in the exponent (0 for a row without keys).
template <typename T>
__device__ __forceinline__ float row_shift(const Score<T>& score, float m, float inverse) {
    return sizeof(T) == 4 ? 0.0f : __builtin_amdgcn_logf(inverse) - m * score.rate;
}
template <typename T>
__device__ __forceinline__ float probability(const Score<T>& score, float t, float m, float inverse, float shift) {
    const float p = score.power(t, m, shift);
    return sizeof(T) == 4 ? p * inverse : p;
}

// Sums of a 32 x 32 result over its diagonals: column l of 16 and row 16 a + b meet in place (l - b) of sum a, or of sum a + 1 where that
// is negative.  A shift within 16 lanes that fills with zeros is part of the addition (DPP): two instructions for a register, none of
// them an LDS atomic, of which one takes 94 cycles for a wavefront (16 of them per tile: 330 us where this takes 101, 32 x 512 tokens, 12 heads
// of 64).  Register r is row 8 (r / 4) + r % 4; the 4 of the upper half wavefront are in the place that the sums are added to.
template <int CTRL>
__device__ __forceinline__ float shifted(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
template <int R>
__device__ __forceinline__ void add_diagonal(float s, float (&x)[3]) {
    constexpr int a = result_row(R) / 16, b = result_row(R) % 16;
    if constexpr (b == 0) {
        x[a] += s;
    } else {
        x[a] += shifted<0x100 + b>(s);              // from b lanes further
        x[a + 1] += shifted<0x110 + 16 - b>(s);     // from 16 - b lanes before
    }
}
template <int... R>
__device__ __forceinline__ void add_diagonals(const f32x16& s, float (&x)[3], std::integer_sequence<int, R...>) {
    (add_diagonal<R>(s[R], x), ...);
}

// dq, D, and the table's gradient: scores transposed as in the forward pass.  The gradients of the biases are summed in float32 by
// relative position (for each half wavefront by itself), those of tiles beyond the reach in the lane.
// D comes from a rounded output, so that the ds of a row add up to a small e instead of 0; what lies beyond the reach, where most of
// a long row's probability is, gets its share of -e back (here, or, where a row's keys are in parts, from finish_kernel).
template <typename T, int DC, int NW, bool BIAS>
__global__ __launch_bounds__(NW * 64) void queries_kernel(SequenceAttention A, AttentionGrads G, int64_t slots, int splits) {
    constexpr int DP = pitch(DC), ND = (DC + 31) / 32;
    using L = Tile<T, DP>;
    constexpr int KEYS = 32, TILE = L::bytes(KEYS);
    extern __shared__ __attribute__((aligned(512))) char lds[];
    char* const tiles = lds;
    uint32_t* const keys = reinterpret_cast<uint32_t*>(lds + 4 * TILE);      // which are not there: two times KEYS
    float* const line = reinterpret_cast<float*>(keys + 2 * KEYS);
    const int entries = 2 * (A.reach + MARGIN) + 1;
    float* const sums = line + entries;                         // (2 NW, entries), then two for each wavefront
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, column = lane & 31;
    int h;
    int64_t slot;
    if (!workgroup_item(blockIdx.x, slots, A.heads, A, true, h, slot)) return;
    const int kh = h / A.share, z = blockIdx.y;
    float* const dtable = BIAS && G.dtable ? G.dtable + (((int64_t)h * splits + z) * slots + slot) * A.buckets : nullptr;
    int b, from;
    bool any = find_slot(A.q_starts, A.q_rows, A.packed, A.batch, NW * 32, slot, lane, b, from);
    Span q{0, 0, 0, 0}, k{0, 0, 0, 0};
    if (any) q = span_of(A.q_starts, A.q_sizes, A.q_rows, A.packed, A.batch, b);
    if (!any || from >= q.rows) {
        if (dtable)
            for (int n = threadIdx.x; n < A.buckets; n += NW * 64) dtable[n] = 0.0f;
        return;
    }
    if (!A.packed || b < A.batch) k = span_of(A.k_starts, A.k_sizes, A.k_rows, A.packed, A.batch, b);
    const int i0 = from + wave * 32, i = i0 + column;
    const bool mine = i < q.there;
    const int shift = shift_of(A, q, k);
    const Score<T> score(A.scale);
    int seen = from < q.there ? k.there : 0;
    if (A.causal) seen = min(seen, min(from + NW * 32, q.there) + shift);
    const int whole = seen > 0 ? (seen + KEYS - 1) / KEYS : 0;
    const int first = (int)((int64_t)whole * z / splits), end = (int)((int64_t)whole * (z + 1) / splits);

    const int64_t row = (q.first + i) * A.heads + h;
    Eight<T> qf[DC / 16], gf[DC / 16], of[DC / 16], rf[sizeof(T) == 2 ? DC / 16 : 1];
    row_operands<T, DC>(qf, row_start<T>(A.q, q, A.packed, h) + (mine ? i : 0) * A.q.row, mine, A.dim, true, lane);
    row_operands<T, DC>(gf, row_start<T>(G.go, q, A.packed, h) + (mine ? i : 0) * G.go.row, mine, A.dim, true, lane);
    row_operands<T, DC>(of, static_cast<const T*>(G.out) + (mine ? row : 0) * A.dim, mine, A.dim, A.dim % L::E == 0, lane);
    if constexpr (sizeof(T) == 2) row_operands<T, DC>(rf, static_cast<const T*>(G.rest) + (mine ? row : 0) * A.dim, mine, A.dim, A.dim % L::E == 0, lane);
    float m = -NONE, inverse = 0.0f;
    if (mine) {
        m = G.stats[2 * row];
        inverse = G.stats[2 * row + 1];
    }
    const T* const k_at = row_start<T>(A.k, k, A.packed, kh);
    const T* const v_at = row_start<T>(A.v, k, A.packed, kh);
    const uint8_t* const mask = A.mask ? A.mask + k.first : nullptr;
    if (BIAS) {
        for (int n = threadIdx.x; n < 2 * NW * entries; n += NW * 64) sums[n] = 0.0f;
    }
    float* const own_sums = sums + (2 * wave + half) * entries;
    float far_ds[2] = {0.0f, 0.0f}, far_p[2] = {0.0f, 0.0f}, all_ds = 0.0f;
    f32x16 dq[ND];
    Scaled<T, ND> scaled;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) dq[d][r] = 0.0f;
    Staged<T, DP, KEYS, NW * 64> kx, vx;
    KeyBits bits;
    uint64_t there = 0;                         // keys of the tile in LDS
    auto fetch = [&](int n) {
        const int j0 = n * KEYS;
        bits.load(mask ? mask + j0 : nullptr, min(k.there - j0, KEYS), lane);
        kx.load(k_at + j0 * A.k.row, A.k.row, k.there - j0, A.dim, threadIdx.x);
        vx.load(v_at + j0 * A.v.row, A.v.row, k.there - j0, A.dim, threadIdx.x);
    };
    auto put = [&](int n) {
        there = bits.get(mask);
        const uint64_t rows = mask ? there | (KEYS < 64 ? ~0ull << (KEYS & 63) : 0ull) : ~0ull;      // (rows behind the last are 0 already)
        if (!all_there<KEYS>(there)) put_keys<KEYS>(keys + (n & 1) * KEYS, there, threadIdx.x);
        kx.store(tiles + (n & 1) * 2 * TILE, threadIdx.x, rows);
        vx.store(tiles + (n & 1) * 2 * TILE + TILE, threadIdx.x, rows);
    };
    if (first < end) fetch(first);
    if (BIAS) fill_line<T>(A, h, line, threadIdx.x, NW * 64);
    float D = 0.0f;
#pragma unroll
    for (int s = 0; s < DC / 16; s++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float o = value<T>(of[s], e);
            if constexpr (sizeof(T) == 2) o += value<T>(rf[s], e);
            D = __builtin_fmaf(value<T>(gf[s], e), o, D);
        }
    D = other_half_sum(D);
    if (z == 0 && half == 0 && i < q.rows) G.rows[row] = D;
    const float off = row_shift(score, m, inverse);
    // 16 bits without a bias: the accumulators of do . v begin at -D, in registers that stay, a subtraction less for each score
    // (4 x 4096, 128 channels with ragged keys, all passes: 2698 -> 2676 us)
    constexpr bool KEPT = !BIAS && sizeof(T) == 2 && DC > 64;
    f32x16 from_D;
#pragma unroll
    for (int r = 0; r < 16; r++) from_D[r] = -D;
    if (first < end) put(first);
    settle<T>(qf);
    settle<T>(gf);
    asm volatile("" : "+v"(m), "+v"(inverse));
    __syncthreads();
    const bool odd = BIAS && any_far_in_scores(line, A.reach);
    for (int n = first; n < end; n++) {
        const uint32_t tile = lds_address(tiles) + (n & 1) * 2 * TILE, kr = tile + L::rows_at(lane), vr = kr + TILE, kc = tile + L::columns_at(lane);
        if (n + 1 < end) fetch(n + 1);
        const int j0 = n * KEYS, low = j0 - (i0 + 31) - shift, high = j0 + 31 - i0 - shift;
        const bool near = BIAS && low < A.reach && high > -A.reach;
        f32x16 s, dp;
        [[maybe_unused]] f32x16 small;
        if constexpr (sizeof(T) == 4)
#pragma unroll
            for (int r = 0; r < 16; r++) small[r] = 0.0f;
        auto products = [&] {
#pragma unroll
            for (int c = 0; c < DC / 16; c++) {
                s = Operand<T>::product(L::template rows<KEYS>(kr, 0, c), qf[c], s);
                if constexpr (sizeof(T) == 4) dp = Operand<T>::product(L::template rows<KEYS>(vr, 0, c), gf[c], dp, small);
                else dp = Operand<T>::product(L::template rows<KEYS>(vr, 0, c), gf[c], dp);
            }
            if constexpr (sizeof(T) == 4) dp += small;
            if (sizeof(T) == 2) reads_ahead<DC / 16 * 2, 4, 1>();
        };
#pragma unroll
        for (int r = 0; r < 16; r++) dp[r] = KEPT ? from_D[r] : 0.0f;
        const bool side = low >= A.reach, begin = near || (odd && far_in_scores(line[side ? 2 * (A.reach + MARGIN) : 0]));
        if (begin) {
            const float* const at = line + (near ? j0 + 4 * half - i - shift + A.reach + MARGIN : side ? 2 * A.reach + MARGIN : 0);
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = at[result_row(r)];
            products();
        } else {
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = 0.0f;
            products();
        }
        const float flat = BIAS && !begin ? line[side ? 2 * (A.reach + MARGIN) : 0] : 0.0f;
        if (!all_there<KEYS>(there)) drop_keys(s, lds_address(keys + (n & 1) * KEYS), lane);
        if (A.causal && high > 0) drop_behind(s, i + shift - j0, lane);
        const float mt = m - flat, offt = off + flat * score.rate;
        if (!BIAS) {
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = probability(score, s[r], mt, inverse, offt) * (KEPT ? dp[r] : dp[r] - D);
        } else if (!near) {
            float ds = 0.0f, ps = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const float p = probability(score, s[r], mt, inverse, offt);
                s[r] = p * (dp[r] - D);
                ds += s[r];
                ps += p;
            }
            far_ds[0] += side ? 0.0f : ds; far_p[0] += side ? 0.0f : ps;
            far_ds[1] += side ? ds : 0.0f; far_p[1] += side ? ps : 0.0f;
            all_ds += ds;
        } else {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[r] = probability(score, s[r], mt, inverse, offt) * (dp[r] - D);
                all_ds += s[r];
            }
            if (i0 + 32 > q.there)      // (rows that are not there meet biases that no row may have)
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = mine ? s[r] : 0.0f;
            float x[3] = {0.0f, 0.0f, 0.0f};
            add_diagonals(s, x, std::make_integer_sequence<int, 16>());
            float* const at = own_sums + (j0 - i0 - shift + 4 * half - (lane & 31) + A.reach + MARGIN);
#pragma unroll
            for (int n16 = 0; n16 < 3; n16++) {      // (no two lanes of a half wavefront in one place, but in those of the next 16)
                at[16 * n16] += x[n16];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        }
        scaled.meet(s, dq);
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const Eight<T> ds = rounded<T>(s, c);
#pragma unroll
            for (int d = 0; d < ND; d++) dq[d] = Operand<T>::product(L::template columns<KEYS>(kc, 16 * c, d), ds, dq[d]);
        }
        if (n + 1 < end) put(n + 1);
        __syncthreads();
    }
    if (i < q.rows) {
        const float factor = A.scale * scaled.back();
        const int64_t rows = (A.packed ? A.q_rows : A.q_rows * A.batch) * A.heads;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                f32x4 x{dq[d][r], dq[d][r + 1], dq[d][r + 2], dq[d][r + 3]};
                x *= factor;
                if (!mine) x = f32x4{0, 0, 0, 0};
                const int c = 32 * d + result_row(r) + 4 * half;
                if (G.dq_parts) put_four<float>(G.dq_parts + (z * rows + row) * A.dim, c, A.dim, x);
                else put_four<T>(static_cast<T*>(G.dq) + row * A.dim, c, A.dim, x);
            }
    }
    if (!BIAS || !dtable) return;
    all_ds = other_half_sum(all_ds);
    float* const far_sums = sums + 2 * NW * entries;
#pragma unroll
    for (int side = 0; side < 2; side++) {
        const float ds = other_half_sum(far_ds[side]), p = other_half_sum(far_p[side]);
        if (G.row_parts && half == 0 && i < q.rows) {
            float* const at = G.row_parts + ((A.packed ? A.q_rows : A.q_rows * A.batch) * A.heads * z + row) * 3;
            at[0] = mine ? all_ds : 0.0f;
            at[1 + side] = mine ? p : 0.0f;
        }
        const float x = wave_sum(mine && half == 0 ? (G.row_parts ? ds : ds - all_ds * p) : 0.0f);
        if (lane == 0) far_sums[2 * wave + side] = x;
    }
    __syncthreads();
    for (int n = threadIdx.x; n < entries; n += NW * 64) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < 2 * NW; w++) x += sums[w * entries + n];
#pragma unroll
        for (int side = 0; side < 2; side++)
            if (n == side * (entries - 1))
#pragma unroll
                for (int w = 0; w < NW; w++) x += far_sums[2 * w + side];
        line[n] = x;
        sums[n] = __int_as_float(A.bucket_of[clamped(n - A.reach - MARGIN, A.reach)]);      // (where the entry's first sum was)
    }
    __syncthreads();
    for (int n = wave; n < A.buckets; n += NW) {
        float x = 0.0f;
        for (int e = lane; e < entries; e += 64) x += __float_as_int(sums[e]) == n ? line[e] : 0.0f;
        x = wave_sum(x);
        if (lane == 0) dtable[n] = x;
    }
}

// ---- backward: keys' side --------------------------------------------------------------------------------------------------------------------
// A wavefront has 32 keys (columns), whose gradients stay in its registers; the workgroup goes through the queries of the heads that
// share the key head, in tiles of 32.  Heads of 128 channels in 16 bits: the wavefront's values stay in LDS, so that two wavefronts
// have room on a SIMD.
template <typename T, int DC>
constexpr bool values_in_lds() { return sizeof(T) == 2 && DC == 128; }
template <typename T, int DC, int NW, bool BIAS>
__global__ __launch_bounds__(NW * 64, (NW == 4 && values_in_lds<T, DC>() ? 2 : 1)) void keys_kernel(SequenceAttention A, AttentionGrads G, int64_t slots, int splits) {
    constexpr int DP = pitch(DC), ND = (DC + 31) / 32;
    using L = Tile<T, DP>;
    constexpr int ROWS = 32, TILE = L::bytes(ROWS);
    extern __shared__ __attribute__((aligned(512))) char lds[];
    char* const tiles = lds;                                            // two pairs: q, do
    float* const row_stats = reinterpret_cast<float*>(lds + 4 * TILE);  // two times (3, ROWS): m or shift, 1 / l, -D
    char* const values = lds + 4 * TILE + 2 * 3 * ROWS * sizeof(float) + (values_in_lds<T, DC>() ? (threadIdx.x >> 6) * TILE : 0);
    float* const line = row_stats + 2 * 3 * ROWS + (values_in_lds<T, DC>() ? NW * TILE / sizeof(float) : 0);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, column = lane & 31;
    int kh;
    int64_t slot;
    if (!workgroup_item(blockIdx.x, slots, A.kv_heads, A, false, kh, slot)) return;
    const int z = blockIdx.y;
    int b, from;
    if (!find_slot(A.k_starts, A.k_rows, A.packed, A.batch, NW * 32, slot, lane, b, from)) return;
    Span k = span_of(A.k_starts, A.k_sizes, A.k_rows, A.packed, A.batch, b);
    if (from >= k.rows) return;
    Span q{0, 0, 0, 0};
    if (!A.packed || b < A.batch) q = span_of(A.q_starts, A.q_sizes, A.q_rows, A.packed, A.batch, b);
    const int j0 = from + wave * 32, j = j0 + column;
    const int shift = shift_of(A, q, k);
    const bool inside = j < k.there;
    const bool mine = inside && (!A.mask || A.mask[k.first + j]);
    const Score<T> score(A.scale);
    // the first tile of queries that sees a key of this workgroup
    int skip = 0;
    if (A.causal) skip = max(0, from - shift) / ROWS;
    const int each = from < k.there ? max(0, (q.there + ROWS - 1) / ROWS - skip) : 0, whole = each * A.share;
    const int first = (int)((int64_t)whole * z / splits), end = (int)((int64_t)whole * (z + 1) / splits);

    // (a masked key's column is computed like the others, and not written)
    Eight<T> kf[DC / 16], vf[values_in_lds<T, DC>() ? 1 : DC / 16];
    [[maybe_unused]] Staged<T, DP, 32, 64> vx;
    {
        const T* const k_row = row_start<T>(A.k, k, A.packed, kh) + (inside ? j : 0) * A.k.row;
        [[maybe_unused]] const T* const v_row = row_start<T>(A.v, k, A.packed, kh) + (inside ? j : 0) * A.v.row;
        row_operands<T, DC>(kf, k_row, inside, A.dim, true, lane);
        if constexpr (values_in_lds<T, DC>()) vx.load(row_start<T>(A.v, k, A.packed, kh) + j0 * A.v.row, A.v.row, k.there - j0, A.dim, lane);
        else row_operands<T, DC>(vf, v_row, inside, A.dim, true, lane);
    }
    f32x16 dk[ND], dv[ND];
    Scaled<T, ND> scaled;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) dk[d][r] = dv[d][r] = 0.0f;
    Staged<T, DP, ROWS, NW * 64> qx, gx;
    float sx[3];
    auto fetch = [&](int n) {
        const int h = kh * A.share + n / each, i0 = (skip + n % each) * ROWS;
        qx.load(row_start<T>(A.q, q, A.packed, h) + i0 * A.q.row, A.q.row, q.there - i0, A.dim, threadIdx.x);
        gx.load(row_start<T>(G.go, q, A.packed, h) + i0 * G.go.row, G.go.row, q.there - i0, A.dim, threadIdx.x);
        if (threadIdx.x < ROWS) {
            float m = -NONE, inverse = 0.0f, D = 0.0f;
            if (i0 + (int)threadIdx.x < q.there) {
                const int64_t row = (q.first + i0 + threadIdx.x) * A.heads + h;
                m = G.stats[2 * row];
                inverse = G.stats[2 * row + 1];
                D = G.rows[row];
            }
            sx[0] = m;
            sx[1] = inverse;
            sx[2] = D;
        }
    };
    auto put = [&](int n) {
        qx.store(tiles + (n & 1) * 2 * TILE, threadIdx.x);
        gx.store(tiles + (n & 1) * 2 * TILE + TILE, threadIdx.x);
        if (threadIdx.x < ROWS) {
            float* const st = row_stats + (n & 1) * 3 * ROWS + threadIdx.x;
            st[0] = sizeof(T) == 4 ? sx[0] : P_LIFT<T> + row_shift(score, sx[0], sx[1]);
            st[ROWS] = sx[1];
            st[2 * ROWS] = -sx[2];
        }
    };
    if (first < end) fetch(first);
    if constexpr (values_in_lds<T, DC>()) vx.store(values, lane);      // (read by this wavefront alone)
    else settle<T>(vf);
    settle<T>(kf);
    if (first < end) put(first);
    int line_of = -1;
    const uint32_t vr = lds_address(values) + L::rows_at(lane);
    (void)vr;
    for (int n = first; n < end; n++) {
        const int h = kh * A.share + n / each, i0 = (skip + n % each) * ROWS;
        if (BIAS && h != line_of) {
            __syncthreads();
            fill_line<T>(A, h, line, threadIdx.x, NW * 64);
            line_of = h;
        }
        __syncthreads();
        const uint32_t tile = lds_address(tiles) + (n & 1) * 2 * TILE, qr = tile + L::rows_at(lane), gr = qr + TILE, qc = tile + L::columns_at(lane),
                       gc = qc + TILE;
        const float* const st = row_stats + (n & 1) * 3 * ROWS + 4 * half;
        if (n + 1 < end) fetch(n + 1);
        f32x16 s, dp;
        const int low = j0 - (i0 + 31) - shift, high = j0 + 31 - i0 - shift;
        if (BIAS && low < A.reach && high > -A.reach) {
            const float* const at = line + (j - i0 - 4 * half - shift + A.reach + MARGIN);
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = at[-result_row(r)];
        } else {
            const float flat = BIAS ? line[low >= A.reach ? 2 * (A.reach + MARGIN) : 0] : 0.0f;
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = flat;
        }
#pragma unroll
        for (int r = 0; r < 16; r += 4) {      // do . v - D
            const f32x4 D4 = *reinterpret_cast<const f32x4*>(st + 2 * ROWS + result_row(r));
#pragma unroll
            for (int e = 0; e < 4; e++) dp[r + e] = D4[e];
        }
#pragma unroll
        for (int c = 0; c < DC / 16; c++) s = Operand<T>::product(L::template rows<ROWS>(qr, 0, c), kf[c], s);
        [[maybe_unused]] f32x16 small;
        if constexpr (sizeof(T) == 4)
#pragma unroll
            for (int r = 0; r < 16; r++) small[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < DC / 16; c++) {
            const Eight<T> gx8 = L::template rows<ROWS>(gr, 0, c);
            if constexpr (sizeof(T) == 4) dp = Operand<T>::product(gx8, vf[c], dp, small);
            else if constexpr (values_in_lds<T, DC>()) dp = Operand<T>::product(gx8, L::template rows<ROWS>(vr, 0, c), dp);
            else dp = Operand<T>::product(gx8, vf[c], dp);
        }
        if constexpr (sizeof(T) == 4) dp += small;
        if (A.causal && high > 0) drop_before(s, j - shift - i0, lane);
        if (BIAS && i0 + ROWS > q.there) drop_behind(s, q.there - 1 - i0, lane);      // (their biases may be plus infinity or NaN)
        f32x16 p;
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const f32x4 m4 = *reinterpret_cast<const f32x4*>(st + result_row(r));
            f32x4 l4{1, 1, 1, 1};
            if (sizeof(T) == 4) l4 = *reinterpret_cast<const f32x4*>(st + ROWS + result_row(r));
#pragma unroll
            for (int e = 0; e < 4; e++) {
                p[r + e] = probability(score, s[r + e], m4[e], l4[e], m4[e]);
                s[r + e] = p[r + e] * dp[r + e];
            }
        }
        scaled.meet(s, dk);
        const Eight<T> pf[2] = {rounded<T>(p, 0), rounded<T>(p, 1)}, ds[2] = {rounded<T>(s, 0), rounded<T>(s, 1)};
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int d = 0; d < ND; d++) {
                dv[d] = Operand<T>::product(L::template columns<ROWS>(gc, 16 * c, d), pf[c], dv[d]);
                dk[d] = Operand<T>::product(L::template columns<ROWS>(qc, 16 * c, d), ds[c], dk[d]);
            }
        if (n + 1 < end) put(n + 1);
    }
    if (j >= k.rows) return;
    const float lift = NARROW<T> ? 0x1p-15f : 1.0f, factor = A.scale * scaled.back() * lift;
    const int64_t row = (k.first + j) * A.kv_heads + kh, rows = (A.packed ? A.k_rows : A.k_rows * A.batch) * A.kv_heads;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            f32x4 x{dk[d][r], dk[d][r + 1], dk[d][r + 2], dk[d][r + 3]}, y{dv[d][r], dv[d][r + 1], dv[d][r + 2], dv[d][r + 3]};
            x *= factor;
            y *= lift;
            if (!mine) x = y = f32x4{0, 0, 0, 0};
            const int c = 32 * d + result_row(r) + 4 * half;
            if (G.dk_parts) {
                put_four<float>(G.dk_parts + (z * rows + row) * A.dim, c, A.dim, x);
                put_four<float>(G.dv_parts + (z * rows + row) * A.dim, c, A.dim, y);
            } else {
                put_four<T>(static_cast<T*>(G.dk) + row * A.dim, c, A.dim, x);
                put_four<T>(static_cast<T*>(G.dv) + row * A.dim, c, A.dim, y);
            }
        }
}

// What the passes left in parts, in one launch: gradients as the sum of their splits, in their order, and the table's.
struct Finish {
    const float* parts[3];
    void* to[3];
    int64_t count[3], blocks[3];      // elements; workgroups (1024 elements each)
    int splits[3];
    const float* table_parts;
    void* dtable;
    int64_t table_count;              // workgroups' sums for a (head, bucket)
    const float* row_parts;           // see AttentionGrads; table_splits, rows without heads
    const int32_t* bucket_of;
    int64_t rows;
    int table_splits, reach;
    int buckets, heads, table_float;
};
template <typename T>
__global__ __launch_bounds__(256) void finish_kernel(Finish F) {
    int64_t block = blockIdx.x;
#pragma unroll
    for (int a = 0; a < 3; a++) {
        if (block >= F.blocks[a]) {
            block -= F.blocks[a];
            continue;
        }
        const int64_t n = (block * 256 + threadIdx.x) * 4, count = F.count[a];
        T* const out = static_cast<T*>(F.to[a]);
        if ((count & 3) == 0) {
            if (n >= count) return;
            f32x4 x{0, 0, 0, 0};
            for (int z = 0; z < F.splits[a]; z++) x += *reinterpret_cast<const f32x4*>(F.parts[a] + z * count + n);
            put_four<T>(out + n, 0, 4, x);
        } else {
            for (int64_t e = n; e < n + 4 && e < count; e++) {
                float x = 0.0f;
                for (int z = 0; z < F.splits[a]; z++) x += F.parts[a][z * count + e];
                out[e] = from_float<T>(x);
            }
        }
        return;
    }
    // a wavefront to a (head, bucket): the workgroups' sums in a fixed order, in 64 bits
    const int64_t at = block * 4 + (threadIdx.x >> 6);
    if (at >= (int64_t)F.heads * F.buckets) return;
    const int h = (int)(at / F.buckets), n = (int)(at - (int64_t)h * F.buckets), lane = threadIdx.x & 63;
    double x = 0.0;
    for (int64_t w = lane; w < F.table_count; w += 64) x += F.table_parts[(h * F.table_count + w) * F.buckets + n];
    if (F.row_parts)
#pragma unroll
        for (int side = 0; side < 2; side++) {
            if (F.bucket_of[side * 2 * F.reach] != n) continue;
            for (int64_t r = lane; r < F.rows; r += 64) {
                float ds = 0.0f, p = 0.0f;
                for (int z = 0; z < F.table_splits; z++) {
                    const float* const at = F.row_parts + ((z * F.rows + r) * F.heads + h) * 3;
                    ds += at[0];
                    p += at[1 + side];
                }
                x -= (double)ds * p;
            }
        }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    if (lane) return;
    if (F.table_float) static_cast<float*>(F.dtable)[(int64_t)n * F.heads + h] = (float)x;
    else static_cast<T*>(F.dtable)[(int64_t)n * F.heads + h] = from_float<T>((float)x);
}
}  // namespace attention

// ---- launches ----------------------------------------------------------------------------------------------------------------------------------
template <typename K, typename... P>
void launch_attention(K kernel, dim3 grid, int threads, size_t lds, hipStream_t st, P... p) {
    if (lds > 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL(kernel, grid, dim3(threads), lds, st, p...);
}
template <typename F>
void with_padded_dim(int dim, F f) {
    if (dim <= 16) f(std::integral_constant<int, 16>());
    else if (dim <= 32) f(std::integral_constant<int, 32>());
    else if (dim <= 64) f(std::integral_constant<int, 64>());
    else if (dim <= 96) f(std::integral_constant<int, 96>());
    else f(std::integral_constant<int, 128>());
}
template <typename F>
void with_choice(bool yes, F f) {
    if (yes) f(std::true_type());
    else f(std::false_type());
}
inline unsigned die_grid(int64_t count) { return (unsigned)((count + 7) / 8 * 8); }

template <typename T>
void sequence_attention_forward(const SequenceAttention& A, const AttentionPlan& P, T* out, T* rest, float* stats, float* scratch, hipStream_t st) {
    using namespace attention;
    with_padded_dim(A.dim, [&](auto dc) {
        with_choice(A.table != nullptr, [&](auto bias) {
            constexpr int DC = decltype(dc)::value, DP = pitch(DC);
            constexpr bool BIAS = decltype(bias)::value;
            const int64_t rows = (A.packed ? A.q_rows : A.q_rows * A.batch) * A.heads;
            if (!P.few) {
                const size_t lds = 4 * Tile<T, DP>::bytes(keys_at_once<T>()) + 2 * keys_at_once<T>() * sizeof(float) + (BIAS ? (2 * (A.reach + MARGIN) + 1) * sizeof(float) : 0);
                launch_attention(tiles_kernel<T, DC, 4, BIAS>, dim3(die_grid((int64_t)P.slots * A.heads)), 256, lds, st, A, out, rest, stats, P.slots);
                return;
            }
            float* const part_o = scratch;
            float* const part_ml = scratch + P.splits * rows * DP;
            const dim3 grid(P.slots, A.kv_heads * ((A.share + 31) / 32), P.splits);
            const int at_once = A.share < 32 ? A.share : 32;
            const size_t line = BIAS && few_line(at_once, A.reach) ? (size_t)at_once * (2 * (A.reach + MARGIN) + 1) * sizeof(float) : 0;
            if (P.waves == 1) launch_attention(few_kernel<T, DC, 1, BIAS, false>, grid, 64, line, st, A, out, rest, stats, part_o, part_ml, P.splits);
            else with_choice(P.past, [&](auto past) {
                launch_attention(few_kernel<T, DC, few_waves(sizeof(T) == 4, DC), BIAS, decltype(past)::value>, grid, P.waves * 64, line, st, A, out, rest, stats,
                                 part_o, part_ml, P.splits);
            });
            if (P.splits > 1)
                launch_attention(combine_parts<T, DC>, dim3((unsigned)((rows + 7) / 8)), 256, 0, st, A, part_o, part_ml, P.splits, rows, out, rest, stats);
        });
    });
}

template <typename T>
void sequence_attention_backward(const SequenceAttention& A, const AttentionGradPlan& P, AttentionGrads G, void* dtable, float* scratch, hipStream_t st) {
    using namespace attention;
    const int64_t q_all = (A.packed ? A.q_rows : A.q_rows * A.batch) * A.heads, k_all = (A.packed ? A.k_rows : A.k_rows * A.batch) * A.kv_heads;
    float* next = scratch;
    auto take = [&](int64_t floats) {      // aligned to 16 bytes
        float* const at = next;
        next += (floats + 3) / 4 * 4;
        return at;
    };
    G.rows = take(q_all);
    if (P.q_splits > 1) G.dq_parts = take(P.q_splits * q_all * A.dim);
    if (P.k_splits > 1) {
        G.dk_parts = take(P.k_splits * k_all * A.dim);
        G.dv_parts = take(P.k_splits * k_all * A.dim);
    }
    if (dtable && P.q_splits > 1) G.row_parts = take(P.q_splits * q_all * 3);
    G.dtable = dtable ? next : nullptr;
    with_padded_dim(A.dim, [&](auto dc) {
        with_choice(A.table != nullptr, [&](auto bias) {
            constexpr int DC = decltype(dc)::value, DP = pitch(DC);
            constexpr bool BIAS = decltype(bias)::value;
            const size_t line = BIAS ? (2 * (A.reach + MARGIN) + 1) * sizeof(float) : 0, tiles = 4 * Tile<T, DP>::bytes(32);
            const size_t queries = queries_lds(sizeof(T) == 4, A.dim, A.reach, BIAS, P.q_waves);
            if (q_all > 0) {
                const dim3 grid(die_grid((int64_t)P.q_slots * A.heads), P.q_splits);
                if (P.q_waves == 1) launch_attention(queries_kernel<T, DC, 1, BIAS>, grid, 64, queries, st, A, G, P.q_slots, P.q_splits);
                else launch_attention(queries_kernel<T, DC, 4, BIAS>, grid, 256, queries, st, A, G, P.q_slots, P.q_splits);
            }
            if (k_all > 0 && G.dk) {
                const dim3 grid(die_grid((int64_t)P.k_slots * A.kv_heads), P.k_splits);
                const size_t lds = tiles + 6 * 32 * sizeof(float) + line + (values_in_lds<T, DC>() ? P.k_waves * Tile<T, DP>::bytes(32) : 0);
                if (P.k_waves == 1) launch_attention(keys_kernel<T, DC, 1, BIAS>, grid, 64, lds, st, A, G, P.k_slots, P.k_splits);
                else launch_attention(keys_kernel<T, DC, 4, BIAS>, grid, 256, lds, st, A, G, P.k_slots, P.k_splits);
            }
        });
    });
    Finish F{};
    int64_t blocks = 0;
    auto add = [&](int at, const float* parts, int splits, int64_t count, void* to) {
        if (!parts || !to) return;
        F.parts[at] = parts; F.to[at] = to; F.splits[at] = splits; F.count[at] = count;
        blocks += F.blocks[at] = (count + 1023) / 1024;
    };
    add(0, G.dq_parts, P.q_splits, q_all * A.dim, G.dq);
    add(1, G.dk_parts, P.k_splits, k_all * A.dim, G.dk);
    add(2, G.dv_parts, P.k_splits, k_all * A.dim, G.dv);
    if (dtable) {
        F.table_parts = G.dtable; F.dtable = dtable;
        F.table_count = q_all > 0 ? P.q_slots * P.q_splits : 0;
        F.row_parts = G.row_parts; F.bucket_of = A.bucket_of; F.rows = A.packed ? A.q_rows : A.q_rows * A.batch;
        F.table_splits = P.q_splits; F.reach = A.reach;
        F.buckets = A.buckets; F.heads = A.heads; F.table_float = A.table_float;
        blocks += ((int64_t)A.heads * A.buckets + 3) / 4;
    }
    if (blocks > 0) launch_attention(finish_kernel<T>, dim3((unsigned)blocks), 256, 0, st, F);
}
}  // namespace cfh
