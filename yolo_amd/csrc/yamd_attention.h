// What the attention kernels share: argument blocks, the layout of a tile in LDS, and the matrix-instruction forms.
//
// All products use v_mfma_f32_32x32x16_bf16.  Lane l holds of A the row l & 31 and of B the column l & 31, both at the
// eight k slots of its half h = l >> 5; of the result it holds column l & 31 and the sixteen rows acc_row(r, h).  Which
// element of the sum a k slot stands for is free as long as A and B agree, so the rows 16 u .. 16 u + 15 of a result are
// used as the B operand of the next product where they are: slot (h, e) stands for row 16 u + 8 (e >> 2) + 4 h + (e & 3).
// The other operand is then needed transposed (eight rows of one column), which the transposing LDS read delivers from
// rows in their natural order: no probability ever moves between lanes.
#pragma once
#include "yamd_common.h"
#include "yamd_distance.h"

#include <cmath>

namespace yamd {

typedef __attribute__((ext_vector_type(4))) short s16x4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMasked = -1e5f;         // a query whose scores with their bias are all below this is left without keys
constexpr int kFewKeys = 256;            // up to here o_exact takes two products without a bias too

struct AttnView {
    const __bf16 *p;
    long long sb, st, sh;                // strides of batch, token and head in elements
};

// A tile of 64 rows in LDS: 16-byte chunks, row r's chunk c at position c ^ swizzle(r).  Rows are unpadded, because loads
// write LDS directly, lane after lane; the swizzle spreads over the 64 banks both the 16-byte reads of 16 rows in one
// column and the transposing reads, which take 64 bytes of each of 4 rows.
template <int D>
struct Tile {
    static constexpr int kChunks = D <= 32 ? 4 : D <= 64 ? 8 : 16;      // per row; D = 96 leaves the last four unused
    static constexpr int kRowBytes = kChunks * 16;
    static constexpr int bytes(int rows) { return rows * kRowBytes; }
    __device__ static __forceinline__ int swizzle(int r)
    {
        if constexpr (kChunks == 4) return (r >> 2) & 3;
        else if constexpr (kChunks == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
        else return ((r & 3) << 2) | ((r >> 2) & 3);
    }
};

__device__ __forceinline__ int acc_row(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

__device__ __forceinline__ f32x16 zero16()
{
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.0f;
    return z;
}

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ s16x4 transposed_quad(const char *at)
{
    typedef __attribute__((address_space(3))) s16x4 lds_quad;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad *)at);
}

// Where a lane reads a tile.  Columns enter a swizzled address as an exclusive or, so one lane constant serves each kind of
// operand: `row` for 16 bytes of row (lane & 31), `quad` for the transposing reads.
template <int D>
struct TileReader {
    using T = Tile<D>;
    unsigned row, quad;

    __device__ __forceinline__ explicit TileReader(int lane)
    {
        const int r = lane & 31, i = lane & 15, g = lane >> 4, rq = 4 * (g >> 1) + (i >> 2);
        row = r * T::kRowBytes + (((lane >> 5) ^ T::swizzle(r)) << 4);
        quad = rq * T::kRowBytes + (((2 * (g & 1) + ((i >> 1) & 1)) ^ T::swizzle(rq)) << 4) + (i & 1) * 8;
    }
    // hides the constants' origin: the addresses made from them are then computed where they are used instead of being kept
    // in registers across the loop, of which wide heads have none to spare
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(row), "+v"(quad)); }

    // A (or B) operand of rows [row0, row0 + 32), columns 16 ks .. 16 ks + 15
    __device__ __forceinline__ bf16x8 rows(const char *tile, int row0, int ks) const
    {
        return *(const bf16x8 *)(tile + row0 * T::kRowBytes + (row ^ (ks << 5)));
    }
    // A operand of the transposed tile: rows are the tile's columns 32 n .. 32 n + 31, k slots its rows in the order that the
    // accumulator rows 0 .. 15 (counted from row0) have as a B operand.  Each group of 16 lanes reads 4 rows of 16 columns and
    // gets them transposed: lane i of the group gives the address of row i / 4, columns 4 (i % 4) .. + 3 and receives the
    // 4 rows of column i.
    __device__ __forceinline__ bf16x8 transposed(const char *tile, int row0, int n) const
    {
        union {
            s16x4 q[2];
            bf16x8 v;
        } o;
        o.q[0] = transposed_quad(tile + row0 * T::kRowBytes + (quad ^ (n << 6)));
        o.q[1] = transposed_quad(tile + (row0 + 8) * T::kRowBytes + (quad ^ (n << 6) ^ 32));      // swizzle(r + 8) = swizzle(r) ^ 2
        return o.v;
    }
};

// B operand from eight consecutive accumulator values
__device__ __forceinline__ bf16x8 acc_operand(const f32x16 &v, int u)
{
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (__bf16)v[8 * u + e];
    return o;
}

// combines a lane's value with that of the lane 32 away (the other half of the same column)
template <typename F>
__device__ __forceinline__ float with_other_half(float v, F f)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    return f(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}

// How the tiles of owned rows (items) become workgroups: the first `whole` items walk the looped axis from end to end, each
// of the `rest` behind them is cut into `splits` parts of `per_split` steps, a workgroup each, whose float32 results another
// kernel joins.
struct WorkSplit {
    int whole, rest, splits, per_split;
    int tile_rows;                       // rows of an item: 128, or all when there are fewer
    __host__ __device__ int whole_grid() const { return (whole + 7) / 8 * 8; }
    int grid() const { return whole_grid() + (rest * splits + 7) / 8 * 8; }
    __host__ __device__ int part_rows() const { return rest * tile_rows; }       // (of one part each: rest < 256)
};
struct Piece {
    int item, split;                     // split < 0: all of the item
    int t0, t1;                          // steps
    int index;                           // among all pieces
};
// The workgroup's piece; false for the ids beyond the work.  Workgroup ids go round-robin to the 8 XCDs: each gets a contiguous
// range of the items, so that the workgroups that share one head's keys share an L2.
__device__ __forceinline__ bool work_piece(const WorkSplit &w, int steps, Piece &p)
{
    const int grid0 = w.whole_grid(), part = blockIdx.x >= grid0;
    const int id = part ? blockIdx.x - grid0 : blockIdx.x, per_xcd = (part ? gridDim.x - grid0 : grid0) >> 3;
    const int at = (id & 7) * per_xcd + (id >> 3);
    if (!part) {
        p = {at, -1, 0, steps, at};
        return at < w.whole;
    }
    const int of = __builtin_amdgcn_readfirstlane(at / w.splits);
    p.item = w.whole + of;
    p.split = at - of * w.splits;
    p.t0 = p.split * w.per_split;
    p.t1 = p.t0 + w.per_split < steps ? p.t0 + w.per_split : steps;
    p.index = w.whole + at;
    return at < w.rest * w.splits;
}
// row of a part's results: parts are laid out [split][item of the rest][row of the item]
__device__ __forceinline__ int part_row(const WorkSplit &w, const Piece &p, int row)
{
    return (p.split * w.rest + p.item - w.whole) * w.tile_rows + row;
}

// Loads that write LDS directly: lane l of the wave takes 16 (4) bytes from `base` + `offset` and they land at byte 16 l
// (4 l) behind `lds`; base and lds are the same for all lanes.  They are written as asm because the compiler, which cannot
// tell the two buffers of a tile apart, would otherwise wait for the next tile's loads before it reads the current tile.
// No register is written; whoever reads the tile waits with landed() and passes a barrier first.
__device__ __forceinline__ unsigned lds_address(const void *p)
{
    return __builtin_amdgcn_readfirstlane((unsigned)(size_t)(const __attribute__((address_space(3))) char *)p);
}
// (m0 is a register that the compiler keeps to itself: it warns about the declaration, and honours it)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_lds_16(const void *base, unsigned offset, const void *lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_address(lds)), "v"(offset), "s"(base)
                 : "memory", "m0");
}
__device__ __forceinline__ void load_lds_4(const void *base, unsigned offset, const void *lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds_address(lds)), "v"(offset), "s"(base)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Fills tiles with rows of a token axis of `len` rows (256 threads, each wave a quarter).  Rows beyond the axis repeat its
// last row, chunks beyond the head width d are left as they are: both are cleared by the caller.
template <int D, int ROWS = kTile>
struct TileLoader {
    using T = Tile<D>;
    static constexpr int N = T::kChunks * ROWS / 256;
    static_assert(N * 256 == T::kChunks * ROWS, "every thread moves whole pieces");
    unsigned offset[N];            // of this lane's pieces of a whole tile
    unsigned row_bytes;
    bool on[N];

    __device__ __forceinline__ TileLoader(long long st, int d, int wave, int lane) : row_bytes((unsigned)st * 2)
    {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int at = (n * 4 + wave) * 64 + lane, r = at / T::kChunks, c = (at % T::kChunks) ^ T::swizzle(r);
            offset[n] = r * row_bytes + 16 * c;
            on[n] = 8 * c < d;
        }
    }
    __device__ __forceinline__ void load(char *tile, const __bf16 *base, int first, int len, int wave, int lane) const
    {
        const char *src = (const char *)base + (long long)first * row_bytes;
        const int last = len - 1 - first;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            unsigned o = offset[n];
            if (last < ROWS - 1) {
                const int r = ((n * 4 + wave) * 64 + lane) / T::kChunks;
                o -= (r > last ? r - last : 0) * row_bytes;
            }
            if (on[n]) load_lds_16(src, o, tile + (n * 4 + wave) * 1024);
        }
    }
};

// `bytes` of LDS (a multiple of 16) set to zero by the workgroup
__device__ __forceinline__ void clear_lds(char *p, int bytes)
{
    for (int at = threadIdx.x * 16; at < bytes; at += 256 * 16) *(uint4 *)(p + at) = make_uint4(0, 0, 0, 0);
}

// zeros in the rows whose bit of `keep` is clear: four threads per row
template <int D, int ROWS = kTile>
__device__ __forceinline__ void clear_rows(char *tile, unsigned long long keep)
{
    using T = Tile<D>;
    const int r = threadIdx.x >> 2;
    if (r >= ROWS || ((keep >> r) & 1)) return;
#pragma unroll
    for (int c = 0; c < T::kChunks / 4; ++c) *(uint4 *)(tile + r * T::kRowBytes + ((threadIdx.x & 3) * (T::kChunks / 4) + c) * 16) = make_uint4(0, 0, 0, 0);
}

// gives -inf to the scores of a tile's rows 32 u .. 32 u + 31 that are not kept
__device__ __forceinline__ void mask_rows(f32x16 &s, unsigned long long keep, int u, int half)
{
    const unsigned bits = (unsigned)(keep >> (32 * u)) >> (4 * half);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = bits & (1u << acc_row(r, 0)) ? s[r] : -INFINITY;
}

__device__ __forceinline__ unsigned long long uniform64(unsigned long long v)
{
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
    return ((unsigned long long)hi << 32) | lo;
}

// bits of the rows first .. first + 63 that are below len
__device__ __forceinline__ unsigned long long rows_below(int first, int len)
{
    return len - first >= kTile ? ~0ull : (1ull << (len - first)) - 1;
}

// The biases of the distances between a workgroup's rows and a tile, staged in LDS: floats `from` .. `from` + n - 1 of a head's
// bias at p[0 ..]; distances outside the table are never read and repeat its ends.
__device__ __forceinline__ void load_window(char *lds, const float *bias, int from, int n, int n_off, int wave, int lane)
{
    for (int at = wave * 64; at < n; at += 256) {
        const int o = from + at + lane;
        load_lds_4(bias, (o < 0 ? 0 : o < n_off ? o : n_off - 1) * 4u, lds + at * 4);
    }
}

// Forms of the bias.  In quads (a sequence, or a map whose width is a multiple of 4) four tokens from a multiple of 4 on
// lie next to each other, so one coordinate serves four rows of an accumulator.
enum Bias { kNoBias, kAnyBias, kQuadBias };

// the biases of a lane's sixteen accumulator rows: win[coord] (SIGN = 1) or win[-coord] for rows 32 u + acc_row(r, half)
template <int BIAS, int SIGN>
__device__ __forceinline__ void read_bias(float (&b)[16], const float *win, const int *coord, int u, int half)
{
    if constexpr (BIAS == kQuadBias) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = coord[32 * u + acc_row(4 * g, half)];
            const float *const p = SIGN > 0 ? win + c : win - c - 3;
#pragma unroll
            for (int j = 0; j < 4; ++j) b[4 * g + j] = p[SIGN > 0 ? j : 3 - j];
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) b[r] = win[SIGN * coord[32 * u + acc_row(r, half)]];
    }
}

static inline Bias bias_form(const float *bias, int map_h, int map_w)
{
    return !bias ? kNoBias : map_h == 1 || map_w % 4 == 0 ? kQuadBias : kAnyBias;
}
// distances between 128 owned rows and a tile of 64, rounded up to what four waves load at once
static inline int window_len(int map_h, int map_w)
{
    const int n = kBlockRows + kTile + (map_h > 1 ? kBlockRows + kTile + 2 * map_w : 0);
    return (n + 255) / 256 * 256;
}

// ---- host side -----------------------------------------------------------------------------------------------------------
// argument checks shared by both directions (yamd_attention.hip)
int check_attention(const yamd_attention_desc *d, const uint8_t *key_mask, long long mask_stride, const float *bias);
int check_tokens(const yamd_attention_desc *d, const yamd_tokens *t, int len, int heads, const char *name);
int check_result(const yamd_attention_desc *d, const yamd_tokens *t, int len, int heads, const char *name);
static inline AttnView view_of(const yamd_tokens *t) { return {(const __bf16 *)t->data, t->batch_stride, t->token_stride, t->head_stride}; }

// the split of `items` items (tiles of an axis of `len` rows) of `steps` steps each, with `resident` workgroups on a CU at a time (what their registers allow),
// `results` results per row, and a step of `step` times the forward kernel's duration
WorkSplit split_work(long long items, int steps, int len, int resident, int results, float step);

// head width of the kernel that serves `d` channels: the channels beyond d are zeros in registers and LDS
static inline int padded_head_dim(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : 128; }

}  // namespace yamd
