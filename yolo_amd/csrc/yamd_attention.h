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

namespace yamd {

typedef __attribute__((ext_vector_type(4))) short s16x4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 64;                // rows of a tile that passes through LDS (keys, or queries in the dK / dV kernel)
constexpr int kBlockRows = 128;          // rows that a workgroup owns: 32 for each of its four waves

struct AttnView {
    const __bf16 *p;
    long long sb, st, sh;                // strides of batch, token and head in elements
};

// a tile row is read 16 bytes at a time by 32 lanes on 32 rows: a row length of an odd multiple of 16 bytes spreads them
template <int D>
constexpr int kRow = D * 2 + 16;

__device__ __forceinline__ int acc_row(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

__device__ __forceinline__ f32x16 zero16()
{
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.0f;
    return z;
}

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// A operand of rows [row0, row0 + 32) of a tile, columns 16 ks .. 16 ks + 15
__device__ __forceinline__ bf16x8 rows_operand(const char *tile, int row_bytes, int row0, int ks, int lane)
{
    return *(const bf16x8 *)(tile + (row0 + (lane & 31)) * row_bytes + (16 * ks + 8 * (lane >> 5)) * 2);
}

__device__ __forceinline__ s16x4 transposed_quad(const char *at)
{
    typedef __attribute__((address_space(3))) s16x4 lds_quad;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad *)at);
}

// A operand of the transposed tile: rows are the tile's columns col0 .. col0 + 31, k slots its rows in the order that the
// accumulator rows 16 u .. 16 u + 15 (counted from row0) have as a B operand.  Each group of 16 lanes reads 4 rows of 16
// columns and gets them transposed: lane i of the group gives the address of row i / 4, columns 4 (i % 4) .. + 3 and
// receives the 4 rows of column i.
__device__ __forceinline__ bf16x8 transposed_operand(const char *tile, int row_bytes, int row0, int col0, int lane)
{
    const int i = lane & 15, g = lane >> 4;
    const char *at = tile + (row0 + 4 * (g >> 1) + (i >> 2)) * row_bytes + (col0 + 16 * (g & 1) + 4 * (i & 3)) * 2;
    union {
        s16x4 q[2];
        bf16x8 v;
    } o;
    o.q[0] = transposed_quad(at);
    o.q[1] = transposed_quad(at + 8 * row_bytes);
    return o.v;
}

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

// Workgroup ids go round-robin to the 8 XCDs: give each a contiguous range of the work, so that the workgroups that share
// one head's keys share an L2.  Returns a value >= total for the ids beyond the work.
__device__ __forceinline__ int work_item()
{
    const int per_xcd = gridDim.x >> 3;
    return (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
}
static inline int work_grid(long long total) { return (int)(ceil_div(total, 8) * 8); }

// A position t of a map of width w at (t / w, t % w) has the coordinate a(t) = (t / w)(2 w - 1) + t % w, and the distance of
// two positions the index a(query) - a(key) + a(last) among the (2 h - 1)(2 w - 1) distances of the map.
__host__ __device__ __forceinline__ int map_coord(int t, int w) { return t + (t / w) * (w - 1); }

// 64 rows of a tile on their way from global memory to LDS: each of 256 threads moves D / 32 pieces of 16 bytes.
template <int D>
struct TilePieces {
    static constexpr int N = D / 32, CPR = D / 8;
    uint4 v[N];

    // rows first .. first + 63 of a token axis with `len` rows; pieces beyond the rows or beyond the head width read as zero
    __device__ __forceinline__ void load(const __bf16 *base, long long st, int first, int len, int d)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = i * 256 + threadIdx.x, row = id / CPR, c = id % CPR, t = first + row;
            if (t < len && 8 * c < d) v[i] = *(const uint4 *)(base + (long long)t * st + 8 * c);
            else v[i] = make_uint4(0, 0, 0, 0);
        }
    }
    // `keep`: one bit per row; a row whose bit is clear is stored as zeros (a masked key may hold anything, NaN included)
    __device__ __forceinline__ void store(char *tile, int row_bytes, unsigned long long keep) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = i * 256 + threadIdx.x, row = id / CPR, c = id % CPR;
            *(uint4 *)(tile + row * row_bytes + c * 16) = (keep >> row) & 1 ? v[i] : make_uint4(0, 0, 0, 0);
        }
    }
};

// ---- host side -----------------------------------------------------------------------------------------------------------
// argument checks shared by both directions (yamd_attention.hip)
int check_attention(const yamd_attention_desc *d, const uint8_t *key_mask, long long mask_stride, const float *bias);
int check_tokens(const yamd_attention_desc *d, const yamd_tokens *t, int len, int heads, const char *name);
static inline AttnView view_of(const yamd_tokens *t) { return {(const __bf16 *)t->data, t->batch_stride, t->token_stride, t->head_stride}; }

// split of the looped axis when the owned rows alone give too few workgroups: the number of parts of `tiles` tiles
int attention_splits(long long workgroups, int tiles, int min_tiles);

// head width of the kernel that serves `d` channels: the channels beyond d are zeros in registers and LDS
static inline int padded_head_dim(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : 128; }

}  // namespace yamd
