// Attention over tokens, backward.  The probabilities are computed again from q, k and the forward pass's logarithm of the
// sums, so nothing of size q_len x k_len is kept:
//   P = exp(scale q k^T + bias - lse),  dP = do v^T,  D = rowsum(do o),  dS = P (dP - D)
//   dv = P^T do,  dk = scale dS^T q,  dq = scale dS k,  d bias[distance] = sum of dS over the pairs at that distance
//
// Two kernels share the work so that every sum has one owner and a fixed order (no atomics on gradients, equal bits on every
// run): one owns keys and walks the queries of all heads that share them (dk, dv), one owns queries and walks the keys (dq,
// bias).  That costs 7 products instead of 5; float32 atomics on dq would instead cost its size once per key block.
// Both take the products so that P and dS come out as the B operand of the product that follows (yamd_attention.h); P and
// dS are rounded to bf16 there, their use in the sums before (bias) stays in float32.  Rounding dS costs dq and dk as much as
// their own rounding (2.4e-3 instead of 1.7e-3 in all); a second product for what is lost took 12 % of the backward pass.
//
// What bounds them: neither unit is full, with two waves per SIMD.  2 images of 8 heads, 6400 x 6400 tokens, d = 64: dkv 373 us,
// 900 TFLOP/s (matrix unit 41 % busy, vector unit 36 %), dq 269 us, 935 TFLOP/s (41 % and 48 %), with a bias 431 and 514 us; d = 128 with
// 4 key heads: dkv 694 - 708 us, 950 TFLOP/s (40 % and 27 %, LDS reads 10 %), dq 446 - 469 us, 1070 - 1130 TFLOP/s (51 % and 38 %).  A third wave does not fit: the
// results and the owned rows alone are 128 registers at d = 64, and asking for it spills.
#include "yamd_attention.h"

#include <cmath>
#include <type_traits>

namespace yamd {

struct AttnBwdArgs {
    AttnView q, k, v, o, go;
    const float *o_exact;          // [batch][heads][q_len][d], in the place of o, or null
    const float *lse;
    float *delta;                  // [batch][heads][q_len]: D
    const uint8_t *mask;
    long long mask_sb;
    const float *bias;
    int n_off, coord_last, map_w;
    int batch, q_len, k_len, d, heads, kv_heads, group;
    float scale;
    // one of the two owning kernels
    int tiles;
    WorkSplit split;
    __bf16 *out0, *out1;           // dk, dv / dq
    long long o0_sb, o0_st, o0_sh, o1_sb, o1_st, o1_sh;
    float *part0, *part1;          // results of parts: [part row][D]
    float *part_bias;              // sums by distance of one workgroup: a row of whole_len for whole items, of part_len for parts
    int ring, whole_len, part_len, window;
};

// the two rings of a wave lie 36 banks apart: the halves hold distances 4 apart, so that their 64 lanes meet 64 banks
constexpr int kRingPad = 36;
constexpr int kMostRing = 2048;                // positions for the widest map (w = 760: 2 * 128 + 8 + 2 * 128 + 2 w)

// where the sums of a piece start
__device__ __forceinline__ long long part_bias_at(const AttnBwdArgs &a, long long piece)
{
    return piece < a.split.whole ? piece * a.whole_len : (long long)a.split.whole * a.whole_len + (piece - a.split.whole) * a.part_len;
}

// ---- dk, dv ------------------------------------------------------------------------------------------------------------
// A wave owns 32 keys (the result's columns); tiles of 64 queries pass through LDS.  S = Q K^T and dP = dO V^T read the
// tile's rows, dV^T += dO^T P and dK^T += Q^T dS read it transposed.
// Wide heads (D > 64) have no registers for the values beside the keys and both results: their values stay in LDS, and the
// tiles are 32 queries so that two workgroups share a CU.
template <int D>
struct KvLds {
    static constexpr int ROWS = D <= 64 ? kTile : 32;
    static constexpr bool VALUES = D > 64;
    static constexpr int T = Tile<D>::bytes(ROWS), BUF = 2 * T, V = 2 * BUF, STATS = V + (VALUES ? Tile<D>::bytes(kBlockRows) : 0);
    static constexpr int WINDOW = STATS + 2 * 3 * ROWS * 4;
    static constexpr int most(bool biased) { return WINDOW + (biased ? 2 * 2048 * 4 : 0); }
};

template <int D, int BIAS>
__global__ __launch_bounds__(256, 2) void attention_dkv_kernel(AttnBwdArgs a)
{
    using L = KvLds<D>;
    constexpr int NKS = D / 16, NB = D / 32, ROWS = L::ROWS;
    constexpr bool EARLY = D <= 64;                    // wider heads have no registers left to request operands ahead
    extern __shared__ __attribute__((aligned(16))) char smem[];

    // the loop runs over (head of the group, tile of queries)
    const int q_tiles = (a.q_len + ROWS - 1) / ROWS;
    Piece piece;
    if (!work_piece(a.split, a.group * q_tiles, piece)) return;
    const int tile = piece.item % a.tiles, kv_head = piece.item / a.tiles % a.kv_heads, b = piece.item / a.tiles / a.kv_heads;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c32 = lane & 31, half = lane >> 5;
    const int key0 = tile * kBlockRows + wave * 32;
    const int key = key0 + c32 < a.k_len ? key0 + c32 : a.k_len - 1;
    const bool valid = key0 + c32 < a.k_len && (!a.mask || a.mask[b * a.mask_sb + key] != 0);
    const bool busy = __any(valid);

    bf16x8 kf[NKS], vf[L::VALUES ? 1 : NKS];
    {
        const __bf16 *kp = a.k.p + b * a.k.sb + (long long)key * a.k.st + kv_head * a.k.sh;
        const __bf16 *vp = a.v.p + b * a.v.sb + (long long)key * a.v.st + kv_head * a.v.sh;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            const int c = 16 * ks + 8 * half;
            if (valid && c < a.d) {
                kf[ks] = *(const bf16x8 *)(kp + c);
                if constexpr (!L::VALUES) vf[ks] = *(const bf16x8 *)(vp + c);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    kf[ks][e] = (__bf16)0.0f;
                    if constexpr (!L::VALUES) vf[ks][e] = (__bf16)0.0f;
                }
            }
        }
    }
    // distance index = a(query) + c_key; a window starts at the distance of the tile's first query and the workgroup's last key
    const int c_key = BIAS ? a.coord_last - map_coord(key, a.map_w) : 0;
    const int last_key = tile * kBlockRows + kBlockRows - 1 < a.k_len ? tile * kBlockRows + kBlockRows - 1 : a.k_len - 1;
    const int c_low = BIAS ? a.coord_last - map_coord(last_key, a.map_w) : 0;

    f32x16 dk[NB], dv[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) dk[n] = zero16(), dv[n] = zero16();
    const float c2 = a.scale * kLog2e, inv_scale = 1.0f / a.scale;

    const int t0 = piece.t0, t1 = piece.t1;
    const TileLoader<D, ROWS> ql(a.q.st, a.d, wave, lane), gl(a.go.st, a.d, wave, lane);
    float lse_n = 0.0f, delta_n = 0.0f;
    auto fetch = [&](int t) {
        const int head = kv_head * a.group + t / q_tiles, first = t % q_tiles * ROWS;
        char *const qt = smem + (t & 1) * L::BUF;
        ql.load(qt, a.q.p + b * a.q.sb + head * a.q.sh, first, a.q_len, wave, lane);
        gl.load(qt + L::T, a.go.p + b * a.go.sb + head * a.go.sh, first, a.q_len, wave, lane);
        if (BIAS)
            load_window(smem + L::WINDOW + (t & 1) * a.window * 4, a.bias + (long long)head * a.n_off, c_low + map_coord(first, a.map_w),
                        a.window, a.n_off, wave, lane);
        if (wave == 0) {
            // rows beyond the queries, and rows without keys, get an infinite sum: their probabilities are exp2(-inf) = 0
            lse_n = INFINITY;
            delta_n = 0.0f;
            if (lane < ROWS && first + lane < a.q_len) {
                const long long w = ((long long)b * a.heads + head) * a.q_len + first + lane;
                lse_n = a.lse[w];
                delta_n = a.delta[w];
            }
        }
    };
    if (a.d < D) {                                     // channels beyond the head width: zeros that no load overwrites
        clear_lds(smem, L::STATS);
        __syncthreads();
    }
    if constexpr (L::VALUES) {
        const TileLoader<D, kBlockRows> vl(a.v.st, a.d, wave, lane);
        vl.load(smem + L::V, a.v.p + b * a.v.sb + kv_head * a.v.sh, tile * kBlockRows, a.k_len, wave, lane);
    }
    if (t0 < t1) fetch(t0);
    __builtin_amdgcn_s_waitcnt(0x0f70);                // (see the forward kernel)
    TileReader<D> reader(lane);
    for (int t = t0; t < t1; ++t) {
        if constexpr (D > 64) reader.forget();
        char *const qt = smem + (t & 1) * L::BUF, *const gt = qt + L::T;
        float *const lse_s = (float *)(smem + L::STATS) + (t & 1) * 3 * ROWS, *const delta = lse_s + ROWS;
        int *const coord = (int *)(delta + ROWS);
        if (wave == 0 && lane < ROWS) {
            lse_s[lane] = lse_n == -INFINITY ? -INFINITY : -lse_n * inv_scale;
            delta[lane] = -delta_n;
        }
        if (BIAS && tid < ROWS) coord[tid] = map_coord(t % q_tiles * ROWS + tid, a.map_w);      // (queries beyond the last one continue)
        landed();
        __syncthreads();
        // read from LDS by all waves, so that they agree on the barrier below
        const unsigned long long keep = uniform64(__ballot(lane >= ROWS || lse_s[lane & (ROWS - 1)] != -INFINITY));
        if (t + 1 < t1) fetch(t + 1);
        if (keep != ~0ull) {                           // a row without keys gives no gradient whatever q and do hold
            clear_rows<D, ROWS>(qt, keep);
            clear_rows<D, ROWS>(gt, keep);
            __syncthreads();
        }
        const float *const win = (const float *)(smem + L::WINDOW) + (t & 1) * a.window +
                                 (BIAS ? c_key - c_low - map_coord(t % q_tiles * ROWS, a.map_w) : 0);
        if (!busy) continue;
        // Operands are requested one stage ahead of the products that use them, as far as registers allow; fences keep the
        // scheduler from putting each read right before its product.  A wave has priority while it issues products, so that the
        // other wave of its SIMD is pushed towards its arithmetic (3 % of the backward pass at d = 64).  Columns (keys) do not mix, so a masked key's column
        // may hold anything until its result is replaced by zeros at the end.
#pragma unroll
        for (int u = 0; u < ROWS / 32; ++u) {
            bf16x8 qr[NKS], gr[NKS];
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) qr[ks] = reader.rows(qt, 32 * u, ks);
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) gr[ks] = reader.rows(gt, 32 * u, ks);
            // both products start from a row's statistics: s from -lse / scale, dP from -D
            f32x16 s, g;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = lse_s[32 * u + acc_row(r, half)];
                g[r] = delta[32 * u + acc_row(r, half)];
            }
            float bias_of[16];
            if constexpr (BIAS) read_bias<BIAS, 1>(bias_of, win, coord, u, half);
            if constexpr (EARLY) __builtin_amdgcn_sched_barrier(0);
            if constexpr (EARLY) __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) s = mfma(qr[ks], kf[ks], s);
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                if constexpr (L::VALUES) g = mfma(gr[ks], reader.rows(smem + L::V, 32 * wave, ks), g);
                else g = mfma(gr[ks], vf[ks], g);
            }
            if constexpr (EARLY) __builtin_amdgcn_s_setprio(0);
            bf16x8 gx[2][NB], qx[2][NB];
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    gx[w][n] = reader.transposed(gt, 32 * u + 16 * w, n);
                    qx[w][n] = reader.transposed(qt, 32 * u + 16 * w, n);
                }
            if constexpr (EARLY) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = __builtin_amdgcn_exp2f(BIAS ? __builtin_fmaf(s[r], c2, bias_of[r] * kLog2e) : s[r] * c2);
                g[r] *= s[r];
            }
            if constexpr (EARLY) __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const bf16x8 pf = acc_operand(s, w), sf = acc_operand(g, w);
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    dv[n] = mfma(gx[w][n], pf, dv[n]);
                    dk[n] = mfma(qx[w][n], sf, dk[n]);
                }
            }
            if constexpr (EARLY) __builtin_amdgcn_s_setprio(0);
        }
    }
    if (key0 + c32 >= a.k_len) return;
    if (!valid) {                                      // a masked key has no gradient whatever the queries hold
#pragma unroll
        for (int n = 0; n < NB; ++n) dk[n] = zero16(), dv[n] = zero16();
    }
    if (piece.split >= 0) {
        const long long at = (long long)part_row(a.split, piece, wave * 32 + c32) * D;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * n + 8 * g + 4 * half;
                *(f32x4 *)(a.part0 + at + c) = f32x4{dk[n][4 * g], dk[n][4 * g + 1], dk[n][4 * g + 2], dk[n][4 * g + 3]};
                *(f32x4 *)(a.part1 + at + c) = f32x4{dv[n][4 * g], dv[n][4 * g + 1], dv[n][4 * g + 2], dv[n][4 * g + 3]};
            }
        return;
    }
    __bf16 *kp = a.out0 + b * a.o0_sb + (long long)key * a.o0_st + kv_head * a.o0_sh;
    __bf16 *vp = a.out1 + b * a.o1_sb + (long long)key * a.o1_st + kv_head * a.o1_sh;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * n + 8 * g + 4 * half;
            if (c < a.d) {
                bf16x4 x, y;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = (__bf16)(dk[n][4 * g + e] * a.scale), y[e] = (__bf16)dv[n][4 * g + e];
                *(bf16x4 *)(kp + c) = x;
                *(bf16x4 *)(vp + c) = y;
            }
        }
}

// ---- dq, bias ----------------------------------------------------------------------------------------------------------
// A wave owns 32 queries (the result's columns); tiles of 64 keys pass through LDS.  S^T = K Q^T and dP^T = V dO^T read the
// tile's rows, dQ^T += K^T dS^T reads the keys transposed.
//
// The bias gradient is summed by distance.  For one key, the 32 queries of a half wave lie at 32 different distances, so
// each half wave adds its dS values into a ring of float32 sums in LDS of its own without two lanes meeting: plain loads
// and stores, in order within a wave.  (An LDS float atomic takes 81 ns per wave and CU, this 4 ns.)  As the
// keys advance the distances fall: those above a(last row) - a(first key of the next tile) are final (yamd_distance.h), and
// after each tile the workgroup adds the eight rings in a fixed order for them, writes them to its row of the workspace and
// clears them.
// Four queries (lanes 4 i .. 4 i + 3) by four keys (accumulator rows r0 .. r0 + 3), both next to each other: lane 4 i + t
// gets the sum of the diagonal that its own query makes with the first key (near), and of the one four distances below
// (far; nothing for t = 0).  Half the additions to the ring are left.
__device__ __forceinline__ void quad_diagonals(const f32x16 &g, int r0, int lane, float &near, float &far)
{
    const int t = lane & 3;
    const float m1 = t < 3 ? 1.0f : 0.0f, m2 = t < 2 ? 1.0f : 0.0f, m3 = t < 1 ? 1.0f : 0.0f;
    auto from = [&](float v, auto ctrl) {          // the value of lane (t + ctrl's rotation) % 4 of the four
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    const float x1 = from(g[r0 + 1], std::integral_constant<int, 0x39>{}), x2 = from(g[r0 + 2], std::integral_constant<int, 0x4e>{}),
                x3 = from(g[r0 + 3], std::integral_constant<int, 0x93>{});
    near = __builtin_fmaf(x3, m3, __builtin_fmaf(x2, m2, __builtin_fmaf(x1, m1, g[r0])));
    far = __builtin_fmaf(x3, 1.0f - m3, __builtin_fmaf(x2, 1.0f - m2, x1 * (1.0f - m1)));
}

template <int D>
struct QLds {
    static constexpr int T = Tile<D>::bytes(kTile), BUF = 2 * T, COORD = 2 * BUF, KEEP = COORD + 2 * kTile * 4, WINDOW = KEEP + 16;
    static constexpr int most(bool biased) { return WINDOW + (biased ? 2 * 2048 * 4 + 8 * (kMostRing + kRingPad) * 4 : 0); }
};

template <int D, int BIAS>
__global__ __launch_bounds__(256, 2) void attention_dq_kernel(AttnBwdArgs a)
{
    using L = QLds<D>;
    constexpr int NKS = D / 16, NB = D / 32;
    constexpr bool EARLY = D <= 64;                    // wider heads have no registers left to request operands ahead
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float *const rings = (float *)(smem + L::WINDOW) + 2 * a.window;

    Piece piece;
    if (!work_piece(a.split, (a.k_len + kTile - 1) / kTile, piece)) return;
    const int tile = piece.item % a.tiles, head = piece.item / a.tiles % a.heads, b = piece.item / a.tiles / a.heads, kv_head = head / a.group;
    const int t0 = piece.t0, t1 = piece.t1;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c32 = lane & 31, half = lane >> 5;
    const int row0 = tile * kBlockRows + wave * 32;
    const int i = row0 + c32 < a.q_len ? row0 + c32 : a.q_len - 1;
    const long long stat = ((long long)b * a.heads + head) * a.q_len + i;
    const float lse = a.lse[stat];
    const bool valid = row0 + c32 < a.q_len && lse != -INFINITY;
    const float lse2 = valid ? lse * kLog2e : INFINITY;
    const bool busy = __any(valid);

    bf16x8 qf[NKS], gf[NKS];
    {
        const __bf16 *qp = a.q.p + b * a.q.sb + (long long)i * a.q.st + head * a.q.sh;
        const __bf16 *gp = a.go.p + b * a.go.sb + (long long)i * a.go.st + head * a.go.sh;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            const int c = 16 * ks + 8 * half;
            if (valid && c < a.d) {
                qf[ks] = *(const bf16x8 *)(qp + c);
                gf[ks] = *(const bf16x8 *)(gp + c);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) qf[ks][e] = gf[ks][e] = (__bf16)0.0f;
            }
        }
    }
    // D = rowsum(do o); a row without keys (lse = -inf) has no gradient whatever do holds.  An error e of D adds -e P to the row's
    // dS.  Where dS cancels that is felt: with o rounded to bf16 the gradient of a bias bucket that holds most of a row's
    // probability was 5e-3 off, dq of queries with 2 keys 4.9e-3 and with 20 keys 2.8e-3 (2.3e-3 is what the roundings of dS and
    // of dq leave).  So o comes unrounded where the caller has it.
    float delta = 0.0f;
    if (valid) {
        const float *ep = a.o_exact + stat * a.d;
        const __bf16 *op = a.o.p + b * a.o.sb + (long long)i * a.o.st + head * a.o.sh;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            const int c = 16 * ks + 8 * half;
            if (c >= a.d) continue;
            if (a.o_exact) {
                const f32x4 o0 = *(const f32x4 *)(ep + c), o1 = *(const f32x4 *)(ep + c + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) delta += o0[e] * (float)gf[ks][e] + o1[e] * (float)gf[ks][4 + e];
            } else {
                const bf16x8 o = *(const bf16x8 *)(op + c);
#pragma unroll
                for (int e = 0; e < 8; ++e) delta += (float)o[e] * (float)gf[ks][e];
            }
        }
    }
    delta = with_other_half(delta, [](float x, float y) { return x + y; });
    if (half == 0 && row0 + c32 < a.q_len && piece.split <= 0) a.delta[stat] = delta;       // for the other kernel
    const __bf16 *kp = a.k.p + b * a.k.sb + kv_head * a.k.sh, *vp = a.v.p + b * a.v.sb + kv_head * a.v.sh;
    const uint8_t *mp = a.mask ? a.mask + b * a.mask_sb : nullptr;

    // distance index of (query, key) = cq - a(key); of the workgroup's first row
    int cq = 0, c_first = 0, high = 0;
    float *ring = nullptr;
    auto final_at = [&](int t) { return final_from(tile, t * kTile, a.coord_last, a.map_w); };
    if constexpr (BIAS) {
        cq = a.coord_last + map_coord(row0 + c32, a.map_w);    // (lanes beyond the queries too have distances of their own)
        c_first = a.coord_last + map_coord(tile * kBlockRows, a.map_w);
        high = final_at(t0);                                   // distances from here on are written out
        ring = rings + (2 * wave + half) * (a.ring + kRingPad);
        for (int e = tid; e < 8 * (a.ring + kRingPad); e += 256) rings[e] = 0.0f;
    }

    f32x16 dq[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) dq[n] = zero16();
    const float c2 = a.scale * kLog2e;

    auto window_from = [&](int t) { return c_first - map_coord(t * kTile + kTile - 1, a.map_w); };
    const TileLoader<D> kl(a.k.st, a.d, wave, lane), vl(a.v.st, a.d, wave, lane);
    unsigned char mask_n = 1;
    auto fetch = [&](int t) {
        char *const kt = smem + (t & 1) * L::BUF;
        kl.load(kt, kp, t * kTile, a.k_len, wave, lane);
        vl.load(kt + L::T, vp, t * kTile, a.k_len, wave, lane);
        if (BIAS)
            load_window(smem + L::WINDOW + (t & 1) * a.window * 4, a.bias + (long long)head * a.n_off, window_from(t), a.window, a.n_off,
                        wave, lane);
        if (mp && wave == 0 && t * kTile + lane < a.k_len) mask_n = mp[t * kTile + lane];
    };
    // coordinate of the last key that the workgroup walks
    const int end_key = t1 * kTile < a.k_len ? t1 * kTile : a.k_len, coord_end = BIAS ? map_coord(end_key - 1, a.map_w) : 0;
    // writes the sums of the distances [low, high) out and clears them
    auto flush = [&](int low) {
        float *out = a.part_bias + part_bias_at(a, piece.index);
        const int base = c_first - coord_end;          // the smallest distance of the workgroup: first query, last key
        for (int e = low + tid; e < high; e += 256) {
            const int at = e & (a.ring - 1);
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                s += rings[w * (a.ring + kRingPad) + at];
                rings[w * (a.ring + kRingPad) + at] = 0.0f;
            }
            out[e - base] = s;
        }
        high = low;
    };
    if (a.d < D) {                                     // channels beyond the head width: zeros that no load overwrites
        clear_lds(smem, 2 * L::BUF);
        __syncthreads();
    }
    if (t0 < t1) fetch(t0);
    __builtin_amdgcn_s_waitcnt(0x0f70);                // (see the forward kernel)
    TileReader<D> reader(lane);
    for (int t = t0; t < t1; ++t) {
        if constexpr (D > 64) reader.forget();
        char *const kt = smem + (t & 1) * L::BUF, *const vt = kt + L::T;
        int *const coord = (int *)(smem + L::COORD) + (t & 1) * kTile;
        unsigned long long *const kept = (unsigned long long *)(smem + L::KEEP) + (t & 1);
        if (BIAS && tid < kTile) coord[tid] = map_coord(t * kTile + tid, a.map_w);      // (keys beyond the last one continue)
        if (mp && wave == 0) {
            const unsigned long long v = __ballot(mask_n != 0);
            if (lane == 0) *kept = v;
        }
        landed();
        __syncthreads();
        unsigned long long keep = rows_below(t * kTile, a.k_len);
        if (mp) keep &= *kept;                         // (from LDS: all waves agree on the barrier below)
        keep = uniform64(keep);
        if (t + 1 < t1) fetch(t + 1);
        if (BIAS && a.part_bias) flush(final_at(t));   // what the tiles before this one left final
        if (keep == 0) continue;
        if (keep != ~0ull) {                           // a masked key may hold anything, NaN included
            clear_rows<D>(kt, keep);
            clear_rows<D>(vt, keep);
            __syncthreads();
        }
        if (!busy) continue;
        const float *const win = (const float *)(smem + L::WINDOW) + (t & 1) * a.window + (BIAS ? cq - window_from(t) : 0);
        // The additions to the ring stand between the products, which hide part of their latency.  Narrow heads take both
        // halves of the tile at once and make two additions at a time: keys 32 apart never put two lanes at one distance,
        // because 32 queries are less than 32 apart.
        constexpr int U = EARLY ? 2 : 1;
        auto add = [&](const int (&d)[U], const float (&v)[U]) {
            float *p[U], x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) p[u] = ring + (d[u] & (a.ring - 1));
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = *p[u];
#pragma unroll
            for (int u = 0; u < U; ++u) *p[u] = x[u] + v[u];
            asm volatile("" ::: "memory");                   // the next addition may read what another lane wrote here
        };
#pragma unroll
        for (int u0 = 0; u0 < 2; u0 += U) {
            bf16x8 kr[U][NKS], vr[U][NKS];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int ks = 0; ks < NKS; ++ks) {
                    kr[u][ks] = reader.rows(kt, 32 * (u0 + u), ks);
                    vr[u][ks] = reader.rows(vt, 32 * (u0 + u), ks);
                }
            if constexpr (EARLY) __builtin_amdgcn_sched_barrier(0);
            if constexpr (EARLY) __builtin_amdgcn_s_setprio(1);
            f32x16 s[U], g[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[u] = zero16(), g[u] = zero16();
#pragma unroll
                for (int ks = 0; ks < NKS; ++ks) s[u] = mfma(kr[u][ks], qf[ks], s[u]);
#pragma unroll
                for (int ks = 0; ks < NKS; ++ks) g[u] = mfma(vr[u][ks], gf[ks], g[u]);
            }
            if constexpr (EARLY) __builtin_amdgcn_s_setprio(0);
            bf16x8 kx[2 * U][NB];
#pragma unroll
            for (int w = 0; w < 2 * U; ++w)
#pragma unroll
                for (int n = 0; n < NB; ++n) kx[w][n] = reader.transposed(kt, 32 * u0 + 16 * w, n);
            if constexpr (EARLY) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < U; ++u) {                    // g: dP to dS
                float x[16];
                if constexpr (BIAS) {
                    read_bias<BIAS, -1>(x, win, coord, u0 + u, half);
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[r] = __builtin_fmaf(x[r], kLog2e, -lse2);
                }
                if (keep != ~0ull) mask_rows(s[u], keep, u0 + u, half);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    g[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], c2, BIAS ? x[r] : -lse2)) * (g[u][r] - delta);
                if constexpr (EARLY && BIAS) __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (EARLY) __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int w = 0; w < 2 * U; ++w) {
                const bf16x8 sf = acc_operand(g[w >> 1], w & 1);
#pragma unroll
                for (int n = 0; n < NB; ++n) dq[n] = mfma(kx[w][n], sf, dq[n]);
                // accumulator rows that go to the ring beside this product
                constexpr int PER = 16 / (2 * U);
#pragma unroll
                for (int r = PER * w; BIAS && r < PER * w + PER; r += BIAS == kQuadBias ? 4 : 1) {
                    if (!a.part_bias) break;                 // a bias without gradient
                    int d[U];
                    float v[U], far[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        d[u] = cq - coord[32 * (u0 + u) + acc_row(r, half)];
                        v[u] = g[u][r];
                        if constexpr (BIAS == kQuadBias) quad_diagonals(g[u], r, lane, v[u], far[u]);
                    }
                    add(d, v);
                    if constexpr (BIAS == kQuadBias) {
#pragma unroll
                        for (int u = 0; u < U; ++u) d[u] -= 4;
                        add(d, far);
                    }
                }
            }
            if constexpr (EARLY) __builtin_amdgcn_s_setprio(0);
        }
    }
    if (BIAS && a.part_bias) {
        __syncthreads();
        flush(c_first - coord_end);
    }
    if (row0 + c32 >= a.q_len) return;
    if (piece.split >= 0) {
        const long long at = (long long)part_row(a.split, piece, wave * 32 + c32) * D;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *(f32x4 *)(a.part0 + at + 32 * n + 8 * g + 4 * half) =
                    f32x4{dq[n][4 * g], dq[n][4 * g + 1], dq[n][4 * g + 2], dq[n][4 * g + 3]};
        return;
    }
    __bf16 *op = a.out0 + b * a.o0_sb + (long long)i * a.o0_st + head * a.o0_sh;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * n + 8 * g + 4 * half;
            if (c < a.d) {
                bf16x4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = (__bf16)(dq[n][4 * g + e] * a.scale);
                *(bf16x4 *)(op + c) = x;
            }
        }
}

// Adds the workgroups' sums by distance: 64 distances x 16 waves per workgroup, a wave takes every 16th of a head's (tile, image)
// pairs and a tree in LDS adds the sixteen.  Which distances a piece has written follows from the coordinates of its rows and
// keys; those need divisions, which would be most of the kernel if each pair made its own, so the lanes work them out for 64
// tiles at a time (832 items of 40 x 40 tokens: 16 us, 23 us without).
__global__ __launch_bounds__(1024) void attention_bias_grad_kernel(AttnBwdArgs a, float *dbias)
{
    __shared__ float part[16][64];
    const int x = threadIdx.x & 63, y = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), off = blockIdx.x * 64 + x, head = blockIdx.y;
    const int per = a.split.per_split * kTile, step_t = 16 / a.batch, step_b = 16 % a.batch;
    float s = 0.0f;
    auto add = [&](long long at, int base, int top) {
        if (off >= base && off <= top) s += a.part_bias[at + off - base];
    };
    for (int t0 = 0; t0 < a.tiles; t0 += 64) {
        const int row = (t0 + x < a.tiles ? t0 + x : a.tiles - 1) * kBlockRows;
        const int first = a.coord_last + map_coord(row, a.map_w);
        const int last = a.coord_last + map_coord(row + kBlockRows < a.q_len ? row + kBlockRows - 1 : a.q_len - 1, a.map_w);
        const int n = a.tiles - t0 < 64 ? a.tiles - t0 : 64;
        for (int t = y / a.batch, b = y % a.batch; t < n;) {
            const int c_first = __builtin_amdgcn_readlane(first, t), c_last = __builtin_amdgcn_readlane(last, t);
            const int item = (b * a.heads + head) * a.tiles + t0 + t;
            if (item < a.split.whole) {
                add((long long)item * a.whole_len, c_first - a.coord_last, c_last);
            } else {
                for (int k = 0; k < a.split.splits; ++k) {
                    const int k0 = k * per, k1 = k0 + per < a.k_len ? k0 + per : a.k_len;
                    add(part_bias_at(a, a.split.whole + (long long)(item - a.split.whole) * a.split.splits + k),
                        c_first - map_coord(k1 - 1, a.map_w), c_last - map_coord(k0, a.map_w));
                }
            }
            t += step_t;
            b += step_b;
            if (b >= a.batch) {
                b -= a.batch;
                ++t;
            }
        }
    }
    part[y][x] = s;
    __syncthreads();
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) {
        if (y < d) part[y][x] += part[y + d][x];
        __syncthreads();
    }
    if (y == 0 && off < a.n_off) dbias[(long long)head * a.n_off + off] = part[0][x];
}

// Adds the parts of split results and rounds them; blockIdx.y picks one of up to three results, so that a backward pass needs
// one launch for all of them (3 images of 1447 tokens, 6 heads, d 64, forward and
// backward: 145 us instead of 152 with a launch each).
struct SumOf {
    const float *parts;
    WorkSplit split;
    int tiles, heads, len;
    float scale;
    __bf16 *out;
    long long sb, st, sh;
};
struct SumArgs {
    SumOf of[3];
    int n, d;
};

template <int D>
__global__ __launch_bounds__(256) void attention_sum_parts_kernel(SumArgs args)
{
    const SumOf a = args.of[blockIdx.y];
    const int id = blockIdx.x * 256 + threadIdx.x, at = id / (D / 4), c = id % (D / 4) * 4, rows = a.split.part_rows();
    if (at >= rows || c >= args.d) return;
    const int item = a.split.whole + at / a.split.tile_rows, t = item % a.tiles * kBlockRows + at % a.split.tile_rows;
    if (t >= a.len) return;
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < a.split.splits; ++k) s += *(const f32x4 *)(a.parts + (long long)(k * rows + at) * D + c);
    const int head = item / a.tiles % a.heads, b = item / a.tiles / a.heads;
    bf16x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (__bf16)(s[e] * a.scale);
    *(bf16x4 *)(a.out + b * a.sb + (long long)t * a.st + head * a.sh + c) = o;
}

namespace {

struct BwdPlan {
    int dpad, kv_tiles, q_tiles, ring, whole_len, part_len;
    WorkSplit kv, q;
    size_t delta, kv_parts, q_parts, bias, workspace;     // bytes
};

size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

// only a bias whose gradient is wanted has sums to keep
BwdPlan plan_backward(const yamd_attention_desc *d, bool biased, bool bias_gradient)
{
    BwdPlan p = {};
    p.dpad = padded_head_dim(d->head_dim);
    const long long bh = (long long)d->batch * d->heads, bk = (long long)d->batch * d->kv_heads;
    const int kt = ceil_div(d->k_len, kTile), qt = ceil_div(d->q_len, p.dpad <= 64 ? kTile : 32) * (d->heads / d->kv_heads);
    p.kv_tiles = ceil_div(d->k_len, kBlockRows);
    p.q_tiles = ceil_div(d->q_len, kBlockRows);
    p.kv = split_work(bk * p.kv_tiles, qt, d->k_len, p.dpad == 32 ? 4 : 2, 2, 2.5f);
    p.q = split_work(bh * p.q_tiles, kt, d->q_len, p.dpad == 32 ? 3 : 2, 1, 2.5f);
    p.delta = up256((size_t)bh * d->q_len * sizeof(float));
    p.kv_parts = up256(2 * (size_t)p.kv.splits * p.kv.part_rows() * p.dpad * sizeof(float));
    p.q_parts = up256((size_t)p.q.splits * p.q.part_rows() * p.dpad * sizeof(float));
    if (biased) {
        p.ring = ring_len(d->map_h, d->map_w);
        p.whole_len = distances_of(d->k_len, d->map_h, d->map_w);
        p.part_len = distances_of(p.q.per_split * kTile < d->k_len ? p.q.per_split * kTile : d->k_len, d->map_h, d->map_w);
        if (bias_gradient) p.bias = up256(((size_t)p.q.whole * p.whole_len + (size_t)p.q.rest * p.q.splits * p.part_len) * sizeof(float));
    }
    p.workspace = p.delta + p.kv_parts + p.q_parts + p.bias;
    return p;
}

template <int D, int BIAS>
int launch_backward(AttnBwdArgs a, const BwdPlan &p, const yamd_tokens *dq, const yamd_tokens *dk, const yamd_tokens *dv, float *dbias,
                    hipStream_t st)
{
    using KvAttr = KernelAttr<&attention_dkv_kernel<D, BIAS>, KvLds<D>::most(BIAS)>;
    using QAttr = KernelAttr<&attention_dq_kernel<D, BIAS>, QLds<D>::most(BIAS)>;
    int rc = KvAttr::ensure();
    if (rc == YAMD_OK) rc = QAttr::ensure();
    if (rc != YAMD_OK) return rc;
    SumArgs sums = {};
    sums.d = a.d;
    // queries first: their kernel leaves D for the other one
    AttnBwdArgs wq = a;
    wq.tiles = p.q_tiles; wq.split = p.q;
    wq.out0 = (__bf16 *)dq->data; wq.o0_sb = dq->batch_stride; wq.o0_st = dq->token_stride; wq.o0_sh = dq->head_stride;
    wq.part0 = a.delta + (p.delta + p.kv_parts) / sizeof(float);
    hipLaunchKernelGGL((attention_dq_kernel<D, BIAS>), dim3(wq.split.grid()), dim3(256),
                       QLds<D>::WINDOW + (BIAS ? 2 * a.window + 8 * (p.ring + kRingPad) : 0) * (int)sizeof(float), st, wq);
    YAMD_LAUNCH_CHECK();
    if (wq.split.rest) sums.of[sums.n++] = {wq.part0, wq.split, wq.tiles, a.heads, a.q_len, a.scale, wq.out0, wq.o0_sb, wq.o0_st, wq.o0_sh};

    AttnBwdArgs wk = a;
    wk.tiles = p.kv_tiles; wk.split = p.kv;
    wk.out0 = (__bf16 *)dk->data; wk.o0_sb = dk->batch_stride; wk.o0_st = dk->token_stride; wk.o0_sh = dk->head_stride;
    wk.out1 = (__bf16 *)dv->data; wk.o1_sb = dv->batch_stride; wk.o1_st = dv->token_stride; wk.o1_sh = dv->head_stride;
    wk.part0 = a.delta + p.delta / sizeof(float);
    wk.part1 = wk.part0 + (size_t)p.kv.splits * p.kv.part_rows() * D;
    hipLaunchKernelGGL((attention_dkv_kernel<D, BIAS>), dim3(wk.split.grid()), dim3(256), KvLds<D>::WINDOW + 2 * a.window * (int)sizeof(float), st, wk);
    YAMD_LAUNCH_CHECK();
    if (wk.split.rest) {
        sums.of[sums.n++] = {wk.part0, wk.split, wk.tiles, a.kv_heads, a.k_len, a.scale, wk.out0, wk.o0_sb, wk.o0_st, wk.o0_sh};
        sums.of[sums.n++] = {wk.part1, wk.split, wk.tiles, a.kv_heads, a.k_len, 1.0f, wk.out1, wk.o1_sb, wk.o1_st, wk.o1_sh};
    }
    if (sums.n) {
        int most = 0;
        for (const SumOf &o : sums.of) most = o.split.part_rows() > most ? o.split.part_rows() : most;
        hipLaunchKernelGGL(attention_sum_parts_kernel<D>, dim3(ceil_div(most * (D / 4), 256), sums.n), dim3(256), 0, st, sums);
        YAMD_LAUNCH_CHECK();
    }
    if (BIAS && dbias) {
        hipLaunchKernelGGL(attention_bias_grad_kernel, dim3(ceil_div(a.n_off, 64), a.heads), dim3(1024), 0, st, wq, dbias);
        YAMD_LAUNCH_CHECK();
    }
    return YAMD_OK;
}

template <int D>
int launch_backward(Bias form, const AttnBwdArgs &a, const BwdPlan &p, const yamd_tokens *dq, const yamd_tokens *dk, const yamd_tokens *dv,
                    float *dbias, hipStream_t st)
{
    if (form == kQuadBias) return launch_backward<D, kQuadBias>(a, p, dq, dk, dv, dbias, st);
    return form == kAnyBias ? launch_backward<D, kAnyBias>(a, p, dq, dk, dv, dbias, st)
                            : launch_backward<D, kNoBias>(a, p, dq, dk, dv, dbias, st);
}

}  // namespace
}  // namespace yamd

using namespace yamd;

extern "C" size_t yamd_attention_backward_workspace_bytes(const yamd_attention_desc *d, int bias_gradient)
{
    if (check_attention(d, nullptr, 0, nullptr) != YAMD_OK) return 0;
    if (bias_gradient && (d->map_h <= 0 || d->map_w <= 0 || (long long)d->map_h * d->map_w != d->k_len)) return 0;
    return plan_backward(d, bias_gradient != 0, bias_gradient != 0).workspace;
}

extern "C" int yamd_attention_backward(const yamd_attention_desc *d, const yamd_tokens *q, const yamd_tokens *k, const yamd_tokens *v,
                                       const uint8_t *key_mask, long long mask_stride, const float *bias, const yamd_tokens *o,
                                       const float *o_exact, const float *lse, const yamd_tokens *d_o, const yamd_tokens *dq, const yamd_tokens *dk,
                                       const yamd_tokens *dv, float *dbias, void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = check_attention(d, key_mask, mask_stride, bias);
    if (rc == YAMD_OK) rc = check_tokens(d, q, d->q_len, d->heads, "q");
    if (rc == YAMD_OK) rc = check_tokens(d, k, d->k_len, d->kv_heads, "k");
    if (rc == YAMD_OK) rc = check_tokens(d, v, d->k_len, d->kv_heads, "v");
    if (rc == YAMD_OK && (o || !o_exact)) rc = check_tokens(d, o, d->q_len, d->heads, "o");
    if (rc == YAMD_OK) rc = check_tokens(d, d_o, d->q_len, d->heads, "do");
    if (rc == YAMD_OK) rc = check_result(d, dq, d->q_len, d->heads, "dq");
    if (rc == YAMD_OK) rc = check_result(d, dk, d->k_len, d->kv_heads, "dk");
    if (rc == YAMD_OK) rc = check_result(d, dv, d->k_len, d->kv_heads, "dv");
    if (rc != YAMD_OK) return rc;
    YAMD_REQUIRE(lse, "attention backward: lse is null");
    YAMD_REQUIRE(!dbias || bias, "attention backward: a bias gradient without a bias");
    YAMD_REQUIRE(!dbias || o_exact, "attention backward: a bias gradient needs o_exact");
    YAMD_REQUIRE(((uintptr_t)o_exact & 15) == 0, "attention backward: o_exact is not 16-byte aligned");
    const BwdPlan p = plan_backward(d, bias != nullptr, dbias != nullptr);
    if (!workspace || workspace_bytes < p.workspace || ((uintptr_t)workspace & 15)) {
        set_error("attention backward: workspace of %zu bytes, needs %zu (16-byte aligned)", workspace ? workspace_bytes : (size_t)0, p.workspace);
        return YAMD_ENOSPC;
    }
    AttnBwdArgs a = {};
    a.q = view_of(q); a.k = view_of(k); a.v = view_of(v); a.go = view_of(d_o);
    if (o) a.o = view_of(o);
    a.lse = lse;
    a.delta = (float *)workspace;
    a.part_bias = dbias ? (float *)((char *)workspace + p.delta + p.kv_parts + p.q_parts) : nullptr;
    a.o_exact = o_exact;
    a.ring = p.ring;
    a.whole_len = p.whole_len;
    a.part_len = p.part_len;
    a.mask = key_mask; a.mask_sb = mask_stride; a.bias = bias;
    if (bias) {
        a.map_w = d->map_h > 1 ? d->map_w : 1;       // (of a sequence the coordinate is the position, also beyond its end)
        a.coord_last = map_coord(d->k_len - 1, a.map_w);
        a.n_off = 2 * a.coord_last + 1;
        a.window = window_len(d->map_h, d->map_w);
    }
    a.batch = d->batch; a.q_len = d->q_len; a.k_len = d->k_len; a.d = d->head_dim;
    a.heads = d->heads; a.kv_heads = d->kv_heads; a.group = d->heads / d->kv_heads; a.scale = d->scale;
    hipStream_t st = (hipStream_t)stream;
    const Bias form = bias_form(bias, d->map_h, d->map_w);
    switch (p.dpad) {
    case 32: return launch_backward<32>(form, a, p, dq, dk, dv, dbias, st);
    case 64: return launch_backward<64>(form, a, p, dq, dk, dv, dbias, st);
    case 96: return launch_backward<96>(form, a, p, dq, dk, dv, dbias, st);
    default: return launch_backward<128>(form, a, p, dq, dk, dv, dbias, st);
    }
}
