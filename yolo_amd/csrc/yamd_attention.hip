// Attention over tokens, forward: o = softmax(scale q k^T + bias) v, bf16 operands, float32 statistics and sums.
//
// A wave owns 32 query rows and keeps them in registers as the B operand; a workgroup of four waves walks the keys in tiles
// of 64 that pass through LDS (two buffers, the next tile's loads in flight under the current one's arithmetic).  The
// products are taken transposed, S^T = K Q^T and O^T = V^T P^T: a lane then owns one query, its running maximum, sum and
// rescaling are scalars of the lane, one exchange between the two halves of the wave completes a maximum, and the
// probabilities are the second product's B operand in the registers where they were computed (yamd_attention.h).
// Probabilities are rounded to bf16 for the second product only (their sum is taken before, in float32): the error of o is
// at most 2^-8 of the weighted mean of |v|, below the rounding of o itself in all but contrived cases.
//
// The backward pass needs o more exactly than that (yamd_attention_backward.hip): with o_exact the second product runs twice,
// for the probabilities rounded to bf16 and for what the rounding left (2^-17 of them is lost), and o is also written in
// float32.  Without a bias only few keys need the second product: what the probabilities of many lose averages out (error of
// dq with one product and with two: 2 keys 2.59e-3 and 2.33e-3, 64 keys 2.40e-3 and 2.36e-3, 600 keys 2.39e-3 and 2.37e-3).
//
// Few query rows: heads that share keys are packed into one tile of rows (row = head in group * q_len + query), and the
// keys are split over workgroups whose float32 parts a second kernel joins.
//
// What bounds it: at d = 64 the vector unit (72 % busy, of which more than half are exponentials, quarter rate; matrix unit
// 39 %): 2 images of 8 heads, 6400 x 6400 tokens take 210 us, 800 TFLOP/s; with a bias 256 us, and 338 us with the second
// product (78 %, the bias adds a load and an addition per score).  At d = 128 nothing is full (vector 45 %, matrix 38 %, two waves per SIMD):
// 375 - 385 us, 870 - 895 TFLOP/s; requesting operands ahead in a ring of registers did not help (386 us against 381 on one card).  One
// query of 8 images on 8400 keys, d 64, moves 69 MB in 18 us with the join.
#include "yamd_attention.h"

#include <algorithm>
#include <cmath>

namespace yamd {

struct AttnFwdArgs {
    AttnView q, k, v;
    __bf16 *o;
    long long o_sb, o_st, o_sh;
    float *o_exact;                // [batch][heads][q_len][d], o before rounding, or null (see below)
    float *lse;                    // [batch][heads][q_len], natural logarithm, or null
    const uint8_t *mask;           // [batch][k_len], 0 = not attended, or null
    long long mask_sb;
    const float *bias;             // [heads][(2 h - 1)(2 w - 1)]
    int n_off, coord_last, map_w, window;
    int batch, q_len, k_len, d, heads, kv_heads, group;
    int packed, rows, q_tiles, grid_heads;
    WorkSplit split;
    float scale;
    float *part_o, *part_ml;       // results of parts: [part row][D] and [part row][2]
};

// LDS: two buffers of a tile of keys and one of values; then the coordinates and the mask of the two tiles' rows, and two
// windows of the bias
template <int D>
struct FwdLds {
    static constexpr int K = Tile<D>::bytes(kTile), BUF = 2 * K, COORD = 2 * BUF, KEEP = COORD + 2 * kTile * 4, WINDOW = KEEP + 16;
    static constexpr int most(bool biased) { return WINDOW + (biased ? 2 * 2048 * 4 : 0); }
};

// EXACT: the second product runs twice
template <int D, int BIAS, bool EXACT>
__global__ __launch_bounds__(256, (D == 64 ? 3 : 2)) void attention_kernel(AttnFwdArgs a)
{
    using L = FwdLds<D>;
    constexpr int NKS = D / 16, NB = D / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];

    Piece piece;
    if (!work_piece(a.split, (a.k_len + kTile - 1) / kTile, piece)) return;
    const int q_tile = piece.item % a.q_tiles, gh = piece.item / a.q_tiles % a.grid_heads, b = piece.item / a.q_tiles / a.grid_heads;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c32 = lane & 31, half = lane >> 5;
    const int row0 = q_tile * kBlockRows + wave * 32;
    const int row = row0 + c32 < a.rows ? row0 + c32 : a.rows - 1;     // lanes beyond the rows repeat the last one
    const int in_group = a.packed ? row / a.q_len : 0;
    const int i = row - in_group * a.q_len;
    const int head = a.packed ? gh * a.group + in_group : gh;
    const int kv_head = a.packed ? gh : gh / a.group;

    bf16x8 qf[NKS];
    {
        const __bf16 *qp = a.q.p + b * a.q.sb + (long long)i * a.q.st + head * a.q.sh;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            const int c = 16 * ks + 8 * half;
            if (c < a.d) qf[ks] = *(const bf16x8 *)(qp + c);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) qf[ks][e] = (__bf16)0.0f;
        }
    }
    const __bf16 *kp = a.k.p + b * a.k.sb + kv_head * a.k.sh, *vp = a.v.p + b * a.v.sb + kv_head * a.v.sh;
    const uint8_t *mp = a.mask ? a.mask + b * a.mask_sb : nullptr;
    f32x16 acc[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[n] = zero16();
    float m = -INFINITY, l = 0.0f;                       // running maximum (units of log 2) and this half's sum
    const float c2 = a.scale * kLog2e;

    const int t0 = piece.t0, t1 = piece.t1;

    // distance index = c_row - a(key); a window starts at the distance of the workgroup's first row and the tile's last key
    const float *bias = BIAS ? a.bias + (long long)gh * a.n_off : nullptr;
    const int c_row = BIAS ? a.coord_last + map_coord(i, a.map_w) : 0;
    const int c_first = BIAS ? a.coord_last + map_coord(q_tile * kBlockRows, a.map_w) : 0;
    auto window_from = [&](int t) { return c_first - map_coord(t * kTile + kTile - 1, a.map_w); };
    const TileLoader<D> kl(a.k.st, a.d, wave, lane), vl(a.v.st, a.d, wave, lane);
    unsigned char mask_n = 1;
    auto fetch = [&](int t) {
        char *const kt = smem + (t & 1) * L::BUF;
        kl.load(kt, kp, t * kTile, a.k_len, wave, lane);
        vl.load(kt + L::K, vp, t * kTile, a.k_len, wave, lane);
        if (BIAS) load_window(smem + L::WINDOW + (t & 1) * a.window * 4, bias, window_from(t), a.window, a.n_off, wave, lane);
        if (mp && wave == 0 && t * kTile + lane < a.k_len) mask_n = mp[t * kTile + lane];
    };
    if (a.d < D) {                                       // channels beyond the head width: zeros that no load overwrites
        clear_lds(smem, 2 * L::BUF);
        __syncthreads();
    }
    if (t0 < t1) fetch(t0);
    // (a wait that the compiler sees: it would otherwise wait for the query rows inside the loop, and for the tiles with them)
    __builtin_amdgcn_s_waitcnt(0x0f70);
    TileReader<D> reader(lane);
    for (int t = t0; t < t1; ++t) {
        if constexpr (D > 64) reader.forget();
        char *const kt = smem + (t & 1) * L::BUF, *const vt = kt + L::K;
        int *const coord = (int *)(smem + L::COORD) + (t & 1) * kTile;
        unsigned long long *const kept = (unsigned long long *)(smem + L::KEEP) + (t & 1);
        if (BIAS && tid < kTile) coord[tid] = map_coord(t * kTile + tid, a.map_w);       // (keys beyond the last one continue)
        if (mp && wave == 0) {
            const unsigned long long v = __ballot(mask_n != 0);
            if (lane == 0) *kept = v;
        }
        landed();
        __syncthreads();
        // the mask that all waves act on is the one in LDS, so they agree on the barrier below whatever memory holds
        unsigned long long keep = rows_below(t * kTile, a.k_len);
        if (mp) keep &= *kept;
        keep = uniform64(keep);
        if (t + 1 < t1) fetch(t + 1);
        if (keep == 0) continue;
        if (keep != ~0ull) {                             // a masked key may hold anything, NaN included
            clear_rows<D>(kt, keep);
            clear_rows<D>(vt, keep);
            __syncthreads();
        }
        if (row0 >= a.rows) continue;

        // operands are requested well ahead of the products that use them (the scheduler would put each read right before
        // its product); the loads of the bias are in flight under the first product, those of half the values under the
        // softmax
        constexpr bool EARLY = D <= 64;                  // wider heads have no registers left for it
        f32x16 s[2];
        bf16x8 kf[2][NKS];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) kf[u][ks] = reader.rows(kt, 32 * u, ks);
        float bias_of[2][16];
        if constexpr (BIAS) {
            const float *const w = (const float *)(smem + L::WINDOW) + (t & 1) * a.window + (c_row - window_from(t));
            read_bias<BIAS, -1>(bias_of[0], w, coord, 0, half);
            read_bias<BIAS, -1>(bias_of[1], w, coord, 1, half);
        }
        if constexpr (EARLY) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            s[u] = zero16();
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) s[u] = mfma(kf[u][ks], qf[ks], s[u]);
        }
        bf16x8 vf[2][NB];
        auto read_values = [&](bf16x8 (&f)[2][NB], int from) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int n = 0; n < NB; ++n) f[u][n] = reader.transposed(vt, from + 16 * u, n);
        };
        if constexpr (EARLY) read_values(vf, 0);
        if constexpr (EARLY) __builtin_amdgcn_sched_barrier(0);
        if constexpr (BIAS) {
#pragma unroll
            for (int r = 0; r < 32; ++r) s[r >> 4][r & 15] = __builtin_fmaf(s[r >> 4][r & 15], a.scale, bias_of[r >> 4][r & 15]);
        }
        if (keep != ~0ull) {
            mask_rows(s[0], keep, 0, half);
            mask_rows(s[1], keep, 1, half);
        }
        float top = s[0][0];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
        top = with_other_half(top, [](float x, float y) { return fmaxf(x, y); });
        const float unit = BIAS ? kLog2e : c2;           // scores to units of log 2
        top *= unit;
        // a tile of masking biases only: no maximum yet (differences of such numbers would mean nothing)
        if (BIAS && top < kMasked * kLog2e) top = -INFINITY;
        if (__any(top > m)) {
            const float m_new = fmaxf(m, top);
            const float f = __builtin_amdgcn_exp2f(m - (m_new == -INFINITY ? 0.0f : m_new));
            m = m_new;
            l *= f;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[n][r] *= f;
        }
        const float sub = m == -INFINITY ? 0.0f : m;     // rows without a key so far: every term below is exp2(-inf) = 0
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], unit, -sub));
                l += s[u][r];
            }
        bf16x8 vg[2][NB];
        if constexpr (EARLY) read_values(vg, 32);
        else read_values(vf, 0);
        if constexpr (EARLY) __builtin_amdgcn_sched_barrier(0);
        auto add_values = [&](const f32x16 &p, const bf16x8 (&f)[2][NB]) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const bf16x8 pf = acc_operand(p, u);
#pragma unroll
                for (int n = 0; n < NB; ++n) acc[n] = mfma(f[u][n], pf, acc[n]);
                if constexpr (EXACT) {
                    bf16x8 rest;
#pragma unroll
                    for (int e = 0; e < 8; ++e) rest[e] = (__bf16)(p[8 * u + e] - (float)pf[e]);
#pragma unroll
                    for (int n = 0; n < NB; ++n) acc[n] = mfma(f[u][n], rest, acc[n]);
                }
            }
        };
        add_values(s[0], vf);
        if constexpr (!EARLY) read_values(vg, 32);
        add_values(s[1], vg);
    }
    l = with_other_half(l, [](float x, float y) { return x + y; });
    if (row0 + c32 >= a.rows) return;
    if (piece.split >= 0) {
        const long long at = part_row(a.split, piece, wave * 32 + c32);
        if (half == 0) *(float2 *)(a.part_ml + 2 * at) = make_float2(m, l);
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 o = {acc[n][4 * g], acc[n][4 * g + 1], acc[n][4 * g + 2], acc[n][4 * g + 3]};
                *(f32x4 *)(a.part_o + at * D + 32 * n + 8 * g + 4 * half) = o;
            }
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    __bf16 *op = a.o + b * a.o_sb + (long long)i * a.o_st + head * a.o_sh;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * n + 8 * g + 4 * half;
            if (c < a.d) {
                bf16x4 o;
                f32x4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = acc[n][4 * g + e] * inv;
                    o[e] = (__bf16)x[e];
                }
                *(bf16x4 *)(op + c) = o;
                if (a.o_exact) *(f32x4 *)(a.o_exact + (((long long)b * a.heads + head) * a.q_len + i) * a.d + c) = x;
            }
        }
    if (a.lse && half == 0)
        a.lse[((long long)b * a.heads + head) * a.q_len + i] = l == 0.0f ? -INFINITY : (m + __builtin_log2f(l)) * 0.6931471805599453f;
}

// Joins the parts of a split key axis.  A lane owns 4 channels of a row and takes its parts four at a time, so that their
// loads overlap.  With many parts a wave works on one row: its 64 / (D / 4) groups of lanes take the parts in turns and are
// joined by exchanges in a fixed order (33 parts of 2400 rows, D 32: 4 us against 18 without); with up to 8 parts the groups
// take a row each (3 parts of 26046 rows, D 64: 7 us against 14).
template <int D>
constexpr int kJoinLanes = D == 96 ? 32 : D / 4;               // (of 32 lanes 24 work for D = 96)
template <int D, bool SHARED>
__global__ __launch_bounds__(256) void attention_join_kernel(AttnFwdArgs a)
{
    constexpr int CH = kJoinLanes<D>, G = SHARED ? 64 / CH : 1;
    const int lane = threadIdx.x & 63, g = SHARED ? lane / CH : 0, c = 4 * (lane % CH);
    const int at = (int)(blockIdx.x * 256 + threadIdx.x) / (CH * G), rows = a.split.part_rows();
    if (at >= rows) return;
    const int item = a.split.whole + at / a.split.tile_rows, row = item % a.q_tiles * kBlockRows + at % a.split.tile_rows;
    if (row >= a.rows) return;
    float m = -INFINITY, l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    auto merge = [&](float pm, float pl, f32x4 po) {
        const float m_new = fmaxf(m, pm), sub = m_new == -INFINITY ? 0.0f : m_new;
        const float f = __builtin_amdgcn_exp2f(m - sub), pf = __builtin_amdgcn_exp2f(pm - sub);
        m = m_new;
        l = l * f + pl * pf;
        o = o * f + po * pf;
    };
    for (int s0 = g; s0 < a.split.splits; s0 += 4 * G) {
        float2 ml[4];
        f32x4 po[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int s = s0 + k * G;
            ml[k] = make_float2(-INFINITY, 0.0f);
            po[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (s < a.split.splits) {
                ml[k] = *(const float2 *)(a.part_ml + 2 * (s * rows + at));
                if (c < D) po[k] = *(const f32x4 *)(a.part_o + (long long)(s * rows + at) * D + c);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) merge(ml[k].x, ml[k].y, po[k]);
    }
#pragma unroll
    for (int d = CH; SHARED && d < 64; d <<= 1) {
        const float pm = __shfl_xor(m, d), pl = __shfl_xor(l, d);
        f32x4 po;
#pragma unroll
        for (int e = 0; e < 4; ++e) po[e] = __shfl_xor(o[e], d);
        merge(pm, pl, po);
    }
    const int gh = item / a.q_tiles % a.grid_heads, b = item / a.q_tiles / a.grid_heads, in_group = a.packed ? row / a.q_len : 0;
    const int i = row - in_group * a.q_len, head = a.packed ? gh * a.group + in_group : gh;
    const long long stat = ((long long)b * a.heads + head) * a.q_len + i;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (g == 0 && c < a.d) {
        bf16x4 w;
        o *= inv;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (__bf16)o[e];
        if (a.o_exact) *(f32x4 *)(a.o_exact + stat * a.d + c) = o;
        *(bf16x4 *)(a.o + b * a.o_sb + (long long)i * a.o_st + head * a.o_sh + c) = w;
    }
    if (a.lse && g == 0 && c == 0) a.lse[stat] = l == 0.0f ? -INFINITY : (m + __builtin_log2f(l)) * 0.6931471805599453f;
}

// ---- host ----------------------------------------------------------------------------------------------------------------
int check_attention(const yamd_attention_desc *d, const uint8_t *key_mask, long long mask_stride, const float *bias)
{
    YAMD_REQUIRE(d, "attention: null descriptor");
    YAMD_REQUIRE(d->batch > 0 && d->q_len > 0 && d->k_len > 0 && d->heads > 0 && d->kv_heads > 0,
                 "attention: bad shape batch=%d q_len=%d k_len=%d heads=%d kv_heads=%d", d->batch, d->q_len, d->k_len, d->heads, d->kv_heads);
    YAMD_REQUIRE(d->heads % d->kv_heads == 0, "attention: %d heads do not share %d key heads evenly", d->heads, d->kv_heads);
    YAMD_REQUIRE(d->head_dim >= 8 && d->head_dim <= 128 && d->head_dim % 8 == 0,
                 "attention: head_dim must be a multiple of 8 up to 128 (got %d)", d->head_dim);
    YAMD_REQUIRE(d->q_len <= (1 << 24) && d->k_len <= (1 << 24), "attention: more than 2^24 tokens (q %d, k %d)", d->q_len, d->k_len);
    YAMD_REQUIRE((long long)d->batch * d->heads <= (1 << 20), "attention: batch * heads = %lld above 2^20", (long long)d->batch * d->heads);
    // (a launch has fewer than 2^32 threads; workgroups take 128 rows or a head each)
    YAMD_REQUIRE((long long)d->batch * d->heads * d->q_len <= (1 << 30) && (long long)d->batch * d->kv_heads * d->k_len <= (1 << 30),
                 "attention: more than 2^30 rows (batch %d, heads %d of %d, q %d, k %d)", d->batch, d->kv_heads, d->heads, d->q_len, d->k_len);
    YAMD_REQUIRE(d->scale >= 1e-20f && d->scale <= 1e20f, "attention: scale must be between 1e-20 and 1e20 (got %g)", (double)d->scale);
    YAMD_REQUIRE(!key_mask || d->batch == 1 || mask_stride >= d->k_len, "attention: mask stride smaller than k_len");
    if (bias) {
        YAMD_REQUIRE(d->map_h > 0 && d->map_w > 0 && d->q_len == d->k_len && (long long)d->map_h * d->map_w == d->q_len,
                     "attention: a position bias needs q_len == k_len == map_h * map_w (got %d, %d, %d x %d)", d->q_len, d->k_len, d->map_h,
                     d->map_w);
        YAMD_REQUIRE(d->heads <= 65535, "attention: a position bias for %d heads (at most 65535)", d->heads);
        YAMD_REQUIRE(d->map_h == 1 || d->map_w <= 760, "attention: a map of several rows is at most 760 wide (got %d x %d)", d->map_h, d->map_w);
    }
    return YAMD_OK;
}

int check_tokens(const yamd_attention_desc *d, const yamd_tokens *t, int len, int heads, const char *name)
{
    YAMD_REQUIRE(t && t->data, "attention: %s is null", name);
    YAMD_REQUIRE(((uintptr_t)t->data & 15) == 0, "attention: %s is not 16-byte aligned", name);
    YAMD_REQUIRE((d->batch == 1 || (t->batch_stride % 8 == 0 && t->batch_stride >= 0)) && (len == 1 || (t->token_stride % 8 == 0 && t->token_stride > 0)) &&
                     (heads == 1 || (t->head_stride % 8 == 0 && t->head_stride > 0)),
                 "attention: strides of %s must be positive multiples of 8 elements", name);
    YAMD_REQUIRE(len == 1 || t->token_stride <= (1 << 23), "attention: tokens of %s are more than 2^23 elements apart", name);
    return YAMD_OK;
}

// rows of a result must not share memory: taken from the shortest stride on, each axis steps over all that the ones before span
int check_result(const yamd_attention_desc *d, const yamd_tokens *t, int len, int heads, const char *name)
{
    const int rc = check_tokens(d, t, len, heads, name);
    if (rc != YAMD_OK) return rc;
    struct Axis {
        long long stride;
        int n;
    } axis[3] = {{t->head_stride, heads}, {t->token_stride, len}, {t->batch_stride, d->batch}};
    std::sort(axis, axis + 3, [](const Axis &x, const Axis &y) { return x.stride < y.stride; });
    long long span = d->head_dim;
    for (const Axis &x : axis) {
        if (x.n == 1) continue;
        YAMD_REQUIRE(x.stride >= span, "attention: rows of %s overlap (strides %lld, %lld, %lld)", name, t->batch_stride, t->token_stride,
                     t->head_stride);
        span += x.stride * (x.n - 1);
    }
    return YAMD_OK;
}

// Costs are in units of a step's time on a CU with enough workgroups.  A CU works through its items one unit per step whether they
// run side by side or one after the other, so what counts is the CU with the most.
//
// From 256 items on, what does not fill all 256 CUs is the loss (6400 keys, d 64: 768 items 208 us, 800 items 270 us, 1024 items
// 280 us): as many items as fill them stay whole, and the rest is cut into parts that fill them once more.
// Below, all items are cut.  The cost is that of a CU with n workgroups, `resident` at a time and each `steps` long (it takes up to
// three to hide the latency of a step, so fewer are no cheaper).
// Both pay for the parts' way through memory and for the launch that joins them.  The numbers were fitted to six shapes of 24 to
// 208 items: 300 queries on 8400 keys, 8 heads: 21 parts 18.4 us, 33 parts 21.3, whole 96; one query of 8 images: 22 parts 17 us,
// 32 parts 20.9.
WorkSplit split_work(long long items, int steps, int len, int resident, int results, float step)
{
    constexpr long long kCus = 256;
    constexpr int kPrologue = 3;                         // steps that a part costs before its first and after its last one
    const bool few = items < kCus;
    const long long whole = few ? 0 : items / kCus * kCus, rest = items - whole;
    const int tile_rows = len < kBlockRows ? len : kBlockRows;
    const float rows = (float)(results * rest) * (float)len / (float)ceil_div(len, kBlockRows);
    WorkSplit w = {(int)items, 0, 1, steps, tile_rows};
    if (rest == 0) return w;
    const float per_part = (0.1f + rows / 5000.0f) / step, join = 12.0f / step;
    const long long least = resident < 3 ? resident : 3;
    float best = INFINITY;
    for (int k = 1; k <= 256;) {
        const int len = (steps + k - 1) / k;
        const long long n = (rest * k + kCus - 1) / kCus;
        float cost;
        if (few) {
            const long long last = n % resident, load = n - last + (last == 0 ? 0 : last > least ? last : least);
            cost = (float)len * (float)load;
        } else {
            cost = (float)(len + (k > 1 ? kPrologue : 0)) * (float)n;
        }
        if (k > 1) cost += per_part * (float)k + join;
        if (cost < best) {
            best = cost;
            if (k > 1) w = {(int)whole, (int)rest, k, len, tile_rows};
        }
        if (len == 1) break;
        k = (steps + len - 2) / (len - 1);               // the next one with shorter parts: more parts of one length only cost more
    }
    w.splits = ceil_div(steps, w.per_split);
    return w;
}

namespace {

struct FwdPlan {
    int packed, rows, q_tiles, grid_heads, dpad;
    WorkSplit split;
    size_t workspace;
};

FwdPlan plan_forward(const yamd_attention_desc *d, bool biased)
{
    FwdPlan p = {};
    const int group = d->heads / d->kv_heads;
    p.dpad = padded_head_dim(d->head_dim);
    // packing shares a tile of keys among the group's heads; with a full tile of queries per head there is nothing to gain
    p.packed = !biased && group > 1 && d->q_len <= kBlockRows / 2;
    p.rows = p.packed ? d->q_len * group : d->q_len;
    p.grid_heads = p.packed ? d->kv_heads : d->heads;
    p.q_tiles = ceil_div(p.rows, kBlockRows);
    p.split = split_work((long long)d->batch * p.grid_heads * p.q_tiles, ceil_div(d->k_len, kTile), p.rows,
                         p.dpad == 32 ? 4 : p.dpad == 64 ? 3 : 2, 1, 1.0f);
    p.workspace = (size_t)p.split.splits * p.split.part_rows() * (p.dpad + 2) * sizeof(float);
    return p;
}

template <int D, int BIAS, bool EXACT>
int launch_forward(const AttnFwdArgs &a, hipStream_t st)
{
    using Attr = KernelAttr<&attention_kernel<D, BIAS, EXACT>, FwdLds<D>::most(BIAS)>;
    const int lds = FwdLds<D>::WINDOW + 2 * a.window * (int)sizeof(float);
    const int rc = Attr::ensure();
    if (rc != YAMD_OK) return rc;
    hipLaunchKernelGGL((attention_kernel<D, BIAS, EXACT>), dim3(a.split.grid()), dim3(256), lds, st, a);
    YAMD_LAUNCH_CHECK();
    if (const int rows = a.split.part_rows()) {
        if (a.split.splits > 8) hipLaunchKernelGGL((attention_join_kernel<D, true>), dim3(ceil_div(rows * 64, 256)), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((attention_join_kernel<D, false>), dim3(ceil_div(rows * kJoinLanes<D>, 256)), dim3(256), 0, st, a);
        YAMD_LAUNCH_CHECK();
    }
    return YAMD_OK;
}

template <int D>
int launch_forward(Bias form, const AttnFwdArgs &a, hipStream_t st)
{
    const bool exact = a.o_exact && (form != kNoBias || a.k_len <= kFewKeys);
    if (form == kNoBias) return exact ? launch_forward<D, kNoBias, true>(a, st) : launch_forward<D, kNoBias, false>(a, st);
    if (form == kQuadBias) return exact ? launch_forward<D, kQuadBias, true>(a, st) : launch_forward<D, kQuadBias, false>(a, st);
    return exact ? launch_forward<D, kAnyBias, true>(a, st) : launch_forward<D, kAnyBias, false>(a, st);
}

}  // namespace
}  // namespace yamd

using namespace yamd;

extern "C" size_t yamd_attention_workspace_bytes(const yamd_attention_desc *d, int biased)
{
    if (check_attention(d, nullptr, 0, nullptr) != YAMD_OK) return 0;
    return plan_forward(d, biased != 0).workspace;
}

extern "C" int yamd_attention(const yamd_attention_desc *d, const yamd_tokens *q, const yamd_tokens *k, const yamd_tokens *v,
                              const uint8_t *key_mask, long long mask_stride, const float *bias, const yamd_tokens *o, float *o_exact,
                              float *lse, void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = check_attention(d, key_mask, mask_stride, bias);
    if (rc == YAMD_OK) rc = check_tokens(d, q, d->q_len, d->heads, "q");
    if (rc == YAMD_OK) rc = check_tokens(d, k, d->k_len, d->kv_heads, "k");
    if (rc == YAMD_OK) rc = check_tokens(d, v, d->k_len, d->kv_heads, "v");
    if (rc == YAMD_OK) rc = check_result(d, o, d->q_len, d->heads, "o");
    if (rc != YAMD_OK) return rc;
    YAMD_REQUIRE(((uintptr_t)o_exact & 15) == 0, "attention: o_exact is not 16-byte aligned");
    const FwdPlan p = plan_forward(d, bias != nullptr);
    if (p.workspace && (!workspace || workspace_bytes < p.workspace || ((uintptr_t)workspace & 15))) {
        set_error("attention: workspace of %zu bytes, needs %zu (16-byte aligned)", workspace ? workspace_bytes : (size_t)0, p.workspace);
        return YAMD_ENOSPC;
    }
    AttnFwdArgs a = {};
    a.q = view_of(q); a.k = view_of(k); a.v = view_of(v);
    a.o = (__bf16 *)o->data; a.o_sb = o->batch_stride; a.o_st = o->token_stride; a.o_sh = o->head_stride;
    a.lse = lse; a.o_exact = o_exact; a.mask = key_mask; a.mask_sb = mask_stride; a.bias = bias;
    if (bias) {
        a.map_w = d->map_h > 1 ? d->map_w : 1;       // (of a sequence the coordinate is the position, also beyond its end)
        a.coord_last = map_coord(d->k_len - 1, a.map_w);
        a.n_off = 2 * a.coord_last + 1;
        a.window = window_len(d->map_h, d->map_w);
    }
    a.batch = d->batch; a.q_len = d->q_len; a.k_len = d->k_len; a.d = d->head_dim; a.heads = d->heads; a.kv_heads = d->kv_heads; a.group = d->heads / d->kv_heads;
    a.packed = p.packed; a.rows = p.rows; a.q_tiles = p.q_tiles; a.grid_heads = p.grid_heads; a.split = p.split; a.scale = d->scale;
    a.part_o = (float *)workspace;
    if (p.workspace) a.part_ml = a.part_o + (size_t)p.split.splits * p.split.part_rows() * p.dpad;
    hipStream_t st = (hipStream_t)stream;
    const Bias form = bias_form(bias, d->map_h, d->map_w);
    switch (p.dpad) {
    case 32: return launch_forward<32>(form, a, st);
    case 64: return launch_forward<64>(form, a, st);
    case 96: return launch_forward<96>(form, a, st);
    default: return launch_forward<128>(form, a, st);
    }
}
