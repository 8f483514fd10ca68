// Layer norm over the channels of a row, forward and backward, float32 or bf16 rows.
//
//   forward    mu = mean x,  r = 1 / sqrt(mean (x - mu)^2 + eps),  y = (x - mu) r w + b
//   backward   xh = (x - mu) r,  g = dy w,  dx = r (g - mean g - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// Both are bound by memory: a row is read once, held in registers between its statistics and its result, and written
// once.  TPR threads share a row (16 to 1024, so that a thread holds at most 16 channels) and every thread keeps its
// channels' weights in registers over all rows that its workgroup takes.  Statistics and sums are float32; the variance is
// that of the centred row, so a large mean costs no bits.  In the backward pass a thread adds dw and db of its channels
// over its rows in registers, a workgroup adds its row groups in a fixed order and writes one partial row, and a second
// kernel adds the partial rows in a fixed order: no atomics, the same bits on every run.
// Measured: 51200 rows of 256 bf16 in 10 us (5.2 TB/s: its 52 MB fit the Infinity Cache; a large copy reaches 4.9), 102400 rows of 512
// with their gradients 90 us in three launches (forward 34, backward 52, sums of the partial rows 4; 101 us over changing inputs,
// 86 us for 420 MB at the rate of a copy).  Several rows are
// in flight per team because one row's loads do not cover the latency of memory (kRowsAtOnce).  Calls of a few hundred rows cost
// their launches.
// VEC > 1 (16-byte accesses) needs channel count, strides and addresses that are multiples of 16 bytes; other rows go
// channel by channel (VEC = 1).
#include "yamd_common.h"

using namespace yamd;

namespace {

constexpr int kMaxChannels = 16384;

template <typename T, int VEC>
struct Pack {
    typedef T type __attribute__((ext_vector_type(VEC)));
};
template <typename T>
struct Pack<T, 1> {
    typedef T type;
};
template <typename T, int VEC>
using pack_t = typename Pack<T, VEC>::type;

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const pack_t<T, VEC> &t, float *v)
{
    if constexpr (VEC == 1) {
        v[0] = (float)t;
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = (float)t[j];
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T *p, const float *v)
{
    if constexpr (VEC == 1) {
        *p = (T)v[0];
    } else {
        pack_t<T, VEC> t;
#pragma unroll
        for (int j = 0; j < VEC; ++j) t[j] = (T)v[j];
        *(pack_t<T, VEC> *)p = t;
    }
}

// a thread's weights or biases (parameters are aligned to their own type only); absent ones read as `none`.  at[k]: first
// channel of its k-th vector
template <typename P, int VEC, int VPT>
__device__ __forceinline__ void load_params_of(const P *p, const int (&at)[VPT], float *v)
{
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        P t[VEC];
        __builtin_memcpy(t, p + at[k], sizeof(t));
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[k * VEC + j] = (float)t[j];
    }
}
template <int VEC, int VPT>
__device__ __forceinline__ void load_params(const void *p, int bf16, const int (&at)[VPT], float none, float *v)
{
    if (!p) {
#pragma unroll
        for (int e = 0; e < VEC * VPT; ++e) v[e] = none;
    } else if (bf16) {
        load_params_of<__bf16, VEC, VPT>((const __bf16 *)p, at, v);
    } else {
        load_params_of<float, VEC, VPT>((const float *)p, at, v);
    }
}

// 1 / sqrt(t): the instruction's result (1 ulp) and one Newton step; t beyond its range (eps = 0, or squares near the end of
// float32; of an overflow 0, not the step's inf * 0) the long way
__device__ __forceinline__ float inverse_sqrt(float t)
{
    if (t < 1e-30f || t > 1e30f) return 1.0f / sqrtf(t);
    const float r = __builtin_amdgcn_rsqf(t);
    return r * (1.5f - 0.5f * t * r * r);
}

template <int CTRL>
__device__ __forceinline__ float add_dpp(float v)
{
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// sum over aligned groups of W lanes, the result in all of them (register exchanges only)
template <int W>
__device__ __forceinline__ float lane_sum(float v)
{
    v = add_dpp<0xb1>(v);                      // lane ^ 1
    v = add_dpp<0x4e>(v);                      // lane ^ 2
    v = add_dpp<0x141>(v);                     // the other four of eight lanes
    v = add_dpp<0x140>(v);                     // the other eight of sixteen
    if constexpr (W >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
        v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    }
    if constexpr (W >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
        v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    }
    return v;
}

// sums over the TPR threads of a row, the results in all of them
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float *lds)
{
    constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = lane_sum<W>(v[n]);
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;
        const int wave = threadIdx.x >> 6;
        __syncthreads();                       // the values of the sum before this one have been read
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) lds[n * NW + wave] = v[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            v[n] = lds[n * NW];
#pragma unroll
            for (int w = 1; w < NW; ++w) v[n] += lds[n * NW + w];
        }
    }
}

// rows that a team takes at once, so that enough loads are in flight
template <int E, int TPR>
constexpr int kRowsAtOnce = TPR > 256 ? 1 : E <= 8 ? 4 : 2;

struct NormArgs {
    const void *x, *dy, *w, *b;
    void *y, *dx;
    float *mean, *rstd;
    const float *mean_in, *rstd_in;
    float *partial;                 // [gridDim.x][2][c]
    long long x_rs, y_rs, dy_rs, dx_rs, rows;
    int c, param_bf16;
    float eps;
};

template <typename T, int VEC, int TPR, int VPT>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layer_norm_kernel(NormArgs a)
{
    constexpr int NT = TPR > 256 ? TPR : 256, RPB = NT / TPR, E = VEC * VPT, R = kRowsAtOnce<E, TPR>;
    __shared__ float lds[R * (NT / 64)];
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const T *x = (const T *)a.x;
    T *y = (T *)a.y;
    const float inv_c = 1.0f / (float)a.c;
    float w[E], b[E];
    bool on[VPT];
    int at[VPT];                               // a thread's vectors beyond the channels repeat the first one and count as zero
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int ch = (k * TPR + lane) * VEC;
        on[k] = ch < a.c;
        at[k] = on[k] ? ch : 0;
    }
    load_params<VEC, VPT>(a.w, a.param_bf16, at, 1.0f, w);
    load_params<VEC, VPT>(a.b, a.param_bf16, at, 0.0f, b);
    for (long long r0 = (long long)blockIdx.x * RPB * R; r0 < a.rows; r0 += (long long)gridDim.x * RPB * R) {
        // all loads first: rows beyond the last one repeat it (their teams still take part in the exchanges)
        pack_t<T, VEC> raw[R][VPT];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const long long r = r0 + q * RPB + group;
            const T *p = x + (r < a.rows ? r : a.rows - 1) * a.x_rs;
#pragma unroll
            for (int k = 0; k < VPT; ++k) raw[q][k] = *(const pack_t<T, VEC> *)(p + at[k]);
        }
        float v[R][E], mu[R], rs[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            mu[q] = 0.0f;
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                unpack<T, VEC>(raw[q][k], v[q] + k * VEC);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[q][k * VEC + j] = on[k] ? v[q][k * VEC + j] : 0.0f;
            }
        }
#pragma unroll
        for (int q = 0; q < R; ++q)
#pragma unroll
            for (int e = 0; e < E; ++e) mu[q] += v[q][e];
        row_sum<TPR>(mu, lds);
#pragma unroll
        for (int q = 0; q < R; ++q) {
            mu[q] *= inv_c;
            rs[q] = 0.0f;
#pragma unroll
            for (int k = 0; k < VPT; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float d = v[q][k * VEC + j] - mu[q];
                    v[q][k * VEC + j] = d;
                    rs[q] += on[k] ? d * d : 0.0f;
                }
        }
        row_sum<TPR>(rs, lds);
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const long long r = r0 + q * RPB + group;
            if (r >= a.rows) continue;
            const float s = inverse_sqrt(rs[q] * inv_c + a.eps);
            if (lane == 0 && a.mean) {
                a.mean[r] = mu[q];
                a.rstd[r] = s;
            }
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                if (!on[k]) continue;
                float o[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) o[j] = v[q][k * VEC + j] * s * w[k * VEC + j] + b[k * VEC + j];
                store_vec<T, VEC>(y + r * a.y_rs + (k * TPR + lane) * VEC, o);
            }
        }
    }
}

template <typename T, int VEC, int TPR, int VPT>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layer_norm_backward_kernel(NormArgs a)
{
    constexpr int NT = TPR > 256 ? TPR : 256, RPB = NT / TPR, E = VEC * VPT, R = E <= 8 ? 2 : 1;
    __shared__ float lds[2 * R * (NT / 64)];
    __shared__ float acc[RPB > 1 ? 2 * TPR * E : 1];
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const T *x = (const T *)a.x, *dy = (const T *)a.dy;
    T *dx = (T *)a.dx;
    const float inv_c = 1.0f / (float)a.c;
    float w[E], dw[E], db[E];
    bool on[VPT];
    int at[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int ch = (k * TPR + lane) * VEC;
        on[k] = ch < a.c;
        at[k] = on[k] ? ch : 0;
    }
    load_params<VEC, VPT>(a.w, a.param_bf16, at, 1.0f, w);
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.0f;
    for (long long r0 = (long long)blockIdx.x * RPB * R; r0 < a.rows; r0 += (long long)gridDim.x * RPB * R) {
        pack_t<T, VEC> raw_x[R][VPT], raw_g[R][VPT];
        float xh[R][E], g[R][E], mu[R], rs[R], s[2 * R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const long long r = r0 + q * RPB + group, rr = r < a.rows ? r : a.rows - 1;
            mu[q] = a.mean_in[rr];
            rs[q] = a.rstd_in[rr];
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                raw_x[q][k] = *(const pack_t<T, VEC> *)(x + rr * a.x_rs + at[k]);
                raw_g[q][k] = *(const pack_t<T, VEC> *)(dy + rr * a.dy_rs + at[k]);
            }
        }
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const bool live = r0 + q * RPB + group < a.rows;
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                unpack<T, VEC>(raw_x[q][k], xh[q] + k * VEC);
                unpack<T, VEC>(raw_g[q][k], g[q] + k * VEC);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    xh[q][k * VEC + j] = live && on[k] ? xh[q][k * VEC + j] : mu[q];
                    g[q][k * VEC + j] = live && on[k] ? g[q][k * VEC + j] : 0.0f;
                }
            }
        }
#pragma unroll
        for (int q = 0; q < R; ++q) {
            s[2 * q] = s[2 * q + 1] = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                xh[q][e] = (xh[q][e] - mu[q]) * rs[q];
                dw[e] += g[q][e] * xh[q][e];
                db[e] += g[q][e];
                g[q][e] *= w[e];
                s[2 * q] += g[q][e];
                s[2 * q + 1] += g[q][e] * xh[q][e];
            }
        }
        if (!a.dx) continue;
        row_sum<TPR>(s, lds);
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const long long r = r0 + q * RPB + group;
            if (r >= a.rows) continue;
            const float m0 = s[2 * q] * inv_c, m1 = s[2 * q + 1] * inv_c;
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                if (!on[k]) continue;
                float o[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) o[j] = rs[q] * (g[q][k * VEC + j] - m0 - xh[q][k * VEC + j] * m1);
                store_vec<T, VEC>(dx + r * a.dx_rs + (k * TPR + lane) * VEC, o);
            }
        }
    }
    if (!a.partial) return;
    if constexpr (RPB > 1) {
        // the row groups of the workgroup, one after the other (channel (k TPR + lane) VEC + j at [(k TPR + lane) VEC + j])
        for (int gi = 0; gi < RPB; ++gi) {
            if (group == gi) {
#pragma unroll
                for (int k = 0; k < VPT; ++k)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const int at = (k * TPR + lane) * VEC + j;
                        acc[at] = (gi ? acc[at] : 0.0f) + dw[k * VEC + j];
                        acc[TPR * E + at] = (gi ? acc[TPR * E + at] : 0.0f) + db[k * VEC + j];
                    }
            }
            __syncthreads();
        }
        float *out = a.partial + (long long)blockIdx.x * 2 * a.c;
        for (int ch = threadIdx.x; ch < a.c; ch += NT) {
            out[ch] = acc[ch];
            out[a.c + ch] = acc[TPR * E + ch];
        }
    } else {
        float *out = a.partial + (long long)blockIdx.x * 2 * a.c;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            if (!on[k]) continue;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                out[(k * TPR + lane) * VEC + j] = dw[k * VEC + j];
                out[a.c + (k * TPR + lane) * VEC + j] = db[k * VEC + j];
            }
        }
    }
}

// column sums of the partial rows: 16 channels x 64 rows of threads per workgroup, blockIdx.y 0 = dw, 1 = db; a thread has
// eight loads in flight
__global__ __launch_bounds__(1024) void norm_param_grad_kernel(const float *partial, int n, int c, void *dw, void *db, int bf16)
{
    __shared__ float lds[64][17];
    const int col = threadIdx.x & 15, row = threadIdx.x >> 4, ch = blockIdx.x * 16 + col;
    float s = 0.0f;
    if (ch < c)
        for (int i0 = row; i0 < n; i0 += 8 * 64) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int i = i0 + 64 * k < n ? i0 + 64 * k : i0;
                v[k] = partial[((long long)i * 2 + blockIdx.y) * c + ch];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) s += i0 + 64 * k < n ? v[k] : 0.0f;
        }
    lds[row][col] = s;
    __syncthreads();
    for (int d = 32; d > 0; d >>= 1) {
        if (row < d) lds[row][col] += lds[row + d][col];
        __syncthreads();
    }
    void *out = blockIdx.y ? db : dw;
    if (row == 0 && ch < c && out) {
        if (bf16) ((__bf16 *)out)[ch] = (__bf16)lds[0][col];
        else ((float *)out)[ch] = lds[0][col];
    }
}

// (threads per row, workgroups at most) for a channel count; the smallest team whose threads hold at most 16 channels
struct Team {
    int tpr, most_blocks;
};

Team team_for(int c, int vec)
{
    const int cap = vec == 1 ? 4 : vec;            // narrow rows: one vector (four single channels) per thread
    if (c <= 16 * cap) return {16, 1024};
    if (vec == 8 && c <= 256) return {32, 1024};
    if (c <= 1024) return {64, 1024};
    if (c <= 4096) return {256, 1024};
    return {1024, 512};
}

// Workgroups of the backward pass.  Each writes one partial row of 2 c floats, so they are kept to what fills the card
// several times, and a workgroup gets at least four rounds of rows where there are enough.
int backward_blocks(long long rows, int c, int vec)
{
    const Team t = team_for(c, vec);
    const long long rpb = t.tpr > 256 ? 1 : 256 / t.tpr;
    const long long n = (rows + 4 * rpb - 1) / (4 * rpb);
    return (int)(n < t.most_blocks ? n : t.most_blocks);
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

template <typename T, int VEC, int TPR, int VPT>
void launch(bool backward, const NormArgs &a, int blocks, hipStream_t st)
{
    constexpr int NT = TPR > 256 ? TPR : 256;
    if (backward) hipLaunchKernelGGL((layer_norm_backward_kernel<T, VEC, TPR, VPT>), dim3(blocks), dim3(NT), 0, st, a);
    else hipLaunchKernelGGL((layer_norm_kernel<T, VEC, TPR, VPT>), dim3(blocks), dim3(NT), 0, st, a);
}

template <typename T>
void dispatch(bool backward, const NormArgs &a, int vec, int blocks, hipStream_t st)
{
    const int c = a.c, tpr = team_for(c, vec).tpr;
    constexpr int V = 16 / sizeof(T);
    if (vec == 1) {
        if (tpr == 16) launch<T, 1, 16, 4>(backward, a, blocks, st);
        else if (tpr == 64 && c <= 256) launch<T, 1, 64, 4>(backward, a, blocks, st);
        else if (tpr == 64) launch<T, 1, 64, 16>(backward, a, blocks, st);
        else if (tpr == 256) launch<T, 1, 256, 16>(backward, a, blocks, st);
        else launch<T, 1, 1024, 16>(backward, a, blocks, st);
    } else if (tpr == 16) {
        launch<T, V, 16, 1>(backward, a, blocks, st);
    } else if (tpr == 32) {
        if constexpr (V == 8) launch<T, 8, 32, 1>(backward, a, blocks, st);
    } else if (tpr == 64) {
        if (c <= 64 * V) launch<T, V, 64, 1>(backward, a, blocks, st);
        else if (c <= 128 * V) launch<T, V, 64, 2>(backward, a, blocks, st);
        else if constexpr (V == 4) launch<T, 4, 64, 4>(backward, a, blocks, st);
    } else if (tpr == 256) {
        if (c <= 512 * V) launch<T, V, 256, 2>(backward, a, blocks, st);
        else if constexpr (V == 4) launch<T, 4, 256, 4>(backward, a, blocks, st);
    } else {
        if (c <= 2048 * V) launch<T, V, 1024, 2>(backward, a, blocks, st);
        else if constexpr (V == 4) launch<T, 4, 1024, 4>(backward, a, blocks, st);
    }
}

int check_common(long long rows, int c, int dtype, int param_dtype)
{
    YAMD_REQUIRE(rows >= 0 && rows <= (1ll << 40) && c > 0 && c <= kMaxChannels, "layer norm: bad shape rows=%lld c=%d (c <= %d)", rows, c,
                 kMaxChannels);
    YAMD_REQUIRE(dtype == YAMD_F32 || dtype == YAMD_BF16, "layer norm: unknown dtype %d", dtype);
    YAMD_REQUIRE(param_dtype == YAMD_F32 || param_dtype == YAMD_BF16, "layer norm: unknown parameter dtype %d", param_dtype);
    return YAMD_OK;
}

bool stride_ok(long long stride, int c, long long rows) { return rows <= 1 || (stride >= c && stride <= (1ll << 31)); }

}  // namespace

extern "C" int yamd_layer_norm(const void *x, long long x_stride, const void *weight, const void *bias, int param_dtype, float eps,
                               void *y, long long y_stride, float *mean, float *rstd, long long rows, int c, int dtype, void *stream)
{
    const int rc = check_common(rows, c, dtype, param_dtype);
    if (rc != YAMD_OK) return rc;
    if (rows == 0) return YAMD_OK;
    YAMD_REQUIRE(x && y, "layer norm: null argument");
    YAMD_REQUIRE((mean == nullptr) == (rstd == nullptr), "layer norm: mean and rstd go together");
    YAMD_REQUIRE(eps >= 0.0f, "layer norm: eps must not be negative (got %g)", (double)eps);
    YAMD_REQUIRE(stride_ok(x_stride, c, rows) && stride_ok(y_stride, c, rows), "layer norm: row stride smaller than c=%d", c);
    // (rows of different workgroups would meet)
    YAMD_REQUIRE(x != y || rows <= 1 || x_stride == y_stride, "layer norm: in place with row strides %lld and %lld", x_stride, y_stride);
    NormArgs a = {};
    a.x = x; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.rstd = rstd;
    a.x_rs = x_stride; a.y_rs = y_stride; a.rows = rows; a.c = c; a.param_bf16 = param_dtype == YAMD_BF16; a.eps = eps;
    const int v = dtype == YAMD_BF16 ? 8 : 4;
    const bool wide = c % v == 0 && x_stride % v == 0 && y_stride % v == 0 && aligned16(x) && aligned16(y);
    const int vec = wide ? v : 1;
    const Team t = team_for(c, vec);
    const long long rpb = t.tpr > 256 ? 1 : 256 / t.tpr;
    const long long want = (rows + rpb - 1) / rpb, most = 256 * (t.tpr > 256 ? 2 : 8);     // (more than the rounds need: they end at once)
    const int blocks = (int)(want < most ? want : most);
    if (dtype == YAMD_BF16) dispatch<__bf16>(false, a, vec, blocks, (hipStream_t)stream);
    else dispatch<float>(false, a, vec, blocks, (hipStream_t)stream);
    YAMD_LAUNCH_CHECK();
    return YAMD_OK;
}

extern "C" size_t yamd_layer_norm_backward_workspace_bytes(long long rows, int c)
{
    if (rows < 0 || c <= 0 || c > kMaxChannels) return 0;
    int most = 1;                                   // the variant is chosen at the call, from the addresses too
    for (int vec : {1, 4, 8}) {
        const int n = backward_blocks(rows, c, vec);
        most = n > most ? n : most;
    }
    return (size_t)most * 2 * c * sizeof(float);
}

extern "C" int yamd_layer_norm_backward(const void *dy, long long dy_stride, const void *x, long long x_stride, const void *weight,
                                        int param_dtype, const float *mean, const float *rstd, void *dx, long long dx_stride,
                                        void *dweight, void *dbias, long long rows, int c, int dtype, void *workspace,
                                        size_t workspace_bytes, void *stream)
{
    const int rc = check_common(rows, c, dtype, param_dtype);
    if (rc != YAMD_OK) return rc;
    YAMD_REQUIRE(dx || dweight || dbias, "layer norm backward: no output");
    const bool params = dweight || dbias;
    NormArgs a = {};
    int blocks = 0;
    if (rows > 0) {
        YAMD_REQUIRE(dy && x && mean && rstd, "layer norm backward: null argument");
        YAMD_REQUIRE(stride_ok(dy_stride, c, rows) && stride_ok(x_stride, c, rows) && (!dx || stride_ok(dx_stride, c, rows)),
                     "layer norm backward: row stride smaller than c=%d", c);
        a.x = x; a.dy = dy; a.w = weight; a.dx = dx; a.mean_in = mean; a.rstd_in = rstd;
        a.x_rs = x_stride; a.dy_rs = dy_stride; a.dx_rs = dx_stride; a.rows = rows; a.c = c;
        a.param_bf16 = param_dtype == YAMD_BF16;
        const int v = dtype == YAMD_BF16 ? 8 : 4;
        const bool wide = c % v == 0 && x_stride % v == 0 && dy_stride % v == 0 && aligned16(x) && aligned16(dy) &&
                          (!dx || (dx_stride % v == 0 && aligned16(dx)));
        const int vec = wide ? v : 1;
        blocks = backward_blocks(rows, c, vec);
        if (params) {
            const size_t need = (size_t)blocks * 2 * c * sizeof(float);
            if (!workspace || workspace_bytes < need) {
                set_error("layer norm backward: workspace of %zu bytes, needs %zu", workspace ? workspace_bytes : (size_t)0, need);
                return YAMD_ENOSPC;
            }
            a.partial = (float *)workspace;
        }
        if (dtype == YAMD_BF16) dispatch<__bf16>(true, a, vec, blocks, (hipStream_t)stream);
        else dispatch<float>(true, a, vec, blocks, (hipStream_t)stream);
        YAMD_LAUNCH_CHECK();
    }
    if (params) {
        hipLaunchKernelGGL(norm_param_grad_kernel, dim3(ceil_div(c, 16), 2), dim3(1024), 0, (hipStream_t)stream, a.partial, blocks, c,
                           dweight, dbias, (int)(param_dtype == YAMD_BF16));
        YAMD_LAUNCH_CHECK();
    }
    return YAMD_OK;
}
