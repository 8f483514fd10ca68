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
__device__ __forceinline__ void load_vec(const T *p, float *v)
{
    if constexpr (VEC == 1) {
        v[0] = (float)*p;
    } else {
        const typename Pack<T, VEC>::type t = *(const typename Pack<T, VEC>::type *)p;
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
        typename Pack<T, VEC>::type t;
#pragma unroll
        for (int j = 0; j < VEC; ++j) t[j] = (T)v[j];
        *(typename Pack<T, VEC>::type *)p = t;
    }
}

// weight / bias of one vector of channels; absent ones read as `none`
template <int VEC>
__device__ __forceinline__ void load_param(const void *p, int bf16, int ch, float none, float *v)
{
    if (!p) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = none;
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = bf16 ? (float)((const __bf16 *)p)[ch + j] : ((const float *)p)[ch + j];
    }
}

// sum over the TPR threads of a row, the result in all of them
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float *lds)
{
    constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int d = W / 2; d > 0; d >>= 1)
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] += __shfl_xor(v[n], d);
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
    constexpr int NT = TPR > 256 ? TPR : 256, RPB = NT / TPR, E = VEC * VPT;
    __shared__ float lds[2 * (NT / 64)];
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const T *x = (const T *)a.x;
    T *y = (T *)a.y;
    const float inv_c = 1.0f / (float)a.c;
    float w[E], b[E];
    bool on[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int ch = (k * TPR + lane) * VEC;
        on[k] = ch < a.c;
        if (on[k]) {
            load_param<VEC>(a.w, a.param_bf16, ch, 1.0f, w + k * VEC);
            load_param<VEC>(a.b, a.param_bf16, ch, 0.0f, b + k * VEC);
        }
    }
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < a.rows; r0 += (long long)gridDim.x * RPB) {
        const long long r = r0 + group;
        const bool live = r < a.rows;          // the other groups of the wave still take part in its exchanges
        float v[E], s[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            if (live && on[k]) {
                load_vec<T, VEC>(x + r * a.x_rs + (k * TPR + lane) * VEC, v + k * VEC);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[k * VEC + j] = 0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) s[0] += v[e];
        row_sum<TPR>(s, lds);
        const float mu = s[0] * inv_c;
        s[0] = 0.0f;
#pragma unroll
        for (int k = 0; k < VPT; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = v[k * VEC + j] - mu;
                v[k * VEC + j] = d;
                s[0] += on[k] ? d * d : 0.0f;
            }
        row_sum<TPR>(s, lds);
        const float rs = 1.0f / sqrtf(s[0] * inv_c + a.eps);
        if (!live) continue;                   // TPR > 64: one group, so all threads or none
        if (lane == 0 && a.mean) {
            a.mean[r] = mu;
            a.rstd[r] = rs;
        }
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            if (!on[k]) continue;
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = v[k * VEC + j] * rs * w[k * VEC + j] + b[k * VEC + j];
            store_vec<T, VEC>(y + r * a.y_rs + (k * TPR + lane) * VEC, o);
        }
    }
}

template <typename T, int VEC, int TPR, int VPT>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layer_norm_backward_kernel(NormArgs a)
{
    constexpr int NT = TPR > 256 ? TPR : 256, RPB = NT / TPR, E = VEC * VPT;
    __shared__ float lds[2 * (NT / 64)];
    __shared__ float acc[RPB > 1 ? 2 * TPR * E : 1];
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const T *x = (const T *)a.x, *dy = (const T *)a.dy;
    T *dx = (T *)a.dx;
    const float inv_c = 1.0f / (float)a.c;
    float w[E], dw[E], db[E];
    bool on[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int ch = (k * TPR + lane) * VEC;
        on[k] = ch < a.c;
#pragma unroll
        for (int j = 0; j < VEC; ++j) w[k * VEC + j] = dw[k * VEC + j] = db[k * VEC + j] = 0.0f;
        if (on[k]) load_param<VEC>(a.w, a.param_bf16, ch, 1.0f, w + k * VEC);
    }
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < a.rows; r0 += (long long)gridDim.x * RPB) {
        const long long r = r0 + group;
        const bool live = r < a.rows;
        float xh[E], g[E], s[2] = {0.0f, 0.0f};
        const float mu = live ? a.mean_in[r] : 0.0f, rs = live ? a.rstd_in[r] : 0.0f;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            if (live && on[k]) {
                load_vec<T, VEC>(x + r * a.x_rs + (k * TPR + lane) * VEC, xh + k * VEC);
                load_vec<T, VEC>(dy + r * a.dy_rs + (k * TPR + lane) * VEC, g + k * VEC);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) xh[k * VEC + j] = mu, g[k * VEC + j] = 0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            xh[e] = (xh[e] - mu) * rs;
            dw[e] += g[e] * xh[e];
            db[e] += g[e];
            g[e] *= w[e];
            s[0] += g[e];
            s[1] += g[e] * xh[e];
        }
        if (!a.dx) continue;
        row_sum<TPR>(s, lds);
        if (!live) continue;
        const float m0 = s[0] * inv_c, m1 = s[1] * inv_c;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            if (!on[k]) continue;
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = rs * (g[k * VEC + j] - m0 - xh[k * VEC + j] * m1);
            store_vec<T, VEC>(dx + r * a.dx_rs + (k * TPR + lane) * VEC, o);
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

// column sums of the partial rows: 16 channels x 64 rows of threads per workgroup, blockIdx.y 0 = dw, 1 = db
__global__ __launch_bounds__(1024) void norm_param_grad_kernel(const float *partial, int n, int c, void *dw, void *db, int bf16)
{
    __shared__ float lds[64][17];
    const int col = threadIdx.x & 15, row = threadIdx.x >> 4, ch = blockIdx.x * 16 + col;
    float s = 0.0f;
    if (ch < c)
        for (int i = row; i < n; i += 64) s += partial[((long long)i * 2 + blockIdx.y) * c + ch];
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
    NormArgs a = {};
    a.x = x; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.rstd = rstd;
    a.x_rs = x_stride; a.y_rs = y_stride; a.rows = rows; a.c = c; a.param_bf16 = param_dtype == YAMD_BF16; a.eps = eps;
    const int v = dtype == YAMD_BF16 ? 8 : 4;
    const bool wide = c % v == 0 && x_stride % v == 0 && y_stride % v == 0 && aligned16(x) && aligned16(y);
    const int vec = wide ? v : 1;
    const Team t = team_for(c, vec);
    const long long rpb = t.tpr > 256 ? 1 : 256 / t.tpr;
    const long long want = (rows + rpb - 1) / rpb, most = 256 * (t.tpr > 256 ? 2 : 8);
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
