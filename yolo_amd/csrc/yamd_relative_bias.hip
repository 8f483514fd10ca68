// A learned position bias by buckets of distance: bias[head][distance] = table[bucket of the distance][head], and the
// gradient of the table.  The attention kernels read the bias by distance ((2 h - 1)(2 w - 1) floats per head, for a 40 x 40
// map 25 KB) and leave the sums of their score gradients by distance, so no array of pairs exists in either
// direction (the sums do take a row of distances for every 128 queries).  Both kernels here move a few hundred kilobytes; a launch is what they cost.
// The gradient adds the distances of one bucket in a fixed order: threads stride over the bucket's list of distances
// (sorted once, when the map of buckets is made) and a tree joins them.
#include "yamd_common.h"

using namespace yamd;

namespace {

__global__ __launch_bounds__(256) void relative_bias_kernel(const void *table, int bf16, const int *bucket_of, int n, int heads,
                                                            int buckets, float *bias)
{
    const int off = blockIdx.x * 256 + threadIdx.x, head = blockIdx.y;
    if (off >= n) return;
    const int bucket = bucket_of[off];
    float v = __builtin_nanf("");            // a bucket that the table does not have
    if (bucket >= 0 && bucket < buckets) {
        const long long at = (long long)bucket * heads + head;
        v = bf16 ? (float)((const __bf16 *)table)[at] : ((const float *)table)[at];
    }
    bias[(long long)head * n + off] = v;
}

// one workgroup per (bucket, head); order[start[bucket] .. start[bucket + 1]) are the distances of the bucket
__global__ __launch_bounds__(256) void relative_bias_backward_kernel(const float *dbias, const int *order, const int *start, int n,
                                                                     int heads, void *dtable, int bf16)
{
    __shared__ float part[4];
    const int bucket = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
    const int e0 = max(start[bucket], 0), e1 = min(start[bucket + 1], n);
    const float *g = dbias + (long long)head * n;
    float s = 0.0f;
    for (int e = e0 + tid; e < e1; e += 256) {
        const int off = order[e];
        if (off >= 0 && off < n) s += g[off];
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
    if ((tid & 63) == 0) part[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) {
        s = (part[0] + part[1]) + (part[2] + part[3]);
        const long long at = (long long)bucket * heads + head;
        if (bf16) ((__bf16 *)dtable)[at] = (__bf16)s;
        else ((float *)dtable)[at] = s;
    }
}

int check_bias(int dtype, int n, int heads, int buckets)
{
    YAMD_REQUIRE(dtype == YAMD_F32 || dtype == YAMD_BF16, "relative bias: unknown dtype %d", dtype);
    YAMD_REQUIRE(n > 0 && n <= (1 << 27) && heads > 0 && heads <= 65535 && buckets > 0 && buckets <= (1 << 20),
                 "relative bias: bad shape distances=%d heads=%d buckets=%d", n, heads, buckets);
    return YAMD_OK;
}

}  // namespace

extern "C" int yamd_relative_bias(const void *table, int table_dtype, const int32_t *bucket_of, int n_distances, int heads, int n_buckets,
                                  float *bias, void *stream)
{
    const int rc = check_bias(table_dtype, n_distances, heads, n_buckets);
    if (rc != YAMD_OK) return rc;
    YAMD_REQUIRE(table && bucket_of && bias, "relative bias: null argument");
    hipLaunchKernelGGL(relative_bias_kernel, dim3(ceil_div(n_distances, 256), heads), dim3(256), 0, (hipStream_t)stream, table,
                       (int)(table_dtype == YAMD_BF16), bucket_of, n_distances, heads, n_buckets, bias);
    YAMD_LAUNCH_CHECK();
    return YAMD_OK;
}

extern "C" int yamd_relative_bias_backward(const float *dbias, const int32_t *order, const int32_t *start, int n_distances, int heads,
                                           int n_buckets, void *dtable, int table_dtype, void *stream)
{
    const int rc = check_bias(table_dtype, n_distances, heads, n_buckets);
    if (rc != YAMD_OK) return rc;
    YAMD_REQUIRE(dbias && order && start && dtable, "relative bias backward: null argument");
    hipLaunchKernelGGL(relative_bias_backward_kernel, dim3(n_buckets, heads), dim3(256), 0, (hipStream_t)stream, dbias, order, start,
                       n_distances, heads, dtable, (int)(table_dtype == YAMD_BF16));
    YAMD_LAUNCH_CHECK();
    return YAMD_OK;
}
