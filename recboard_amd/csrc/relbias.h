// The bucket half of the relative position bias, shared by the standalone operator and by attention.
#pragma once
#include "re_types.h"

#define RB_MAX_DISTANCE 1024
#define RB_MAX_BUCKETS 256

static inline bool rb_sizes_ok(int64_t max_distance, int64_t buckets) {
    return max_distance >= 1 && max_distance <= RB_MAX_DISTANCE && buckets >= 1 && buckets <= RB_MAX_BUCKETS;
}

#ifdef __HIPCC__
// line[d] = table[map[d], h] for the 2 * max_distance + 1 clipped distances; an entry of the map that is no bucket reads as 0
__device__ __forceinline__ float rb_entry(const void* table, int32_t dtype, const int32_t* map, int d, int buckets, int64_t H, int64_t h) {
    const int k = map[d];
    return (unsigned)k < (unsigned)buckets ? re_load_as_float(table, k * H + h, dtype) : 0.f;
}

// out[k] = the sum of line[d] over the distances in bucket k, by a workgroup of THREADS (line in LDS, complete; `ids`: n ints of LDS, `tmp`: THREADS
// floats).  Fixed order: every bucket is cut into the same slices whatever the launch.
template <int THREADS>
__device__ __forceinline__ void rb_line_to_buckets(const float* line, const int32_t* __restrict__ map, int n, int buckets, float* out, int* ids, float* tmp) {
    for (int d = threadIdx.x; d < n; d += THREADS) ids[d] = map[d];
    __syncthreads();
    int p = 1;
    while (p < buckets && p < THREADS) p <<= 1;
    const int slice = threadIdx.x / p, slices = THREADS / p;
    const int per = (n + slices - 1) / slices, from = slice * per, to = min(n, from + per);
    for (int k0 = 0; k0 < buckets; k0 += p) {
        const int k = k0 + (threadIdx.x & (p - 1));
        float acc = 0.f;
#pragma unroll 8
        for (int d = from; d < to; ++d) acc += ids[d] == k ? line[d] : 0.f;
        __syncthreads();                               // (the last round's parts have been read)
        tmp[threadIdx.x] = acc;
        __syncthreads();
        if (slice == 0 && k < buckets) {
            for (int s = 1; s < slices; ++s) acc += tmp[s * p + (k - k0)];
            out[k] = acc;
        }
    }
}

// dtable[k, h] = sum over r < rows of part[b][h][r][k] (b < B): one workgroup per head, 1024 lanes = bucket x slice (a few loads in flight each:
// the launch is their latency), fixed order
static __global__ __launch_bounds__(1024) void rb_reduce_k(const float* __restrict__ part, int64_t B, int64_t H, int64_t rows, int buckets, void* dtable,
                                                           int32_t dtype) {
    __shared__ float tmp[1024];
    int p = 1;
    while (p < buckets) p <<= 1;
    const int k = threadIdx.x & (p - 1), slice = threadIdx.x / p, slices = 1024 / p;
    const int64_t h = blockIdx.x, n = B * rows;
    float acc = 0.f;
    if (k < buckets) {
#pragma unroll 8
        for (int64_t i = slice; i < n; i += slices) {
            const int64_t b = i / rows, r = i - b * rows;
            acc += part[((b * H + h) * rows + r) * buckets + k];
        }
    }
    tmp[threadIdx.x] = acc;
    __syncthreads();
    if (slice == 0 && k < buckets) {
        for (int s = 1; s < slices; ++s) acc += tmp[s * p + k];
        re_store_float(dtable, k * H + h, dtype, acc);
    }
}
#endif
