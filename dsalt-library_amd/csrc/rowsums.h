// Rows held in registers by the waves of a workgroup: their sums, and column sums over rows.
#pragma once

#include "lanes.h"
#include "rows.h"

namespace dsalt {
namespace {

__device__ __forceinline__ void load8_dt(const void *p, int64_t chunk, int dtype, float (&v)[8]) {
    if (dtype == DSALT_DTYPE_F32) {
        Raw8<F32> r;
        r.load(p, chunk);
        r.get(v);
    } else if (dtype == DSALT_DTYPE_BF16) {
        Raw8<BF16> r;
        r.load(p, chunk);
        r.get(v);
    } else {
        Raw8<F16> r;
        r.load(p, chunk);
        r.get(v);
    }
}
__device__ __forceinline__ float load1_dt(const void *p, int64_t i, int dtype) {
    return dtype == DSALT_DTYPE_F32 ? Elem<F32>::ld(p, i) : dtype == DSALT_DTYPE_BF16 ? Elem<BF16>::ld(p, i) : Elem<F16>::ld(p, i);
}
__device__ __forceinline__ void store1_dt(void *p, int64_t i, int dtype, float v) {
    if (dtype == DSALT_DTYPE_F32) Elem<F32>::st(p, i, v);
    else if (dtype == DSALT_DTYPE_BF16) Elem<BF16>::st(p, i, v);
    else Elem<F16>::st(p, i, v);
}

// Sums of N values over a row's WPR waves; every lane receives them. The LDS slots of
// consecutive calls alternate, so one barrier a call is enough: a wave that writes a slot again
// has passed the barrier of the call between, which every wave entered after reading it.
template <int WPR, int N>
struct RowSums {
    float *lds;  // [2][WPR][N]
    int phase = 0;
    __device__ __forceinline__ void operator()(float (&v)[N], int count) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < count) v[i] = group_sum_lanes(v[i], 64);
        if constexpr (WPR > 1) {
            float *s = lds + phase * WPR * N;
            phase ^= 1;
            const int wave = (threadIdx.x >> 6) % WPR;
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int i = 0; i < N; ++i) s[wave * N + i] = v[i];
            __syncthreads();
            const int lane = threadIdx.x & (WPR - 1);  // each lane takes one wave's sum, in every group of WPR lanes
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = group_sum_lanes(s[lane * N + i], WPR);
        }
    }
};

// WPR waves a row, ROWS rows a workgroup at a time: every wave keeps the barriers of the row
// sums, also where its row is past the last.
template <int WPR>
struct RowShape {
    static constexpr int WAVES = WPR > 8 ? WPR : 8, ROWS = WAVES / WPR, THREADS = 64 * WAVES;
};

// Column sums over the workgroups' partials: 32 columns per workgroup, 32 threads per column,
// each over every 32nd partial. blockIdx.y: which of the N sums; partials lie as [workgroup][N][d].
template <int N>
struct SumOut {
    void *out[N];
    int dtype[N];
    int groups[N];  // workgroups with partials: none of a sum that is zero
};
template <int N>
__global__ void __launch_bounds__(1024) column_sums_kernel(const float *__restrict__ part, const SumOut<N> o, int d) {
    __shared__ float lds[32][33];
    const int q = blockIdx.y;
    if (!o.out[q]) return;
    const int groups = o.groups[q];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), r = threadIdx.x >> 5;
    float t = 0.f;
    if (col < d) {
        for (int g = r; g < groups; g += 32 * 4) {
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = g + 32 * u < groups ? part[((int64_t)(g + 32 * u) * N + q) * d + col] : 0.f;
            t += (v[0] + v[1]) + (v[2] + v[3]);
        }
    }
    lds[r][threadIdx.x & 31] = t;
    __syncthreads();
    if (r == 0 && col < d) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += lds[i][threadIdx.x];
        store1_dt(o.out[q], col, o.dtype[q], s);
    }
}

}  // namespace
}  // namespace dsalt
