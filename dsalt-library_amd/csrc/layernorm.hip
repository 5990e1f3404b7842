// Layer norm of rows, and of the sum of a residual stream and a branch, forward and backward, one
// pass each. Per row of d columns:
//   z    = x + h                               z = x without h; x_out = z in x's dtype
//   mean = sum(z) / d,  r = rsqrt(sum((z - mean)^2) / d + eps)
//   y    = n * w + b,  n = (z - mean) r        w = 1 without it, b = 0
// y is formed from the fp32 sum. The backward forms z again from x and h (a 16-bit x_out has lost
// bits of it that fp32 gradients of w would show; an fp32 one is z and is read instead):
//   a  = dy * w,  dz = dx_out + r (a - sum(a) / d - n sum(a n) / d)
//   dw = sum over rows of dy n,  db = sum over rows of dy
// The variance is summed from the centred row, which the registers hold: a sum of squares would lose
// it where the mean is large. The centred row's own sum over d is what the mean's rounding to fp32 left
// of it, and is taken off too: a row of equal values is zeros then, and not rounding errors over
// sqrt(eps). Sums are fp32 in a fixed order: per lane over the rows of a workgroup, over its waves in
// LDS, then over the workgroups.
//
// Bound by HBM bytes: a row lies in the registers of one to sixteen waves (eight columns a lane), so that
// each operand is read once and each result written once. 16384 x 4096 bf16 with a branch: 96 us forward
// (5.6 TB/s), 142 us backward (4.7 TB/s) and 5 for the sums over its workgroups; 6473 x 1024, fp32 stream
// and bf16 branch: 17.4 us (4.6 TB/s), 21.9 (4.8) and 3.9; a copy of 1 GiB reaches 5.1 TB/s. One row takes
// 2.8 us: a launch and two exchanges. Widths that are no multiple of 8 and unaligned rows go element by element, two to
// four times as slow: bf16 with a branch, one call after another on the same rows, 6473 x 1023 24 us forward and 47
// backward with its sums (1024: 11 and 17), 16384 x 4097 258 and 520 (4096: 98 and 118).
#include "launch.h"
#include "rowsums.h"

#include <algorithm>

namespace dsalt {
namespace {

enum { kSumW = 0, kSumB = 1 };

struct LayerParams {
    const void *x, *h, *w, *b;
    void *x_out, *y;
    float *stats;  // [3][rows]: mean, what its rounding left, r; may be NULL in the forward
    const void *dx_out, *dy;
    void *dx, *dh;
    float *part;  // [workgroup][2][d]
    int64_t rows;
    int y_dtype, w_dtype, b_dtype, dh_dtype;
    int sums;  // bit kSum*: that column sum is wanted
    int d;
    float inv_d, eps;
};

// A lane's eight columns of a row: VEC: the consecutive ones of its chunk, 16 bytes at a time (d a
// multiple of 8, aligned tensors); otherwise every 64 WPR-th, an element at a time.
template <int WPR, bool VEC>
struct Columns {
    int ch, d;
    // Unhoisted: element offsets formed in the loop over the rows; kept across it, with every tensor's
    // addresses, they take more registers than a workgroup of 16 waves has.
    __device__ __forceinline__ Columns unhoisted() const {
        Columns c = *this;
        if constexpr (!VEC) asm volatile("" : "+v"(c.ch));
        return c;
    }
    __device__ __forceinline__ int col(int e) const { return VEC ? ch * 8 + e : ch + e * 64 * WPR; }
    __device__ __forceinline__ bool in(int e) const { return col(e) < d; }
    // the row's first element (uniform over the wave: the lanes add 32-bit offsets)
    template <typename DT>
    __device__ __forceinline__ const char *row_of(const void *p, int64_t row) const {
        return static_cast<const char *>(p) + row * d * (std::is_same<DT, F32>::value ? 4 : 2);
    }
    // elements of row `row` as fp32, zeros past d
    template <typename DT>
    __device__ __forceinline__ void load(const void *p, int64_t row, float (&v)[8]) const {
        if constexpr (VEC) {
            Raw8<DT> raw = {};
            if (in(0)) raw.load(p, row * (d >> 3) + ch);
            raw.get(v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = in(e) ? Elem<DT>::ld(row_of<DT>(p, row), (uint32_t)col(e)) : 0.f;
        }
    }
    __device__ __forceinline__ void load_dt(const void *p, int64_t row, int dtype, float (&v)[8]) const {
        if (dtype == DSALT_DTYPE_F32) load<F32>(p, row, v);
        else if (dtype == DSALT_DTYPE_BF16) load<BF16>(p, row, v);
        else load<F16>(p, row, v);
    }
    template <typename DT>
    __device__ __forceinline__ void store(void *p, int64_t row, const float (&v)[8]) const {
        if constexpr (VEC) {
            if (in(0)) store8<DT>(p, row * (d >> 3) + ch, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (in(e)) Elem<DT>::st(const_cast<char *>(row_of<DT>(p, row)), (uint32_t)col(e), v[e]);
        }
    }
    __device__ __forceinline__ void store_dt(void *p, int64_t row, int dtype, const float (&v)[8]) const {
        if (dtype == DSALT_DTYPE_F32) store<F32>(p, row, v);
        else if (dtype == DSALT_DTYPE_BF16) store<BF16>(p, row, v);
        else store<F16>(p, row, v);
    }
};

template <typename DX, typename DH, int WPR, bool VEC>
__global__ void __launch_bounds__(RowShape<WPR>::THREADS) layer_fwd_kernel(const LayerParams p) {
    constexpr int ROWS = RowShape<WPR>::ROWS;
    __shared__ float lds[ROWS][2 * 2 * WPR];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slot = wave / WPR;
    const Columns<WPR, VEC> cols{(int)((wave % WPR) * 64 + (threadIdx.x & 63)), p.d};
    RowSums<WPR, 2> row_sum{lds[slot]};
    float w[8], b[8] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.f;
    if (p.w) cols.load_dt(p.w, 0, p.w_dtype, w);
    if (p.b) cols.load_dt(p.b, 0, p.b_dtype, b);
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < p.rows; r0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = r0 + slot;
        const Columns<WPR, VEC> at = cols.unhoisted();
        const bool live = row < p.rows;  // uniform over the wave
        float z[8] = {}, s[2] = {0.f, 0.f};
        if (live) {
            at.template load<DX>(p.x, row, z);
            if (p.h) {
                float h[8];
                at.template load<DH>(p.h, row, h);
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] += h[e];
                at.template store<DX>(p.x_out, row, z);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) s[0] += z[e];
        row_sum(s, 1);
        float mean = s[0] * p.inv_d;
        asm volatile("" : "+v"(mean));  // the rounded one, as the backward has it: not z - s inv_d in one step
        s[0] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            z[e] = at.in(e) ? z[e] - mean : 0.f;
            s[0] += z[e];
            s[1] = fmaf(z[e], z[e], s[1]);
        }
        row_sum(s, 2);
        const float rest = s[0] * p.inv_d;
        const float r = rsqrtf(fmaxf(fmaf(-s[0], rest, s[1]), 0.f) * p.inv_d + p.eps);
        if (!live) continue;
        if (p.stats && at.ch == 0) {
            p.stats[row] = mean;
            p.stats[p.rows + row] = rest;
            p.stats[2 * p.rows + row] = r;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = fmaf((z[e] - rest) * r, w[e], b[e]);
        at.store_dt(p.y, row, p.y_dtype, z);
    }
}

template <typename DX, typename DH, int WPR, bool VEC>
__global__ void __launch_bounds__(RowShape<WPR>::THREADS) layer_bwd_kernel(const LayerParams p) {
    constexpr int ROWS = RowShape<WPR>::ROWS;
    __shared__ float lds[ROWS][2 * 2 * WPR];
    __shared__ float acc[ROWS > 1 ? ROWS : 1][8][ROWS > 1 ? 64 * WPR : 1];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slot = wave / WPR;
    const Columns<WPR, VEC> cols{(int)((wave % WPR) * 64 + (threadIdx.x & 63)), p.d};
    RowSums<WPR, 2> row_sum{lds[slot]};
    float w[8], sum[2][8] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.f;
    if (p.w) cols.load_dt(p.w, 0, p.w_dtype, w);
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < p.rows; r0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = r0 + slot;
        const Columns<WPR, VEC> at = cols.unhoisted();
        const bool live = row < p.rows;
        float n[8] = {}, a[8] = {}, dz[8] = {}, mean = 0.f, rest = 0.f, r = 0.f;
        if (live) {
            at.template load<DX>(p.x, row, n);
            at.load_dt(p.dy, row, p.y_dtype, a);
            if (p.dx_out) at.template load<DX>(p.dx_out, row, dz);
            mean = p.stats[row];
            rest = p.stats[p.rows + row];
            r = p.stats[2 * p.rows + row];
            if (p.h) {
                float h[8];
                at.template load<DH>(p.h, row, h);
#pragma unroll
                for (int e = 0; e < 8; ++e) n[e] += h[e];
            }
        }
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            n[e] = ((n[e] - mean) - rest) * r;  // past d: a = 0
            sum[kSumW][e] = fmaf(a[e], n[e], sum[kSumW][e]);
            sum[kSumB][e] += a[e];
            a[e] *= w[e];
            s[0] += a[e];
            s[1] = fmaf(a[e], n[e], s[1]);
        }
        if (!p.dx && !p.dh) continue;  // uniform over the grid
        row_sum(s, 2);
        if (!live) continue;
        const float c0 = s[0] * p.inv_d, c1 = s[1] * p.inv_d;
#pragma unroll
        for (int e = 0; e < 8; ++e) dz[e] = fmaf(r, fmaf(-n[e], c1, a[e] - c0), dz[e]);
        if (p.dx) at.template store<DX>(p.dx, row, dz);
        if (p.dh) at.store_dt(p.dh, row, p.dh_dtype, dz);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        if (!((p.sums >> q) & 1)) continue;
        if constexpr (ROWS > 1) {
            __syncthreads();  // the previous sums have been read
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[slot][e][cols.ch] = sum[q][e];
            __syncthreads();
            if (slot) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int i = 1; i < ROWS; ++i) sum[q][e] += acc[i][e][cols.ch];
        }
        cols.template store<F32>(p.part, (int64_t)blockIdx.x * 2 + q, sum[q]);
    }
}

constexpr int kLayerMaxGroups = 512;  // workgroups of the backward, whose sums the second kernel reads

int row_waves(int d) { return d <= 512 ? 1 : d <= 1024 ? 2 : d <= 2048 ? 4 : d <= 4096 ? 8 : 16; }
int64_t row_groups(int64_t rows, int d) {
    const int per = std::max(8 / row_waves(d), 1);
    return (rows + per - 1) / per;
}
int layer_bwd_groups(int64_t rows, int d) { return (int)std::min<int64_t>(row_groups(rows, d), kLayerMaxGroups); }

template <typename DX, typename DH, int WPR, bool VEC>
void launch_shape(const LayerParams &p, bool bwd, hipStream_t stream) {
    const dim3 block(RowShape<WPR>::THREADS);
    if (bwd)
        hipLaunchKernelGGL((layer_bwd_kernel<DX, DH, WPR, VEC>), dim3(layer_bwd_groups(p.rows, p.d)), block, 0, stream, p);
    else
        hipLaunchKernelGGL((layer_fwd_kernel<DX, DH, WPR, VEC>),
                           dim3((unsigned)std::min<int64_t>(row_groups(p.rows, p.d), 2048)), block, 0, stream, p);
}

template <typename DX, typename DH, bool VEC>
void launch_width(const LayerParams &p, bool bwd, hipStream_t stream) {
    switch (row_waves(p.d)) {
        case 1: return launch_shape<DX, DH, 1, VEC>(p, bwd, stream);
        case 2: return launch_shape<DX, DH, 2, VEC>(p, bwd, stream);
        case 4: return launch_shape<DX, DH, 4, VEC>(p, bwd, stream);
        case 8: return launch_shape<DX, DH, 8, VEC>(p, bwd, stream);
        default: return launch_shape<DX, DH, 16, VEC>(p, bwd, stream);
    }
}

hipError_t launch_layer(const dsalt_layer_norm_args &a, bool bwd, hipStream_t stream) {
    LayerParams p = {};
    p.x = a.x;
    p.h = a.h;
    p.w = a.weight;
    p.b = a.bias;
    p.x_out = a.x_out;
    p.y = a.y;
    p.stats = a.stats;
    p.dx_out = a.dx_out;
    p.dy = a.dy;
    p.dx = a.dx;
    p.dh = a.dh;
    p.part = static_cast<float *>(a.workspace);
    p.rows = a.rows;
    p.y_dtype = a.y_dtype;
    p.w_dtype = a.w_dtype;
    p.b_dtype = a.b_dtype;
    p.dh_dtype = a.h_dtype;
    p.d = a.d;
    p.inv_d = 1.f / (float)a.d;
    p.eps = a.eps;
    const int groups = layer_bwd_groups(a.rows, a.d);
    const SumOut<2> o = {{a.d_weight, a.d_bias}, {a.w_dtype, a.b_dtype}, {groups, groups}};
    const bool sums = bwd && (a.d_weight || a.d_bias);
    p.sums = (a.d_weight ? 1 << kSumW : 0) | (a.d_bias ? 1 << kSumB : 0);
    if (a.rows > 0) {
        uintptr_t all = (uintptr_t)(a.d % 8 * 2);  // 16-byte pieces of every tensor
        for (const void *t : {a.x, a.h, a.weight, a.bias, (const void *)a.x_out, (const void *)a.y, a.dx_out, a.dy,
                              (const void *)a.dx, (const void *)a.dh, (const void *)a.workspace})
            all |= (uintptr_t)t;
        const auto go = [&](auto dx, auto dh) {
            if (all % 16 == 0) launch_width<decltype(dx), decltype(dh), true>(p, bwd, stream);
            else launch_width<decltype(dx), decltype(dh), false>(p, bwd, stream);
        };
        if (a.x_dtype == DSALT_DTYPE_BF16) go(BF16(), BF16());
        else if (a.x_dtype == DSALT_DTYPE_F16) go(F16(), F16());
        else if (a.h && a.h_dtype == DSALT_DTYPE_BF16) go(F32(), BF16());
        else if (a.h && a.h_dtype == DSALT_DTYPE_F16) go(F32(), F16());
        else go(F32(), F32());
    }
    if (sums) hipLaunchKernelGGL(column_sums_kernel<2>, dim3((a.d + 31) / 32, 2), dim3(1024), 0, stream, p.part, o, a.d);
    return hipGetLastError();
}

}  // namespace

int layer_norm_max_dim() { return 8192; }
int64_t layer_norm_workspace_bytes(int64_t rows, int d) { return (int64_t)layer_bwd_groups(rows, d) * 2 * d * 4; }
hipError_t launch_layer_norm(const dsalt_layer_norm_args &a, hipStream_t stream) { return launch_layer(a, false, stream); }
hipError_t launch_layer_norm_bwd(const dsalt_layer_norm_args &a, hipStream_t stream) { return launch_layer(a, true, stream); }

}  // namespace dsalt
