// A block's branch joined to its residual stream, forward and backward, one pass each. Per row:
//   hd = dropout(h)                        philox.h; hd = h without
//   n  = hd * rh * w_post, rh = rsqrt(mean(hd^2) + post_eps)       n = hd without w_post
//   z  = residual_scale * x + gate * n     gate: per channel, per row, or 1
//   y  = z * r * w, r = rsqrt(mean(z^2) + eps)                     no y without w
// z goes out in x's dtype, y is formed from the fp32 sum. rh and r are kept for the backward,
// which recomputes z from x and h (both of which it needs whatever was kept, where there is a
// gate or a norm of the branch): with dz, dy given and xh = z r, hh = hd rh,
//   t  = dz + r (a - xh mean(a xh)), a = dy * w
//   dx = residual_scale * t,  dw = sum_rows dy xh,  dgate = sum t n over rows or the row
//   b  = gate * t * w_post,  dw_post = sum_rows gate * t * hh
//   dh = dropout(rh (b - hh mean(b hh)))
// Sums are fp32 in a fixed order: per lane over the rows of a workgroup, over its waves in LDS,
// then over the workgroups.
//
// Bound by HBM bytes: a row stays in registers, eight columns a lane, so that every tensor is read
// and written once. Rows of up to 512 columns take one wave, longer ones 2, 4, 8 or 16 whose
// sums are joined in LDS. With 16 columns a lane and half the waves the backward's registers
// leave two waves on a SIMD instead of four, and too few loads in flight: 16384 x 4096 bf16
// backward 178 us (805 MB, 4.5 TB/s) against 212, 6473 x 1024 with an fp32 stream 23.8 us (119 MB,
// 5.0 TB/s) against 29.6. Forward 102 us (537 MB, 5.3 TB/s) and 16.3 us (80 MB, 4.9 TB/s).
#include "launch.h"
#include "lanes.h"
#include "philox.h"
#include "rows.h"

#include <algorithm>

namespace dsalt {
namespace {

enum { kGateNone = 0, kGateChannel = 1, kGateRow = 2 };
enum { kSumW = 0, kSumPost = 1, kSumGate = 2 };

struct BranchParams {
    const void *x, *h, *w, *w_post, *gate;
    int w_dtype, post_dtype, gate_dtype, gate_kind;
    void *x_out, *y;
    int y_dtype;
    float *rstd, *rstd_post;
    const void *dx_out, *dy;
    void *dx, *dh, *d_gate_row;
    float *part;     // [workgroup][3][d]
    int sums;        // bit kSum*: that column sum is wanted
    int64_t rows;
    int nch;         // chunks of eight elements per row
    float inv_d, eps, post_eps, rs;
    DropoutParams drop;
    int dropout;
};

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

template <typename DX, typename DH, int WPR>
__global__ void __launch_bounds__(RowShape<WPR>::THREADS) branch_fwd_kernel(const BranchParams p) {
    constexpr int ROWS = RowShape<WPR>::ROWS;
    __shared__ float lds[ROWS][2 * WPR];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slot = wave / WPR;
    const int ch = (wave % WPR) * 64 + (threadIdx.x & 63);  // the lane's chunk of a row
    const bool in = ch < p.nch;
    RowSums<WPR, 1> row_sum{lds[slot]};
    const uint64_t seed = p.dropout ? dropout_seed(p.drop) : 0;
    float wp[8] = {}, wf[8] = {}, gc[8] = {};
    if (in) {
        if (p.w_post) load8_dt(p.w_post, ch, p.post_dtype, wp);
        if (p.w) load8_dt(p.w, ch, p.w_dtype, wf);
        if (p.gate_kind == kGateChannel) load8_dt(p.gate, ch, p.gate_dtype, gc);
    }
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < p.rows; r0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = r0 + slot, at = row * p.nch + ch;
        const bool live = in && row < p.rows;
        float n[8] = {}, z[8] = {}, g = 1.f, ss[1] = {0.f};
        if (live) {
            Raw8<DX> xv;
            Raw8<DH> hv;
            xv.load(p.x, at);
            hv.load(p.h, at);
            if (p.gate_kind == kGateRow) g = load1_dt(p.gate, row, p.gate_dtype);
            hv.get(n);
            if (p.dropout) apply_keep(keep8<true>((uint64_t)at, p.drop, seed), p.drop.scale, n);
            xv.get(z);
        }
        if (p.w_post) {
#pragma unroll
            for (int e = 0; e < 8; ++e) ss[0] = fmaf(n[e], n[e], ss[0]);
            row_sum(ss, 1);
            const float rh = rsqrtf(ss[0] * p.inv_d + p.post_eps);
            if (live && ch == 0 && p.rstd_post) p.rstd_post[row] = rh;
#pragma unroll
            for (int e = 0; e < 8; ++e) n[e] = n[e] * rh * wp[e];
        }
        ss[0] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            z[e] = fmaf(p.rs, z[e], p.gate_kind == kGateChannel ? gc[e] * n[e] : g * n[e]);
            ss[0] = fmaf(z[e], z[e], ss[0]);
        }
        if (live) store8<DX>(p.x_out, at, z);
        if (!p.w) continue;
        row_sum(ss, 1);
        const float r = rsqrtf(ss[0] * p.inv_d + p.eps);
        if (live) {
            if (ch == 0 && p.rstd) p.rstd[row] = r;
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = z[e] * r * wf[e];
            store8_dt(p.y, at, z, p.y_dtype);
        }
    }
}

template <typename DX, typename DH, int WPR>
__global__ void __launch_bounds__(RowShape<WPR>::THREADS) branch_bwd_kernel(const BranchParams p) {
    constexpr int ROWS = RowShape<WPR>::ROWS;
    __shared__ float lds[ROWS][2 * 2 * WPR];
    __shared__ float4 acc[ROWS > 1 ? ROWS : 1][2][ROWS > 1 ? 64 * WPR : 1];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slot = wave / WPR;
    const int ch = (wave % WPR) * 64 + (threadIdx.x & 63);
    const bool in = ch < p.nch;
    RowSums<WPR, 2> row_sum{lds[slot]};
    const uint64_t seed = p.dropout ? dropout_seed(p.drop) : 0;
    float wp[8], wf[8], gc[8], sum[3][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        wp[e] = gc[e] = 1.f;
        wf[e] = sum[0][e] = sum[1][e] = sum[2][e] = 0.f;
    }
    if (in) {
        if (p.w_post) load8_dt(p.w_post, ch, p.post_dtype, wp);
        if (p.w) load8_dt(p.w, ch, p.w_dtype, wf);
        if (p.gate_kind == kGateChannel) load8_dt(p.gate, ch, p.gate_dtype, gc);
    }
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < p.rows; r0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = r0 + slot, at = row * p.nch + ch;
        const bool live = in && row < p.rows;
        float a[8] = {}, hh[8] = {}, t[8] = {}, dz[8] = {}, r = 0.f, rh = 1.f, g = 1.f;
        uint32_t keep = 0xffu;
        if (live) {
            Raw8<DX> xv, zv = {};
            Raw8<DH> hv;
            xv.load(p.x, at);
            hv.load(p.h, at);
            if (p.dx_out) zv.load(p.dx_out, at);
            if (p.dy) {
                load8_dt(p.dy, at, p.y_dtype, a);
                r = p.rstd[row];
            }
            if (p.w_post) rh = p.rstd_post[row];
            if (p.gate_kind == kGateRow) g = load1_dt(p.gate, row, p.gate_dtype);
            hv.get(hh);
            if (p.dropout) {
                keep = keep8<true>((uint64_t)at, p.drop, seed);
                apply_keep(keep, p.drop.scale, hh);
            }
            xv.get(t);
            zv.get(dz);
        }
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            hh[e] *= rh;
            t[e] = fmaf(p.rs, t[e], g * gc[e] * (hh[e] * wp[e])) * r;  // xh
            sum[kSumW][e] = fmaf(a[e], t[e], sum[kSumW][e]);
            a[e] *= wf[e];
            s[0] = fmaf(a[e], t[e], s[0]);
        }
        if (p.dy) row_sum(s, 1);
        const float c1 = s[0] * p.inv_d;
        s[0] = s[1] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            t[e] = p.dy ? fmaf(r, fmaf(-t[e], c1, a[e]), dz[e]) : dz[e];
            dz[e] = p.rs * t[e];
            const float tn = t[e] * hh[e];
            sum[kSumGate][e] = fmaf(tn, wp[e], sum[kSumGate][e]);
            sum[kSumPost][e] = fmaf(tn, g * gc[e], sum[kSumPost][e]);
            s[1] = fmaf(tn, wp[e], s[1]);
            t[e] *= g * gc[e] * wp[e];
            s[0] = fmaf(t[e], hh[e], s[0]);
        }
        if (live && p.dx) store8<DX>(p.dx, at, dz);
        if (p.w_post || p.d_gate_row) row_sum(s, 2);
        if (!live) continue;
        if (p.d_gate_row && ch == 0) store1_dt(p.d_gate_row, row, p.gate_dtype, s[1]);
        if (p.dh) {
            const float c2 = p.w_post ? s[0] * p.inv_d : 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = rh * fmaf(-hh[e], c2, t[e]);
            if (p.dropout) apply_keep(keep, p.drop.scale, t);
            store8<DH>(p.dh, at, t);
        }
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        if (!((p.sums >> q) & 1)) continue;
        float4 lo = make_float4(sum[q][0], sum[q][1], sum[q][2], sum[q][3]);
        float4 hi = make_float4(sum[q][4], sum[q][5], sum[q][6], sum[q][7]);
        if constexpr (ROWS > 1) {
            __syncthreads();  // the previous sums have been read
            acc[slot][0][ch] = lo;
            acc[slot][1][ch] = hi;
            __syncthreads();
            if (slot) continue;
#pragma unroll
            for (int w = 1; w < ROWS; ++w) {
                const float4 b = acc[w][0][ch], c = acc[w][1][ch];
                lo.x += b.x; lo.y += b.y; lo.z += b.z; lo.w += b.w;
                hi.x += c.x; hi.y += c.y; hi.z += c.z; hi.w += c.w;
            }
        }
        if (in) {
            float4 *out = reinterpret_cast<float4 *>(p.part) + (((int64_t)blockIdx.x * 3 + q) * p.nch + ch) * 2;
            out[0] = lo;
            out[1] = hi;
        }
    }
}

// Column sums over the workgroups' partials: 32 columns per workgroup, 32 threads per column,
// each over every 32nd partial. blockIdx.y: which of the three sums.
struct SumOut {
    void *out[3];
    int dtype[3];
    int groups[3];  // workgroups with partials: none of a sum that is zero
};
__global__ void __launch_bounds__(1024) branch_sums_kernel(const float *__restrict__ part, const SumOut o, int d) {
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
            for (int u = 0; u < 4; ++u) v[u] = g + 32 * u < groups ? part[((int64_t)(g + 32 * u) * 3 + q) * d + col] : 0.f;
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

constexpr int kBranchMaxGroups = 512;  // workgroups of the backward: what its registers allow, two per CU

int row_waves(int d) { return d <= 512 ? 1 : d <= 1024 ? 2 : d <= 2048 ? 4 : d <= 4096 ? 8 : 16; }
int64_t row_groups(int64_t rows, int d) {
    const int per = std::max(8 / row_waves(d), 1);
    return (rows + per - 1) / per;
}
int branch_bwd_groups(int64_t rows, int d) { return (int)std::min<int64_t>(row_groups(rows, d), kBranchMaxGroups); }

template <typename DX, typename DH, int WPR>
void launch_shape(const BranchParams &p, bool bwd, hipStream_t stream) {
    const dim3 block(RowShape<WPR>::THREADS);
    const int64_t groups = row_groups(p.rows, p.nch * 8);
    if (bwd)
        hipLaunchKernelGGL((branch_bwd_kernel<DX, DH, WPR>), dim3(branch_bwd_groups(p.rows, p.nch * 8)), block, 0, stream, p);
    else
        hipLaunchKernelGGL((branch_fwd_kernel<DX, DH, WPR>), dim3((unsigned)std::min<int64_t>(groups, 2048)), block, 0,
                           stream, p);
}

template <typename DX, typename DH>
void launch_types(const BranchParams &p, bool bwd, hipStream_t stream) {
    switch (row_waves(p.nch * 8)) {
        case 1: return launch_shape<DX, DH, 1>(p, bwd, stream);
        case 2: return launch_shape<DX, DH, 2>(p, bwd, stream);
        case 4: return launch_shape<DX, DH, 4>(p, bwd, stream);
        case 8: return launch_shape<DX, DH, 8>(p, bwd, stream);
        default: return launch_shape<DX, DH, 16>(p, bwd, stream);
    }
}

hipError_t launch_branch(const dsalt_branch_norm_args &a, bool bwd, hipStream_t stream) {
    BranchParams p = {};
    p.x = a.x;
    p.h = a.h;
    p.w = a.weight;
    p.w_post = a.post_weight;
    p.gate = a.gate;
    p.w_dtype = a.w_dtype;
    p.post_dtype = a.post_dtype;
    p.gate_dtype = a.gate_dtype;
    p.gate_kind = a.gate_kind;
    p.x_out = a.x_out;
    p.y = a.y;
    p.y_dtype = a.y_dtype;
    p.rstd = a.rstd;
    p.rstd_post = a.rstd_post;
    p.dx_out = a.dx_out;
    p.dy = a.dy;
    p.dx = a.dx;
    p.dh = a.dh;
    p.d_gate_row = a.gate_kind == kGateRow ? a.d_gate : nullptr;
    p.part = static_cast<float *>(a.workspace);
    p.rows = a.rows;
    p.nch = a.d / 8;
    p.inv_d = 1.f / (float)a.d;
    p.eps = a.eps;
    p.post_eps = a.post_eps;
    p.rs = a.residual_scale;
    p.dropout = a.threshold < 65536;
    p.drop = dropout_params(a.threshold, a.seed, a.seed_ptr, a.offset);
    const int groups = branch_bwd_groups(a.rows, a.d);
    // without a gradient of y that of its norm's weight is zero
    SumOut o = {{a.d_weight, a.d_post_weight, a.gate_kind == kGateChannel ? a.d_gate : nullptr},
                {a.w_dtype, a.post_dtype, a.gate_dtype},
                {a.dy ? groups : 0, groups, groups}};
    bool sums = false;
    for (int q = 0; bwd && q < 3; ++q) {
        p.sums |= o.out[q] && o.groups[q] ? 1 << q : 0;
        sums |= o.out[q] != nullptr;
    }
    if (a.rows > 0) {
        if (a.x_dtype == DSALT_DTYPE_BF16) launch_types<BF16, BF16>(p, bwd, stream);
        else if (a.x_dtype == DSALT_DTYPE_F16) launch_types<F16, F16>(p, bwd, stream);
        else if (a.h_dtype == DSALT_DTYPE_BF16) launch_types<F32, BF16>(p, bwd, stream);
        else if (a.h_dtype == DSALT_DTYPE_F16) launch_types<F32, F16>(p, bwd, stream);
        else launch_types<F32, F32>(p, bwd, stream);
    }
    if (sums)
        hipLaunchKernelGGL(branch_sums_kernel, dim3((a.d + 31) / 32, 3), dim3(1024), 0, stream, p.part, o, a.d);
    return hipGetLastError();
}

}  // namespace

int branch_norm_max_dim() { return 8192; }
int64_t branch_norm_workspace_bytes(int64_t rows, int d) { return (int64_t)branch_bwd_groups(rows, d) * 3 * d * 4; }
hipError_t launch_branch_norm(const dsalt_branch_norm_args &a, hipStream_t stream) { return launch_branch(a, false, stream); }
hipError_t launch_branch_norm_bwd(const dsalt_branch_norm_args &a, hipStream_t stream) { return launch_branch(a, true, stream); }

}  // namespace dsalt
