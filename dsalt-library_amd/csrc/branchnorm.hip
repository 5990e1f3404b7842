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
// Bound by HBM bytes: a row stays in the registers of one wave (d <= 1024), four (d <= 4096) or
// eight, so that every tensor is read and written once.
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
            const int wave = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int i = 0; i < N; ++i) s[wave * N + i] = v[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float t = 0.f;
#pragma unroll
                for (int w = 0; w < WPR; ++w) t += s[w * N + i];
                v[i] = t;
            }
        }
    }
};

constexpr int branch_waves(int wpr) { return wpr > 4 ? wpr : 4; }

// A wave's share of its rows: chunk c of lane l is chunk c * 64 WPR + l of the row. All rows of a
// workgroup with WPR > 1 are the same row, so its barriers are met by every wave.
template <typename DX, typename DH, int NCH, int WPR>
__global__ void __launch_bounds__(64 * branch_waves(WPR)) branch_fwd_kernel(const BranchParams p) {
    constexpr int NW = branch_waves(WPR), ROWS = NW / WPR;
    __shared__ float lds[2 * WPR];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l = (wave % WPR) * 64 + (threadIdx.x & 63);
    RowSums<WPR, 1> row_sum{lds};
    const uint64_t seed = p.dropout ? dropout_seed(p.drop) : 0;
    float wp[NCH][8], wf[NCH][8], gc[NCH][8];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int ch = c * 64 * WPR + l;
        if (ch < p.nch) {
            if (p.w_post) load8_dt(p.w_post, ch, p.post_dtype, wp[c]);
            if (p.w) load8_dt(p.w, ch, p.w_dtype, wf[c]);
            if (p.gate_kind == kGateChannel) load8_dt(p.gate, ch, p.gate_dtype, gc[c]);
        }
    }
    for (int64_t row = (int64_t)blockIdx.x * ROWS + wave / WPR; row < p.rows; row += (int64_t)gridDim.x * ROWS) {
        const int64_t base = row * p.nch;
        Raw8<DX> xv[NCH];
        Raw8<DH> hv[NCH];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int ch = c * 64 * WPR + l;
            if (ch < p.nch) {
                xv[c].load(p.x, base + ch);
                hv[c].load(p.h, base + ch);
            }
        }
        float n[NCH][8], g = 1.f, ss[1] = {0.f};
        if (p.gate_kind == kGateRow) g = load1_dt(p.gate, row, p.gate_dtype);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int ch = c * 64 * WPR + l;
            if (ch < p.nch) {
                hv[c].get(n[c]);
                if (p.dropout) apply_keep(keep8<true>((uint64_t)(base + ch), p.drop, seed), p.drop.scale, n[c]);
#pragma unroll
                for (int e = 0; e < 8; ++e) ss[0] = fmaf(n[c][e], n[c][e], ss[0]);
            }
        }
        if (p.w_post) {
            row_sum(ss, 1);
            const float rh = rsqrtf(ss[0] * p.inv_d + p.post_eps);
            if (l == 0 && p.rstd_post) p.rstd_post[row] = rh;
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) n[c][e] = n[c][e] * rh * wp[c][e];
        }
        ss[0] = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int ch = c * 64 * WPR + l;
            if (ch < p.nch) {
                float z[8];
                xv[c].get(z);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float gn = p.gate_kind == kGateChannel ? gc[c][e] * n[c][e] : g * n[c][e];
                    z[e] = fmaf(p.rs, z[e], gn);
                    n[c][e] = z[e];
                    ss[0] = fmaf(z[e], z[e], ss[0]);
                }
                store8<DX>(p.x_out, base + ch, z);
            }
        }
        if (!p.w) continue;
        row_sum(ss, 1);
        const float r = rsqrtf(ss[0] * p.inv_d + p.eps);
        if (l == 0 && p.rstd) p.rstd[row] = r;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int ch = c * 64 * WPR + l;
            if (ch < p.nch) {
#pragma unroll
                for (int e = 0; e < 8; ++e) n[c][e] = n[c][e] * r * wf[c][e];
                store8_dt(p.y, base + ch, n[c], p.y_dtype);
            }
        }
    }
}

template <typename DX, typename DH, int NCH, int WPR>
__global__ void __launch_bounds__(64 * branch_waves(WPR)) branch_bwd_kernel(const BranchParams p) {
    constexpr int NW = branch_waves(WPR), ROWS = NW / WPR;
    __shared__ float lds[2 * 2 * WPR];
    __shared__ float4 acc[WPR == 1 ? NW : 1][NCH * 2][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int l = (wave % WPR) * 64 + lane;
    RowSums<WPR, 2> row_sum{lds};
    const uint64_t seed = p.dropout ? dropout_seed(p.drop) : 0;
    float wp[NCH][8], wf[NCH][8], gc[NCH][8], sum[3][NCH][8];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int ch = c * 64 * WPR + l;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            wp[c][e] = gc[c][e] = 1.f;
            wf[c][e] = 0.f;
            sum[0][c][e] = sum[1][c][e] = sum[2][c][e] = 0.f;
        }
        if (ch < p.nch) {
            if (p.w_post) load8_dt(p.w_post, ch, p.post_dtype, wp[c]);
            if (p.w) load8_dt(p.w, ch, p.w_dtype, wf[c]);
            if (p.gate_kind == kGateChannel) load8_dt(p.gate, ch, p.gate_dtype, gc[c]);
        }
    }
    for (int64_t row = (int64_t)blockIdx.x * ROWS + wave / WPR; row < p.rows; row += (int64_t)gridDim.x * ROWS) {
        const int64_t base = row * p.nch;
        Raw8<DX> xv[NCH], zv[NCH];
        Raw8<DH> hv[NCH];
        float a[NCH][8];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int ch = c * 64 * WPR + l;
            if (ch < p.nch) {
                xv[c].load(p.x, base + ch);
                hv[c].load(p.h, base + ch);
                if (p.dx_out) zv[c].load(p.dx_out, base + ch);
                if (p.dy) load8_dt(p.dy, base + ch, p.y_dtype, a[c]);
            }
        }
        const float r = p.dy ? p.rstd[row] : 0.f, rh = p.w_post ? p.rstd_post[row] : 1.f;
        const float g = p.gate_kind == kGateRow ? load1_dt(p.gate, row, p.gate_dtype) : 1.f;
        uint32_t keep[NCH];
        float hh[NCH][8], t[NCH][8], s[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int ch = c * 64 * WPR + l;
            keep[c] = 0xffu;
            if (ch < p.nch) {
                hv[c].get(hh[c]);
                if (p.dropout) {
                    keep[c] = keep8<true>((uint64_t)(base + ch), p.drop, seed);
                    apply_keep(keep[c], p.drop.scale, hh[c]);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) hh[c][e] *= rh;
                if (p.dy) {
                    xv[c].get(t[c]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float xh = fmaf(p.rs, t[c][e], g * gc[c][e] * (hh[c][e] * wp[c][e])) * r;
                        sum[kSumW][c][e] = fmaf(a[c][e], xh, sum[kSumW][c][e]);
                        a[c][e] *= wf[c][e];
                        t[c][e] = xh;
                        s[0] = fmaf(a[c][e], xh, s[0]);
                    }
                }
            }
        }
        float c1 = 0.f;
        if (p.dy) {
            row_sum(s, 1);
            c1 = s[0] * p.inv_d;
        }
        s[0] = s[1] = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int ch = c * 64 * WPR + l;
            if (ch < p.nch) {
                float o[8];
                if (p.dx_out) zv[c].get(o);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float dn = p.dy ? r * fmaf(-t[c][e], c1, a[c][e]) : 0.f;
                    t[c][e] = p.dx_out ? o[e] + dn : dn;
                    o[e] = p.rs * t[c][e];
                }
                if (p.dx) store8<DX>(p.dx, base + ch, o);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float tn = t[c][e] * hh[c][e];
                    sum[kSumGate][c][e] = fmaf(tn, wp[c][e], sum[kSumGate][c][e]);
                    sum[kSumPost][c][e] = fmaf(tn, g * gc[c][e], sum[kSumPost][c][e]);
                    s[1] = fmaf(tn, wp[c][e], s[1]);
                    t[c][e] *= g * gc[c][e] * wp[c][e];
                    s[0] = fmaf(t[c][e], hh[c][e], s[0]);
                }
            }
        }
        if (p.w_post || p.d_gate_row) row_sum(s, 2);
        if (p.d_gate_row && l == 0) store1_dt(p.d_gate_row, row, p.gate_dtype, s[1]);
        if (p.dh) {
            const float c2 = p.w_post ? s[0] * p.inv_d : 0.f;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int ch = c * 64 * WPR + l;
                if (ch < p.nch) {
                    float o[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] = rh * fmaf(-hh[c][e], c2, t[c][e]);
                    if (p.dropout) apply_keep(keep[c], p.drop.scale, o);
                    store8<DH>(p.dh, base + ch, o);
                }
            }
        }
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        if (!((p.sums >> q) & 1)) continue;
        float4 *out = reinterpret_cast<float4 *>(p.part) + ((int64_t)blockIdx.x * 3 + q) * p.nch * 2;
        if constexpr (WPR > 1) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int ch = c * 64 * WPR + l;
                if (ch < p.nch) {
                    const float *v = sum[q][c];
                    out[2 * ch] = make_float4(v[0], v[1], v[2], v[3]);
                    out[2 * ch + 1] = make_float4(v[4], v[5], v[6], v[7]);
                }
            }
        } else {
            __syncthreads();  // the previous sums have been read
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const float *v = sum[q][c];
                acc[wave][2 * c][lane] = make_float4(v[0], v[1], v[2], v[3]);
                acc[wave][2 * c + 1][lane] = make_float4(v[4], v[5], v[6], v[7]);
            }
            __syncthreads();
            for (int i = threadIdx.x; i < NCH * 2 * 64; i += 64 * NW) {
                const int ln = i & 63, hc = i >> 6;
                float4 s = acc[0][hc][ln];
#pragma unroll
                for (int w = 1; w < NW; ++w) {
                    const float4 b = acc[w][hc][ln];
                    s.x += b.x; s.y += b.y; s.z += b.z; s.w += b.w;
                }
                const int ch = (hc >> 1) * 64 + ln;
                if (ch < p.nch) out[2 * ch + (hc & 1)] = s;
            }
        }
    }
}

// Column sums over the workgroups' partials: 32 columns per workgroup, 32 threads per column,
// each over every 32nd partial. blockIdx.y: which of the three sums.
struct SumOut {
    void *out[3];
    int dtype[3];
};
__global__ void __launch_bounds__(1024) branch_sums_kernel(const float *__restrict__ part, const SumOut o, int groups, int d) {
    __shared__ float lds[32][33];
    const int q = blockIdx.y;
    if (!o.out[q]) return;
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

constexpr int kBranchMaxGroups = 512;

int64_t row_groups(int64_t rows, int d) {
    const int per = d <= 1024 ? 4 : 1;
    return (rows + per - 1) / per;
}
int branch_bwd_groups(int64_t rows, int d) { return (int)std::min<int64_t>(row_groups(rows, d), kBranchMaxGroups); }

template <typename DX, typename DH, int NCH, int WPR>
void launch_shape(const BranchParams &p, bool bwd, hipStream_t stream) {
    const dim3 block(64 * branch_waves(WPR));
    if (bwd)
        hipLaunchKernelGGL((branch_bwd_kernel<DX, DH, NCH, WPR>), dim3(branch_bwd_groups(p.rows, p.nch * 8)), block, 0,
                           stream, p);
    else
        hipLaunchKernelGGL((branch_fwd_kernel<DX, DH, NCH, WPR>),
                           dim3((unsigned)std::min<int64_t>(row_groups(p.rows, p.nch * 8), 2048)), block, 0, stream, p);
}

template <typename DX, typename DH>
void launch_types(const BranchParams &p, bool bwd, hipStream_t stream) {
    if (p.nch <= 64) launch_shape<DX, DH, 1, 1>(p, bwd, stream);
    else if (p.nch <= 128) launch_shape<DX, DH, 2, 1>(p, bwd, stream);
    else if (p.nch <= 256) launch_shape<DX, DH, 1, 4>(p, bwd, stream);
    else if (p.nch <= 512) launch_shape<DX, DH, 2, 4>(p, bwd, stream);
    else launch_shape<DX, DH, 2, 8>(p, bwd, stream);
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
    SumOut o = {{a.dy || a.rows == 0 ? a.d_weight : nullptr, a.d_post_weight, a.gate_kind == kGateChannel ? a.d_gate : nullptr},
                {a.w_dtype, a.post_dtype, a.gate_dtype}};
    if (bwd)
        for (int q = 0; q < 3; ++q) p.sums |= o.out[q] ? 1 << q : 0;
    if (a.rows > 0) {
        if (a.x_dtype == DSALT_DTYPE_BF16) launch_types<BF16, BF16>(p, bwd, stream);
        else if (a.x_dtype == DSALT_DTYPE_F16) launch_types<F16, F16>(p, bwd, stream);
        else if (a.h_dtype == DSALT_DTYPE_BF16) launch_types<F32, BF16>(p, bwd, stream);
        else if (a.h_dtype == DSALT_DTYPE_F16) launch_types<F32, F16>(p, bwd, stream);
        else launch_types<F32, F32>(p, bwd, stream);
    }
    if (p.sums)
        hipLaunchKernelGGL(branch_sums_kernel, dim3((a.d + 31) / 32, 3), dim3(1024), 0, stream, p.part, o,
                           branch_bwd_groups(a.rows, a.d), a.d);
    return hipGetLastError();
}

}  // namespace

int branch_norm_max_dim() { return 8192; }
int64_t branch_norm_workspace_bytes(int64_t rows, int d) { return (int64_t)branch_bwd_groups(rows, d) * 3 * d * 4; }
hipError_t launch_branch_norm(const dsalt_branch_norm_args &a, hipStream_t stream) { return launch_branch(a, false, stream); }
hipError_t launch_branch_norm_bwd(const dsalt_branch_norm_args &a, hipStream_t stream) { return launch_branch(a, true, stream); }

}  // namespace dsalt
