// Gated feed-forward block, forward and backward:
//   g = x Wg^T, u = x Wu^T, a = act(g) * u, y = a Wd^T
//   da = dy Wd, dg = da * u * act'(g), du = da * act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T a
// Reference: SwiGLUFFN (dsalt/modules/dsalt_transformer.py:10-21) with torch's autograd.
//
// Gate and up projection, activation and product are one kernel: a workgroup's B tile holds
// the same columns of both weights, so that a lane ends with g and u of the same elements
// in its fp32 accumulators and rounds only a (and g, u where a backward will read them). The
// backward's first kernel ends da = dy Wd in the gradients of g and u the same way: da is
// never written.
#include "gemm.h"
#include "launch.h"

#include <algorithm>

namespace dsalt {
namespace {

constexpr float kGeluTanhC = 0.7978845608028654f;  // sqrt(2 / pi)

// act(g) and act'(g) in fp32. exp and reciprocal are the hardware's (1 ulp): their results are
// rounded to 16 bits next.
template <int ACT>
__device__ __forceinline__ void act_grad(float g, float &v, float &slope) {
    if constexpr (ACT == DSALT_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + fast_exp2(-g * kLog2e));
        v = g * s;
        slope = s * (1.f + g * (1.f - s));
    } else if constexpr (ACT == DSALT_ACT_GELU_TANH) {
        // 0.5 (1 + tanh z) = sigmoid(2 z); past |g| = 30 it is 0 or 1 and z would overflow
        const float c = fminf(fmaxf(g, -30.f), 30.f), c2 = c * c;
        const float z2 = 2.f * kGeluTanhC * c * (1.f + 0.044715f * c2);
        const float s = __builtin_amdgcn_rcpf(1.f + fast_exp2(-z2 * kLog2e));
        v = g * s;
        slope = s + g * s * (1.f - s) * (2.f * kGeluTanhC) * (1.f + 3.f * 0.044715f * c2);
    } else if constexpr (ACT == DSALT_ACT_GELU) {
        const float phi = 0.5f * erfcf(-0.7071067811865476f * g);
        v = g * phi;
        slope = phi + g * 0.3989422804014327f * fast_exp2(-0.5f * kLog2e * g * g);
    } else {
        const bool off = g <= 0.f;  // NaN stays NaN
        v = off ? 0.f : g;
        slope = off ? 0.f : 1.f;
    }
}
template <int ACT>
__device__ __forceinline__ float act_value(float g) {
    float v, s;
    act_grad<ACT>(g, v, s);
    return v;
}

struct FfnParams {
    GemmOperand a[2], b[2];
    int64_t m, n, k;     // of the product (PAIR: n of one matrix)
    int tiles_m, tiles_n;
    char *out[2];
    int64_t out_ld;      // bytes
    const char *gu;      // gate | up, row stride gu_ld bytes, up at gu + up_off
    int64_t gu_ld, up_off;
};

// Tile of workgroup `id`: each XCD takes a contiguous range of ids, ids run over kGroup m-tiles
// before the next n-tile, so that the workgroups that run at a time share operand rows in their L2.
constexpr int kGroup = 8;
__device__ __forceinline__ bool tile_of(int id, int tiles_m, int tiles_n, int &tm, int &tn) {
    const int l = xcd_remap(id, gridDim.x);
    if (l >= tiles_m * tiles_n) return false;
    const int per = kGroup * tiles_n, g = l / per, r = l - g * per, rows = min(kGroup, tiles_m - g * kGroup);
    tn = r / rows;
    tm = g * kGroup + r - tn * rows;
    return true;
}

enum { kEpiUp, kEpiUpSave, kEpiStore, kEpiGrad };

template <class DT, int BM, int BN, int WM, int WN, int ALAY, int BLAY, int SEGMENTS, int EPI, int ACT>
__global__ void __launch_bounds__(WM *WN * 64) ffn_kernel(FfnParams p) {
    constexpr bool PAIR = EPI == kEpiUp || EPI == kEpiUpSave;
    typedef GemmCore<DT, BM, BN, WM, WN, ALAY, BLAY, PAIR> Core;
    __shared__ __attribute__((aligned(16))) char lds[Core::LDS_BYTES];
    int tm, tn;
    if (!tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn)) return;
    constexpr int BNO = PAIR ? BN / 2 : BN;  // columns of the output
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BNO;
    const int z = blockIdx.y;  // independent products of one shape: their a operand and output
    Core c;
    if constexpr (SEGMENTS == 1 && !PAIR) {
        c.template run<1>(lds, &p.a[z], &p.b[0], m0, n0, p.k, 0, (int)((p.k + kGemmBK - 1) / kGemmBK));
    } else {
        c.template run<SEGMENTS>(lds, p.a, p.b, m0, n0, p.k, 0, SEGMENTS * (int)((p.k + kGemmBK - 1) / kGemmBK));
    }
#pragma unroll
    for (int i = 0; i < Core::FM; ++i) {
        const int64_t m = m0 + c.row(i);
        if (m >= p.m) continue;
        constexpr int FO = PAIR ? Core::FN / 2 : Core::FN;
#pragma unroll
        for (int j = 0; j < FO; ++j) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int64_t n = n0 + (c.wn * FO + j) * 32 + c.col(half);
                float v[8], u[8], w[8];
                c.values(c.acc[i][j], half, v);
                if constexpr (PAIR) {
                    c.values(c.acc[i][FO + j], half, u);
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = act_value<ACT>(v[e]) * u[e];
                }
                if (n >= p.n) continue;
                if constexpr (PAIR) {
                    *reinterpret_cast<uint4 *>(p.out[0] + m * p.out_ld + n * 2) = pack8<DT>(w);
                    if constexpr (EPI == kEpiUpSave) {
                        char *gu = p.out[1] + m * p.gu_ld + n * 2;
                        *reinterpret_cast<uint4 *>(gu) = pack8<DT>(v);
                        *reinterpret_cast<uint4 *>(gu + p.up_off) = pack8<DT>(u);
                    }
                } else if constexpr (EPI == kEpiStore) {
                    *reinterpret_cast<uint4 *>(p.out[z] + m * p.out_ld + n * 2) = pack8<DT>(v);
                } else {
                    const char *gu = p.gu + m * p.gu_ld + n * 2;
                    float g[8];
                    unpack8<DT>(*reinterpret_cast<const uint4 *>(gu), g);
                    unpack8<DT>(*reinterpret_cast<const uint4 *>(gu + p.up_off), u);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float act, slope;
                        act_grad<ACT>(g[e], act, slope);
                        w[e] = v[e] * act;
                        v[e] = v[e] * u[e] * slope;
                    }
                    char *o = p.out[0] + m * p.out_ld + n * 2;
                    *reinterpret_cast<uint4 *>(o) = pack8<DT>(v);
                    *reinterpret_cast<uint4 *>(o + p.up_off) = pack8<DT>(w);
                }
            }
        }
    }
}

template <class DT, int ALAY, int BLAY, int SEGMENTS, int EPI, int ACT>
void launch_product(FfnParams p, int batch, hipStream_t stream) {
    constexpr int BM = 128, BN = 128;
    constexpr bool PAIR = EPI == kEpiUp || EPI == kEpiUpSave;
    p.tiles_m = (int)((p.m + BM - 1) / BM);
    p.tiles_n = (int)((p.n + (PAIR ? BN / 2 : BN) - 1) / (PAIR ? BN / 2 : BN));
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    if (tiles == 0) return;
    const dim3 grid((unsigned)((tiles + 7) / 8 * 8), (unsigned)batch);
    hipLaunchKernelGGL((ffn_kernel<DT, BM, BN, 2, 2, ALAY, BLAY, SEGMENTS, EPI, ACT>), grid, dim3(256), 0, stream, p);
}

template <class DT, int ALAY, int BLAY, int SEGMENTS, int EPI>
void launch_act(const FfnParams &p, int act, hipStream_t stream) {
    switch (act) {
        case DSALT_ACT_SILU: return launch_product<DT, ALAY, BLAY, SEGMENTS, EPI, DSALT_ACT_SILU>(p, 1, stream);
        case DSALT_ACT_GELU: return launch_product<DT, ALAY, BLAY, SEGMENTS, EPI, DSALT_ACT_GELU>(p, 1, stream);
        case DSALT_ACT_GELU_TANH: return launch_product<DT, ALAY, BLAY, SEGMENTS, EPI, DSALT_ACT_GELU_TANH>(p, 1, stream);
        default: return launch_product<DT, ALAY, BLAY, SEGMENTS, EPI, DSALT_ACT_RELU>(p, 1, stream);
    }
}

GemmOperand operand(const void *p, int64_t ld, int64_t rows) { return {static_cast<const char *>(p), ld * 2, rows}; }

template <class DT>
void forward(const dsalt_gated_ffn_args &a, hipStream_t stream) {
    FfnParams p{};
    p.m = a.rows;
    p.n = a.f;
    p.k = a.d;
    p.a[0] = operand(a.x, a.x_stride, a.rows);
    p.b[0] = operand(a.w_gate, a.w_gate_stride, a.f);
    p.b[1] = operand(a.w_up, a.w_up_stride, a.f);
    p.out[0] = static_cast<char *>(a.act);
    p.out_ld = (int64_t)a.f * 2;
    if (a.gate_up) {
        p.out[1] = static_cast<char *>(a.gate_up);
        p.gu_ld = (int64_t)a.f * 4;
        p.up_off = (int64_t)a.f * 2;
        launch_act<DT, kKContig, kKContig, 1, kEpiUpSave>(p, a.activation, stream);
    } else {
        launch_act<DT, kKContig, kKContig, 1, kEpiUp>(p, a.activation, stream);
    }
    FfnParams q{};
    q.m = a.rows;
    q.n = a.e;
    q.k = a.f;
    q.a[0] = operand(a.act, a.f, a.rows);
    q.b[0] = operand(a.w_down, a.w_down_stride, a.e);
    q.out[0] = static_cast<char *>(a.y);
    q.out_ld = (int64_t)a.e * 2;
    launch_product<DT, kKContig, kKContig, 1, kEpiStore, 0>(q, 1, stream);
}

template <class DT>
void backward(const dsalt_gated_ffn_args &a, hipStream_t stream) {
    const int64_t f2 = (int64_t)a.f * 2;  // bytes of [f], elements of gate | up
    if (a.dw_down) {
        FfnParams p{};
        p.m = a.e;
        p.n = a.f;
        p.k = a.rows;
        p.a[0] = operand(a.dy, a.dy_stride, a.e);
        p.b[0] = operand(a.act, a.f, a.f);
        p.out[0] = static_cast<char *>(a.dw_down);
        p.out_ld = f2;
        launch_product<DT, kRContig, kRContig, 1, kEpiStore, 0>(p, 1, stream);
    }
    if (a.d_gate_up) {
        FfnParams p{};
        p.m = a.rows;
        p.n = a.f;
        p.k = a.e;
        p.a[0] = operand(a.dy, a.dy_stride, a.rows);
        p.b[0] = operand(a.w_down, a.w_down_stride, a.f);
        p.out[0] = static_cast<char *>(a.d_gate_up);
        p.out_ld = p.gu_ld = f2 * 2;
        p.gu = static_cast<const char *>(a.gate_up);
        p.up_off = f2;
        launch_act<DT, kKContig, kRContig, 1, kEpiGrad>(p, a.activation, stream);
    }
    const GemmOperand dg = operand(a.d_gate_up, f2, 0), du = {dg.base + f2, dg.ld, 0};
    if (a.dx) {
        FfnParams p{};
        p.m = a.rows;
        p.n = a.d;
        p.k = a.f;
        p.a[0] = {dg.base, dg.ld, a.rows};
        p.a[1] = {du.base, du.ld, a.rows};
        p.b[0] = operand(a.w_gate, a.w_gate_stride, a.d);
        p.b[1] = operand(a.w_up, a.w_up_stride, a.d);
        p.out[0] = static_cast<char *>(a.dx);
        p.out_ld = (int64_t)a.d * 2;
        launch_product<DT, kKContig, kRContig, 2, kEpiStore, 0>(p, 1, stream);
    }
    if (a.dw_gate || a.dw_up) {
        FfnParams p{};
        p.m = a.f;
        p.n = a.d;
        p.k = a.rows;
        int batch = 0;
        if (a.dw_gate) {
            p.a[batch] = {dg.base, dg.ld, a.f};
            p.out[batch++] = static_cast<char *>(a.dw_gate);
        }
        if (a.dw_up) {
            p.a[batch] = {du.base, du.ld, a.f};
            p.out[batch++] = static_cast<char *>(a.dw_up);
        }
        p.b[0] = operand(a.x, a.x_stride, a.d);
        p.out_ld = (int64_t)a.d * 2;
        launch_product<DT, kRContig, kRContig, 1, kEpiStore, 0>(p, batch, stream);
    }
}

}  // namespace

hipError_t launch_gated_ffn(const dsalt_gated_ffn_args &a, hipStream_t stream) {
    if (a.rows == 0) return hipSuccess;
    if (a.dtype == DSALT_DTYPE_BF16) forward<BF16>(a, stream);
    else forward<F16>(a, stream);
    return hipGetLastError();
}

hipError_t launch_gated_ffn_bwd(const dsalt_gated_ffn_args &a, hipStream_t stream) {
    if (a.dtype == DSALT_DTYPE_BF16) backward<BF16>(a, stream);
    else backward<F16>(a, stream);
    return hipGetLastError();
}

int64_t gated_ffn_workspace_bytes(int64_t, int, int, int, bool) { return 0; }
int64_t gated_ffn_max_ld() { return kGemmMaxLd; }

}  // namespace dsalt
