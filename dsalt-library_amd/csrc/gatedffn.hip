// Gated feed-forward block, forward and backward:
//   g = x Wg^T, u = x Wu^T, a = act(g) * u, y = a Wd^T
//   da = dy Wd, dg = da * u * act'(g), du = da * act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T a
// Reference: SwiGLUFFN (dsalt/modules/dsalt_transformer.py:10-21) with torch's autograd.
//
// Gate and up projection, activation and product are one kernel: a workgroup's B tile holds
// the same columns of both weights, so that a lane ends with g and u of the same elements
// in its fp32 accumulators and rounds only a. Where a backward will read g and u they are
// kept in more bits than the element type's (see Kept). The backward's first kernel ends
// da = dy Wd in the gradients of g and u the same way: da is never written.
#include "gemm.h"
#include "launch.h"

#include <algorithm>
#include <type_traits>

namespace dsalt {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

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
        // The tail 0.5 erfc(|g| / sqrt 2) is exp(-g^2 / 2), which the slope takes too, times t P(t) with
        // t = 1 / (1 + 0.375 x), x = |g| / sqrt 2: as erfc(x) exp(x^2) falls like 1 / x, seven terms hold
        // its relative error below 2^-20 for every x of a normal result (fitted in float64, the largest
        // relative error least). The exponent's fp32 rounding adds 2^-16 of the tail at |g| = 13, 2^-19
        // below 4. Abramowitz and Stegun's 7.1.26, two terms less, holds the absolute error instead
        // and is 2 % off at -10; 8192 x 1024 x 2816 took 1 % less with it.
        const float x = 0.7071067811865476f * fabsf(g), t = __builtin_amdgcn_rcpf(1.f + 0.375f * x);
        const float ex = fast_exp2(-0.5f * kLog2e * g * g);
        const float tail = 0.5f * ex * t *
            (0.211339448f + t * (0.215689182f + t * (0.166664559f + t * (0.283061556f +
             t * (-0.129597319f + t * (0.387937839f + t * -0.135095904f))))));
        const float phi = g < 0.f ? tail : 1.f - tail;
        v = g * phi;
        slope = phi + g * 0.3989422804014327f * ex;
    } else {
        const bool off = g <= 0.f;  // NaN stays NaN
        v = off ? 0.f : g;
        slope = off ? 0.f : 1.f;
    }
}
// Eight at a time inside the choice of the activation, so that their chains of exp and
// reciprocal overlap.
template <int ACT>
__device__ __forceinline__ void gated8(const float (&g)[8], const float (&u)[8], float (&a)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float v, s;
        act_grad<ACT>(g[e], v, s);
        a[e] = v * u[e];
    }
}
__device__ __forceinline__ void gated8(int act, const float (&g)[8], const float (&u)[8], float (&a)[8]) {
    if (act == DSALT_ACT_SILU) gated8<DSALT_ACT_SILU>(g, u, a);
    else if (act == DSALT_ACT_GELU) gated8<DSALT_ACT_GELU>(g, u, a);
    else if (act == DSALT_ACT_GELU_TANH) gated8<DSALT_ACT_GELU_TANH>(g, u, a);
    else gated8<DSALT_ACT_RELU>(g, u, a);
}
// da becomes the gradient of g, u that of u.
template <int ACT>
__device__ __forceinline__ void gated_grad8(const float (&g)[8], float (&u)[8], float (&da)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float v, s;
        act_grad<ACT>(g[e], v, s);
        const float d = da[e];
        da[e] = d * u[e] * s;
        u[e] = d * v;
    }
}
__device__ __forceinline__ void gated_grad8(int act, const float (&g)[8], float (&u)[8], float (&da)[8]) {
    if (act == DSALT_ACT_SILU) gated_grad8<DSALT_ACT_SILU>(g, u, da);
    else if (act == DSALT_ACT_GELU) gated_grad8<DSALT_ACT_GELU>(g, u, da);
    else if (act == DSALT_ACT_GELU_TANH) gated_grad8<DSALT_ACT_GELU_TANH>(g, u, da);
    else gated_grad8<DSALT_ACT_RELU>(g, u, da);
}

// g and u kept for the backward. Their gradients are rounded to the element type once, as operands
// of the matrix units have to be, and so is every result; g and u rounded to it too would put
// a third rounding into dx and the weights' gradients (1.8 times the error of the last rounding
// alone, against 1.4 so; the extra byte costs under 1 % of a training pass of 16384 rows). So they
// keep the upper 20 bits of their fp32 value beside bf16 (four bits more than it has), and the upper
// 24 beside fp16 (five more): the upper 16 bits in a plane of gate | up rows, the rest in a plane
// behind it, a byte for both (low half g) or a byte each.
template <class DT>
struct Kept {
    static constexpr bool NIBBLE = std::is_same<DT, BF16>::value;
    static constexpr int LOW = NIBBLE ? 4 : 8;                // bits in the second plane
    static constexpr int LOW_BYTES = NIBBLE ? 1 : 2;          // of a (g, u) pair there
    static __device__ __forceinline__ uint32_t round(float x) {
        const uint32_t b = __float_as_uint(x), r = b + (1u << (15 - LOW));  // to nearest
        return (b & 0x7fffffffu) > 0x7f800000u ? b : r;                    // a NaN stays one
    }
    // eight columns: the planes' words
    static __device__ __forceinline__ void pack(const float (&v)[8], uint4 &high, uint32_t (&low)[2]) {
        uint32_t h[4];
        low[0] = low[1] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t x = round(v[2 * e]), y = round(v[2 * e + 1]);
            h[e] = (x >> 16) | (y & 0xffff0000u);
            low[e >> 1] |= (((x & 0xffffu) >> (16 - LOW)) | (((y & 0xffffu) >> (16 - LOW)) << 8)) << (16 * (e & 1));
        }
        high = make_uint4(h[0], h[1], h[2], h[3]);
    }
    static __device__ __forceinline__ void store(const float (&g)[8], const float (&u)[8], char *high, char *low, int64_t up_off) {
        uint4 gh, uh;
        uint32_t gl[2], ul[2];
        pack(g, gh, gl);
        pack(u, uh, ul);
        *reinterpret_cast<uint4 *>(high) = gh;
        *reinterpret_cast<uint4 *>(high + up_off) = uh;
        if constexpr (NIBBLE) {
            *reinterpret_cast<uint2 *>(low) = make_uint2(gl[0] | (ul[0] << 4), gl[1] | (ul[1] << 4));
        } else {
            *reinterpret_cast<uint2 *>(low) = make_uint2(gl[0], gl[1]);
            *reinterpret_cast<uint2 *>(low + up_off / 2) = make_uint2(ul[0], ul[1]);
        }
    }
    // low: the bytes of one matrix, shift: where its nibble is in them
    static __device__ __forceinline__ void unpack(uint4 high, uint2 low, int shift, float (&v)[8]) {
        const uint32_t h[4] = {high.x, high.y, high.z, high.w}, l[2] = {low.x >> shift, low.y >> shift};
        constexpr uint32_t MASK = (1u << LOW) - 1;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t top = e & 1 ? h[e >> 1] & 0xffff0000u : h[e >> 1] << 16;
            v[e] = __uint_as_float(top | (((l[e >> 2] >> (8 * (e & 3))) & MASK) << (16 - LOW)));
        }
    }
};

// One product of a launch: out [m, n] = sum over the segments of a[s] b[s] (pair: n columns of
// each of b[0] and b[1]).
struct Product {
    GemmOperand a[2], b[2];
    int64_t m, n;
    int tiles_m, tiles_n;
    char *out;
    int64_t out_ld;  // bytes
};

constexpr int kMaxProducts = 3;
struct FfnParams {
    Product prod[kMaxProducts];
    int products;
    int64_t k;        // of every product and segment
    int act;
    char *gu, *low;   // the planes of gate | up (Kept): written (pair; gu NULL: not kept) or read (gradient)
    int64_t gu_ld, up_off, low_ld;  // bytes; up at gu + up_off and, with a byte of its own, low + up_off / 2
    int whole;        // tiles computed by one workgroup each; the others by `split` workgroups,
    int split;        // whose fp32 partial sums go to `part` and are joined by a second launch
    float *part;
};

// A launch's tiles in order: product by product, in each kGroup m-tiles before the next n-tile,
// so that the workgroups that run at a time on one XCD share operand rows in its L2.
constexpr int kGroup = 8;
__device__ __forceinline__ const Product &tile_of(const FfnParams &p, int tile, int &tm, int &tn) {
    int z = 0;
    while (z + 1 < p.products && tile >= p.prod[z].tiles_m * p.prod[z].tiles_n) {
        tile -= p.prod[z].tiles_m * p.prod[z].tiles_n;
        ++z;
    }
    const Product &q = p.prod[z];
    const int per = kGroup * q.tiles_n, g = tile / per, r = tile - g * per, rows = min(kGroup, q.tiles_m - g * kGroup);
    tn = r / rows;
    tm = g * kGroup + r - tn * rows;
    return q;
}

enum { kEpiPair, kEpiStore, kEpiGrad };

// g and u of a tile's elements, in the epilogue's pieces, loaded kAhead turns before they are used:
// one after the other they would cost a trip to memory for every 16 bytes of a lane. (All of
// them loaded as the product starts, where the registers hold them, measured no faster.)
// Bounds by descriptor: the largest size's da took 528 us with addresses and bounds per lane, 497 so
// (both with g and u of 16 bits, on the core's earlier matrix instructions).
constexpr int kAhead = 3;
template <class DT, class Core>
struct GateUp {
    u32x4 g[kAhead], u[kAhead];
    u32x2 gl[kAhead], ul[kAhead];
    // piece t of the wave's row block `block`
    __device__ __forceinline__ void load(const FfnParams &p, const Product &q, const Core &c, int block, int t, int64_t m0,
                                         int64_t n0) {
        const int64_t mb = m0 + (c.wm * Core::FM + block) * 32, nb = n0 + c.wn * Core::COLS;
        const int64_t rows = min(q.m - mb, (int64_t)32), cols = q.n - nb;
        const bool some = rows > 0 && cols > 0, in = c.piece_col() < cols;
        const int at = t % kAhead;
        // past the last row, and past the row's end, nothing is read
        auto rsrc = [&](const char *plane, int64_t ld, int64_t off, int size) {
            return __builtin_amdgcn_make_buffer_rsrc((void *)(plane + mb * ld + nb * size + off), (short)0,
                                                     (int)(some ? (rows - 1) * ld + cols * size : 0), 0x00020000);
        };
        const int off = in ? (int)((uint32_t)c.piece_row(t) * (uint32_t)p.gu_ld) + c.piece_col() * 2 : (int)kOutOfRange;
        g[at] = __builtin_amdgcn_raw_buffer_load_b128(rsrc(p.gu, p.gu_ld, 0, 2), off, 0, 0);
        u[at] = __builtin_amdgcn_raw_buffer_load_b128(rsrc(p.gu, p.gu_ld, p.up_off, 2), off, 0, 0);
        const int low = in ? (int)((uint32_t)c.piece_row(t) * (uint32_t)p.low_ld) + c.piece_col() : (int)kOutOfRange;
        gl[at] = __builtin_amdgcn_raw_buffer_load_b64(rsrc(p.low, p.low_ld, 0, 1), low, 0, 0);
        if constexpr (!Kept<DT>::NIBBLE)
            ul[at] = __builtin_amdgcn_raw_buffer_load_b64(rsrc(p.low, p.low_ld, p.up_off / 2, 1), low, 0, 0);
    }
    __device__ __forceinline__ void get(int t, float (&gate)[8], float (&up)[8]) const {
        const int at = t % kAhead;
        Kept<DT>::unpack(bitcast<uint4>(g[at]), bitcast<uint2>(gl[at]), 0, gate);
        if constexpr (Kept<DT>::NIBBLE) Kept<DT>::unpack(bitcast<uint4>(u[at]), bitcast<uint2>(gl[at]), 4, up);
        else Kept<DT>::unpack(bitcast<uint4>(u[at]), bitcast<uint2>(ul[at]), 0, up);
    }
};

// The tile's row blocks first .. first + ROWS - 1 from their accumulators: the activation and
// product of a pair, a plain store, or the gradients of gate and up from that of the product.
template <class DT, class Core, int EPI, int ROWS>
__device__ __forceinline__ void epilogue(const FfnParams &p, const Product &q, const Core &c,
                                         const f32x4 (&acc)[ROWS][Core::FN][4], int first, int64_t m0, int64_t n0, char *lds) {
    constexpr int WIDTH = EPI == kEpiPair ? Core::COLS / 2 : Core::COLS;  // output columns of a wave
    const int64_t nb = n0 + c.wn * WIDTH;
    const bool inside = nb + c.piece_col() < q.n;
    const uint32_t ld = (uint32_t)q.out_ld, gu_ld = (uint32_t)p.gu_ld, low_ld = (uint32_t)p.low_ld;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t mb = m0 + (c.wm * Core::FM + first + i) * 32;
        const int rows = (int)min(q.m - mb, (int64_t)32);
        // wave-uniform bases, 32-bit lane offsets
        char *out = q.out + mb * q.out_ld + nb * 2, *gu_out = p.gu + mb * p.gu_ld + nb * 2, *low_out = p.low + mb * p.low_ld + nb;
        const uint32_t off = (uint32_t)(c.lane / Core::PIECES) * ld + c.piece_col() * 2,
                       gu_off = (uint32_t)(c.lane / Core::PIECES) * gu_ld + c.piece_col() * 2,
                       low_off = (uint32_t)(c.lane / Core::PIECES) * low_ld + c.piece_col();
        GateUp<DT, Core> gu;
        if constexpr (EPI == kEpiGrad) {
#pragma unroll
            for (int t = 0; t < kAhead && t < Core::TURNS; ++t) gu.load(p, q, c, first + i, t, m0, n0);
        }
        c.put(lds, acc[i]);
#pragma unroll
        for (int t = 0; t < Core::TURNS; ++t) {
            float v[8], u[8], w[8];
            c.get(lds, t, 0, v);
            if constexpr (EPI == kEpiPair) c.get(lds, t, WIDTH, u);
            if (inside && c.piece_row(t) < rows) {
                char *o = out + (uint32_t)(t * Core::TURN_ROWS) * ld;
                if constexpr (EPI == kEpiPair) {
                    if (p.gu)
                        Kept<DT>::store(v, u, gu_out + (uint32_t)(t * Core::TURN_ROWS) * gu_ld + gu_off,
                                        low_out + (uint32_t)(t * Core::TURN_ROWS) * low_ld + low_off, p.up_off);
                    gated8(p.act, v, u, w);
                    *reinterpret_cast<uint4 *>(o + off) = pack8<DT>(w);
                } else if constexpr (EPI == kEpiStore) {
                    *reinterpret_cast<uint4 *>(o + off) = pack8<DT>(v);
                } else {
                    gu.get(t, w, u);
                    gated_grad8(p.act, w, u, v);
                    *reinterpret_cast<uint4 *>(o + off) = pack8<DT>(v);
                    *reinterpret_cast<uint4 *>(o + p.up_off + off) = pack8<DT>(u);
                }
            }
            if constexpr (EPI == kEpiGrad)
                if (t + kAhead < Core::TURNS) gu.load(p, q, c, first + i, t + kAhead, m0, n0);
            __builtin_amdgcn_sched_barrier(0);  // no more turns in registers at a time than these
        }
        __builtin_amdgcn_wave_barrier();  // the next block overwrites this one
    }
}

template <int BM_, int BN_, int RA_, int RB_, int WM_, int WN_>
struct Shape {
    static constexpr int BM = BM_, BN = BN_, RA = RA_, RB = RB_, WM = WM_, WN = WN_;
};
template <class DT, class S, int ALAY, int BLAY, int EPI>
using Core = GemmCore<DT, S::BM, S::BN, 64, S::RA, S::RB, S::WM, S::WN, ALAY, BLAY, EPI == kEpiPair>;

// Partial sums of piece `piece` of split tile r: [piece][r][i][j][quarter][thread] float4.
template <class C>
__device__ __forceinline__ float4 *partial(const FfnParams &p, int r, int piece, int tiles, int i, int j, int thread) {
    return reinterpret_cast<float4 *>(p.part) +
           ((((int64_t)piece * tiles + r) * C::FM + i) * C::FN + j) * 4 * C::THREADS + thread;
}

template <class DT, class S, int ALAY, int BLAY, int SEGMENTS, int EPI>
__global__ void __launch_bounds__(S::WM *S::WN * 64) ffn_kernel(const FfnParams p) {
    typedef Core<DT, S, ALAY, BLAY, EPI> C;
    __shared__ __attribute__((aligned(256))) char lds[C::LDS_BYTES];
    constexpr int BNO = EPI == kEpiPair ? S::BN / 2 : S::BN;  // columns of the output
    // the whole tiles come first; each XCD takes a contiguous range of them
    int id = blockIdx.x, r = 0, piece = 0;
    const int steps = SEGMENTS * (int)((p.k + C::BK - 1) / C::BK);
    int first = 0, last = steps;
    if (id < (p.whole & ~7)) id = xcd_remap(id, p.whole & ~7);
    const bool split = id >= p.whole && p.split > 1;
    if (split) {
        r = (id - p.whole) / p.split;
        piece = (id - p.whole) - r * p.split;
        id = p.whole + r;
        first = (int)((int64_t)steps * piece / p.split);
        last = (int)((int64_t)steps * (piece + 1) / p.split);
    }
    int tm, tn;
    const Product &q = tile_of(p, id, tm, tn);
    const int64_t m0 = (int64_t)tm * S::BM, n0 = (int64_t)tn * BNO;
    C c;
    c.template run<SEGMENTS>(lds, q.a, q.b, m0, n0, p.k, first, last);
    if (split) {
        const int tiles = (gridDim.x - p.whole) / p.split;
#pragma unroll
        for (int i = 0; i < C::FM; ++i)
#pragma unroll
            for (int j = 0; j < C::FN; ++j)
#pragma unroll
                for (int h = 0; h < 4; ++h)
                    partial<C>(p, r, piece, tiles, i, j, threadIdx.x)[h * C::THREADS] = bitcast<float4>(c.acc[i][j][h]);
        return;
    }
    epilogue<DT, C, EPI, C::FM>(p, q, c, c.acc, 0, m0, n0, lds);
}

// The split tiles' partial sums added in order, and their epilogue: a workgroup of one wave for
// each row block of each of the tile's waves (a CU alone reads too slowly for more).
template <class DT, class S, int ALAY, int BLAY, int EPI>
__global__ void __launch_bounds__(64) ffn_join_kernel(const FfnParams p) {
    typedef Core<DT, S, ALAY, BLAY, EPI> C;
    constexpr int BNO = EPI == kEpiPair ? S::BN / 2 : S::BN;
    const int tiles = gridDim.x / (C::FM * C::NW), r = blockIdx.x / (C::FM * C::NW);
    const int i = blockIdx.x / C::NW % C::FM, wave = blockIdx.x % C::NW;
    int tm, tn;
    const Product &q = tile_of(p, p.whole + r, tm, tn);
    __shared__ __attribute__((aligned(256))) char lds[32 * C::COLS * 4];
    C c;  // the only wave of its workgroup, in the place of one of the tile's
    c.wm = wave % S::WM;
    c.wn = wave / S::WM;
    f32x4 acc[1][C::FN][4];
    const int64_t stride = (int64_t)tiles * C::FM * C::FN * 4 * C::THREADS;
    constexpr int kPieces = 8;  // partial sums in flight: one after the other each is a trip to memory
#pragma unroll
    for (int j = 0; j < C::FN; ++j) {
#pragma unroll
        for (int h = 0; h < 4; ++h) acc[0][j][h] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float4 *first = partial<C>(p, r, 0, tiles, i, j, wave * 64 + threadIdx.x);
        for (int s0 = 0; s0 < p.split; s0 += kPieces) {
            float4 v[kPieces][4];
#pragma unroll
            for (int s = 0; s < kPieces; ++s)
#pragma unroll
                for (int h = 0; h < 4; ++h)
                    v[s][h] = first[min(s0 + s, p.split - 1) * stride + h * C::THREADS];
#pragma unroll
            for (int s = 0; s < kPieces; ++s)
#pragma unroll
                for (int h = 0; s0 + s < p.split && h < 4; ++h) acc[0][j][h] += bitcast<f32x4>(v[s][h]);
        }
    }
    const int64_t m0 = (int64_t)tm * S::BM, n0 = (int64_t)tn * BNO;
    epilogue<DT, C, EPI, 1>(p, q, c, acc, i, m0, n0, lds);
}

// Few rows (up to 16 TT): bound by the weights' bytes, and by the latency of a call this short.
// A workgroup takes 16 weight rows (pair: the same 8 of both weights) and all rows of x; its waves
// take every NW-th 32 of k straight from memory into the operands of v_mfma_f32_16x16x32, so that
// nothing waits on LDS until their sums are added there, in order. Every workgroup reads all of x,
// so that its time grows with the rows while the tiles' stays; the two products took (bf16, us under
// the profiler, weights from memory; tiles with the join of their split)
//     d, f            1 row   16 rows   32 rows   tiles, 1 to 64 rows
//     1024, 2816       12.9      15.8      20.6   30.4 to 31.2
//     2048, 5504       21.2      27.8      39.1   38.7 to 40.3
//     4096, 11008      58.8      80.4     112.2   74.7 to 77.1
// The limit is that of the block's widths; at 4096 x 11008 tiles are ahead from 16 rows on.
// 1 row of 1024: 17.3 MB of weights, 1.4 TB/s; a launch of nothing takes 2 us of each 6, and the
// second product's 64 workgroups leave three quarters of the CUs without one.
constexpr int kFewRows = 32;
template <class DT, int TT, int NW, int EPI>
__global__ void __launch_bounds__(NW * 64) ffn_few_kernel(const FfnParams p) {
    constexpr bool PAIR = EPI == kEpiPair;
    // weight loads in flight a lane: gate and up of d 4096, f 11008 took 36.0 us with 8, 40.8 with 4 (5.0
    // TB/s); 32 rows' registers hold 4, and gained nothing from more
    constexpr int UNROLL = TT == 1 ? 8 : 4;
    __shared__ float4 part[NW][TT][64];
    const Product &q = p.prod[0];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l16 = lane & 15;
    const int n0 = blockIdx.x * (PAIR ? 8 : 16);
    // the lane's weight row: gate or up row n0 + l16 % 8 of a pair
    const GemmOperand &b = PAIR && l16 >= 8 ? q.b[1] : q.b[0];
    const int n = n0 + (PAIR ? l16 & 7 : l16), kl = (lane >> 4) * 8;
    const char *w = b.base + (int64_t)n * b.ld + kl * 2, *x[TT];
    bool xin[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        xin[t] = t * 16 + l16 < q.m;
        x[t] = q.a[0].base + (int64_t)(t * 16 + l16) * q.a[0].ld + kl * 2;
    }
    const bool win = n < q.n;
    const int k = (int)p.k;
    f32x4 acc[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = wave * 32; k0 < k; k0 += NW * 32 * UNROLL) {
        uint4 wv[UNROLL], xv[UNROLL][TT];
#pragma unroll
        for (int s = 0; s < UNROLL; ++s) {
            const int at = k0 + s * NW * 32;
            const bool in = at + kl < k;
            wv[s] = in && win ? *reinterpret_cast<const uint4 *>(w + at * 2) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int t = 0; t < TT; ++t)
                xv[s][t] = in && xin[t] ? *reinterpret_cast<const uint4 *>(x[t] + at * 2) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int s = 0; s < UNROLL; ++s)
#pragma unroll
            for (int t = 0; t < TT; ++t) acc[t] = mfma16<DT>(wv[s], xv[s][t], acc[t]);
    }
    // lane l holds rows 4 (l / 16) .. + 3 of the 16 weight rows for x row t * 16 + l % 16
#pragma unroll
    for (int t = 0; t < TT; ++t) part[wave][t][lane] = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
    __syncthreads();
    // a thread forms eight columns of one row: the gates and ups of a pair, or one half of 16
    const int id = threadIdx.x, half = PAIR ? 0 : id / (16 * TT), r = id % (16 * TT);
    if (id >= 16 * TT * (PAIR ? 1 : 2) || r >= q.m) return;
    auto sum = [&](int group, float (&v)[8]) {  // of weight rows 4 group .. + 7
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float4 s = part[0][r >> 4][(group + h) * 16 + (r & 15)];
            for (int wv = 1; wv < NW; ++wv) {
                const float4 o = part[wv][r >> 4][(group + h) * 16 + (r & 15)];
                s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w;
            }
            v[4 * h] = s.x; v[4 * h + 1] = s.y; v[4 * h + 2] = s.z; v[4 * h + 3] = s.w;
        }
    };
    float v[8], u[8], a[8];
    const int64_t col = n0 + half * 8;
    if (col >= q.n) return;
    sum(half * 2, v);
    char *o = q.out + (int64_t)r * q.out_ld + col * 2;
    if constexpr (PAIR) {
        sum(2, u);
        if (p.gu) Kept<DT>::store(v, u, p.gu + (int64_t)r * p.gu_ld + col * 2, p.low + (int64_t)r * p.low_ld + col, p.up_off);
        gated8(p.act, v, u, a);
        *reinterpret_cast<uint4 *>(o) = pack8<DT>(a);
    } else {
        *reinterpret_cast<uint4 *>(o) = pack8<DT>(v);
    }
}

template <class DT, int EPI>
hipError_t launch_few(const FfnParams &p, hipStream_t stream) {
    // the second product's k is the longer one, and its grid the smaller
    constexpr int NW = EPI == kEpiPair ? 8 : 16;
    const Product &q = p.prod[0];
    const dim3 grid((unsigned)((q.n + (EPI == kEpiPair ? 7 : 15)) / (EPI == kEpiPair ? 8 : 16))), block(NW * 64);
    if (q.m <= 16) hipLaunchKernelGGL((ffn_few_kernel<DT, 1, NW, EPI>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((ffn_few_kernel<DT, 2, NW, EPI>), grid, block, 0, stream, p);
    return hipGetLastError();
}

// How a launch covers its tiles: the shape, and into how many pieces the tiles past the last full
// round of workgroups are cut along k.
//
// The times are fits to measurements: us of one 64-wide k-step with all slots busy and with few
// (a CU alone has more of the caches, of the memory and of the power budget), and the share of
// the epilogue's bytes, at kMemory, that nothing else runs under (one of two workgroups on a CU
// computes while the other stores). With each shape forced (bf16, us under the profiler; largest is
// 16384 rows, d 2048, f 5504, ragged 6473, 1024, 2816, small 1500, 512, 1408; + the join):
//                     256 x 256   256 x 128   128 x 128    64 x 128
//   largest, gate|up        722         917         887         972
//   largest, down           325         388         369         470 + 7
//   largest, da             477         508         516         541
//   largest, dx             589         762         724         955 + 8
//   largest, weights        864 + 11   1064 + 8    1086 + 7    1758 + 9
//   ragged,  gate|up        104         109          89         103
//   ragged,  down            65          44          43          48 + 5
//   ragged,  da              68 + 15     80          68          67
//   ragged,  dx              76 + 14     95          91         102 + 6
//   ragged,  weights        139         118 + 6     106 + 6     144 + 8
//   small,   gate|up         24          16          16          14
//   small,   down            15 + 8      12 + 5      17          14
//   small,   da              32          20          17          13
//   small,   dx              21 + 9      18 + 5      14 + 5      14 + 5
//   small,   weights         20 + 9      27          21          19
// The constants below were fitted to such a table of earlier kernels, 8 % slower throughout, in which
// the same shapes led, row by row. A split costs a join of 5 to 6 us, less what it saves: dx of 575, 264, 712 took
// 17.2 us whole and 13.6 in pieces, of 3000, 768, 2048 50.4 and 37.5, down of 1500, 1024, 2816 27.9 and 24.6.
struct Plan {
    int shape, whole, split, tiles;
    int64_t part_bytes;
};
struct ShapeCost {
    int bm, bn, slots;  // workgroups that run at a time
    double busy, alone, bare, tile;  // tile: us of a tile besides its k-steps and bytes
};
constexpr ShapeCost kShapes[] = {
    {256, 256, 256, 1.80, 1.20, 1.0, 4.0},
    {256, 128, 256, 1.10, 0.80, 1.0, 3.0},
    {128, 128, 512, 1.12, 0.60, 0.65, 3.0},
    {64, 128, 768, 1.00, 0.50, 0.4, 3.0},
};
constexpr int kShapeCount = 4, kMaxSplit = 8;
constexpr int64_t kMaxTiles = 1 << 22;  // of one launch: with up to 512 threads each, half of what a grid may hold
constexpr double kJoin = 4.0, kMemory = 5.0e6, kPartials = 4.0e6;  // us, bytes per us twice

int64_t tiles_of(int64_t m, int64_t n, int shape, bool pair) {
    const int bn = kShapes[shape].bn / (pair ? 2 : 1);
    return ((m + kShapes[shape].bm - 1) / kShapes[shape].bm) * ((n + bn - 1) / bn);
}

struct Extent {
    int64_t m, n;
};
// io: bytes that an output element's epilogue moves.
Plan plan(const Extent *e, int count, int64_t k, int segments, bool pair, int io) {
    const int64_t steps = segments * ((k + 63) / 64);
    Plan best{};
    double least = 0;
    for (int s = 0; s < kShapeCount; ++s) {
        const ShapeCost &c = kShapes[s];
        int64_t tiles = 0;
        for (int z = 0; z < count; ++z) tiles += tiles_of(e[z].m, e[z].n, s, pair);
        if (tiles == 0) return best;
        if (tiles > kMaxTiles) continue;  // not of the largest tile: gated_ffn_fits()
        const double out = (double)c.bm * c.bn / (pair ? 2 : 1) * io * c.bare / kMemory;  // us per workgroup of a round
        const int64_t rounds = tiles / c.slots, rest = tiles - rounds * c.slots;
        const int most = rest ? (int)std::min<int64_t>(std::min<int64_t>(c.slots / rest, kMaxSplit), steps / 4) : 1;
        for (int split = 1; split <= std::max(most, 1); ++split) {
            double t = rounds * (steps * c.busy + c.tile + out * c.slots);
            const double busy = (double)rest * split / c.slots, bytes = split > 1 ? (double)rest * split * c.bm * c.bn * 4 : 0;
            if (rest) {
                t += (steps + split - 1) / split * (c.alone + (c.busy - c.alone) * busy) + c.tile;
                t += split > 1 ? kJoin + 2 * bytes / kPartials : out * rest;
            }
            if (best.tiles == 0 || t < least) {
                least = t;
                best = {s, (int)(split > 1 ? tiles - rest : tiles), split, (int)tiles, (int64_t)bytes};
            }
        }
    }
    return best;
}
// What each kind of launch moves per output element: see epilogue().
constexpr int kIoStore = 2, kIoGrad = 9;
int io_pair(bool keep) { return keep ? 7 : 2; }

template <class DT, class S, int ALAY, int BLAY, int SEGMENTS, int EPI>
hipError_t launch_shape(const FfnParams &p, const Plan &w, hipStream_t stream) {
    typedef Core<DT, S, ALAY, BLAY, EPI> C;
    const int rest = w.tiles - w.whole;
    hipLaunchKernelGGL((ffn_kernel<DT, S, ALAY, BLAY, SEGMENTS, EPI>), dim3(w.whole + rest * w.split), dim3(C::THREADS), 0,
                       stream, p);
    if (rest)
        hipLaunchKernelGGL((ffn_join_kernel<DT, S, ALAY, BLAY, EPI>), dim3(rest * C::FM * C::NW), dim3(64), 0, stream,
                           p);
    return hipGetLastError();
}

template <class DT, int ALAY, int BLAY, int SEGMENTS, int EPI>
hipError_t launch_product(FfnParams p, void *workspace, hipStream_t stream) {
    constexpr bool PAIR = EPI == kEpiPair;
    Extent e[kMaxProducts];
    for (int z = 0; z < p.products; ++z) e[z] = {p.prod[z].m, p.prod[z].n};
    const int io = EPI == kEpiPair ? io_pair(p.gu != nullptr) : EPI == kEpiGrad ? kIoGrad : kIoStore;
    const Plan w = plan(e, p.products, p.k, SEGMENTS, PAIR, io);
    if (w.tiles == 0) return hipSuccess;
    for (int z = 0; z < p.products; ++z) {
        const int bm = kShapes[w.shape].bm, bn = kShapes[w.shape].bn / (PAIR ? 2 : 1);
        p.prod[z].tiles_m = (int)((e[z].m + bm - 1) / bm);
        p.prod[z].tiles_n = (int)((e[z].n + bn - 1) / bn);
    }
    p.whole = w.whole;
    p.split = w.split;
    p.part = static_cast<float *>(workspace);
    switch (w.shape) {
        case 0: return launch_shape<DT, Shape<256, 256, 3, 2, 4, 2>, ALAY, BLAY, SEGMENTS, EPI>(p, w, stream);
        case 1: return launch_shape<DT, Shape<256, 128, 3, 3, 4, 2>, ALAY, BLAY, SEGMENTS, EPI>(p, w, stream);
        case 2: return launch_shape<DT, Shape<128, 128, 2, 2, 2, 2>, ALAY, BLAY, SEGMENTS, EPI>(p, w, stream);
        default: return launch_shape<DT, Shape<64, 128, 2, 2, 2, 2>, ALAY, BLAY, SEGMENTS, EPI>(p, w, stream);
    }
}

// The planes of the kept gate | up of `rows` rows.
template <class DT>
void set_kept(FfnParams &p, void *gate_up, int64_t rows, int64_t f) {
    p.gu = static_cast<char *>(gate_up);
    p.gu_ld = f * 4;
    p.up_off = f * 2;
    p.low = p.gu + rows * p.gu_ld;
    p.low_ld = f * Kept<DT>::LOW_BYTES;
}

GemmOperand operand(const void *p, int64_t ld, int64_t rows) { return {static_cast<const char *>(p), ld * 2, rows}; }

Product product(GemmOperand a, GemmOperand b, int64_t m, int64_t n, void *out, int64_t out_ld) {
    Product q{};
    q.a[0] = a;
    q.b[0] = b;
    q.m = m;
    q.n = n;
    q.out = static_cast<char *>(out);
    q.out_ld = out_ld * 2;
    return q;
}

template <class DT>
hipError_t forward(const dsalt_gated_ffn_args &a, hipStream_t stream) {
    FfnParams p{};
    p.products = 1;
    p.k = a.d;
    p.act = a.activation;
    p.prod[0] = product(operand(a.x, a.x_stride, a.rows), operand(a.w_gate, a.w_gate_stride, a.f), a.rows, a.f, a.act, a.f);
    p.prod[0].b[1] = operand(a.w_up, a.w_up_stride, a.f);
    if (a.gate_up) set_kept<DT>(p, a.gate_up, a.rows, a.f);
    const bool few = a.rows <= kFewRows;
    hipError_t e = few ? launch_few<DT, kEpiPair>(p, stream)
                       : launch_product<DT, kKContig, kKContig, 1, kEpiPair>(p, a.workspace, stream);
    if (e != hipSuccess) return e;
    FfnParams q{};
    q.products = 1;
    q.k = a.f;
    q.prod[0] = product(operand(a.act, a.f, a.rows), operand(a.w_down, a.w_down_stride, a.e), a.rows, a.e, a.y, a.e);
    return few ? launch_few<DT, kEpiStore>(q, stream)
               : launch_product<DT, kKContig, kKContig, 1, kEpiStore>(q, a.workspace, stream);
}

template <class DT>
hipError_t backward(const dsalt_gated_ffn_args &a, hipStream_t stream) {
    const int64_t up = (int64_t)a.f * 2;  // bytes from gate to up in a row of gate | up
    const char *dgu = static_cast<const char *>(a.d_gate_up);
    if (a.d_gate_up) {
        FfnParams p{};
        p.products = 1;
        p.k = a.e;
        p.act = a.activation;
        p.prod[0] = product(operand(a.dy, a.dy_stride, a.rows), operand(a.w_down, a.w_down_stride, a.f), a.rows, a.f,
                            a.d_gate_up, 2 * (int64_t)a.f);
        set_kept<DT>(p, a.gate_up, a.rows, a.f);
        hipError_t e = launch_product<DT, kKContig, kRContig, 1, kEpiGrad>(p, a.workspace, stream);
        if (e != hipSuccess) return e;
    }
    if (a.dx) {
        FfnParams p{};
        p.products = 1;
        p.k = a.f;
        p.prod[0] = product(operand(dgu, 2 * (int64_t)a.f, a.rows), operand(a.w_gate, a.w_gate_stride, a.d), a.rows, a.d, a.dx, a.d);
        p.prod[0].a[1] = operand(dgu + up, 2 * (int64_t)a.f, a.rows);
        p.prod[0].b[1] = operand(a.w_up, a.w_up_stride, a.d);
        hipError_t e = launch_product<DT, kKContig, kRContig, 2, kEpiStore>(p, a.workspace, stream);
        if (e != hipSuccess) return e;
    }
    // the weights' gradients share their k axis, the rows: one launch
    FfnParams p{};
    p.k = a.rows;
    const GemmOperand x = operand(a.x, a.x_stride, a.d);
    if (a.dw_gate) p.prod[p.products++] = product(operand(dgu, 2 * (int64_t)a.f, a.f), x, a.f, a.d, a.dw_gate, a.d);
    if (a.dw_up) p.prod[p.products++] = product(operand(dgu + up, 2 * (int64_t)a.f, a.f), x, a.f, a.d, a.dw_up, a.d);
    if (a.dw_down)
        p.prod[p.products++] = product(operand(a.dy, a.dy_stride, a.e), operand(a.act, a.f, a.f), a.e, a.f, a.dw_down, a.f);
    return launch_product<DT, kRContig, kRContig, 1, kEpiStore>(p, a.workspace, stream);
}

}  // namespace

hipError_t launch_gated_ffn(const dsalt_gated_ffn_args &a, hipStream_t stream) {
    if (a.rows == 0) return hipSuccess;
    return a.dtype == DSALT_DTYPE_BF16 ? forward<BF16>(a, stream) : forward<F16>(a, stream);
}

hipError_t launch_gated_ffn_bwd(const dsalt_gated_ffn_args &a, hipStream_t stream) {
    return a.dtype == DSALT_DTYPE_BF16 ? backward<BF16>(a, stream) : backward<F16>(a, stream);
}

int64_t gated_ffn_workspace_bytes(int64_t rows, int d, int f, int e, bool bwd) {
    if (!bwd) {
        if (rows <= kFewRows) return 0;
        const Extent up{rows, f}, down{rows, e};
        int64_t most = plan(&down, 1, f, 1, false, kIoStore).part_bytes;
        for (bool keep : {false, true}) most = std::max(most, plan(&up, 1, d, 1, true, io_pair(keep)).part_bytes);
        return most;
    }
    const Extent da{rows, f}, dx{rows, d}, dw[3] = {{f, d}, {f, d}, {e, f}}, two[2] = {dw[0], dw[2]};
    int64_t most = std::max(plan(&da, 1, e, 1, false, kIoGrad).part_bytes, plan(&dx, 1, f, 2, false, kIoStore).part_bytes);
    // any of the three weight gradients may be wanted
    most = std::max(most, plan(two, 2, rows, 1, false, kIoStore).part_bytes);
    for (int first = 0; first < 3; ++first)
        for (int count = 1; first + count <= 3; ++count)
            most = std::max(most, plan(dw + first, count, rows, 1, false, kIoStore).part_bytes);
    return most;
}

bool gated_ffn_fits(int64_t rows, int d, int f, int e, bool bwd) {
    const auto tiles = [](int64_t m, int64_t n, bool pair) { return tiles_of(m, n, 0, pair); };
    if (!bwd) return tiles(rows, f, true) <= kMaxTiles && tiles(rows, e, false) <= kMaxTiles;
    return tiles(rows, f, false) <= kMaxTiles && tiles(rows, d, false) <= kMaxTiles &&
           2 * tiles(f, d, false) + tiles(e, f, false) <= kMaxTiles;
}

int64_t gated_ffn_kept_bytes(int64_t rows, int f, int dtype) {
    return rows * f * (4 + (dtype == DSALT_DTYPE_BF16 ? Kept<BF16>::LOW_BYTES : Kept<F16>::LOW_BYTES));
}
int64_t gated_ffn_max_ld() { return kGemmMaxLd; }

}  // namespace dsalt
