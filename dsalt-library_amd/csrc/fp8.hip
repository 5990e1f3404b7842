// Products of 8-bit floats (e4m3) with a scale for each block of 128, and the quantisation that makes
// their operands:
//   C[m, n] = sum over blocks b of k:  sa[m, b] sb[n / 128, b] sum_{k in b} A[m, k] B[n, k]  (+ bias[n])
// A [M, K] holds activations with a scale for 128 elements of a row, B [N, K] weights with one for a tile
// of 128 x 128. Products and sums are fp32; C is rounded once.
//
// Quantisation gives a block the smallest power of two that brings its largest magnitude to at most 448,
// e4m3's largest: the division is exact then, an element is rounded once, and what a scale of amax / 448
// would add to the range (less than a factor of two) an element's relative precision does not show.
#include "launch.h"
#include "fp8.h"
#include "rows.h"

#include <algorithm>

namespace dsalt {
namespace {

// ---- quantisation ---------------------------------------------------------------------------
struct QuantParams {
    const void *x;
    int64_t x_stride, rows;
    int k, blocks;
    uint8_t *q;  // [rows, k]
    void *scale;
    int64_t scale_stride;  // elements of a row of scales
    int scale_f32;
    int vec;  // rows of x can be read 16 bytes at a time
};

// Eight consecutive elements from column c of a row (zeros past k) as fp32.
template <typename DT>
__device__ __forceinline__ void load8(const QuantParams &p, int64_t row, int c, float (&v)[8]) {
    constexpr int SZ = std::is_same<DT, F32>::value ? 4 : 2;
    const char *at = static_cast<const char *>(p.x) + (row * p.x_stride + c) * SZ;
    if (p.vec && c + 8 <= p.k) {
        Elem<DT>::template ldv<8>(at, 0, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < p.k ? Elem<DT>::ld(at, e) : 0.f;
    }
}
__device__ __forceinline__ uint32_t amax8(const float (&v)[8]) {
    uint32_t m = 0;  // of magnitudes' bits: NaN and infinities are the largest
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
    return m;
}
__device__ __forceinline__ uint32_t row16_max(uint32_t m) {
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, false));
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, false));
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xF, 0xF, false));
    return max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x140, 0xF, 0xF, false));
}
__device__ __forceinline__ uint2 quantised(const float (&v)[8], uint32_t e8) {
    const float s = inverse_scale(e8);
    return make_uint2(pack_e4m3(v[0] * s, v[1] * s, v[2] * s, v[3] * s), pack_e4m3(v[4] * s, v[5] * s, v[6] * s, v[7] * s));
}
__device__ __forceinline__ void store_q(const QuantParams &p, int64_t row, int c, uint2 v) {
    uint8_t *at = p.q + row * p.k + c;
    if (c + 8 <= p.k && p.k % 8 == 0) {
        *reinterpret_cast<uint2 *>(at) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < p.k) at[e] = (uint8_t)((e < 4 ? v.x : v.y) >> (8 * (e & 3)));
    }
}
__device__ __forceinline__ void store_scale(const QuantParams &p, int64_t row, int block, uint32_t e8) {
    const int64_t at = row * p.scale_stride + block;
    if (p.scale_f32) static_cast<float *>(p.scale)[at] = e8m0_f32(e8);
    else static_cast<uint8_t *>(p.scale)[at] = (uint8_t)e8;
}

// Sixteen lanes a block of 128 of a row.
template <typename DT>
__global__ void __launch_bounds__(256) quant_rows_kernel(const QuantParams p) {
    const int64_t items = p.rows * p.blocks;
    const int l = threadIdx.x & 15;
    for (int64_t item = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); item < items; item += (int64_t)gridDim.x * 16) {
        const int64_t row = item / p.blocks;
        const int block = (int)(item - row * p.blocks), c = block * kFp8Block + l * 8;
        float v[8];
        load8<DT>(p, row, c, v);
        const uint32_t e8 = e8m0_of_amax(row16_max(amax8(v)));
        if (c < p.k) store_q(p, row, c, quantised(v, e8));
        if (l == 0) store_scale(p, row, block, e8);
    }
}

// A workgroup a tile of 128 x 128.
template <typename DT>
__global__ void __launch_bounds__(256) quant_tile_kernel(const QuantParams p) {
    __shared__ uint32_t lds[16];
    const int block = blockIdx.x % p.blocks, l = threadIdx.x & 15, c = block * kFp8Block + l * 8;
    const int64_t r0 = (int64_t)(blockIdx.x / p.blocks) * kFp8Block;
    float v[8][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = r0 + i * 16 + (threadIdx.x >> 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
        if (row < p.rows) load8<DT>(p, row, c, v[i]);
        m = max(m, amax8(v[i]));
    }
    m = row16_max(m);
    if (l == 0) lds[threadIdx.x >> 4] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, lds[i]);
    const uint32_t e8 = e8m0_of_amax(m);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = r0 + i * 16 + (threadIdx.x >> 4);
        if (row < p.rows && c < p.k) store_q(p, row, c, quantised(v[i], e8));
    }
    if (threadIdx.x == 0) store_scale(p, blockIdx.x / p.blocks, block, e8);
}

// ---- products -------------------------------------------------------------------------------
struct Fp8Params {
    GemmOperand a, b;  // ld in bytes
    Fp8Scales sa, sb;
    int64_t m, n, k;
    int kb;  // blocks of k
    const void *bias;
    int bias_dtype;
    void *out;
    int out_dtype;
    float *part;  // [splits][m][n], where k is split
    int splits;
    int tiles_m, tiles_n;
    int a_dtype;  // few rows: of x, which is quantised on the way
};

__device__ __forceinline__ float load_dt(const void *p, int64_t i, int dtype) {
    return dtype == DSALT_DTYPE_F32 ? Elem<F32>::ld(p, i) : dtype == DSALT_DTYPE_BF16 ? Elem<BF16>::ld(p, i) : Elem<F16>::ld(p, i);
}
__device__ __forceinline__ void store_dt(void *p, int64_t i, int dtype, float v) {
    if (dtype == DSALT_DTYPE_F32) Elem<F32>::st(p, i, v);
    else if (dtype == DSALT_DTYPE_BF16) Elem<BF16>::st(p, i, v);
    else Elem<F16>::st(p, i, v);
}
// N (4 or 8) results of columns col .. of a row, with the bias; whole: all lie inside and vectors may be written.
template <int N>
__device__ __forceinline__ void store_out(const Fp8Params &p, int64_t row, int64_t col, float (&v)[N]) {
    const int64_t at = row * p.n + col;
    if (p.bias)
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (col + e < p.n) v[e] += load_dt(p.bias, col + e, p.bias_dtype);
    if (p.n % N == 0) {  // rows start on the vectors' boundaries; col < n then means col + N <= n
        if (p.out_dtype == DSALT_DTYPE_F32) {
#pragma unroll
            for (int e = 0; e < N; e += 4)
                reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at)[e / 4] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        } else {
            uint32_t w[N / 2];
#pragma unroll
            for (int e = 0; e < N; e += 2)
                w[e / 2] = p.out_dtype == DSALT_DTYPE_BF16 ? BF16::pack2(v[e], v[e + 1]) : F16::pack2(v[e], v[e + 1]);
            uint16_t *o = static_cast<uint16_t *>(p.out) + at;
            if constexpr (N == 8) *reinterpret_cast<uint4 *>(o) = make_uint4(w[0], w[1], w[2], w[3]);
            else *reinterpret_cast<uint2 *>(o) = make_uint2(w[0], w[1]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (col + e < p.n) store_dt(p.out, at + e, p.out_dtype, v[e]);
    }
}

// A workgroup's tile: WM x WN waves over BM x BN, two stages of one block of k in LDS. MX: both scales
// are e8m0 and the matrix instruction applies them; otherwise both are fp32, and a block's product is formed
// from zero and added to the sums times the product of the scales, four multiply-adds an instruction.
//
// A wave holds one set of B's operands and a ring of four of A's, each read two groups of products (a
// group: one of A's with all of B's) before its own. The barrier that frees a stage stands before the last
// two groups of a step: what they need is in registers by then and the next stage has landed. Under them
// the next step's first two of A's are read, and each of B's as soon as its last product has been issued: it
// is needed a group later.
template <bool MX, int BM, int BN, int WM, int WN>
struct Fp8Core {
    static constexpr int NW = WM * WN, THREADS = NW * 64, M16 = BM / WM / 16, N16 = BN / WN / 16;
    typedef GemmTile<kKContig, BM, 64, NW> TA;  // 64 pairs of bytes: a block
    typedef GemmTile<kKContig, BN, 64, NW> TB;
    static constexpr int LA = TA::LPW, LB = TB::LPW, LT = LA + LB + 1;
    // a stage: A's tile, B's tile, and 64 scales a wave: A's rows, then B's blocks
    static constexpr int ASTAGE = BM * 128, BSTAGE = BN * 128, SSTAGE = NW * 256, STAGE = ASTAGE + BSTAGE + SSTAGE;
    static constexpr int LDS_BYTES = 2 * STAGE;
    static_assert(BM % 64 == 0 && BM / 64 < NW && BN / WN <= kFp8Block, "a wave for B's scales beside A's");
    static_assert(M16 % 4 == 0 && N16 % 2 == 0, "the ring of A's operands, and the pairs of the epilogue");

    f32x4 acc[M16][N16];
    int lane, wave, wm, wn;

    __device__ __forceinline__ Fp8Core() {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        wm = wave % WM;
        wn = wave / WM;
    }

    __device__ __forceinline__ void run(char *lds, const Fp8Params &p, int64_t m0, int64_t n0, int first, int last) {
        const uint32_t base = lds_addr(lds);
        const int64_t k2 = p.k / 2;
        const TA ta(wave, lane, (uint32_t)p.a.ld);
        const TB tb(wave, lane, (uint32_t)p.b.ld);
        const GemmFrag<kKContig, BM, 64> fa(lane);
        const GemmFrag<kKContig, BN, 64> fb(lane);
        // the wave's 64 scales of a step
        const bool is_a = wave < BM / 64;
        const Fp8Scales &sc = is_a ? p.sa : p.sb;
        const int64_t srow = is_a ? m0 + wave * 64 : n0 / kFp8Block;
        const int64_t sleft = wave > BM / 64 ? 0 : sc.rows - srow;
        constexpr uint32_t ssize = MX ? 1 : 4;
        const int slots = is_a ? 64 : (BN + kFp8Block - 1) / kFp8Block;
        const uint32_t soff = lane < sleft && lane < slots ? (uint32_t)(lane * sc.row_stride) * ssize : kOutOfRange;
        typename TA::Step da;
        typename TB::Step db;
        i32x4 ds;
        // past `last` the loads read nothing, so that every step counts the same number of loads
        auto prepare = [&](int step) {
            const bool on = step < last;
            da = ta.step(p.a, m0, on ? (int64_t)step * 64 : k2, k2);
            db = tb.step(p.b, n0, on ? (int64_t)step * 64 : k2, k2);
            const char *q = sc.base + (srow * sc.row_stride + (on ? step : 0) * sc.k_stride) * ssize;
            ds = uniform_rsrc(buffer_rsrc(q, on && sleft > 0 ? kOutOfRange - 1 : 0));
        };
        auto issue = [&](int stage, int u) {
            const uint32_t at = base + stage * STAGE;
            if (u < LA) TA::issue(da, u, at, wave);
            else if (u < LA + LB) TB::issue(db, u - LA, at + ASTAGE, wave);
            else {
                const uint32_t to = __builtin_amdgcn_readfirstlane(at + ASTAGE + BSTAGE + wave * 256);
                if constexpr (MX) dma1(soff, ds, to);
                else dma4(soff, ds, to);
            }
        };
#pragma unroll
        for (int i = 0; i < M16; ++i)
#pragma unroll
            for (int j = 0; j < N16; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (first >= last) return;
        Fp8Frag ra[4], rb[N16];
        uint32_t sa[4], sb, sb_next;
        auto read_a = [&](const char *at, int i) {
            ra[i % 4] = fp8_frag(fa.read(at, wm * M16 + i, 0), fa.read(at, wm * M16 + i, 1));
            sa[i % 4] = reinterpret_cast<const uint32_t *>(at + ASTAGE + BSTAGE)[(wm * M16 + i) * 16 + (lane & 15)];
        };
        auto read_b = [&](const char *at, int j) {
            rb[j] = fp8_frag(fb.read(at + ASTAGE, wn * N16 + j, 0), fb.read(at + ASTAGE, wn * N16 + j, 1));
        };
        auto read_sb = [&](const char *at) {
            return reinterpret_cast<const uint32_t *>(at + ASTAGE + BSTAGE)[BM + wn * (N16 * 16) / kFp8Block];
        };
        prepare(first);
#pragma unroll
        for (int u = 0; u < LT; ++u) issue(0, u);
        prepare(first + 1);
#pragma unroll
        for (int u = 0; u < LT; ++u) issue(1, u);
        tile_barrier<LT>();
        // in the loop's order: its first waits then count the same reads behind theirs on every step
        sb = read_sb(lds);
        read_a(lds, 0);
        __builtin_amdgcn_sched_barrier(0);
        read_a(lds, 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < N16; ++j) {
            read_b(lds, j);
            __builtin_amdgcn_sched_barrier(0);
        }
        int stage = 0;
        for (int t = first; t < last; ++t) {
            const char *at = lds + stage * STAGE, *next = lds + (stage ^ 1) * STAGE;
            float sbf = 0.f;
            if constexpr (!MX) sbf = __uint_as_float(sb);
#pragma unroll
            for (int i = 0; i < M16; ++i) {
                if (i == M16 - 2) {
                    prepare(t + 2);
                    __builtin_amdgcn_sched_barrier(0);
                    tile_barrier<0>();
                    sb_next = read_sb(next);
                }
                if (i < M16 - 2) read_a(at, i + 2);
                else read_a(next, i - M16 + 2);
                float s = 0.f;
                if constexpr (!MX) s = __uint_as_float(sa[i % 4]) * sbf;
#pragma unroll
                for (int j = 0; j < N16; ++j) {
                    if constexpr (MX) {
                        acc[i][j] = mfma_fp8(rb[j], ra[i % 4], acc[i][j], (int)sb, (int)sa[i % 4]);
                        // held here: a product has no side effect that would keep it from drifting behind the
                        // loads and the barrier, with copies of all that it needs
                        asm volatile("" : "+v"(acc[i][j]));
                    } else {
                        const f32x4 d = mfma_fp8(rb[j], ra[i % 4]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[e], s, acc[i][j][e]);
                    }
                    if (i == M16 - 1) {
                        __builtin_amdgcn_sched_barrier(0);  // not before the product that still needs the old one
                        read_b(next, j);
                    }
                    // the loads of step t + 2, spread over the groups behind the barrier
                    if (i >= M16 - 2) {
                        constexpr int NM = 2 * N16;
#pragma unroll
                        for (int u = 0; u < LT; ++u)
                            if (u * NM / LT == (i - M16 + 2) * N16 + j) issue(stage, u);
                    }
                }
                if constexpr (!MX)
#pragma unroll
                    for (int j = 0; j < N16; ++j)
                        if (i > 0) asm volatile("" : "+v"(acc[i - 1][j]));
                __builtin_amdgcn_sched_barrier(0);
            }
            sb = sb_next;
            stage ^= 1;
        }
        tile_barrier<0>();  // no load may land in LDS that another workgroup has by then
    }

    // Calls f(row, column, v) for eight consecutive columns of the tile a lane. The accumulators hold four
    // consecutive n of one m; of two neighbouring blocks of 16 columns a lane takes eight of one, in exchange
    // with the lanes 16 further on.
    template <class F>
    __device__ __forceinline__ void each_piece(F f) const {
        const int g = lane >> 4;
#pragma unroll
        for (int i = 0; i < M16; ++i)
#pragma unroll
            for (int j = 0; j < N16; j += 2) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // lane groups (0, 1, 2, 3) of the pair: (j, j + 1, j, j + 1) at columns (0, 0, 8, 8)
                    auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[i][j][e]), __float_as_uint(acc[i][j + 1][e]), false, false);
                    v[e] = __uint_as_float(x[0]);
                    v[4 + e] = __uint_as_float(x[1]);
                }
                f((wm * M16 + i) * 16 + (lane & 15), (wn * N16 + j + (g & 1)) * 16 + (g >> 1) * 8, v);
            }
    }
};

// Tile of a workgroup: consecutive ids of one XCD take groups of eight tile rows, so that the tiles that run
// beside each other share their operands' rows in that XCD's L2.
__device__ __forceinline__ bool fp8_tile(const Fp8Params &p, int &tm, int &tn, int &split) {
    const int per = p.tiles_m * p.tiles_n, id = xcd_remap(blockIdx.x, gridDim.x);
    if (id >= per * p.splits) return false;
    split = id / per;
    const int t = id - split * per;
    constexpr int G = 8;
    const int group = t / (G * p.tiles_n), in = t - group * G * p.tiles_n, rows = min(G, p.tiles_m - group * G);
    tm = group * G + in % rows;
    tn = in / rows;
    return true;
}

template <bool MX, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM *WN * 64) fp8_tile_kernel(const Fp8Params p) {
    typedef Fp8Core<MX, BM, BN, WM, WN> Core;
    extern __shared__ char lds[];
    int tm, tn, split;
    if (!fp8_tile(p, tm, tn, split)) return;
    Core core;
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int per = (p.kb + p.splits - 1) / p.splits, first = split * per;
    core.run(lds, p, m0, n0, first, min(first + per, p.kb));
    float *part = p.splits > 1 ? p.part + split * p.m * p.n : nullptr;
    core.each_piece([&](int r, int c, float (&v)[8]) {
        const int64_t row = m0 + r, col = n0 + c;
        if (row >= p.m || col >= p.n) return;
        if (!part) return store_out<8>(p, row, col, v);
        float *o = part + row * p.n + col;
        if (p.n % 4 == 0 && col + 8 <= p.n) {
            reinterpret_cast<float4 *>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4 *>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (col + e < p.n) o[e] = v[e];
        }
    });
}

// Sum of the splits' parts in their order.
__global__ void __launch_bounds__(256) fp8_join_kernel(const Fp8Params p) {
    const int64_t total = p.m * p.n, per = (p.n + 3) / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.m * per; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per, col = (i - row * per) * 4;
        const float *in = p.part + row * p.n + col;
        float v[4] = {};
        for (int s = 0; s < p.splits; ++s, in += total) {
            if (p.n % 4 == 0) {
                const float4 f = *reinterpret_cast<const float4 *>(in);
                v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (col + e < p.n) v[e] += in[e];
            }
        }
        store_out<4>(p, row, col, v);
    }
}

// Up to 16 MF rows against 16 rows of weights a wave: the weights come straight from memory, eight blocks of k
// in flight, and KW waves of the workgroup share out k and join their sums in LDS. TX: the rows are x's
// element type and each wave quantises what it reads of them; void: they are e4m3 with scales.
constexpr int kRowWaves = 8;
template <typename TX, int MF, int KW>
__global__ void __launch_bounds__(64 * kRowWaves) fp8_rows_kernel(const Fp8Params p) {
    constexpr bool QUANT = !std::is_void<TX>::value;
    constexpr int U = 4;
    __shared__ f32x4 lds[KW > 1 ? kRowWaves : 1][MF][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int kw = wave % KW, group = lane >> 4;
    const int64_t n0 = ((int64_t)blockIdx.x * (kRowWaves / KW) + wave / KW) * 16;
    const int64_t brow = n0 + (lane & 15);
    const bool b_in = brow < p.n;
    const char *bp = p.b.base + (b_in ? brow : 0) * p.b.ld;
    const int64_t nb = min(n0, p.n - 1) / kFp8Block;
    f32x4 acc[MF] = {};
    const int per = (p.kb + KW - 1) / KW, first = kw * per, last = n0 < p.n ? min(first + per, p.kb) : 0;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    // one block of k: the weights w against the rows
    const auto block = [&](int kb, Fp8Frag w) {
        const int64_t k0 = (int64_t)kb * kFp8Block + group * 16;
        const float sb = p.sb.at(nb, kb);
#pragma unroll
        for (int i = 0; i < MF; ++i) {
            const int64_t row = i * 16 + (lane & 15);
            const bool in = row < p.m;
            Fp8Frag fa = fp8_frag(zero, zero);
            float s = 0.f;
            if constexpr (QUANT) {
                const char *ap = p.a.base + (in ? row : 0) * p.a.ld;
                Raw8<TX> r0 = {}, r1 = {}, r2 = {}, r3 = {};
                if (in && k0 < p.k) {
                    r0.load(ap, k0 / 8);
                    r1.load(ap, k0 / 8 + 1);
                }
                if (in && k0 + 64 < p.k) {
                    r2.load(ap, k0 / 8 + 8);
                    r3.load(ap, k0 / 8 + 9);
                }
                float v0[8], v1[8], v2[8], v3[8];
                r0.get(v0);
                r1.get(v1);
                r2.get(v2);
                r3.get(v3);
                uint32_t m = max(max(amax8(v0), amax8(v1)), max(amax8(v2), amax8(v3)));
                m = max(m, (uint32_t)__shfl_xor((int)m, 16));
                m = max(m, (uint32_t)__shfl_xor((int)m, 32));
                const uint32_t e8 = e8m0_of_amax(m);
                const uint2 q0 = quantised(v0, e8), q1 = quantised(v1, e8), q2 = quantised(v2, e8), q3 = quantised(v3, e8);
                fa = fp8_frag(make_uint4(q0.x, q0.y, q1.x, q1.y), make_uint4(q2.x, q2.y, q3.x, q3.y));
                s = e8m0_f32(e8);
            } else if (in) {
                const char *ap = p.a.base + row * p.a.ld;
                uint4 lo = zero, hi = zero;
                if (k0 < p.k) lo = *reinterpret_cast<const uint4 *>(ap + k0);
                if (k0 + 64 < p.k) hi = *reinterpret_cast<const uint4 *>(ap + k0 + 64);
                fa = fp8_frag(lo, hi);
                s = p.sa.at(row, kb);
            }
            const f32x4 d = mfma_fp8(w, fa);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][e] = fmaf(d[e], s * sb, acc[i][e]);
        }
    };
    for (int t = first; t < last; t += U) {
        Fp8Frag fb[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k0 = (int64_t)(t + u) * kFp8Block + group * 16;
            uint4 lo = zero, hi = zero;
            if (t + u < last && b_in && k0 < p.k) lo = *reinterpret_cast<const uint4 *>(bp + k0);
            if (t + u < last && b_in && k0 + 64 < p.k) hi = *reinterpret_cast<const uint4 *>(bp + k0 + 64);
            fb[u] = fp8_frag(lo, hi);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (t + u < last) block(t + u, fb[u]);
        }
    }
    if constexpr (KW > 1) {
#pragma unroll
        for (int i = 0; i < MF; ++i) lds[wave][i][lane] = acc[i];
        __syncthreads();
        if (kw) return;
#pragma unroll
        for (int w = 1; w < KW; ++w)
#pragma unroll
            for (int i = 0; i < MF; ++i) {
                const f32x4 o = lds[wave + w][i][lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][e] += o[e];
            }
    }
    const int64_t col = n0 + group * 4;
#pragma unroll
    for (int i = 0; i < MF; ++i) {
        const int64_t row = i * 16 + (lane & 15);
        float v[4] = {acc[i][0], acc[i][1], acc[i][2], acc[i][3]};
        if (row < p.m && col < p.n) store_out<4>(p, row, col, v);
    }
}

constexpr int kFewRows = 32;

// ---- launches -------------------------------------------------------------------------------
template <bool MX, int BM, int BN, int WM, int WN>
hipError_t launch_tile(Fp8Params p, hipStream_t stream) {
    typedef Fp8Core<MX, BM, BN, WM, WN> Core;
    p.tiles_m = (int)((p.m + BM - 1) / BM);
    p.tiles_n = (int)((p.n + BN - 1) / BN);
    const int64_t groups = (int64_t)p.tiles_m * p.tiles_n * p.splits;
    const auto kernel = fp8_tile_kernel<MX, BM, BN, WM, WN>;
    if (Core::LDS_BYTES > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 Core::LDS_BYTES);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)((groups + 7) / 8 * 8)), dim3(Core::THREADS), Core::LDS_BYTES, stream, p);
    return hipGetLastError();
}

enum { kTile256, kTile128, kTile64 };  // 256 x 256 (x 128 without MX), 128 x 128, 64 x 128
struct Plan {
    int tile, splits;
};

Plan plan(int64_t m, int64_t n, int64_t k) {
    const int kb = (int)((k + kFp8Block - 1) / kFp8Block);
    for (int t : {kTile256, kTile128, kTile64}) {
        const int64_t bm = t == kTile256 ? 256 : t == kTile128 ? 128 : 64, bn = t == kTile256 ? 256 : 128;
        const int64_t tiles = ((m + bm - 1) / bm) * ((n + bn - 1) / bn);
        if (tiles >= 256 || t == kTile64) {
            int splits = 1;
            while (t == kTile64 && tiles * splits * 2 <= 512 && kb / (splits * 2) >= 4) splits *= 2;
            return {t, splits};
        }
    }
    return {kTile64, 1};
}

template <bool MX>
hipError_t launch_tiles(const Fp8Params &p, int tile, hipStream_t stream) {
    switch (tile) {
        case kTile256:  // without MX a wave's 128 x 64 would need more registers than two waves a SIMD have
            if constexpr (MX) return launch_tile<true, 256, 256, 2, 4>(p, stream);
            else return launch_tile<false, 256, 128, 4, 2>(p, stream);
        case kTile128: return launch_tile<MX, 128, 128, 2, 2>(p, stream);
        default: return launch_tile<MX, 64, 128, 1, 4>(p, stream);
    }
}

template <typename TX, int MF>
void launch_few(const Fp8Params &p, hipStream_t stream) {
    // waves along k until the card has two a SIMD, each with two blocks of k at least
    const int64_t tiles = (p.n + 15) / 16;
    int kw = 1;
    while (kw < kRowWaves && tiles * kw < 2048 && p.kb >= kw * 4) kw *= 2;
    const dim3 block(64 * kRowWaves), grid((unsigned)((tiles * kw + kRowWaves - 1) / kRowWaves));
    switch (kw) {
        case 1: hipLaunchKernelGGL((fp8_rows_kernel<TX, MF, 1>), grid, block, 0, stream, p); break;
        case 2: hipLaunchKernelGGL((fp8_rows_kernel<TX, MF, 2>), grid, block, 0, stream, p); break;
        case 4: hipLaunchKernelGGL((fp8_rows_kernel<TX, MF, 4>), grid, block, 0, stream, p); break;
        default: hipLaunchKernelGGL((fp8_rows_kernel<TX, MF, 8>), grid, block, 0, stream, p); break;
    }
}
template <typename TX>
void launch_few_rows(const Fp8Params &p, hipStream_t stream) {
    if (p.m <= 16) launch_few<TX, 1>(p, stream);
    else launch_few<TX, 2>(p, stream);
}

template <typename DT>
void launch_quant(const QuantParams &p, bool tile, hipStream_t stream) {
    if (tile) {
        const int64_t groups = (p.rows + kFp8Block - 1) / kFp8Block * p.blocks;
        hipLaunchKernelGGL(quant_tile_kernel<DT>, dim3((unsigned)groups), dim3(256), 0, stream, p);
    } else {
        const int64_t groups = (p.rows * p.blocks + 15) / 16;
        hipLaunchKernelGGL(quant_rows_kernel<DT>, dim3((unsigned)std::min<int64_t>(groups, 1 << 20)), dim3(256), 0, stream, p);
    }
}

}  // namespace

int fp8_few_rows() { return kFewRows; }

int64_t fp8_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    if (m <= kFewRows) return 0;
    const Plan pl = plan(m, n, k);
    return pl.splits > 1 ? pl.splits * m * n * 4 : 0;
}

hipError_t launch_fp8_quantize(const dsalt_fp8_quantize_args &a, hipStream_t stream) {
    if (a.rows == 0) return hipSuccess;
    QuantParams p = {};
    p.x = a.x;
    p.x_stride = a.x_stride;
    p.rows = a.rows;
    p.k = a.k;
    p.blocks = (a.k + kFp8Block - 1) / kFp8Block;
    p.q = static_cast<uint8_t *>(a.q);
    p.scale = a.scale;
    p.scale_stride = a.scale_stride;
    p.scale_f32 = a.scale_f32;
    const int size = a.x_dtype == DSALT_DTYPE_F32 ? 4 : 2;
    p.vec = (uintptr_t)a.x % 16 == 0 && a.x_stride * size % 16 == 0;
    if (a.x_dtype == DSALT_DTYPE_BF16) launch_quant<BF16>(p, a.tile, stream);
    else if (a.x_dtype == DSALT_DTYPE_F16) launch_quant<F16>(p, a.tile, stream);
    else launch_quant<F32>(p, a.tile, stream);
    return hipGetLastError();
}

hipError_t launch_fp8_matmul(const dsalt_fp8_matmul_args &a, hipStream_t stream) {
    if (a.m == 0) return hipSuccess;
    Fp8Params p = {};
    const int xsize = a.a_dtype == DSALT_DTYPE_E4M3 ? 1 : a.a_dtype == DSALT_DTYPE_F32 ? 4 : 2;
    p.a = {static_cast<const char *>(a.a), a.a_stride * xsize, a.m};
    p.b = {static_cast<const char *>(a.b), a.b_stride, a.n};
    p.m = a.m;
    p.n = a.n;
    p.k = a.k;
    p.kb = (a.k + kFp8Block - 1) / kFp8Block;
    p.sa = {static_cast<const char *>(a.a_scale), a.a_scale_stride_m, a.a_scale_stride_k, a.m, a.a_scale_e8m0};
    p.sb = {static_cast<const char *>(a.b_scale), a.b_scale_stride_n, a.b_scale_stride_k, (a.n + kFp8Block - 1) / kFp8Block,
            a.b_scale_e8m0};
    p.bias = a.bias;
    p.bias_dtype = a.bias_dtype;
    p.out = a.out;
    p.out_dtype = a.out_dtype;
    p.a_dtype = a.a_dtype;
    if (a.m <= kFewRows) {
        if (a.a_dtype == DSALT_DTYPE_E4M3) launch_few_rows<void>(p, stream);
        else if (a.a_dtype == DSALT_DTYPE_BF16) launch_few_rows<BF16>(p, stream);
        else if (a.a_dtype == DSALT_DTYPE_F16) launch_few_rows<F16>(p, stream);
        else launch_few_rows<F32>(p, stream);
        return hipGetLastError();
    }
    const Plan pl = plan(a.m, a.n, a.k);
    p.splits = pl.splits;
    p.part = static_cast<float *>(a.workspace);
    const hipError_t e = p.sa.e8m0 && p.sb.e8m0 ? launch_tiles<true>(p, pl.tile, stream) : launch_tiles<false>(p, pl.tile, stream);
    if (e != hipSuccess || p.splits == 1) return e;
    const int64_t items = p.m * ((p.n + 3) / 4);
    hipLaunchKernelGGL(fp8_join_kernel, dim3((unsigned)std::min<int64_t>((items + 255) / 256, 4096)), dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace dsalt
