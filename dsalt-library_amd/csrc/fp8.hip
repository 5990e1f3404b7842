// Products of 8-bit floats (e4m3) with a scale for each block of 128, and the quantisation that makes
// their operands:
//   C[m, n] = sum over blocks b of k:  sa[m, b] sb[n / 128, b] sum_{k in b} A[m, k] B[n, k]  (+ bias[n])
// A [M, K] holds activations with a scale for 128 elements of a row, B [N, K] weights with one for a tile
// of 128 x 128. Of the products of eight consecutive k the matrix instruction cuts what lies 13 bits below the
// largest one's exponent: at most 7 2^-13 of that product a group, 1.5e-5 of a result of normal values (fp8.h). All other sums,
// the scales and the bias are fp32; C is rounded once.
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

// Sixteen lanes a block of 128 of a row, kQuantRun blocks a lane in flight. Bound by HBM bytes: 8192 x 11008
// bf16 45 us (6.0 TB/s), 8192 x 1024 5.6 us; with one block a lane the latter took 9.
constexpr int kQuantRun = 4;
template <typename DT>
__global__ void __launch_bounds__(256) quant_rows_kernel(const QuantParams p) {
    const uint32_t items = (uint32_t)(p.rows * p.blocks);  // below 2^30
    const uint32_t first = blockIdx.x * (16 * kQuantRun) + (threadIdx.x >> 4);
    const int l = threadIdx.x & 15;
    float v[kQuantRun][8];
    uint32_t row[kQuantRun], block[kQuantRun];
#pragma unroll
    for (int u = 0; u < kQuantRun; ++u) {
        const uint32_t item = min(first + u * 16, items - 1);  // past the end: the last one again
        row[u] = item / (uint32_t)p.blocks;
        block[u] = item - row[u] * p.blocks;
        load8<DT>(p, row[u], block[u] * kFp8Block + l * 8, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kQuantRun; ++u) {
        const int c = block[u] * kFp8Block + l * 8;
        const uint32_t e8 = e8m0_of_amax(row16_max(amax8(v[u])));
        if (first + u * 16 >= items) break;
        if (c < p.k) store_q(p, row[u], c, quantised(v[u], e8));
        if (l == 0) store_scale(p, row[u], block[u], e8);
    }
}

// A workgroup a tile of 128 x 128. Bound by HBM bytes: 28672 x 8192 bf16 130 us (5.4 TB/s), 32000 x 1024 18 us, 5632 x
// 1024 7.6 us.
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
    float *part;  // [splits][m][part_ld], where k is split
    int splits, per_split;
    int64_t part_ld;  // n rounded up to a multiple of eight
    int tiles_m, tiles_n;
};

__device__ __forceinline__ float load_dt(const void *p, int64_t i, int dtype) {
    return dtype == DSALT_DTYPE_F32 ? Elem<F32>::ld(p, i) : dtype == DSALT_DTYPE_BF16 ? Elem<BF16>::ld(p, i) : Elem<F16>::ld(p, i);
}
__device__ __forceinline__ void store_dt(void *p, int64_t i, int dtype, float v) {
    if (dtype == DSALT_DTYPE_F32) Elem<F32>::st(p, i, v);
    else if (dtype == DSALT_DTYPE_BF16) Elem<BF16>::st(p, i, v);
    else Elem<F16>::st(p, i, v);
}
// Four results of columns col .. of a row, with the bias.
__device__ __forceinline__ void store_out(const Fp8Params &p, int64_t row, int64_t col, float (&v)[4]) {
    const int64_t at = row * p.n + col;
    if (p.bias)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < p.n) v[e] += load_dt(p.bias, col + e, p.bias_dtype);
    if (p.n % 4 == 0) {  // rows start on the vectors' boundaries; col < n then means col + 4 <= n
        if (p.out_dtype == DSALT_DTYPE_F32) {
            *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            const bool bf16 = p.out_dtype == DSALT_DTYPE_BF16;
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + at) =
                make_uint2(bf16 ? BF16::pack2(v[0], v[1]) : F16::pack2(v[0], v[1]),
                           bf16 ? BF16::pack2(v[2], v[3]) : F16::pack2(v[2], v[3]));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < p.n) store_dt(p.out, at + e, p.out_dtype, v[e]);
    }
}

// The kernel's arguments, read where they are needed: held in scalar registers over the loop over the
// blocks, they would not fit beside its own.
typedef const __attribute__((address_space(4))) Fp8Params *Fp8Args;
__device__ __forceinline__ Fp8Args fp8_args(bool first = false) {
    Fp8Args a = (Fp8Args)__builtin_amdgcn_kernarg_segment_ptr();
    if (!first) asm volatile("" : "+s"(a));
    return a;
}

// Tile number `w` of a launch: its corner and its blocks of k. Consecutive numbers go down groups of eight
// tile rows, so that tiles that run beside each other share their operands' rows in an XCD's L2.
struct Fp8Item {
    int m0, n0, first, steps;  // steps = 0: no such tile
    int split;
};
template <int BM, int BN>
__device__ __forceinline__ Fp8Item fp8_item(const Fp8Args p, int w) {
    const int tiles_m = p->tiles_m, tiles_n = p->tiles_n, per = tiles_m * tiles_n;
    Fp8Item it = {};
    if (w >= per * p->splits) return it;
    const auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };  // quotients come from vector units
    it.split = p->splits == 1 ? 0 : uniform(w / per);
    const int t = w - it.split * per;
    constexpr int G = 8;
    const int group = uniform(t / (G * tiles_n)), in = t - group * G * tiles_n, rows = min(G, tiles_m - group * G);
    const int column = uniform(in / rows);
    it.m0 = (group * G + in - column * rows) * BM;
    it.n0 = column * BN;
    it.first = it.split * p->per_split;
    it.steps = min(p->per_split, p->kb - it.first);
    return it;
}

// A stream of an operand's tiles: ROWS rows, a block of k a step, to LDS as GemmTile lays it out.
template <int ROWS, int NW>
struct Fp8Stream {
    typedef GemmTile<kKContig, ROWS, 64, NW> Tile;  // 64 pairs of bytes: a block
    static constexpr int LOADS = Tile::LPW, OFFS = Tile::OFFS;
    Tile tile;
    const char *at;  // the tile's first row at the step's block
    int bytes;       // from there to the end of its last row; 0: nothing to load
    uint32_t ld;
    i32x4 rsrc;
    uint32_t v[OFFS];
    __device__ __forceinline__ Fp8Stream(int wave, int lane, uint32_t ld_) : tile(wave, lane, ld_), at(nullptr), bytes(0), ld(ld_) {}
    __device__ __forceinline__ void start(const char *base, int64_t r0, int64_t rows, int kb, int k) {
        at = base + r0 * (int64_t)ld + (int64_t)kb * kFp8Block;
        const int n = (int)min(rows - r0, (int64_t)ROWS);
        bytes = n > 0 ? (n - 1) * (int)ld + k - kb * kFp8Block : 0;
    }
    // The loads of the step whose first byte of k has `left` bytes behind it, and on to the next. A chunk past k
    // would read the next row's first bytes.
    __device__ __forceinline__ void prepare(int left) {
        rsrc = uniform_rsrc(buffer_rsrc(at, (uint32_t)bytes));
#pragma unroll
        for (int u = 0; u < OFFS; ++u) v[u] = tile.kchunk[u] * 16 >= left ? kOutOfRange : tile.off[u];
        at += kFp8Block;
        bytes = max(bytes - kFp8Block, 0);
    }
    __device__ __forceinline__ void issue(int u, uint32_t lds, int wave) const {
        dma16(v[u % OFFS] + (uint32_t)(u / OFFS * OFFS * Tile::RPL) * ld, rsrc,
              __builtin_amdgcn_readfirstlane(lds + (wave * LOADS + u) * 1024));
    }
};

// A workgroup goes through tiles of BM x BN with WM x WN waves, over two stages of one block of k in LDS. MX: both scales
// are e8m0 and the matrix instruction applies them; otherwise both are fp32, and a block's product is formed
// from zero and added to the sums times the product of the scales, four multiply-adds an instruction.
//
// A wave holds one set of B's operands and a ring of four of A's, each read two groups of products (a
// group: one of A's with all of B's) before its own. The barrier that frees a stage stands before the last
// two groups of a step: what they need is in registers by then and the next stage has landed. Under them
// the next step's first two of A's are read, and each of B's as soon as its last product has been issued: it
// is needed a group later.
//
// The loads run two steps ahead of the products and from one tile straight into the next, so that a tile's
// results are stored while the next one's operands arrive.
//
// Bound by the matrix units' power at large sizes: 8192^3 with e8m0 scales 403-423 us (2.6-2.7 PFLOP/s), the
// matrix units busy 66 % of the cycles, at a clock that a loop of nothing but products lowers too (3.4-4.1
// PFLOP/s). 16384 x 2048 x 11008: 324-331 us (2.25 PFLOP/s), of which 55 are loads, 55 stores. With fp32 scales the
// multiply-adds and the narrower tile's LDS reads (128 bytes a cycle, what LDS gives) count: 435 us. Small
// ones wait for the first loads and the last stores: 6473 x 1360 x 1001 in fp16 21.5 us, of which 10
// stay with one block of k.
template <bool MX, int BM, int BN, int WM, int WN>
struct Fp8Core {
    static constexpr int NW = WM * WN, THREADS = NW * 64, M16 = BM / WM / 16, N16 = BN / WN / 16;
    static constexpr int LA = Fp8Stream<BM, NW>::LOADS, LB = Fp8Stream<BN, NW>::LOADS, LT = LA + LB + 1;
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

    // Tiles w, w + stride, ..
    __device__ __forceinline__ void run(char *lds, int w, int stride) {
        const uint32_t base = lds_addr(lds);
        Fp8Item cur = fp8_item<BM, BN>(fp8_args(true), w);
        if (!cur.steps) return;
        const GemmFrag<kKContig, BM, 64> fa(lane);
        const GemmFrag<kKContig, BN, 64> fb(lane);
        // the loads' streams, up to two steps ahead of the products: A, B and the wave's 64 scales of a step (rows
        // of A, or one wave B's blocks)
        Fp8Stream<BM, NW> da(wave, lane, (uint32_t)fp8_args(true)->a.ld);
        Fp8Stream<BN, NW> db(wave, lane, (uint32_t)fp8_args(true)->b.ld);
        const bool is_a = wave < BM / 64;
        constexpr int ssize = MX ? 1 : 4;
        const char *sat = nullptr;
        int sstep, ahead_w = w, ahead = 0, left = 0;
        uint32_t soff = kOutOfRange;
        i32x4 ds;
        auto start = [&](const Fp8Args p, const Fp8Item &it) {  // the streams go on to tile `it`
            ahead = it.steps;
            if (!ahead) {  // behind the last tile they read nothing, so that every step counts the same number of loads
                da.bytes = db.bytes = 0;
                soff = kOutOfRange;
                return;
            }
            da.start(p->a.base, it.m0, p->a.rows, it.first, (int)p->k);
            db.start(p->b.base, it.n0, p->b.rows, it.first, (int)p->k);
            left = (int)p->k - it.first * kFp8Block;
            const int64_t rs = is_a ? p->sa.row_stride : p->sb.row_stride, ks = is_a ? p->sa.k_stride : p->sb.k_stride;
            const int64_t row = is_a ? it.m0 + wave * 64 : it.n0 / kFp8Block;
            const int64_t rows = (is_a ? p->sa.rows : p->sb.rows) - row;
            const int slots = is_a ? 64 : wave == BM / 64 ? (BN + kFp8Block - 1) / kFp8Block : 0;
            sat = (is_a ? p->sa.base : p->sb.base) + (row * rs + it.first * ks) * ssize;
            sstep = (int)ks * ssize;
            soff = lane < slots && lane < rows ? (uint32_t)(lane * rs) * ssize : kOutOfRange;
        };
        auto prepare = [&] {
            da.prepare(left);
            db.prepare(left);
            ds = uniform_rsrc(buffer_rsrc(sat, kOutOfRange - 1));
            left -= kFp8Block;
            sat += sstep;
        };
        auto issue = [&](int stage, int u) {
            const uint32_t at = base + stage * STAGE;
            if (u < LA) da.issue(u, at, wave);
            else if (u < LA + LB) db.issue(u - LA, at + ASTAGE, wave);
            else {
                const uint32_t to = __builtin_amdgcn_readfirstlane(at + ASTAGE + BSTAGE + wave * 256);
                if constexpr (MX) dma1(soff, ds, to);
                else dma4(soff, ds, to);
            }
        };
        auto next_tile = [&] {  // behind a step's loads: on to the next tile where this one has no step left
            if (ahead && --ahead == 0) {
                const Fp8Args p = fp8_args();
                start(p, fp8_item<BM, BN>(p, ahead_w += stride));
            }
        };
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
        start(fp8_args(true), cur);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            prepare();
#pragma unroll
            for (int u = 0; u < LT; ++u) issue(t, u);
            next_tile();
        }
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
        for (;;) {
#pragma unroll
            for (int i = 0; i < M16; ++i)
#pragma unroll
                for (int j = 0; j < N16; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int t = 0; t < cur.steps; ++t) {
                const char *at = lds + stage * STAGE, *next = lds + (stage ^ 1) * STAGE;
                float sbf = 0.f, s[2];  // without MX: B's scale, and its product with A's of two groups
                f32x4 d[3];
                if constexpr (!MX) sbf = __uint_as_float(sb);
                auto add = [&](int q, f32x4 v) {
                    asm volatile("" : "+v"(v));  // no sooner: it would wait for the product
                    f32x4 &c = acc[q / N16][q % N16];
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[e] = fmaf(v[e], s[q / N16 % 2], c[e]);
                    asm volatile("" : "+v"(c));
                };
#pragma unroll
                for (int i = 0; i < M16; ++i) {
                    if (i == M16 - 2) {
                        prepare();
                        __builtin_amdgcn_sched_barrier(0);
                        tile_barrier<0>();
                        sb_next = read_sb(next);
                    }
                    if (i < M16 - 2) read_a(at, i + 2);
                    else read_a(next, i - M16 + 2);
                    if constexpr (!MX) s[i % 2] = __uint_as_float(sa[i % 4]) * sbf;
#pragma unroll
                    for (int j = 0; j < N16; ++j) {
                        if constexpr (MX) {
                            acc[i][j] = mfma_fp8(rb[j], ra[i % 4], acc[i][j], (int)sb, (int)sa[i % 4]);
                            // held here: a product has no side effect that would keep it from drifting behind the
                            // loads and the barrier, with copies of all that it needs
                            asm volatile("" : "+v"(acc[i][j]));
                        } else {
                            constexpr int D = 2;  // products between one and its sum: its latency
                            const int q = i * N16 + j;
                            d[q % (D + 1)] = mfma_fp8(rb[j], ra[i % 4]);
                            asm volatile("" : "+v"(d[q % (D + 1)]));
                            if (q >= D) add(q - D, d[(q - D) % (D + 1)]);
                            if (q == M16 * N16 - 1)
#pragma unroll
                                for (int r = q - D + 1; r <= q; ++r) add(r, d[r % (D + 1)]);
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
                    __builtin_amdgcn_sched_barrier(0);
                }
                next_tile();
                sb = sb_next;
                stage ^= 1;
            }
            store(cur);
            cur = fp8_item<BM, BN>(fp8_args(), w += stride);
            if (!cur.steps) break;
        }
        tile_barrier<0>();  // no load may land in LDS that another workgroup has by then
    }

    // The tile's results. The accumulators hold four consecutive n of one m; of two neighbouring blocks of 16
    // columns a lane takes eight of one, in exchange with the lanes 16 further on, and writes 16 bytes. Rows
    // past the operand's fall out of the descriptors, columns take an offset that does.
    __device__ __forceinline__ void store(const Fp8Item &it) {
        const Fp8Args p = fp8_args();
        const int g = lane >> 4, row = wm * M16 * 16 + (lane & 15);
        const bool part = p->splits > 1;
        const void *bias = p->bias;
        if (bias && !part)
#pragma unroll
            for (int j = 0; j < N16; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int64_t col = it.n0 + (wn * N16 + j) * 16 + g * 4 + e;
                    const float b = col < p->n ? load_dt(bias, col, p->bias_dtype) : 0.f;
#pragma unroll
                    for (int i = 0; i < M16; ++i) acc[i][j][e] += b;
                }
        const int64_t ld = part ? p->part_ld : p->n, m = p->m;
        char *out = part ? reinterpret_cast<char *>(p->part + it.split * m * ld) : static_cast<char *>(p->out);
        const int dtype = part ? DSALT_DTYPE_F32 : p->out_dtype;
        if (ld % 8) {
            if (dtype == DSALT_DTYPE_F32) return store_ragged<F32>(out, ld, it, m);
            if (dtype == DSALT_DTYPE_BF16) return store_ragged<BF16>(out, ld, it, m);
            return store_ragged<F16>(out, ld, it, m);
        }
        const int64_t col = it.n0 + wn * N16 * 16 + (g & 1) * 16 + (g >> 1) * 8;
        if (dtype == DSALT_DTYPE_F32) store_rows<F32>(out, ld, it, m, row, col);
        else if (dtype == DSALT_DTYPE_BF16) store_rows<BF16>(out, ld, it, m, row, col);
        else store_rows<F16>(out, ld, it, m, row, col);
    }
    template <typename DT>
    __device__ __forceinline__ void store_rows(char *out, int64_t ld, const Fp8Item &it, int64_t m, int row, int64_t col) const {
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        constexpr int SZ = std::is_same<DT, F32>::value ? 4 : 2;
        const int64_t total = (min(m - it.m0, (int64_t)BM) * ld - it.n0) * SZ;
        char *base = out + ((int64_t)it.m0 * ld + it.n0) * SZ;
        const uint32_t lane_off = (uint32_t)((row * ld + (col - it.n0)) * SZ);
#pragma unroll
        for (int i = 0; i < M16; ++i) {
            const int64_t skip = i * 16 * ld * SZ;
            const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(base + skip, (short)0, (int)max(total - skip, (int64_t)0), 0x00020000);
#pragma unroll
            for (int j = 0; j < N16; j += 2) {
                const uint32_t off = col + j * 16 < ld ? lane_off + j * 16 * SZ : kOutOfRange;
                if constexpr (SZ == 4) {
                    u32x4 lo, hi;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[i][j][e]),
                                                                        __float_as_uint(acc[i][j + 1][e]), false, false);
                        lo[e] = x[0];
                        hi[e] = x[1];
                    }
                    __builtin_amdgcn_raw_buffer_store_b128(lo, rsrc, off, 0, 0);
                    __builtin_amdgcn_raw_buffer_store_b128(hi, rsrc, off + 16, 0, 0);
                } else {
                    const f32x4 c = acc[i][j], d = acc[i][j + 1];
                    const auto x = __builtin_amdgcn_permlane16_swap(DT::pack2(c[0], c[1]), DT::pack2(d[0], d[1]), false, false);
                    const auto y = __builtin_amdgcn_permlane16_swap(DT::pack2(c[2], c[3]), DT::pack2(d[2], d[3]), false, false);
                    __builtin_amdgcn_raw_buffer_store_b128(u32x4{x[0], y[0], x[1], y[1]}, rsrc, off, 0, 0);
                }
            }
        }
    }
    // Rows that do not start on 16 bytes: the same pieces, written to wherever they lie.
    template <typename DT>
    __device__ __forceinline__ void store_ragged(char *out, int64_t ld, const Fp8Item &it, int64_t m) const {
        constexpr int SZ = std::is_same<DT, F32>::value ? 4 : 2;
        struct __attribute__((packed, aligned(4))) Piece {
            uint32_t w[2 * SZ];
        };
        struct __attribute__((packed, aligned(4))) Inner {
            uint32_t w[3];
        };
        const int g = lane >> 4;
#pragma unroll
        for (int i = 0; i < M16; ++i) {
            const int64_t row = it.m0 + (wm * M16 + i) * 16 + (lane & 15);
#pragma unroll
            for (int j = 0; j < N16; j += 2) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[i][j][e]), __float_as_uint(acc[i][j + 1][e]),
                                                                    false, false);
                    v[e] = __uint_as_float(x[0]);
                    v[4 + e] = __uint_as_float(x[1]);
                }
                const int64_t col = it.n0 + (wn * N16 + j + (g & 1)) * 16 + (g >> 1) * 8;
                char *to = out + (row * ld + col) * SZ;
                if (row < m && col + 8 <= ld) {
                    Piece q;
#pragma unroll
                    for (int e = 0; e < 2 * SZ; ++e) {
                        if constexpr (SZ == 4) q.w[e] = __float_as_uint(v[e]);
                        else q.w[e] = DT::pack2(v[2 * e], v[2 * e + 1]);
                    }
                    if (SZ == 4 || ((uintptr_t)to & 3) == 0) {
                        *reinterpret_cast<Piece *>(to) = q;
                    } else {  // rows of odd length: an element, six on dwords, an element
                        uint16_t *o = reinterpret_cast<uint16_t *>(to);
                        o[0] = (uint16_t)q.w[0];
                        Inner in;
#pragma unroll
                        for (int e = 0; e < 3; ++e) in.w[e] = q.w[e] >> 16 | q.w[e + 1] << 16;
                        *reinterpret_cast<Inner *>(o + 1) = in;
                        o[7] = (uint16_t)(q.w[3] >> 16);
                    }
                } else if (row < m) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (col + e < ld) Elem<DT>::st(to, e, v[e]);
                }
            }
        }
    }
};

template <bool MX, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM *WN * 64) fp8_tile_kernel(const Fp8Params) {
    typedef Fp8Core<MX, BM, BN, WM, WN> Core;
    extern __shared__ char lds[];
    Core core;
    core.run(lds, xcd_remap(blockIdx.x, gridDim.x), gridDim.x);
}

// Sum of the splits' parts in their order.
__global__ void __launch_bounds__(256) fp8_join_kernel(const Fp8Params p) {
    const int64_t total = p.m * p.part_ld, per = (p.n + 3) / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.m * per; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per, col = (i - row * per) * 4;
        const float *in = p.part + row * p.part_ld + col;
        float v[4] = {};
        for (int s = 0; s < p.splits; ++s, in += total) {
            const float4 f = *reinterpret_cast<const float4 *>(in);
            v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
        }
        store_out(p, row, col, v);
    }
}

// Up to 16 MF rows against 16 NT rows of weights: the eight waves of a workgroup share out the blocks of k, read
// the weights straight from memory and join their sums in LDS. TX: the rows are x's element type and a wave
// quantises what it reads of them, once for all its NT; void: they are e4m3 with scales. Bound by the
// weights' bytes, and by latency where they are few: all loads of a wave's blocks go out before the first
// product (U blocks at a time). 1 x 1024 x 32000 9.4 us (3.5 TB/s), 23 x 2816 x 1024 6.5 us.
constexpr int kRowWaves = 8;
template <typename TX, int MF, int NT>
__global__ void __launch_bounds__(64 * kRowWaves) fp8_rows_kernel(const Fp8Params p) {
    constexpr bool QUANT = !std::is_void<TX>::value;
    constexpr int U = NT > 2 ? 1 : 4 / NT;
    __shared__ f32x4 lds[kRowWaves][NT * MF][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, group = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NT);
    const char *bp[NT];
    bool b_in[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t row = n0 + j * 16 + (lane & 15);
        b_in[j] = row < p.n;
        bp[j] = p.b.base + (b_in[j] ? row : 0) * p.b.ld + group * 16;
    }
    f32x4 acc[NT][MF] = {};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int t = wave; t < p.kb; t += kRowWaves * U) {
        Fp8Frag fb[U][NT];
        float sb[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kb = t + u * kRowWaves;
            const int64_t k0 = (int64_t)kb * kFp8Block, k = k0 + group * 16;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                uint4 lo = zero, hi = zero;
                if (kb < p.kb && b_in[j] && k < p.k) lo = *reinterpret_cast<const uint4 *>(bp[j] + k0);
                if (kb < p.kb && b_in[j] && k + 64 < p.k) hi = *reinterpret_cast<const uint4 *>(bp[j] + k0 + 64);
                fb[u][j] = fp8_frag(lo, hi);
                sb[u][j] = kb < p.kb ? p.sb.at(min(n0 + j * 16, p.n - 1) / kFp8Block, kb) : 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kb = t + u * kRowWaves;
            if (kb >= p.kb) continue;
            const int64_t k = (int64_t)kb * kFp8Block + group * 16;
#pragma unroll
            for (int i = 0; i < MF; ++i) {
                const int64_t row = i * 16 + (lane & 15);
                const bool in = row < p.m;
                Fp8Frag fa = fp8_frag(zero, zero);
                float s = 0.f;
                if constexpr (QUANT) {
                    const char *ap = p.a.base + (in ? row : 0) * p.a.ld;
                    Raw8<TX> r0 = {}, r1 = {}, r2 = {}, r3 = {};
                    if (in && k < p.k) {
                        r0.load(ap, k / 8);
                        r1.load(ap, k / 8 + 1);
                    }
                    if (in && k + 64 < p.k) {
                        r2.load(ap, k / 8 + 8);
                        r3.load(ap, k / 8 + 9);
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
                    if (k < p.k) lo = *reinterpret_cast<const uint4 *>(ap + k);
                    if (k + 64 < p.k) hi = *reinterpret_cast<const uint4 *>(ap + k + 64);
                    fa = fp8_frag(lo, hi);
                    s = p.sa.at(row, kb);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const f32x4 d = mfma_fp8(fb[u][j], fa);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[j][i][e] = fmaf(d[e], s * sb[u][j], acc[j][i][e]);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MF; ++i) lds[wave][j * MF + i][lane] = acc[j][i];
    __syncthreads();
    for (int q = wave; q < NT * MF; q += kRowWaves) {
        f32x4 sum = lds[0][q][lane];
#pragma unroll
        for (int w = 1; w < kRowWaves; ++w) {
            const f32x4 o = lds[w][q][lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += o[e];
        }
        const int64_t row = q % MF * 16 + (lane & 15), col = n0 + q / MF * 16 + group * 4;
        float v[4] = {sum[0], sum[1], sum[2], sum[3]};
        if (row < p.m && col < p.n) store_out(p, row, col, v);
    }
}

constexpr int kFewRows = 32;

// ---- launches -------------------------------------------------------------------------------
template <bool MX, int BM, int BN, int WM, int WN>
hipError_t launch_tile(Fp8Params p, hipStream_t stream) {
    typedef Fp8Core<MX, BM, BN, WM, WN> Core;
    p.tiles_m = (int)((p.m + BM - 1) / BM);
    p.tiles_n = (int)((p.n + BN - 1) / BN);
    // as many workgroups as the card holds at once (LDS): they go through the tiles
    const int64_t groups = std::min<int64_t>((int64_t)p.tiles_m * p.tiles_n * p.splits, 256 * (163840 / Core::LDS_BYTES));
    const auto kernel = fp8_tile_kernel<MX, BM, BN, WM, WN>;
    if (Core::LDS_BYTES > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 Core::LDS_BYTES);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)((groups + 7) / 8 * 8)), dim3(Core::THREADS), Core::LDS_BYTES, stream, p);
    return hipGetLastError();
}

enum { kTile256, kTile128, kTile64 };  // 256 x 256, 128 x 128, 64 x 128
struct Plan {
    int tile, splits;
};

// The tile and the number of splits of k with the least time by a model of what they measured, in us: a
// workgroup's `start` (launch, first loads, results) and the steps over its blocks of k, which take longer the
// more workgroups share a CU, once for each round of the card. 512 x 2816 x 1024: 64 x 128 tiles 11.5, 128 x 128
// 14.8, 256 x 256 33.5; 8192 x 1024 x 5632: 73, 61, 55; 1000 x 4096 x 4096: 24.7, 28, 48. Splits cost a second
// launch and the traffic of their parts: 64 x 4096 x 4096 14.9, 12.7, 11.7 and 14.2 with 1, 2, 4 and 8.
// The largest tile is for e8m0 scales only: with fp32 ones a wave's 128 x 64 would need more registers than
// two waves a SIMD have, and 256 x 128, which fits, was no faster than 128 x 128 anywhere (8192^3: 601
// against 581; 6473 x 1360 x 1001: 23.3 against 22.3).
Plan plan(int64_t m, int64_t n, int64_t k, bool mx) {
    struct Tile {
        int bm, bn, per_cu;
        double start, step[3];
    };
    static const Tile tiles[] = {{256, 256, 1, 6.0, {1.4}}, {128, 128, 2, 4.5, {0.7, 0.95}}, {64, 128, 3, 4.0, {0.39, 0.6, 0.8}}};
    const int kb = (int)((k + kFp8Block - 1) / kFp8Block);
    Plan best = {kTile64, 1};
    double least = 1e30;
    for (int t : {kTile256, kTile128, kTile64}) {
        if (t == kTile256 && !mx) continue;
        for (int splits = 1; splits <= (t == kTile64 ? 16 : 1) && splits <= kb; splits *= 2) {
            const Tile &tile = tiles[t];
            const int per = (kb + splits - 1) / splits, used = (kb + per - 1) / per;  // none of them empty
            const int64_t groups = ((m + tile.bm - 1) / tile.bm) * ((n + tile.bn - 1) / tile.bn) * used;
            const int64_t rounds = (groups + 256 * tile.per_cu - 1) / (256 * tile.per_cu);
            const int shared = rounds > 1 ? tile.per_cu : (int)((groups + 255) / 256);
            double time = (double)rounds * (tile.start + per * tile.step[shared - 1]);
            if (used > 1) time += 3.0 + (double)used * (double)m * (double)n * 8.0 / 3e6;
            if (time < least) {
                least = time;
                best = {t, used};
            }
        }
    }
    return best;
}

template <bool MX>
hipError_t launch_tiles(const Fp8Params &p, int tile, hipStream_t stream) {
    if constexpr (MX)
        if (tile == kTile256) return launch_tile<true, 256, 256, 2, 4>(p, stream);
    return tile == kTile128 ? launch_tile<MX, 128, 128, 2, 2>(p, stream) : launch_tile<MX, 64, 128, 1, 4>(p, stream);
}

// Columns of a few-row workgroup, in 16s: wider ones quantise and read the rows less often; narrower ones where
// there would be fewer than two a CU.
int few_columns(int64_t n) { return n >= 4 * 16 * 480 ? 4 : n >= 2 * 16 * 480 ? 2 : 1; }

template <typename TX, int MF>
void launch_few(const Fp8Params &p, hipStream_t stream) {
    const auto go = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        hipLaunchKernelGGL((fp8_rows_kernel<TX, MF, NT>), dim3((unsigned)((p.n + 16 * NT - 1) / (16 * NT))), dim3(64 * kRowWaves), 0,
                           stream, p);
    };
    switch (few_columns(p.n)) {
        case 4: return go(std::integral_constant<int, 4>());
        case 2: return go(std::integral_constant<int, 2>());
        default: return go(std::integral_constant<int, 1>());
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
        const int64_t groups = (p.rows * p.blocks + 16 * kQuantRun - 1) / (16 * kQuantRun);
        hipLaunchKernelGGL(quant_rows_kernel<DT>, dim3((unsigned)groups), dim3(256), 0, stream, p);
    }
}

}  // namespace

int fp8_few_rows() { return kFewRows; }

Fp8Plan fp8_plan(int64_t m, int64_t n, int64_t k, bool e8m0) {
    if (m <= kFewRows) return {m <= 16 ? 16 : 32, few_columns(n) * 16, 1};
    const Plan pl = plan(m, n, k, e8m0);
    return {pl.tile == kTile256 ? 256 : pl.tile == kTile128 ? 128 : 64, pl.tile == kTile256 ? 256 : 128, pl.splits};
}

int64_t fp8_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    if (m <= kFewRows) return 0;
    const int64_t splits = std::max(plan(m, n, k, true).splits, plan(m, n, k, false).splits);
    return splits > 1 ? splits * m * ((n + 7) / 8 * 8) * 4 : 0;
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
    if (a.m <= kFewRows) {
        if (a.a_dtype == DSALT_DTYPE_E4M3) launch_few_rows<void>(p, stream);
        else if (a.a_dtype == DSALT_DTYPE_BF16) launch_few_rows<BF16>(p, stream);
        else if (a.a_dtype == DSALT_DTYPE_F16) launch_few_rows<F16>(p, stream);
        else launch_few_rows<F32>(p, stream);
        return hipGetLastError();
    }
    const bool mx = p.sa.e8m0 && p.sb.e8m0;
    const Plan pl = plan(a.m, a.n, a.k, mx);
    p.splits = pl.splits;
    p.per_split = (p.kb + pl.splits - 1) / pl.splits;
    p.part_ld = (p.n + 7) / 8 * 8;
    p.part = static_cast<float *>(a.workspace);
    const hipError_t e = mx ? launch_tiles<true>(p, pl.tile, stream) : launch_tiles<false>(p, pl.tile, stream);
    if (e != hipSuccess || p.splits == 1) return e;
    const int64_t items = p.m * ((p.n + 3) / 4);
    hipLaunchKernelGGL(fp8_join_kernel, dim3((unsigned)std::min<int64_t>((items + 255) / 256, 4096)), dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace dsalt
