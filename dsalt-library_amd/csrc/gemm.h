// Tile products C[m, n] = sum_k A(m, k) B(n, k) of 16-bit matrices on v_mfma_f32_16x16x32 with
// fp32 accumulators, for the kernels that end a product in an epilogue of their own.
//
// Large products run at the card's power limit, and there the smaller blocks are the cheaper ones (a
// result element is read and written once per 32 of k instead of 16): operands held in registers,
// random bf16, 2077 TFLOP/s against 1301 with v_mfma_f32_32x32x16 in the same loop. Of whole
// training passes, where loads and LDS reads take their share, 4 % came of it at 16384 x 2048 x 5504,
// 2 % at 6473 x 1024 x 2816; 3000 x 768 x 2048, below that limit, takes 4 % more.
//
// An operand's element (r, k) lies at base[r * ld + k] (kKContig: weights and hidden states of a
// forward product) or at base[k * ld + r] (kRContig: the same tensors in their gradients'
// products). Either way a tile of ROWS x 64 elements goes to LDS as it lies in memory, with
// direct 16-byte loads whose chunks are XOR-swizzled, and the lanes read it back with k
// contiguous: kKContig rows by ds_read_b128, kRContig ones by ds_read_b64_tr_b16.
//
// Every load is bounds-checked by its buffer descriptor, which is rebuilt per k-step over what
// is left of the operand: rows past the operand and k past its end read zeros, so that
// any m, n and k (multiples of 8 along the contiguous axis) run without a padded copy, and
// offsets inside a descriptor stay below 2^31 whatever the tensor's size.
//
// C's tile is formed transposed (first MFMA operand B, second A): a lane then holds four
// consecutive n of one m per register group, 16 bytes of an fp32 row.
#pragma once

#include "tiles.h"

#include <type_traits>

namespace dsalt {

typedef float f32x4 __attribute__((ext_vector_type(4)));

enum { kKContig = 0, kRContig = 1 };
constexpr uint32_t kOutOfRange = 0x80000000u;  // above every descriptor's size (kGemmMaxLd)
constexpr int64_t kGemmMaxLd = 1 << 21;        // elements of a row stride: 256 rows stay below 2^30 bytes

struct GemmOperand {
    const char *base;
    int64_t ld;   // bytes
    int64_t rows; // extent of r
};

// What a chunk's place in a row of `CPR` chunks is XORed with.
template <int LAY, int CPR>
__device__ __forceinline__ int gemm_swizzle(int row) {
    static_assert(CPR == 8 || (LAY == kRContig && CPR >= 16), "a swizzle stays inside its row");
    if constexpr (LAY == kKContig) return (row >> 1) & 7;
    else if constexpr (CPR >= 16) return ((row & 3) << 2) | ((row >> 2) & 2);
    else return (row & 2) | ((row >> 1) & 4);
}

// One operand's tile: ROWS rows of r, BK of k, filled by NW waves.
//
// LDS has 64 banks of 4 bytes, and a 16-byte read serves 16 lanes at a time: the swizzle puts the
// same chunk of 16 consecutive rows on 16 different places of 256 bytes (two rows of 64): 4.2
// clocks a read, against 8.3 with chunk ^ (row & 7), which spreads 8 rows. A transposing read's 32
// lanes take 32 bytes of each of eight rows, r .. r + 3 and r + 8 .. r + 11: the first four go to
// different 64-byte places, the others to those places' other halves (of 128-byte rows, two to
// a 256 bytes, to four 32-byte places each).
template <int LAY, int ROWS, int BK, int NW>
struct GemmTile {
    static constexpr int BYTES = ROWS * BK * 2;
    static constexpr int LPW = BYTES / 16 / (64 * NW);               // 16-byte loads per lane
    static constexpr int CPR = LAY == kKContig ? BK / 8 : ROWS / 8;  // chunks per LDS row
    static constexpr int RPL = 64 / CPR;                             // LDS rows per load instruction
    static_assert(BYTES % (16 * 64 * NW) == 0, "the waves cover the tile");
    // loads of a wave after which the swizzle is that of the first again
    static constexpr int OFFS = LAY == kRContig && CPR == 16 && LPW == 4 ? 4 : 2;
    static_assert(LAY == kKContig || OFFS * RPL % 16 == 0 || (LPW * RPL == 8 && OFFS * RPL % 4 == 0), "swizzle's period");
    uint32_t off[OFFS];
    int kchunk[OFFS];  // kKContig: their chunks of k

    __device__ __forceinline__ GemmTile(int wave, int lane, uint32_t ld) {
#pragma unroll
        for (int u = 0; u < OFFS; ++u) {
            const int row = (wave * LPW + u) * RPL + lane / CPR, chunk = (lane % CPR) ^ gemm_swizzle<LAY, CPR>(row);
            kchunk[u] = chunk;
            off[u] = (uint32_t)row * ld + (chunk << 4);
        }
    }

    // The loads of k0 .. k0 + BK - 1 (k in all) of rows r0 .. r0 + ROWS - 1.
    struct Step {
        i32x4 rsrc;
        uint32_t v[OFFS], ld;
    };
    __device__ __forceinline__ Step step(const GemmOperand &o, int64_t r0, int64_t k0, int64_t k) const {
        const int64_t left = k - k0;
        const char *p;
        int64_t bytes;
        if constexpr (LAY == kKContig) {
            const int64_t rows = min(o.rows - r0, (int64_t)ROWS);
            p = o.base + r0 * o.ld + k0 * 2;
            bytes = rows > 0 && left > 0 ? (rows - 1) * o.ld + left * 2 : 0;
        } else {
            p = o.base + k0 * o.ld + r0 * 2;
            bytes = left > 0 && o.rows > r0 ? (min(left, (int64_t)BK) - 1) * o.ld + (o.rows - r0) * 2 : 0;
        }
        Step s;
        s.rsrc = uniform_rsrc(buffer_rsrc(p, (uint32_t)bytes));
        s.ld = (uint32_t)o.ld;
#pragma unroll
        for (int u = 0; u < OFFS; ++u) s.v[u] = off[u];
        if constexpr (LAY == kKContig) {  // a chunk past k would read the next row's first elements
#pragma unroll
            for (int u = 0; u < OFFS; ++u)
                if (kchunk[u] * 8 >= left) s.v[u] = kOutOfRange;
        }
        return s;
    }
    // Load `u` of LPW to the tile at LDS byte `lds`.
    static __device__ __forceinline__ void issue(const Step &s, int u, uint32_t lds, int wave) {
        dma16(s.v[u % OFFS] + (uint32_t)(u / OFFS * OFFS * RPL) * s.ld, s.rsrc,
              __builtin_amdgcn_readfirstlane(lds + (wave * LPW + u) * 1024));
    }
};

// Reads of a tile as MFMA operands: the lane's r = 16 block + lane % 16, k = 32 sub + 8 (lane / 16) .. + 7.
template <int LAY, int ROWS, int BK>
struct GemmFrag {
    uint32_t a;  // byte of the lane's first element in block 0, sub-step 0
    __device__ __forceinline__ explicit GemmFrag(int lane) {
        constexpr int CPR = LAY == kKContig ? BK / 8 : ROWS / 8;
        if constexpr (LAY == kKContig) {
            const int row = lane & 15;
            a = row * (BK * 2) + (((lane >> 4) ^ gemm_swizzle<LAY, CPR>(row)) << 4);
        } else {
            // ds_read_b64_tr_b16 gives lane l element l % 4 of the 8-byte pieces that lanes
            // 16 (l / 16) + 4 e + (l % 16) / 4, e = 0..3, address: a lane addresses k-row
            // (l % 16) / 4 and columns 4 (l % 4) of its 16 lanes' block
            const int krow = ((lane >> 4) << 3) + ((lane >> 2) & 3);
            a = krow * (ROWS * 2) + ((((lane & 3) >> 1) ^ gemm_swizzle<LAY, CPR>(krow)) << 4) + ((lane & 1) << 3);
        }
    }
    __device__ __forceinline__ uint4 read(const char *tile, int block, int sub) const {
        if constexpr (LAY == kKContig) {
            return *reinterpret_cast<const uint4 *>(tile + (a ^ (sub << 6)) + block * (16 * BK * 2));
        } else {
            const char *p = tile + (a ^ ((block & 7) << 5)) + (block >> 3) * 256 + sub * (32 * ROWS * 2);
            const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *)p);
            const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) shortx4 *)(p + 4 * ROWS * 2));
            const uint2 l2 = bitcast<uint2>(lo), h2 = bitcast<uint2>(hi);
            return make_uint4(l2.x, l2.y, h2.x, h2.y);
        }
    }
};

template <class DT>
__device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
    if constexpr (std::is_same<DT, BF16>::value)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bitcast<bf16x8>(a), bitcast<bf16x8>(b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(bitcast<f16x8>(a), bitcast<f16x8>(b), c, 0, 0, 0);
}

// A workgroup's tile of the product: WM x WN waves over BM x BN, each FM x FN blocks of 32 x 32.
// PAIR: the B tile's first half are rows of one matrix and its second half the same rows of
// another (gate and up), and a wave holds the same n of both.
//
// RA and RB = RA or RA - 1 stages of the A and B tiles: a step's loads are issued RA - 1 and
// RB - 1 steps before it is read, into the stages that the barrier of the step before has freed.
template <class DT, int BM, int BN, int BK_, int RA, int RB, int WM, int WN, int ALAY, int BLAY, bool PAIR>
struct GemmCore {
    static constexpr int BK = BK_, NW = WM * WN, THREADS = NW * 64, FM = BM / WM / 32, FN = BN / WN / 32, SUBS = BK / 32;
    static constexpr int BNB = PAIR ? BN / 2 : BN, NWB = PAIR ? NW / 2 : NW;  // of one B matrix
    typedef GemmTile<ALAY, BM, BK, NW> TA;
    typedef GemmTile<BLAY, BNB, BK, NWB> TB;
    static constexpr int ASTAGE = BM * BK * 2, BSTAGE = BN * BK * 2, LDS_BYTES = RA * ASTAGE + RB * BSTAGE;
    static constexpr int LA = TA::LPW, LB = TB::LPW;
    static_assert(SUBS % 2 == 0, "the operand registers alternate from one step to the next");
    static_assert(RB >= 2 && (RA == RB || RA == RB + 1), "see the waits in run()");

    f32x4 acc[FM][FN][4];  // of a block's quarters: 16 rows each, then 16 columns
    int wm, wn, lane, wave;

    __device__ __forceinline__ GemmCore() {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        wm = wave % WM;
        wn = wave / WM;
    }

    // `SEGMENTS` products of the operands a[s], b[s] (PAIR: b[0], b[1] are the two matrices and
    // there is one segment) over steps first .. last - 1 of their k-steps in order.
    template <int SEGMENTS>
    __device__ __forceinline__ void run(char *lds, const GemmOperand *a, const GemmOperand *b, int64_t m0, int64_t n0,
                                        int64_t k, int first, int last) {
        const uint32_t base = lds_addr(lds);
        const int per = (int)((k + BK - 1) / BK);  // steps of a segment
        const int bwave = PAIR ? wave % NWB : wave;
        const bool second = PAIR && wave >= NWB;
        const int from = SEGMENTS > 1 && first >= per ? 1 : 0;  // the first step's segment
        TA ta(wave, lane, (uint32_t)a[from].ld);
        TB tb(bwave, lane, (uint32_t)(second ? b[1].ld : b[from].ld));
        const uint32_t bbase = base + RA * ASTAGE + (second ? TB::BYTES : 0);
        const GemmFrag<ALAY, BM, BK> fa(lane);
        const GemmFrag<BLAY, BNB, BK> fb(lane);
        typename TA::Step sa;
        typename TB::Step sb;
        // past `last` the loads read nothing, so that every step counts the same number of loads; steps are
        // prepared in order, and where the second segment starts the lanes take its row strides
        auto prepare_a = [&](int step) {
            const int s = SEGMENTS > 1 && step >= per ? 1 : 0;
            if constexpr (SEGMENTS > 1)
                if (step == per) ta = TA(wave, lane, (uint32_t)a[1].ld);
            sa = ta.step(a[s], m0, step < last ? (int64_t)(step - s * per) * BK : k, k);
        };
        auto prepare_b = [&](int step) {
            const int s = SEGMENTS > 1 && step >= per ? 1 : 0;
            if constexpr (SEGMENTS > 1)
                if (step == per) tb = TB(bwave, lane, (uint32_t)b[1].ld);
            sb = tb.step(PAIR ? (second ? b[1] : b[0]) : b[s], n0, step < last ? (int64_t)(step - s * per) * BK : k, k);
        };
        // load u of a step: B's first, as its step is needed first where RA > RB
        auto issue = [&](int sta, int stb, int u) {
            if (u < LB) TB::issue(sb, u, bbase + stb * BSTAGE, bwave);
            else TA::issue(sa, u - LB, base + sta * ASTAGE, wave);
        };
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int h = 0; h < 4; ++h) acc[i][j][h] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (first >= last) return;

        constexpr int M16 = 2 * FM, N16 = 2 * FN, READS = M16 + N16;
        uint4 ra[2][M16], rb[2][N16];
        // operand read r of READS, in the order of the products' use: b0 a0 b1 b2 .. a1 ..
        auto read = [&](int sta, int stb, int sub, int r, int buf) {
            const char *at = lds + sta * ASTAGE, *bt = lds + RA * ASTAGE + stb * BSTAGE;
            if (r == 0 || (r >= 2 && r <= N16)) {
                const int j = r == 0 ? 0 : r - 1;
                if constexpr (PAIR) rb[buf][j] = fb.read(bt + (j < FN ? 0 : TB::BYTES), wn * FN + j % FN, sub);
                else rb[buf][j] = fb.read(bt, wn * N16 + j, sub);
            } else {
                const int i = r == 1 ? 0 : r - N16;
                ra[buf][i] = fa.read(at, wm * M16 + i, sub);
            }
        };
        auto mul = [&](int q, int buf) {
            const int i = q / N16, j = q % N16;
            f32x4 &c = acc[i >> 1][j >> 1][(i & 1) * 2 + (j & 1)];
            c = mfma16<DT>(rb[buf][j], ra[buf][i], c);
        };
        constexpr int NM = M16 * N16, LT = LA + LB;
        auto read_before = [&](int sta, int stb, int sub, int q, int buf) {
#pragma unroll
            for (int r = 0; r < READS; ++r)  // spread over three quarters of the products
                if (r * (NM * 3 / 4) / READS == q) read(sta, stb, sub, r, buf);
        };
        // the loads of a group are spread over the SUBS sub-steps after the barrier that frees their
        // stages (part 0 .. SUBS - 1), one after every few products, so that they do not fill the memory
        // pipe's queue and hold the wave's products back (in the first half of each sub-step: up to 4 %
        // slower dx, 2 % faster down)
        auto issue_after = [&](int sta, int stb, int part, int q) {
#pragma unroll
            for (int u = 0; u < LT; ++u)
                if (u * SUBS / LT == part && (u * SUBS % LT * NM + LT * NM / 2 / LT) / LT == q) issue(sta, stb, u);
        };
        // group order: (A0 where RA > RB,) then B(t), A(t + RA - RB) for t = 0, 1, ..
        if constexpr (RA > RB) {
            prepare_a(first);
#pragma unroll
            for (int u = LB; u < LT; ++u) issue(0, 0, u);
        }
#pragma unroll
        for (int t = 0; t < RB; ++t) {
            prepare_b(first + t);
            prepare_a(first + t + RA - RB);
#pragma unroll
            for (int u = 0; u < LT; ++u)
                if (t < RB - 1 || u * SUBS / LT == 0) issue(t + RA - RB, t, u);
        }
        constexpr int PART0 = (LT + SUBS - 1) / SUBS;  // loads of a group's part 0
        tile_barrier<PART0 + (RB - 2) * LT + (RA - RB) * LA>();
#pragma unroll
        for (int r = 0; r < READS; ++r) read(0, 0, 0, r, 0);
        int sta = 0, stb = 0, olda = RA - 1, oldb = RB - 1;
        for (int t = first; t < last; ++t) {
            // a read of the next sub-step's operands between one product and the next; the compiler orders
            // two products at a time (one: 1 to 3 % slower, four: 1 %)
#pragma unroll
            for (int s = 0; s < SUBS - 1; ++s)
#pragma unroll
                for (int q = 0; q < NM; ++q) {
                    read_before(sta, stb, s + 1, q, (s + 1) & 1);
                    mul(q, s & 1);
                    issue_after(olda, oldb, s + 1, q);
                    if (q % 2) __builtin_amdgcn_sched_barrier(0);
                }
            olda = sta;
            oldb = stb;
            sta = sta + 1 == RA ? 0 : sta + 1;
            stb = stb + 1 == RB ? 0 : stb + 1;
            prepare_b(t + RB);
            prepare_a(t + RA);
            __builtin_amdgcn_sched_barrier(0);
            // every wave is done reading the old stages, and the next step's tiles have landed: of the
            // loads issued since, only whole groups (and A's part of one) may be outstanding
            tile_barrier<(RB - 2) * LT + (RA - RB) * LA>();
#pragma unroll
            for (int q = 0; q < NM; ++q) {
                read_before(sta, stb, 0, q, 0);
                mul(q, 1);
                issue_after(olda, oldb, 0, q);
                if (q % 2) __builtin_amdgcn_sched_barrier(0);
            }
        }
        tile_barrier<0>();  // no load may land in LDS that another workgroup has by then
    }

    // The accumulators hold one row m per lane; memory wants whole rows. Each wave turns its row
    // blocks (32 rows of FN * 32 fp32 columns) in its own part of LDS, free after run(): it
    // writes them with put() and reads them with get() as pieces of eight columns, piece t * 64 +
    // lane of the block's pieces in row order, so that loads and stores of 16 bits a column cover
    // 16-byte pieces of whole rows. XOR with the row spreads the rows over the banks.
    static constexpr int COLS = FN * 32, PIECES = (PAIR ? COLS / 2 : COLS) / 8, TURNS = 32 * PIECES / 64;
    __device__ __forceinline__ char *turn(char *lds) const { return lds + wave * (32 * COLS * 4); }
    __device__ __forceinline__ void put(char *lds, const f32x4 (&row)[FN][4]) const {
        char *p = turn(lds) + (lane & 15) * (COLS * 4);
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int h = 0; h < 4; ++h)
                *reinterpret_cast<f32x4 *>(p + (h >> 1) * (16 * COLS * 4) +
                                           (((j * 8 + (h & 1) * 4 + (lane >> 4)) ^ (lane & 15)) << 4)) = row[j][h];
        __builtin_amdgcn_wave_barrier();
    }
    // Row and first column (of the wave's) of the lane's piece in turn t.
    static constexpr int TURN_ROWS = 64 / PIECES;
    static_assert(64 % PIECES == 0, "a turn covers whole rows");
    __device__ __forceinline__ int piece_row(int t) const { return t * TURN_ROWS + lane / PIECES; }
    __device__ __forceinline__ int piece_col() const { return lane % PIECES * 8; }
    // offset: columns from the piece's (PAIR: COLS / 2 reaches the second matrix)
    __device__ __forceinline__ void get(const char *lds, int t, int offset, float (&v)[8]) const {
        const int r = piece_row(t), c = (piece_col() + offset) / 4;
        const char *p = turn(const_cast<char *>(lds)) + r * (COLS * 4);
        const float4 lo = *reinterpret_cast<const float4 *>(p + ((c ^ (r & 15)) << 4));
        const float4 hi = *reinterpret_cast<const float4 *>(p + (((c + 1) ^ (r & 15)) << 4));
        v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
        v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
    }
};

template <class DT>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    return make_uint4(DT::pack2(v[0], v[1]), DT::pack2(v[2], v[3]), DT::pack2(v[4], v[5]), DT::pack2(v[6], v[7]));
}

}  // namespace dsalt
