// Tile products C[m, n] = sum_k A(m, k) B(n, k) of 16-bit matrices on v_mfma_f32_32x32x16 with
// fp32 accumulators, for the kernels that end a product in an epilogue of their own.
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
// consecutive n of one m per register group, and one lane-half swap makes them eight, 16 bytes
// of a 16-bit row.
#pragma once

#include "tiles.h"

namespace dsalt {

enum { kKContig = 0, kRContig = 1 };
constexpr int kGemmBK = 64;
constexpr uint32_t kOutOfRange = 0x80000000u;  // above every descriptor's size (kGemmMaxLd)
constexpr int64_t kGemmMaxLd = 1 << 21;        // elements of a row stride: 256 rows stay below 2^30 bytes

struct GemmOperand {
    const char *base;
    int64_t ld;   // bytes
    int64_t rows; // extent of r
};

// One operand's tile: ROWS rows of r, kGemmBK of k, filled by NW waves.
template <int LAY, int ROWS, int NW>
struct GemmTile {
    static constexpr int BYTES = ROWS * kGemmBK * 2;
    static constexpr int LPW = ROWS * 8 / (64 * NW);  // 16-byte loads per lane
    static constexpr int CPR = LAY == kKContig ? 8 : ROWS / 8;  // chunks per LDS row
    static constexpr int RPL = 64 / CPR;                        // LDS rows per load instruction
    static_assert(ROWS * 8 % (64 * NW) == 0, "the waves cover the tile");

    uint32_t off[2];  // of a wave's even and odd loads
    int kchunk;       // kKContig: the lane's chunk of k

    __device__ __forceinline__ GemmTile(int wave, int lane, uint32_t ld) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = (wave * LPW + u) * RPL + lane / CPR, slot = lane % CPR;
            if constexpr (LAY == kKContig) {
                kchunk = slot ^ (row & 7);
                off[u] = (uint32_t)row * ld + (kchunk << 4);
            } else {
                kchunk = 0;
                off[u] = (uint32_t)row * ld + ((slot ^ ((row & 3) << 1)) << 4);
            }
        }
    }

    // Loads k0 .. k0 + 63 (k in all) of rows r0 .. r0 + ROWS - 1 to the tile at LDS byte `lds`.
    __device__ __forceinline__ void load(uint32_t lds, int wave, const GemmOperand &o, int64_t r0, int64_t k0,
                                         int64_t k) const {
        const int64_t left = k - k0;
        const char *p;
        int64_t bytes;
        if constexpr (LAY == kKContig) {
            const int64_t rows = min(o.rows - r0, (int64_t)ROWS);
            p = o.base + r0 * o.ld + k0 * 2;
            bytes = rows > 0 && left > 0 ? (rows - 1) * o.ld + left * 2 : 0;
        } else {
            p = o.base + k0 * o.ld + r0 * 2;
            bytes = left > 0 && o.rows > r0 ? (min(left, (int64_t)kGemmBK) - 1) * o.ld + (o.rows - r0) * 2 : 0;
        }
        const i32x4 rsrc = uniform_rsrc(buffer_rsrc(p, (uint32_t)bytes));
        uint32_t v[2] = {off[0], off[1]};
        if constexpr (LAY == kKContig) {
            // a chunk past k would read the next row's first elements
            if (kchunk * 8 >= left) v[0] = v[1] = kOutOfRange;
        }
        const uint32_t ld = (uint32_t)o.ld;
#pragma unroll
        for (int u = 0; u < LPW; ++u)
            dma16(v[u & 1] + (uint32_t)((u & ~1) * RPL) * ld, rsrc,
                  __builtin_amdgcn_readfirstlane(lds + (wave * LPW + u) * 1024));
    }
};

// Reads of a tile as MFMA operands: the lane's r = r0 + lane % 32, k = 16 step + 8 (lane / 32) .. + 7.
template <int LAY, int ROWS>
struct GemmFrag {
    uint32_t a[2];  // byte of the lane's first element; kRContig: for even and odd 32-row blocks
    __device__ __forceinline__ explicit GemmFrag(int lane) {
        if constexpr (LAY == kKContig) {
            const int row = lane & 31;
            a[0] = a[1] = row * 128 + (((lane >> 5) ^ (row & 7)) << 4);
        } else {
            // ds_read_b64_tr_b16 gives lane l element l % 4 of the 8-byte pieces that lanes
            // 16 (l / 16) + 4 e + (l % 16) / 4, e = 0..3, address: a lane addresses k-row
            // (l % 16) / 4 and columns 16 ((l / 16) % 2) + 4 (l % 4) of its half's block
            const int krow = ((lane >> 5) << 3) + ((lane >> 2) & 3);
            const int chunk = (((lane >> 4) & 1) << 1) + ((lane & 3) >> 1);
#pragma unroll
            for (int p = 0; p < 2; ++p)
                a[p] = krow * (ROWS * 2) + (((chunk + 4 * p) ^ ((krow & 3) << 1)) << 4) + ((lane & 1) << 3);
        }
    }
    // block: r0 / 32
    __device__ __forceinline__ uint4 read(const char *tile, int block, int step) const {
        if constexpr (LAY == kKContig) {
            return *reinterpret_cast<const uint4 *>(tile + (a[0] ^ (step << 5)) + block * 4096);
        } else {
            const char *p = tile + a[block & 1] + (block >> 1) * 128 + step * (16 * ROWS * 2);
            const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *)p);
            const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) shortx4 *)(p + 4 * ROWS * 2));
            const uint2 l2 = bitcast<uint2>(lo), h2 = bitcast<uint2>(hi);
            return make_uint4(l2.x, l2.y, h2.x, h2.y);
        }
    }
};

// A workgroup's tile of the product: WM x WN waves over BM x BN, each FM x FN blocks of 32 x 32.
// PAIR: the B tile's first half are rows of one matrix and its second half the same rows of
// another (gate and up), and a wave holds the same n of both.
template <class DT, int BM, int BN, int WM, int WN, int ALAY, int BLAY, bool PAIR>
struct GemmCore {
    static constexpr int NW = WM * WN, THREADS = NW * 64, FM = BM / WM / 32, FN = BN / WN / 32, BK = kGemmBK;
    static constexpr int STAGE = (BM + BN) * BK * 2, LDS_BYTES = 2 * STAGE;
    static constexpr int LOADS = (BM + BN) * 8 / THREADS;
    typedef GemmTile<ALAY, BM, NW> TA;
    typedef GemmTile<BLAY, PAIR ? BN / 2 : BN, PAIR ? NW / 2 : NW> TB;

    f32x16 acc[FM][FN];
    int wm, wn, lane, wave;

    __device__ __forceinline__ GemmCore() {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        wm = wave % WM;
        wn = wave / WM;
    }
    // `segments` products of the operands a[s], b[s] (PAIR: b[0], b[1] are the two matrices and
    // there is one segment) over steps first .. last - 1 of their k-steps in order.
    template <int SEGMENTS>
    __device__ __forceinline__ void run(char *lds, const GemmOperand *a, const GemmOperand *b, int64_t m0, int64_t n0,
                                        int64_t k, int first, int last) {
        const uint32_t base = lds_addr(lds);
        const int per = (int)((k + BK - 1) / BK);  // steps of a segment
        const TA ta(wave, lane, (uint32_t)a[0].ld);
        const int bwave = PAIR ? wave % (NW / 2) : wave;
        const bool second = PAIR && wave >= NW / 2;
        const TB tb(bwave, lane, (uint32_t)(second ? b[1].ld : b[0].ld));
        const uint32_t bbase = BM * BK * 2 + (second ? BN * BK : 0);
        const GemmFrag<ALAY, BM> fa(lane);
        const GemmFrag<BLAY, PAIR ? BN / 2 : BN> fb(lane);
        auto load = [&](int stage, int step) {
            const int s = SEGMENTS > 1 && step >= per ? 1 : 0;
            const int64_t k0 = (int64_t)(step - s * per) * BK;
            ta.load(base + stage * STAGE, wave, a[s], m0, k0, k);
            tb.load(base + stage * STAGE + bbase, bwave, PAIR ? (second ? b[1] : b[0]) : b[s], n0, k0, k);
        };
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = f32x16{};
        if (first >= last) return;

        uint4 ra[2][FM], rb[2][FN];
        auto read = [&](int stage, int step, uint4 (&qa)[FM], uint4 (&qb)[FN]) {
            const char *at = lds + stage * STAGE, *bt = at + BM * BK * 2;
#pragma unroll
            for (int i = 0; i < FM; ++i) qa[i] = fa.read(at, wm * FM + i, step);
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                if constexpr (PAIR) {  // two tiles of BN / 2 rows
                    const int blk = wn * (FN / 2) + j % (FN / 2);
                    qb[j] = fb.read(bt + (j < FN / 2 ? 0 : BN * BK), blk, step);
                } else {
                    qb[j] = fb.read(bt, wn * FN + j, step);
                }
            }
        };
        auto mul = [&](const uint4 (&qa)[FM], const uint4 (&qb)[FN]) {
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = DT::mfma(bitcast<typename DT::vec8>(qb[j]), bitcast<typename DT::vec8>(qa[i]), acc[i][j]);
        };
        load(0, first);
        if (first + 1 < last) {
            load(1, first + 1);
            tile_barrier<LOADS>();
        } else {
            tile_barrier<0>();
        }
        read(0, 0, ra[0], rb[0]);
        for (int t = first; t < last; ++t) {
            const int stage = (t - first) & 1;
#pragma unroll
            for (int s = 0; s < 3; ++s) {
                read(stage, s + 1, ra[(s + 1) & 1], rb[(s + 1) & 1]);
                mul(ra[s & 1], rb[s & 1]);
            }
            // every wave is done reading this stage, and the next step's tiles have landed
            tile_barrier<0>();
            if (t + 2 < last) load(stage, t + 2);
            if (t + 1 < last) read(stage ^ 1, 0, ra[0], rb[0]);
            mul(ra[1], rb[1]);
        }
    }

    // The lane's 16-byte piece `half` (0, 1) of block (i, j): m = m0 + row(i), n = n0 + j * 32 + col(half)
    __device__ __forceinline__ int row(int i) const { return (wm * FM + i) * 32 + (lane & 31); }
    __device__ __forceinline__ int col(int half) const { return half * 16 + (lane >> 5) * 8; }
    // eight fp32 values of consecutive n
    __device__ __forceinline__ void values(const f32x16 &c, int half, float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(c[half * 8 + e]), __float_as_uint(c[half * 8 + 4 + e]),
                                                      false, false);
            v[e] = __uint_as_float(r[0]);
            v[4 + e] = __uint_as_float(r[1]);
        }
    }
};

template <class DT>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    return make_uint4(DT::pack2(v[0], v[1]), DT::pack2(v[2], v[3]), DT::pack2(v[4], v[5]), DT::pack2(v[6], v[7]));
}
template <class DT>
__device__ __forceinline__ void unpack8(uint4 w, float (&v)[8]) {
    const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] = DT::lo_f32(q[e]);
        v[2 * e + 1] = DT::hi_f32(q[e]);
    }
}

}  // namespace dsalt
