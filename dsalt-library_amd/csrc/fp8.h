// 8-bit floats with scales: e4m3 conversions, scale reads and the matrix instruction.
//
// v_mfma_f32_16x16x128_f8f6f4 takes a whole block of 128 along k in one instruction: a lane holds 32
// bytes of its row (lane % 16), and every element of a block has the same scale, so that any
// assignment of k to lanes and bytes will do that both operands share. Here lane group g = lane / 16
// holds the 16-byte chunks g and g + 4 of the block: the two halves that GemmFrag reads.
//
// The instruction adds the products of eight consecutive k aligned to the largest of them, to 13 bits
// below its exponent; what lies lower is cut. All beyond such a group is fp32. That is its only rounding
// below 32 bits, and the price of its rate, twice that of 16-bit operands: against float64 a product of
// normal values is off by 1.5e-5 (2-norm) at every k from 128 to 16384, where the rounding of the
// operands to four bits has cost 4e-2 before it and a bf16 result's rounding costs 1.7e-3 after it.
#pragma once

#include "gemm.h"

namespace dsalt {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kFp8Block = 128;
constexpr int kUnitScale = 127;  // 2^0 as e8m0

typedef i32x8 Fp8Frag;  // a lane's chunks g and g + 4
__device__ __forceinline__ Fp8Frag fp8_frag(uint4 lo, uint4 hi) {
    return Fp8Frag{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}
// c + a b 2^(sa + sb - 254) over a block, with the scales of the lanes' rows (e8m0, low byte).
__device__ __forceinline__ f32x4 mfma_fp8(Fp8Frag a, Fp8Frag b, f32x4 c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}
// a b over a block, unscaled.
__device__ __forceinline__ f32x4 mfma_fp8(Fp8Frag a, Fp8Frag b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0,
                                                            kUnitScale, 0, kUnitScale);
}

// An e8m0 scale as fp32: 2^(b - 127), NaN of 255.
__device__ __forceinline__ float e8m0_f32(uint32_t b) {
    return __uint_as_float(b == 0 ? 0x00400000u : b == 255 ? 0x7fc00000u : b << 23);
}
// The scale of a block whose largest magnitude has the fp32 bits `amax`, as e8m0: the smallest power of two
// that brings it to at most 448 = 1.75 2^8, 1 of a block of zeros, NaN of one that holds no finite largest.
__device__ __forceinline__ uint32_t e8m0_of_amax(uint32_t amax) {
    if (amax >= 0x7f800000u) return 255;
    if (amax == 0) return kUnitScale;
    const int b = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u);
    return (uint32_t)max(b, 0);
}
// What a block's elements are multiplied by before their rounding; exact, being a power of two.
__device__ __forceinline__ float inverse_scale(uint32_t e8m0) {
    return e8m0 == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((254u - e8m0) << 23);
}
// Four values as e4m3, rounded to nearest even; magnitudes up to 448.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// One 4-byte element (or byte, as 32 bits) a lane at byte offset voff of the buffer, to LDS byte lds + 4 lane.
__device__ __forceinline__ void dma4(uint32_t voff, i32x4 rsrc, uint32_t lds) {
    asm volatile("buffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "{m0}"(lds) : "memory");
}
__device__ __forceinline__ void dma1(uint32_t voff, i32x4 rsrc, uint32_t lds) {
    asm volatile("buffer_load_ubyte %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "{m0}"(lds) : "memory");
}

// Scales [rows, blocks of k], fp32 or e8m0, any strides (in elements).
struct Fp8Scales {
    const char *base;
    int64_t row_stride, k_stride;
    int64_t rows;
    int e8m0;
    __device__ __forceinline__ int size() const { return e8m0 ? 1 : 4; }
    __device__ __forceinline__ float at(int64_t row, int64_t kb) const {
        const char *p = base + (row * row_stride + kb * k_stride) * size();
        return e8m0 ? e8m0_f32(*reinterpret_cast<const uint8_t *>(p)) : *reinterpret_cast<const float *>(p);
    }
};

}  // namespace dsalt
