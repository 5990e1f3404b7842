// Row tensors read and written eight elements at a time.
#pragma once

#include "../../include/dsalt_hip.h"
#include "common.h"
#include "rotary.h"  // the F32 element tag

#include <type_traits>

namespace dsalt {
namespace {

// Eight consecutive elements as loaded.
template <typename DT>
struct Raw8 {
    uint4 v;
    __device__ __forceinline__ void load(const void *p, int64_t chunk) { v = static_cast<const uint4 *>(p)[chunk]; }
    __device__ __forceinline__ void get(float *f) const {
        const uint32_t a[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[2 * e] = DT::lo_f32(a[e]);
            f[2 * e + 1] = DT::hi_f32(a[e]);
        }
    }
};
template <>
struct Raw8<F32> {
    float4 a, b;
    __device__ __forceinline__ void load(const void *p, int64_t chunk) {
        a = static_cast<const float4 *>(p)[2 * chunk];
        b = static_cast<const float4 *>(p)[2 * chunk + 1];
    }
    __device__ __forceinline__ void get(float *f) const {
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
};

template <typename DT>
__device__ __forceinline__ void store8(void *p, int64_t chunk, const float *f) {
    if constexpr (std::is_same<DT, F32>::value) {
        float4 *o = static_cast<float4 *>(p) + 2 * chunk;
        o[0] = make_float4(f[0], f[1], f[2], f[3]);
        o[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        static_cast<uint4 *>(p)[chunk] = make_uint4(DT::pack2(f[0], f[1]), DT::pack2(f[2], f[3]),
                                                    DT::pack2(f[4], f[5]), DT::pack2(f[6], f[7]));
    }
}
__device__ __forceinline__ void store8_dt(void *p, int64_t chunk, const float *f, int dtype) {
    if (dtype == DSALT_DTYPE_BF16) store8<BF16>(p, chunk, f);
    else if (dtype == DSALT_DTYPE_F16) store8<F16>(p, chunk, f);
    else store8<F32>(p, chunk, f);
}

}  // namespace
}  // namespace dsalt
