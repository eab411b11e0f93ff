// row_run.h -- runs of consecutive values of a row, loaded and stored as one
// piece of up to 16 bytes, and sums over rows.  Not part of the ABI.
#pragma once

#include "mfma_common.h"

namespace race {

// V consecutive values.
template <typename TIn, int V>
struct Run {
    static constexpr int kWords = V * int(sizeof(TIn)) / 4 > 0 ? V * int(sizeof(TIn)) / 4 : 1;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const TIn* p) {
        if constexpr (V * sizeof(TIn) == 16) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (V * sizeof(TIn) == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x, w[1] = v.y;
        } else if constexpr (V * sizeof(TIn) == 4 && V == 2) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (sizeof(TIn) == 4) {
            w[0] = __float_as_uint(*p);
        } else {
            w[0] = *p;
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (sizeof(TIn) == 4) return __uint_as_float(w[e]);
        return (e & 1) ? mfma::hi_half(w[e >> 1]) : mfma::lo_half(w[e >> 1]);
    }
    __device__ __forceinline__ static void store(TIn* p, const float (&x)[V]) {
        if constexpr (V * sizeof(TIn) == 16 && sizeof(TIn) == 4)
            *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        else if constexpr (V * sizeof(TIn) == 16)
            *reinterpret_cast<uint4*>(p) = make_uint4(mfma::pack2(x[0], x[1]), mfma::pack2(x[2], x[3]),
                                                      mfma::pack2(x[4], x[5]), mfma::pack2(x[6], x[7]));
        else if constexpr (V * sizeof(TIn) == 8 && sizeof(TIn) == 4)
            *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
        else if constexpr (V * sizeof(TIn) == 8)
            *reinterpret_cast<uint2*>(p) = make_uint2(mfma::pack2(x[0], x[1]), mfma::pack2(x[2], x[3]));
        else if constexpr (V == 2)
            *reinterpret_cast<uint32_t*>(p) = mfma::pack2(x[0], x[1]);
        else
            store_val(p, x[0]);
    }
};

// out[c] (nullable) = the sum of partial[rows][d] over its rows, in fp32 or bf16: a workgroup
// of 1024 threads takes 32 columns in 32 runs of rows, in a fixed order.
__device__ __forceinline__ void column_sums(const float* partial, int rows, int d, void* out, int f32) {
    __shared__ float sums[32][33];
    const int cl = threadIdx.x & 31, run = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
    const int per = (rows + 31) / 32, from = run * per, to = min(rows, from + per);
    float s = 0.f;
    if (c < d && out) {
#pragma unroll 8
        for (int r = from; r < to; ++r) s += partial[int64_t(r) * d + c];
    }
    sums[run][cl] = s;
    __syncthreads();
    if (run != 0 || c >= d || !out) return;
    float total = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) total += sums[r][cl];
    if (f32)
        static_cast<float*>(out)[c] = total;
    else
        static_cast<bf16_t*>(out)[c] = f32_to_bf16(total);
}

}  // namespace race
