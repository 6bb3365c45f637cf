// Activations as the attention operators take them: fp32, fp16 or bf16 bits,
// eight consecutive elements at a time (16 bytes of a 16-bit type, 32 of
// fp32), computed on in fp32 and rounded once to nearest even when stored.
#pragma once

#include "frq_common.h"

namespace frq {

constexpr int kTypeF32 = 0, kTypeF16 = 1, kTypeBF16 = 30;    // GGML type ids

__device__ __forceinline__ uint16_t f32_to_bf16_bits(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ uint16_t f32_to_f16_bits(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }

template <int TYPE>
struct Val;

template <>
struct Val<kTypeF32> {
    using Elem = float;
    static __device__ __forceinline__ void load8(const Elem* p, float (&f)[8]) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
    static __device__ __forceinline__ void store8(Elem* p, const float (&f)[8]) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
    static __device__ __forceinline__ Elem one(float x) { return x; }
};

template <>
struct Val<kTypeF16> {
    using Elem = uint16_t;
    static __device__ __forceinline__ void load8(const Elem* p, float (&f)[8]) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = f16_bits_to_f32(w[i]);
            f[2 * i + 1] = f16_bits_to_f32(w[i] >> 16);
        }
    }
    static __device__ __forceinline__ void store8(Elem* p, const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = f32_to_f16_bits(f[2 * i]) | ((uint32_t)f32_to_f16_bits(f[2 * i + 1]) << 16);
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ Elem one(float x) { return f32_to_f16_bits(x); }
};

template <>
struct Val<kTypeBF16> {
    using Elem = uint16_t;
    static __device__ __forceinline__ void load8(const Elem* p, float (&f)[8]) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __builtin_bit_cast(float, w[i] << 16);
            f[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ void store8(Elem* p, const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = f32_to_bf16_bits(f[2 * i]) | ((uint32_t)f32_to_bf16_bits(f[2 * i + 1]) << 16);
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ Elem one(float x) { return f32_to_bf16_bits(x); }
};

// f(Int<type>{}) for a type id checked by the caller.
template <typename F>
hipError_t with_type(int type, F&& f) {
    switch (type) {
        case kTypeF32: return f(Int<kTypeF32>{});
        case kTypeF16: return f(Int<kTypeF16>{});
        case kTypeBF16: return f(Int<kTypeBF16>{});
        default: return hipErrorInvalidValue;
    }
}

}  // namespace frq
