// Device code shared by the kernels of the 4-bit KV cache.
#pragma once
#include "sd_kvq.hpp"

namespace sd {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));

// One nibble position of a word pair as two fp16 codes c - 8, exactly: the
// nibble under the exponent of 1024 is 1024 + c, in the next nibble 1024 + 16 c.
__device__ __forceinline__ half2v kvq_low(uint32_t w) {
    const uint32_t u = (w & 0x000f000fu) | 0x64006400u;
    return __builtin_bit_cast(half2v, u) + half2v{(_Float16)-1032.f, (_Float16)-1032.f};
}
__device__ __forceinline__ half2v kvq_high(uint32_t w) {
    const uint32_t u = (w & 0x00f000f0u) | 0x64006400u;
    const half2v s = {(_Float16)0.0625f, (_Float16)0.0625f}, b = {(_Float16)-72.f, (_Float16)-72.f};
    return __builtin_elementwise_fma(__builtin_bit_cast(half2v, u), s, b);
}
__device__ __forceinline__ uint32_t h2bits(half2v v) { return __builtin_bit_cast(uint32_t, v); }

// the 8 channels of a K word as fp16 values, in channel order
__device__ __forceinline__ uintx4 kvq_expand_k(uint32_t w, half2v d) {
    return uintx4{h2bits(kvq_low(w) * d), h2bits(kvq_high(w) * d), h2bits(kvq_low(w >> 8) * d),
                  h2bits(kvq_high(w >> 8) * d)};
}

}  // namespace sd
