// Device code shared by the kernels of the paged KV caches.
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

// Where row r of a call lives: its page id, or -1 where the row is left out.
__device__ __forceinline__ int kvq_row_page(const KvqRows &t, const KvqLayer &L, int r, int &slot) {
    const int s = t.seq ? t.seq[r] : 0;
    slot = t.slot ? t.slot[r] : t.slot0 + r;
    if (s < 0 || s >= t.n_seqs || slot < 0) return -1;
    const int at = slot >> L.page_shift;
    if (at >= t.table_ld) return -1;
    const int page = t.table[(int64_t)s * t.table_ld + at];
    return page >= 0 && page < L.n_pages ? page : -1;
}

// The value of another lane of the same four (XOR 1 or 2) without LDS.
template <int X> __device__ __forceinline__ uint32_t quad_xor(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, X == 1 ? 0xB1 : 0x4E, 0xf, 0xf, true);
}
template <int X> __device__ __forceinline__ double quad_xor(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)quad_xor<X>((uint32_t)b) | ((uint64_t)quad_xor<X>((uint32_t)(b >> 32)) << 32));
}

template <bool F32> __device__ __forceinline__ void load8(const void *base, int64_t at, float (&x)[8]) {
    if constexpr (F32) {
        const float4 a = *(const float4 *)((const float *)base + at), b = *(const float4 *)((const float *)base + at + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const half8 h = *(const half8 *)((const _Float16 *)base + at);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)h[i];
    }
}

// x[0..7] (channels 8 w ..) rotated in T: with neighbouring pairs inside the
// thread, with halves against channels 8 w +- hd / 2 (y).
template <typename T, int HD>
__device__ __forceinline__ void rotate8(const float (&x)[8], const float (&y)[8], const float *cos_r, const float *sin_r,
                                        int w, bool pairs, T (&out)[8]) {
    if (pairs) {
        const float4 c = *(const float4 *)(cos_r + 4 * w), s = *(const float4 *)(sin_r + 4 * w);
        const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const T a = x[2 * i], b = x[2 * i + 1], C = cc[i], S = ss[i];
            out[2 * i] = a * C - b * S;
            out[2 * i + 1] = b * C + a * S;
        }
    } else {
        const bool upper = w >= HD / 16;
        const int at = (8 * w) & (HD / 2 - 1);
        const float4 c0 = *(const float4 *)(cos_r + at), c1 = *(const float4 *)(cos_r + at + 4);
        const float4 s0 = *(const float4 *)(sin_r + at), s1 = *(const float4 *)(sin_r + at + 4);
        const float cc[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
        const float ss[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const T a = x[i], b = y[i], C = cc[i], S = upper ? ss[i] : -ss[i];
            out[i] = a * C + b * S;
        }
    }
}

}  // namespace sd
