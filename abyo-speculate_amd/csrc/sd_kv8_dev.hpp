// Device code shared by the kernels of the 8-bit KV cache.
#pragma once
#include "sd_kv8.hpp"
#include "sd_kvq_dev.hpp"

namespace sd {

typedef float float2v __attribute__((ext_vector_type(2)));

constexpr int kKv8T = 256;  // threads that build a block: 8 to a position
// Channel of the i-th of a thread's HD / 8 values: 8 from c0 = 8 (thread % 8) and, with 128
// channels, the 8 that lie half a head away (which halves rotate with).
template <int HD> __host__ __device__ constexpr int kv8_ch(int c0, int i) { return c0 + (i & 7) + (i >> 3) * 64; }

// 2^e, e in [-126, 127]
__device__ __forceinline__ float kv8_two_to(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The smallest e with a <= 448 * 2^e = 1.75 * 2^(8 + e), for a finite a >= 0 (a
// subnormal's result is wrong, but below the least scale in any case).
__device__ __forceinline__ int kv8_exp(float a) {
    const uint32_t b = __float_as_uint(a);
    return (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u);
}

// x in 32 bits such that comparing it with a number of fewer bits, or rounding it to
// fewer, gives what x itself would: what does not fit goes into the last bit
__device__ __forceinline__ float kv8_odd(double x) {
    const float f = (float)x;
    const double d = (double)f;
    if (d == x) return f;
    const uint32_t b = __float_as_uint(f);
    return __uint_as_float((fabs(d) > fabs(x) ? b - 1 : b) | 1u);
}
__device__ __forceinline__ float kv8_odd(float x) { return x; }

// four codes of x * r
__device__ __forceinline__ uint32_t kv8_pack(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return (uint32_t)w;
}
__device__ __forceinline__ float kv8_value(uint32_t code, float scale) {
    return __builtin_amdgcn_cvt_f32_fp8((int)code, 0) * scale;
}
// eight codes as fp16 values, exactly
__device__ __forceinline__ uintx4 kv8_expand(uint32_t a, uint32_t b, float scale) {
    return uintx4{h2bits(__builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, false))),
                  h2bits(__builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, true))),
                  h2bits(__builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, false))),
                  h2bits(__builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, true)))};
}

// 8 x 8 bytes of the eight lanes that are 8 apart, lane 8 k + j the k-th of them: it has byte
// k of the i-th's at byte i afterwards
__device__ __forceinline__ uintx2 kv8_transpose(uintx2 w, int lane) {
    const auto far = __builtin_amdgcn_permlane32_swap(w.x, w.y, false, false);
    const auto mid = __builtin_amdgcn_permlane16_swap(__builtin_amdgcn_perm(far[1], far[0], 0x05040100u),
                                                      __builtin_amdgcn_perm(far[1], far[0], 0x07060302u), false, false);
    w = uintx2{__builtin_amdgcn_perm(mid[1], mid[0], 0x05040100u), __builtin_amdgcn_perm(mid[1], mid[0], 0x07060302u)};
    const uint32_t pick = lane & 8 ? 0x03070105u : 0x06020400u;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t of = (uint32_t)__builtin_amdgcn_mov_dpp((int)w[i], 0x128, 0xf, 0xf, true);  // lane ^ 8
        w[i] = __builtin_amdgcn_perm(of, w[i], pick);
    }
    return w;
}

// A block's keys or values from the values of its positions (keys that were rotated in
// f64 as kv8_odd leaves them): thread t has the
// channels kv8_ch(8 (t & 7), .) of position t >> 3 in x (live: the position holds
// something), in LDS `codes` come the block's 32 HD bytes of codes.  Returns the
// scale and the NaN bits.  All 256 threads call it; what they read of `codes`
// before, they have read when the first barrier is passed.
struct Kv8Sh {
    __align__(16) uint8_t codes[32 * 128];
    int exp[4];
    uint32_t nan[4];
};
template <int HD, bool V>
__device__ __forceinline__ void kv8_build(Kv8Sh &sh, const float (&x)[HD / 8], bool live, bool nan, float &scale, uint32_t &nans) {
    constexpr int C = HD / 8;
    const int tid = threadIdx.x, k = tid >> 3, c0 = (tid & 7) * 8, lane = tid & 63;
    float top = fabsf(x[0]);
    bool bad = !(top <= 65504.f);
#pragma unroll
    for (int i = 1; i < C; i++) {
        const float a = fabsf(x[i]);
        bad |= !(a <= 65504.f);
        top = fmaxf(top, a);
    }
    const uint64_t wave_bad = __builtin_amdgcn_ballot_w64(live && (bad || nan));
    const bool row_bad = (wave_bad >> (lane & 56) & 0xff) != 0;
    int e = live && !row_bad && top > 0.f ? min(max(kv8_exp(top), kKv8MinExp), kKv8MaxExp) : kKv8MinExp;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) e = max(e, __shfl_xor(e, o));
    if (lane == 0) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) m |= (uint32_t)((wave_bad >> (8 * i) & 0xff) != 0) << i;
        sh.exp[tid >> 6] = e;
        sh.nan[tid >> 6] = m;
    }
    __syncthreads();
    e = max(max(sh.exp[0], sh.exp[1]), max(sh.exp[2], sh.exp[3]));
    nans = sh.nan[0] | sh.nan[1] << 8 | sh.nan[2] << 16 | sh.nan[3] << 24;
    scale = kv8_two_to(e);
    const float r = live && !row_bad ? kv8_two_to(-e) : 0.f;
    uint32_t w[C / 4];
#pragma unroll
    for (int i = 0; i < C; i += 4) {
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            y[j] = r == 0.f ? 0.f : x[i + j] * r;  // (not NaN or infinity times 0)
            if (e == kKv8MaxExp) y[j] = fminf(fmaxf(y[j], -240.f), 240.f);  // 256 of it are more than fp16 holds
        }
        w[i / 4] = kv8_pack(y[0], y[1], y[2], y[3]);
    }
#pragma unroll
    for (int i = 0; i < C / 4; i += 2) {
        const uintx2 v{w[i], w[i + 1]};
        const int c = kv8_ch<HD>(c0, 4 * i);
        if constexpr (!V) *(uintx2 *)(sh.codes + kv8_k_at(k, c, HD)) = v;
        else *(uintx2 *)(sh.codes + kv8_v_at(k & 24, c + (k & 7), HD)) = kv8_transpose(v, lane);
    }
    __syncthreads();
}
// the codes in LDS to a block's keys or values in memory
template <int HD> __device__ __forceinline__ void kv8_codes_out(const Kv8Sh &sh, uint8_t *at) {
    if constexpr (HD == 128) *(uintx4 *)(at + threadIdx.x * 16) = *(const uintx4 *)(sh.codes + threadIdx.x * 16);
    else *(uintx2 *)(at + threadIdx.x * 8) = *(const uintx2 *)(sh.codes + threadIdx.x * 8);
}
// the values of 4 codes
__device__ __forceinline__ void kv8_values(uint32_t w, float scale, float *x) {
    const float2v a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = a.x * scale, x[1] = a.y * scale, x[2] = b.x * scale, x[3] = b.y * scale;
}
// as kv8_build takes them, a thread's channels of its position from a block's keys or values; all lanes of a wave call it
template <int HD, bool V> __device__ __forceinline__ void kv8_held(const uint8_t *codes, float scale, float (&x)[HD / 8]) {
    const int k = threadIdx.x >> 3, c0 = (threadIdx.x & 7) * 8, lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < HD / 8; i += 8) {
        const int c = kv8_ch<HD>(c0, i);
        const uintx2 w = V ? kv8_transpose(*(const uintx2 *)(codes + kv8_v_at(k & 24, c + (k & 7), HD)), lane)
                           : *(const uintx2 *)(codes + kv8_k_at(k, c, HD));
        kv8_values(w.x, scale, x + i);
        kv8_values(w.y, scale, x + i + 4);
    }
}
// the channels kv8_ch(c0, .) of position k of a block's keys
template <int HD> __device__ __forceinline__ void kv8_key(const uint8_t *codes, int k, int c0, float scale, float (&x)[HD / 8]) {
#pragma unroll
    for (int i = 0; i < HD / 8; i += 8) {
        const uintx2 w = *(const uintx2 *)(codes + kv8_k_at(k, kv8_ch<HD>(c0, i), HD));
        kv8_values(w.x, scale, x + i);
        kv8_values(w.y, scale, x + i + 4);
    }
}

}  // namespace sd
