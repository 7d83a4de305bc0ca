// What every position of the 8-bit cache gets of its sequence's attention weight,
// added to what it had: out = decay in + sum over the rows, and the query heads of its
// KV head, that see it of exp(scale q k - lse).
//
// A wave has 32 or 64 positions' keys in registers as operands of 32x32x16 MFMA (column
// = position) and meets all queries of the sequence, 32 at a time, which the four
// waves of a workgroup share through LDS: keys are read and expanded once, no result
// leaves a lane before the end, and each position has one writer, so the order of the
// additions is always the same.
#include "sd_kv8_attn_dev.hpp"

#pragma clang fp contract(fast)

namespace sd {

typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kWgtWaves = 4;
template <int HD> struct Kv8Queries {
    uintx4 q[HD / 16][64];  // [chunk of 16 channels][lane]: the MFMA's operands
    __align__(16) float lse[32];  // in base 2; infinite where the query does not exist or sees nothing
};

template <int HD, int NB>
__global__ __launch_bounds__(64 * kWgtWaves) __attribute__((amdgpu_waves_per_eu(2))) void k_kv8_weights(const Kv8Weights p) {
    constexpr int NC = HD / 16, NQ = HD / 64;  // chunks; 16-byte pieces of a tile of queries to a thread
    __shared__ Kv8Queries<HD> sh[2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r32 = lane & 31, hh = lane >> 5;
    const int s = blockIdx.z, h = blockIdx.y;
    const Kv8Layer L(p.a.L);
    Kv8Work W;
    if (!kv8_work(p.a, s, 0, 32, W)) return;
    const int T = (int)min((int64_t)W.T, p.ld), tiles = (W.nq + 31) / 32;
    const float sl2 = p.a.scale * 1.4426950408889634f;
    constexpr int kMine = 32 * NB, kChunk = kMine * kWgtWaves;
    for (int64_t c0 = (int64_t)blockIdx.x * kChunk; c0 < T; c0 += (int64_t)gridDim.x * kChunk) {
        // the wave's keys: lane (r32, hh) has the channels 16 c + 8 hh .. of position r32
        const int base = (int)c0 + wave * kMine;
        half8 kf[NB][NC];
        uint32_t nan[NB];
        bool have[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int pos = base + 32 * b;
            int page = -1;
            if (pos < T && (pos >> p.a.L.page_shift) < p.a.table_ld) page = p.a.table[(int64_t)s * p.a.table_ld + (pos >> p.a.L.page_shift)];
            page = __builtin_amdgcn_readfirstlane(page);
            have[b] = page >= 0 && page < p.a.L.n_pages;
            nan[b] = 0;
            if (have[b]) {
                const uint8_t *codes = L.codes(page, h, pos);
                const Kv8Head hd = *L.head(page, h, pos);
                uintx2 w[NC];
#pragma unroll
                for (int c = 0; c < NC; c++) w[c] = *(const uintx2 *)(codes + kv8_k_at(r32, 16 * c + 8 * hh, HD));
                nan[b] = hd.nan[0];
#pragma unroll
                for (int c = 0; c < NC; c++) kf[b][c] = __builtin_bit_cast(half8, kv8_expand(w[c].x, w[c].y, hd.scale[0]));
            } else {
#pragma unroll
                for (int c = 0; c < NC; c++) kf[b][c] = __builtin_bit_cast(half8, uintx4{0, 0, 0, 0});
            }
        }
        // tiles of queries that see some of the workgroup's positions: without a tree's mask not those in front of the first
        // or, with a window that has left all of them behind, after the last
        int t0 = 0, t1 = tiles;
        if (!p.a.mask) t0 = min(tiles, (int)(max((int64_t)0, c0 - W.P) * p.a.n_rep / 32));
        if (p.a.window > 0 && c0 >= p.a.sinks) {
            const int64_t last = min(c0 + kChunk, (int64_t)T) - 1 + p.a.window - 1 - W.P;  // the last row that sees one
            t1 = (int)max((int64_t)t0, min((int64_t)tiles, last < 0 ? (int64_t)0 : (last * p.a.n_rep + p.a.n_rep - 1) / 32 + 1));
        }
        uintx4 piece[NQ];
        float lse = 0.f;
        auto request = [&](int t) {
#pragma unroll
            for (int i = 0; i < NQ; i++) {
                const int u = threadIdx.x + i * 256, c = u >> 6, ln = u & 63, q = t * 32 + (ln & 31);
                piece[i] = *(const uintx4 *)(kvq_query(p.a, W, h, q) + 16 * c + 8 * (ln >> 5));
                if (q >= W.nq) piece[i] = uintx4{0, 0, 0, 0};
            }
            const int q = t * 32 + r32, qc = min(q, W.nq - 1);
            const float x = p.a.lse[(int64_t)(W.r0 + qc / p.a.n_rep) * p.a.n_heads + h * p.a.n_rep + qc % p.a.n_rep];
            lse = q >= W.nq || x == -INFINITY ? INFINITY : x * 1.4426950408889634f;
        };
        auto put = [&](Kv8Queries<HD> &S) {
#pragma unroll
            for (int i = 0; i < NQ; i++) {
                const int u = threadIdx.x + i * 256;
                S.q[u >> 6][u & 63] = piece[i];
            }
            if (threadIdx.x < 32) S.lse[threadIdx.x] = lse;
        };
        float sum[NB] = {};
        if (t0 < t1) {
            request(t0);
            put(sh[0]);
        }
        __syncthreads();
        for (int t = t0; t < t1; t++) {
            const Kv8Queries<HD> &S = sh[(t - t0) & 1];
            if (t + 1 < t1) request(t + 1);
            const int m_first = t * 32 / p.a.n_rep, m_last = (min(t * 32 + 32, W.nq) - 1) / p.a.n_rep;
            const int any_end = p.a.mask ? W.T : min(W.T, W.P + m_last + 1), all_end = p.a.mask ? W.P : min(W.T, W.P + m_first + 1);
            floatx16 acc[NB];
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int j = 0; j < 16; j++) acc[b][j] = 0.f;
            const bool some = base < any_end && (have[0] || have[NB - 1]);
            if (some) {
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const half8 a = __builtin_bit_cast(half8, S.q[c][lane]);
#pragma unroll
                    for (int b = 0; b < NB; b++) acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, kf[b][c], acc[b], 0, 0, 0);
                }
                float4 ls[4];
#pragma unroll
                for (int i = 0; i < 4; i++) ls[i] = *(const float4 *)&S.lse[8 * i + 4 * hh];
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const int pos0 = base + 32 * b;
                    if (pos0 >= any_end || !have[b]) continue;
                    const bool full = nan[b] == 0 && pos0 + 32 <= all_end &&
                                      (p.a.window <= 0 || pos0 > W.P + m_last - p.a.window || pos0 + 32 <= p.a.sinks);
                    float part = 0.f;
                    if (full) {
#pragma unroll
                        for (int j = 0; j < 16; j++) part += __builtin_amdgcn_exp2f(acc[b][j] * sl2 - ((const float *)&ls[j >> 2])[j & 3]);
                    } else {
                        const int pos = pos0 + r32;
                        const bool bad = nan[b] >> r32 & 1;
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            const int q = t * 32 + 8 * (j >> 2) + 4 * hh + (j & 3);
                            const uint32_t vis = kv8_visible<32>(p.a, W, min(q, W.nq - 1) / p.a.n_rep, pos0);
                            const float x = bad ? NAN : __builtin_amdgcn_exp2f(acc[b][j] * sl2 - ((const float *)&ls[j >> 2])[j & 3]);
                            if (q < W.nq && pos < T && (vis >> r32 & 1)) part += x;
                        }
                    }
                    sum[b] += part;
                }
            }
            if (t + 1 < t1) put(sh[(t + 1 - t0) & 1]);
            __syncthreads();
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum[b]), __float_as_uint(sum[b]), false, false);
            const float total = __uint_as_float(x[0]) + __uint_as_float(x[1]);
            const int pos = base + 32 * b + r32;
            if (hh == 0 && pos < T) {
                const int64_t at = ((int64_t)s * p.a.L.n_kv + h) * p.ld + pos;
                p.out[at] = p.in && p.decay != 0.f ? p.decay * p.in[at] + total : total;
            }
        }
    }
}

// 64 positions a wave where that still gives every CU a workgroup
void launch_kv8_weights(const Kv8Weights &in, hipStream_t st) {
    Kv8Weights p = in;
    int dev = 0, cus = 0;
    SD_HIP_CHECK(hipGetDevice(&dev));
    SD_HIP_CHECK(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    const int64_t groups = (int64_t)p.a.L.n_kv * p.a.n_seqs, len = std::max<int64_t>(1, std::min(p.max_len, p.ld));
    const bool two = (len + 255) / 256 * groups >= cus;
    const int64_t chunk = two ? 256 : 128, most = std::max<int64_t>(1, ((int64_t)1 << 23) / groups);
    const dim3 g((unsigned)std::min((len + chunk - 1) / chunk, most), (unsigned)p.a.L.n_kv, (unsigned)p.a.n_seqs), b(64 * kWgtWaves);
    if (p.a.L.hd == 128) {
        if (two) k_kv8_weights<128, 2><<<g, b, 0, st>>>(p);
        else k_kv8_weights<128, 1><<<g, b, 0, st>>>(p);
    } else {
        if (two) k_kv8_weights<64, 2><<<g, b, 0, st>>>(p);
        else k_kv8_weights<64, 1><<<g, b, 0, st>>>(p);
    }
    SD_HIP_CHECK(hipGetLastError());
}

}  // namespace sd
