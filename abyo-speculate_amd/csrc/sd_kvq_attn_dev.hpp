// Device code that the attention kernels of the 4-bit and the 8-bit cache share.
#pragma once
#include "sd_attn_dev.hpp"
#include "sd_kvq_dev.hpp"

// products and sums may fuse within this code (the includer's setting is
// restored at the end of the file: -ffp-contract=on)
#pragma clang fp contract(fast)

namespace sd {

constexpr int kKvqT = 256, kKvqWaves = kKvqT / 64;

// Weights are 2^(score - m) in fp16 with m, a query's reference, this much below
// a maximum of its scores: the largest of the scores so far weighs 2^7 or more,
// so that a million positions of 2^-24 of its weight each still count (fp16 ends
// at 2^-24; a weight is rounded by 2^-11 of itself, or by 2^-32 of the largest).
// The headroom costs the many-row kernel 3 % (2048 rows over 8191 positions).
constexpr float kKvqHead = 7.f;

// the rows of sequence s: n of them from r0; false where there are none inside the call's
__device__ __forceinline__ bool kvq_seq_rows(const KvqAttn &p, int s, int &r0, int &n) {
    r0 = p.row_start ? p.row_start[s] : 0;
    const int end = p.row_start ? p.row_start[s + 1] : p.rows;
    n = end - r0;
    return r0 >= 0 && end > r0 && end <= p.rows;
}

__device__ __forceinline__ uint32_t kvq_pair(float a, float b) { return (uint32_t)f2h(a) | ((uint32_t)f2h(b) << 16); }
// C channels from k of a row of the result, in the activation layout or in rows
template <int C>
__device__ __forceinline__ void kvq_put(const KvqAttn &p, int row, int64_t k, const float (&o)[C], float inv) {
#pragma unroll
    for (int c = 0; c < C; c += 4) {
        if (p.out_act)
            *(uintx2 *)(p.out + act_index(row, k + c, (int)p.out_ld, p.out_act == 2)) =
                uintx2{kvq_pair(o[c] * inv, o[c + 2] * inv), kvq_pair(o[c + 1] * inv, o[c + 3] * inv)};
        else
            *(uintx2 *)(p.out + (int64_t)row * p.out_ld + k + c) =
                uintx2{kvq_pair(o[c] * inv, o[c + 1] * inv), kvq_pair(o[c + 2] * inv, o[c + 3] * inv)};
    }
}
// C channels from tc of a query's result: normalised, or a split's part (o, and once per query its maximum and sum)
template <int C>
__device__ __forceinline__ void kvq_emit(const KvqAttn &p, int split, int row, int head, int tc, float (&o)[C], float M, float l,
                                         bool first) {
    if (p.nsplit == 1) {
        kvq_put<C>(p, row, (int64_t)head * p.L.hd + tc, o, l == 0.f ? 0.f : 1.f / l);
        return;
    }
    const int64_t at = ((int64_t)split * p.rows + row) * p.n_heads + head;
    float *po = p.part_o + at * p.L.hd + tc;
#pragma unroll
    for (int c = 0; c < C; c += 4) *(float4 *)(po + c) = float4{o[c], o[c + 1], o[c + 2], o[c + 3]};
    if (first) *(float2 *)(p.part_ml + 2 * at) = float2{M, l};
}

// Workgroup id -> (sequence, KV head, tile, split): the splits one after the
// other, a split's groups turned by its number.  XCDs take workgroups in turn
// (8 of them), and the first splits are the ones every sequence has: with the
// splits next to each other all short sequences of a batch met on one XCD
// (16 sequences of up to 9001 positions in 32 splits: 19.5 us, in 35 14.8).
// With heads next to each other a head's tiles read its blocks through one L2.
struct KvqPlace {
    int s, h, tile, split;
};
__device__ __forceinline__ KvqPlace kvq_place(const KvqAttn &p) {
    KvqPlace r;
    const uint32_t id = blockIdx.x, n = (uint32_t)p.groups;
    r.split = (int)(id / n);
    uint32_t i = id % n + (uint32_t)r.split;
    i = i >= n ? i % n : i;
    r.h = (int)(i % (uint32_t)p.L.n_kv);
    i /= (uint32_t)p.L.n_kv;
    r.tile = (int)(i % (uint32_t)p.tiles);
    r.s = (int)(i / (uint32_t)p.tiles);
    return r;
}

// The page of block b, asked for before it is known whether the sequence has
// the block: one round trip to memory less before the first one is requested.
__device__ __forceinline__ int kvq_page(const KvqAttn &p, int s, int b) {
    return p.table[(int64_t)s * p.table_ld + min(b >> (p.L.page_shift - 5), p.table_ld - 1)];
}

// a query's channels
template <typename W> __device__ __forceinline__ const uint16_t *kvq_query(const KvqAttn &p, const W &w, int h, int q) {
    q = min(q, w.nq - 1);
    return p.q + (int64_t)(w.r0 + q / p.n_rep) * p.q_row + (int64_t)(h * p.n_rep + q % p.n_rep) * p.q_head;
}

// fp16 weights of eight scores (in base-2 units) against the reference, and their sum
__device__ __forceinline__ uintx4 kvq_weights(const float (&s)[8], float mu, float &sum) {
    uintx4 pk;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float a = __builtin_amdgcn_exp2f(s[2 * j] - mu), b = __builtin_amdgcn_exp2f(s[2 * j + 1] - mu);
        sum += a + b;
        pk[j] = h2bits(half2v{(_Float16)a, (_Float16)b});
    }
    return pk;
}

}  // namespace sd

#pragma clang fp contract(on)
