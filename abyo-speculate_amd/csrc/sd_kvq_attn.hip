// Attention over the 4-bit paged KV cache (sd_kvq.hpp).
//
// Split flash-decoding: a workgroup takes one query tile (QT x 16 queries of
// one KV head: rows times the heads that share it) and one range of 32-position
// blocks; its four waves take the range's blocks in turn.  A block's codes
// become fp16 values in registers (exactly the values the codes stand for),
// scores are computed transposed, S^T = K Q^T, so that a lane's eight
// probabilities are the operand of O^T = V^T P^T, and each wave keeps a running
// maximum and sum in f32.  The waves meet in LDS, the splits in a second launch.
#include "sd_attn_dev.hpp"
#include "sd_kvq_dev.hpp"

#pragma clang fp contract(fast)

namespace sd {

constexpr int kKvqT = 256, kKvqWaves = kKvqT / 64;

// What a wave loads of one block: the words of its lane.
template <int HD> struct KvqStep {
    uintx4 kc[HD / 64];  // [kt] at hd 128, both kt at 64
    uint32_t ks;         // steps of kt 0 and 1
    uintx4 vc[2];        // 8 positions' words
    uintx4 vs;           // their 8 steps
};

template <int HD>
__device__ __forceinline__ void kvq_load(KvqStep<HD> &b, const uint8_t *blk, int lane) {
    const int r16 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < HD / 64; i++) b.kc[i] = *(const uintx4 *)(blk + i * 1024 + lane * 16);
    b.ks = *(const uint32_t *)(blk + 16 * HD + (r16 + 16 * (HD == 128 ? g : g >> 1)) * 4);
    const uint8_t *v = blk + 18 * HD + ((HD == 128 ? r16 : r16 >> 1) + (HD / 8) * g) * 32;
    b.vc[0] = *(const uintx4 *)v;
    b.vc[1] = *(const uintx4 *)(v + 16);
    b.vs = *(const uintx4 *)(blk + 34 * HD + ((HD == 128 ? r16 >> 2 : r16 >> 3) * 4 + g) * 16);
}

template <int HD, int QT> struct KvqState {
    uintx4 q[QT][HD / 32];
    floatx4 o[QT][HD / 16];
    float m[QT], l[QT];
};

// the rows of sequence s: n of them from r0; false where there are none inside the call's
__device__ __forceinline__ bool kvq_seq_rows(const KvqAttn &p, int s, int &r0, int &n) {
    r0 = p.row_start ? p.row_start[s] : 0;
    const int end = p.row_start ? p.row_start[s + 1] : p.rows;
    n = end - r0;
    return r0 >= 0 && end > r0 && end <= p.rows;
}

// bit j: position j of the lane's 8 is a number's (its V step is not NaN)
__device__ __forceinline__ uint32_t kvq_nan_steps(const uintx4 &vs) {
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        bad |= (uint32_t)((vs[i] & 0x7fffu) > 0x7c00u) << (2 * i);
        bad |= (uint32_t)((vs[i] & 0x7fff0000u) > 0x7c000000u) << (2 * i + 1);
    }
    return bad;
}

template <int HD, int QT>
__global__ __launch_bounds__(kKvqT) void k_kvq_attn(const KvqAttn p) {
    constexpr int NDC = HD / 32, NDT = HD / 16;
    __shared__ float sh_o[kKvqWaves][16][HD];
    __shared__ float sh_ml[kKvqWaves][16][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, g = lane >> 4;
    const int split = blockIdx.x, s = blockIdx.z;
    const int h = blockIdx.y % p.L.n_kv, tile = blockIdx.y / p.L.n_kv;
    int r0, n;
    if (!kvq_seq_rows(p, s, r0, n)) return;
    const int T = p.row_start ? p.kv_len[s] : p.len0;
    const int nq = min(n, p.max_rows) * p.n_rep, q0 = tile * QT * 16;
    if (q0 >= nq) return;
    const int P = T - n;  // row i is position P + i
    const int m_last = (min(q0 + QT * 16, nq) - 1) / p.n_rep, m_first = q0 / p.n_rep;
    // positions any of the tile's rows may see, and those that all of them see
    const int t_end = p.mask ? T : min(T, P + m_last + 1);
    const int t_all = p.mask ? P : P + m_first + 1;
    const int nblk = t_end > 0 ? (int)min((int64_t)((t_end - 1) / 32 + 1), (int64_t)p.table_ld << (p.L.page_shift - 5)) : 0;
    const int b0 = (int)((int64_t)nblk * split / p.nsplit), b1 = (int)((int64_t)nblk * (split + 1) / p.nsplit);

    KvqState<HD, QT> S;
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int q = min(q0 + t * 16 + r16, nq - 1);
        const uint16_t *qr = p.q + (int64_t)(r0 + q / p.n_rep) * p.q_row + (int64_t)(h * p.n_rep + q % p.n_rep) * p.q_head;
#pragma unroll
        for (int dc = 0; dc < NDC; dc++) S.q[t][dc] = *(const uintx4 *)(qr + 8 * (g * NDC + dc));
#pragma unroll
        for (int dt = 0; dt < NDT; dt++) S.o[t][dt] = floatx4{0.f, 0.f, 0.f, 0.f};
        S.m[t] = -INFINITY;
        S.l[t] = 0.f;
    }
    const float sl2 = p.scale * 1.4426950408889634f;
    const int *table = p.table + (int64_t)s * p.table_ld;
    for (int b = b0 + wave; b < b1; b += kKvqWaves) {
        const int page = __builtin_amdgcn_readfirstlane(table[b >> (p.L.page_shift - 5)]);
        if (page < 0 || page >= p.L.n_pages) continue;  // holds no positions
        KvqStep<HD> k;
        kvq_load<HD>(k, p.L.block(page, h, b * 32), lane);
        const int key0 = b * 32 + 8 * g;
        const bool full = b * 32 + 32 <= t_all && b * 32 + 32 <= T;
        // K operands
        uintx4 ka[2][NDC];
        {
            const uint32_t k0 = k.ks & 0xffffu, k1 = k.ks >> 16;
            const half2v d0 = __builtin_bit_cast(half2v, k0 | (k0 << 16)), d1 = __builtin_bit_cast(half2v, k1 | (k1 << 16));
#pragma unroll
            for (int dc = 0; dc < NDC; dc++) {
                ka[0][dc] = kvq_expand_k(HD == 128 ? k.kc[0][dc] : k.kc[0][dc], d0);
                ka[1][dc] = kvq_expand_k(HD == 128 ? k.kc[HD / 64 - 1][dc] : k.kc[0][2 + dc], d1);
            }
        }
        // V operands: a position pair's nibbles n are channels n (hd 128) or 4 (r16 & 1) + n (64) of the lane's word
        uintx4 va[NDT];
        uint32_t bad = 0;
        if (!full) {
            bad = kvq_nan_steps(k.vs);
            if (bad) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (bad >> (2 * i) & 1) k.vs[i] &= 0xffff0000u;
                    if (bad >> (2 * i + 1) & 1) k.vs[i] &= 0x0000ffffu;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t wa = k.vc[j >> 1][(2 * j) & 3], wb = k.vc[j >> 1][(2 * j + 1) & 3];
            const half2v d = __builtin_bit_cast(half2v, (uint32_t)k.vs[j]);
#pragma unroll
            for (int u = 0; u < NDT / 4; u++) {
                const uint32_t sel = HD == 128 ? (u ? 0x07060302u : 0x05040100u) : (r16 & 1 ? 0x07060302u : 0x05040100u);
                const uint32_t x = __builtin_amdgcn_perm(wb, wa, sel);
                va[4 * u][j] = h2bits(kvq_low(x) * d);
                va[4 * u + 1][j] = h2bits(kvq_high(x) * d);
                va[4 * u + 2][j] = h2bits(kvq_low(x >> 8) * d);
                va[4 * u + 3][j] = h2bits(kvq_high(x >> 8) * d);
            }
        }
#pragma unroll
        for (int t = 0; t < QT; t++) {
            if (q0 + t * 16 >= nq) break;
            floatx4 st[2];
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                st[kt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int dc = 0; dc < NDC; dc++)
                    st[kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, ka[kt][dc]),
                                                                    __builtin_bit_cast(half8, S.q[t][dc]), st[kt], 0, 0, 0);
            }
            // bit j: the query sees position key0 + j
            uint32_t vis = 0xffu;
            if (!full) {
                const int m = min(q0 + t * 16 + r16, nq - 1) / p.n_rep;
                vis = 0;
                if (p.mask) {
                    const uint64_t *mk = p.mask + (int64_t)(r0 + m) * p.mask_words;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int x = key0 + j - P;
                        bool see = x < 0;
                        if (x >= 0 && x < n && (x >> 6) < p.mask_words) see = (mk[x >> 6] >> (x & 63)) & 1;
                        vis |= (uint32_t)see << j;
                    }
                } else {
                    const int seen = min(max(P + m + 1 - key0, 0), 8);  // of the lane's 8
                    vis = (1u << seen) - 1u;
                }
            }
            float lmax = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float v = st[j >> 2][j & 3] * sl2;
                if (!full) v = (vis >> j) & 1 ? v : -INFINITY;
                st[j >> 2][j & 3] = v;
                lmax = fmaxf(lmax, v);
            }
            // the maximum moves only for a score above it by more than 8: weights stay below 2^8
            if (__builtin_amdgcn_ballot_w64(lmax > S.m[t] + 8.f) != 0) {
                const float cm = xmax4(lmax);
                if (cm > S.m[t] + 8.f) {
                    const float alpha = __builtin_amdgcn_exp2f(S.m[t] - cm);
                    S.m[t] = cm;
                    S.l[t] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) S.o[t][dt] *= alpha;
                }
            }
            const float mu = S.m[t] == -INFINITY ? 0.f : S.m[t];
            float ps = 0.f, e[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                e[j] = __builtin_amdgcn_exp2f(st[j >> 2][j & 3] - mu);
                ps += e[j];
            }
            S.l[t] += ps;
            uintx4 pk;
#pragma unroll
            for (int j = 0; j < 4; j++) pk[j] = (uint32_t)f2h(e[2 * j]) | ((uint32_t)f2h(e[2 * j + 1]) << 16);
#pragma unroll
            for (int dt = 0; dt < NDT; dt++)
                S.o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, va[dt]),
                                                                    __builtin_bit_cast(half8, pk), S.o[t][dt], 0, 0, 0);
            if (!full && __builtin_amdgcn_ballot_w64(bad != 0) != 0) {
                // NaN groups among the block's values: they reach the queries that see them and no others.
                // Lane (q, g) knows the visibility of its 8 positions; the groups' flags are in lanes with the
                // same g: one flag byte per group e, from lane e * (64 / HD * 8 ...) of this g.
                uint32_t hit = 0;
#pragma unroll
                for (int e2 = 0; e2 < HD / 32; e2++) {
                    const int from = g * 16 + e2 * (16 / (HD / 32));
                    const uint32_t fl = (uint32_t)__shfl((int)bad, from);
                    hit |= (uint32_t)((fl & vis) != 0) << e2;
                }
                hit |= (uint32_t)__shfl_xor((int)hit, 16);
                hit |= (uint32_t)__shfl_xor((int)hit, 32);
                // the lane's accumulators are channels (HD / 4) g ..: group (HD / 4) g / 32
                if ((hit >> (HD == 128 ? g : g >> 1)) & 1) {
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) S.o[t][dt] = floatx4{NAN, NAN, NAN, NAN};
                }
            }
        }
    }
    // the four waves' states, one query tile at a time
#pragma unroll
    for (int t = 0; t < QT; t++) {
        if (q0 + t * 16 >= nq) break;
        const float l = xsum4(S.l[t]);
        if (g == 0) {
            sh_ml[wave][r16][0] = S.m[t];
            sh_ml[wave][r16][1] = l;
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int dt = 0; dt < NDT; dt++) sh_o[wave][r16][(HD / 4) * g + NDT * i + dt] = S.o[t][dt][i];
        __syncthreads();
        // thread: query tq, HD / 16 channels from tc
        const int tq = threadIdx.x >> 4, tc = (threadIdx.x & 15) * (HD / 16);
        const int q = q0 + t * 16 + tq;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kKvqWaves; w++) M = fmaxf(M, sh_ml[w][tq][0]);
        const float Mu = M == -INFINITY ? 0.f : M;
        float lw = 0.f, o[HD / 16];
#pragma unroll
        for (int c = 0; c < HD / 16; c++) o[c] = 0.f;
#pragma unroll
        for (int w = 0; w < kKvqWaves; w++) {
            const float f = __builtin_amdgcn_exp2f(sh_ml[w][tq][0] - Mu);
            lw += sh_ml[w][tq][1] * f;
#pragma unroll
            for (int c = 0; c < HD / 16; c++) o[c] += sh_o[w][tq][tc + c] * f;
        }
        if (q < nq) {
            const int row = r0 + q / p.n_rep, head = h * p.n_rep + q % p.n_rep;
            if (p.nsplit == 1) {
                const float inv = lw == 0.f ? 0.f : 1.f / lw;
                if (p.out_act) {
#pragma unroll
                    for (int c = 0; c < HD / 16; c += 4)
                        *(uintx2 *)(p.out + act_index(row, (int64_t)head * HD + tc + c, (int)p.out_ld, p.out_act == 2)) =
                            uintx2{(uint32_t)f2h(o[c] * inv) | ((uint32_t)f2h(o[c + 2] * inv) << 16),
                                   (uint32_t)f2h(o[c + 1] * inv) | ((uint32_t)f2h(o[c + 3] * inv) << 16)};
                } else {
                    uint16_t *dst = p.out + (int64_t)row * p.out_ld + (int64_t)head * HD + tc;
#pragma unroll
                    for (int c = 0; c < HD / 16; c += 4)
                        *(uintx2 *)(dst + c) = uintx2{(uint32_t)f2h(o[c] * inv) | ((uint32_t)f2h(o[c + 1] * inv) << 16),
                                                      (uint32_t)f2h(o[c + 2] * inv) | ((uint32_t)f2h(o[c + 3] * inv) << 16)};
                }
            } else {
                const int64_t at = ((int64_t)split * p.rows + row) * p.n_heads + head;
                float *po = p.part_o + at * HD + tc;
#pragma unroll
                for (int c = 0; c < HD / 16; c += 4) *(float4 *)(po + c) = float4{o[c], o[c + 1], o[c + 2], o[c + 3]};
                if (tc == 0) {
                    p.part_ml[2 * at] = M;
                    p.part_ml[2 * at + 1] = lw;
                }
            }
        }
        __syncthreads();
    }
}

// One wave per (row, head): the splits in order.
template <int HD> __global__ __launch_bounds__(256) void k_kvq_combine(const KvqAttn p) {
    const int s = blockIdx.y, lane = threadIdx.x & 63;
    int r0, n;
    if (!kvq_seq_rows(p, s, r0, n)) return;
    const int at = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int m = at / p.n_heads, head = at % p.n_heads;
    if (m >= min(n, p.max_rows)) return;
    const int row = r0 + m;
    float M = -INFINITY;
    for (int k = 0; k < p.nsplit; k++) M = fmaxf(M, p.part_ml[2 * (((int64_t)k * p.rows + row) * p.n_heads + head)]);
    const float Mu = M == -INFINITY ? 0.f : M;
    constexpr int C = HD / 64;
    float l = 0.f, o[C] = {};
    for (int k = 0; k < p.nsplit; k++) {
        const int64_t i = ((int64_t)k * p.rows + row) * p.n_heads + head;
        const float f = __builtin_amdgcn_exp2f(p.part_ml[2 * i] - Mu);
        l += p.part_ml[2 * i + 1] * f;
#pragma unroll
        for (int c = 0; c < C; c++) o[c] += p.part_o[i * HD + lane * C + c] * f;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int64_t k = (int64_t)head * HD + lane * C + c;
        p.out[p.out_act ? act_index(row, k, (int)p.out_ld, p.out_act == 2) : (int64_t)row * p.out_ld + k] = f2h(o[c] * inv);
    }
}

// Splits so that the workgroups fill the card about twice, each with at least
// one block for each of its waves.
KvqPlan kvq_attn_plan(int n_heads, int n_kv, int hd, int n_seqs, int max_rows, int64_t max_len, int cus) {
    KvqPlan r{};
    const int nq = max_rows * (n_heads / n_kv);
    r.qt = nq <= 16 ? 1 : nq <= 32 ? 2 : 4;
    r.tiles = (nq + 16 * r.qt - 1) / (16 * r.qt);
    const int64_t groups = (int64_t)r.tiles * n_kv * n_seqs, blocks = (max_len + 31) / 32;
    const int64_t want = (2 * cus + groups - 1) / groups, most = std::max<int64_t>(1, blocks / kKvqWaves);
    r.nsplit = (int)std::max<int64_t>(1, std::min({want, most, (int64_t)64}));
    return r;
}

void launch_kvq_attention(const KvqAttn &in, const KvqPlan &plan, void *ws, hipStream_t st) {
    KvqAttn p = in;
    p.nsplit = plan.nsplit;
    p.qt = plan.qt;
    p.tiles = plan.tiles;
    p.part_o = (float *)ws;
    p.part_ml = p.part_o + (int64_t)p.nsplit * p.rows * p.n_heads * p.L.hd;
    const dim3 g((unsigned)p.nsplit, (unsigned)(p.tiles * p.L.n_kv), (unsigned)p.n_seqs), b(kKvqT);
#define KVQ_ATTN(HD)                                            \
    if (p.qt == 1) k_kvq_attn<HD, 1><<<g, b, 0, st>>>(p);       \
    else if (p.qt == 2) k_kvq_attn<HD, 2><<<g, b, 0, st>>>(p);  \
    else k_kvq_attn<HD, 4><<<g, b, 0, st>>>(p)
    if (p.L.hd == 128) {
        KVQ_ATTN(128);
    } else {
        KVQ_ATTN(64);
    }
#undef KVQ_ATTN
    SD_HIP_CHECK(hipGetLastError());
    if (p.nsplit > 1) {
        const dim3 cg((unsigned)((p.max_rows * p.n_heads + 3) / 4), (unsigned)p.n_seqs);
        if (p.L.hd == 128) k_kvq_combine<128><<<cg, dim3(256), 0, st>>>(p);
        else k_kvq_combine<64><<<cg, dim3(256), 0, st>>>(p);
        SD_HIP_CHECK(hipGetLastError());
    }
}

}  // namespace sd
