// Attention over the 4-bit paged KV cache (sd_kvq.hpp).
//
// Split flash-decoding in two kernels.  A block's codes become fp16 values
// (exactly the values the codes stand for), scores are computed transposed,
// S^T = K Q^T, so that a lane's probabilities are its operand of O^T = V^T P^T,
// and a running maximum and sum in f32 follow the blocks.
//
// Up to 64 queries of a KV head (rows times the heads that share it):
// k_kvq_attn, whose four waves take the blocks of a key range in turn, codes
// straight from memory into registers.  A value costs two VALU operations
// (mask and exponent, then the exact subtraction and the step, two values
// each); with softmax, products, prologue and merge a block of 4.6 KB is some 540
// VALU instructions of a wave for up to 32 queries, 540 cycles of a CU, whose
// share of the memory's rate brings it in 410.
// 5 rows of 32 heads over 8 and 32768 positions, 37.7 MB of blocks: 17 us, 6.2 at
// the rate of a large read.  VALU instructions are issued in 59 % of the CUs' busy
// cycles, matrix instructions take 13 %, and waves wait for 27 % of theirs: each
// has four blocks here, of which it requests one ahead.
// More: k_kvq_wide, whose waves have 32 queries each and share the values of
// 64 positions through LDS, expanded once for up to 256 queries (two key groups
// of 128 queries halve the partial results where the context is short).
// 2048 rows of 32 heads over 8191 positions: 291 us once the clocks have settled
// (307 to 332 in the first ten calls), 825 TFLOP/s; a large product of fp16 matrices
// reaches 1190.  A stage of 64 positions is 2048 cycles of matrix instructions
// and some 2300 of VALU work (253 instructions a wave, 32 of them exponentials)
// on a SIMD, whose two waves overlap them in part: of the CUs' busy cycles the
// matrix pipes take 40 % and VALU instructions 50 %.  A CU has one tile, and causal
// tiles differ in length: the longest is 1.14 times the mean here, 1.94 times in
// the first 2048 positions of a prompt (83 us, 416 TFLOP/s).
// 60 rows over 8192 positions: 29 us, in which the CUs' matrix pipes take 17 %,
// VALU instructions 36 %, and waves wait for 39 % (four stages to a key group).
// Key ranges (splits) meet in k_kvq_combine (60 rows of 32 heads in 16 ranges,
// 16 MB of fp32: 6.1 us; 5 rows in 64 ranges 4.3, most of it latency).
#include <atomic>
#include <type_traits>

#include "sd_kvq_attn_dev.hpp"

#pragma clang fp contract(fast)

namespace sd {

typedef float floatx16 __attribute__((ext_vector_type(16)));

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

// bit j: the V step of position j of the lane's 8 is NaN
__device__ __forceinline__ uint32_t kvq_nan_steps(const uintx4 &vs) {
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        bad |= (uint32_t)((vs[i] & 0x7fffu) > 0x7c00u) << (2 * i);
        bad |= (uint32_t)((vs[i] & 0x7fff0000u) > 0x7c000000u) << (2 * i + 1);
    }
    return bad;
}

// blocks of t positions that the table has pages for
__device__ __forceinline__ int kvq_blocks(const KvqAttn &p, int t) {
    return t > 0 ? (int)min((int64_t)((t - 1) / 32 + 1), (int64_t)p.table_ld << (p.L.page_shift - 5)) : 0;
}
// splits of a sequence of T positions: at least one
__device__ __forceinline__ int kvq_splits(const KvqAttn &p, int T) {
    return min(p.nsplit, max(1, (kvq_blocks(p, T) + p.chunk - 1) / p.chunk));
}

// What a workgroup works on: rows and positions of its sequence, its queries,
// its range of blocks.  False: nothing.
struct KvqWork {
    int r0, n, T, P;  // row i of n is row r0 + i of the call and position P + i
    int nq, q0;       // queries of the KV head, the tile's first
    int t_end, t_all; // positions that some of the tile's rows see end before t_end, all of them see those before t_all
    int b0, b1;       // blocks
};
__device__ __forceinline__ bool kvq_work(const KvqAttn &p, int s, int split, int tile, int tile_q, KvqWork &w) {
    w.T = p.row_start ? p.kv_len[s] : p.len0;
    if (!kvq_seq_rows(p, s, w.r0, w.n)) return false;
    w.nq = min(w.n, p.max_rows) * p.n_rep;
    w.q0 = tile * tile_q;
    if (w.q0 >= w.nq) return false;
    w.P = w.T - w.n;
    const int m_first = w.q0 / p.n_rep, m_last = (min(w.q0 + tile_q, w.nq) - 1) / p.n_rep;
    w.t_end = p.mask ? w.T : min(w.T, w.P + m_last + 1);
    w.t_all = p.mask ? w.P : w.P + m_first + 1;
    // split k: blocks [k chunk, (k + 1) chunk), the last one to the end
    if (split >= kvq_splits(p, w.T)) return false;
    const int nblk = kvq_blocks(p, w.t_end);
    w.b0 = min(split * p.chunk, nblk);
    w.b1 = split == p.nsplit - 1 ? nblk : min(w.b0 + p.chunk, nblk);
    return true;
}

// bit j: row m sees position key0 + j, j < 8
__device__ __forceinline__ uint32_t kvq_visible(const KvqAttn &p, const KvqWork &w, int m, int key0) {
    if (!p.mask) return (1u << min(max(w.P + m + 1 - key0, 0), 8)) - 1u;
    // eight bits from x0 of the row's words: both words they can lie in are loaded at once, whatever x0 is
    const uint64_t *mk = p.mask + (int64_t)(w.r0 + m) * p.mask_words;
    const int x0 = key0 - w.P, a = x0 >> 6, s = x0 & 63, left = w.n - x0;
    const uint64_t w0 = mk[min(max(a, 0), p.mask_words - 1)], w1 = mk[min(max(a + 1, 0), p.mask_words - 1)];
    const uint64_t lo = a >= 0 && a < p.mask_words ? w0 : 0, hi = a + 1 >= 0 && a + 1 < p.mask_words ? w1 : 0;
    uint32_t vis = (uint32_t)(lo >> s | (hi << 1) << (63 - s)) & 0xffu;
    if (left < 8) vis &= (1u << max(left, 0)) - 1u;
    if (x0 < 0) vis |= (1u << min(-x0, 8)) - 1u;  // the prefix
    return vis;
}

// bit j: row m sees position key0 + j, j < 64
__device__ __forceinline__ uint64_t kvq_visible64(const KvqAttn &p, const KvqWork &w, int m, int key0) {
    if (!p.mask) {
        const int n = w.P + m + 1 - key0;
        return n >= 64 ? ~0ull : (1ull << max(n, 0)) - 1u;
    }
    const uint64_t *mk = p.mask + (int64_t)(w.r0 + m) * p.mask_words;
    const int x0 = key0 - w.P, a = x0 >> 6, s = x0 & 63, left = w.n - x0;
    const uint64_t w0 = mk[min(max(a, 0), p.mask_words - 1)], w1 = mk[min(max(a + 1, 0), p.mask_words - 1)];
    const uint64_t lo = a >= 0 && a < p.mask_words ? w0 : 0, hi = a + 1 >= 0 && a + 1 < p.mask_words ? w1 : 0;
    uint64_t vis = lo >> s | (hi << 1) << (63 - s);
    if (left < 64) vis &= (1ull << max(left, 0)) - 1u;
    if (x0 < 0) vis |= x0 <= -64 ? ~0ull : (1ull << -x0) - 1u;  // the prefix
    return vis;
}

// ---- up to 64 queries, 16 or 32 to a workgroup ------------------------------------
template <int HD, int QT>
__global__ __launch_bounds__(kKvqT) __attribute__((amdgpu_waves_per_eu(2))) void k_kvq_attn(const KvqAttn p) {
    constexpr int NDC = HD / 32, NDT = HD / 16;
    __shared__ float sh_o[kKvqWaves][16][HD];
    __shared__ float sh_ml[kKvqWaves][16][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, g = lane >> 4;
    const KvqPlace at = kvq_place(p);
    const int split = at.split, h = at.h;
    const int pg0 = kvq_page(p, at.s, split * p.chunk + wave + lane * kKvqWaves);
    KvqWork W;
    if (!kvq_work(p, at.s, split, at.tile, QT * 16, W)) return;

    uintx4 qf[QT][NDC];
    floatx4 o[QT][NDT];
    float m[QT], l[QT];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const uint16_t *qr = kvq_query(p, W, h, W.q0 + t * 16 + r16);
#pragma unroll
        for (int dc = 0; dc < NDC; dc++) qf[t][dc] = *(const uintx4 *)(qr + 8 * (g * NDC + dc));
#pragma unroll
        for (int dt = 0; dt < NDT; dt++) o[t][dt] = floatx4{0.f, 0.f, 0.f, 0.f};
        m[t] = -INFINITY;
        l[t] = 0.f;
    }
    const float sl2 = p.scale * 1.4426950408889634f;  // scores in base-2 units
    const int steps = (W.b1 - W.b0 - wave + kKvqWaves - 1) / kKvqWaves;  // blocks b0 + wave + 4 i
    // lane i holds the page of step i of 64; -1: holds no positions
    auto pages = [&](int i0, int pg) { return i0 + lane < steps && pg >= 0 && pg < p.L.n_pages ? pg : -1; };
    auto fetch = [&](KvqStep<HD> &k, int i, int page) {
        if (page >= 0) kvq_load<HD>(k, p.L.block(page, h, (W.b0 + wave + i * kKvqWaves) * 32), lane);
    };
    int pg = pages(0, pg0);
    KvqStep<HD> next{};
    int page = __builtin_amdgcn_readlane(pg, 0);
    if (steps > 0) fetch(next, 0, page);
    for (int i = 0; i < steps; i++) {
        KvqStep<HD> k = next;
        const bool have = page >= 0;
        if (i + 1 < steps) {
            if (((i + 1) & 63) == 0) pg = pages(i + 1, kvq_page(p, at.s, W.b0 + wave + (i + 1 + lane) * kKvqWaves));
            page = __builtin_amdgcn_readlane(pg, (i + 1) & 63);
            fetch(next, i + 1, page);
        }
        if (!have) continue;
        const int b = W.b0 + wave + i * kKvqWaves, key0 = b * 32 + 8 * g;
        const bool full = b * 32 + 32 <= W.t_all && b * 32 + 32 <= W.T;
        float st[QT][8];
        {
            const uint32_t k0 = k.ks & 0xffffu, k1 = k.ks >> 16;
            const half2v d0 = __builtin_bit_cast(half2v, k0 | (k0 << 16)), d1 = __builtin_bit_cast(half2v, k1 | (k1 << 16));
            floatx4 acc[QT][2];
#pragma unroll
            for (int t = 0; t < QT; t++) acc[t][0] = acc[t][1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int dc = 0; dc < NDC; dc++) {
                const half8 a0 = __builtin_bit_cast(half8, kvq_expand_k(k.kc[0][dc], d0));
                const half8 a1 = __builtin_bit_cast(half8, kvq_expand_k(HD == 128 ? k.kc[HD / 64 - 1][dc] : k.kc[0][2 + dc], d1));
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    acc[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, __builtin_bit_cast(half8, qf[t][dc]), acc[t][0], 0, 0, 0);
                    acc[t][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, __builtin_bit_cast(half8, qf[t][dc]), acc[t][1], 0, 0, 0);
                }
            }
#pragma unroll
            for (int t = 0; t < QT; t++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    // rounded here, not inside the weight: beyond 2^28 the rounding is more than fp16 has room for, so what is
                    // weighed must be what the maximum is taken of
#pragma clang fp contract(off)
                    st[t][j] = acc[t][j >> 2][j & 3] * sl2;
                }
        }
        uint32_t bad = 0, vis[QT];
        if (!full) {
            bad = kvq_nan_steps(k.vs);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (bad >> (2 * j) & 1) k.vs[j] &= 0xffff0000u;
                if (bad >> (2 * j + 1) & 1) k.vs[j] &= 0x0000ffffu;
            }
#pragma unroll
            for (int t = 0; t < QT; t++) {
                vis[t] = kvq_visible(p, W, min(W.q0 + t * 16 + r16, W.nq - 1) / p.n_rep, key0);
#pragma unroll
                for (int j = 0; j < 8; j++) st[t][j] = (vis[t] >> j) & 1 ? st[t][j] : -INFINITY;
            }
        }
        uintx4 pk[QT];
#pragma unroll
        for (int t = 0; t < QT; t++) {
            float top = st[t][0];
#pragma unroll
            for (int j = 1; j < 8; j++) top = fmaxf(top, st[t][j]);
            // The reference moves only for a score that would weigh more than 2^15.  By the difference, which is exact for
            // neighbouring scores: beyond 2^27 the reference and 15 add up to the score that is 16 above it.
            if (__builtin_amdgcn_ballot_w64(top - m[t] > 15.f) != 0) {
                const float tm = xmax4(top);
                if (tm - m[t] > 15.f) {
                    const float cm = tm - kKvqHead, alpha = __builtin_amdgcn_exp2f(m[t] - cm);
                    m[t] = cm;
                    l[t] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) o[t][dt] *= alpha;
                }
            }
            pk[t] = kvq_weights(st[t], m[t] == -INFINITY ? 0.f : m[t], l[t]);
        }
        // V operands: a position pair's nibbles n are channels n (hd 128) or 4 (r16 & 1) + n (64) of the lane's word
#pragma unroll
        for (int u = 0; u < NDT / 4; u++) {
            uintx4 va[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t wa = k.vc[j >> 1][(2 * j) & 3], wb = k.vc[j >> 1][(2 * j + 1) & 3];
                const half2v d = __builtin_bit_cast(half2v, (uint32_t)k.vs[j]);
                const uint32_t sel = HD == 128 ? (u ? 0x07060302u : 0x05040100u) : (r16 & 1 ? 0x07060302u : 0x05040100u);
                const uint32_t x = __builtin_amdgcn_perm(wb, wa, sel);
                va[0][j] = h2bits(kvq_low(x) * d);
                va[1][j] = h2bits(kvq_high(x) * d);
                va[2][j] = h2bits(kvq_low(x >> 8) * d);
                va[3][j] = h2bits(kvq_high(x >> 8) * d);
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int t = 0; t < QT; t++)
                    o[t][4 * u + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        __builtin_bit_cast(half8, va[e]), __builtin_bit_cast(half8, pk[t]), o[t][4 * u + e], 0, 0, 0);
        }
        if (!full && __builtin_amdgcn_ballot_w64(bad != 0) != 0) {
            // NaN groups among the block's values reach the queries that see them and no others.  Lane (q, g) knows what
            // q sees of the positions 8 g ..; their flags for group e are in the lanes of the same g with its words.
#pragma unroll
            for (int t = 0; t < QT; t++) {
                uint32_t hit = 0;
#pragma unroll
                for (int e = 0; e < HD / 32; e++)
                    hit |= (uint32_t)(((uint32_t)__shfl((int)bad, g * 16 + e * (512 / HD)) & vis[t]) != 0) << e;
                hit |= (uint32_t)__shfl_xor((int)hit, 16);
                hit |= (uint32_t)__shfl_xor((int)hit, 32);
                // the lane's accumulators are channels (HD / 4) g ..: group (HD / 4) g / 32
                if ((hit >> (HD == 128 ? g : g >> 1)) & 1) {
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) o[t][dt] = floatx4{NAN, NAN, NAN, NAN};
                }
            }
        }
    }
    // the four waves' states, one query tile at a time
#pragma unroll
    for (int t = 0; t < QT; t++) {
        if (W.q0 + t * 16 >= W.nq) break;
        const float lq = xsum4(l[t]);
        if (g == 0) {
            sh_ml[wave][r16][0] = m[t];
            sh_ml[wave][r16][1] = lq;
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int dt = 0; dt < NDT; dt += 4)
                *(floatx4 *)&sh_o[wave][r16][(HD / 4) * g + NDT * i + dt] =
                    floatx4{o[t][dt][i], o[t][dt + 1][i], o[t][dt + 2][i], o[t][dt + 3][i]};
        __syncthreads();
        // thread: query tq, HD / 16 channels from tc
        const int tq = threadIdx.x >> 4, tc = (threadIdx.x & 15) * (HD / 16), q = W.q0 + t * 16 + tq;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kKvqWaves; w++) M = fmaxf(M, sh_ml[w][tq][0]);
        const float Mu = M == -INFINITY ? 0.f : M;
        float lw = 0.f, oc[HD / 16];
#pragma unroll
        for (int c = 0; c < HD / 16; c++) oc[c] = 0.f;
#pragma unroll
        for (int w = 0; w < kKvqWaves; w++) {
            const float f = __builtin_amdgcn_exp2f(sh_ml[w][tq][0] - Mu);
            lw += sh_ml[w][tq][1] * f;
#pragma unroll
            for (int c = 0; c < HD / 16; c++) oc[c] += sh_o[w][tq][tc + c] * f;
        }
        if (q < W.nq) kvq_emit<HD / 16>(p, split, W.r0 + q / p.n_rep, h * p.n_rep + q % p.n_rep, tc, oc, M, lw, tc == 0);
        __syncthreads();
    }
}

// ---- more ------------------------------------------------------------------------
// NW waves of 32 queries (32x32x16 MFMA: column = query).  Stages of two blocks
// go through LDS as operands, 1 KiB each: lane r + 32 h of an operand holds 8
// values.  K, chunk c of 16 channels: row r (position k with bits 2 and 3
// exchanged), channels 16 c + 8 h ..; so a lane's scores 8 c .. 8 c + 7 are the
// positions 16 c + 8 h ..  V, tile tt and chunk c of 16 positions: positions
// 16 c + 8 h .. of channel (hd 128) 8 (r >> 1) + 2 tt + (r & 1) or (64)
// 8 (r >> 2) + 4 tt + (r & 3): the channels of a word are rows next to each other.
// A stage is expanded by all waves while the one before it is multiplied (two
// buffers, one barrier a stage).
constexpr int kMfma = 0x008, kDsRead = 0x100, kValu = 0x402;  // instruction classes of a scheduling group
template <int HD> struct KvqStage {
    uintx4 k[2][HD / 16][64];  // [block][chunk][lane]
    uintx4 v[2][HD / 16][64];  // [block][2 tile + chunk][lane]
    __align__(16) uint32_t bad[2][HD / 32];  // [block][group]: positions whose values are NaN (held as 0)
};

// A unit of a stage: 0, 1 the K halves of block 0 (kt), 2, 3 its V halves, 4 .. 7 block 1's.
template <int HD> struct KvqUnit {
    uintx4 a, b, s;
};

template <int HD, int NW, int KG>
__global__ __launch_bounds__(64 * NW * KG) __attribute__((amdgpu_waves_per_eu(2))) void k_kvq_wide(const KvqAttn p) {
    constexpr int NC = HD / 16, NT = HD / 32, NU = 8 / NW;
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 63, id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r32 = lane & 31, hh = lane >> 5;
    const int wave = id % NW, kg = id / NW;
    KvqStage<HD> *stage = (KvqStage<HD> *)smem + 2 * kg;
    const KvqPlace at = kvq_place(p);
    const int split = at.split, h = at.h;
    int pages = kvq_page(p, at.s, split * p.chunk + lane);
    KvqWork W;
    if (!kvq_work(p, at.s, split, at.tile, NW * 32, W)) return;
    const int q0 = W.q0 + wave * 32;            // this wave's queries
    const bool idle = q0 >= W.nq;
    const int m_first = min(q0, W.nq - 1) / p.n_rep, m_last = (min(q0 + 32, W.nq) - 1) / p.n_rep;
    const int t_end = p.mask ? W.T : min(W.T, W.P + m_last + 1), t_all = p.mask ? W.P : min(W.T, W.P + m_first + 1);
    const int my_m = min(q0 + r32, W.nq - 1) / p.n_rep;

    uintx4 qf[NC];
    const uint16_t *qr = kvq_query(p, W, h, q0 + r32);
#pragma unroll
    for (int c = 0; c < NC; c++) qf[c] = *(const uintx4 *)(qr + 16 * c + 8 * hh);
    floatx16 o[NT];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[t][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float sl2 = p.scale * 1.4426950408889634f;  // scores in base-2 units
    const int all = (W.b1 - W.b0 + 1) / 2, stages = (all - kg + KG - 1) / KG;  // the range's and this key group's

    // in `pages` lane k holds the page of block b0 + 64 j + k; -1: holds no positions
    KvqUnit<HD> un[NU];
    int page[2] = {-1, -1};  // of the stage in un
    auto fetch = [&](int n) {
        const int i = n * KG + kg;
        if ((i & 31) < KG) {
            const int b = W.b0 + 2 * (i & ~31) + lane;
            if (n > 0) pages = kvq_page(p, at.s, b);
            pages = b < W.b1 && pages >= 0 && pages < p.L.n_pages ? pages : -1;
        }
        page[0] = __builtin_amdgcn_readlane(pages, 2 * i & 63);
        page[1] = __builtin_amdgcn_readlane(pages, (2 * i + 1) & 63);
#pragma unroll
        for (int u = 0; u < NU; u++) {
            const int id = wave * NU + u, blk = id >> 2, part = id & 3;
            const int pg = blk ? page[1] : page[0];
            if (pg < 0) continue;
            const uint8_t *base = p.L.block(pg, h, (W.b0 + 2 * i + blk) * 32);
            if (part < 2) {
                // K half: position rows of key tile `part`; the lane's (rho, lane group) as stored
                const int rho = lane & 15, g = lane >> 4;
                if constexpr (HD == 128) {
                    un[u].a = *(const uintx4 *)(base + part * 1024 + lane * 16);
                    un[u].s.x = *(const uint16_t *)(base + 16 * HD + (rho + 16 * g) * 4 + 2 * part);
                } else {
                    const uintx2 w = *(const uintx2 *)(base + lane * 16 + 8 * part);
                    un[u].a = uintx4{w.x, w.y, 0, 0};
                    un[u].s.x = *(const uint16_t *)(base + 16 * HD + (rho + 16 * (g >> 1)) * 4 + 2 * part);
                }
            } else {
                // V half: hd 128: word lane & 15, positions 8 (lane >> 4) ..; 64: word lane & 7, positions 8 ((lane >> 3) & 3) ..
                const int w = HD == 128 ? lane & 15 : lane & 7, g = HD == 128 ? lane >> 4 : (lane >> 3) & 3;
                const uint8_t *v = base + 18 * HD + (w + (HD / 8) * g) * 32;
                un[u].a = *(const uintx4 *)v;
                un[u].b = *(const uintx4 *)(v + 16);
                un[u].s = *(const uintx4 *)(base + 34 * HD + ((w >> 2) * 4 + g) * 16);
            }
        }
    };
    auto expand = [&](KvqStage<HD> &S) {
#pragma unroll
        for (int u = 0; u < NU; u++) {
            const int id = wave * NU + u, blk = id >> 2, part = id & 3;
            if ((blk ? page[1] : page[0]) < 0) {
                // nobody sees the positions: their weights are 0, and so must the values be
                if (part == 2 && lane < HD / 32) S.bad[blk][lane] = 0;
                if (part >= 2)
                    for (int e = 0; e < HD / 32; e++) S.v[blk][(part - 2) * (HD / 32) + e][lane] = uintx4{0, 0, 0, 0};
                continue;
            }
            if (part < 2) {
                const int rho = lane & 15, g = lane >> 4;
                // position 8 (rho >> 2) + 4 part + (rho & 3) is row 16 (rho >> 3) + 8 part + 4 ((rho >> 2) & 1) + (rho & 3)
                const int row = 16 * (rho >> 3) + 8 * part + 4 * ((rho >> 2) & 1) + (rho & 3);
                const uint32_t s = un[u].s.x & 0xffffu;
                const half2v d = __builtin_bit_cast(half2v, s | (s << 16));
#pragma unroll
                for (int e = 0; e < HD / 32; e++) {
                    const int w = g * (HD / 32) + e;  // channels 8 w ..: chunk w >> 1, half w & 1
                    S.k[blk][w >> 1][row + 32 * (w & 1)] = kvq_expand_k(un[u].a[e], d);
                }
            } else {
                const int w = HD == 128 ? lane & 15 : lane & 7, g = HD == 128 ? lane >> 4 : (lane >> 3) & 3;
                const uint32_t bad = kvq_nan_steps(un[u].s);
                if (bad) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if (bad >> (2 * j) & 1) un[u].s[j] &= 0xffff0000u;
                        if (bad >> (2 * j + 1) & 1) un[u].s[j] &= 0x0000ffffu;
                    }
                }
                if (part == 2 && (w & 3) == 0 && (HD == 128 || lane < 32)) ((uint8_t *)&S.bad[blk][w >> 2])[g] = (uint8_t)bad;
                // nibbles 4 (part - 2) .. of the words; hd 64 gives each half of the wave two of them
                const uint32_t sel = part == 3 ? 0x07060302u : 0x05040100u;
                uintx4 va[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uintx4 &x4 = j < 2 ? un[u].a : un[u].b;
                    const uint32_t x = __builtin_amdgcn_perm(x4[(2 * j + 1) & 3], x4[(2 * j) & 3], sel);
                    const half2v d = __builtin_bit_cast(half2v, (uint32_t)un[u].s[j]);
                    va[0][j] = h2bits(kvq_low(x) * d);
                    va[1][j] = h2bits(kvq_high(x) * d);
                    va[2][j] = h2bits(kvq_low(x >> 8) * d);
                    va[3][j] = h2bits(kvq_high(x >> 8) * d);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int n = 4 * (part - 2) + e;  // nibble: hd 128: tile n >> 1, row 2 w + (n & 1); 64: tile n >> 2, row 4 w + (n & 3)
                    const int tt = HD == 128 ? n >> 1 : n >> 2, row = HD == 128 ? 2 * w + (n & 1) : 4 * w + (n & 3);
                    if (HD == 128 || lane < 32) S.v[blk][2 * tt + (g >> 1)][row + 32 * (g & 1)] = va[e];
                }
            }
        }
    };
    const float hidden = sl2 < 0.f ? INFINITY : -INFINITY;  // a masked score before it is scaled
    // a block's scores move their query's reference
    auto raise = [&](const floatx16 &st) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 16; j++) top = fmaxf(top, st[j] * sl2);
        const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        const float cm = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])) - kKvqHead;
        if (cm > m) {
            const float alpha = __builtin_amdgcn_exp2f(m - cm);
            m = cm;
            l *= alpha;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int j = 0; j < 16; j++) o[t][j] *= alpha;
        }
    };
    // fp16 weights of a block's scores and their sum; with `rounded` of the scaled scores as raise() compares them, else in
    // one fused operation each
    auto weigh = [&](const floatx16 &st, uintx4 (&pk)[2], auto rounded) {
        const float mu = m == -INFINITY ? 0.f : m;
        float sum = 0.f;
        auto weight = [&](float s) {
#pragma clang fp contract(off)
            return __builtin_amdgcn_exp2f(decltype(rounded)::value ? s * sl2 - mu : __builtin_fmaf(s, sl2, -mu));
        };
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float x = weight(st[8 * c + 2 * j]), y = weight(st[8 * c + 2 * j + 1]);
                sum += x + y;
                pk[c][j] = h2bits(half2v{(_Float16)x, (_Float16)y});
            }
        return sum;
    };
    // A stage: the products of one block run beside the softmax of the other.  No maximum is looked for: a query
    // keeps the reference of its first block until its weights add up to more than 2^15 in half a block (they stay
    // below fp16's range); then the reference is raised and they are taken again.  A fused weight is of the unrounded
    // score, which beyond 2^28 may lie more than 16 from the rounded one that the reference came from, past fp16's end
    // on either side: where the reference is beyond 2^24, weights are always taken again, of the rounded scores.
    constexpr float kMost = 32768.f, kFused = 16777216.f;
    auto multiply = [&](const KvqStage<HD> &S, int base, bool first, bool second) {
        const bool full = first && second && base + 64 <= t_all;
        floatx16 st[2];
        uintx4 pk[2][2];
        uint64_t seen = ~0ull;  // bit j: the lane's query sees position base + j
        if (!full) seen = kvq_visible64(p, W, my_m, base) & ((first ? 0xffffffffull : 0) | (second ? 0xffffffffull << 32 : 0));
#pragma unroll
        for (int j = 0; j < 16; j++) st[0][j] = st[1][j] = 0.f;
        auto mask = [&](int blk) {
            if (full) return;
            const uint32_t vis = (uint32_t)(seen >> (32 * blk + 8 * hh));
#pragma unroll
            for (int j = 0; j < 16; j++) st[blk][j] = (vis >> (j + (j & 8))) & 1 ? st[blk][j] : hidden;
        };
        auto scores = [&](int blk) {
#pragma unroll
            for (int c = 0; c < NC; c++)
                st[blk] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, S.k[blk][c][lane]),
                                                                 __builtin_bit_cast(half8, qf[c]), st[blk], 0, 0, 0);
        };
        auto values = [&](int blk) {
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int t = 0; t < NT; t++)
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, S.v[blk][2 * t + c][lane]),
                                                                  __builtin_bit_cast(half8, pk[blk][c]), o[t], 0, 0, 0);
        };
        // scores of block 0, its operands requested four ahead
        __builtin_amdgcn_sched_barrier(0);
        scores(0);
        __builtin_amdgcn_sched_group_barrier(kDsRead, 4, 0);
#pragma unroll
        for (int c = 0; c < NC - 4; c++) {
            __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kMfma, 4, 0);
        __builtin_amdgcn_sched_barrier(0);
        mask(0);
        // scores of block 1 beside the weights of block 0
        __builtin_amdgcn_sched_barrier(0);
        scores(1);
        float sum = weigh(st[0], pk[0], std::false_type{});
        __builtin_amdgcn_sched_group_barrier(kDsRead, 4, 0);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kValu, 56 / NC, 0);
            if (c + 4 < NC) __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (__builtin_amdgcn_ballot_w64(sum > kMost || !(fabsf(m) < kFused)) != 0) {
            raise(st[0]);
            sum = weigh(st[0], pk[0], std::true_type{});
        }
        l += sum;
        mask(1);
        // values of block 0 beside the weights of block 1
        __builtin_amdgcn_sched_barrier(0);
        values(0);
        sum = weigh(st[1], pk[1], std::false_type{});
        __builtin_amdgcn_sched_group_barrier(kDsRead, 4, 0);
#pragma unroll
        for (int c = 0; c < 2 * NT; c++) {
            __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kValu, 56 / (2 * NT), 0);
            if (c + 4 < 2 * NT) __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (__builtin_amdgcn_ballot_w64(sum > kMost || !(fabsf(m) < kFused)) != 0) {
            raise(st[1]);
            sum = weigh(st[1], pk[1], std::true_type{});
        }
        l += sum;
        __builtin_amdgcn_sched_barrier(0);
        values(1);
        uintx4 bad[2];
        if constexpr (HD == 128) {
            bad[0] = *(const uintx4 *)S.bad[0], bad[1] = *(const uintx4 *)S.bad[1];
        } else {
            const uintx4 b = *(const uintx4 *)S.bad[0];
            bad[0] = uintx4{b.x, b.y, 0, 0}, bad[1] = uintx4{b.z, b.w, 0, 0};
        }
        __builtin_amdgcn_sched_group_barrier(kDsRead, 4, 0);
#pragma unroll
        for (int c = 0; c < 2 * NT - 3; c++) {
            __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kMfma, 3, 0);
        __builtin_amdgcn_sched_barrier(0);
        // NaN groups among the values reach the queries that see them
        uint32_t any = 0;
#pragma unroll
        for (int e = 0; e < HD / 32; e++) any |= bad[0][e] | bad[1][e];
        if (__builtin_amdgcn_readfirstlane(any) != 0) {
#pragma unroll
            for (int blk = 0; blk < 2; blk++) {
#pragma unroll
                for (int e = 0; e < HD / 32; e++)
                    if (bad[blk][e] & (uint32_t)(seen >> (32 * blk))) {
                        // accumulator j of any tile is a channel of word (hd 128) 4 (j >> 2) + 2 hh + ((j >> 1) & 1),
                        // (64) 2 (j >> 2) + hh
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            const int w = HD == 128 ? 4 * (j >> 2) + 2 * hh + ((j >> 1) & 1) : 2 * (j >> 2) + hh;
                            if (w >> 2 == e)
#pragma unroll
                                for (int t = 0; t < NT; t++) o[t][j] = NAN;
                        }
                    }
            }
        }
    };
    // In an interval stage i is multiplied, stage i + 1 expanded and stage i + 2 requested.  Half of the waves, one of the
    // two of a SIMD, expand first: the matrix instructions of one wave then run beside the other's VALU work (2048 rows
    // over 8191 positions: 3 % less time than with all expanding first).
    const bool early = NW * KG == 8 && id >= 4;
    int now = 0, next = 0;  // bit b: block b of the stage holds positions
    if (stages > 0) fetch(0);
    auto prepare = [&](int i) {
        if (i + 1 >= stages) return;
        next = (page[0] >= 0) | (page[1] >= 0) << 1;
        expand(stage[(i + 1) & 1]);
        if (i + 2 < stages) fetch(i + 2);
    };
    for (int i = -1; i < (all + KG - 1) / KG; i++) {
        if (early) prepare(i);
        const int base = (W.b0 + 2 * (i * KG + kg)) * 32;
        if (i >= 0 && i < stages && !idle && now && base < t_end) multiply(stage[i & 1], base, now & 1, now >> 1);
        if (!early) prepare(i);
        now = next;
        __syncthreads();
    }
    if constexpr (KG == 2) {
        // group 1's state goes to the wave of group 0 with the same queries, lane to lane
        float4 *box = (float4 *)smem + wave * 64 * (4 * NT + 1) + lane;
        if (kg == 1) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    box[64 * (4 * t + i)] = float4{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
            box[64 * 4 * NT] = float4{m, l, 0.f, 0.f};
        }
        __syncthreads();
        if (kg == 1) return;
        const float4 ml = box[64 * 4 * NT];
        const float M = fmaxf(m, ml.x), Mu = M == -INFINITY ? 0.f : M;
        const float f0 = __builtin_amdgcn_exp2f(m - Mu), f1 = __builtin_amdgcn_exp2f(ml.x - Mu);
        m = M;
        l = l * f0 + ml.y * f1;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float4 b = box[64 * (4 * t + i)];
                o[t][4 * i] = o[t][4 * i] * f0 + b.x * f1;
                o[t][4 * i + 1] = o[t][4 * i + 1] * f0 + b.y * f1;
                o[t][4 * i + 2] = o[t][4 * i + 2] * f0 + b.z * f1;
                o[t][4 * i + 3] = o[t][4 * i + 3] * f0 + b.w * f1;
            }
    }
    if (idle) return;
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    const int q = q0 + r32;
    if (q >= W.nq) return;
    const int row = W.r0 + q / p.n_rep, head = h * p.n_rep + q % p.n_rep;
    // word w's 8 channels: hd 128: tiles 0 .. 3 of accumulators j, j + 1 (j even); 64: tiles 0, 1 of four accumulators
    auto words = [&](auto &&put) {
#pragma unroll
        for (int j = 0; j < 16; j += HD == 128 ? 2 : 4) {
            float oc[8];
#pragma unroll
            for (int n = 0; n < 8; n++) oc[n] = HD == 128 ? o[n >> 1][j + (n & 1)] : o[(n >> 2) % NT][(j + (n & 3)) & 15];
            put((HD == 128 ? 4 * (j >> 2) + ((j >> 1) & 1) : 2 * (j >> 2)) * 8, oc);
        }
    };
    const int c0 = (HD == 128 ? 2 : 1) * 8 * hh;  // the lane's first channel
    if (p.nsplit > 1) {
        const int64_t i = ((int64_t)split * p.rows + row) * p.n_heads + head;
        float *po = p.part_o + i * HD + c0;
        words([&](int c, const float (&oc)[8]) {
            *(float4 *)(po + c) = float4{oc[0], oc[1], oc[2], oc[3]};
            *(float4 *)(po + c + 4) = float4{oc[4], oc[5], oc[6], oc[7]};
        });
        if (hh == 0) *(float2 *)(p.part_ml + 2 * i) = float2{m, l};
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    words([&](int c, const float (&oc)[8]) { kvq_put<8>(p, row, (int64_t)head * HD + c0 + c, oc, inv); });
}

// ---- the splits ------------------------------------------------------------------
// One workgroup per (row, head): every wave knows all weights (lane k: split
// k's) and takes a part of the splits, HD / 4 lanes to a split, four loads in
// flight; the first of them go out with those of the maxima and sums.
template <int HD> __global__ __launch_bounds__(256) void k_kvq_combine(const KvqAttn p) {
    constexpr int LS = HD / 4, N = 256 / LS, U = 4;  // lanes of a split, splits of a round, rounds in flight
    __shared__ __align__(16) float sh[N][HD];
    const int s = blockIdx.y, lane = threadIdx.x & 63, mine = threadIdx.x / LS, c = threadIdx.x % LS * 4;
    const int T = p.row_start ? p.kv_len[s] : p.len0;
    int r0, n;
    if (!kvq_seq_rows(p, s, r0, n)) return;
    const int mr = blockIdx.x / p.n_heads, head = blockIdx.x % p.n_heads;
    if (mr >= min(n, p.max_rows)) return;
    const int row = r0 + mr, ns = kvq_splits(p, T);
    const int64_t at = (int64_t)row * p.n_heads + head, step = (int64_t)p.rows * p.n_heads;
    const float2 ml = lane < ns ? *(const float2 *)(p.part_ml + 2 * (at + lane * step)) : float2{-INFINITY, 0.f};
    float4 v[U];
    auto load = [&](int k0) {
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = *(const float4 *)(p.part_o + (at + min(k0 + u * N + mine, ns - 1) * step) * HD + c);
    };
    load(0);
    float M = ml.x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    const float f = lane < ns ? __builtin_amdgcn_exp2f(ml.x - (M == -INFINITY ? 0.f : M)) : 0.f;
    float l = ml.y * f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
    float4 acc{0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < ns; k0 += U * N) {
        if (k0 > 0) load(k0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = k0 + u * N + mine;
            const float w = __shfl(f, k & 63);
            if (k < ns) acc.x += v[u].x * w, acc.y += v[u].y * w, acc.z += v[u].z * w, acc.w += v[u].w * w;
        }
    }
    *(float4 *)&sh[mine][c] = acc;
    __syncthreads();
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int d = threadIdx.x;
    if (d < HD) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) x += sh[i][d];
        const int64_t k = (int64_t)head * HD + d;
        p.out[p.out_act ? act_index(row, k, (int)p.out_ld, p.out_act == 2) : (int64_t)row * p.out_ld + k] = f2h(x * inv);
    }
}

// Queries of a KV head: up to 64 in tiles of 16 or 32 of the small kernel, which
// for two tiles expands every value twice but waits for no LDS (a decoder's pass
// of 16 rows, 32 heads over 8, 8 layers: 32768 positions 858 us, 120000 1199; in
// a tile of 64 of the wide kernel 959 and 1438, of 128 946 and 1459).
// More: tiles of 256 expand every value once but leave, with the splits
// that a short context needs to fill the card, twice the partial results of
// tiles of 128 in two key groups.  They are taken where they fill the card alone
// or a split is more than 12 blocks long (a decoder's pass of 60 rows, 32 heads
// over 8, 8 layers: 8192 positions 1113 us with 128 and 1126 with 256, 32768
// 1451 and 1394).
// Splits: the wide kernel's workgroup has a CU to itself, the small one's four
// waves share it with another (8 layers of 32 heads over 8, 120000 positions, one
// row: a pass of 720 us, 763 with one to a CU; 32768 positions, 5 rows: no
// difference).  In a batch the lengths differ, so four times as many ranges even
// the load (16 sequences of up to 9001 positions: 17.6 us, 19.2 without).  No
// range is shorter than a block for each wave.
KvqPlan kvq_attn_plan(int n_heads, int n_kv, int hd, int n_seqs, int max_rows, int64_t max_len, int cus) {
    KvqPlan r{};
    const int64_t nq = (int64_t)max_rows * (n_heads / n_kv);
    const int64_t blocks = (max_len + 31) / 32, big = (nq + 255) / 256 * n_kv * n_seqs;
    r.tile_q = nq <= 16 ? 16 : nq <= 64 ? 32 : nq > 128 && (big >= cus || big * blocks > 12 * cus) ? 256 : 128;
    r.tiles = (int)((nq + r.tile_q - 1) / r.tile_q);
    const int64_t groups = (int64_t)r.tiles * n_kv * n_seqs;
    const int64_t fill = r.tile_q > 32 ? cus : n_seqs > 1 ? 8 * cus : 2 * cus;
    int64_t want = (fill + groups - 1) / groups, most = std::max<int64_t>(1, blocks / 4);
    r.nsplit = (int)std::max<int64_t>(1, std::min({want, most, (int64_t)64}));
    r.chunk = (int)std::max<int64_t>(1, (blocks + r.nsplit - 1) / r.nsplit);
    return r;
}

template <int HD, int NW, int KG> static void launch_wide(const KvqAttn &p, hipStream_t st) {
    constexpr int lds = 2 * KG * (int)sizeof(KvqStage<HD>);
    static_assert(lds <= 160 * 1024, "two stages of each key group in LDS");
    static_assert(KG == 1 || NW * 64 * (HD / 8 + 1) * 16 <= lds, "a key group's state in LDS");
    if constexpr (lds > 64 * 1024) {
        static std::atomic<uint64_t> done{0};  // bit per device
        int dev = 0;
        SD_HIP_CHECK(hipGetDevice(&dev));
        const uint64_t bit = 1ull << (dev & 63);
        if (!(done.load(std::memory_order_acquire) & bit) || dev > 63) {
            SD_HIP_CHECK(hipFuncSetAttribute((const void *)k_kvq_wide<HD, NW, KG>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
            done.fetch_or(bit, std::memory_order_release);
        }
    }
    k_kvq_wide<HD, NW, KG><<<dim3((unsigned)(p.nsplit * p.groups)), dim3(64 * NW * KG), lds, st>>>(p);
}

template <int HD> static void launch_attn(const KvqAttn &p, hipStream_t st) {
    const dim3 g((unsigned)(p.nsplit * p.groups)), b(kKvqT);
    switch (p.tile_q) {
    case 16: k_kvq_attn<HD, 1><<<g, b, 0, st>>>(p); break;
    case 32: k_kvq_attn<HD, 2><<<g, b, 0, st>>>(p); break;
    case 128: launch_wide<HD, 4, 2>(p, st); break;
    default: launch_wide<HD, 8, 1>(p, st); break;
    }
    SD_HIP_CHECK(hipGetLastError());
    if (p.nsplit > 1) {
        k_kvq_combine<HD><<<dim3((unsigned)(p.max_rows * p.n_heads), (unsigned)p.n_seqs), dim3(256), 0, st>>>(p);
        SD_HIP_CHECK(hipGetLastError());
    }
}

void launch_kvq_attention(const KvqAttn &in, const KvqPlan &plan, void *ws, hipStream_t st) {
    KvqAttn p = in;
    p.nsplit = plan.nsplit;
    p.tile_q = plan.tile_q;
    p.tiles = plan.tiles;
    p.chunk = plan.chunk;
    p.groups = p.tiles * p.L.n_kv * p.n_seqs;
    p.part_o = (float *)ws;
    p.part_ml = p.part_o + (int64_t)p.nsplit * p.rows * p.n_heads * p.L.hd;
    if (p.L.hd == 128) launch_attn<128>(p, st);
    else launch_attn<64>(p, st);
}

}  // namespace sd
