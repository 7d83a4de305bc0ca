// Attention over the 8-bit paged KV cache (sd_kv8.hpp), the whole of it or a
// sliding window behind first positions that stay visible.
//
// Split flash-decoding in two kernels, as over the 4-bit cache: scores are computed
// transposed, S^T = K Q^T, so that a lane's probabilities are its operand of
// O^T = V^T P^T, and a running reference and sum in f32 follow the blocks.  Codes
// become fp16 values (exactly what they stand for) in one conversion per two of them,
// which takes the block's scale.  No code is ever NaN or infinite, so what a
// probability of 0 meets is finite; the rows that are NaN are bits in the header.
// Probabilities are rounded to fp16 (2^-11 of each, see kKvqHead) since the matrix
// instruction takes both its operands in 16 bits, and the values fill fp16's; sums,
// references and results stay in f32.
//
// A value costs half a VALU operation, so no value is expanded for more than the wave
// that needs it: codes go from memory straight into registers, two buffers of a block
// each, and nothing waits for LDS before the waves' states are joined.  A block of 8.2 KB
// is some 190 VALU operations and 512 cycles of matrix instructions for 32 queries.
// 2048 rows of 32 heads over 8191 positions: 268 us, 900 TFLOP/s (a large product of
// fp16 matrices reaches 1196); VALU instructions are issued in 64 % of the CUs' busy
// cycles, matrix instructions take 39 %, and the two waves of a SIMD overlap them in
// part.  5 rows over 32768 positions, 67 MB of blocks: 16.6 us, 11.2 at the rate of a
// large read; the chain to the first block (arguments, lengths, page, block) is some
// 3 us, joining the waves 1.5.
// Tried and dropped: the values of a block multiplied beside the weights of the next
// (2048 rows 435 us: the registers do not hold it), tiles of 64 queries with one wave a
// SIMD (410), wave priorities around the products (no difference), a separate maximum
// for each block (300).
#include "sd_kv8_attn_dev.hpp"

#pragma clang fp contract(fast)

namespace sd {

// What a tile's blocks are cut into: ranges of `chunk` blocks, none shorter than min_blocks unless it is the only one.
struct Kv8Cut {
    int n, chunk;
};
__device__ __forceinline__ Kv8Cut kv8_cut(const Kv8Attn &p, int total) {
    Kv8Cut c;
    const int want = max(1, min(p.nsplit, total / p.min_blocks));
    c.chunk = max(1, (total + want - 1) / want);
    c.n = max(1, (total + c.chunk - 1) / c.chunk);
    return c;
}
__device__ __forceinline__ float kv8_lse(float m, float l) { return (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f; }

// What a wave loads of one block: the codes of its lane.
template <int HD> struct Kv8Step {
    uintx4 k[2][HD / 64];  // [kt][16 channels each]
    uintx4 v[HD / 32];     // [two channels each]
};
// (nothing is read where bytes is 0)
template <int HD> __device__ __forceinline__ void kv8_load(Kv8Step<HD> &b, const uint8_t *codes, uint32_t bytes, int lane) {
    const rsrc_t r = make_rsrc(codes, bytes);
#pragma unroll
    for (int kt = 0; kt < 2; kt++)
#pragma unroll
        for (int i = 0; i < HD / 64; i++) b.k[kt][i] = bld16(r, lane * 16, (kt * (HD / 64) + i) * 1024);
#pragma unroll
    for (int i = 0; i < HD / 32; i++) b.v[i] = bld16(r, lane * 16, 32 * HD + i * 1024);
}

// ---- 16 or 32 queries to a workgroup ------------------------------------------------
// Four waves take the blocks of a key range in turn, codes straight from memory
// into registers.
template <int HD, int QT>
__global__ __launch_bounds__(kKvqT) __attribute__((amdgpu_waves_per_eu(2))) void k_kv8_attn(const Kv8Attn p) {
    constexpr int NDC = HD / 32, NDT = HD / 16;
    __shared__ float sh_o[kKvqWaves][16][HD];
    __shared__ float sh_ml[kKvqWaves][16][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, g = lane >> 4;
    warm_kernargs<sizeof(Kv8Attn)>();
    const KvqPlace at = kv8_place(p);
    const int split = at.split, h = at.h;
    Kv8Work W;
    if (!kv8_work(p, at.s, at.tile, QT * 16, W)) return;
    const Kv8Cut cut = kv8_cut(p, W.total);
    if (split >= cut.n) return;
    const int b0 = split * cut.chunk, b1 = min(b0 + cut.chunk, W.total);
    const Kv8Layer L(p.L);

    uintx4 qf[QT][NDC];
    floatx4 o[QT][NDT];
    float m[QT], l[QT];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const uint16_t *qr = kv8_query(p, W, h, W.q0 + t * 16 + r16);
#pragma unroll
        for (int dc = 0; dc < NDC; dc++) qf[t][dc] = *(const uintx4 *)(qr + 8 * (g * NDC + dc));
#pragma unroll
        for (int dt = 0; dt < NDT; dt++) o[t][dt] = floatx4{0.f, 0.f, 0.f, 0.f};
        m[t] = -INFINITY;
        l[t] = 0.f;
    }
    const float sl2 = p.scale * 1.4426950408889634f;  // scores in base-2 units
    const int steps = (b1 - b0 - wave + kKvqWaves - 1) / kKvqWaves;  // blocks b0 + wave + 4 i
    auto block = [&](int i) { return kv8_nth(W, b0 + wave + i * kKvqWaves); };
    // Lane k holds the page (-1: holds no positions) and the header of the step whose number modulo 64 is k, 32 of them asked for
    // at a time: those of the steps before are still needed.
    int pg = -1;
    uintx4 heads = {0, 0, 0, 0};
    auto pages = [&](int i0) {
        const int i = i0 + (lane & 31);
        if ((lane ^ i0) & 32) return;
        pg = i < steps ? kvq_page(p, at.s, block(i)) : -1;
        if (pg < 0 || pg >= p.L.n_pages) pg = -1;
        else heads = *(const uintx4 *)L.head(pg, h, block(i) * 32);
    };
    // The loads of a step past the end, or without a page, are issued all the same and read nothing: how many are in flight is
    // always known.
    auto fetch = [&](Kv8Step<HD> &b, int i) __attribute__((always_inline)) {
        const int page = i < steps ? __builtin_amdgcn_readlane(pg, i & 63) : -1;
        kv8_load<HD>(b, L.codes(max(page, 0), h, block(min(i, steps - 1)) * 32), page >= 0 ? 64 * HD : 0, lane);
    };
    const float hidden = sl2 < 0.f ? INFINITY : -INFINITY;  // a masked score before it is scaled
    // No maximum is looked for: a query keeps the reference of its first block until eight of its weights add up to more than
    // 2^15 (below fp16's range); then the reference is raised and they are taken again.  A fused weight is of the unrounded
    // score, which beyond 2^28 may lie more than 16 from the rounded one that the reference came from, past fp16's end on
    // either side: where the reference is beyond 2^24, weights are always taken again, of the rounded scores.
    constexpr float kMost = 32768.f, kFused = 16777216.f;
    auto process = [&](const Kv8Step<HD> &k, int i) __attribute__((always_inline)) {
        if (__builtin_amdgcn_readlane(pg, i & 63) < 0) return;
        uint32_t hd[4];
#pragma unroll
        for (int j = 0; j < 4; j++) hd[j] = (uint32_t)__builtin_amdgcn_readlane((int)heads[j], i & 63);
        const float ks = __uint_as_float(hd[0]), vs = __uint_as_float(hd[1]);
        const int base = block(i) * 32, key0 = base + 8 * g;
        const bool clean = (hd[2] | hd[3]) == 0, full = clean && kv8_full(p, W, base, 32);
        floatx4 acc[QT][2];
#pragma unroll
        for (int t = 0; t < QT; t++) acc[t][0] = acc[t][1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int dc = 0; dc < NDC; dc++) {
            half8 a[2];
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
                a[kt] = __builtin_bit_cast(half8, kv8_expand(k.k[kt][dc >> 1][2 * (dc & 1)], k.k[kt][dc >> 1][2 * (dc & 1) + 1], ks));
#pragma unroll
            for (int t = 0; t < QT; t++)
#pragma unroll
                for (int kt = 0; kt < 2; kt++)
                    acc[t][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[kt], __builtin_bit_cast(half8, qf[t][dc]), acc[t][kt], 0, 0, 0);
        }
        uint32_t vis[QT];
        if (!full) {
            const uint32_t kn = hd[2] >> (8 * g) & 0xffu;
#pragma unroll
            for (int t = 0; t < QT; t++) {
                vis[t] = kv8_visible(p, W, p.by_rep.quot(min(W.q0 + t * 16 + r16, W.nq - 1)), key0);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    float &s = ((float *)&acc[t][j >> 2])[j & 3];
                    if (!clean && (kn >> j & 1)) s = NAN;
                    s = (vis[t] >> j) & 1 ? s : hidden;
                }
            }
        }
        uintx4 pk[QT];
        float sum[QT];
        bool again = false;
#pragma unroll
        for (int t = 0; t < QT; t++) {
            const float mu = m[t] == -INFINITY ? 0.f : m[t];
            sum[t] = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[t][j >> 1][(2 * j) & 3], sl2, -mu));
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[t][j >> 1][(2 * j + 1) & 3], sl2, -mu));
                sum[t] += x + y;
                pk[t][j] = h2bits(half2v{(_Float16)x, (_Float16)y});
            }
            again |= sum[t] > kMost || !(fabsf(m[t]) < kFused);
        }
        if (__builtin_amdgcn_ballot_w64(again) != 0) {
#pragma unroll
            for (int t = 0; t < QT; t++) {
                float st[8], top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    // rounded here, not inside the weight: what is weighed is what the maximum is taken of
#pragma clang fp contract(off)
                    st[j] = acc[t][j >> 2][j & 3] * sl2;
                    top = fmaxf(top, st[j]);
                }
                const float cm = xmax4(top) - kKvqHead;
                if (cm > m[t]) {
                    const float alpha = __builtin_amdgcn_exp2f(m[t] - cm);
                    m[t] = cm;
                    l[t] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) o[t][dt] *= alpha;
                }
                sum[t] = 0.f;
                pk[t] = kvq_weights(st, m[t] == -INFINITY ? 0.f : m[t], sum[t]);
            }
        }
#pragma unroll
        for (int t = 0; t < QT; t++) l[t] += sum[t];
#pragma unroll
        for (int dt = 0; dt < NDT; dt++) {
            const half8 a = __builtin_bit_cast(half8, kv8_expand(k.v[dt >> 1][2 * (dt & 1)], k.v[dt >> 1][2 * (dt & 1) + 1], vs));
#pragma unroll
            for (int t = 0; t < QT; t++)
                o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, __builtin_bit_cast(half8, pk[t]), o[t][dt], 0, 0, 0);
        }
        if (!full && hd[3] != 0) {
            // NaN rows among the block's values reach the queries that see them and no others
#pragma unroll
            for (int t = 0; t < QT; t++) {
                uint32_t hit = vis[t] & (hd[3] >> (8 * g));
                hit |= (uint32_t)__shfl_xor((int)hit, 16);
                hit |= (uint32_t)__shfl_xor((int)hit, 32);
                if (hit) {
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) o[t][dt] = floatx4{NAN, NAN, NAN, NAN};
                }
            }
        }
    };
    if (steps > 0) {
        Kv8Step<HD> even, odd;
        pages(0);
        fetch(even, 0);
        fetch(odd, 1);
        for (int i = 0; i < steps; i += 2) {
            process(even, i);
            if (((i + 2) & 31) == 0) pages(i + 2);
            fetch(even, i + 2);
            if (i + 1 < steps) process(odd, i + 1);
            fetch(odd, i + 3);
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
        if (q < W.nq) {
            const int m = p.by_rep.quot(q), row = W.r0 + m, head = h * p.n_rep + q - m * p.n_rep;
            kvq_emit<HD / 16>(p, split, row, head, tc, oc, M, lw, tc == 0);
            if (p.nsplit == 1 && p.lse && tc == 0) p.lse[(int64_t)row * p.n_heads + head] = kv8_lse(M, lw);
        }
        __syncthreads();
    }
}

// ---- the splits ------------------------------------------------------------------
// One workgroup per (row, head): every wave knows all weights (lane k: split
// k's) and takes a part of the splits, HD / 4 lanes to a split, four loads in
// flight; the first of them go out with those of the maxima and sums.
template <int HD> __global__ __launch_bounds__(256) void k_kv8_combine(const Kv8Attn p) {
    constexpr int LS = HD / 4, N = 256 / LS, U = 4;  // lanes of a split, splits of a round, rounds in flight
    __shared__ __align__(16) float sh[N][HD];
    const int s = blockIdx.y, lane = threadIdx.x & 63, mine = threadIdx.x / LS, c = threadIdx.x % LS * 4;
    warm_kernargs<sizeof(Kv8Attn)>();
    // (heads are n_rep to each of the KV heads)
    const int mh = p.by_rep.quot(blockIdx.x), mr = p.by_kv.quot(mh), r = blockIdx.x - mh * p.n_rep;
    const int head = (mh - mr * p.L.n_kv) * p.n_rep + r, tile = (mr * p.n_rep + r) >> (31 - __builtin_clz((unsigned)p.tile_q));
    Kv8Work W;
    if (!kv8_work(p, s, tile, p.tile_q, W)) return;
    if (mr >= min(W.n, p.max_rows)) return;
    const int row = W.r0 + mr, ns = kv8_cut(p, W.total).n;
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
    if (p.lse && d == 0) p.lse[at] = kv8_lse(M, l);
}

// Measured with heads of 128 channels; those of 64 follow the same rules.
// Tiles: of 16 queries up to 64 of them, which expand every value for each tile but
// leave registers for more waves (5 rows of 32 heads over 8 and 32768 positions 19.8 us,
// with one tile of 32 21.1; 16 rows 25.3 and 26.5), of 32 above (60 rows over 8192
// positions 28.5 us, with 16 29.5; 2048 rows over 8191 267 and 324).  Ranges: as many as
// give every CU two workgroups, one where there is a single tile in a single sequence
// (5 rows over 8192 positions in one tile 14.1 us, with two 16.9; a batch of 16
// sequences with two 17.2 us, with one 19.5, with eight 20; 60 rows over 8192 positions
// with two 28.2, with four 33.6), each of at least a block for each wave.  A sequence's
// own length decides how many of them it has and how long they are.
KvqPlan kv8_attn_plan(int n_heads, int n_kv, int n_seqs, int max_rows, int64_t max_len, int window, int sinks, int cus) {
    KvqPlan r{};
    const int64_t nq = (int64_t)max_rows * (n_heads / n_kv);
    r.tile_q = nq <= 64 ? 16 : 32;
    r.tiles = (int)((nq + r.tile_q - 1) / r.tile_q);
    // most blocks that a tile sees
    int64_t blocks = (max_len + 31) / 32;
    if (window > 0) blocks = std::min(blocks, ((int64_t)window + r.tile_q + 62) / 32 + ((int64_t)sinks + 31) / 32);
    const int64_t groups = (int64_t)r.tiles * n_kv * n_seqs, fill = groups > n_kv ? 2 * cus : cus;
    const int64_t want = (fill + groups - 1) / groups, most = std::max<int64_t>(1, blocks / 4);
    r.nsplit = (int)std::max<int64_t>(1, std::min({want, most, (int64_t)64}));
    return r;
}

template <int HD> static void launch_attn(const Kv8Attn &p, hipStream_t st) {
    const dim3 g((unsigned)(p.nsplit * p.groups)), b(kKvqT);
    if (p.tile_q == 16) k_kv8_attn<HD, 1><<<g, b, 0, st>>>(p);
    else k_kv8_attn<HD, 2><<<g, b, 0, st>>>(p);
    SD_HIP_CHECK(hipGetLastError());
    if (p.nsplit > 1) {
        k_kv8_combine<HD><<<dim3((unsigned)(p.max_rows * p.n_heads), (unsigned)p.n_seqs), dim3(256), 0, st>>>(p);
        SD_HIP_CHECK(hipGetLastError());
    }
}

void launch_kv8_attention(const Kv8Attn &in, const KvqPlan &plan, void *ws, hipStream_t st) {
    Kv8Attn p = in;
    p.nsplit = plan.nsplit;
    p.tile_q = plan.tile_q;
    p.tiles = plan.tiles;
    p.min_blocks = 4;
    p.groups = p.tiles * p.L.n_kv * p.n_seqs;
    p.by_rep = Kv8Div::by((uint32_t)p.n_rep);
    p.by_kv = Kv8Div::by((uint32_t)p.L.n_kv);
    p.by_tiles = Kv8Div::by((uint32_t)p.tiles);
    p.by_groups = Kv8Div::by((uint32_t)p.groups);
    p.part_o = (float *)ws;
    p.part_ml = p.part_o + (int64_t)p.nsplit * p.rows * p.n_heads * p.L.hd;
    if (p.L.hd == 128) launch_attn<128>(p, st);
    else launch_attn<64>(p, st);
}

}  // namespace sd
