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

constexpr int kWgtWaves = 4, kWgtStages = 2;
template <int HD> struct Kv8Queries {
    uintx4 q[HD / 16][64];  // [chunk of 16 channels][lane]: the MFMA's operands
};

// Queries that see a position j: those from from(j) on and before to(j), numbered as
// row x n_rep + head.  Without a tree's mask that is all there is to visibility.
struct Kv8Range {
    int P, n_rep, window, sinks;
    __device__ __forceinline__ static int clip(int64_t x) { return (int)min(max(x, (int64_t)0), (int64_t)0x7fffffff); }
    __device__ __forceinline__ int from(int j) const { return clip((int64_t)(j - P) * n_rep); }
    __device__ __forceinline__ int to(int j) const {
        return window <= 0 || j < sinks ? 0x7fffffff : clip(((int64_t)j - P + window) * n_rep);
    }
};

// A tile of queries is multiplied while the weights of the one before are taken, is in
// LDS one tile ahead and on its way from memory two ahead.  512 rows of 32 heads over 8
// and 16384 positions: 97 us, 700 TFLOP/s; without that overlap and with a division for
// each query's address 157.  Matrix instructions take 38 % of the CUs' busy cycles, VALU
// instructions (of which 32 exponentials for each 64 positions and 32 queries) are issued
// in 50 %, waves wait for 38 % of theirs: four of them meet at each tile.  A batch of
// single rows (4 sequences, 15273 positions): 8 us, of which the keys' bytes are 1.3; the
// rest is the chain of lengths, page, keys, and the queries behind them.
template <int HD, int NB>
__global__ __launch_bounds__(64 * kWgtWaves) __attribute__((amdgpu_waves_per_eu(2))) void k_kv8_weights(const Kv8Weights p) {
    constexpr int NC = HD / 16, NQ = HD / 64;  // chunks; 16-byte pieces of a tile of queries to a thread
    __shared__ Kv8Queries<HD> sh[kWgtStages];
    // in base 2, read a tile later than the queries
    __shared__ __align__(16) float sh_lse[4][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r32 = lane & 31, hh = lane >> 5;
    warm_kernargs<sizeof(Kv8Weights)>();
    const int s = blockIdx.z, h = blockIdx.y;
    const Kv8Layer L(p.a.L);
    Kv8Work W;
    if (!kv8_work(p.a, s, 0, 32, W)) return;
    const int T = (int)min((int64_t)W.T, p.ld), tiles = (W.nq + 31) / 32, n_rep = p.a.n_rep;
    const Kv8Range see{W.P, n_rep, p.a.window, p.a.sinks};
    const bool tree = p.a.mask != nullptr;
    const float sl2 = p.a.scale * 1.4426950408889634f;
    constexpr int kMine = 32 * NB, kChunk = kMine * kWgtWaves;
    for (int64_t c0 = (int64_t)blockIdx.x * kChunk; c0 < T; c0 += (int64_t)gridDim.x * kChunk) {
        // the wave's keys: lane (r32, hh) has the channels 16 c + 8 hh .. of position r32
        const int base = (int)c0 + wave * kMine;
        half8 kf[NB][NC];
        uint32_t nan[NB];
        int q_from[NB], q_to[NB];  // the lane's position is seen by the queries in between (a tree's own rows: by its bits)
        bool clean = base + kMine <= T;  // no position is past the end, absent or NaN
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int pos = base + 32 * b;
            int page = -1;
            if (pos < T && (pos >> p.a.L.page_shift) < p.a.table_ld) page = p.a.table[(int64_t)s * p.a.table_ld + (pos >> p.a.L.page_shift)];
            page = __builtin_amdgcn_readfirstlane(page);
            const bool have = page >= 0 && page < p.a.L.n_pages;
            const uint8_t *codes = have ? L.codes(page, h, pos) : p.a.L.base;
            const Kv8Head hd = *(have ? L.head(page, h, pos) : (const Kv8Head *)p.a.L.base);
            uintx2 w[NC];
#pragma unroll
            for (int c = 0; c < NC; c++) w[c] = *(const uintx2 *)(codes + kv8_k_at(r32, 16 * c + 8 * hh, HD));
            const float scale = have ? hd.scale[0] : 1.f;
#pragma unroll
            for (int c = 0; c < NC; c++) kf[b][c] = __builtin_bit_cast(half8, kv8_expand(w[c].x, w[c].y, scale));
            nan[b] = have ? hd.nan[0] : 0;
            const int mine = pos + r32;
            q_from[b] = !have || mine >= T ? 0x7fffffff : tree ? 0 : see.from(mine);
            q_to[b] = see.to(mine);
            clean = clean && have && nan[b] == 0;
        }
        // tiles of queries that see some of the workgroup's positions, some and all of the wave's
        const int c1 = (int)min(c0 + kChunk, (int64_t)T) - 1, last = base + kMine - 1;
        const int t0 = tree ? 0 : min(tiles, see.from((int)c0) / 32);
        const int t1 = c0 < p.a.sinks ? tiles : max(t0, min(tiles, (int)(((int64_t)see.to(c1) + 31) / 32)));
        const int some0 = tree ? 0 : see.from(base) / 32, some1 = base < p.a.sinks ? tiles : (int)(((int64_t)see.to(last) + 31) / 32);
        const int all0 = tree ? (last < W.P ? 0 : tiles) : (int)(((int64_t)see.from(last) + 31) / 32);
        const int all1 = min(W.nq, p.a.window <= 0 || last < p.a.sinks ? 0x7fffffff : min(see.to(base), see.to(max(base, p.a.sinks)))) / 32;

        uintx4 piece[2][NQ];
        float lse[2];
        // The thread's query of the tile that is asked for next, and how far the next tile's is; past the last one it is the
        // sequence's first.
        const int rows = p.a.by_rep.quot(W.nq), step_row = p.a.by_rep.quot(32), step_rep = 32 - step_row * n_rep;
        const int64_t q_step = step_row * p.a.q_row + step_rep * p.a.q_head, q_wrap = p.a.q_row - n_rep * p.a.q_head;
        const int64_t s_step = step_row * (int64_t)p.a.n_heads + step_rep, s_wrap = p.a.n_heads - n_rep;
        const uint16_t *q_first = p.a.q + (int64_t)W.r0 * p.a.q_row + (int64_t)h * n_rep * p.a.q_head + 16 * wave + 8 * hh;
        const float *s_first = p.a.lse + (int64_t)W.r0 * p.a.n_heads + h * n_rep;
        int row = 0, rep = 0;
        const uint16_t *q_at = q_first;
        const float *s_at = s_first;
        auto start = [&](int t) __attribute__((always_inline)) {
            const int q = t * 32 + r32;
            row = p.a.by_rep.quot(q), rep = q - row * n_rep;
            q_at = q_first + row * p.a.q_row + rep * p.a.q_head;
            s_at = s_first + row * (int64_t)p.a.n_heads + rep;
        };
        auto request = [&](int slot) __attribute__((always_inline)) {
            const bool in = row < rows;
            const uint16_t *q = in ? q_at : q_first;
#pragma unroll
            for (int i = 0; i < NQ; i++) piece[slot][i] = *(const uintx4 *)(q + 64 * i);
            lse[slot] = *(in ? s_at : s_first);
            row += step_row, rep += step_rep, q_at += q_step, s_at += s_step;
            if (rep >= n_rep) rep -= n_rep, row++, q_at += q_wrap, s_at += s_wrap;
        };
        auto put = [&](int slot, Kv8Queries<HD> &S, int t) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < NQ; i++) S.q[wave + 4 * i][lane] = piece[slot][i];
            // (a query that sees nothing has no weight to give)
            if (threadIdx.x < 32) sh_lse[t & 3][threadIdx.x] = lse[slot] == -INFINITY ? INFINITY : lse[slot] * 1.4426950408889634f;
        };
        float sum[NB][2] = {};
        floatx16 acc[2][NB];
        auto scores = [&](int k, const Kv8Queries<HD> &S) __attribute__((always_inline)) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int j = 0; j < 16; j++) acc[k][b][j] = 0.f;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const half8 a = __builtin_bit_cast(half8, S.q[c][lane]);
#pragma unroll
                for (int b = 0; b < NB; b++) acc[k][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, kf[b][c], acc[k][b], 0, 0, 0);
            }
        };
        // register j of a score tile is query 8 (j >> 2) + 4 hh + (j & 3), the lane's column its position
        float4 ls[4];
        auto stats = [&](int t) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; i++) ls[i] = *(const float4 *)&sh_lse[t & 3][8 * i + 4 * hh];
        };
        auto add = [&](int k) __attribute__((always_inline)) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int j = 0; j < 16; j++)
                    sum[b][j & 1] += __builtin_amdgcn_exp2f(acc[k][b][j] * sl2 - ((const float *)&ls[j >> 2])[j & 3]);
        };
        // A tile of which the position is seen by some, those of numbers [from, to) and, of a tree's own rows, those whose mask
        // has the position's bit (bit j of `vis`: the query of register j).
        auto add_some = [&](int k, int t) __attribute__((always_inline)) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const int x = base + 32 * b + r32 - W.P, q0 = t * 32 + 4 * hh;
                const int from = q_from[b], to = min(q_to[b], W.nq);
                const bool bad = nan[b] >> r32 & 1;
                uint32_t vis = 0xffffu;
                if (tree && base + 32 * b + 31 >= W.P) {
                    const bool own = x >= 0, known = x < W.n && (x >> 6) < p.a.mask_words;
                    if (own) vis = 0;
#pragma unroll 1
                    for (int j = 0; j < 16; j++) {
                        const int q = q0 + 8 * (j >> 2) + (j & 3);
                        if (own && known && q < W.nq)
                            vis |= (uint32_t)(p.a.mask[(int64_t)(W.r0 + p.a.by_rep.quot(q)) * p.a.mask_words + (x >> 6)] >> (x & 63) & 1) << j;
                    }
                }
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const int q = q0 + 8 * (j >> 2) + (j & 3);
                    const float w = __builtin_amdgcn_exp2f(acc[k][b][j] * sl2 - ((const float *)&ls[j >> 2])[j & 3]);
                    sum[b][j & 1] += q >= from && q < to && (vis >> j & 1) ? (bad ? NAN : w) : 0.f;
                }
            }
        };
        if (t0 < t1) {
            start(t0);
            request(0);
            request(1);
            put(0, sh[0], t0);
        }
        __syncthreads();
        // kinds of a tile: 0 no position of the wave is seen, 1 all are, 2 some
        int pending = 0, stage = 0;
        auto turn = [&](int k, int t) __attribute__((always_inline)) {  // tile t into acc[k]; what waits is in acc[k ^ 1]; the request for tile t + 2 goes to slot k
            const int kind = t < some0 || t >= some1 || (!tree && base >= T) ? 0 : clean && t >= all0 && t < all1 ? 1 : 2;
            const int next = stage == kWgtStages - 1 ? 0 : stage + 1;
            request(k);  // (past the last tile too: its wait is then always for the loads of the tile before)
            if (kind == 1 && pending == 1) {
                stats(t - 1);
                __builtin_amdgcn_sched_barrier(0);
                scores(k, sh[stage]);
                add(k ^ 1);
                __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
                for (int c = 0; c < NC; c++) {
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x402, 48 / NC, 0);
                    }
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            } else {
                if (pending == 1) stats(t - 1), add(k ^ 1);
                else if (pending == 2) stats(t - 1), add_some(k ^ 1, t - 1);
                if (kind) scores(k, sh[stage]);
            }
            pending = kind;
            if (t + 1 < t1) put(k ^ 1, sh[next], t + 1);
            __syncthreads();
            stage = next;
        };
        int t = t0;
        for (; t + 1 < t1; t += 2) {
            turn(0, t);
            turn(1, t + 1);
        }
        if (t < t1) {
            turn(0, t);
            if (pending == 1) stats(t), add(0);
            else if (pending == 2) stats(t), add_some(0, t);
        } else if (t0 < t1) {
            if (pending == 1) stats(t - 1), add(1);
            else if (pending == 2) stats(t - 1), add_some(1, t - 1);
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const float mine = sum[b][0] + sum[b][1];
            const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(mine), __float_as_uint(mine), false, false);
            const float total = __uint_as_float(x[0]) + __uint_as_float(x[1]);
            const int pos = base + 32 * b + r32;
            if (hh == 0 && pos < T) {
                const int64_t at = ((int64_t)s * p.a.L.n_kv + h) * p.ld + pos;
                const bool had = p.decay != 0.f && !(p.anew && pos >= W.P);
                p.out[at] = had ? p.decay * p.in[at] + total : total;
            }
        }
        __syncthreads();
    }
}

// 64 positions a wave where that still gives every CU a workgroup
void launch_kv8_weights(const Kv8Weights &in, hipStream_t st) {
    Kv8Weights p = in;
    if (!p.in) p.decay = 0.f;  // nothing is read then
    p.a.by_rep = Kv8Div::by((uint32_t)p.a.n_rep);
    const int64_t groups = (int64_t)p.a.L.n_kv * p.a.n_seqs, len = std::max<int64_t>(1, std::min(p.max_len, p.ld));
    const bool two = (len + 255) / 256 * groups >= p.cus;
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
