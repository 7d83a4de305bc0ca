// Eviction from the 8-bit cache by the positions' accumulated weights: which ones of
// every sequence and KV head stay, and moving them together.
#include <type_traits>

#include "sd_kv8_dev.hpp"

namespace sd {

// Positions of a sequence that exist: the table has pages and the scores entries for them.
__device__ __forceinline__ int kv8_evict_len(const Kv8Evict &p, int s) {
    const int64_t cap = min((int64_t)p.table_ld << p.L.page_shift, min(p.scores_ld, (int64_t)kKv8MaxEvict));
    return (int)max((int64_t)0, min((int64_t)p.kv_len[s], cap));
}

// A score's rank as an unsigned number, never 0: larger for a larger score, NaN below all, -0 as 0.
__device__ __forceinline__ uint32_t kv8_rank(float x) {
    if (x != x) return 1;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}

// One workgroup per (KV head, sequence).  The rank of the last position that stays is
// found 11, 11 and 10 bits at a time, each by a histogram of the positions that agree
// with the bits found so far; then every wave counts what it keeps of its part of the
// positions, in order, and writes it.  Equal scores stay from the lowest position on.
// Ranks are held in LDS, 32768 at a time: a sequence up to that length is read once, a
// longer one once for each of the four rounds (32769 positions 41 us, 131072 112).  32768
// positions: 20 us on the one CU that a head has, where VALU instructions are issued in
// more than half of its cycles (equal scores meet in one bin: 53 us); with the
// first histogram behind the reading, bounds checked at every position and one position a
// lane in the counts 28.  2176 positions: 9, most of them the rounds' barriers.
constexpr int kSelT = 1024, kSelWaves = kSelT / 64, kSelBins = 2048, kSelChunk = 32768;
static_assert(kSelChunk % (8 * kSelT) == 0, "a full chunk has no position past its end");
constexpr uint32_t kSelForced = ~0u;  // the rank of a first or last position
struct Kv8Select {
    __align__(16) uint32_t bins[kSelBins][2];  // of even and odd lanes: fewer meet in one
    uint32_t part[kSelWaves], eq_part[kSelWaves];
    uint32_t found[2];  // bin, positions in bins above it
};
// the sum of the first n of 16 numbers in LDS, in every lane
__device__ __forceinline__ uint32_t kv8_sum_first(const uint32_t *v, int n, int lane) {
    int x = (lane & 15) < n ? (int)v[lane & 15] : 0;
    x += __builtin_amdgcn_mov_dpp(x, 0xB1, 0xf, 0xf, true);   // lane ^ 1
    x += __builtin_amdgcn_mov_dpp(x, 0x4E, 0xf, 0xf, true);   // lane ^ 2
    x += __builtin_amdgcn_mov_dpp(x, 0x141, 0xf, 0xf, true);  // 7 - lane of each 8
    x += __builtin_amdgcn_mov_dpp(x, 0x140, 0xf, 0xf, true);  // 15 - lane of each 16
    return (uint32_t)x;
}
// bits of m below the lane's own
__device__ __forceinline__ uint32_t kv8_below(uint64_t m) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}
__global__ __launch_bounds__(kSelT) void k_kv8_select(const Kv8Evict p) {
    extern __shared__ __align__(16) uint32_t sel_rank[];
    __shared__ Kv8Select sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = blockIdx.x, s = blockIdx.y;
    const int T = kv8_evict_len(p, s), n = min(T, p.budget);
    const int64_t u = (int64_t)s * p.L.n_kv + h;
    const float *x = p.scores + u * p.scores_ld;
    int *kept = p.kept + u * p.budget;
    if (h == 0 && tid == 0) p.new_len[s] = n;
    for (int i = n + tid; i < p.budget; i += kSelT) kept[i] = -1;
    if (T <= p.budget) {
        for (int i = tid; i < T; i += kSelT) kept[i] = i;
        return;
    }
    const int lo = p.sinks, hi = T - p.recent;  // candidates [lo, hi)
    const bool once = T <= kSelChunk;
    // ranks of the positions from `at` on, zeros up to a multiple of a round; the first time counted by their highest 11 bits
    auto load = [&](int at, auto first) {
        const int m = min(kSelChunk, T - at), round = (m + kSelT - 1) / kSelT * kSelT;
        float v[8], w[8];
        auto ask = [&](int i0) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = x[at + min(i0 + j * kSelT, m - 1)];
        };
        ask(tid);
        __syncthreads();
        for (int i0 = tid; i0 < round; i0 += 8 * kSelT) {
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = v[j];
            if (i0 + 8 * kSelT < round) ask(i0 + 8 * kSelT);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int i = i0 + j * kSelT, from = at + i - tid;
                if (from >= lo && from + kSelT <= hi) {  // (i < m: hi is at most T, and a chunk whole strides)
                    const uint32_t r = kv8_rank(w[j]);
                    sel_rank[i] = r;
                    if (first) atomicAdd(&sh.bins[r >> 21][lane & 1], 1u);
                    continue;
                }
                const bool open = i < m && at + i >= lo && at + i < hi;
                const uint32_t r = i >= m ? 0 : open ? kv8_rank(w[j]) : kSelForced;
                if (i < round) sel_rank[i] = r;
                if (first && open) atomicAdd(&sh.bins[r >> 21][lane & 1], 1u);
            }
        }
        __syncthreads();
        return m;
    };
    *(uintx4 *)&sh.bins[2 * tid][0] = uintx4{0, 0, 0, 0};
    int m = 0;
    for (int at = 0; at < T; at += kSelChunk) m = load(at, std::true_type{});
    uint32_t need = (uint32_t)(p.budget - p.sinks - p.recent);  // candidates that stay
    const bool any = need > 0;
    uint32_t prefix = any ? 0 : kSelForced - 1;  // the bits found of the last one's rank
    int shift = 32;
    for (int pass = 0; pass < 3 && any; pass++) {
        const int bits = pass < 2 ? 11 : 10, above = shift;  // bits of the prefix end at `above`
        shift -= bits;
        if (pass > 0) {
            *(uintx4 *)&sh.bins[2 * tid][0] = uintx4{0, 0, 0, 0};
            __syncthreads();
        }
        for (int at = 0; pass > 0 && at < T; at += kSelChunk) {
            if (!once) m = load(at, std::false_type{});
            const uint32_t low = (1u << bits) - 1u;
#pragma unroll 2
            for (int i = 4 * tid; i < m; i += 4 * kSelT) {
                // (forced ones' highest bits are no number's; the zeros past the end come behind all that can be looked for)
                const uintx4 q = *(const uintx4 *)&sel_rank[i];
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (q[j] >> above == prefix)
                        atomicAdd(&sh.bins[(q[j] >> shift) & low][lane & 1], 1u);
            }
        }
        __syncthreads();
        // thread t has the bins 2047 - 2 t and 2046 - 2 t: from the top down
        const uintx4 ba = *(const uintx4 *)&sh.bins[kSelBins - 2 - 2 * tid][0];
        const uint32_t a = ba.z + ba.w, b = ba.x + ba.y;
        uint32_t run = a + b;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t v = __shfl_up(run, o);
            if (lane >= o) run += v;
        }
        if (lane == 63) sh.part[wave] = run;
        __syncthreads();
        const uint32_t before = run - a - b + kv8_sum_first(sh.part, wave, lane);
        if (before < need && before + a >= need) sh.found[0] = (uint32_t)(kSelBins - 1 - 2 * tid), sh.found[1] = before;
        else if (before + a < need && before + a + b >= need) sh.found[0] = (uint32_t)(kSelBins - 2 - 2 * tid), sh.found[1] = before + a;
        __syncthreads();
        prefix = prefix << bits | sh.found[0];
        need -= sh.found[1];
    }
    // `prefix` is the last one's rank, `need` of its equals stay
    uint32_t at_chunk = 0, eq_chunk = 0;  // what is above it and what equals it in front of the chunk
    for (int at = 0; at < T; at += kSelChunk) {
        if (!once) m = load(at, std::false_type{});
        // wave w has the positions [first, last) of the chunk, whole rounds of 64
        const int seg = (m + kSelT - 1) / kSelT * 64, first = wave * seg, last = first + seg;
        uint32_t count = 0;  // of those above it, and 65536 times that of its equals
        for (int i = first + 4 * lane; i < last; i += 256) {
            const uintx4 q = *(const uintx4 *)&sel_rank[i];
#pragma unroll
            for (int j = 0; j < 4; j++) count += (q[j] > prefix ? 1u : 0u) + (q[j] == prefix ? 65536u : 0u);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) count += __shfl_xor(count, o);
        __syncthreads();  // the parts of the pass or chunk before have been read
        if (lane == 0) sh.part[wave] = count & 0xffffu, sh.eq_part[wave] = count >> 16;
        __syncthreads();
        uint32_t seen = eq_chunk + kv8_sum_first(sh.eq_part, wave, lane);
        uint32_t to = at_chunk + kv8_sum_first(sh.part, wave, lane) + min(seen, need);
        at_chunk += kv8_sum_first(sh.part, kSelWaves, lane);
        eq_chunk += kv8_sum_first(sh.eq_part, kSelWaves, lane);
#pragma unroll 4
        for (int i = first; i < last; i += 64) {
            const uint32_t r = sel_rank[i + lane];
            bool stay = r > prefix;
            const uint64_t e = __builtin_amdgcn_ballot_w64(r == prefix);
            if (e != 0) {
                stay |= r == prefix && seen + kv8_below(e) < need;
                seen += (uint32_t)__popcll(e);
            }
            const uint64_t k = __builtin_amdgcn_ballot_w64(stay);
            if (stay) kept[to + kv8_below(k)] = at + i + lane;
            to += (uint32_t)__popcll(k);
        }
    }
    if (p.scores_out != p.scores) return;  // (elsewhere they go with the keys)
    __threadfence_block();
    __syncthreads();
    // the scores move to the front: what a round writes, later ones do not read
    float *y = p.scores_out + u * p.scores_out_ld;
    for (int i0 = 0; i0 < n; i0 += kSelT) {
        const int i = i0 + tid;
        const float v = i < n ? x[__hip_atomic_load(&kept[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)] : 0.f;
        __syncthreads();
        if (i < n) y[i] = v;
        __syncthreads();
    }
}

// Block d of what a sequence's head keeps, keys or values: its positions' codes from
// wherever they are, as one block.  In place it goes to the workspace, since other
// workgroups still read where it belongs, and k_kv8_place brings it there.
struct Kv8Spot {
    uint8_t *codes;
    Kv8Head *head;
};
template <int HD> __device__ __forceinline__ Kv8Spot kv8_in_ws(void *ws, int n_seqs, int n_kv, int nblk, int s, int h, int d) {
    const int64_t i = ((int64_t)s * n_kv + h) * nblk + d, all = (int64_t)n_seqs * n_kv * nblk;
    return {(uint8_t *)ws + i * kv8_block_bytes(HD), (Kv8Head *)((uint8_t *)ws + all * kv8_block_bytes(HD)) + i};
}
// where block d belongs; codes null: its page is not there
__device__ __forceinline__ Kv8Spot kv8_in_pool(const Kv8Evict &p, int s, int h, int d) {
    const int *table = p.new_table ? p.new_table : p.table;
    const int ld = p.new_table ? p.new_ld : p.table_ld, at = d >> (p.L.page_shift - 5);
    const int page = at < ld ? table[(int64_t)s * ld + at] : -1;
    if (page < 0 || page >= p.L.n_pages) return {nullptr, nullptr};
    return {p.L.codes(page, h, d * 32), p.L.head(page, h, d * 32)};
}
template <int HD> __device__ __forceinline__ Kv8Spot kv8_to(const Kv8Evict &p, void *ws, int s, int h, int d) {
    return p.new_table ? kv8_in_pool(p, s, h, d) : kv8_in_ws<HD>(ws, p.n_seqs, p.L.n_kv, (p.budget + 31) / 32, s, h, d);
}
// Keys: 8 threads to a position, whose codes are 8 bytes next to each other.
template <int HD>
__device__ __forceinline__ void kv8_gather_k(const Kv8Evict &p, void *ws, Kv8Sh &sh, int s, int h, int d, int n) {
    const int k = threadIdx.x >> 3, c0 = (threadIdx.x & 7) * 8, i = d * 32 + k;
    float x[HD / 8] = {};
    bool nan = false;
    if (i < n) {
        const int64_t head = (int64_t)s * p.L.n_kv + h;
        const int pos = p.kept[head * p.budget + i];
        const int page = p.table[(int64_t)s * p.table_ld + (pos >> p.L.page_shift)];
        if (p.scores_out && p.scores_out != p.scores && c0 == 0)
            p.scores_out[head * p.scores_out_ld + i] = p.scores[head * p.scores_ld + pos];
        if (page >= 0 && page < p.L.n_pages) {  // (a position without a page is zeros)
            const Kv8Head *of = p.L.head(page, h, pos);
            kv8_key<HD>(p.L.codes(page, h, pos), pos & 31, c0, of->scale[0], x);
            nan = of->nan[0] >> (pos & 31) & 1;
        }
    }
    float scale;
    uint32_t nans;
    kv8_build<HD, false>(sh, x, i < n, nan, scale, nans);
    const Kv8Spot to = kv8_to<HD>(p, ws, s, h, d);
    if (!to.codes) return;
    kv8_codes_out<HD>(sh, to.codes);
    if (threadIdx.x == 0) {
        to.head->scale[0] = scale;
        to.head->nan[0] = nans;
    }
}
// Values: a position's bytes are 8 apart, between those of 7 others, so the groups of
// 8 positions that have some of the 32 go to LDS as they are, once each, and a thread
// picks 8 positions of one or two channels, which are what it writes.
constexpr int kGroups = 16;  // at a time: with 32 half as many workgroups fit a CU
template <int HD> struct Kv8Groups {
    __align__(16) uint8_t codes[kGroups][HD * 8];
    const uint8_t *from[32];
    float scale[32];
    uint16_t at[32];  // of position k: its group's place and its byte
    uint32_t nan;
    int n, exp[4];
};
template <int HD>
__device__ __forceinline__ void kv8_gather_v(const Kv8Evict &p, void *ws, Kv8Groups<HD> &G, int s, int h, int d, int n) {
    constexpr int NT = HD / 64, NI = HD / 32;
    const int tid = threadIdx.x, lane = tid & 63;
    if (tid < 64) {
        const int i = d * 32 + lane;
        int pos = -1;
        float scale = 0.f;  // (what is past the end, or has no page, is zeros)
        uint32_t nan = 0;
        const uint8_t *from = p.L.base;
        if (lane < 32 && i < n) {
            pos = p.kept[((int64_t)s * p.L.n_kv + h) * p.budget + i];
            const int page = p.table[(int64_t)s * p.table_ld + (pos >> p.L.page_shift)];
            if (page >= 0 && page < p.L.n_pages) {
                const Kv8Head *head = p.L.head(page, h, pos);
                from = p.L.codes(page, h, pos) + 32 * HD + (pos >> 3 & 3) * 256;
                scale = head->scale[1];
                nan = head->nan[1] >> (pos & 31) & 1;
            }
        }
        const int before = __shfl_up(pos, 1);
        const bool fresh = lane == 0 || (lane < 32 && pos >> 3 != before >> 3);
        const uint64_t starts = __builtin_amdgcn_ballot_w64(fresh), nans = __builtin_amdgcn_ballot_w64(nan != 0);
        if (lane < 32) {
            const int slot = (int)__popcll(starts & ((2ull << lane) - 1ull)) - 1;
            if (fresh) G.from[slot] = from;
            G.scale[lane] = scale;
            G.at[lane] = (uint16_t)(slot << 3 | (pos & 7));
        }
        if (lane == 0) G.n = (int)__popcll(starts), G.nan = (uint32_t)nans;
    }
    __syncthreads();
    // task: channel (HD / 16) r + 2 i + e, positions 8 g ..
    float x[NT][8], top = 0.f;
    const int groups = G.n;
    for (int s0 = 0; s0 < groups; s0 += kGroups) {
        if (s0) __syncthreads();
        for (int u = tid; u < min(groups - s0, kGroups) * (HD / 2); u += kKv8T) {
            const int slot = u / (HD / 2), w = u % (HD / 2);
            *(uintx4 *)&G.codes[slot][w * 16] = *(const uintx4 *)(G.from[s0 + slot] + (w >> 4) * 1024 + (w & 15) * 16);
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < NT; m++) {
            const int u = tid + kKv8T * m, rest = u >> 5, g = rest / NI, in = (rest % NI) * 256 + (u & 31) * 8;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int at = G.at[8 * g + j], slot = (at >> 3) - s0;
                if (slot < 0 || slot >= kGroups) continue;
                x[m][j] = kv8_value(G.codes[slot][in + (at & 7)], G.scale[8 * g + j]);
                top = fmaxf(top, fabsf(x[m][j]));
            }
        }
    }
    int e = top > 0.f ? min(max(kv8_exp(top), kKv8MinExp), kKv8MaxExp) : kKv8MinExp;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) e = max(e, __shfl_xor(e, o));
    if (lane == 0) G.exp[tid >> 6] = e;
    __syncthreads();
    e = max(max(G.exp[0], G.exp[1]), max(G.exp[2], G.exp[3]));
    const Kv8Spot to = kv8_to<HD>(p, ws, s, h, d);
    if (!to.codes) return;
    const float back = kv8_two_to(-e);
#pragma unroll
    for (int m = 0; m < NT; m++) {
        const int u = tid + kKv8T * m, rest = u >> 5, g = rest / NI;
        uintx2 w;
#pragma unroll
        for (int j = 0; j < 2; j++)
            w[j] = kv8_pack(x[m][4 * j] * back, x[m][4 * j + 1] * back, x[m][4 * j + 2] * back, x[m][4 * j + 3] * back);
        *(uintx2 *)(to.codes + 32 * HD + (rest % NI) * 1024 + g * 256 + (u & 31) * 8) = w;
    }
    if (tid == 0) {
        to.head->scale[1] = kv8_two_to(e);
        to.head->nan[1] = G.nan;
    }
}
// 8 sequences of some 2200 positions cut to 2048, 4 heads of 128 channels, 31 MB moved:
// 16 us; 32768 positions of 8 heads cut to 4096, 17 MB: 14 us, in which 43 MB are fetched,
// since a position's values lie in one byte of eight of its group's.
template <int HD> __global__ __launch_bounds__(kKv8T) void k_kv8_gather(const Kv8Evict p, void *ws) {
    __shared__ union Sh {
        Kv8Sh k;
        Kv8Groups<HD> v;
        __device__ Sh() {}
    } sh;
    const int s = blockIdx.z, d = blockIdx.x, n_kv = p.L.n_kv, u = blockIdx.y;
    const int T = kv8_evict_len(p, s), n = min(T, p.budget);
    if (d * 32 >= n) return;
    if (T <= p.budget && !p.new_table) {  // stays where it is
        if (u < n_kv && threadIdx.x < 32 && p.scores_out && p.scores_out != p.scores && d * 32 + (int)threadIdx.x < n) {
            const int64_t head = (int64_t)s * n_kv + u, i = d * 32 + threadIdx.x;
            p.scores_out[head * p.scores_out_ld + i] = p.scores[head * p.scores_ld + i];
        }
        return;
    }
    if (u < n_kv) kv8_gather_k<HD>(p, ws, sh.k, s, u, d, n);
    else kv8_gather_v<HD>(p, ws, sh.v, s, u - n_kv, d, n);
}
template <int HD> __global__ __launch_bounds__(kKv8T) void k_kv8_place(const Kv8Evict p, void *ws) {
    const int s = blockIdx.z, d = blockIdx.x, h = blockIdx.y;
    const int T = kv8_evict_len(p, s);
    if (T <= p.budget || d * 32 >= p.budget) return;
    const Kv8Spot from = kv8_in_ws<HD>(ws, p.n_seqs, p.L.n_kv, (p.budget + 31) / 32, s, h, d), to = kv8_in_pool(p, s, h, d);
    if (!to.codes) return;
#pragma unroll
    for (int i = 0; i < HD / 64; i++)
        *(uintx4 *)(to.codes + (i * kKv8T + threadIdx.x) * 16) = *(const uintx4 *)(from.codes + (i * kKv8T + threadIdx.x) * 16);
    if (threadIdx.x == 0) *to.head = *from.head;
}

void kv8_prepare() {
    SD_HIP_CHECK(hipFuncSetAttribute((const void *)k_kv8_select, hipFuncAttributeMaxDynamicSharedMemorySize, kSelChunk * 4));
}

size_t kv8_evict_ws_bytes(int n_seqs, int n_kv, int hd, int budget) {
    return (size_t)n_seqs * n_kv * ((budget + 31) / 32) * (kv8_block_bytes(hd) + sizeof(Kv8Head));
}

void launch_kv8_evict(const Kv8Evict &p, void *ws, hipStream_t st) {
    const unsigned kv = (unsigned)p.L.n_kv, seqs = (unsigned)p.n_seqs, nblk = (unsigned)((p.budget + 31) / 32);
    const int64_t most = std::min<int64_t>(((int64_t)p.table_ld << p.L.page_shift), p.scores_ld);
    const int lds = (int)std::min<int64_t>((most + kSelT - 1) / kSelT * kSelT, kSelChunk) * 4;
    k_kv8_select<<<dim3(kv, seqs), dim3(kSelT), lds, st>>>(p);
    SD_HIP_CHECK(hipGetLastError());
    if (nblk == 0) return;
    const dim3 b(kKv8T);
    if (p.L.hd == 128) k_kv8_gather<128><<<dim3(nblk, 2 * kv, seqs), b, 0, st>>>(p, ws);
    else k_kv8_gather<64><<<dim3(nblk, 2 * kv, seqs), b, 0, st>>>(p, ws);
    SD_HIP_CHECK(hipGetLastError());
    if (p.new_table) return;
    if (p.L.hd == 128) k_kv8_place<128><<<dim3(nblk, kv, seqs), b, 0, st>>>(p, ws);
    else k_kv8_place<64><<<dim3(nblk, kv, seqs), b, 0, st>>>(p, ws);
    SD_HIP_CHECK(hipGetLastError());
}

}  // namespace sd
