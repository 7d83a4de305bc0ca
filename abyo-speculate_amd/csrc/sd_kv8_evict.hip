// Eviction from the 8-bit cache by the positions' accumulated weights: which ones of
// every sequence and KV head stay, and moving them together.
#include "sd_kv8_dev.hpp"

namespace sd {

// Positions of a sequence that exist: the table has pages and the scores entries for them.
__device__ __forceinline__ int kv8_evict_len(const Kv8Evict &p, int s) {
    const int64_t cap = min((int64_t)p.table_ld << p.L.page_shift, min(p.scores_ld, (int64_t)kKv8MaxEvict));
    return (int)max((int64_t)0, min((int64_t)p.kv_len[s], cap));
}

// A score's rank as an unsigned number: larger for a larger score, NaN below all, -0 as 0.
__device__ __forceinline__ uint32_t kv8_rank(float x) {
    if (x != x) return 0;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One workgroup per (KV head, sequence).  The rank of the last position that stays is
// found 11, 11 and 10 bits at a time, each by a histogram of the positions that agree
// with the bits found so far; then every wave counts what it keeps of its part of the
// positions, in order, and writes it.  Equal scores stay from the lowest position on.
constexpr int kSelT = 1024, kSelWaves = kSelT / 64, kSelBins = 2048;
__global__ __launch_bounds__(kSelT) void k_kv8_select(const Kv8Evict p) {
    __shared__ uint32_t bins[kSelBins];
    __shared__ uint32_t part[kSelWaves], eq_part[kSelWaves];
    __shared__ uint32_t found[2];  // bin, positions in bins above it
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = blockIdx.x, s = blockIdx.y;
    const int T = kv8_evict_len(p, s), n = min(T, p.budget);
    const int64_t u = (int64_t)s * p.L.n_kv + h;
    const float *x = p.scores + u * p.scores_ld;
    float *y = p.scores_out ? p.scores_out + u * p.scores_out_ld : nullptr;
    int *kept = p.kept + u * p.budget;
    if (h == 0 && tid == 0) p.new_len[s] = n;
    for (int i = n + tid; i < p.budget; i += kSelT) kept[i] = -1;
    if (T <= p.budget) {
        for (int i = tid; i < T; i += kSelT) {
            kept[i] = i;
            if (y && y != x) y[i] = x[i];
        }
        return;
    }
    const int lo = p.sinks, hi = T - p.recent;  // candidates [lo, hi)
    uint32_t need = (uint32_t)(p.budget - p.sinks - p.recent);  // of them stay
    uint32_t prefix = 0;  // the bits found of the last one's rank
    if (need > 0) {
        int shift = 32;
        for (int pass = 0; pass < 3; pass++) {
            const int bits = pass < 2 ? 11 : 10;
            const int above = shift;  // bits of the prefix end here
            shift -= bits;
            for (int i = tid; i < kSelBins; i += kSelT) bins[i] = 0;
            __syncthreads();
            for (int i = lo + tid; i < hi; i += kSelT) {
                const uint32_t r = kv8_rank(x[i]);
                if (pass == 0 || r >> above == prefix) atomicAdd(&bins[(r >> shift) & ((1u << bits) - 1u)], 1u);
            }
            __syncthreads();
            // wave w has bins 128 w .. 128 w + 127, two to a lane, from the top down
            const uint32_t a = bins[kSelBins - 1 - 2 * tid], b = bins[kSelBins - 2 - 2 * tid];
            uint32_t run = a + b;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t v = __shfl_up(run, o);
                if (lane >= o) run += v;
            }
            if (lane == 63) part[wave] = run;
            __syncthreads();
            uint32_t before = run - a - b;
            for (int w = 0; w < wave; w++) before += part[w];
            if (before < need && before + a >= need) found[0] = (uint32_t)(kSelBins - 1 - 2 * tid), found[1] = before;
            else if (before + a < need && before + a + b >= need) found[0] = (uint32_t)(kSelBins - 2 - 2 * tid), found[1] = before + a;
            __syncthreads();
            prefix = prefix << bits | found[0];
            need -= found[1];
            __syncthreads();
        }
    }
    // `prefix` is the last one's rank, `need` of its equals stay
    const int each = (T + kSelWaves * 64 - 1) / (kSelWaves * 64) * 64, w0 = min(wave * each, T), w1 = min(w0 + each, T);
    const bool any = p.budget > p.sinks + p.recent;
    auto look = [&](int i, bool &stay, bool &equal) {
        stay = equal = false;
        if (i >= w1) return;
        if (i < lo || i >= hi) stay = true;
        else if (any) {
            const uint32_t r = kv8_rank(x[i]);
            stay = r > prefix;
            equal = r == prefix;
        }
    };
    uint32_t count = 0, equals = 0;
    for (int i0 = w0; i0 < w1; i0 += 64) {
        bool stay, equal;
        look(i0 + lane, stay, equal);
        count += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(stay));
        equals += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(equal));
    }
    if (lane == 0) part[wave] = count, eq_part[wave] = equals;
    __syncthreads();
    uint32_t at = 0, seen = 0;  // positions kept and equals met in front of this wave's
    for (int w = 0; w < wave; w++) {
        at += part[w] + (seen < need ? min(eq_part[w], need - seen) : 0);
        seen += eq_part[w];
    }
    const uint64_t below = (1ull << lane) - 1ull;
    for (int i0 = w0; i0 < w1; i0 += 64) {
        bool stay, equal;
        look(i0 + lane, stay, equal);
        const uint64_t e = __builtin_amdgcn_ballot_w64(equal);
        stay = stay || (equal && seen + (uint32_t)__popcll(e & below) < need);
        seen += (uint32_t)__popcll(e);
        const uint64_t k = __builtin_amdgcn_ballot_w64(stay);
        if (stay) kept[at + (uint32_t)__popcll(k & below)] = i0 + lane;
        at += (uint32_t)__popcll(k);
    }
    if (!y) return;
    __threadfence_block();
    __syncthreads();
    // the scores move to the front: what a round writes, later ones do not read
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
template <int HD, bool V>
__device__ __forceinline__ void kv8_gather(const Kv8Evict &p, void *ws, Kv8Sh &sh, int s, int h, int d, int n) {
    constexpr int C = HD / 8;
    const int k = threadIdx.x >> 3, c0 = (threadIdx.x & 7) * C, i = d * 32 + k;
    float x[C] = {};
    bool nan = false;
    if (i < n) {
        const int pos = p.kept[((int64_t)s * p.L.n_kv + h) * p.budget + i];
        const int page = p.table[(int64_t)s * p.table_ld + (pos >> p.L.page_shift)];
        if (page >= 0 && page < p.L.n_pages) {  // (a position without a page is zeros)
            const Kv8Head hd = *p.L.head(page, h, pos);
            kv8_row<HD, V>(p.L.codes(page, h, pos) + (V ? 32 * HD : 0), pos & 31, c0, hd.scale[V], x);
            nan = hd.nan[V] >> (pos & 31) & 1;
        }
    }
    float scale;
    uint32_t nans;
    kv8_build<HD, V>(sh, x, i < n, nan, scale, nans);
    const Kv8Spot to = p.new_table ? kv8_in_pool(p, s, h, d)
                                   : kv8_in_ws<HD>(ws, p.n_seqs, p.L.n_kv, (p.budget + 31) / 32, s, h, d);
    if (!to.codes) return;
    kv8_codes_out<HD>(sh, to.codes + (V ? 32 * HD : 0));
    if (threadIdx.x == 0) {
        to.head->scale[V] = scale;
        to.head->nan[V] = nans;
    }
}
template <int HD> __global__ __launch_bounds__(kKv8T) void k_kv8_gather(const Kv8Evict p, void *ws) {
    __shared__ Kv8Sh sh;
    const int s = blockIdx.z, d = blockIdx.x, n_kv = p.L.n_kv, u = blockIdx.y;
    const int T = kv8_evict_len(p, s), n = min(T, p.budget);
    if (d * 32 >= n || (T <= p.budget && !p.new_table)) return;
    if (u < n_kv) kv8_gather<HD, false>(p, ws, sh, s, u, d, n);
    else kv8_gather<HD, true>(p, ws, sh, s, u - n_kv, d, n);
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

size_t kv8_evict_ws_bytes(int n_seqs, int n_kv, int hd, int budget) {
    return (size_t)n_seqs * n_kv * ((budget + 31) / 32) * (kv8_block_bytes(hd) + sizeof(Kv8Head));
}

void launch_kv8_evict(const Kv8Evict &p, void *ws, hipStream_t st) {
    const unsigned kv = (unsigned)p.L.n_kv, seqs = (unsigned)p.n_seqs, nblk = (unsigned)((p.budget + 31) / 32);
    k_kv8_select<<<dim3(kv, seqs), dim3(kSelT), 0, st>>>(p);
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
