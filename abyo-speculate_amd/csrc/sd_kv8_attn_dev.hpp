// What the attention over the 8-bit cache and the sums of its weights share:
// which blocks a tile of queries sees, and which of their positions.
#pragma once
#include "sd_kv8_dev.hpp"
#include "sd_kvq_attn_dev.hpp"

namespace sd {

// kvq_place and kvq_query without divisions
__device__ __forceinline__ KvqPlace kv8_place(const Kv8Attn &p) {
    KvqPlace r;
    const uint32_t id = blockIdx.x, n = (uint32_t)p.groups;
    r.split = (int)p.by_groups.quot(id);
    uint32_t i = id - r.split * n + (uint32_t)r.split;
    i -= p.by_groups.quot(i) * n;
    const uint32_t a = p.by_kv.quot(i);
    r.h = (int)(i - a * (uint32_t)p.L.n_kv);
    r.s = (int)p.by_tiles.quot(a);
    r.tile = (int)(a - r.s * (uint32_t)p.tiles);
    return r;
}

// Rows and positions of a workgroup's sequence, its queries and their blocks.
struct Kv8Work {
    int r0, n, T, P;   // row i of n is row r0 + i of the call and position P + i
    int nq, q0;        // queries of the KV head, the tile's first
    int t_end, t_all;  // positions that some of the tile's rows see end before t_end, without a window all see those before t_all
    int w_any, w_all;  // with a window: besides the first `sinks`, some rows see positions from w_any on, all of them from w_all
    int nsink, b_win;  // blocks: [0, nsink) for the first positions, then from b_win to the end
    int total;         // blocks in all
};

// the k-th block that a tile sees
__device__ __forceinline__ int kv8_nth(const Kv8Work &w, int k) { return k < w.nsink ? k : k - w.nsink + w.b_win; }

__device__ __forceinline__ bool kv8_work(const Kv8Attn &p, int s, int tile, int tile_q, Kv8Work &w) {
    w.T = p.row_start ? p.kv_len[s] : p.len0;
    if (!kvq_seq_rows(p, s, w.r0, w.n)) return false;
    w.nq = min(w.n, p.max_rows) * p.n_rep;
    w.q0 = tile * tile_q;
    if (w.q0 >= w.nq) return false;
    w.T = min(w.T, kKv8MaxLen);
    w.P = w.T - w.n;
    const int m_first = p.by_rep.quot(w.q0), m_last = p.by_rep.quot(min(w.q0 + tile_q, w.nq) - 1);
    w.t_end = p.mask ? w.T : min(w.T, w.P + m_last + 1);
    w.t_all = p.mask ? w.P : w.P + m_first + 1;
    // blocks that hold positions the table has pages for
    const int nblk = w.t_end > 0 ? (int)min((int64_t)((w.t_end - 1) / 32 + 1), (int64_t)p.table_ld << (p.L.page_shift - 5)) : 0;
    w.w_any = w.w_all = w.nsink = w.b_win = 0;
    if (p.window > 0) {
        w.w_any = max(0, w.P + m_first - p.window + 1);
        w.w_all = max(0, w.P + m_last - p.window + 1);
        w.b_win = min(w.w_any >> 5, nblk);
        w.nsink = min((int)(((int64_t)p.sinks + 31) >> 5), w.b_win);
    }
    w.total = w.nsink + nblk - w.b_win;
    return true;
}
__device__ __forceinline__ const uint16_t *kv8_query(const Kv8Attn &p, const Kv8Work &w, int h, int q) {
    q = min(q, w.nq - 1);
    const int m = p.by_rep.quot(q);
    return p.q + (int64_t)(w.r0 + m) * p.q_row + (int64_t)(h * p.n_rep + q - m * p.n_rep) * p.q_head;
}
// whether every row of the tile sees all of positions [a, a + n)
__device__ __forceinline__ bool kv8_full(const Kv8Attn &p, const Kv8Work &w, int a, int n) {
    return a + n <= w.t_all && a + n <= w.T && (p.window <= 0 || a >= w.w_all || a + n <= p.sinks);
}

// the lowest n of 8 bits
__device__ __forceinline__ uint32_t kv8_low(int n) { return n >= 8 ? 0xffu : (1u << max(n, 0)) - 1u; }
// bit j: row m sees position key0 + j, j < 8; key0 a multiple of 8
__device__ __forceinline__ uint32_t kv8_visible(const Kv8Attn &p, const Kv8Work &w, int m, int key0) {
    uint32_t vis;
    if (!p.mask) {
        vis = kv8_low(w.P + m + 1 - key0);
    } else {
        // 8 bits from x0 of the row's words: both words they can lie in are loaded at once, whatever x0 is
        const uint64_t *mk = p.mask + (int64_t)(w.r0 + m) * p.mask_words;
        const int x0 = key0 - w.P, a = x0 >> 6, s = x0 & 63;
        const uint64_t w0 = mk[min(max(a, 0), p.mask_words - 1)], w1 = mk[min(max(a + 1, 0), p.mask_words - 1)];
        const uint64_t lo = a >= 0 && a < p.mask_words ? w0 : 0, hi = a + 1 >= 0 && a + 1 < p.mask_words ? w1 : 0;
        vis = (uint32_t)(lo >> s | (hi << 1) << (63 - s)) & kv8_low(w.n - x0);
        if (x0 < 0) vis |= kv8_low(-x0);  // the prefix
    }
    if (p.window > 0) vis &= kv8_low(p.sinks - key0) | ~kv8_low(w.P + m - p.window + 1 - key0);
    return vis;
}

}  // namespace sd
