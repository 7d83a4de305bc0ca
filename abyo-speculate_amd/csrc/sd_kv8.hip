// The 8-bit paged KV cache: appending rows (RoPE and quantisation on the way),
// reading them back, moving accepted tree rows.  The format and the block layout
// are in sd_kv8.hpp.
#include "sd_kv8_dev.hpp"

namespace sd {

// The channels kv8_ch(c0, .) of a head's row, rotated in T by the pairs' or halves' angles (from f64: as kv8_odd leaves them)
template <typename T, int HD, bool F32, bool PAIRS>
__device__ __forceinline__ void kv8_rotated(const void *src, int64_t at, int c0, const float *cos_r, const float *sin_r,
                                            float (&x)[HD / 8]) {
    constexpr int N = HD / 64;
    float a[2][8] = {};  // with 64 channels the second eight are those that the first rotate with
    load8<F32>(src, at + c0, a[0]);
    if (N == 2 || !PAIRS) load8<F32>(src, at + (c0 + HD / 2) % HD, a[1]);
    if constexpr (N == 2 && !PAIRS) {
        // both halves' channels at once, which need the same numbers
        float c[8], s[8];
        load8<true>(cos_r, c0, c);
        load8<true>(sin_r, c0, s);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const T A = a[0][j], B = a[1][j], C = c[j], S = s[j];
            x[j] = kv8_odd(A * C + B * -S);
            x[8 + j] = kv8_odd(B * C + A * S);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            T o[8];
            rotate8<T, HD>(a[i], a[i ^ 1], cos_r, sin_r, c0 / 8 + 8 * i, PAIRS, o);
#pragma unroll
            for (int j = 0; j < 8; j++) x[8 * i + j] = kv8_odd(o[j]);
        }
    }
}

// The channels kv8_ch(c0, .) of query head h of the row at position pos (row pos + shift), if it is one before hi
template <int HD, bool F32, bool PAIRS>
__device__ __forceinline__ void kv8_turn_q(const Kv8Append &p, int pos, int hi, int shift, int h, int c0) {
    constexpr int C = HD / 8;
    if (pos >= hi) return;
    const int row = pos + shift, at = p.pos ? p.pos[row] : pos;
    float x[C];
    if (at >= 0 && at < p.max_pos) {
        kv8_rotated<float, HD, F32, PAIRS>(p.q, (int64_t)row * p.q_ld + (int64_t)h * HD, c0, p.cos_t + (int64_t)at * (HD / 2),
                                           p.sin_t + (int64_t)at * (HD / 2), x);
    } else {
#pragma unroll
        for (int i = 0; i < C; i++) x[i] = NAN;
    }
    uint16_t *out = p.q_out + ((int64_t)row * p.n_heads + h) * HD;
#pragma unroll
    for (int i = 0; i < C; i += 8) {
        uintx4 v;
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = (uint32_t)f2h(x[i + 2 * j]) | (uint32_t)f2h(x[i + 2 * j + 1]) << 16;
        *(uintx4 *)(out + kv8_ch<HD>(c0, i)) = v;
    }
}

// One workgroup per block and unit: the keys of a KV head, the values of one, or
// 32 pairs of a row and a query head; 8 threads to a position or pair.  Blocks of a
// sequence are dealt round gridDim.x workgroups.  What a block holds in front of the
// call's rows is read, and the whole block written: its scale may have changed.  Keys
// are rotated and rounded in f64, so that no code depends on the order of roundings.
// 16384 fp16 rows of 8 KV heads of 128 channels, 100 MB: 35 us, 21 at the rate of a
// large copy; VALU instructions, most of them the f64 rotation's, are issued in 69 % of
// the CUs' busy cycles and waves wait for 54 % of theirs.  Five waves a SIMD: with four
// 6 us more, with six registers spill and it is 3 us more.  (8 channels a thread, 16
// threads to a position: 193 us for rows and queries, 107 so.)
template <int HD, bool F32, bool PAIRS>
__global__ __launch_bounds__(kKv8T) __attribute__((amdgpu_waves_per_eu(5))) void k_kv8_append(const Kv8Append p) {
    constexpr int C = HD / 8;
    __shared__ Kv8Sh sh;
    const int s = blockIdx.z, n_kv = p.L.n_kv, tid = threadIdx.x;
    const int r0 = p.seqs.row_start ? p.seqs.row_start[s] : 0;
    const int end = p.seqs.row_start ? p.seqs.row_start[s + 1] : p.seqs.rows;
    const int T = p.seqs.row_start ? p.seqs.kv_len[s] : p.seqs.len0;
    if (r0 < 0 || end <= r0 || end > p.seqs.rows || T < 1 || T > kKv8MaxLen) return;
    // row i is position P + i; of the positions [first, last)
    const int n = end - r0, P = T - n, first = max(P, 0), last = P + min(n, p.seqs.max_rows);
    const int unit = blockIdx.y;
    for (int b = (first >> 5) + (int)blockIdx.x; (int64_t)b * 32 < last; b += gridDim.x) {
        const int lo = max(first, b * 32), hi = min(last, b * 32 + 32);
        if (unit >= 2 * n_kv) {
            kv8_turn_q<HD, F32, PAIRS>(p, lo + ((unit - 2 * n_kv) * 32 + (tid >> 3)) / p.n_heads, hi, r0 - P,
                                       ((unit - 2 * n_kv) * 32 + (tid >> 3)) % p.n_heads, (tid & 7) * 8);
            continue;
        }
        const bool is_v = unit >= n_kv;
        const int h = is_v ? unit - n_kv : unit, slot = b >> (p.L.page_shift - 5);
        const int page = slot < p.seqs.table_ld ? p.seqs.table[(int64_t)s * p.seqs.table_ld + slot] : -1;
        if (page < 0 || page >= p.L.n_pages) continue;
        uint8_t *codes = p.L.codes(page, h, b * 32) + (is_v ? 32 * HD : 0);
        Kv8Head *head = p.L.head(page, h, b * 32);
        const int k = tid >> 3, c0 = (tid & 7) * 8, pos = b * 32 + k;
        const bool live = pos < hi, held = pos < lo;
        float scale = 1.f;
        uint32_t nans = 0;
        const int row = r0 + pos - P;
        if (lo > b * 32) {
            scale = head->scale[is_v];
            nans = head->nan[is_v];
        }
        // (the barriers of kv8_build are behind all reads of the block)
        float x[C] = {};
        if (is_v) {
            if (lo > b * 32) kv8_held<HD, true>(codes, scale, x);
            if (live && !held) {
                const int64_t at = (int64_t)row * p.v_ld + (int64_t)h * HD;
#pragma unroll
                for (int i = 0; i < C; i += 8) {
                    float a[8];
                    load8<F32>(p.v, at + kv8_ch<HD>(c0, i), a);
#pragma unroll
                    for (int j = 0; j < 8; j++) x[i + j] = a[j];
                }
            }
            // a row whose rotation position does not exist is NaN in its values too
            const bool lost = live && !held && p.pos && (p.pos[row] < 0 || p.pos[row] >= p.max_pos);
            const bool past = live && !held && !p.pos && pos >= p.max_pos;
            kv8_build<HD, true>(sh, x, live, lost || past || (held && (nans >> k & 1)), scale, nans);
        } else {
            bool lost = held && (nans >> k & 1);
            if (held) {
                kv8_key<HD>(codes, k, c0, scale, x);
            } else if (live) {
                const int at = p.pos ? p.pos[row] : pos;
                lost = at < 0 || at >= p.max_pos;
                if (!lost)
                    kv8_rotated<double, HD, F32, PAIRS>(p.k, (int64_t)row * p.k_ld + (int64_t)h * HD, c0,
                                                        p.cos_t + (int64_t)at * (HD / 2), p.sin_t + (int64_t)at * (HD / 2), x);
            }
            kv8_build<HD, false>(sh, x, live, lost, scale, nans);
        }
        kv8_codes_out<HD>(sh, codes);
        if (tid == 0) {
            head->scale[is_v] = scale;
            head->nan[is_v] = nans;
        }
        __syncthreads();  // the codes in LDS are free again
    }
}

// The queries by themselves: a thread's registers are then few enough for a CU's whole
// complement of waves.  16384 rows of 32 heads, 268 MB: 57 us, 4.7 TB/s, a large copy's
// rate (54 to 57); a small call keeps them in the launch above, which saves a launch of 3 us: from
// kApart pairs of a row and a head on the shorter kernel outweighs it.
constexpr int64_t kApart = 1 << 16;
template <int HD, bool F32, bool PAIRS>
__global__ __launch_bounds__(kKv8T) void k_kv8_queries(const Kv8Append p) {
    const int s = blockIdx.z, tid = threadIdx.x;
    const int r0 = p.seqs.row_start ? p.seqs.row_start[s] : 0;
    const int end = p.seqs.row_start ? p.seqs.row_start[s + 1] : p.seqs.rows;
    const int T = p.seqs.row_start ? p.seqs.kv_len[s] : p.seqs.len0;
    if (r0 < 0 || end <= r0 || end > p.seqs.rows || T < 1 || T > kKv8MaxLen) return;
    const int n = end - r0, P = T - n, first = max(P, 0), last = P + min(n, p.seqs.max_rows);
    for (int64_t a = (int64_t)first + blockIdx.x * 32; a < last; a += (int64_t)gridDim.x * 32) {
        const int u = blockIdx.y * 32 + (tid >> 3), m = u / p.n_heads;
        kv8_turn_q<HD, F32, PAIRS>(p, (int)a + m, min(last, (int)a + 32), r0 - P, u - m * p.n_heads, (tid & 7) * 8);
    }
}

template <int HD, bool F32> static void launch_append(const Kv8Append &p, bool queries, dim3 g, hipStream_t st) {
    const dim3 b(kKv8T);
    if (queries) {
        if (p.interleaved) k_kv8_queries<HD, F32, true><<<g, b, 0, st>>>(p);
        else k_kv8_queries<HD, F32, false><<<g, b, 0, st>>>(p);
    } else {
        if (p.interleaved) k_kv8_append<HD, F32, true><<<g, b, 0, st>>>(p);
        else k_kv8_append<HD, F32, false><<<g, b, 0, st>>>(p);
    }
    SD_HIP_CHECK(hipGetLastError());
}
static void launch_append(const Kv8Append &p, bool queries, dim3 g, hipStream_t st) {
    if (p.L.hd == 128) p.f32 ? launch_append<128, true>(p, queries, g, st) : launch_append<128, false>(p, queries, g, st);
    else p.f32 ? launch_append<64, true>(p, queries, g, st) : launch_append<64, false>(p, queries, g, st);
}
void launch_kv8_append(const Kv8Append &in, hipStream_t st) {
    if (in.seqs.rows < 1) return;
    Kv8Append p = in;
    const int seqs = p.seqs.n_seqs, kv = 2 * p.L.n_kv;
    // blocks that max_rows rows can touch; a sequence's are dealt round as many workgroups as even ragged lengths need
    const int64_t blocks = (p.seqs.max_rows + 30) / 32 + 1, mean = (p.seqs.rows / 32 + 3 * (int64_t)seqs - 1) / seqs;
    const int q = p.q ? (int)(((int64_t)std::min(32, p.seqs.max_rows) * p.n_heads + 31) / 32) : 0;
    // (a grid holds fewer than 2^32 threads)
    auto grid = [&](int64_t units) {
        const int64_t most = ((int64_t)1 << 23) / (units * seqs);
        if (most < 1) throw BackendError("append: too many sequences and heads in one call");
        return dim3((unsigned)std::min({blocks, 4 * mean, most}), (unsigned)units, (unsigned)seqs);
    };
    // many queries in a launch of their own
    const bool apart = q && (int64_t)p.seqs.rows * p.n_heads >= kApart;
    if (apart) launch_append(p, true, grid(q), st);
    launch_append(p, false, grid(kv + (apart ? 0 : q)), st);
}

// ---- read ----------------------------------------------------------------------
// A wave has 8 rows of 64 channels of one KV head's keys or values, kReadU times: lane
// 8 k + j the channels 8 j .. of row k.  Rows that are 8 positions of one group of a
// block share the bytes that their values lie in: then lane 8 k + j loads the 8
// positions of channel 8 j + k and the eight lanes exchange them; otherwise a lane
// picks its 8 bytes.  16384 rows of 8 heads, 34 MB of blocks and 67 MB of rows: 20 us,
// a large copy's rate (31 where every lane picks).
constexpr int kReadU = 2;
template <int HD>
__global__ __launch_bounds__(256) void k_kv8_read(const Kv8Layer L, const KvqRows rows, uint16_t *k_out, uint16_t *v_out) {
    constexpr int PARTS = HD / 64, GROUPS = 4 / PARTS;  // of 64 channels, of 8 rows
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool is_v = (int)blockIdx.y >= L.n_kv;
    const int h = is_v ? (int)blockIdx.y - L.n_kv : (int)blockIdx.y;
    uint16_t *out = is_v ? v_out : k_out;
    if (!out) return;
    const int r0 = ((int)blockIdx.x * GROUPS + wave / PARTS) * 8 * kReadU + (lane >> 3), c0 = wave % PARTS * 64 + (lane & 7) * 8;
    int slot[kReadU], page[kReadU];
#pragma unroll
    for (int u = 0; u < kReadU; u++) {
        const int r = r0 + 8 * u;
        page[u] = r < rows.n ? kvq_row_page(rows, L, r, slot[u]) : -1;
        if (page[u] < 0) slot[u] = 0;
    }
    uintx2 w[kReadU];
    Kv8Head head[kReadU];
    bool turn[kReadU];
#pragma unroll
    for (int u = 0; u < kReadU; u++) {
        const int k = slot[u] & 31, at = max(page[u], 0);
        const uint8_t *codes = L.codes(at, h, slot[u]) + (is_v ? 32 * HD : 0);
        head[u] = *L.head(at, h, slot[u]);
        const int first = __builtin_amdgcn_readfirstlane(slot[u]), of = __builtin_amdgcn_readfirstlane(page[u]);
        turn[u] = is_v && __builtin_amdgcn_ballot_w64(page[u] < 0 || of != page[u] || (first & 7) != 0 || slot[u] != first + (lane >> 3)) == 0;
        if (turn[u]) {
            w[u] = *(const uintx2 *)(codes + kv8_v_at(k & 24, c0 + (lane >> 3), HD));
        } else if (is_v) {
            w[u] = uintx2{0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++) w[u][i >> 2] |= (uint32_t)codes[kv8_v_at(k, c0 + i, HD)] << (8 * (i & 3));
        } else {
            w[u] = *(const uintx2 *)(codes + kv8_k_at(k, c0, HD));
        }
    }
#pragma unroll
    for (int u = 0; u < kReadU; u++) {
        if (turn[u]) w[u] = kv8_transpose(w[u], lane);
        uintx4 v = kv8_expand(w[u].x, w[u].y, head[u].scale[is_v]);
        if (head[u].nan[is_v] >> (slot[u] & 31) & 1) v = uintx4{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};
        if (page[u] >= 0) *(uintx4 *)(out + ((int64_t)(r0 + 8 * u) * L.n_kv + h) * HD + c0) = v;
    }
}

void launch_kv8_read(const Kv8Layer &L, const KvqRows &rows, uint16_t *k_out, uint16_t *v_out, hipStream_t st) {
    if (rows.n < 1) return;
    const int each = 8 * kReadU * (4 / (L.hd / 64));
    const dim3 g((unsigned)((rows.n + each - 1) / each), (unsigned)(2 * L.n_kv)), b(256);
    if (L.hd == 128) k_kv8_read<128><<<g, b, 0, st>>>(L, rows, k_out, v_out);
    else k_kv8_read<64><<<g, b, 0, st>>>(L, rows, k_out, v_out);
    SD_HIP_CHECK(hipGetLastError());
}

// ---- keep accepted tree rows ------------------------------------------------------
// One workgroup per (layer, KV head, keys or values): the accepted rows' codes go to
// LDS, with their scales, then the blocks from P's on are built again from what stays
// in front of P and the rows.
constexpr int kKeepMax = 128;
template <int HD, bool V>
__device__ void kv8_keep(Kv8Sh &sh, uint8_t (&code)[kKeepMax][HD], float (&scales)[kKeepMax], uint32_t (&bad)[kKeepMax],
                         const Kv8Layer &L, int h, const int *table, int P, const int *src, int n) {
    constexpr int C = HD / 8;
    const int tid = threadIdx.x;
    for (int i = tid; i < n * 8; i += kKv8T) {
        const int j = i >> 3, c0 = (i & 7) * 8, pos = P + src[j], page = table[pos >> L.page_shift];
        const uint8_t *b = L.codes(page, h, pos) + (V ? 32 * HD : 0);
#pragma unroll
        for (int n = 0; n < C; n++) {
            const int c = kv8_ch<HD>(c0, n);
            code[j][c] = b[V ? kv8_v_at(pos & 31, c, HD) : kv8_k_at(pos & 31, c, HD)];
        }
        if ((i & 7) == 0) {
            const Kv8Head *head = L.head(page, h, pos);
            scales[j] = head->scale[V];
            bad[j] = head->nan[V] >> (pos & 31) & 1;
        }
    }
    __syncthreads();
    const int k = tid >> 3, c0 = (tid & 7) * 8;
    for (int b = P >> 5; b * 32 < P + n; b++) {
        const int page = table[b * 32 >> L.page_shift], pos = b * 32 + k, j = pos - P;
        uint8_t *codes = L.codes(page, h, b * 32) + (V ? 32 * HD : 0);
        Kv8Head *head = L.head(page, h, b * 32);
        float scale = head->scale[V];
        uint32_t nans = head->nan[V];
        float x[C] = {};
        bool lost = false;
        kv8_held<HD, V>(codes, scale, x);
        if (j < 0) {
            lost = nans >> k & 1;
        } else if (j < n) {
#pragma unroll
            for (int c = 0; c < C; c++) x[c] = kv8_value(code[j][kv8_ch<HD>(c0, c)], scales[j]);
            lost = bad[j] != 0;
        }
        kv8_build<HD, V>(sh, x, j < n, lost, scale, nans);  // (its first barrier: the block has been read)
        kv8_codes_out<HD>(sh, codes);
        if (tid == 0) {
            head->scale[V] = scale;
            head->nan[V] = nans;
        }
        __syncthreads();
    }
}
template <int HD>
__global__ __launch_bounds__(kKv8T) void k_kv8_keep_tail(const Kv8Layer L0, int64_t layer_bytes, const int *table, int P,
                                                         const int *src, int n) {
    __shared__ Kv8Sh sh;
    __shared__ uint8_t code[kKeepMax][HD];
    __shared__ float scales[kKeepMax];
    __shared__ uint32_t bad[kKeepMax];
    Kv8Layer L = L0;
    const int u = blockIdx.x % (2 * L.n_kv);
    L.base += (int64_t)(blockIdx.x / (2 * L.n_kv)) * layer_bytes;
    if (u < L.n_kv) kv8_keep<HD, false>(sh, code, scales, bad, L, u, table, P, src, n);
    else kv8_keep<HD, true>(sh, code, scales, bad, L, u - L.n_kv, table, P, src, n);
}

void launch_kv8_keep_tail(const Kv8Layer &L0, int64_t layer_bytes, int n_layers, const int *table, int P, const int *src,
                          int n, hipStream_t st) {
    if (n < 1) return;
    if (n > kKeepMax) throw BackendError("keep_tail: at most 128 rows");
    const dim3 g((unsigned)(n_layers * 2 * L0.n_kv)), b(kKv8T);
    if (L0.hd == 128) k_kv8_keep_tail<128><<<g, b, 0, st>>>(L0, layer_bytes, table, P, src, n);
    else k_kv8_keep_tail<64><<<g, b, 0, st>>>(L0, layer_bytes, table, P, src, n);
    SD_HIP_CHECK(hipGetLastError());
}

}  // namespace sd
