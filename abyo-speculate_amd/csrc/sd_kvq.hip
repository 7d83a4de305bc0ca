// The 4-bit paged KV cache: appending rows (RoPE and quantisation on the
// way), reading them back, moving accepted tree rows.  The attention over it
// is in sd_kvq_attn.hip, the format and the block layout in sd_kvq.hpp.
#include "sd_buffer.hpp"
#include "sd_kvq_dev.hpp"

namespace sd {

// Where row r of a call lives: its page id, or -1 where the row is left out.
__device__ __forceinline__ int kvq_row_page(const KvqRows &t, const KvqLayer &L, int r, int &slot) {
    const int s = t.seq ? t.seq[r] : 0;
    slot = t.slot ? t.slot[r] : t.slot0 + r;
    if (s < 0 || s >= t.n_seqs || slot < 0) return -1;
    const int at = slot >> L.page_shift;
    if (at >= t.table_ld) return -1;
    const int page = t.table[(int64_t)s * t.table_ld + at];
    return page >= 0 && page < L.n_pages ? page : -1;
}

// ---- append --------------------------------------------------------------------
// The value of another lane of the same four (XOR 1 or 2) without LDS.
template <int X> __device__ __forceinline__ uint32_t quad_xor(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, X == 1 ? 0xB1 : 0x4E, 0xf, 0xf, true);
}
template <int X> __device__ __forceinline__ double quad_xor(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)quad_xor<X>((uint32_t)b) | ((uint64_t)quad_xor<X>((uint32_t)(b >> 32)) << 32));
}

// c + 8 of clamp(rint(x / d), -8, 7).  The product with 1 / d is within 2^-49
// of the quotient, so only a value that close to a half needs the division.
__device__ __forceinline__ uint32_t group_code(double x, double d, double rd) {
    const double y = x * rd;
    double r = rint(y);
    if (fabs(y - r) > 0.5 - 1e-9) r = rint(x / d);
    return (uint32_t)((int)fmin(fmax(r, -8.0), 7.0) + 8);
}

template <bool F32> __device__ __forceinline__ void load8(const void *base, int64_t at, float (&x)[8]) {
    if constexpr (F32) {
        const float4 a = *(const float4 *)((const float *)base + at), b = *(const float4 *)((const float *)base + at + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const half8 h = *(const half8 *)((const _Float16 *)base + at);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)h[i];
    }
}

// x[0..7] (channels 8 w ..) rotated in T: with neighbouring pairs inside the
// thread, with halves against channels 8 w +- hd / 2 (y).
template <typename T, int HD>
__device__ __forceinline__ void rotate8(const float (&x)[8], const float (&y)[8], const float *cos_r, const float *sin_r,
                                        int w, bool pairs, T (&out)[8]) {
    if (pairs) {
        const float4 c = *(const float4 *)(cos_r + 4 * w), s = *(const float4 *)(sin_r + 4 * w);
        const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const T a = x[2 * i], b = x[2 * i + 1], C = cc[i], S = ss[i];
            out[2 * i] = a * C - b * S;
            out[2 * i + 1] = b * C + a * S;
        }
    } else {
        const bool upper = w >= HD / 16;
        const int at = (8 * w) & (HD / 2 - 1);
        const float4 c0 = *(const float4 *)(cos_r + at), c1 = *(const float4 *)(cos_r + at + 4);
        const float4 s0 = *(const float4 *)(sin_r + at), s1 = *(const float4 *)(sin_r + at + 4);
        const float cc[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
        const float ss[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const T a = x[i], b = y[i], C = cc[i], S = upper ? ss[i] : -ss[i];
            out[i] = a * C + b * S;
        }
    }
}

__global__ __launch_bounds__(256) void k_kvq_tables(float *cos_t, float *sin_t, int64_t n, int half, double base) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const double a = (double)(i / half) * pow(base, -(double)(i % half) / half);
    cos_t[i] = (float)cos(a);
    sin_t[i] = (float)sin(a);
}
void launch_kvq_tables(float *cos_t, float *sin_t, int max_pos, int hd, double base, hipStream_t st) {
    const int64_t n = (int64_t)max_pos * (hd / 2);
    k_kvq_tables<<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st>>>(cos_t, sin_t, n, hd / 2, base);
    SD_HIP_CHECK(hipGetLastError());
}

constexpr int kAppendT = 256;

// c + 8 for a value that fp32 holds: the fp32 quotient is within 2^-22 of its
// own size of the exact one, so only a value that close to a half needs more.
__device__ __forceinline__ uint32_t group_code(float x, float d, float rd) {
    const float y = x * rd;
    float r = rintf(y);
    if (fabsf(y - r) > 0.5f - 1e-5f) r = (float)rint((double)x / (double)d);
    return (uint32_t)((int)fminf(fmaxf(r, -8.f), 7.f) + 8);
}

// the step of 32 channels from the extremes of four lanes' 8 each
template <typename T> __device__ __forceinline__ T quad_max(T v) {
    v = fmax(v, quad_xor<1>(v));
    return fmax(v, quad_xor<2>(v));
}
template <> __device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __uint_as_float(quad_xor<1>(__float_as_uint(v))));
    return fmaxf(v, __uint_as_float(quad_xor<2>(__float_as_uint(v))));
}
template <typename T> __device__ __forceinline__ _Float16 group_step(const T (&x)[8]) {
    T hi = x[0], lo = -x[0];
    uint32_t bad = x[0] != x[0];
#pragma unroll
    for (int i = 1; i < 8; i++) {
        hi = fmax(hi, x[i]);
        lo = fmax(lo, -x[i]);
        bad |= x[i] != x[i];
    }
    hi = quad_max(hi);
    lo = quad_max(lo);
    bad |= quad_xor<1>(bad);
    bad |= quad_xor<2>(bad);
    const T a = fmax(hi, lo);
    if (bad || !(a <= (T)65504)) return (_Float16)__builtin_nanf("");
    const _Float16 d = (_Float16)(float)(a * (T)0.125);
    return hi > lo ? -d : d;
}

// the codes of a word's 8 channels; 8s where the step is 0 or NaN
template <typename T> __device__ __forceinline__ uint32_t group_word(const T (&x)[8], _Float16 d, bool is_v) {
    if (!(d != (_Float16)0.f && d == d)) return 0x88888888u;
    const T dd = (T)(float)d, rd = (T)1 / dd;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int n = is_v ? i : (i >> 1) + 4 * (i & 1);
        word |= group_code(x[i], dd, rd) << (4 * n);
    }
    return word;
}

// One thread per 8 channels of one head of one row, so a group of 32 is four
// neighbouring lanes and its extremes two quad exchanges.  grid (rows, chunks of
// units): first the row's K and V heads, then its q heads, which keeps the two
// kinds of work in different workgroups and gives a single row three of them.
// K values are rotated and divided in f64: a code that lies at a border in fp32
// (about one value in a million) would depend on the order of two roundings.
// Values need no rotation, and fp32 with a check near the borders decides their
// codes; with the grid by rows that took append and read of 16384 rows from 136
// to 114 us.  Memory bounds it: 16384 fp16 rows of 32 query heads and 8 KV heads
// of 128 channels take 87 us, 74 at the rate of a large copy (4-byte words of codes
// 32 bytes apart: 235 MB are written where 172 would do); 2501 fp32 rows 20 (18).
template <int HD, bool F32>
__global__ __launch_bounds__(kAppendT) void k_kvq_append(const KvqAppend p, int kv_chunks) {
    constexpr int W = HD / 8, U = kAppendT / W;  // units of a workgroup
    const int r = blockIdx.x, w = threadIdx.x % W, unit = threadIdx.x / W, n_kv = p.L.n_kv;
    const bool is_q = (int)blockIdx.y >= kv_chunks;
    const int u = (is_q ? (int)blockIdx.y - kv_chunks : (int)blockIdx.y) * U + unit;
    if (u >= (is_q ? p.n_heads : 2 * n_kv)) return;
    const bool is_v = !is_q && u >= n_kv;
    const int h = is_v ? u - n_kv : u, other = (w + W / 2) % W;
    const bool pairs = p.interleaved != 0;
    // the row's values do not wait for its place
    float a[8], b[8] = {};
    {
        const void *src = is_q ? p.q : is_v ? p.v : p.k;
        const int64_t at = (int64_t)r * (is_q ? p.q_ld : is_v ? p.v_ld : p.k_ld) + h * HD;
        load8<F32>(src, at + 8 * w, a);
        if (!pairs && !is_v) load8<F32>(src, at + 8 * other, b);
    }
    int slot;
    const int page = kvq_row_page(p.rows, p.L, r, slot);
    const int pos = p.pos ? p.pos[r] : slot;
    if (page < 0 || pos < 0 || pos >= p.max_pos) return;
    const float *cos_r = p.cos_t + (int64_t)pos * (HD / 2), *sin_r = p.sin_t + (int64_t)pos * (HD / 2);
    if (is_q) {
        float o[8];
        rotate8<float, HD>(a, b, cos_r, sin_r, w, pairs, o);
        uintx4 v;
        v.x = (uint32_t)f2h(o[0]) | ((uint32_t)f2h(o[1]) << 16);
        v.y = (uint32_t)f2h(o[2]) | ((uint32_t)f2h(o[3]) << 16);
        v.z = (uint32_t)f2h(o[4]) | ((uint32_t)f2h(o[5]) << 16);
        v.w = (uint32_t)f2h(o[6]) | ((uint32_t)f2h(o[7]) << 16);
        *(uintx4 *)(p.q_out + (int64_t)r * p.q_out_row + (int64_t)h * p.q_out_head + 8 * w) = v;
        return;
    }
    const int k = slot & 31;
    uint8_t *blk = p.L.block(page, h, slot);
    if (is_v) {
        const _Float16 d = group_step(a);
        *(uint32_t *)(blk + kvq_v_code(k, w, HD)) = group_word(a, d, true);
        if ((w & 3) == 0) *(_Float16 *)(blk + kvq_v_step(k, w >> 2, HD)) = d;
    } else {
        double x[8];
        rotate8<double, HD>(a, b, cos_r, sin_r, w, pairs, x);
        const _Float16 d = group_step(x);
        *(uint32_t *)(blk + kvq_k_code(k, w, HD)) = group_word(x, d, false);
        if ((w & 3) == 0) *(_Float16 *)(blk + kvq_k_step(k, w >> 2, HD)) = d;
    }
}

void launch_kvq_append(const KvqAppend &p, hipStream_t st) {
    if (p.rows.n < 1) return;
    const int U = kAppendT / (p.L.hd / 8), kv = (2 * p.L.n_kv + U - 1) / U, q = p.q ? (p.n_heads + U - 1) / U : 0;
    const dim3 g((unsigned)p.rows.n, (unsigned)(kv + q)), b(kAppendT);
    if (p.L.hd == 128) {
        if (p.f32) k_kvq_append<128, true><<<g, b, 0, st>>>(p, kv);
        else k_kvq_append<128, false><<<g, b, 0, st>>>(p, kv);
    } else {
        if (p.f32) k_kvq_append<64, true><<<g, b, 0, st>>>(p, kv);
        else k_kvq_append<64, false><<<g, b, 0, st>>>(p, kv);
    }
    SD_HIP_CHECK(hipGetLastError());
}

// ---- read ----------------------------------------------------------------------
// The same threads the other way: 16384 rows of 8 heads 29 us, 18 at the rate of
// a large copy.  A workgroup has one row, whose 4-byte words lie 32 bytes apart,
// so that the seven rows beside it fetch the same sectors again.
template <int HD>
__global__ __launch_bounds__(kAppendT) void k_kvq_read(const KvqLayer L, const KvqRows rows, uint16_t *k_out,
                                                       uint16_t *v_out) {
    constexpr int W = HD / 8;
    const int r = blockIdx.x, w = threadIdx.x % W, u = blockIdx.y * (kAppendT / W) + threadIdx.x / W;
    if (u >= 2 * L.n_kv) return;
    const bool is_v = u >= L.n_kv;
    uint16_t *out = is_v ? v_out : k_out;
    int slot;
    const int page = kvq_row_page(rows, L, r, slot);
    if (!out || page < 0) return;
    const int h = is_v ? u - L.n_kv : u, k = slot & 31;
    const uint8_t *blk = L.block(page, h, slot);
    const _Float16 d = *(const _Float16 *)(blk + (is_v ? kvq_v_step(k, w >> 2, HD) : kvq_k_step(k, w >> 2, HD)));
    uint32_t word = *(const uint32_t *)(blk + (is_v ? kvq_v_code(k, w, HD) : kvq_k_code(k, w, HD)));
    if (is_v) {
        // channels in pairs (i, i + 4), as a K word has them
        uint32_t a = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) a |= ((word >> (4 * i)) & 15u) << (4 * ((i >> 1) + 4 * (i & 1)));
        word = a;
    }
    *(uintx4 *)(out + ((int64_t)r * L.n_kv + h) * HD + 8 * w) = kvq_expand_k(word, half2v{d, d});
}

void launch_kvq_read(const KvqLayer &L, const KvqRows &rows, uint16_t *k_out, uint16_t *v_out, hipStream_t st) {
    if (rows.n < 1) return;
    const int U = kAppendT / (L.hd / 8);
    const dim3 g((unsigned)rows.n, (unsigned)((2 * L.n_kv + U - 1) / U)), b(kAppendT);
    if (L.hd == 128) k_kvq_read<128><<<g, b, 0, st>>>(L, rows, k_out, v_out);
    else k_kvq_read<64><<<g, b, 0, st>>>(L, rows, k_out, v_out);
    SD_HIP_CHECK(hipGetLastError());
}

// ---- keep accepted tree rows ------------------------------------------------------
// One workgroup per (layer, KV head): the accepted rows are gathered into LDS
// and written back behind the prefix, as rows of one call may overlap.
constexpr int kKeepMax = 128;
template <int HD>
__global__ __launch_bounds__(256) void k_kvq_keep_tail(const KvqLayer L0, int64_t layer_bytes, const int *table, int P,
                                                       const int *src, int n) {
    constexpr int W = HD / 8, E = HD / 32;
    __shared__ uint32_t code[2][kKeepMax][W];
    __shared__ uint16_t step[2][kKeepMax][E];
    KvqLayer L = L0;
    L.base += (int64_t)(blockIdx.x / L.n_kv) * layer_bytes;
    const int h = blockIdx.x % L.n_kv;
    for (int i = threadIdx.x; i < n * W; i += 256) {
        const int j = i / W, w = i % W, pos = P + src[j], k = pos & 31;
        const uint8_t *b = L.block(table[pos >> L.page_shift], h, pos);
        code[0][j][w] = *(const uint32_t *)(b + kvq_k_code(k, w, HD));
        code[1][j][w] = *(const uint32_t *)(b + kvq_v_code(k, w, HD));
        if (w < E) {
            step[0][j][w] = *(const uint16_t *)(b + kvq_k_step(k, w, HD));
            step[1][j][w] = *(const uint16_t *)(b + kvq_v_step(k, w, HD));
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * W; i += 256) {
        const int j = i / W, w = i % W, pos = P + j, k = pos & 31;
        uint8_t *b = L.block(table[pos >> L.page_shift], h, pos);
        *(uint32_t *)(b + kvq_k_code(k, w, HD)) = code[0][j][w];
        *(uint32_t *)(b + kvq_v_code(k, w, HD)) = code[1][j][w];
        if (w < E) {
            *(uint16_t *)(b + kvq_k_step(k, w, HD)) = step[0][j][w];
            *(uint16_t *)(b + kvq_v_step(k, w, HD)) = step[1][j][w];
        }
    }
}

void launch_kvq_keep_tail(const KvqLayer &L0, int64_t layer_bytes, int n_layers, const int *table, int P,
                          const int *src, int n, hipStream_t st) {
    if (n < 1) return;
    if (n > kKeepMax) throw BackendError("keep_tail: at most 128 rows");
    const dim3 g((unsigned)(n_layers * L0.n_kv)), b(256);
    if (L0.hd == 128) k_kvq_keep_tail<128><<<g, b, 0, st>>>(L0, layer_bytes, table, P, src, n);
    else k_kvq_keep_tail<64><<<g, b, 0, st>>>(L0, layer_bytes, table, P, src, n);
    SD_HIP_CHECK(hipGetLastError());
}

}  // namespace sd
