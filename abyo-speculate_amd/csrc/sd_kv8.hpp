// The 8-bit paged KV cache: layout, parameter blocks and launchers (sd_kv8.hip,
// sd_kv8_attn.hip, sd_kv8_weights.hip, sd_kv8_evict.hip); the host handle is in
// sd_kvpool.cpp.
//
// 32 positions of one KV head are a block, whose keys and whose values have one
// scale each: the smallest 2^E, E in [-15, 8], with A <= 448 * 2^E, A the largest
// magnitude of what the block holds.  A value x is held as the 8-bit float (e4m3,
// finite, up to 448) nearest to x / 2^E, halves to even, and stands for the code
// times 2^E, which fp16 holds exactly (with E = 8 codes end at 240: 65536 is none).  A row (one position of a head, keys or
// values) with a value that is not finite or above 65504 in magnitude stands for
// NaN in every channel: a bit in the block's header, its codes are 0, so that no
// code is ever NaN.  The scale being a power of two, what a block holds changes its
// scale without loss, except that values below 2^(E - 6) are rounded to multiples
// of 2^(E - 9).
//
// A block's codes are 64 * hd bytes, laid out as the operands of the attention's
// 16x16x32 MFMA (lane = r + 16 g), 1 KiB of 16 bytes a lane at a time:
//   K: position k (0..31) is row rho = 4 (k >> 3) + (k & 3) of the key tile
//      kt = (k >> 2) & 1, so that a lane group's 8 scores of the transposed product
//      S^T = K Q^T are the positions 8 g .. 8 g + 7; lane rho + 16 g has the
//      channels (hd / 4) g ..: [kt][16 channels each][lane][16]
//   V: lane r + 16 g has the positions 8 g .. of the channels (hd / 16) r ..:
//      [two channels each][lane][channel][8 positions]
// The header (16 bytes) is the scales as fp32 and a bit for each NaN row.  A page
// holds page_tokens / 32 blocks of each KV head, head after head, then their headers
// in the same order; a layer holds all pages.
#pragma once
#include "sd_kvq.hpp"

namespace sd {

constexpr int kKv8Block = 32;
constexpr int kKv8MaxLen = 0x7fffffc0;  // positions of a sequence
constexpr int kKv8MaxEvict = 1 << 30;    // of one that is cut down
constexpr int kKv8MinExp = -15, kKv8MaxExp = 8;

struct Kv8Head {
    float scale[2];   // of the keys and the values
    uint32_t nan[2];  // bit k: position k's row is NaN
};
static_assert(sizeof(Kv8Head) == 16, "one 16-byte access");

__host__ __device__ inline int kv8_block_bytes(int hd) { return 64 * hd; }
__host__ __device__ inline int64_t kv8_page_bytes(int n_kv, int hd, int page_tokens) {
    return (int64_t)n_kv * (page_tokens / kKv8Block) * (kv8_block_bytes(hd) + (int)sizeof(Kv8Head));
}
__host__ __device__ inline int kv8_k_at(int k, int c, int hd) {
    const int rho = 4 * (k >> 3) + (k & 3), kt = (k >> 2) & 1;
    return hd == 128 ? kt * 2048 + ((c >> 4) & 1) * 1024 + (rho + 16 * (c >> 5)) * 16 + (c & 15)
                     : kt * 1024 + (rho + 16 * (c >> 4)) * 16 + (c & 15);
}
// (from the block's values, which lie 32 hd bytes behind its keys)
__host__ __device__ inline int kv8_v_at(int k, int c, int hd) {
    const int n = hd / 16, r = c / n, d = c % n;
    return (d >> 1) * 1024 + (r + 16 * (k >> 3)) * 16 + (d & 1) * 8 + (k & 7);
}

// One layer of a pool as the kernels see it.
struct Kv8Layer : KvqLayer {
    __host__ __device__ Kv8Layer() : KvqLayer{} {}
    __host__ __device__ explicit Kv8Layer(const KvqLayer &l) : KvqLayer(l) {}
    __host__ __device__ int blocks() const { return 1 << (page_shift - 5); }
    __host__ __device__ int index(int h, int pos) const { return h * blocks() + ((pos >> 5) & (blocks() - 1)); }
    // codes and header of the block of position `pos` of KV head h in page `page`
    __host__ __device__ uint8_t *codes(int page, int h, int pos) const {
        return base + (int64_t)page * page_bytes + (int64_t)index(h, pos) * kv8_block_bytes(hd);
    }
    __host__ __device__ Kv8Head *head(int page, int h, int pos) const {
        return (Kv8Head *)(base + (int64_t)page * page_bytes + (int64_t)n_kv * blocks() * kv8_block_bytes(hd)) + index(h, pos);
    }
};

// Rows row_start[s] .. row_start[s + 1) of a call are the last positions of
// sequence s, which holds kv_len[s]; its page slot / page_tokens is table[s][...].
struct Kv8Seqs {
    int rows, n_seqs, max_rows;
    const int *row_start;  // null: one sequence of all rows, len0 positions
    const int *kv_len;
    int len0;
    const int *table;
    int table_ld;
};

struct Kv8Append {
    Kv8Layer L;
    Kv8Seqs seqs;
    const int *pos;             // rotation positions, or null: the rows' own
    const float *cos_t, *sin_t; // [max_pos][hd / 2]
    int max_pos;
    int interleaved;            // 1: pairs (2i, 2i+1); 0: pairs (i, i + hd/2)
    int n_heads;
    int f32;                    // rows are f32, else fp16
    const void *q, *k, *v;      // row strides in elements; q null: no queries
    int64_t q_ld, k_ld, v_ld;
    uint16_t *q_out;            // fp16 [rows][n_heads][hd]
};
void launch_kv8_append(const Kv8Append &p, hipStream_t st);

// rows of a layer as fp16 [n][n_kv][hd]; either output may be null
void launch_kv8_read(const Kv8Layer &L, const KvqRows &rows, uint16_t *k_out, uint16_t *v_out, hipStream_t st);

// position P + j <- position P + src[j] (src increasing, n <= 128) of every layer
// of one sequence whose pages are table[0 ..], which then ends at P + n
void launch_kv8_keep_tail(const Kv8Layer &L0, int64_t layer_bytes, int n_layers, const int *table, int P, const int *src,
                          int n, hipStream_t st);

// Division by a number that the host knows, of n < 2^31: with 2^L >= d, m = floor(2^(31 + L) / d) + 1
// is at most 2^L / 2^(31 + L) of a quotient's unit too large for each unit of n.
struct Kv8Div {
    uint32_t d, m;
    int shift;
    static Kv8Div by(uint32_t d) {
        int l = 0;
        while ((1ull << l) < d) l++;
        return {d, (uint32_t)((1ull << (31 + l)) / d + 1), 31 + l};
    }
    __device__ __forceinline__ uint32_t quot(uint32_t n) const { return (uint32_t)(((uint64_t)n * m) >> shift); }
};

// Attention: the 4-bit one's parameters (L the 8-bit layer's), and
struct Kv8Attn : KvqAttn {
    int window, sinks;  // 0: no window; else row p sees of what its mask shows the positions below sinks and above p - window
    float *lse;         // [rows][n_heads] ln of the sum of exp(score), or null
    int min_blocks;     // of a key range, from the plan
    Kv8Div by_rep, by_kv, by_tiles, by_groups;  // n_rep, KV heads, tiles, groups
};
KvqPlan kv8_attn_plan(int n_heads, int n_kv, int n_seqs, int max_rows, int64_t max_len, int window, int sinks, int cus);
void launch_kv8_attention(const Kv8Attn &p, const KvqPlan &plan, void *ws, hipStream_t st);

// out[s][h][j] = decay * in[s][h][j] + what position j of sequence s gets from its
// rows' weights in the query heads of KV head h (p.lse is read); anew: the first
// term is 0 for the positions of the rows themselves
struct Kv8Weights {
    Kv8Attn a;
    const float *in;  // or null: zeros
    float *out;
    int64_t ld;
    float decay;
    int anew;
    int64_t max_len;
    int cus;
};
void launch_kv8_weights(const Kv8Weights &p, hipStream_t st);

struct Kv8Evict {
    Kv8Layer L;
    int n_seqs;
    const int *kv_len, *table;
    int table_ld;
    const int *new_table;  // null: in place
    int new_ld;
    const float *scores;   // [n_seqs][n_kv][scores_ld]
    int64_t scores_ld;
    float *scores_out;     // or null
    int64_t scores_out_ld;
    int budget, sinks, recent;
    int *kept;             // [n_seqs][n_kv][budget]
    int *new_len;          // [n_seqs]
};
// allows the kernels their LDS on the current device; once before the first call there
void kv8_prepare();
size_t kv8_evict_ws_bytes(int n_seqs, int n_kv, int hd, int budget);
void launch_kv8_evict(const Kv8Evict &p, void *ws, hipStream_t st);

}  // namespace sd
