// The 4-bit paged KV cache: layout, parameter blocks and launchers (sd_kvq.hip,
// sd_kvq_attn.hip) and the host handle (sd_kvpool.cpp).
//
// A group of 32 channels of one position and KV head shares one fp16 step d.
// With A the group's largest magnitude, |d| = fp16(fp32(A / 8)), negative when
// the largest magnitude is a positive number's alone, so that this number
// stands on -8; channel x has the code c = clamp(rint(x / d), -8, 7) and stands
// for fp16(d * c).  A group with a value that is not finite or exceeds 65504
// has d = NaN and stands for NaN.
//
// 32 positions of one KV head are a block of 36 * hd bytes, laid out so that
// every operand of the attention's 16x16x32 MFMA is a whole-word load of one
// lane (lane = r + 16 g) and so that a position's 8 channels are one 32-bit
// word: appending a position never reads or rewrites another position's bits.
//   K codes (16 hd) | K steps (2 hd) | V codes (16 hd) | V steps (2 hd)
// Position k (0..31) of a block is row rho = 4 (k >> 3) + (k & 3) of the key
// tile kt = (k >> 2) & 1: a lane group's 8 scores of the transposed product
// S^T = K Q^T are then the positions 8 g .. 8 g + 7, the ones whose values the
// lane holds for O^T = V^T P^T.
//   K word w (channels 8 w ..): hd 128 [kt][rho + 16 (w >> 2)][w & 3],
//                               hd 64  [rho + 16 (w >> 1)][kt][w & 1]
//     nibble n holds channel 8 w + 2 (n & 3) + (n >> 2)
//   K step of group e: [rho + 16 e][kt]
//   V word w: [w + (hd / 8) (k >> 3)][k & 7], nibble n holds channel 8 w + n
//   V step of group e: [e][k >> 3][k & 7]
// Codes are stored as c + 8.  A page holds page_tokens / 32 blocks of each KV
// head, head after head; a layer holds all pages.
#pragma once
#include <memory>
#include <vector>

#include "sd_common.hpp"
#include "sd_kernels.hpp"

namespace sd {

constexpr int kKvqBlock = 32;  // positions of a block
__host__ __device__ inline int kvq_block_bytes(int hd) { return 36 * hd; }
__host__ __device__ inline int kvq_k_code(int k, int w, int hd) {
    const int rho = 4 * (k >> 3) + (k & 3), kt = (k >> 2) & 1;
    return hd == 128 ? kt * 1024 + (rho + 16 * (w >> 2)) * 16 + (w & 3) * 4
                     : (rho + 16 * (w >> 1)) * 16 + kt * 8 + (w & 1) * 4;
}
__host__ __device__ inline int kvq_k_step(int k, int e, int hd) {
    const int rho = 4 * (k >> 3) + (k & 3), kt = (k >> 2) & 1;
    return 16 * hd + ((rho + 16 * e) * 2 + kt) * 2;
}
__host__ __device__ inline int kvq_v_code(int k, int w, int hd) {
    return 18 * hd + ((w + (hd / 8) * (k >> 3)) * 8 + (k & 7)) * 4;
}
__host__ __device__ inline int kvq_v_step(int k, int e, int hd) { return 34 * hd + ((e * 4 + (k >> 3)) * 8 + (k & 7)) * 2; }

// One layer of a pool as the kernels see it.
struct KvqLayer {
    uint8_t *base;
    int64_t page_bytes;
    int n_pages;
    int page_shift;  // log2(page_tokens), at least 5
    int n_kv, hd;
    // block of position `pos` of KV head h in page `page`
    __host__ __device__ uint8_t *block(int page, int h, int pos) const {
        const int bpp = 1 << (page_shift - 5);
        return base + (int64_t)page * page_bytes +
               (int64_t)(h * bpp + ((pos >> 5) & (bpp - 1))) * kvq_block_bytes(hd);
    }
};

// Where the rows of a call live: row r is position slot[r] (slot0 + r without
// slot) of sequence seq[r] (0 without seq), whose page slot / page_tokens is
// table[seq][...].  A row whose sequence, position or page lies outside is
// left out.
struct KvqRows {
    int n;
    const int *seq, *slot;
    int slot0;
    const int *table;
    int n_seqs, table_ld;
};

struct KvqAppend {
    KvqLayer L;
    KvqRows rows;
    const int *pos;             // rotation positions, or null: the slots
    const float *cos_t, *sin_t; // [max_pos][hd / 2]
    int max_pos;
    int interleaved;            // 1: pairs (2i, 2i+1); 0: pairs (i, i + hd/2)
    int n_heads;
    int f32;                    // rows are f32, else fp16
    const void *q, *k, *v;      // row strides in elements; q null: no queries
    int64_t q_ld, k_ld, v_ld;
    uint16_t *q_out;            // fp16; element c of head h of row r at q_out[r * q_out_row + h * q_out_head + c]
    int64_t q_out_row, q_out_head;
};
void launch_kvq_append(const KvqAppend &p, hipStream_t st);
// RoPE tables [max_pos][hd / 2]: cos and sin of pos * base^(-2i / hd), angles in f64
void launch_kvq_tables(float *cos_t, float *sin_t, int max_pos, int hd, double base, hipStream_t st);

// rows of a layer as fp16 [n][n_kv][hd]; either output may be null
void launch_kvq_read(const KvqLayer &L, const KvqRows &rows, uint16_t *k_out, uint16_t *v_out, hipStream_t st);

// position P + j <- position P + src[j] (src increasing, n <= 128) of every
// layer of one sequence whose pages are table[0 ..]
void launch_kvq_keep_tail(const KvqLayer &L0, int64_t layer_bytes, int n_layers, const int *table, int P,
                          const int *src, int n, hipStream_t st);

struct KvqAttn {
    KvqLayer L;
    const uint16_t *q;     // fp16; channel c of head h of row r at q[r * q_row + h * q_head + c]
    int64_t q_row, q_head;
    uint16_t *out;         // [rows][out_ld] fp16: heads side by side, or the next matmul's input (act_index)
    int64_t out_ld;
    int out_act;           // 0: plain rows; 1: fragment order; 2: operand order
    int rows;              // rows of q and out
    int n_seqs;
    const int *row_start;  // [n_seqs + 1]; null: one sequence of all rows, len0 positions
    const int *kv_len;     // [n_seqs] positions held, the sequence's rows among them (the last ones)
    int len0;
    const int *table;
    int table_ld;
    const uint64_t *mask;  // [rows][mask_words]: bit j = row j of the same sequence; null: causal
    int mask_words;
    int max_rows;          // most rows of one sequence
    int n_heads, n_rep;
    float scale;
    // from the plan
    int nsplit, tile_q, tiles, chunk, groups;
    float *part_o, *part_ml;
};
// The work split of a call: query tiles, key splits and the workspace they need.
struct KvqPlan {
    int tile_q, tiles, nsplit, chunk;  // queries of a tile, tiles, key ranges, blocks of a range
    size_t ws_bytes;
};
KvqPlan kvq_attn_plan(int n_heads, int n_kv, int hd, int n_seqs, int max_rows, int64_t max_len, int cus);
void launch_kvq_attention(const KvqAttn &p, const KvqPlan &plan, void *ws, hipStream_t st);

}  // namespace sd
