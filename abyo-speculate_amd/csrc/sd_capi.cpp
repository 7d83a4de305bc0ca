// extern "C" boundary (include/speculate_hip.h) over Model / Decoder.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <string>

#include "speculate_hip.h"
#include "sd_model.hpp"
#include "sd_common.hpp"
#include "sd_draft.hpp"
#include "sd_gguf.hpp"
#include "sd_kvpool.hpp"
#include "sd_qcodes.hpp"
#include "sd_tiles.hpp"

struct sd_model {
    std::unique_ptr<sd::Model> model;
    std::unique_ptr<sd::Decoder> dec;
};

struct sd_gguf {
    std::unique_ptr<sd::GgufFile> file;
};

struct sd_draft2 {
    std::unique_ptr<sd::Draft2> d;
};
struct sd_draft3 {
    std::unique_ptr<sd::Draft3> d;
};

struct sd_kvpool {
    std::unique_ptr<sd::KvPool> p;
};
struct sd_kv8 {
    std::unique_ptr<sd::KvPool> p;
};
struct sd_sampler {
    std::unique_ptr<sd::Sampler> s;
};

static thread_local std::string g_err;

template <typename F> static sd_status guard(F &&f) {
    try {
        f();
        return SD_OK;
    } catch (const sd::SamplingError &e) {
        g_err = e.what();
        return SD_ERR_SAMPLING;
    } catch (const sd::RollbackError &e) {
        g_err = e.what();
        return SD_ERR_ROLLBACK;
    } catch (const sd::ArgError &e) {
        g_err = e.what();
        return SD_ERR_ARG;
    } catch (const sd::UnsupportedError &e) {
        g_err = e.what();
        return SD_ERR_UNSUPPORTED;
    } catch (const sd::BackendError &e) {
        g_err = e.what();
        return SD_ERR_BACKEND;
    } catch (const std::exception &e) {
        g_err = e.what();
        return SD_ERR_BACKEND;
    }
}

static void need(const sd_model *m) {
    if (!m || !m->model) throw sd::ArgError("null model handle");
}
static void need_weights(const sd_model *m) {
    need(m);
    if (!m->model->weights_ready()) throw sd::ArgError("model weights are not fully set");
}
static void need(const sd_kvpool *c) {
    if (!c || !c->p) throw sd::ArgError("null pool handle");
}
static void need(const sd_kv8 *c) {
    if (!c || !c->p) throw sd::ArgError("null pool handle");
}
// elements of a row: the caller's stride, or a dense row's
static int64_t row_stride(size_t ld, int64_t dense, const char *what) {
    if (ld == 0) return dense;
    if (ld > ((size_t)1 << 40) || (int64_t)ld < dense) throw sd::ArgError(std::string(what) + ": rows overlap");
    return (int64_t)ld;
}
static void need_aligned(const void *p, int64_t row_bytes, int align, const char *what) {
    if ((uintptr_t)p % align || row_bytes % align)
        throw sd::ArgError(std::string(what) + ": rows must start at multiples of " + std::to_string(align) + " bytes");
}
static sd::KvqRows kv_rows(const sd_kv_rows *r) {
    if (!r || !r->slot || !r->table) throw sd::ArgError("null argument");
    // a grid holds fewer than 2^32 threads, 256 of them to a row
    if (r->n > ((size_t)1 << 23)) throw sd::ArgError("at most 2^23 rows");
    if (r->n_seqs < 1 || r->table_ld < 1) throw sd::ArgError("n_seqs and table_ld must be positive");
    return sd::KvqRows{(int)r->n, r->seq, r->slot, 0, r->table, r->n_seqs, r->table_ld};
}
static std::unique_ptr<sd::KvPool> make_pool(const sd_kvpool_config &cfg, int bits) {
    sd::KvPoolCfg c;
    c.n_layers = cfg.n_layers;
    c.n_heads = cfg.n_heads;
    c.n_kv_heads = cfg.n_kv_heads;
    c.head_dim = cfg.head_dim;
    c.n_pages = cfg.n_pages;
    c.page_tokens = cfg.page_tokens;
    c.max_pos = cfg.max_pos;
    c.interleaved = cfg.interleaved != 0;
    c.rope_theta = cfg.rope_theta;
    c.device = cfg.device;
    c.bits = bits;
    if (c.max_pos < 1) throw sd::ArgError("kvpool: max_pos must be positive");
    return std::make_unique<sd::KvPool>(c);
}
// A window of as many positions as a sequence can have is none; the kernels' sums of
// positions and windows are of 32 bits.
static void kv8_window(const sd_kv_window *win, int &window, int &sinks) {
    window = sinks = 0;
    if (!win || win->window >= (size_t)sd::kKv8MaxLen) return;
    if (win->window > ((size_t)1 << 30)) throw sd::ArgError("window must be at most 2^30, or from 2^31 - 64 on none");
    window = (int)win->window;
    sinks = (int)std::min(win->sinks, (size_t)sd::kKv8MaxLen);
}
// What an attention call and a call for its weights have in common: the rows, the
// sequences, the mask and the window of a query over an 8-bit pool.
static sd::Kv8Attn kv8_query(const sd::KvPool &P, int32_t layer, const sd_kv_query *qy, const sd_kv_window *win) {
    P.check_layer(layer);
    if (!qy->q || !qy->row_start || !qy->kv_len || !qy->table) throw sd::ArgError("null argument");
    if (qy->n_seqs < 1 || qy->table_ld < 1) throw sd::ArgError("n_seqs and table_ld must be positive");
    if (qy->mask && qy->mask_words < 1) throw sd::ArgError("mask_words must be positive");
    if (!std::isfinite(qy->scale * 1.4426950408889634f)) throw sd::ArgError("scale must be finite, in base 2 too");
    const int hd = P.cfg.head_dim;
    const size_t most = (size_t)1 << 30;
    sd::Kv8Attn a{};
    a.L = P.layer(layer);
    a.q = qy->q;
    a.q_row = row_stride(qy->q_ld, (int64_t)P.cfg.n_heads * hd, "q");
    a.q_head = hd;
    need_aligned(a.q, a.q_row * 2, 16, "q");
    a.rows = (int)std::min(qy->rows, most);
    a.n_seqs = qy->n_seqs;
    a.row_start = qy->row_start;
    a.kv_len = qy->kv_len;
    a.table = qy->table;
    a.table_ld = qy->table_ld;
    a.mask = qy->mask;
    a.mask_words = qy->mask_words;
    a.max_rows = (int)std::min(qy->max_rows, most);
    a.n_heads = P.cfg.n_heads;
    a.n_rep = P.cfg.n_heads / P.cfg.n_kv_heads;
    a.scale = qy->scale == 0.f ? (float)(1.0 / std::sqrt((double)hd)) : qy->scale;
    kv8_window(win, a.window, a.sinks);
    return a;
}
static sd::KvqPlan kv8_plan(const sd::KvPool &P, size_t rows, size_t n_seqs, size_t max_rows, size_t max_len,
                            const sd_kv_window *win) {
    const size_t most = (size_t)1 << 40;
    int window, sinks;
    kv8_window(win, window, sinks);
    return P.plan((int64_t)std::min(rows, most), (int64_t)std::min(n_seqs, most), (int64_t)std::min(max_rows, most),
                  (int64_t)std::min(max_len, most), window, sinks);
}
// one range of memory
static sd::RowBytes bytes_at(const void *p, int64_t bytes) { return {p, 0, bytes, 1}; }
static void setdev(sd_model *m) { SD_HIP_CHECK(hipSetDevice(m->model->cfg.device)); }

extern "C" {

const char *sd_last_error(void) { return g_err.c_str(); }

sd_status sd_model_create(const sd_config *cfg, sd_model **out) {
    return guard([&] {
        if (!cfg || !out) throw sd::ArgError("null argument");
        *out = nullptr;
        sd::ModelCfg c;
        c.arch = cfg->arch;
        if (c.arch != SD_ARCH_LLAMA && c.arch != SD_ARCH_QWEN2) throw sd::ArgError("unknown arch");
        c.n_layers = cfg->n_layers;
        c.hidden = cfg->hidden;
        c.n_heads = cfg->n_heads;
        c.n_kv_heads = cfg->n_kv_heads;
        c.head_dim = cfg->head_dim;
        c.ffn = cfg->ffn;
        c.vocab = cfg->vocab;
        c.rope_theta = cfg->rope_theta;
        c.rms_eps = cfg->rms_eps;
        c.ctx_len = cfg->ctx_len;
        c.max_batch = cfg->max_batch;
        c.tied_output = cfg->tied_output;
        c.device = cfg->device;
        if (c.hidden != c.n_heads * c.head_dim) throw sd::UnsupportedError("hidden must equal n_heads * head_dim");
        auto h = std::make_unique<sd_model>();
        h->model = std::make_unique<sd::Model>(c);
        h->dec = std::make_unique<sd::Decoder>(h->model.get());
        // set-up of the allocation-free entry points: this device's scratch
        // address, resolved while the device is current (Model set it)
        sd::noalloc_scratch(c.device);
        *out = h.release();
    });
}

void sd_model_destroy(sd_model *m) { delete m; }

sd_status sd_model_set_tensor(sd_model *m, int32_t layer, int32_t kind, int32_t fmt, const void *data, size_t bytes) {
    return guard([&] {
        need(m);
        if (!data) throw sd::ArgError("null data");
        m->model->set_tensor(layer, kind, fmt, data, bytes);
        m->dec->last_valid = false;
    });
}

sd_status sd_model_get_tensor(sd_model *m, int32_t layer, int32_t kind, void *out, size_t bytes) {
    return guard([&] {
        need(m);
        if (!out) throw sd::ArgError("null output");
        m->model->get_tensor(layer, kind, out, bytes);
    });
}

sd_status sd_model_tensor_info(sd_model *m, int32_t layer, int32_t kind, int32_t *fmt, int32_t *rows, int32_t *cols,
                               size_t *gguf_bytes) {
    return guard([&] {
        need(m);
        int f, r, k;
        size_t b;
        m->model->tensor_info(layer, kind, &f, &r, &k, &b);
        if (fmt) *fmt = f;
        if (rows) *rows = r;
        if (cols) *cols = k;
        if (gguf_bytes) *gguf_bytes = b;
    });
}

sd_status sd_model_synthesize(sd_model *m, int32_t mix, uint64_t seed, float stdv) {
    return guard([&] {
        need(m);
        m->model->synthesize(mix, seed, stdv);
        m->dec->last_valid = false;
    });
}

sd_status sd_gguf_open(const char *path, sd_gguf **out) {
    return guard([&] {
        if (!path || !out) throw sd::ArgError("null argument");
        *out = nullptr;
        auto g = std::make_unique<sd_gguf>();
        g->file = std::make_unique<sd::GgufFile>(path);
        *out = g.release();
    });
}

void sd_gguf_close(sd_gguf *g) { delete g; }

static const sd::GgufFile &gfile(const sd_gguf *g) {
    if (!g || !g->file) throw sd::ArgError("null gguf handle");
    return *g->file;
}

sd_status sd_gguf_config(const sd_gguf *g, int32_t arch, sd_config *cfg) {
    return guard([&] {
        if (!cfg) throw sd::ArgError("null argument");
        const sd::ModelCfg c = gfile(g).config(arch);
        sd_config o;
        o.arch = c.arch;
        o.n_layers = c.n_layers;
        o.hidden = c.hidden;
        o.n_heads = c.n_heads;
        o.n_kv_heads = c.n_kv_heads;
        o.head_dim = c.head_dim;
        o.ffn = c.ffn;
        o.vocab = c.vocab;
        o.rope_theta = c.rope_theta;
        o.rms_eps = c.rms_eps;
        o.ctx_len = c.ctx_len;
        o.max_batch = c.max_batch;
        o.tied_output = c.tied_output;
        o.device = c.device;
        *cfg = o;
    });
}

sd_status sd_gguf_layout(const sd_gguf *g, uint32_t *version, uint64_t *alignment, uint64_t *data_offset) {
    return guard([&] {
        const sd::GgufFile &f = gfile(g);
        if (version) *version = f.version;
        if (alignment) *alignment = f.alignment;
        if (data_offset) *data_offset = f.data_start;
    });
}

size_t sd_gguf_tensor_count(const sd_gguf *g) { return g && g->file ? g->file->tensors.size() : 0; }

sd_status sd_gguf_tensor_info(const sd_gguf *g, const char *name, int32_t *type, int32_t *n_dims, uint64_t *ne,
                              uint64_t *offset) {
    return guard([&] {
        if (!name) throw sd::ArgError("null name");
        const sd::GgufTensor &t = gfile(g).tensor(name);
        if (type) *type = (int32_t)t.type;
        if (n_dims) *n_dims = (int32_t)t.n_dims;
        if (ne)
            for (int d = 0; d < 4; d++) ne[d] = t.ne[d];
        if (offset) *offset = t.offset;
    });
}

sd_status sd_model_load_gguf(sd_model *m, const sd_gguf *g) {
    return guard([&] {
        need(m);
        const sd::GgufFile &f = gfile(g);
        f.load(*m->model);
        m->dec->last_valid = false;
    });
}

sd_status sd_model_dequant_tensor(sd_model *m, int32_t layer, int32_t kind, float *out) {
    return guard([&] {
        need(m);
        if (!out) throw sd::ArgError("null output");
        m->model->dequant_tensor(layer, kind, out);
    });
}

sd_status sd_model_qmatmul(sd_model *m, int32_t layer, int32_t kind, const float *x, size_t rows, float *y) {
    return guard([&] {
        need(m);
        if (!x || !y) throw sd::ArgError("null argument");
        m->model->qmatmul(layer, kind, x, (int)rows, y);
    });
}

sd_status sd_model_qmatmul_noalloc(sd_model *m, int32_t layer, int32_t kind, const float *x_dev, size_t rows,
                                   float *y_dev, void *stream) {
    return guard([&] {
        need(m);
        if (!x_dev || !y_dev) throw sd::ArgError("null argument");
        if (rows < 1 || rows > 128) throw sd::ArgError("rows must be in [1, 128]");
        setdev(m);
        // resolved at sd_model_create for this device; a kept pointer, no allocation
        void *scr = sd::noalloc_scratch(m->model->cfg.device);
        m->model->qmatmul_into(layer, kind, x_dev, (int)rows, y_dev, (hipStream_t)stream, scr);
    });
}

sd_status sd_bench_qmatmul(sd_model *m, int32_t layer, int32_t kind, size_t rows, int32_t iters, double *us,
                           double *bytes) {
    return guard([&] {
        need_weights(m);
        if (!us) throw sd::ArgError("null argument");
        *us = m->model->bench_qmatmul(layer, kind, (int)rows, iters, bytes);
    });
}

size_t sd_vocab_size(const sd_model *m) { return m && m->model ? (size_t)m->model->cfg.vocab : 0; }
size_t sd_history_len(const sd_model *m) { return m && m->dec ? m->dec->history.size() : 0; }
size_t sd_history(const sd_model *m, uint32_t *out, size_t cap) {
    if (!m || !m->dec) return 0;
    const size_t n = std::min(cap, m->dec->history.size());
    if (out && n) std::memcpy(out, m->dec->history.data(), n * 4);
    return n;
}
void sd_reset(sd_model *m) {
    if (m && m->dec) m->dec->reset();
}
size_t sd_num_hidden_layers(const sd_model *m) { return m && m->model ? (size_t)m->model->cfg.n_layers : 0; }
size_t sd_hidden_size(const sd_model *m) { return m && m->model ? (size_t)m->model->cfg.hidden : 0; }

sd_status sd_observe(sd_model *m, const uint32_t *ids, size_t n) {
    return guard([&] {
        need_weights(m);
        if (n && !ids) throw sd::ArgError("null ids");
        setdev(m);
        m->dec->observe(ids, n);
    });
}

sd_status sd_next_logits(sd_model *m, float *out) {
    return guard([&] {
        need_weights(m);
        setdev(m);
        m->dec->next_logits(out);
    });
}

sd_status sd_batched_logits(sd_model *m, const uint32_t *drafts, size_t k, float *out) {
    return guard([&] {
        need_weights(m);
        if (k && !drafts) throw sd::ArgError("null drafts");
        setdev(m);
        m->dec->batched_logits(drafts, k, out);
    });
}

sd_status sd_rollback_to(sd_model *m, size_t len) {
    return guard([&] {
        need(m);
        m->dec->rollback_to(len);
    });
}

sd_status sd_set_eos_token_ids(sd_model *m, const uint32_t *ids, size_t n) {
    return guard([&] {
        need(m);
        if (n && !ids) throw sd::ArgError("null ids");
        m->dec->eos.assign(ids, ids + n);
    });
}

size_t sd_eos_token_ids(const sd_model *m, uint32_t *out, size_t cap) {
    if (!m || !m->dec) return 0;
    const size_t n = std::min(cap, m->dec->eos.size());
    if (out && n) std::memcpy(out, m->dec->eos.data(), n * 4);
    return m->dec->eos.size();
}

sd_status sd_tree_logits_keep_kv(sd_model *m, const uint32_t *tokens, const uint32_t *parents, size_t n,
                                 float *out_logits, float *out_hidden) {
    return guard([&] {
        need_weights(m);
        if (!tokens || !parents) throw sd::ArgError("null tree");
        setdev(m);
        m->dec->tree_logits_keep_kv(tokens, parents, n, out_logits, out_hidden);
    });
}

sd_status sd_tree_logits(sd_model *m, const uint32_t *tokens, const uint32_t *parents, size_t n, float *out_logits) {
    return guard([&] {
        need_weights(m);
        if (!tokens || !parents) throw sd::ArgError("null tree");
        setdev(m);
        m->dec->tree_logits(tokens, parents, n, out_logits);
    });
}

sd_status sd_commit_tree_path(sd_model *m, const uint32_t *tokens, const uint32_t *parents, size_t n,
                              const uint32_t *accepted, size_t n_accepted) {
    return guard([&] {
        need_weights(m);
        if (!tokens || !parents || (n_accepted && !accepted)) throw sd::ArgError("null argument");
        setdev(m);
        m->dec->commit_tree_path(tokens, parents, n, accepted, n_accepted);
    });
}

sd_status sd_last_hidden_state(sd_model *m, float *out) {
    return guard([&] {
        need_weights(m);
        setdev(m);
        m->dec->last_hidden_state(out);
    });
}

sd_status sd_observe_returning_last_hidden(sd_model *m, const uint32_t *ids, size_t n, float *out) {
    return guard([&] {
        need_weights(m);
        if (n && !ids) throw sd::ArgError("null ids");
        setdev(m);
        m->dec->observe_returning_last_hidden(ids, n, out);
    });
}

sd_status sd_last_hidden_states_multi(sd_model *m, const uint32_t *layers, size_t n_layers, float *out_final,
                                      float *out_layers) {
    return guard([&] {
        need_weights(m);
        if (n_layers && !layers) throw sd::ArgError("null layers");
        setdev(m);
        m->dec->last_hidden_states_multi(layers, n_layers, out_final, out_layers);
    });
}

sd_status sd_apply_lm_head(sd_model *m, const float *hidden, size_t rows, float *out) {
    return guard([&] {
        need_weights(m);
        if (!hidden || !out) throw sd::ArgError("null argument");
        setdev(m);
        m->model->lm_head_rows(hidden, (int)rows, out);
    });
}

sd_status sd_embed_tokens(sd_model *m, const uint32_t *ids, size_t n, float *out) {
    return guard([&] {
        need_weights(m);
        if (!ids || !out) throw sd::ArgError("null argument");
        setdev(m);
        std::vector<int> v(ids, ids + n);
        for (size_t i = 0; i < n; i++)
            if (ids[i] >= (uint32_t)m->model->cfg.vocab) throw sd::ArgError("token id out of range");
        m->model->embed_rows(v.data(), (int)n, out);
    });
}

sd_status sd_verify_greedy_linear(sd_model *m, const uint32_t *drafts, size_t k, uint32_t *commits,
                                  size_t *n_commit, size_t *n_accepted) {
    return guard([&] {
        need_weights(m);
        if ((k && !drafts) || !commits || !n_commit || !n_accepted) throw sd::ArgError("null argument");
        setdev(m);
        m->dec->verify_greedy_linear(drafts, k, commits, n_commit, n_accepted);
    });
}

sd_status sd_verify_greedy_tree(sd_model *m, const uint32_t *tokens, const uint32_t *parents, size_t n,
                                int32_t strict, uint32_t *path, size_t *path_len, uint32_t *bonus,
                                int32_t *bonus_node, uint32_t *committed, size_t *n_committed, size_t *keep_len,
                                int32_t *stop) {
    return guard([&] {
        need_weights(m);
        if (!tokens || !parents || !path || !path_len || !bonus || !bonus_node || !n_committed || !keep_len || !stop)
            throw sd::ArgError("null argument");
        setdev(m);
        m->dec->verify_greedy_tree(tokens, parents, n, strict, path, path_len, bonus, bonus_node, committed,
                                   n_committed, keep_len, stop);
    });
}

sd_status sd_verify_rejection_linear(sd_model *m, const uint32_t *drafts, size_t k, const float *q_rows,
                                     const float *uniforms, size_t n_uniforms, float temperature, size_t max_commit,
                                     uint32_t *commits, size_t *n_commit, size_t *n_accepted, size_t *n_used) {
    return guard([&] {
        need_weights(m);
        if ((k && (!drafts || !q_rows)) || !uniforms || !commits || !n_commit || !n_accepted || !n_used)
            throw sd::ArgError("null argument");
        setdev(m);
        m->dec->verify_rejection_linear(drafts, k, q_rows, uniforms, n_uniforms, temperature, max_commit, commits,
                                        n_commit, n_accepted, n_used);
    });
}

sd_status sd_verify_rejection_linear_device_q(sd_model *m, const uint32_t *drafts, size_t k, const float *q_rows_dev,
                                              const float *uniforms, size_t n_uniforms, float temperature,
                                              size_t max_commit, uint32_t *commits, size_t *n_commit,
                                              size_t *n_accepted, size_t *n_used) {
    return guard([&] {
        need_weights(m);
        if ((k && (!drafts || !q_rows_dev)) || !uniforms || !commits || !n_commit || !n_accepted || !n_used)
            throw sd::ArgError("null argument");
        setdev(m);
        m->dec->verify_rejection_linear(drafts, k, q_rows_dev, uniforms, n_uniforms, temperature, max_commit, commits,
                                        n_commit, n_accepted, n_used, true);
    });
}

sd_status sd_verify_rejection_tree(sd_model *m, const uint32_t *tokens, const uint32_t *parents, size_t n,
                                   const float *q_rows, size_t q_rows_n, size_t q_vocab, const int32_t *q_row_of,
                                   const float *uniforms, size_t n_uniforms, float temperature, int32_t use_t2d,
                                   int32_t siblings, size_t max_commit, uint32_t *path, size_t *path_len,
                                   int32_t *token, size_t *n_used) {
    return guard([&] {
        need_weights(m);
        if (!tokens || !parents || !q_row_of || !uniforms || !path || !path_len || !token || !n_used ||
            (q_rows_n && !q_rows))
            throw sd::ArgError("null argument");
        setdev(m);
        m->dec->verify_rejection_tree(tokens, parents, n, q_rows, q_rows_n, q_vocab, q_row_of, uniforms, n_uniforms,
                                      temperature, use_t2d, siblings, max_commit, path, path_len, token, n_used);
    });
}

sd_status sd_verify_rejection_tree_device_q(sd_model *m, const uint32_t *tokens, const uint32_t *parents, size_t n,
                                            const float *q_rows_dev, size_t q_rows_n, size_t q_vocab,
                                            const int32_t *q_row_of, const float *uniforms, size_t n_uniforms,
                                            float temperature, int32_t use_t2d, int32_t siblings, size_t max_commit,
                                            uint32_t *path, size_t *path_len, int32_t *token, size_t *n_used) {
    return guard([&] {
        need_weights(m);
        if (!tokens || !parents || !q_row_of || !uniforms || !path || !path_len || !token || !n_used ||
            (q_rows_n && !q_rows_dev))
            throw sd::ArgError("null argument");
        setdev(m);
        m->dec->verify_rejection_tree(tokens, parents, n, q_rows_dev, q_rows_n, q_vocab, q_row_of, uniforms,
                                      n_uniforms, temperature, use_t2d, siblings, max_commit, path, path_len, token,
                                      n_used, true);
    });
}

sd_status sd_set_d2t(sd_model *m, const int64_t *d2t, size_t n) {
    return guard([&] {
        need(m);
        if (!d2t) throw sd::ArgError("null d2t");
        setdev(m);
        m->dec->set_d2t(d2t, n);
    });
}

sd_status sd_draft_to_target(sd_model *m, const uint32_t *draft_ids, size_t n, uint32_t *out) {
    return guard([&] {
        need(m);
        if ((n && (!draft_ids || !out))) throw sd::ArgError("null argument");
        const auto &d2t = m->dec->d2t_host;
        if (d2t.empty()) throw sd::ArgError("no d2t table (sd_set_d2t)");
        for (size_t i = 0; i < n; i++)
            if (draft_ids[i] >= d2t.size())
                throw sd::SamplingError("draft id " + std::to_string(draft_ids[i]) + " out of range (" +
                                        std::to_string(d2t.size()) + ")");
        for (size_t i = 0; i < n; i++) out[i] = (uint32_t)d2t[draft_ids[i]];
    });
}

size_t sd_t2d_mask(const sd_model *m, uint8_t *out, size_t cap) {
    if (!m || !m->dec || m->dec->t2d_host.empty()) return 0;
    const auto &inv = m->dec->t2d_host;
    const size_t n = std::min(cap, inv.size());
    for (size_t i = 0; i < n && out; i++) out[i] = inv[i] >= 0 ? 1 : 0;
    return inv.size();
}

sd_status sd_last_argmax(sd_model *m, int32_t *out, size_t n) {
    return guard([&] {
        need(m);
        if (!out) throw sd::ArgError("null output");
        setdev(m);
        m->dec->argmax_rows(out, n);
    });
}

static sd::SampleParams filters_of(const sd_sampling *f) {
    if (!f) throw sd::ArgError("null argument");
    sd::SampleParams p{};
    p.temperature = f->temperature;
    p.top_k = f->top_k;
    p.top_p = f->top_p;
    p.min_p = f->min_p;
    return p;
}

sd_status sd_sample_next(sd_model *m, const sd_sampling *params, float uniform, int32_t *token) {
    return guard([&] {
        need_weights(m);
        if (!token) throw sd::ArgError("null output");
        const sd::SampleParams f = filters_of(params);
        setdev(m);
        m->dec->sample_next(f, uniform, token);
    });
}

sd_status sd_sample_rows(sd_model *m, const sd_sampling *params, const float *uniforms, size_t n, int32_t *tokens) {
    return guard([&] {
        need(m);
        if (!uniforms || !tokens) throw sd::ArgError("null argument");
        const sd::SampleParams f = filters_of(params);
        setdev(m);
        m->dec->sample_rows(f, uniforms, n, tokens);
    });
}

sd_status sd_model_set_kv_format(sd_model *m, int32_t format) {
    return guard([&] {
        need(m);
        if (m->dec->cache_len || !m->dec->history.empty()) throw sd::ArgError("the cache must be empty (reset first)");
        setdev(m);
        m->model->set_kv_format(format);
    });
}

sd_status sd_prime_synthetic(sd_model *m, const uint32_t *ids, size_t n, uint64_t kv_seed) {
    return guard([&] {
        need(m);
        if (!ids) throw sd::ArgError("null ids");
        setdev(m);
        m->dec->prime_synthetic(ids, n, kv_seed);
    });
}

sd_status sd_profile_enable(sd_model *m, int32_t on) {
    return guard([&] {
        need(m);
        m->model->prof_on = on != 0;
    });
}

size_t sd_profile_read(sd_model *m, int32_t *cls, double *bytes, float *ms, size_t cap) {
    if (!m || !m->model) return 0;
    auto &P = m->model->prof;
    (void)hipSetDevice(m->model->cfg.device);
    (void)hipStreamSynchronize(m->model->st);
    size_t n = 0;
    for (auto &e : P) {
        if (n >= cap) break;
        float t = 0.f;
        (void)hipEventElapsedTime(&t, m->model->ev_pool[e.ev], m->model->ev_pool[e.ev + 1]);
        if (cls) cls[n] = e.cls;
        if (bytes) bytes[n] = e.bytes;
        if (ms) ms[n] = t;
        n++;
    }
    m->model->prof_reset();
    return n;
}

sd_status sd_synchronize(sd_model *m) {
    return guard([&] {
        need(m);
        setdev(m);
        m->model->sync();
    });
}

sd_status sd_read_kv_rows(sd_model *m, int32_t layer, int32_t which, int32_t head, size_t pos0, size_t n,
                          uint16_t *out) {
    return guard([&] {
        need(m);
        const sd::ModelCfg &c = m->model->cfg;
        if (!out) throw sd::ArgError("null output");
        if (layer < 0 || layer >= c.n_layers || which < 0 || which > 1 || head < 0 || head >= c.n_kv_heads)
            throw sd::ArgError("kv row selector out of range");
        m->model->read_kv_rows(layer, which, head, pos0, n, out);
    });
}

size_t sd_cache_len(const sd_model *m) { return m && m->dec ? (size_t)m->dec->cache_len : 0; }

static int64_t quant_rows_check(int32_t fmt, size_t rows, size_t K) {
    if (fmt != SD_Q4_K && fmt != SD_Q5_K && fmt != SD_Q6_K && fmt != SD_Q8_0)
        throw sd::UnsupportedError("format must be Q4_K, Q5_K, Q6_K or Q8_0");
    if (rows == 0 || rows % 16 || K == 0 || K % 256) throw sd::ArgError("rows must be a multiple of 16 and K of 256");
    return (int64_t)(K / 256);
}

sd_status sd_repack_gguf(int32_t fmt, const void *gguf, size_t rows, size_t K, void *out) {
    return guard([&] {
        if (!gguf || !out) throw sd::ArgError("null argument");
        const int64_t nsb = quant_rows_check(fmt, rows, K);
        const int sbb = sd::fmt_sb_bytes(fmt), tbb = sd::tile_block_bytes(fmt);
        const uint8_t *src = (const uint8_t *)gguf;
        uint8_t *dst = (uint8_t *)out;
        for (size_t r = 0; r < rows; r++)
            for (int64_t sb = 0; sb < nsb; sb++)
                sd::pack_sb(fmt, src + ((int64_t)r * nsb + sb) * sbb, dst + ((int64_t)(r >> 4) * nsb + sb) * tbb,
                            (int)(r & 15));
    });
}

sd_status sd_unpack_tiles(int32_t fmt, const void *tiles, size_t rows, size_t K, void *gguf_out) {
    return guard([&] {
        if (!tiles || !gguf_out) throw sd::ArgError("null argument");
        const int64_t nsb = quant_rows_check(fmt, rows, K);
        const int sbb = sd::fmt_sb_bytes(fmt), tbb = sd::tile_block_bytes(fmt);
        const uint8_t *src = (const uint8_t *)tiles;
        uint8_t *dst = (uint8_t *)gguf_out;
        for (size_t r = 0; r < rows; r++)
            for (int64_t sb = 0; sb < nsb; sb++)
                sd::unpack_sb(fmt, src + ((int64_t)(r >> 4) * nsb + sb) * tbb, (int)(r & 15),
                              dst + ((int64_t)r * nsb + sb) * sbb);
    });
}

sd_status sd_lane_codes(int32_t fmt, const void *tile_block, int32_t lane, int32_t chunk, uint32_t *out) {
    return guard([&] {
        if (!tile_block || !out) throw sd::ArgError("null argument");
        if (lane < 0 || lane > 63 || chunk < 0 || chunk > 7) throw sd::ArgError("lane in [0, 64), chunk in [0, 8)");
        const uint8_t *tb = (const uint8_t *)tile_block;
        auto v4 = [&](int off) {
            sd::uintx4 v;
            std::memcpy(&v, tb + off, 16);
            return v;
        };
        const int g = lane >> 4;
        if (fmt == SD_Q4_K) {
            sd::LaneQ4K d;
            d.hdr = v4(d.off_hdr(lane));
            d.q0 = v4(d.off_q0(lane));
            d.q1 = v4(d.off_q1(lane));
            d.codes(g, chunk, out);
        } else if (fmt == SD_Q5_K) {
            sd::LaneQ5K d;
            d.hdr = v4(d.off_hdr(lane));
            std::memcpy(&d.qh, tb + d.off_qh(lane), 8);
            d.q0 = v4(d.off_q0(lane));
            d.q1 = v4(d.off_q1(lane));
            d.codes(g, chunk, out);
        } else if (fmt == SD_Q6_K) {
            sd::LaneQ6K d;
            d.n0 = v4(d.off_n0(lane));
            d.n1 = v4(d.off_n1(lane));
            d.hb = v4(d.off_hb(lane));
            d.codes(g, chunk, out);
        } else if (fmt == SD_Q8_0) {
            sd::LaneQ80 d;
            d.a0 = v4(d.off_part(lane, 0));
            d.a1 = v4(d.off_part(lane, 1));
            d.b0 = v4(d.off_part(lane, 2));
            d.b1 = v4(d.off_part(lane, 3));
            d.codes(g, chunk, out);
        } else {
            throw sd::UnsupportedError("format must be Q4_K, Q5_K, Q6_K or Q8_0");
        }
    });
}

sd_status sd_tree_cartesian(uint32_t root, const uint32_t *cand, const uint32_t *branching, size_t depth,
                            uint32_t *tokens, uint32_t *parents, size_t cap, size_t *n) {
    return guard([&] {
        if (!n || (depth && (!cand || !branching))) throw sd::ArgError("null argument");
        const size_t need = sd::cartesian_size(branching, depth);
        *n = need;
        if (!tokens || !parents) return;  // size query
        if (need > cap) throw sd::ArgError("output capacity smaller than the Cartesian tree");
        const sd::DraftTreeC t = sd::cartesian_tree(root, cand, branching, depth);
        std::memcpy(tokens, t.tokens.data(), need * 4);
        std::memcpy(parents, t.parents.data(), need * 4);
    });
}

sd_status sd_tree_prune(const uint32_t *tokens, const uint32_t *parents, size_t n, const float *log_probs,
                        const uint32_t *branching, size_t depth, size_t max_total, uint32_t *out_tokens,
                        uint32_t *out_parents, size_t *n_out) {
    return guard([&] {
        if (!tokens || !parents || !out_tokens || !out_parents || !n_out || (depth && (!log_probs || !branching)))
            throw sd::ArgError("null argument");
        const sd::DraftTreeC full = sd::DraftTreeC::from_arrays(tokens, parents, n);
        const sd::DraftTreeC t = sd::prune_cartesian(full, log_probs, branching, depth, max_total);
        std::memcpy(out_tokens, t.tokens.data(), t.size() * 4);
        std::memcpy(out_parents, t.parents.data(), t.size() * 4);
        *n_out = t.size();
    });
}


/* ---- EAGLE-3 draft (crates/speculate/src/methods/eagle3.rs) ---- */
static void need3(const sd_draft3 *d) {
    if (!d || !d->d) throw sd::ArgError("null draft handle");
}

sd_status sd_draft3_create(const sd_draft3_config *cfg, sd_draft3 **out) {
    return guard([&] {
        if (!cfg || !out) throw sd::ArgError("null argument");
        *out = nullptr;
        sd::Draft3Cfg c;
        c.hidden = cfg->hidden;
        c.n_heads = cfg->n_heads;
        c.n_kv_heads = cfg->n_kv_heads;
        c.ffn = cfg->ffn;
        c.draft_vocab = cfg->draft_vocab;
        c.target_vocab = cfg->target_vocab;
        c.rms_eps = cfg->rms_eps;
        c.rope_theta = cfg->rope_theta;
        c.max_pos = cfg->max_pos;
        c.device = cfg->device;
        auto h = std::make_unique<sd_draft3>();
        h->d = std::make_unique<sd::Draft3>(c);
        *out = h.release();
    });
}

void sd_draft3_destroy(sd_draft3 *d) { delete d; }

size_t sd_draft3_tensor_bytes(const sd_draft3 *d, int32_t kind) {
    if (!d || !d->d || kind < 0 || kind >= sd::D3_NUM) return 0;
    return d->d->tensor_bytes(kind);
}

sd_status sd_draft3_set_tensor(sd_draft3 *d, int32_t kind, const void *data, size_t bytes) {
    return guard([&] {
        need3(d);
        d->d->set_tensor(kind, data, bytes);
    });
}

sd_status sd_draft3_get_tensor(const sd_draft3 *d, int32_t kind, void *data, size_t bytes) {
    return guard([&] {
        need3(d);
        if (!data) throw sd::ArgError("null data");
        d->d->get_tensor(kind, data, bytes);
    });
}

sd_status sd_draft3_synthesize(sd_draft3 *d, uint64_t seed, float weight_std) {
    return guard([&] {
        need3(d);
        d->d->synthesize(seed, weight_std);
    });
}

sd_status sd_draft3_reset(sd_draft3 *d) {
    return guard([&] {
        need3(d);
        d->d->reset();
    });
}

sd_status sd_draft3_forward(sd_draft3 *d, const float *hidden_in, size_t n_in, const float *input_emb,
                            size_t position, float *out_hidden, float *out_logits) {
    return guard([&] {
        need3(d);
        if (!hidden_in || !input_emb) throw sd::ArgError("null argument");
        if (position > (size_t)INT32_MAX) throw sd::ArgError("position out of range");
        d->d->step_host(hidden_in, n_in, input_emb, (int)position, out_hidden, out_logits);
    });
}

sd_status sd_draft3_round(sd_draft3 *d, sd_model *m, const uint32_t *layers, size_t depth, const int32_t *top_k,
                          int32_t *target_ids, int32_t *draft_ids, float *log_probs) {
    return guard([&] {
        need3(d);
        need_weights(m);
        if (!layers || !top_k || !target_ids || !draft_ids || !log_probs) throw sd::ArgError("null argument");
        if (depth < 1 || depth > (size_t)sd::kDraftMaxSteps) throw sd::ArgError("draft depth out of range");
        setdev(m);
        d->d->round(*m->model, *m->dec, layers, (int)depth, top_k, target_ids, draft_ids, log_probs);
    });
}


/* ---- EAGLE-2 draft (crates/speculate/src/methods/eagle.rs) ---- */
static void need2(const sd_draft2 *d) {
    if (!d || !d->d) throw sd::ArgError("null draft handle");
}

sd_status sd_draft2_create(const sd_draft2_config *cfg, sd_draft2 **out) {
    return guard([&] {
        if (!cfg || !out) throw sd::ArgError("null argument");
        *out = nullptr;
        sd::Draft2Cfg c;
        c.hidden = cfg->hidden;
        c.n_heads = cfg->n_heads;
        c.n_kv_heads = cfg->n_kv_heads;
        c.ffn = cfg->ffn;
        c.vocab = cfg->vocab;
        c.rms_eps = cfg->rms_eps;
        c.rope_theta = cfg->rope_theta;
        c.max_pos = cfg->max_pos;
        c.device = cfg->device;
        auto h = std::make_unique<sd_draft2>();
        h->d = std::make_unique<sd::Draft2>(c);
        *out = h.release();
    });
}

void sd_draft2_destroy(sd_draft2 *d) { delete d; }

size_t sd_draft2_tensor_bytes(const sd_draft2 *d, int32_t kind) {
    if (!d || !d->d || kind < 0 || kind >= sd::D2_NUM) return 0;
    return d->d->tensor_bytes(kind);
}

sd_status sd_draft2_set_tensor(sd_draft2 *d, int32_t kind, const void *data, size_t bytes) {
    return guard([&] {
        need2(d);
        d->d->set_tensor(kind, data, bytes);
    });
}

sd_status sd_draft2_get_tensor(const sd_draft2 *d, int32_t kind, void *data, size_t bytes) {
    return guard([&] {
        need2(d);
        if (!data) throw sd::ArgError("null data");
        d->d->get_tensor(kind, data, bytes);
    });
}

sd_status sd_draft2_synthesize(sd_draft2 *d, uint64_t seed, float weight_std) {
    return guard([&] {
        need2(d);
        d->d->synthesize(seed, weight_std);
    });
}

sd_status sd_draft2_reset(sd_draft2 *d) {
    return guard([&] {
        need2(d);
        d->d->reset();
    });
}

sd_status sd_draft2_forward(sd_draft2 *d, const float *target_hidden, size_t n, uint32_t token, size_t position,
                            float *out_hidden) {
    return guard([&] {
        need2(d);
        if (!target_hidden) throw sd::ArgError("null argument");
        if (n != (size_t)d->d->cfg.hidden) throw sd::ArgError("target_hidden must be hidden wide");
        if (position > (size_t)INT32_MAX) throw sd::ArgError("position out of range");
        d->d->step_host(target_hidden, token, (int)position, out_hidden);
    });
}

sd_status sd_draft2_round(sd_draft2 *d, sd_model *m, const float *target_hidden, size_t depth, const int32_t *top_k,
                          int32_t *ids, float *log_probs) {
    return guard([&] {
        need2(d);
        need_weights(m);
        if (!target_hidden || !top_k || !ids || !log_probs) throw sd::ArgError("null argument");
        if (depth < 1 || depth > (size_t)sd::kDraftMaxSteps) throw sd::ArgError("draft depth out of range");
        setdev(m);
        d->d->round(*m->model, *m->dec, target_hidden, (int)depth, top_k, ids, log_probs);
    });
}

sd_status sd_kvpool_create(const sd_kvpool_config *cfg, sd_kvpool **out) {
    return guard([&] {
        if (!cfg || !out) throw sd::ArgError("null argument");
        *out = nullptr;
        auto h = std::make_unique<sd_kvpool>();
        h->p = make_pool(*cfg, 4);
        *out = h.release();
    });
}
void sd_kvpool_destroy(sd_kvpool *c) { delete c; }
size_t sd_kvpool_page_bytes(const sd_kvpool *c) { return c && c->p ? (size_t)c->p->layer(0).page_bytes : 0; }

sd_status sd_kvpool_append(sd_kvpool *c, int32_t layer, const sd_kv_rows *rows, int32_t fmt, const void *q, size_t q_ld,
                           const void *k, size_t k_ld, const void *v, size_t v_ld, const int32_t *pos, uint16_t *q_out,
                           void *stream) {
    return guard([&] {
        need(c);
        const sd::KvPool &P = *c->p;
        P.check_layer(layer);
        sd::KvqAppend a{};
        a.rows = kv_rows(rows);
        if (fmt != SD_F16 && fmt != SD_F32) throw sd::UnsupportedError("append: rows must be F16 or F32");
        if (!k || !v || (q && !q_out)) throw sd::ArgError("null argument");
        const int size = fmt == SD_F32 ? 4 : 2, hd = P.cfg.head_dim;
        a.L = P.layer(layer);
        a.pos = pos;
        a.cos_t = P.cos_t;
        a.sin_t = P.sin_t;
        a.max_pos = P.cfg.max_pos;
        a.interleaved = P.cfg.interleaved;
        a.n_heads = P.cfg.n_heads;
        a.f32 = fmt == SD_F32;
        a.q = q;
        a.k = k;
        a.v = v;
        a.q_ld = row_stride(q_ld, (int64_t)P.cfg.n_heads * hd, "q");
        a.k_ld = row_stride(k_ld, (int64_t)P.cfg.n_kv_heads * hd, "k");
        a.v_ld = row_stride(v_ld, (int64_t)P.cfg.n_kv_heads * hd, "v");
        a.q_out = q_out;
        a.q_out_row = (int64_t)P.cfg.n_heads * hd;
        a.q_out_head = hd;
        if (q) need_aligned(q, a.q_ld * size, 16, "q");
        need_aligned(k, a.k_ld * size, 16, "k");
        need_aligned(v, a.v_ld * size, 16, "v");
        if (q) {
            need_aligned(q_out, 16, 16, "q_out");
            const int64_t n = a.rows.n, qb = (int64_t)P.cfg.n_heads * hd, kb = (int64_t)P.cfg.n_kv_heads * hd * size;
            const sd::RowBytes out{q_out, qb * 2, qb * 2, n};
            if (rows_meet(out, {q, a.q_ld * size, qb * size, n}) || rows_meet(out, {k, a.k_ld * size, kb, n}) ||
                rows_meet(out, {v, a.v_ld * size, kb, n}))
                throw sd::ArgError("q_out must not overlap q, k or v");
        }
        sd::DeviceScope dev(P.cfg.device);
        sd::launch_kvq_append(a, (hipStream_t)stream);
    });
}

sd_status sd_kvpool_read(sd_kvpool *c, int32_t layer, const sd_kv_rows *rows, uint16_t *k_out, uint16_t *v_out,
                         void *stream) {
    return guard([&] {
        need(c);
        c->p->check_layer(layer);
        const sd::KvqRows r = kv_rows(rows);
        need_aligned(k_out, 16, 16, "k_out");
        need_aligned(v_out, 16, 16, "v_out");
        if (!k_out && !v_out) return;
        sd::DeviceScope dev(c->p->cfg.device);
        sd::launch_kvq_read(c->p->layer(layer), r, k_out, v_out, (hipStream_t)stream);
    });
}

size_t sd_kvpool_attend_workspace(const sd_kvpool *c, size_t rows, size_t n_seqs, size_t max_rows, size_t max_len) {
    size_t bytes = 0;
    guard([&] {
        need(c);
        const size_t most = (size_t)1 << 40;
        bytes = c->p->plan((int64_t)std::min(rows, most), (int64_t)std::min(n_seqs, most),
                           (int64_t)std::min(max_rows, most), (int64_t)std::min(max_len, most)).ws_bytes;
    });
    return bytes;
}

sd_status sd_kvpool_attend(sd_kvpool *c, int32_t layer, const sd_kv_query *qy, void *ws, size_t ws_bytes, void *stream) {
    return guard([&] {
        need(c);
        const sd::KvPool &P = *c->p;
        P.check_layer(layer);
        if (!qy) throw sd::ArgError("null argument");
        if (qy->rows == 0) return;
        if (!qy->q || !qy->out || !qy->row_start || !qy->kv_len || !qy->table) throw sd::ArgError("null argument");
        if (qy->n_seqs < 1 || qy->table_ld < 1) throw sd::ArgError("n_seqs and table_ld must be positive");
        if (qy->mask && qy->mask_words < 1) throw sd::ArgError("mask_words must be positive");
        const size_t most = (size_t)1 << 40;
        const sd::KvqPlan plan = P.plan((int64_t)std::min(qy->rows, most), qy->n_seqs, (int64_t)std::min(qy->max_rows, most),
                                        (int64_t)std::min(qy->max_len, most));
        if (plan.ws_bytes && (!ws || ws_bytes < plan.ws_bytes))
            throw sd::ArgError("attend: the workspace needs " + std::to_string(plan.ws_bytes) + " bytes");
        need_aligned(ws, 16, 16, "workspace");
        if (!std::isfinite(qy->scale)) throw sd::ArgError("scale must be finite");
        const int hd = P.cfg.head_dim;
        sd::KvqAttn a{};
        a.L = P.layer(layer);
        a.q = qy->q;
        a.q_row = row_stride(qy->q_ld, (int64_t)P.cfg.n_heads * hd, "q");
        a.q_head = hd;
        a.out = qy->out;
        a.out_ld = row_stride(qy->out_ld, (int64_t)P.cfg.n_heads * hd, "out");
        need_aligned(a.q, a.q_row * 2, 16, "q");
        need_aligned(a.out, a.out_ld * 2, 8, "out");
        const int64_t row = (int64_t)P.cfg.n_heads * hd * 2;
        const sd::RowBytes q{a.q, a.q_row * 2, row, (int64_t)qy->rows}, out{a.out, a.out_ld * 2, row, (int64_t)qy->rows};
        const sd::RowBytes work{ws, 0, (int64_t)plan.ws_bytes, 1};
        if (rows_meet(q, out) || rows_meet(q, work) || rows_meet(out, work))
            throw sd::ArgError("attend: q, out and the workspace must not overlap");
        a.rows = (int)qy->rows;
        a.n_seqs = qy->n_seqs;
        a.row_start = qy->row_start;
        a.kv_len = qy->kv_len;
        a.table = qy->table;
        a.table_ld = qy->table_ld;
        a.mask = qy->mask;
        a.mask_words = qy->mask_words;
        a.max_rows = (int)qy->max_rows;
        a.n_heads = P.cfg.n_heads;
        a.n_rep = P.cfg.n_heads / P.cfg.n_kv_heads;
        a.scale = qy->scale == 0.f ? (float)(1.0 / std::sqrt((double)hd)) : qy->scale;
        sd::DeviceScope dev(P.cfg.device);
        sd::launch_kvq_attention(a, plan, ws, (hipStream_t)stream);
    });
}

sd_status sd_kv8_create(const sd_kvpool_config *cfg, sd_kv8 **out) {
    return guard([&] {
        if (!cfg || !out) throw sd::ArgError("null argument");
        *out = nullptr;
        auto h = std::make_unique<sd_kv8>();
        h->p = make_pool(*cfg, 8);
        *out = h.release();
    });
}
void sd_kv8_destroy(sd_kv8 *c) { delete c; }
size_t sd_kv8_page_bytes(const sd_kv8 *c) { return c && c->p ? (size_t)c->p->page_bytes() : 0; }

sd_status sd_kv8_append(sd_kv8 *c, int32_t layer, const sd_kv_seqs *seqs, int32_t fmt, const void *q, size_t q_ld,
                        const void *k, size_t k_ld, const void *v, size_t v_ld, const int32_t *pos, uint16_t *q_out,
                        void *stream) {
    return guard([&] {
        need(c);
        const sd::KvPool &P = *c->p;
        P.check_layer(layer);
        if (!seqs) throw sd::ArgError("null argument");
        if (fmt != SD_F16 && fmt != SD_F32) throw sd::UnsupportedError("append: rows must be F16 or F32");
        if (seqs->rows == 0) return;
        if (!seqs->row_start || !seqs->kv_len || !seqs->table || !k || !v || (q && !q_out)) throw sd::ArgError("null argument");
        if (seqs->rows > ((size_t)1 << 24)) throw sd::ArgError("append: at most 2^24 rows");
        if (seqs->max_rows < 1 || seqs->max_rows > seqs->rows) throw sd::ArgError("append: max_rows must be in [1, rows]");
        if (seqs->n_seqs < 1 || seqs->n_seqs > 65535) throw sd::ArgError("append: n_seqs must be in [1, 65535]");
        if (seqs->table_ld < 1) throw sd::ArgError("append: table_ld must be positive");
        // a grid holds fewer than 2^32 threads
        if ((int64_t)seqs->n_seqs * (2 * P.cfg.n_kv_heads + P.cfg.n_heads) > (1 << 23))
            throw sd::UnsupportedError("append: too many sequences and heads in one call");
        const int size = fmt == SD_F32 ? 4 : 2, hd = P.cfg.head_dim;
        sd::Kv8Append a{};
        a.L = sd::Kv8Layer(P.layer(layer));
        a.seqs = {(int)seqs->rows, seqs->n_seqs, (int)seqs->max_rows, seqs->row_start, seqs->kv_len, 0, seqs->table, seqs->table_ld};
        a.pos = pos;
        a.cos_t = P.cos_t;
        a.sin_t = P.sin_t;
        a.max_pos = P.cfg.max_pos;
        a.interleaved = P.cfg.interleaved;
        a.n_heads = P.cfg.n_heads;
        a.f32 = fmt == SD_F32;
        a.q = q;
        a.k = k;
        a.v = v;
        a.q_ld = row_stride(q_ld, (int64_t)P.cfg.n_heads * hd, "q");
        a.k_ld = row_stride(k_ld, (int64_t)P.cfg.n_kv_heads * hd, "k");
        a.v_ld = row_stride(v_ld, (int64_t)P.cfg.n_kv_heads * hd, "v");
        a.q_out = q_out;
        need_aligned(k, a.k_ld * size, 16, "k");
        need_aligned(v, a.v_ld * size, 16, "v");
        if (q) {
            need_aligned(q, a.q_ld * size, 16, "q");
            need_aligned(q_out, 16, 16, "q_out");
            const int64_t n = a.seqs.rows, qb = (int64_t)P.cfg.n_heads * hd, kb = (int64_t)P.cfg.n_kv_heads * hd * size;
            const sd::RowBytes out{q_out, qb * 2, qb * 2, n};
            if (rows_meet(out, {q, a.q_ld * size, qb * size, n}) || rows_meet(out, {k, a.k_ld * size, kb, n}) ||
                rows_meet(out, {v, a.v_ld * size, kb, n}))
                throw sd::ArgError("q_out must not overlap q, k or v");
        }
        sd::DeviceScope dev(P.cfg.device);
        sd::launch_kv8_append(a, (hipStream_t)stream);
    });
}

sd_status sd_kv8_read(sd_kv8 *c, int32_t layer, const sd_kv_rows *rows, uint16_t *k_out, uint16_t *v_out, void *stream) {
    return guard([&] {
        need(c);
        c->p->check_layer(layer);
        const sd::KvqRows r = kv_rows(rows);
        need_aligned(k_out, 16, 16, "k_out");
        need_aligned(v_out, 16, 16, "v_out");
        const int64_t bytes = (int64_t)r.n * c->p->cfg.n_kv_heads * c->p->cfg.head_dim * 2;
        if (rows_meet(bytes_at(k_out, bytes), bytes_at(v_out, bytes))) throw sd::ArgError("read: k_out and v_out must not overlap");
        if (!k_out && !v_out) return;
        sd::DeviceScope dev(c->p->cfg.device);
        sd::launch_kv8_read(sd::Kv8Layer(c->p->layer(layer)), r, k_out, v_out, (hipStream_t)stream);
    });
}

size_t sd_kv8_attend_workspace(const sd_kv8 *c, size_t rows, size_t n_seqs, size_t max_rows, size_t max_len,
                               const sd_kv_window *window) {
    size_t bytes = 0;
    guard([&] {
        need(c);
        bytes = kv8_plan(*c->p, rows, n_seqs, max_rows, max_len, window).ws_bytes;
    });
    return bytes;
}

sd_status sd_kv8_attend(sd_kv8 *c, int32_t layer, const sd_kv_query *qy, const sd_kv_window *window, float *lse, void *ws,
                        size_t ws_bytes, void *stream) {
    return guard([&] {
        need(c);
        const sd::KvPool &P = *c->p;
        P.check_layer(layer);
        if (!qy) throw sd::ArgError("null argument");
        if (qy->rows == 0) return;
        if (!qy->out) throw sd::ArgError("null argument");
        sd::Kv8Attn a = kv8_query(P, layer, qy, window);
        const sd::KvqPlan plan = kv8_plan(P, qy->rows, (size_t)qy->n_seqs, qy->max_rows, qy->max_len, window);
        if (plan.ws_bytes && (!ws || ws_bytes < plan.ws_bytes))
            throw sd::ArgError("attend: the workspace needs " + std::to_string(plan.ws_bytes) + " bytes");
        need_aligned(ws, 16, 16, "workspace");
        need_aligned(lse, 4, 4, "lse");
        a.out = qy->out;
        a.out_ld = row_stride(qy->out_ld, (int64_t)P.cfg.n_heads * P.cfg.head_dim, "out");
        need_aligned(a.out, a.out_ld * 2, 8, "out");
        a.lse = lse;
        const int64_t row = (int64_t)P.cfg.n_heads * P.cfg.head_dim * 2, n = a.rows;
        const sd::RowBytes q{a.q, a.q_row * 2, row, n}, out{a.out, a.out_ld * 2, row, n};
        const sd::RowBytes work = bytes_at(ws, (int64_t)plan.ws_bytes), stat = bytes_at(lse, n * P.cfg.n_heads * 4);
        if (rows_meet(q, out) || rows_meet(q, work) || rows_meet(out, work) || rows_meet(stat, q) || rows_meet(stat, out) ||
            rows_meet(stat, work))
            throw sd::ArgError("attend: q, out, lse and the workspace must not overlap");
        sd::DeviceScope dev(P.cfg.device);
        sd::launch_kv8_attention(a, plan, ws, (hipStream_t)stream);
    });
}

sd_status sd_kv8_weights(sd_kv8 *c, int32_t layer, const sd_kv_query *qy, const sd_kv_window *window, const float *lse,
                         const sd_kv_scores *scores, void *stream) {
    return guard([&] {
        need(c);
        const sd::KvPool &P = *c->p;
        P.check_layer(layer);
        if (!qy || !scores) throw sd::ArgError("null argument");
        if (qy->rows == 0) return;
        if (!lse || !scores->out) throw sd::ArgError("null argument");
        kv8_plan(P, qy->rows, (size_t)std::max(qy->n_seqs, 0), qy->max_rows, qy->max_len, window);  // the sizes
        sd::Kv8Weights w{};
        w.a = kv8_query(P, layer, qy, window);
        w.a.lse = (float *)lse;
        w.in = scores->in;
        w.out = scores->out;
        if (scores->ld < 1 || scores->ld > ((size_t)1 << 30)) throw sd::ArgError("weights: ld must be in [1, 2^30]");
        if (!std::isfinite(scores->decay)) throw sd::ArgError("weights: decay must be finite");
        w.ld = (int64_t)scores->ld;
        w.decay = scores->decay;
        w.anew = scores->own_rows_anew != 0;
        w.max_len = (int64_t)qy->max_len;
        w.cus = P.cus;
        need_aligned(lse, 4, 4, "lse");
        need_aligned(w.in, 4, 4, "scores");
        need_aligned(w.out, 4, 4, "scores");
        const int64_t n = (int64_t)w.a.n_seqs * P.cfg.n_kv_heads * w.ld * 4, row = (int64_t)P.cfg.n_heads * P.cfg.head_dim * 2;
        const sd::RowBytes out = bytes_at(w.out, n);
        if (w.in != w.out && rows_meet(out, bytes_at(w.in, n))) throw sd::ArgError("weights: the scores overlap in part");
        if (rows_meet(out, {w.a.q, w.a.q_row * 2, row, w.a.rows}) || rows_meet(out, bytes_at(lse, (int64_t)w.a.rows * P.cfg.n_heads * 4)))
            throw sd::ArgError("weights: the scores must not overlap q or lse");
        sd::DeviceScope dev(P.cfg.device);
        sd::launch_kv8_weights(w, (hipStream_t)stream);
    });
}

// whether n_seqs x budget is a size that a call can have
static void check_evict(const sd::KvPool &P, int64_t n_seqs, size_t budget) {
    if (n_seqs < 1 || n_seqs > 65535) throw sd::ArgError("evict: n_seqs must be in [1, 65535]");
    if (budget > ((size_t)1 << 30)) throw sd::ArgError("evict: budget must be at most 2^30");
    // a grid holds fewer than 2^32 threads
    const int64_t blocks = std::max<int64_t>(4, ((int64_t)budget + 31) / 32);
    if (blocks > ((int64_t)1 << 23) / (2 * P.cfg.n_kv_heads * n_seqs))
        throw sd::UnsupportedError("evict: too many sequences and blocks in one call");
}

size_t sd_kv8_evict_workspace(const sd_kv8 *c, size_t n_seqs, size_t budget) {
    size_t bytes = 0;
    guard([&] {
        need(c);
        check_evict(*c->p, (int64_t)std::min(n_seqs, (size_t)1 << 40), budget);
        bytes = sd::kv8_evict_ws_bytes((int)n_seqs, c->p->cfg.n_kv_heads, c->p->cfg.head_dim, (int)budget);
    });
    return bytes;
}

sd_status sd_kv8_evict(sd_kv8 *c, int32_t layer, const sd_kv_evict *e, void *ws, size_t ws_bytes, void *stream) {
    return guard([&] {
        need(c);
        const sd::KvPool &P = *c->p;
        P.check_layer(layer);
        if (!e || !e->kv_len || !e->table || !e->scores || !e->new_len || (e->budget && !e->kept)) throw sd::ArgError("null argument");
        if (e->table_ld < 1 || (e->new_table && e->new_table_ld < 1)) throw sd::ArgError("table_ld must be positive");
        check_evict(P, e->n_seqs, e->budget);
        if (e->sinks > e->budget || e->recent > e->budget - e->sinks) throw sd::ArgError("evict: sinks and recent exceed the budget");
        if (e->scores_ld < 1 || e->scores_ld > ((size_t)1 << 30)) throw sd::ArgError("evict: scores_ld must be in [1, 2^30]");
        const size_t out_ld = e->scores_out_ld ? e->scores_out_ld : e->budget;
        if (e->scores_out && (out_ld < e->budget || out_ld > ((size_t)1 << 30))) throw sd::ArgError("evict: scores_out: rows overlap");
        const int kv = P.cfg.n_kv_heads;
        const int64_t need_ws = e->new_table ? 0 : (int64_t)sd::kv8_evict_ws_bytes(e->n_seqs, kv, P.cfg.head_dim, (int)e->budget);
        if (need_ws && (!ws || ws_bytes < (size_t)need_ws))
            throw sd::ArgError("evict: the workspace needs " + std::to_string(need_ws) + " bytes");
        need_aligned(ws, 16, 16, "workspace");
        for (const void *p : {(const void *)e->scores, (const void *)e->scores_out, (const void *)e->kept, (const void *)e->new_len})
            need_aligned(p, 4, 4, "evict");
        const int64_t heads = (int64_t)e->n_seqs * kv;
        const bool same = e->scores_out == e->scores && out_ld == e->scores_ld;
        // (tables of several layers' calls, kv_len and scores are inputs; nothing written may meet them or each other)
        const sd::RowBytes outs[] = {bytes_at(e->kept, heads * (int64_t)e->budget * 4), bytes_at(e->new_len, (int64_t)e->n_seqs * 4),
                                     bytes_at(ws, need_ws), bytes_at(e->scores_out, heads * (int64_t)out_ld * 4)};
        const sd::RowBytes ins[] = {bytes_at(e->kv_len, (int64_t)e->n_seqs * 4), bytes_at(e->table, (int64_t)e->n_seqs * e->table_ld * 4),
                                    bytes_at(e->new_table, (int64_t)e->n_seqs * e->new_table_ld * 4),
                                    bytes_at(e->scores, heads * (int64_t)e->scores_ld * 4)};
        for (int i = 0; i < 4; i++) {
            for (int j = 0; j < i; j++)
                if (rows_meet(outs[i], outs[j])) throw sd::ArgError("evict: outputs and the workspace must not overlap");
            for (int j = 0; j < 4; j++)
                if (!(i == 3 && j == 3 && same) && rows_meet(outs[i], ins[j]))
                    throw sd::ArgError("evict: outputs and the workspace must not overlap the inputs");
        }
        sd::Kv8Evict a{};
        a.L = sd::Kv8Layer(P.layer(layer));
        a.n_seqs = e->n_seqs;
        a.kv_len = e->kv_len;
        a.table = e->table;
        a.table_ld = e->table_ld;
        a.new_table = e->new_table;
        a.new_ld = e->new_table_ld;
        a.scores = e->scores;
        a.scores_ld = (int64_t)e->scores_ld;
        a.scores_out = e->scores_out;
        a.scores_out_ld = (int64_t)out_ld;
        a.budget = (int)e->budget;
        a.sinks = (int)e->sinks;
        a.recent = (int)e->recent;
        a.kept = e->kept;
        a.new_len = e->new_len;
        sd::DeviceScope dev(P.cfg.device);
        sd::launch_kv8_evict(a, ws, (hipStream_t)stream);
    });
}

sd_status sd_sampler_create(int32_t vocab, int32_t max_rows, int32_t device, sd_sampler **out) {
    return guard([&] {
        if (!out) throw sd::ArgError("null argument");
        *out = nullptr;
        auto h = std::make_unique<sd_sampler>();
        h->s = std::make_unique<sd::Sampler>(vocab, max_rows, device);
        *out = h.release();
    });
}
void sd_sampler_destroy(sd_sampler *s) { delete s; }

sd_status sd_sampler_run(sd_sampler *s, const float *logits, size_t ld, size_t rows, const sd_sampling *params,
                         const float *uniforms, int32_t *tokens, float *probs, void *stream) {
    return guard([&] {
        if (!s || !s->s) throw sd::ArgError("null sampler handle");
        if (!params) throw sd::ArgError("null argument");
        if (rows > 65535 || ld > ((size_t)1 << 40)) throw sd::ArgError("sampler: rows or ld out of range");
        sd::SampleParams p{};
        p.logits = logits;
        p.ld = (int64_t)ld;
        p.rows = (int)rows;
        p.temperature = params->temperature;
        p.top_k = params->top_k;
        p.top_p = params->top_p;
        p.min_p = params->min_p;
        p.u = uniforms;
        p.tokens = tokens;
        p.probs = probs;
        s->s->run(p, (hipStream_t)stream);
    });
}

}  // extern "C"
