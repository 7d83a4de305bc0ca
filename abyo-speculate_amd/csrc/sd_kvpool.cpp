// Host side of the paged KV caches and the sampler.  See sd_kvpool.hpp.
#include "sd_kvpool.hpp"

#include <cmath>

#include "sd_model.hpp"

namespace sd {

DeviceScope::DeviceScope(int device) {
    SD_HIP_CHECK(hipGetDevice(&prev));
    if (prev == device) prev = -1;
    else SD_HIP_CHECK(hipSetDevice(device));
}
DeviceScope::~DeviceScope() {
    if (prev >= 0) (void)hipSetDevice(prev);
}

bool rows_meet(const RowBytes &a, const RowBytes &b) {
    if (!a.at || !b.at || a.n < 1 || b.n < 1 || a.row < 1 || b.row < 1) return false;
    // (a stride of 2^42 bytes times 2^24 rows passes 64 bits)
    typedef unsigned __int128 wide;
    auto start = [](const RowBytes &x, int64_t i) { return (wide)(uintptr_t)x.at + (wide)i * (wide)x.ld; };
    if (start(a, a.n - 1) + a.row <= start(b, 0) || start(b, b.n - 1) + b.row <= start(a, 0)) return false;
    for (int64_t i = 0, j = 0; i < a.n && j < b.n;) {
        const wide ea = start(a, i) + a.row, eb = start(b, j) + b.row;
        if (start(a, i) < eb && start(b, j) < ea) return true;
        (ea < eb ? i : j)++;
    }
    return false;
}

KvPool::KvPool(const KvPoolCfg &c) : cfg(c) {
    if (c.n_layers < 1 || c.n_heads < 1 || c.n_kv_heads < 1 || c.n_pages < 1) throw ArgError("kvpool: all sizes must be positive");
    if (c.n_heads % c.n_kv_heads) throw ArgError("kvpool: n_heads must be a multiple of n_kv_heads");
    if (c.n_heads > 4096) throw UnsupportedError("kvpool: at most 4096 heads");
    if (c.head_dim != 64 && c.head_dim != 128) throw UnsupportedError("kvpool: head_dim must be 64 or 128");
    if (c.page_tokens < 32 || c.page_tokens > 4096 || (c.page_tokens & (c.page_tokens - 1)))
        throw UnsupportedError("kvpool: page_tokens must be a power of two from 32 to 4096");
    if (c.max_pos < 0 || c.max_pos > (1 << 24)) throw ArgError("kvpool: max_pos must be in [0, 2^24]");
    if (c.max_pos && !(c.rope_theta > 0.f && std::isfinite(c.rope_theta))) throw ArgError("kvpool: rope_theta must be positive");
    const double bytes = (double)c.n_layers * c.n_pages * (double)page_bytes();
    if (bytes > 1e12) throw ArgError("kvpool: more than 1 TB of pages");
    DeviceScope dev(c.device);
    SD_HIP_CHECK(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, c.device));
    layer_bytes = c.n_pages * page_bytes();
    if (c.bits == 8) kv8_prepare();
    try {
        SD_HIP_CHECK(hipMalloc(&mem, (size_t)layer_bytes * c.n_layers + 256));
        SD_HIP_CHECK(hipMemset(mem, 0, (size_t)layer_bytes * c.n_layers + 256));
        if (c.max_pos) {
            const size_t n = (size_t)c.max_pos * (c.head_dim / 2) * sizeof(float);
            SD_HIP_CHECK(hipMalloc(&cos_t, n));
            SD_HIP_CHECK(hipMalloc(&sin_t, n));
            launch_kvq_tables(cos_t, sin_t, c.max_pos, c.head_dim, c.rope_theta, nullptr);
        }
        SD_HIP_CHECK(hipDeviceSynchronize());
    } catch (...) {
        for (void *p : {(void *)mem, (void *)cos_t, (void *)sin_t})
            if (p) (void)hipFree(p);
        throw;
    }
}

KvPool::~KvPool() {
    int prev = -1;
    (void)hipGetDevice(&prev);
    (void)hipSetDevice(cfg.device);
    for (void *p : {(void *)mem, (void *)cos_t, (void *)sin_t})
        if (p) (void)hipFree(p);
    if (prev >= 0) (void)hipSetDevice(prev);
}

int64_t KvPool::page_bytes() const {
    return cfg.bits == 8 ? kv8_page_bytes(cfg.n_kv_heads, cfg.head_dim, cfg.page_tokens)
                         : (int64_t)cfg.n_kv_heads * (cfg.page_tokens / kKvqBlock) * kvq_block_bytes(cfg.head_dim);
}

KvqLayer KvPool::layer(int l) const {
    KvqLayer L;
    L.base = mem + (int64_t)l * layer_bytes;
    L.page_bytes = page_bytes();
    L.n_pages = cfg.n_pages;
    L.page_shift = __builtin_ctz((unsigned)cfg.page_tokens);
    L.n_kv = cfg.n_kv_heads;
    L.hd = cfg.head_dim;
    return L;
}

void KvPool::check_layer(int l) const {
    if (l < 0 || l >= cfg.n_layers) throw ArgError("kvpool: layer out of range");
}

KvqPlan KvPool::plan(int64_t rows, int64_t n_seqs, int64_t max_rows, int64_t max_len, int window, int sinks) const {
    if (rows < 1 || rows > (1 << 24)) throw ArgError("kvpool: rows must be in [1, 2^24]");
    if (n_seqs < 1 || n_seqs > 65535) throw ArgError("kvpool: n_seqs must be in [1, 65535]");
    if (max_rows < 1 || max_rows > rows) throw ArgError("kvpool: max_rows must be in [1, rows]");
    if (max_len < 0 || max_len > 0x7fffffc0) throw ArgError("kvpool: max_len out of range");
    // (before the plan's numbers are of 32 bits; below, tiles are fewer than that)
    if (max_rows * (cfg.n_heads / cfg.n_kv_heads) > (1 << 30)) throw UnsupportedError("kvpool: too many rows in one call");
    KvqPlan p = cfg.bits == 8 ? kv8_attn_plan(cfg.n_heads, cfg.n_kv_heads, (int)n_seqs, (int)max_rows, max_len, window, sinks, cus)
                              : kvq_attn_plan(cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, (int)n_seqs, (int)max_rows, max_len, cus);
    // a grid holds fewer than 2^32 threads, at up to 512 a workgroup
    if ((int64_t)p.tiles * cfg.n_kv_heads * n_seqs > (1 << 22)) throw UnsupportedError("kvpool: too many rows in one call");
    p.ws_bytes = p.nsplit > 1 ? (size_t)p.nsplit * (size_t)rows * cfg.n_heads * (cfg.head_dim + 2) * sizeof(float) : 0;
    return p;
}

Sampler::Sampler(int v, int n, int d) : vocab(v), max_rows(n), device(d) {
    if (v < 1 || n < 1) throw ArgError("sampler: vocab and max_rows must be positive");
    if (v > kSmpMaxVocab) throw UnsupportedError("sampler: at most 262144 tokens");
    if (n > 65535) throw ArgError("sampler: at most 65535 rows");
    DeviceScope dev(device);
    SD_HIP_CHECK(hipMalloc(&ws, sample_ws_bytes(vocab, max_rows)));
}

Sampler::~Sampler() {
    int prev = -1;
    (void)hipGetDevice(&prev);
    (void)hipSetDevice(device);
    if (ws) (void)hipFree(ws);
    if (prev >= 0) (void)hipSetDevice(prev);
}

void Sampler::check(float temperature, int64_t top_k, float top_p, float min_p) {
    if (!(temperature >= 0.f) || !std::isfinite(temperature)) throw SamplingError("temperature must be finite and not negative");
    if (top_k < 0) throw SamplingError("top_k must not be negative (0: off)");
    if (!(top_p >= 0.f && top_p <= 1.f)) throw SamplingError("top_p must be in [0, 1] (1: off)");
    if (!(min_p >= 0.f && min_p <= 1.f)) throw SamplingError("min_p must be in [0, 1] (0: off)");
}

void Sampler::run(SampleParams p, hipStream_t st) {
    check(p.temperature, p.top_k, p.top_p, p.min_p);
    if (p.rows < 0 || p.rows > max_rows) throw ArgError("sampler: rows must be in [0, max_rows]");
    if (p.rows == 0) return;
    if (!p.logits || !p.u || !p.tokens) throw ArgError("sampler: null argument");
    if (p.ld == 0) p.ld = vocab;
    if (p.ld < vocab) throw ArgError("sampler: rows overlap (ld < vocab)");
    const int64_t row = (int64_t)vocab * sizeof(float);
    if (rows_meet({p.probs, row, row, p.rows}, {p.logits, p.ld * (int64_t)sizeof(float), row, p.rows}))
        throw ArgError("sampler: probs must not overlap the logits");
    DeviceScope dev(device);
    p.V = vocab;
    p.ws = ws;
    launch_sample(p, st);
}

}  // namespace sd
