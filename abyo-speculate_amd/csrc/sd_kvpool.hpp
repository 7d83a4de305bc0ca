// Host handles of the operators on device memory: the 4-bit paged KV cache
// and the sampler.
#pragma once
#include "sd_kvq.hpp"
#include "sd_sample.hpp"

namespace sd {

struct KvPoolCfg {
    int n_layers = 0, n_heads = 0, n_kv_heads = 0, head_dim = 0;
    int n_pages = 0, page_tokens = 64;
    int max_pos = 0;  // rows of the RoPE tables; 0: the caller has tables
    int interleaved = 0;
    float rope_theta = 10000.f;
    int device = 0;
};

// Makes a device current and the previous one current again at the end.
class DeviceScope {
  public:
    explicit DeviceScope(int device);
    ~DeviceScope();

  private:
    int prev = -1;
};

// Whether two sets of rows (n rows of `row` bytes, `ld` bytes apart) have a byte
// in common.  Rows of one buffer may lie between the other's.
struct RowBytes {
    const void *at;
    int64_t ld, row, n;
};
bool rows_meet(const RowBytes &a, const RowBytes &b);

// The pages of every layer in one allocation.
class KvPool {
  public:
    explicit KvPool(const KvPoolCfg &c);
    ~KvPool();
    KvPool(const KvPool &) = delete;
    KvPool &operator=(const KvPool &) = delete;

    KvPoolCfg cfg;
    float *cos_t = nullptr, *sin_t = nullptr;
    int64_t layer_bytes = 0;
    int cus = 0;

    KvqLayer layer(int l) const;
    void check_layer(int l) const;
    // the plan of a call (ArgError for sizes that no call can have)
    KvqPlan plan(int64_t rows, int64_t n_seqs, int64_t max_rows, int64_t max_len) const;

  private:
    uint8_t *mem = nullptr;
};

class Sampler {
  public:
    Sampler(int vocab, int max_rows, int device);
    ~Sampler();
    Sampler(const Sampler &) = delete;
    Sampler &operator=(const Sampler &) = delete;

    int vocab, max_rows, device;
    // checks the filters and sizes and enqueues (p.ws and p.V are the handle's)
    void run(SampleParams p, hipStream_t st);
    static void check(float temperature, int64_t top_k, float top_p, float min_p);

  private:
    void *ws = nullptr;
};

}  // namespace sd
