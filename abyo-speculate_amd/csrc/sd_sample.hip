// Sampling: one token per row of logits from a given uniform, after the
// filters in this order:
//   w_i  = exp((l_i - max) / T)          (T = 0: the first maximum alone)
//   top-k  the k largest, of equal ones the first
//   top-p  the shortest run of the rest, largest first (of equal ones the
//          first), whose weights reach p times the rest's sum
//   min-p  of those the ones with w_i >= min_p
//   token  the first kept i whose running sum, by index, exceeds u times the
//          sum of the kept
// Weights are computed in f64 and summed as integers of 2^-44, so no sum
// depends on an order; a decision can differ from exact arithmetic only within
// about 1e-11 of a border.
//
// Both top-k and top-p keep a prefix of the order (value descending, index
// ascending), so together they are one bound on the pair (value, index).  Two
// launches find it: k_smp_slices (a workgroup per 8192 entries) leaves each
// slice's maximum and a histogram of counts and weights over bins of equal
// width in l / T; k_smp_draw (a workgroup per row) adds the histograms, finds
// the bin in which the bound lies, takes that bin's entries (or, when they are
// few, all entries down to that bin) into LDS, finds the bound by radix
// selection and draws.  k_smp_probs writes the kept distribution when asked.
#include "sd_sample.hpp"
#include "sd_common.hpp"

namespace sd {

constexpr int kSmpT = 1024, kSmpPer = kSmpSlice / kSmpT, kSmpWaves = kSmpT / 64;
constexpr int kSmpList = 2048;  // entries taken into LDS
constexpr double kOne = 17592186044416.0;  // 2^44

// Per slice: the largest entry's order key, whether an entry is NaN or +inf,
// the sum of the weights relative to the slice's maximum.
struct SmpSlice {
    uint32_t key;
    uint32_t bad;
    uint64_t mass;
};
// What k_smp_draw leaves for k_smp_probs.
struct SmpRow {
    uint64_t cut;   // kept: order_of(key, index) >= cut ...
    uint64_t total; // sum of the kept weights; 0: no distribution
    float max;
    float pad;
};

struct SmpWs {
    SmpSlice *slice;  // [rows][slices]
    uint64_t *mass;   // [rows][slices][kSmpBins]
    uint32_t *count;  // [rows][slices][kSmpBins]
    SmpRow *row;      // [rows]
};
static __host__ __device__ inline int smp_slices(int V) { return (V + kSmpSlice - 1) / kSmpSlice; }
static SmpWs smp_ws(void *p, int V, int rows) {
    const size_t n = (size_t)rows * smp_slices(V);
    SmpWs w;
    w.mass = (uint64_t *)p;
    w.slice = (SmpSlice *)(w.mass + n * kSmpBins);
    w.row = (SmpRow *)(w.slice + n);
    w.count = (uint32_t *)(w.row + rows);
    return w;
}
size_t sample_ws_bytes(int V, int rows) {
    const size_t n = (size_t)rows * smp_slices(V);
    return n * kSmpBins * 12 + n * sizeof(SmpSlice) + (size_t)rows * sizeof(SmpRow);
}

// order key of a logit: unsigned order is value order, +0 and -0 alike
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(l + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // key_of(-inf); an entry at or below it has no weight
// value descending, then index ascending, as one number to compare (50 bits)
__device__ __forceinline__ uint64_t order_of(uint32_t key, int i) {
    return ((uint64_t)key << 18) | (uint32_t)(kSmpMaxVocab - 1 - i);
}
// bin grid in l / T, the same for all slices; monotone in l
__device__ __forceinline__ int bin_of(float l, float bins_per) {
    return (int)floorf(fminf(fmaxf(l * bins_per, -1.0e9f), 1.0e9f));
}
// exp2((l - max) * c) to 1e-11, c = log2(e) / T: the power of two of the
// rounded exponent times the exponential series of the rest (|y| < 0.347,
// tenth term 2e-13 ...)
__device__ __forceinline__ double weight(float l, float max, double c) {
    const double t = ((double)l - (double)max) * c;
    if (!(t > -1000.0)) return 0.0;
    const double n = rint(t), y = (t - n) * 0.6931471805599453;
    double e = 1.0 / 3628800.0;
    e = e * y + 1.0 / 362880.0;
    e = e * y + 1.0 / 40320.0;
    e = e * y + 1.0 / 5040.0;
    e = e * y + 1.0 / 720.0;
    e = e * y + 1.0 / 120.0;
    e = e * y + 1.0 / 24.0;
    e = e * y + 1.0 / 6.0;
    e = e * y + 0.5;
    e = e * y + 1.0;
    e = e * y + 1.0;
    return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, e) + ((uint64_t)(int64_t)(int)n << 52));
}
// a value in [0, 2^51) rounded to an integer
__device__ __forceinline__ uint64_t to_int(double x) {
    return __builtin_bit_cast(uint64_t, x + 4503599627370496.0) & 0xfffffffffffffull;
}

struct SmpCfg {
    const float *logits;
    int64_t ld;
    int V, nsl;
    double c;        // log2(e) / T
    float bins_per;  // bins per unit of l
    int top_k;
    double top_p, min_p;
    int filtered;    // top-k or top-p: histograms
    const float *u;
    int *tokens;
    float *probs;
    SmpWs ws;
};

// ---- slices ----------------------------------------------------------------------
__global__ __launch_bounds__(kSmpT) void k_smp_slices(const SmpCfg p) {
    __shared__ uint64_t mass[kSmpBins];
    __shared__ uint32_t count[kSmpBins];
    __shared__ uint32_t s_key, s_bad;
    __shared__ uint64_t s_mass;
    const int sl = blockIdx.x, r = blockIdx.y, t = threadIdx.x;
    const float *row = p.logits + (int64_t)r * p.ld;
    if (t == 0) s_key = s_bad = 0, s_mass = 0;
    if (p.filtered) mass[t] = 0, count[t] = 0;
    float l[kSmpPer];
    uint32_t key = 0, bad = 0;
#pragma unroll
    for (int i = 0; i < kSmpPer; i++) {
        const int x = sl * kSmpSlice + i * kSmpT + t;
        l[i] = x < p.V ? row[x] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < kSmpPer; i++) {
        bad |= l[i] != l[i] || l[i] == INFINITY;
        key = max(key, key_of(l[i]));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        key = max(key, (uint32_t)__shfl_xor((int)key, o));
        bad |= (uint32_t)__shfl_xor((int)bad, o);
    }
    __syncthreads();
    if ((t & 63) == 0) {
        atomicMax(&s_key, key);
        if (bad) atomicOr(&s_bad, 1u);
    }
    __syncthreads();
    key = s_key;
    SmpSlice *out = p.ws.slice + (int64_t)r * p.nsl + sl;
    if (s_bad || key <= kKeyNegInf) {
        // nothing to weigh: the histograms of a slice with key <= -inf are not read
        if (t == 0) *out = SmpSlice{key, s_bad, 0};
        return;
    }
    const float m = of_key(key);
    const int top = bin_of(m, p.bins_per);
    uint64_t sum = 0;
#pragma unroll
    for (int i = 0; i < kSmpPer; i++) {
        if (l[i] == -INFINITY) continue;
        const uint64_t w = to_int(weight(l[i], m, p.c) * kOne);
        if (p.filtered) {
            const int b = min(top - bin_of(l[i], p.bins_per), kSmpBins - 1);
            atomicAdd(&count[b], 1u);
            if (w) atomicAdd((unsigned long long *)&mass[b], (unsigned long long)w);
        } else {
            sum += w;
        }
    }
    if (p.filtered) {
        __syncthreads();
        const int64_t at = ((int64_t)r * p.nsl + sl) * kSmpBins + t;
        p.ws.mass[at] = mass[t];
        p.ws.count[at] = count[t];
        if (t == 0) *out = SmpSlice{key, 0, 0};
        return;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += (uint64_t)__shfl_xor((long long)sum, o);
    if ((t & 63) == 0) atomicAdd((unsigned long long *)&s_mass, (unsigned long long)sum);
    __syncthreads();
    if (t == 0) *out = SmpSlice{key, 0, s_mass};
}

// ---- draw ------------------------------------------------------------------------
struct SmpShared {
    uint64_t mass[kSmpBins];  // running sums down to and including the bin
    uint32_t count[kSmpBins];
    uint64_t lmass[kSmpList];
    uint64_t lorder[kSmpList];
    uint64_t dmass[256];
    uint32_t dcount[256];
    uint64_t wsum[kSmpWaves];
    uint32_t wcnt[kSmpWaves];
    double f[64];
    int shift[64];
    uint64_t a, b;
    int n, i;
};
static_assert(kSmpMaxVocab / kSmpSlice <= 64, "slices of a row");

__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += (uint64_t)__shfl_xor((long long)v, o);
    return v;
}
// the workgroup's sum, to every thread
__device__ uint64_t group_sum(SmpShared &S, uint64_t v) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) S.wsum[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
    for (int w = 0; w < kSmpWaves; w++) t += S.wsum[w];
    return t;
}

// Entries to select from: the list in LDS, or the row's entries of bins
// [lo, hi] (counted from the row's top bin).
struct ListSource {
    SmpShared &S;
    int n;
    uint64_t least;  // entries below are left out
    __device__ int size() const { return n; }
    __device__ bool get(int i, uint64_t &order, uint64_t &mass) const {
        order = S.lorder[i];
        mass = S.lmass[i];
        return order >= least;
    }
};
struct RowSource {
    const SmpCfg &p;
    const float *row;
    float max;
    int top, lo, hi;
    uint64_t least;
    __device__ int size() const { return p.V; }
    __device__ bool get(int i, uint64_t &order, uint64_t &mass) const {
        const float l = row[i];
        if (l == -INFINITY) return false;
        const int b = min(top - bin_of(l, p.bins_per), kSmpBins - 1);
        if (b < lo || b > hi) return false;
        order = order_of(key_of(l), i);
        if (order < least) return false;
        mass = to_int(weight(l, max, p.c) * kOne);
        return true;
    }
};

// The entry at which the running count (or sum) over the source, in
// descending order, first reaches `target`; the last entry if it never does.
// Eight bits of the order number at a time.  All threads; returns its order.
template <typename Src> __device__ uint64_t select(SmpShared &S, const Src &src, bool by_mass, uint64_t target) {
    const int t = threadIdx.x;
    uint64_t prefix = 0;
    for (int shift = 48; shift >= 0; shift -= 8) {  // 50 bits: digits of 8 from bit 48 (the first has 2)
        __syncthreads();
        if (t < 256) S.dmass[t] = 0, S.dcount[t] = 0;
        __syncthreads();
        for (int i = t; i < src.size(); i += kSmpT) {
            uint64_t order, mass;
            if (!src.get(i, order, mass) || (order >> (shift + 8)) != prefix) continue;
            const int d = (int)(order >> shift) & 255;
            atomicAdd(&S.dcount[d], 1u);
            if (by_mass && mass) atomicAdd((unsigned long long *)&S.dmass[d], (unsigned long long)mass);
        }
        __syncthreads();
        if (t < 64) {
            // lane t holds digits 255 - 4 t .. 252 - 4 t, in descending order
            uint64_t v[4], sum = 0;
            uint32_t any = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int d = 255 - 4 * t - k;
                v[k] = by_mass ? S.dmass[d] : S.dcount[d];
                any |= (uint32_t)(S.dcount[d] != 0) << k;
                sum += v[k];
            }
            uint64_t run = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint64_t up = (uint64_t)__shfl_up((long long)run, o);
                if (t >= o) run += up;
            }
            uint64_t before = run - sum;
            int pick = -1;
            uint64_t left = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (pick < 0 && (any >> k & 1) && before + v[k] >= target) {
                    pick = 255 - 4 * t - k;
                    left = target - before;  // target > before: an earlier digit would have been taken
                }
                before += v[k];
            }
            const uint64_t found = __ballot(pick >= 0);
            // none reaches it (rounded sums): the last digit present, its last entry
            const uint64_t has = __ballot(any != 0);
            if (found) {
                if (t == __ffsll((unsigned long long)found) - 1) {
                    S.i = pick;
                    S.a = left;
                }
            } else if (has && t == 63 - __clzll((long long)has)) {
                int k = 31 - __clz((int)any);
                S.i = 255 - 4 * t - k;
                S.a = ~0ull >> 1;
            } else if (!has && t == 0) {
                S.i = 0;
                S.a = 0;
            }
        }
        __syncthreads();
        prefix = (prefix << 8) | (uint64_t)S.i;
        target = S.a;
    }
    return prefix;
}

// The first index of [x0, x1) whose running kept weight reaches target,
// the last one with any weight if none does; -1 without weight.
struct Kept {
    const SmpCfg &p;
    const float *row;
    float max;
    uint64_t cut;
    __device__ uint64_t mass(int i) const {
        const float l = row[i];
        if (l == -INFINITY || order_of(key_of(l), i) < cut) return 0;
        const double w = weight(l, max, p.c);
        return w >= p.min_p ? to_int(w * kOne) : 0;
    }
};
// per-wave sums of contiguous parts of [x0, x1) in S.wsum; returns the part's size
__device__ int part_sums(SmpShared &S, const Kept &k, int x0, int x1) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int seg = ((x1 - x0 + kSmpWaves - 1) / kSmpWaves + 63) / 64 * 64;
    const int a = x0 + wave * seg, b = min(x1, a + seg);
    uint64_t s = 0;
    for (int i = a + lane; i < b; i += 64) s += k.mass(i);
    s = wave_sum(s);
    __syncthreads();
    if (lane == 0) S.wsum[wave] = s;
    __syncthreads();
    return seg;
}
__device__ int draw_row(SmpShared &S, const Kept &k, int x0, int x1, uint64_t target) {
    // narrow to at most one entry per thread
    while (x1 - x0 > kSmpT) {
        const int seg = part_sums(S, k, x0, x1);
        int pick = -1, last = -1;
        uint64_t before = 0, left = 0;
        for (int w = 0; w < kSmpWaves; w++) {
            const uint64_t s = S.wsum[w];
            if (s) last = w;
            if (pick < 0 && s && before + s >= target) {
                pick = w;
                left = target - before;
            }
            before += s;
        }
        if (pick < 0) {
            if (last < 0) return -1;
            pick = last;
            left = ~0ull >> 1;
        }
        x0 += pick * seg;
        x1 = min(x1, x0 + seg);
        target = left;
        __syncthreads();
    }
    const int t = threadIdx.x, i = x0 + t, lane = t & 63, wave = t >> 6;
    const uint64_t m = i < x1 ? k.mass(i) : 0;
    uint64_t run = m;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t up = (uint64_t)__shfl_up((long long)run, o);
        if (lane >= o) run += up;
    }
    if (t == 0) S.n = 0x7fffffff, S.i = -1;
    __syncthreads();
    if (lane == 63) S.wsum[wave] = run;
    __syncthreads();
    for (int w = 0; w < wave; w++) run += S.wsum[w];
    if (m) {
        if (run >= target) atomicMin(&S.n, i);
        atomicMax(&S.i, i);
    }
    __syncthreads();
    return S.n != 0x7fffffff ? S.n : S.i;
}

// the row's entries of bins [lo, hi] into the list; returns their number
__device__ int gather(SmpShared &S, const RowSource &src) {
    __syncthreads();
    if (threadIdx.x == 0) S.n = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < src.size(); i += kSmpT) {
        uint64_t order, mass;
        if (!src.get(i, order, mass)) continue;
        const int at = atomicAdd(&S.n, 1);
        if (at < kSmpList) {
            S.lorder[at] = order;
            S.lmass[at] = mass;
        }
    }
    __syncthreads();
    return min(S.n, kSmpList);
}

// first bin whose running count (or sum) reaches target, else the last bin
__device__ int bin_reaching(SmpShared &S, bool by_mass, uint64_t target) {
    __syncthreads();
    if (threadIdx.x == 0) S.i = kSmpBins - 1;
    __syncthreads();
    const int b = threadIdx.x;
    if ((by_mass ? S.mass[b] : S.count[b]) >= target) atomicMin(&S.i, b);
    __syncthreads();
    return S.i;
}

// u times sum as the least running sum that exceeds it
__device__ __forceinline__ uint64_t draw_target(float u, uint64_t sum) {
    const double t = fmin(fmax((double)u, 0.0), 1.0) * (double)sum;
    return min((uint64_t)t + 1, sum);
}

__global__ __launch_bounds__(kSmpT) void k_smp_draw(const SmpCfg p) {
    __shared__ SmpShared S;
    const int r = blockIdx.x, t = threadIdx.x;
    const float *row = p.logits + (int64_t)r * p.ld;
    const SmpSlice *sl = p.ws.slice + (int64_t)r * p.nsl;
    uint32_t key = 0, bad = 0;
    for (int s = 0; s < p.nsl; s++) {
        key = max(key, sl[s].key);
        bad |= sl[s].bad;
    }
    if (bad || key <= kKeyNegInf) {
        if (t == 0) {
            p.tokens[r] = -1;
            p.ws.row[r] = SmpRow{0, 0, 0.f, 0.f};
        }
        return;
    }
    const float max = of_key(key);
    const int top = bin_of(max, p.bins_per);
    if (t < p.nsl) {
        const bool some = sl[t].key > kKeyNegInf;
        const float m = of_key(sl[t].key);
        S.f[t] = some ? weight(m, max, p.c) : 0.0;
        S.shift[t] = some ? min(top - bin_of(m, p.bins_per), kSmpBins) : -1;
    }
    const float u = p.u[r];
    uint64_t cut = 0, total = 0;
    int token;
    if (!p.filtered && p.min_p <= 0.0) {
        // the slice from the slices' sums, the entry from the slice
        __syncthreads();
        for (int s = 0; s < p.nsl; s++) total += (uint64_t)rint((double)sl[s].mass * S.f[s]);
        uint64_t target = draw_target(u, total), before = 0;
        int pick = 0;
        for (int s = 0; s < p.nsl; s++) {
            const uint64_t m = (uint64_t)rint((double)sl[s].mass * S.f[s]);
            if (!m) continue;
            pick = s;
            if (before + m >= target) break;
            before += m;
        }
        const Kept k{p, row, max, 0};
        token = draw_row(S, k, pick * kSmpSlice, min(p.V, (pick + 1) * kSmpSlice), target - before);
    } else if (!p.filtered) {
        const Kept k{p, row, max, 0};
        uint64_t mine = 0;
        for (int i = t; i < p.V; i += kSmpT) mine += k.mass(i);
        total = group_sum(S, mine);
        token = draw_row(S, k, 0, p.V, draw_target(u, total));
    } else {
        S.mass[t] = 0;
        S.count[t] = 0;
        __syncthreads();
        for (int s = 0; s < p.nsl; s++) {
            if (S.shift[s] < 0) continue;
            const int64_t at = ((int64_t)r * p.nsl + s) * kSmpBins + t;
            const uint32_t c = p.ws.count[at];
            if (!c) continue;
            const int b = min(t + S.shift[s], kSmpBins - 1);
            const uint64_t m = (uint64_t)rint((double)p.ws.mass[at] * S.f[s]);
            atomicAdd(&S.count[b], c);
            if (m) atomicAdd((unsigned long long *)&S.mass[b], (unsigned long long)m);
        }
        __syncthreads();
        {
            // running sums over the bins
            const int lane = t & 63, wave = t >> 6;
            uint64_t m = S.mass[t];
            uint32_t c = S.count[t];
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint64_t um = (uint64_t)__shfl_up((long long)m, o);
                const uint32_t uc = (uint32_t)__shfl_up((int)c, o);
                if (lane >= o) m += um, c += uc;
            }
            if (lane == 63) S.wsum[wave] = m, S.wcnt[wave] = c;
            __syncthreads();
            for (int w = 0; w < wave; w++) m += S.wsum[w], c += S.wcnt[w];
            S.mass[t] = m;
            S.count[t] = c;
            __syncthreads();
        }
        const uint32_t entries = S.count[kSmpBins - 1];
        const bool k_on = p.top_k > 0 && (uint32_t)p.top_k < entries, p_on = p.top_p < 1.0;
        uint64_t kept = S.mass[kSmpBins - 1];  // sum of the entries left so far
        int hi = kSmpBins - 1;                 // their last bin
        int listed_lo = 0, listed_hi = -1, n = 0;  // bins in the list
        if (k_on) hi = bin_reaching(S, false, (uint64_t)p.top_k);
        else if (p_on) hi = bin_reaching(S, true, (uint64_t)ceil(p.top_p * (double)kept));
        RowSource src{p, row, max, top, 0, hi, 0};
        const bool all = S.count[hi] <= (uint32_t)kSmpList;  // everything down to that bin fits the list
        if (all) {
            n = gather(S, src);
            listed_hi = hi;
        }
        // the selection inside bin b after `before` entries (weight) of the bins above
        auto bound = [&](int b, bool by_mass, uint64_t target) -> uint64_t {
            const uint64_t above = b ? (by_mass ? S.mass[b - 1] : S.count[b - 1]) : 0;
            const uint32_t in_bin = S.count[b] - (b ? S.count[b - 1] : 0);
            src.lo = src.hi = b;
            src.least = cut;
            if (!all && in_bin > (uint32_t)kSmpList) return select(S, src, by_mass, target > above ? target - above : 1);
            if (!all && (listed_lo != b || listed_hi != b)) {
                src.least = 0;
                n = gather(S, src);
                listed_lo = listed_hi = b;
            }
            const ListSource ls{S, n, cut};
            if (all) return select(S, ls, by_mass, target);
            return select(S, ls, by_mass, target > above ? target - above : 1);
        };
        // the weight of the entries at or above `cut`, which lies in bin b
        auto weight_to = [&](int b) -> uint64_t {
            uint64_t mine = 0, order, m;
            if (all || (listed_lo == b && listed_hi == b)) {
                for (int i = t; i < n; i += kSmpT)
                    if (S.lorder[i] >= cut) mine += S.lmass[i];
            } else {
                src.lo = src.hi = b;
                src.least = cut;
                for (int i = t; i < p.V; i += kSmpT)
                    if (src.get(i, order, m)) mine += m;
            }
            return group_sum(S, mine) + (all || !b ? 0 : S.mass[b - 1]);
        };
        if (k_on) {
            cut = bound(hi, false, (uint64_t)p.top_k);
            kept = weight_to(hi);
        }
        if (p_on) {
            const uint64_t target = std::max<uint64_t>(1, (uint64_t)ceil(p.top_p * (double)kept));
            const int b = std::min(hi, bin_reaching(S, true, target));
            cut = std::max(cut, bound(b, true, target));
        }
        // the kept entries' sum and the draw
        if (all) {
            uint64_t mine = 0;
            __syncthreads();
            for (int i = t; i < n; i += kSmpT) {
                const uint64_t o = S.lorder[i];
                const bool keep = o >= cut && weight(of_key((uint32_t)(o >> 18)), max, p.c) >= p.min_p;
                if (!keep) S.lmass[i] = 0;
                mine += S.lmass[i];
                S.lorder[i] = keep ? (o & (kSmpMaxVocab - 1)) : 0;  // by index from here on
            }
            total = group_sum(S, mine);
            const ListSource ls{S, n, 0};
            token = kSmpMaxVocab - 1 - (int)select(S, ls, true, draw_target(u, total));
        } else {
            const Kept k{p, row, max, cut};
            uint64_t mine = 0;
            for (int i = t; i < p.V; i += kSmpT) mine += k.mass(i);
            total = group_sum(S, mine);
            token = draw_row(S, k, 0, p.V, draw_target(u, total));
        }
    }
    if (t == 0) {
        p.tokens[r] = token;
        p.ws.row[r] = SmpRow{cut, total, max, 0.f};
    }
}

// ---- the kept distribution ----------------------------------------------------------
__global__ __launch_bounds__(256) void k_smp_probs(const SmpCfg p) {
    const int r = blockIdx.y, x0 = blockIdx.x * 2048 + threadIdx.x;
    const SmpRow s = p.ws.row[r];
    const float *row = p.logits + (int64_t)r * p.ld;
    float *out = p.probs + (int64_t)r * p.V;
    const double inv = s.total ? kOne / (double)s.total : 0.0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int x = x0 + i * 256;
        if (x >= p.V) return;
        const float l = row[x];
        double w = 0.0;
        if (s.total && l > -INFINITY && order_of(key_of(l), x) >= s.cut) w = weight(l, s.max, p.c);
        out[x] = w >= p.min_p ? (float)(w * inv) : 0.f;
    }
}

void launch_sample(const SampleParams &in, hipStream_t st) {
    if (in.rows < 1) return;
    SmpCfg p{};
    p.logits = in.logits;
    p.ld = in.ld;
    p.V = in.V;
    p.nsl = smp_slices(in.V);
    const bool greedy = in.temperature == 0.f;
    const double T = greedy ? 1.0 : (double)in.temperature;
    p.c = 1.4426950408889634 / T;
    p.bins_per = (float)std::min(32.0 / T, 1e30);
    p.top_k = greedy ? 1 : in.top_k;
    p.top_p = in.top_p;
    p.min_p = in.min_p;
    p.filtered = p.top_k > 0 || p.top_p < 1.0;
    p.u = in.u;
    p.tokens = in.tokens;
    p.probs = in.probs;
    p.ws = smp_ws(in.ws, in.V, in.rows);
    k_smp_slices<<<dim3((unsigned)p.nsl, (unsigned)in.rows), dim3(kSmpT), 0, st>>>(p);
    SD_HIP_CHECK(hipGetLastError());
    k_smp_draw<<<dim3((unsigned)in.rows), dim3(kSmpT), 0, st>>>(p);
    SD_HIP_CHECK(hipGetLastError());
    if (p.probs) {
        k_smp_probs<<<dim3((unsigned)((in.V + 2047) / 2048), (unsigned)in.rows), dim3(256), 0, st>>>(p);
        SD_HIP_CHECK(hipGetLastError());
    }
}

}  // namespace sd
