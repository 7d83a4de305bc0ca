// Sampling: one token per row of logits from a given uniform, after the
// filters in this order:
//   w_i  = exp((l_i - max) / T)          (T = 0: the first maximum alone)
//   top-k  the k largest, of equal ones the first
//   top-p  the shortest run of the rest, largest first (of equal ones the
//          first), whose weights reach p times the rest's sum
//   min-p  of those the ones with w_i >= min_p
//   token  the first kept i whose running sum, by index, exceeds u times the
//          sum of the kept
// Weights are computed in f64 and summed as integers, so no sum depends on an
// order: of 2^-44 in the sums that a token is drawn from, of 2^-36 in the
// histograms.  A weight is within 1e-11 of itself, and a rounded sum of V of them
// loses at most half a unit for each, so a decision can differ from exact
// arithmetic only within 1e-11 and V * 2^-45 of the sum (with histograms V * 2^-37)
// of a border.
//
// Both top-k and top-p keep a prefix of the order (value descending, index
// ascending), so together they are one bound on the pair (value, index).  Two
// launches find it: k_smp_slices (a workgroup per 8192 entries) leaves each
// slice's maximum, a histogram over bins of equal width in l / T and its
// entries' places ordered by bin (for a top-k of up to 256 its up to 256 largest
// entries instead); k_smp_draw (a workgroup per row) adds the histograms, finds
// the bin in which the bound lies, takes that bin's entries (or, when they are
// few, all entries down to that bin) into LDS, finds the bound among them and
// draws: a slice by the slices' sums, then an entry of it.  k_smp_probs writes
// the kept distribution when asked.  (One row of 128256 with top-k 40: 6.5 us of
// slices and 10 of draw; 60 rows of 152064 with top-p: 29 and 23.)
//
// A row's draw is a chain of short steps that each run once, so its time is
// memory round trips and instruction fetches (about 0.15 us for a cache line of
// code that no wave has run yet): loads go out in batches, and what is done
// with them is a rolled loop, not sixteen copies of the f64 series.
#include "sd_sample.hpp"
#include "sd_common.hpp"

namespace sd {

constexpr int kSmpT = 1024, kSmpWaves = kSmpT / 64;  // of the draw
constexpr int kSmpList = 2048;             // entries taken into LDS
constexpr int kSmpCand = 256;              // largest entries kept of a slice
constexpr int kMaxSlices = kSmpMaxVocab / kSmpSlice;
constexpr double kOne = 17592186044416.0;  // 2^44
// A histogram word: the bin's weight in units of 2^-36 above 14 bits of its
// count (8192 weights of at most 1 make 49 bits).
constexpr double kBinOne = 68719476736.0;  // 2^36
constexpr int kCountBits = 14, kFactorBits = 8;  // kOne / kBinOne: 2^8

// Per slice: the largest entry's order key, whether an entry is NaN or +inf,
// the sum of the weights relative to the slice's maximum (kSmpSum), the entries
// listed and the number of bins whose entries all are (kSmpTopK), the finite
// entries (kSmpHist).
struct SmpSlice {
    uint32_t key, bad;
    uint64_t mass;
    int n, bins;
};
// What k_smp_draw leaves for k_smp_probs.
struct SmpRow {
    uint64_t cut;   // kept: order_of(key, index) >= cut ...
    uint64_t total; // sum of the kept weights; 0: no distribution
    float max;
    float pad;
};

struct SmpWs {
    uint64_t *hist;   // [rows][slices][kSmpBins]
    uint64_t *cand;   // [rows][slices][kSmpCand], kSmpTopK
    uint16_t *place;  // [rows][slices][kSmpSlice], kSmpHist: the entries' places by bin
    uint16_t *first;  // [rows][slices][kSmpBins]: entries of the bins above each
    SmpSlice *slice;  // [rows][slices]
    SmpRow *row;      // [rows]
};
static __host__ __device__ inline int smp_slices(int V) { return (V + kSmpSlice - 1) / kSmpSlice; }
static SmpWs smp_ws(void *p, int V, int rows) {
    const size_t n = (size_t)rows * smp_slices(V);
    SmpWs w;
    w.hist = (uint64_t *)p;
    w.cand = w.hist + n * kSmpBins;
    w.place = (uint16_t *)(w.cand + n * kSmpCand);
    w.first = w.place + n * kSmpSlice;
    w.slice = (SmpSlice *)(w.first + n * kSmpBins);
    w.row = (SmpRow *)(w.slice + n);
    return w;
}
size_t sample_ws_bytes(int V, int rows) {
    const size_t n = (size_t)rows * smp_slices(V);
    return n * ((kSmpBins + kSmpCand) * sizeof(uint64_t) + sizeof(SmpSlice) + (kSmpSlice + kSmpBins) * sizeof(uint16_t)) +
           (size_t)rows * sizeof(SmpRow);
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
__device__ __forceinline__ int index_of(uint64_t order) { return kSmpMaxVocab - 1 - (int)(order & (kSmpMaxVocab - 1)); }
__device__ __forceinline__ float value_of(uint64_t order) { return of_key((uint32_t)(order >> 18)); }
// bin grid in l / T, the same for all slices; monotone in l
__device__ __forceinline__ int bin_of(float l, float bins_per) {
    return (int)floorf(fminf(fmaxf(l * bins_per, -1.0e9f), 1.0e9f));
}
// exp2((l - max) * c) to 1e-11, c = log2(e) / T: the power of two of the
// rounded exponent times ten terms of the exponential series of the rest
// (|y| < 0.347: the eleventh is below 3e-13)
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
    int mode;        // SmpMode
    const float *u;
    int *tokens;
    float *probs;
    SmpWs ws;
};

__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// running sum over the lanes, the lane's own value included
template <typename T> __device__ __forceinline__ T wave_run(T v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T up = __shfl_up(v, o);
        if (lane >= o) v += up;
    }
    return v;
}

// ---- slices ----------------------------------------------------------------------
// What the first launch leaves: the slice's sum (no bound to find), counts only
// inside it and its candidates (a top-k that they can hold), or the histogram
// and the candidates.
enum SmpMode : int { kSmpSum = 0, kSmpTopK = 1, kSmpHist = 2 };

// A workgroup's time is the length of its chain (one row of 128256 is 16
// workgroups on 256 CUs) and of the code that it runs once: 1024 threads with
// two loads of four entries each, rolled loops over the entries (32 entries a
// thread, unrolled: 10 us for one row, 4 of them fetching the last loop's code;
// now 6.5).  Many rows are bound by VALU work, 82 instructions an entry and a
// quarter of them f64, issued in 91 % of the CUs' busy cycles: 60 rows of 152064
// take 29 us, 6 at the rate of a large read (and 30 MB of places and histograms
// are written).  The histogram's loop therefore takes two entries a turn (one: 31
// us; four: the same as two; entries in LDS instead of turned registers: 31).
constexpr int kSlT = 1024, kSlPer = kSmpSlice / kSlT;
typedef float floatx4r __attribute__((ext_vector_type(4), aligned(4)));

// the next N of a thread's entries into l[0] ..
template <int N, typename T> __device__ __forceinline__ void turn(T (&l)[kSlPer]) {
    T first[N];
#pragma unroll
    for (int k = 0; k < N; k++) first[k] = l[k];
#pragma unroll
    for (int k = 0; k + N < kSlPer; k++) l[k] = l[k + N];
#pragma unroll
    for (int k = 0; k < N; k++) l[kSlPer - N + k] = first[k];
}

template <int MODE> __global__ __launch_bounds__(kSlT) void k_smp_slices(const SmpCfg p) {
    __shared__ uint64_t hist[MODE == kSmpHist ? kSmpBins : 1];
    __shared__ uint32_t cnt[MODE == kSmpTopK ? kSmpBins : 1];
    __shared__ __align__(16) uint16_t place[MODE == kSmpHist ? kSmpSlice : 1];
    __shared__ uint32_t wcnt[kSlT / 64], s_key, s_bad, s_n;
    __shared__ uint64_t s_mass;
    __shared__ int s_bins;
    const int sl = blockIdx.x, r = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const float *row = p.logits + (int64_t)r * p.ld + (int64_t)sl * kSmpSlice;
    const int len = min(kSmpSlice, p.V - sl * kSmpSlice);
    // entry k of the thread is x = 4096 (k >> 2) + 4 t + (k & 3)
    float l[kSlPer];
#pragma unroll
    for (int i = 0; i < kSlPer / 4; i++) {
        const int x = i * 4 * kSlT + 4 * t;
        if (x + 4 <= len) {
            const floatx4r v = *(const floatx4r *)(row + x);
            l[4 * i] = v.x, l[4 * i + 1] = v.y, l[4 * i + 2] = v.z, l[4 * i + 3] = v.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) l[4 * i + k] = x + k < len ? row[x + k] : -INFINITY;
        }
    }
    if (t == 0) s_key = s_bad = s_n = 0, s_mass = 0, s_bins = kSmpBins;
    if constexpr (MODE == kSmpHist) hist[t] = 0;
    if constexpr (MODE == kSmpTopK) cnt[t] = 0;
    float m = -INFINITY;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < kSlPer; i++) {
        bad |= l[i] != l[i] || l[i] == INFINITY;
        m = fmaxf(m, l[i]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    bad = __ballot(bad != 0) != 0;
    __syncthreads();
    if (lane == 0) {
        atomicMax(&s_key, key_of(m));
        if (bad) s_bad = 1;
    }
    __syncthreads();
    const uint32_t key = s_key;
    SmpSlice *out = p.ws.slice + (int64_t)r * p.nsl + sl;
    if (s_bad || key <= kKeyNegInf) {
        // nothing to weigh: the histogram of a slice with key <= -inf is not read
        if (t == 0) *out = SmpSlice{key, s_bad, 0, 0, kSmpBins};
        return;
    }
    m = of_key(key);
    const int top = bin_of(m, p.bins_per);
    uint64_t sum = 0;
    uint32_t at[kSlPer];  // kSmpHist: the entry's bin and its rank in it (bin << 16 | rank)
    constexpr int kStep = MODE == kSmpHist ? 2 : 1;
#pragma unroll 1
    for (int i = 0; i < kSlPer; i += kStep) {
#pragma unroll
        for (int k = 0; k < kStep; k++) {
            if constexpr (MODE == kSmpSum) {
                sum += to_int(weight(l[k], m, p.c) * kOne);  // -inf weighs 0
                continue;
            }
            at[k] = ~0u;
            if (l[k] > -INFINITY) {
                const int b = min(top - bin_of(l[k], p.bins_per), kSmpBins - 1);
                if constexpr (MODE == kSmpTopK)
                    atomicAdd(&cnt[b], 1u);
                else
                    at[k] = (uint32_t)b << 16 |
                            ((uint32_t)atomicAdd((unsigned long long *)&hist[b],
                                                 (unsigned long long)((to_int(weight(l[k], m, p.c) * kBinOne) << kCountBits) + 1)) &
                             ((1u << kCountBits) - 1));
            }
        }
        if constexpr (MODE == kSmpHist) turn<kStep>(at);
        turn<kStep>(l);
    }
    if constexpr (MODE == kSmpSum) {
        sum = wave_sum(sum);
        if (lane == 0) atomicAdd((unsigned long long *)&s_mass, (unsigned long long)sum);
        __syncthreads();
        if (t == 0) *out = SmpSlice{key, 0, s_mass, 0, kSmpBins};
        return;
    }
    __syncthreads();
    // entries of the bins above, and with the thread's own bin
    const uint64_t h = MODE == kSmpHist ? hist[t] : 0;
    const uint32_t c = MODE == kSmpHist ? (uint32_t)h & ((1u << kCountBits) - 1) : cnt[MODE == kSmpTopK ? t : 0];
    uint32_t run = wave_run(c);
    if (lane == 63) wcnt[wave] = run;
    __syncthreads();
    uint32_t before = lane < wave ? wcnt[lane & 15] : 0;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) before += __shfl_xor(before, o);
    run += __shfl(before, 0);
    if constexpr (MODE == kSmpHist) {
        hist[t] = run - c;
        p.ws.hist[((int64_t)r * p.nsl + sl) * kSmpBins + t] = h;
        p.ws.first[((int64_t)r * p.nsl + sl) * kSmpBins + t] = (uint16_t)(run - c);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSlPer; i++)
            if (at[i] != ~0u)
                place[(uint32_t)hist[at[i] >> 16] + (at[i] & 0xffffu)] = (uint16_t)((i >> 2) * 4 * kSlT + 4 * t + (i & 3));
        __syncthreads();
        // (places past the finite entries are not read)
        *(uintx4 *)(p.ws.place + ((int64_t)r * p.nsl + sl) * kSmpSlice + 8 * t) = *(const uintx4 *)(place + 8 * t);
        if (t == kSlT - 1) *out = SmpSlice{key, 0, 0, (int)run, kSmpBins};
    } else {
        // the one bin at which the running count passes the candidates
        if (run > (uint32_t)kSmpCand && run - c <= (uint32_t)kSmpCand) s_bins = t;
        __syncthreads();
        const int bins = s_bins;
        uint64_t *cand = p.ws.cand + ((int64_t)r * p.nsl + sl) * kSmpCand;
#pragma unroll 1
        for (int i = 0; i < kSlPer; i++) {
            if (l[0] > -INFINITY && min(top - bin_of(l[0], p.bins_per), kSmpBins - 1) < bins)
                cand[atomicAdd(&s_n, 1u)] = order_of(key_of(l[0]), sl * kSmpSlice + (i >> 2) * 4 * kSlT + 4 * t + (i & 3));
            turn<1>(l);
        }
        __syncthreads();
        if (t == 0) *out = SmpSlice{key, 0, 0, (int)s_n, bins};
    }
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
    uint64_t smass[kMaxSlices];
    double f[kMaxSlices];
    int shift[kMaxSlices];  // of the slice's bins against the row's; -1: a slice without entries
    int n_in[kMaxSlices], bins[kMaxSlices];
    int seg[kMaxSlices], seg_at[kMaxSlices + 1];  // a bin range's entries: first place of each slice, entries before it
    uint64_t a;
    int n, i;
};

// sum of the waves' values before this one's (v: the wave's, in any lane 63), total: of all
template <typename T> __device__ __forceinline__ T waves_before(T *sh, T wave_total, T &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 63) sh[wave] = wave_total;
    __syncthreads();
    const T v = wave_run(sh[lane & 15]);
    total = __shfl(v, 15);
    return wave ? __shfl(v, max(wave - 1, 0)) : 0;
}
// the workgroup's sum, to every thread
__device__ __forceinline__ uint64_t group_sum(SmpShared &S, uint64_t v) {
    v = wave_sum(v);
    __syncthreads();
    uint64_t total;
    waves_before(S.wsum, v, total);
    return total;
}

// Entries to select from, those at or above `least`: the list in LDS, the
// row's entries of some bins (their places from set_segments), the whole row.
struct ListSource {
    SmpShared &S;
    int n;
    uint64_t least;
    template <typename F> __device__ __forceinline__ void each(F &&f) const {
#pragma unroll 1
        for (int i = threadIdx.x; i < n; i += kSmpT)
            if (S.lorder[i] >= least) f(S.lorder[i], S.lmass[i]);
    }
};
struct BinSource {
    SmpShared &S;
    const SmpCfg &p;
    const float *row;
    float max;
    int r;
    uint64_t least;
    __device__ __forceinline__ uint64_t order_at(int i) const {
        int s = 0;
#pragma unroll
        for (int o = kMaxSlices / 2; o > 0; o >>= 1)
            if (s + o < p.nsl && S.seg_at[s + o] <= i) s += o;
        const int x = s * kSmpSlice + p.ws.place[((int64_t)r * p.nsl + s) * kSmpSlice + S.seg[s] + (i - S.seg_at[s])];
        return order_of(key_of(row[x]), x);
    }
    template <typename F> __device__ __forceinline__ void each(F &&f) const {
        const int n = S.seg_at[p.nsl];
#pragma unroll 1
        for (int i = threadIdx.x; i < n; i += kSmpT) {
            const uint64_t order = order_at(i);
            if (order >= least) f(order, to_int(weight(value_of(order), max, p.c) * kOne));
        }
    }
};
struct RowSource {
    const SmpCfg &p;
    const float *row;
    float max;
    uint64_t least;
    template <typename F> __device__ __forceinline__ void each(F &&f) const {
        constexpr int kDeep = 8;
#pragma unroll 1
        for (int x = threadIdx.x; x < p.V; x += kDeep * kSmpT) {
            float l[kDeep];
#pragma unroll
            for (int k = 0; k < kDeep; k++) l[k] = row[min(x + k * kSmpT, p.V - 1)];
#pragma unroll 1
            for (int k = 0; k < kDeep; k++) {
                const int i = x + k * kSmpT;
                if (i < p.V && l[0] > -INFINITY && order_of(key_of(l[0]), i) >= least)
                    f(order_of(key_of(l[0]), i), to_int(weight(l[0], max, p.c) * kOne));
#pragma unroll
                for (int e = 0; e + 1 < kDeep; e++) l[e] = l[e + 1];
            }
        }
    }
};

// The entry at which the running count (or sum) over the source, in
// descending order, first reaches `target`; the last entry if it never does.
// Eight bits of the order number at a time, from bit `shift` on, the bits
// above being `prefix`; it ends early with an entry that is alone.  All
// threads; returns its order.
template <typename Src>
__device__ __forceinline__ uint64_t select(SmpShared &S, const Src &src, bool by_mass, uint64_t target, int shift, uint64_t prefix) {
    const int t = threadIdx.x;
#pragma unroll 1
    for (; shift >= 0; shift -= 8) {
        __syncthreads();
        if (t < 256) S.dmass[t] = 0, S.dcount[t] = 0;
        __syncthreads();
        src.each([&](uint64_t order, uint64_t mass) {
            if ((order >> (shift + 8)) != prefix) return;
            const int d = (int)(order >> shift) & 255;
            atomicAdd(&S.dcount[d], 1u);
            if (by_mass && mass) atomicAdd((unsigned long long *)&S.dmass[d], (unsigned long long)mass);
        });
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
            uint64_t before = wave_run(sum) - sum;
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
                S.i = 255 - 4 * t - (31 - __clz((int)any));
                S.a = ~0ull >> 1;
            } else if (!has && t == 0) {
                S.i = 0;
                S.a = 0;
            }
        }
        __syncthreads();
        prefix = (prefix << 8) | (uint64_t)S.i;
        target = S.a;
        if (shift && S.dcount[S.i] == 1) {
            __syncthreads();
            src.each([&](uint64_t order, uint64_t) {
                if ((order >> shift) == prefix) S.a = order;
            });
            __syncthreads();
            return S.a;
        }
    }
    return prefix;
}
constexpr int kOrderShift = 48, kIndexShift = 16;  // of 50 and 18 bits
// the same on the list, from the first digit in which its entries differ
__device__ __forceinline__ uint64_t select_list(SmpShared &S, int n, uint64_t least, bool by_mass, uint64_t target) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const uint64_t some = S.lorder[0];
    uint64_t diff = 0;
#pragma unroll 1
    for (int i = t; i < n; i += kSmpT) diff |= S.lorder[i] ^ some;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) diff |= __shfl_xor(diff, o);
    __syncthreads();
    if (lane == 0) S.wsum[wave] = diff;
    __syncthreads();
    diff = S.wsum[lane & 15];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) diff |= __shfl_xor(diff, o);
    diff = __shfl(diff, 0);
    const int shift = diff ? (63 - __clzll((long long)diff)) / 8 * 8 : 0;
    return select(S, ListSource{S, n, least}, by_mass, target, shift, some >> (shift + 8));
}

// The weight of an entry if it is kept, `one` units for a weight of 1.
struct Kept {
    const SmpCfg &p;
    const float *row;
    float max;
    uint64_t cut;
    __device__ __forceinline__ uint64_t mass(int i, float l, double one = kOne) const {
        if (l == -INFINITY || order_of(key_of(l), i) < cut) return 0;
        const double w = weight(l, max, p.c);
        return w >= p.min_p ? to_int(w * one) : 0;
    }
};
// the slices' kept weights from the row itself, a slice to a wave, into S.smass
__device__ __forceinline__ void row_sums(SmpShared &S, const Kept &k) {
    constexpr int kDeep = 8;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll 1
    for (int sl = wave; sl < k.p.nsl; sl += kSmpWaves) {
        const int a = sl * kSmpSlice, b = min(k.p.V, a + kSmpSlice);
        uint64_t s = 0;
#pragma unroll 1
        for (int i = a + lane; i < b; i += kDeep * 64) {
            float l[kDeep];
#pragma unroll
            for (int d = 0; d < kDeep; d++) l[d] = k.row[min(i + d * 64, b - 1)];
#pragma unroll 1
            for (int d = 0; d < kDeep; d++) {
                if (i + d * 64 < b) s += k.mass(i + d * 64, l[0]);
#pragma unroll
                for (int e = 0; e + 1 < kDeep; e++) l[e] = l[e + 1];
            }
        }
        s = wave_sum(s);
        if (lane == 0) S.smass[sl] = s;
    }
    __syncthreads();
}

// u times sum as the least running sum that exceeds it
__device__ __forceinline__ uint64_t draw_target(float u, uint64_t sum) {
    const double t = fmin(fmax((double)u, 0.0), 1.0) * (double)sum;
    return min((uint64_t)t + 1, sum);
}

// The draw: a slice by the slices' sums, then the first of its entries whose
// running kept weight reaches what is left of the target (the last kept one
// where rounded sums leave more than the slice has).
// A slice may be far below the row's maximum (its sum some units of 2^-44, each
// of its entries less than half a unit), so inside it weights and target are
// in units of 2^-44 of its maximum's power of two: the maximum, which is
// kept where anything of the slice is, weighs 2^44 or more, and a slice that
// is picked always has an entry to give.
__device__ __forceinline__ int draw_slices(SmpShared &S, const Kept &k, float u, uint64_t &total) {
    const int t = threadIdx.x, lane = t & 63;
    const uint64_t sm = lane < k.p.nsl ? S.smass[lane & (kMaxSlices - 1)] : 0, sr = wave_run(sm);
    total = __shfl(sr, 63);
    uint64_t target = draw_target(u, total);
    uint64_t hit = __ballot(sm && sr >= target);
    if (!hit) hit = 1;  // no weight at all
    const int pick = __ffsll((unsigned long long)hit) - 1;
    target -= min(__shfl(sr - sm, pick), target - 1);
    // its maximum's exponent, from the factor of its sums; a sum of a unit or more has a maximum of 2^-58 or more (8192
    // entries, half a unit lost to rounding)
    const int e = (int)(__builtin_bit_cast(uint64_t, S.f[pick]) >> 52) - (k.p.mode == kSmpHist ? kFactorBits : 0);
    const int down = min(1023 - e, 58);
    const double one = __builtin_bit_cast(double, (uint64_t)(1023 + 44 + down) << 52);
    target = ((target - 1) << down) + 1;
    // eight entries to a thread, in order
    const int x0 = pick * kSmpSlice + 8 * t, len = k.p.V - x0;
    float l[8];
#pragma unroll
    for (int e = 0; e < 2; e++)
        if (4 * e + 4 <= len) {
            const floatx4r v = *(const floatx4r *)(k.row + x0 + 4 * e);
            l[4 * e] = v.x, l[4 * e + 1] = v.y, l[4 * e + 2] = v.z, l[4 * e + 3] = v.w;
        } else {
#pragma unroll
            for (int i = 4 * e; i < 4 * e + 4; i++) l[i] = i < len ? k.row[x0 + i] : -INFINITY;
        }
    uint64_t mine = 0, m[8];
#pragma unroll 1
    for (int e = 0; e < 8; e++) {
        const uint64_t w = k.mass(x0 + e, l[0], one);
        mine += w;
#pragma unroll
        for (int i = 0; i < 7; i++) l[i] = l[i + 1], m[i] = m[i + 1];
        m[7] = w;
    }
    uint64_t run = wave_run(mine), all;
    __syncthreads();
    if (t == 0) S.n = 0x7fffffff, S.i = -1;
    run += waves_before(S.wsum, run, all);
    uint64_t before = run - mine;
    int first = 0x7fffffff, last = -1;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        before += m[e];
        if (m[e]) {
            if (before >= target) first = min(first, x0 + e);
            last = x0 + e;
        }
    }
    if (first != 0x7fffffff) atomicMin(&S.n, first);
    if (last >= 0 && target > all) atomicMax(&S.i, last);
    __syncthreads();
    return S.n != 0x7fffffff ? S.n : S.i;
}

// the places of the row's entries in bins [lo, hi]; returns their number
__device__ __forceinline__ int set_segments(SmpShared &S, const SmpCfg &p, int r, int lo, int hi) {
    const int t = threadIdx.x;
    __syncthreads();
    if (t < 64) {
        int n = 0;
        if (t < p.nsl && S.shift[t] >= 0) {
            // the slice's own bins; its last one holds what lies below them all
            const int a = max(lo - S.shift[t], 0), b = hi == kSmpBins - 1 ? kSmpBins - 1 : hi - S.shift[t];
            const uint16_t *first = p.ws.first + ((int64_t)r * p.nsl + t) * kSmpBins;
            if (a <= b) {
                const int start = first[a], end = b == kSmpBins - 1 ? S.n_in[t] : first[b + 1];
                S.seg[t] = start;
                n = end - start;
            }
        }
        const int run = wave_run(n);
        if (t < kMaxSlices) S.seg_at[t] = run - n;
        if (t == 63) S.seg_at[p.nsl] = run;
    }
    __syncthreads();
    return S.seg_at[p.nsl];
}

// The row's entries of bins [lo, hi], at most kSmpList of them, into the list
// with their weights; returns their number.
__device__ __forceinline__ int gather(SmpShared &S, const BinSource &src, int lo, int hi) {
    const int n = min(set_segments(S, src.p, src.r, lo, hi), kSmpList);
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += kSmpT) {
        const uint64_t o = src.order_at(i);
        S.lorder[i] = o;
        S.lmass[i] = to_int(weight(value_of(o), src.max, src.p.c) * kOne);
    }
    __syncthreads();
    return n;
}

// the slices' weights in the bins above `b`, into S.smass
__device__ __forceinline__ void slice_sums(SmpShared &S, const SmpCfg &p, int r, int b) {
    const int s = threadIdx.x >> 5, j = threadIdx.x & 31;
    uint64_t sum = 0;
    if (s < p.nsl && S.shift[s] >= 0) {
        const uint64_t *h = p.ws.hist + ((int64_t)r * p.nsl + s) * kSmpBins;
        const int end = min(b - S.shift[s], kSmpBins);  // local bins below it lie above b
        const double f = S.f[s];
#pragma unroll 1
        for (int i = j; i < end; i += 32 * 8) {
            uint64_t v[8];
#pragma unroll
            for (int d = 0; d < 8; d++) v[d] = i + 32 * d < end ? h[i + 32 * d] : 0;
#pragma unroll
            for (int d = 0; d < 8; d++) sum += (uint64_t)rint((double)(v[d] >> kCountBits) * f);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (j == 0) S.smass[s] = sum;
    __syncthreads();
}

// All filters on a list of up to 64 entries that holds every entry down to the
// bounds' bin (sum: the weight of all entries of the row): one wave, an entry
// in each lane, no barriers.
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)v, lane) |
           (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), lane) << 32;
}
__device__ __forceinline__ int draw_wave(const SmpCfg &p, uint64_t mine, int n, bool k_on, bool p_on, uint64_t sum, float max,
                                         float u, uint64_t &cut, uint64_t &total) {
    const int t = threadIdx.x;
    const double w = weight(value_of(mine), max, p.c);
    uint64_t m = t < n ? to_int(w * kOne) : 0;
    int rank = 0;
    uint64_t above = 0;
#pragma unroll 1
    for (int j = 0; j < n; j++) {
        const bool hi = lane_u64(mine, j) > mine;
        const uint64_t mj = lane_u64(m, j);
        rank += hi;
        above += hi ? mj : 0;
    }
    bool keep = t < n && (!k_on || rank < p.top_k);
    if (p_on) {
        const uint64_t of = k_on ? wave_sum(keep ? m : 0) : sum;
        keep = keep && (above < (uint64_t)ceil(p.top_p * (double)of) || rank == 0);
    }
    // the entry that k and p keep last is the bound
    const uint64_t kept = __ballot(keep);
    int lowest = keep ? rank : -1;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) lowest = ::max(lowest, __shfl_xor(lowest, o));
    cut = k_on || p_on ? lane_u64(mine, __ffsll((unsigned long long)__ballot(keep && rank == lowest)) - 1) : 0;
    keep = keep && w >= p.min_p;
    if (!keep) m = 0;
    total = wave_sum(m);
    const uint32_t x = (uint32_t)mine & (kSmpMaxVocab - 1);  // larger: earlier
    uint64_t before = 0;
#pragma unroll 1
    for (uint64_t left = kept; left; left &= left - 1) {
        const int j = __ffsll((unsigned long long)left) - 1;
        const uint64_t mj = lane_u64(m, j);
        before += (uint32_t)__builtin_amdgcn_readlane(x, j) > x ? mj : 0;
    }
    int token = keep && m && before + m >= draw_target(u, total) ? index_of(mine) : 0x7fffffff;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) token = min(token, __shfl_xor(token, o));
    return token;
}

// first bin whose running sum reaches target, else the last bin
__device__ __forceinline__ int bin_reaching(SmpShared &S, uint64_t target) {
    __syncthreads();
    if (threadIdx.x == 0) S.i = kSmpBins - 1;
    __syncthreads();
    const int b = threadIdx.x;
    if (S.mass[b] >= target && (b == 0 || S.mass[b - 1] < target)) S.i = b;
    __syncthreads();
    return S.i;
}

// a - b within [0, kSmpBins], for bins up to 1e9 either way
__device__ __forceinline__ int max_sub(int a, int b) { return (int)min(std::max<int64_t>((int64_t)a - b, 0), (int64_t)kSmpBins); }

__global__ __launch_bounds__(kSmpT) void k_smp_draw(const SmpCfg p) {
    __shared__ SmpShared S;
    const int r = blockIdx.x, t = threadIdx.x, lane = t & 63;
    const float *row = p.logits + (int64_t)r * p.ld;
    // every wave finds the row's maximum from the slices'
    const SmpSlice mine = lane < p.nsl ? p.ws.slice[(int64_t)r * p.nsl + lane] : SmpSlice{0, 0, 0, 0, 0};
    const float u = p.u[r];
    uint32_t key = mine.key, bad = mine.bad;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor(key, o));
    key = max(key, __shfl_xor(key, 32));
    if (__ballot(bad != 0) || key <= kKeyNegInf) {
        if (t == 0) {
            p.tokens[r] = -1;
            p.ws.row[r] = SmpRow{0, 0, 0.f, 0.f};
        }
        return;
    }
    const float max = of_key(key);
    const int top = bin_of(max, p.bins_per);
    if (t < p.nsl) {
        const bool some = mine.key > kKeyNegInf;
        const float m = of_key(mine.key);
        const double f = some ? weight(m, max, p.c) : 0.0;
        S.f[t] = f * (p.mode == kSmpHist ? kOne / kBinOne : 1.0);
        S.shift[t] = some ? min(top - bin_of(m, p.bins_per), kSmpBins) : -1;
        S.smass[t] = (uint64_t)rint((double)mine.mass * f);
        S.n_in[t] = mine.n;
        S.bins[t] = mine.bins;
    }
    S.mass[t] = 0;
    S.count[t] = 0;
    if (t == 0) S.n = S.i = kSmpBins - 1;
    uint64_t cut = 0, total = 0;
    int token;
    __syncthreads();
    const BinSource src{S, p, row, max, r, 0};
    if (p.mode == kSmpSum) {
        const Kept k{p, row, max, 0};
        token = draw_slices(S, k, u, total);
    } else if (p.mode == kSmpTopK) {
        // the candidates of all slices, in registers, and their counts by bin
        constexpr int kPer = kMaxSlices * kSmpCand / kSmpT;
        uint64_t o[kPer];
#pragma unroll
        for (int k = 0; k < kPer; k++) {
            const int y = t + k * kSmpT, s = y / kSmpCand;
            const bool has = s < p.nsl && S.shift[s] >= 0 && y % kSmpCand < S.n_in[s];
            o[k] = has ? p.ws.cand[(int64_t)r * p.nsl * kSmpCand + y] : 0;
        }
#pragma unroll
        for (int k = 0; k < kPer; k++)
            if (o[k]) atomicAdd(&S.count[min(top - bin_of(value_of(o[k]), p.bins_per), kSmpBins - 1)], 1u);
        __syncthreads();
        {
            const uint32_t own = S.count[t];
            uint32_t all, c = wave_run(own);
            c += waves_before(S.wcnt, c, all);
            // the one bin at which the running count reaches top_k; the last where none does
            if (c >= (uint32_t)p.top_k && c - own < (uint32_t)p.top_k) S.n = t;
            S.count[t] = c;
            __syncthreads();
        }
        const int hi = S.n, few = (int)S.count[hi];
        const int s = lane & (kMaxSlices - 1);
        // A slice's entries down to hi are all listed (the row's last bin takes what lies below it, however far down), or
        // top_k of its largest are, and what it does not list is none of the row's top_k.
        const int need = hi == kSmpBins - 1 ? kSmpBins : hi - S.shift[s] + 1;
        const bool short_of = s < p.nsl && S.shift[s] >= 0 && need > S.bins[s] && S.n_in[s] < p.top_k;
        const bool whole = few <= kSmpList && __ballot(short_of) == 0;
        const bool p_on = p.top_p < 1.0;
        __syncthreads();
        if (t == 0) S.n = 0;
        __syncthreads();
        if (whole) {
#pragma unroll
            for (int k = 0; k < kPer; k++)
                if (o[k] && min(top - bin_of(value_of(o[k]), p.bins_per), kSmpBins - 1) <= hi) S.lorder[atomicAdd(&S.n, 1)] = o[k];
            __syncthreads();
        }
        const int n = S.n;
        if (whole && n <= 64) {
            if (t >= 64) return;
            token = draw_wave(p, t < n ? S.lorder[t] : 0, n, true, p_on, 0, max, u, cut, total);
        } else {
            // more entries, or (not whole) more than 256 of a slice too close together: then from the row
            if (whole) {
#pragma unroll 1
                for (int i = t; i < n; i += kSmpT) S.lmass[i] = to_int(weight(value_of(S.lorder[i]), max, p.c) * kOne);
                __syncthreads();
                cut = select_list(S, n, 0, false, (uint64_t)p.top_k);
            } else {
                cut = select(S, RowSource{p, row, max, 0}, false, (uint64_t)p.top_k, kOrderShift, 0);
            }
            if (p_on) {
                uint64_t sum = 0;
                if (whole) ListSource{S, n, cut}.each([&](uint64_t, uint64_t m) { sum += m; });
                else RowSource{p, row, max, cut}.each([&](uint64_t, uint64_t m) { sum += m; });
                const uint64_t target = std::max<uint64_t>(1, (uint64_t)ceil(p.top_p * (double)group_sum(S, sum)));
                cut = whole ? select_list(S, n, cut, true, target)
                            : select(S, RowSource{p, row, max, cut}, true, target, kOrderShift, 0);
            }
            const Kept k{p, row, max, cut};
            if (whole) {
                // the slices' sums from the list
                __syncthreads();
                if (t < kMaxSlices) S.smass[t] = 0;
                __syncthreads();
#pragma unroll 1
                for (int i = t; i < n; i += kSmpT)
                    if (S.lorder[i] >= cut && weight(value_of(S.lorder[i]), max, p.c) >= p.min_p)
                        atomicAdd((unsigned long long *)&S.smass[index_of(S.lorder[i]) / kSmpSlice], (unsigned long long)S.lmass[i]);
                __syncthreads();
            } else {
                row_sums(S, k);
            }
            token = draw_slices(S, k, u, total);
        }
    } else {
        // the slices' histograms, sixteen words in flight
#pragma unroll 1
        for (int s0 = 0; s0 < p.nsl; s0 += 16) {
            uint64_t h[16];
#pragma unroll
            for (int s = 0; s < 16; s++) {
                const bool has = s0 + s < p.nsl && S.shift[min(s0 + s, p.nsl - 1)] >= 0;
                h[s] = has ? p.ws.hist[((int64_t)r * p.nsl + s0 + s) * kSmpBins + t] : 0;
            }
#pragma unroll
            for (int s = 0; s < 16; s++) {
                const uint32_t c = (uint32_t)h[s] & ((1u << kCountBits) - 1);
                if (!c) continue;
                const int b = min(t + S.shift[s0 + s], kSmpBins - 1);
                atomicAdd(&S.count[b], c);
                const uint64_t w = (uint64_t)rint((double)(h[s] >> kCountBits) * S.f[s0 + s]);
                if (w) atomicAdd((unsigned long long *)&S.mass[b], (unsigned long long)w);
            }
        }
        __syncthreads();
        const uint32_t own_c = S.count[t];
        const uint64_t own_m = S.mass[t];
        uint64_t kept, m = wave_run(own_m);  // kept: the sum of the entries left so far
        uint32_t entries, c = wave_run(own_c);
        m += waves_before(S.wsum, m, kept);
        c += waves_before(S.wcnt, c, entries);
        // the one bin at which the running count (sum) reaches the bound; the last where none does
        if (c >= (uint32_t)p.top_k && c - own_c < (uint32_t)p.top_k) S.n = t;
        const uint64_t p_target = std::max<uint64_t>(1, (uint64_t)ceil(p.top_p * (double)kept));
        if (m >= p_target && m - own_m < p_target) S.i = t;
        S.mass[t] = m;
        S.count[t] = c;
        __syncthreads();
        bool k_on = p.top_k > 0 && (uint32_t)p.top_k < entries, p_on = p.top_p < 1.0;
        int hi = kSmpBins - 1;  // the bin of the last entry left
        if (k_on) hi = S.n;
        else if (p_on) hi = S.i;
        // min-p keeps all of the bins above m_lo and nothing below m_hi: its bound is in [m_lo, m_hi]
        int m_lo = kSmpBins, m_hi = kSmpBins - 1;
        if (p.min_p > 0.0) {
            // the bound as a float is off by less than its neighbours
            const float at = (float)((double)max + log2(p.min_p) / p.c);
            m_lo = max_sub(top, bin_of(nextafterf(at, INFINITY), p.bins_per));
            m_hi = min(max_sub(top, bin_of(nextafterf(at, -INFINITY), p.bins_per)), kSmpBins - 1);
        }
        const bool by_min = m_hi < hi && !(k_on && p_on);  // the other bound lies below min-p's: min-p alone decides
        if (by_min || !(k_on || p_on)) {
            k_on = p_on = false;
            hi = m_hi;
        }
        // all entries down to hi, if the list holds them; else the bins of the bounds one after the other
        const bool all = S.count[hi] <= (uint32_t)kSmpList;
        int n = 0;
        if (all) n = gather(S, src, 0, hi);
        if (all && n <= 64) {
            if (t >= 64) return;
            token = draw_wave(p, t < n ? S.lorder[t] : 0, n, k_on, p_on, kept, max, u, cut, total);
        } else {
            // the bound in bin b at `target`, counted from the row's first entry; leaves the bin's entries in the list
            // where it holds them
            bool listed = false;
            auto bound = [&](int b, bool by_mass, uint64_t target) -> uint64_t {
                if (all) return select_list(S, n, cut, by_mass, target);
                const uint64_t above = b ? (by_mass ? S.mass[b - 1] : S.count[b - 1]) : 0;
                const uint32_t in_bin = S.count[b] - (b ? S.count[b - 1] : 0);
                target = target > above ? target - above : 1;
                listed = in_bin <= (uint32_t)kSmpList;
                if (listed) {
                    n = gather(S, src, b, b);
                    return select_list(S, n, cut, by_mass, target);
                }
                set_segments(S, p, r, b, b);
                return select(S, BinSource{S, p, row, max, r, cut}, by_mass, target, kOrderShift, 0);
            };
            if (k_on) {
                cut = bound(hi, false, (uint64_t)p.top_k);
                if (p_on) {
                    uint64_t sum = 0;
                    if (all || listed) ListSource{S, n, cut}.each([&](uint64_t, uint64_t w) { sum += w; });
                    else BinSource{S, p, row, max, r, cut}.each([&](uint64_t, uint64_t w) { sum += w; });
                    kept = group_sum(S, sum) + (all || !hi ? 0 : S.mass[hi - 1]);
                }
            }
            if (p_on) {
                const uint64_t target = std::max<uint64_t>(1, (uint64_t)ceil(p.top_p * (double)kept));
                hi = std::min(hi, bin_reaching(S, target));
                cut = std::max(cut, bound(hi, true, target));
            }
            // Of the bins above lo every entry is kept, of [lo, end] those that the bounds keep, below none.
            int lo = std::min(hi, m_lo);
            const int end = std::min(hi, m_hi);
            __syncthreads();
            if (all) lo = 0;
            slice_sums(S, p, r, lo);
            auto add = [&](uint64_t order, uint64_t w) {
                if (p.min_p <= 0.0 || weight(value_of(order), max, p.c) >= p.min_p)
                    atomicAdd((unsigned long long *)&S.smass[index_of(order) / kSmpSlice], (unsigned long long)w);
            };
            if (all || (listed && lo == hi)) {
                ListSource{S, n, cut}.each(add);
            } else {
                set_segments(S, p, r, lo, end);
                BinSource{S, p, row, max, r, cut}.each(add);
            }
            __syncthreads();
            const Kept k{p, row, max, cut};
            token = draw_slices(S, k, u, total);
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
    // A slice's candidates hold a top-k of up to 256 (of the whole row, so of any slice); histograms for the other
    // bounds, min-p alone among them (2 rows of 128256: 21 us; the draw's one workgroup adding up its row again 60).
    p.mode = p.top_k > 0 && p.top_k <= kSmpCand ? kSmpTopK : p.top_k > 0 || p.top_p < 1.0 || p.min_p > 0.0 ? kSmpHist : kSmpSum;
    p.u = in.u;
    p.tokens = in.tokens;
    p.probs = in.probs;
    p.ws = smp_ws(in.ws, in.V, in.rows);
    const dim3 g((unsigned)p.nsl, (unsigned)in.rows), b(kSlT);
    if (p.mode == kSmpSum) k_smp_slices<kSmpSum><<<g, b, 0, st>>>(p);
    else if (p.mode == kSmpTopK) k_smp_slices<kSmpTopK><<<g, b, 0, st>>>(p);
    else k_smp_slices<kSmpHist><<<g, b, 0, st>>>(p);
    SD_HIP_CHECK(hipGetLastError());
    k_smp_draw<<<dim3((unsigned)in.rows), dim3(kSmpT), 0, st>>>(p);
    SD_HIP_CHECK(hipGetLastError());
    if (p.probs) {
        k_smp_probs<<<dim3((unsigned)((in.V + 2047) / 2048), (unsigned)in.rows), dim3(256), 0, st>>>(p);
        SD_HIP_CHECK(hipGetLastError());
    }
}

}  // namespace sd
