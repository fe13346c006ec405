// Sampling of one token per row of logits: temperature, top-k, top-p, min-p and one given
// uniform number per row.
//
// w_i = exp((x_i - max) / T). In the order of falling logits, ties by rising index, the kept
// entries are the first k (top-k), of those the shortest prefix that holds p of their weight
// (top-p), of those the entries with w >= min_p (min-p; max w is 1). The token is the first,
// in index order, at which the kept weight exceeds u times all of it. Borders decide, so
// weights are computed in 64 bits (2e-12 relative) and summed as integers in units of 2^-44:
// a sum is then the same in whatever order its parts arrive.
//
// Four launches, the first three with several workgroups a row where rows are few:
//   top_kernel   the largest logit of each slice of a row;
//   hist_kernel  top-k: a histogram of the largest of every eight logits, over bins of 2^-7
//                octave: k of those are above a border, so at least k logits are, and few
//                more. Top-p without top-k: histograms of all logits' weights and counts (of
//                16-bit logits counts alone: a bin's weight is that of its few values times
//                their counts, so that no logit needs an exponential of its own). Neither, nor
//                min-p: the weight of every 512 logits;
//   list_kernel  top-k and min-p: the entries above the border go to a list, 8192 at most.
//                Top-p without top-k: those of the border's bin alone, and what lies above it
//                as weight by 512 indices;
//   pick_kernel  one workgroup a row: the exact borders on the list (by comparing each of up
//                to 256 entries with each, else by radix selection over ordered 32-bit keys),
//                then the token by the kept weight of every 512 indices and, in the 512 that
//                pass u, of every one.
// A row whose border lies too low for the list has its selection over all of the row.
//
// Measured, each launch in turn: 1 x 151936 fp16, top-k and top-p, 2.7 + 4.4 + 8.4 + 8.5 us, all
// latency; 32 x 128256 fp32, top-p alone, 5 + 19 + 16 + 17 (the 64-bit weights of all logits bind
// the second: 16.4 MB at 0.9 TB/s); 256 x 151936 bf16 with settings of every kind 16 + 43 + 43 +
// 20 (the first reads its 78 MB at 5 TB/s, the next two are vector instructions a logit).
#include <algorithm>
#include <cmath>

#include "common.h"

namespace ortmi {
namespace sample {

constexpr int kThreads = 1024, kWaves = 16, kBins = 2048, kVec = 8;
constexpr int kSmall = 256;  // entries that are compared each with each
constexpr int kBlock = 512, kBlocks = 512;  // indices summed together; 262144 columns
constexpr int kList = 8192, kSlices = 32;
constexpr int kHist = 4096;  // bins of a row's histogram
constexpr double kUnit = 17592186044416.0;  // 2^44
constexpr uint32_t kNoKey = 0;              // -inf and NaN: never taken
constexpr uint32_t kOver = 0xFFFFFFFFu;

struct Entry {
    uint32_t key, index;
};

// What the launches leave for each other, one for each row.
struct Record {
    uint32_t slice_top[kSlices];  // keys
    unsigned long long mass[kHist];
    uint32_t count[kHist];
    unsigned long long rest;      // weight below the bins
    unsigned long long block[kBlocks];
    unsigned long long mass_above, all;
    uint32_t listed;              // kOver: the list does not have what the row needs
    uint32_t high;                // bin only: the largest key of the border's bin
    Entry list[kList];
};
struct Params {
    const void* x;
    const float* uniform;
    const float *temperature, *top_p, *min_p;  // per row, or null: the values below
    const int32_t* top_k;
    float temperature_value, top_p_value, min_p_value;
    int32_t top_k_value;
    int64_t* ids;
    float* logprobs;
    int64_t cols, row0;
    Record* records;
    int blocks;        // of 512 indices in a row
    int slices, per;   // `per` blocks a slice
};

// Order-preserving key; equal numbers (0 and -0 among them) have equal keys. NaN and -inf: 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return kNoKey;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// Weights by 2^z = 2^n 2^(i/32) 2^r: the middle from a table in LDS, |r| <= 1/64 by the power
// series of exp to the fourth term (1.2e-12 relative).
constexpr int kTable = 32;

// The table, before a barrier: exp's power series to the term of 2e-16 on [0, 1) by halves.
__device__ __forceinline__ void fill_table(double* table) {
    if (threadIdx.x < kTable) {
        const double t = (double)threadIdx.x * (0.69314718055994530942 / (2 * kTable));
        double r = 1.0;
#pragma unroll
        for (int i = 12; i >= 1; --i) r = fma(r, t * (1.0 / i), 1.0);
        table[threadIdx.x] = r * r;  // exp(t)^2
    }
}

struct Weight {
    double top, c;  // the row's maximum, log2(e) / T
    const double* table;
    // The largest weighs 1 (an infinity as the largest finite: beside it all else weighs 0).
    __device__ __forceinline__ double of(float x) const {
        const double z = fmax(((double)fminf(x, 3.402823466e38f) - top) * c, -1000.0);
        const double kd = fma(z, (double)kTable, 6755399441055744.0);  // 1.5 2^52: an integer's bits
        const int k = (int)(uint32_t)__builtin_bit_cast(uint64_t, kd);
        const double r = fma(kd - 6755399441055744.0, -1.0 / kTable, z);
        double e = fma(r, 0.0096181291076284772, 0.055504108664821580);  // ln2^4 / 24, ln2^3 / 6
        e = fma(r, e, 0.24022650695910071);
        e = fma(r, e, 0.69314718055994531);
        e = fma(r, e, 1.0);
        return ldexp(e * table[k & (kTable - 1)], k >> 5);
    }
    __device__ static __forceinline__ uint64_t units_of(double w) {  // at most 2^44: exact in 2^52
        const double v = w * kUnit + 4503599627370496.0;
        return __builtin_bit_cast(uint64_t, v) & 0xFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ uint64_t units(float x) const { return units_of(of(x)); }
};

// Bins of a row's histogram, from the largest logit down, 128 an octave. A largest that is
// positive: 2048 bins (16 octaves) of positive logits, one of all between, 2047 of negative
// ones from 8 octaves below the largest's magnitude (at least 2^-9) on. One that is not: one
// of magnitudes below 2^-16, or the largest's, 4095 of larger ones.
struct Bins {
    int top;      // the largest's magnitude, in units of 2^16 of its bits
    bool positive;
    __device__ __forceinline__ Bins(uint32_t top_key)
        : top((int)((__float_as_uint(value_of(top_key)) & 0x7FFFFFFFu) >> 16)),
          positive(top_key > 0x80000000u) {}
    __device__ __forceinline__ int low() const {
        return positive ? max(top - 1024, 0x3B00) : max(top, 0x3780);
    }
    // The bin of values that have no bin of their own.
    __device__ __forceinline__ uint32_t between() const { return positive ? 2048u : 0u; }
    // NaN, -inf and what lies below the bins: kOver.
    __device__ __forceinline__ uint32_t of(float x) const {
        const uint32_t u = __float_as_uint(x + 0.f);
        const int h = (int)((u & 0x7FFFFFFFu) >> 16), l = low(), base = (int)between();
        const int neg = h < l ? base : base + 1 + h - l;
        const int d = u >= 0x80000000u ? neg : (positive ? min(top - h, 2048) : 0);
        return ((x > -INFINITY) & (d < kHist)) ? (uint32_t)d : kOver;
    }
    // The keys of bin d.
    __device__ __forceinline__ void keys(int d, uint32_t& first, uint32_t& last) const {
        auto pos = [](int h) { return 0x80000000u | ((uint32_t)h << 16); };
        const int base = (int)between();
        if (d < base) {
            first = pos(max(top - d, 0));
            last = first + 0xFFFFu;
        } else if (d == base) {
            first = ~pos(low()) + 1;
            last = positive ? pos(max(top - 2047, 0)) - 1 : 0x80000000u;
        } else {
            last = ~pos(low() + d - base - 1);
            first = last - 0xFFFFu;
        }
    }
};

struct Shared {
    uint64_t mass[kBins];
    uint32_t count[kBins];
    uint64_t block[kBlocks], inside[kBlock];
    uint64_t wave_mass[kWaves];
    uint32_t wave_count[kWaves];
    // What one thread finds for all.
    uint32_t bin, above, in_bin, hit, listed;
    uint64_t mass_above, mass_in, before;
    int64_t index;
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int o) {
    const uint32_t lo = __shfl_up((uint32_t)v, o, 64), hi = __shfl_up((uint32_t)(v >> 32), o, 64);
    return ((uint64_t)hi << 32) | lo;
}

// Sums over the threads before this one (exclusive), and over all.
__device__ __forceinline__ void block_scan(Shared& sh, uint32_t& c, uint64_t& m, uint32_t& call,
                                           uint64_t& mall) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t ci = c;
    uint64_t mi = m;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t cv = __shfl_up(ci, o, 64);
        const uint64_t mv = shfl_up64(mi, o);
        if (lane >= o) {
            ci += cv;
            mi += mv;
        }
    }
    __syncthreads();
    if (lane == 63) {
        sh.wave_count[wave] = ci;
        sh.wave_mass[wave] = mi;
    }
    __syncthreads();
    uint32_t cb = 0;
    uint64_t mb = 0;
    call = 0;
    mall = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w == wave) {
            cb = call;
            mb = mall;
        }
        call += sh.wave_count[w];
        mall += sh.wave_mass[w];
    }
    c = cb + ci - c;
    m = mb + mi - m;
}

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const uint32_t lo = __shfl_xor((uint32_t)v, o, 64), hi = __shfl_xor((uint32_t)(v >> 32), o, 64);
        v += ((uint64_t)hi << 32) | lo;
    }
    return v;
}

// Sum over the workgroup, in every thread.
__device__ __forceinline__ uint64_t block_sum(Shared& sh, uint64_t v) {
    v = wave_sum_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave_mass[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t r = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) r += sh.wave_mass[w];
    return r;
}


typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));  // rows begin anywhere

// The row's logits, 512 a wave and step, eight a lane; -inf behind its end.
template <typename T>
struct Row {
    const T* x;
    int cols;
    __device__ __forceinline__ Row(const Params& p, int64_t row)
        : x(static_cast<const T*>(p.x) + (p.row0 + row) * p.cols), cols((int)p.cols) {}
    static constexpr int kWords = sizeof(T) == 2 ? 4 : 8;
    __device__ __forceinline__ void bits(int i0, uint32_t (&w)[kWords]) const {
        if (i0 + kVec <= cols) {
#pragma unroll
            for (int v = 0; v < kWords / 4; ++v) {
                const u32x4_any q = *reinterpret_cast<const u32x4_any*>(x + i0 + v * kVec / (kWords / 4));
#pragma unroll
                for (int i = 0; i < 4; ++i) w[4 * v + i] = q[i];
            }
        } else if constexpr (sizeof(T) == 2) {
            const uint32_t none = std::is_same<T, half_t>::value ? 0xFC00u : 0xFF80u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a = i0 + 2 * i < cols ? __builtin_bit_cast(uint16_t, x[i0 + 2 * i]) : none;
                const uint32_t b = i0 + 2 * i + 1 < cols ? __builtin_bit_cast(uint16_t, x[i0 + 2 * i + 1]) : none;
                w[i] = a | (b << 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = i0 + i < cols ? __float_as_uint(x[i0 + i]) : 0xFF800000u;
        }
    }
    __device__ static __forceinline__ float value(const uint32_t (&w)[kWords], int e) {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
        else return to_f32(__builtin_bit_cast(T, (uint16_t)(w[e / 2] >> (16 * (e & 1)))));
    }
    __device__ __forceinline__ uint32_t key_at(int64_t i) const { return key_of(to_f32(x[i])); }

    // f(key, index) for the elements of this thread.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        for (int b = threadIdx.x >> 6; b * kBlock < cols; b += kWaves) {
            const int i0 = b * kBlock + (int)(threadIdx.x & 63) * kVec;
            uint32_t w[kWords];
            bits(i0, w);
#pragma unroll
            for (int e = 0; e < kVec; ++e) f(key_of(value(w, e)), i0 + e);
        }
    }
    // Sums of part(key, index) by 512 indices, into zeroed words; of one of the 512 by index.
    template <typename F>
    __device__ __forceinline__ void sum_blocks(uint64_t* block, F part) const {
        for (int b = threadIdx.x >> 6; b * kBlock < cols; b += kWaves) {
            const int i0 = b * kBlock + (int)(threadIdx.x & 63) * kVec;
            uint32_t w[kWords];
            bits(i0, w);
            uint64_t m = 0;
#pragma unroll
            for (int e = 0; e < kVec; ++e) m += part(key_of(value(w, e)), i0 + e);
            m = wave_sum_u64(m);
            if ((threadIdx.x & 63) == 0) block[b] = m;
        }
    }
    template <typename F>
    __device__ __forceinline__ void fill_block(uint32_t b, uint64_t* inside, F part) const {
        const int i = (int)(b * kBlock + threadIdx.x);
        if (threadIdx.x < kBlock && i < cols) inside[threadIdx.x] = part(key_of(to_f32(x[i])), i);
    }
};

// The listed entries, in no order.
struct List {
    const Entry* e;
    int n;
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        for (int i = threadIdx.x; i < n; i += kThreads) f(e[i].key, (int)e[i].index);
    }
    template <typename F>
    __device__ __forceinline__ void sum_blocks(uint64_t* block, F part) const {
        each([&](uint32_t k, int i) {
            const uint64_t m = part(k, i);
            if (m) atomicAdd(reinterpret_cast<unsigned long long*>(block + i / kBlock), (unsigned long long)m);
        });
    }
    template <typename F>
    __device__ __forceinline__ void fill_block(uint32_t b, uint64_t* inside, F part) const {
        each([&](uint32_t k, int i) {
            if ((uint32_t)i / kBlock == b) inside[i % kBlock] = part(k, i);
        });
    }
};

// Radix selection from the largest key down. By count: the key at which `need` keys are
// reached. By weight (MASS): the key at which `mass_above` and the weight of the keys >=
// floor_key reach `target` units. Gives the key, and of the keys above it the number and the
// weight; of the equal ones sh.in_bin and sh.mass_in. Nothing found (no keys): key 0.
template <bool MASS, typename A>
__device__ __forceinline__ uint32_t select(const A& acc, const Weight& w, Shared& sh,
                                           uint32_t need, double target, uint32_t floor_key,
                                           uint32_t& above, uint64_t& mass_above) {
    uint32_t prefix = 0;
    above = 0;
    for (int level = 0; level < 3; ++level) {
        const int shift = level == 0 ? 21 : (level == 1 ? 10 : 0), bits = level == 2 ? 10 : 11;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) {
            sh.count[i] = 0;
            sh.mass[i] = 0;
        }
        if (threadIdx.x == 0) {
            sh.bin = sh.above = sh.in_bin = 0;
            sh.mass_above = sh.mass_in = 0;
        }
        __syncthreads();
        acc.each([&](uint32_t k, int) {
            const bool in = k > kNoKey && k >= floor_key &&
                            (level == 0 || k >> (shift + bits) == prefix);
            if (in) {
                const uint32_t bin = (k >> shift) & ((1u << bits) - 1);
                atomicAdd(&sh.count[bin], 1u);
                if constexpr (MASS)
                    atomicAdd(reinterpret_cast<unsigned long long*>(&sh.mass[bin]),
                              (unsigned long long)w.units(value_of(k)));
            }
        });
        __syncthreads();
        // Bins from the top, two a thread.
        const int b0 = kBins - 1 - 2 * threadIdx.x, b1 = b0 - 1;
        const uint32_t c0 = sh.count[b0], c1 = sh.count[b1];
        const uint64_t m0 = sh.mass[b0], m1 = sh.mass[b1];
        uint32_t c = c0 + c1, call;
        uint64_t m = m0 + m1, mall;
        block_scan(sh, c, m, call, mall);
        auto reached = [&](uint32_t cc, uint64_t mm) {
            return MASS ? (double)(mass_above + mm) >= target : above + cc >= need;
        };
        // The bin that reaches it, or the last one that holds anything (rounding of target).
        const bool before0 = c > 0 && reached(c, m), before1 = c + c0 > 0 && reached(c + c0, m + m0);
        const bool last0 = c + c0 == call, last1 = c + c0 + c1 == call;
        if (c0 && !before0 && (reached(c + c0, m + m0) || last0)) {
            sh.bin = b0;
            sh.above = c;
            sh.mass_above = m;
            sh.in_bin = c0;
            sh.mass_in = m0;
        } else if (c1 && !before1 && (reached(c + c0 + c1, m + m0 + m1) || last1)) {
            sh.bin = b1;
            sh.above = c + c0;
            sh.mass_above = m + m0;
            sh.in_bin = c1;
            sh.mass_in = m1;
        }
        __syncthreads();
        prefix = (prefix << bits) | sh.bin;
        above += sh.above;
        mass_above += sh.mass_above;
    }
    __syncthreads();
    return prefix;
}

// Whether `own` behind `cum` is the place that `want` falls on; the last part where rounding
// leaves it behind all of them.
__device__ __forceinline__ bool falls_on(uint64_t cum, uint64_t own, double want, uint64_t total) {
    return own && !((double)cum > want) && ((double)(cum + own) > want || cum + own == total);
}

// The thread t < 512 on whose part[t] `want` falls, as sh.hit, the parts before it as
// sh.before; want is u times the whole for u >= 0, else `rank`. Returns the whole.
__device__ __forceinline__ uint64_t find_part(Shared& sh, const uint64_t* part, double u,
                                              uint64_t before, uint64_t whole, bool top_level,
                                              double& want) {
    const uint64_t own = threadIdx.x < kBlocks ? part[threadIdx.x] : 0;
    uint32_t c = 0, call;
    uint64_t m = own, mall;
    if (threadIdx.x == 0) sh.hit = kOver;
    block_scan(sh, c, m, call, mall);
    if (top_level) {
        whole = mall;
        if (u >= 0.0) want = u * (double)whole;
    }
    if (falls_on(before + m, own, want, whole)) {
        sh.hit = threadIdx.x;
        sh.before = before + m;
    }
    __syncthreads();
    return whole;
}

// The index, in index order, at which the cumulative part(key, index) exceeds u times the
// whole (u < 0: exceeds `rank`), as sh.index (-1: there is no part). Returns the whole.
template <typename A, typename F>
__device__ __forceinline__ uint64_t locate(const A& acc, Shared& sh, double u, double rank, F part) {
    __syncthreads();
    if (threadIdx.x < kBlocks) sh.block[threadIdx.x] = 0;
    if (threadIdx.x < kBlock) sh.inside[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.index = -1;
    __syncthreads();
    acc.sum_blocks(sh.block, part);
    __syncthreads();
    double want = rank;
    const uint64_t whole = find_part(sh, sh.block, u, 0, 0, true, want);
    const uint32_t b = sh.hit;
    const uint64_t before = sh.before;
    if (b != kOver) {
        acc.fill_block(b, sh.inside, part);
        __syncthreads();
        find_part(sh, sh.inside, u, before, whole, false, want);
        if (threadIdx.x == 0) sh.index = (int64_t)b * kBlock + sh.hit;
    }
    __syncthreads();
    return whole;
}

struct Settings {
    float temperature, top_p, min_p, u;
    int top_k;
    __device__ __forceinline__ Settings(const Params& p, int64_t row) {
        const int64_t r = p.row0 + row;
        temperature = p.temperature ? p.temperature[r] : p.temperature_value;
        top_p = p.top_p ? p.top_p[r] : p.top_p_value;
        min_p = p.min_p ? p.min_p[r] : p.min_p_value;
        top_k = p.top_k ? p.top_k[r] : p.top_k_value;
        if (top_k >= p.cols || top_k < 0) top_k = 0;
        const float v = p.uniform[r];
        u = v < 1.f ? (v > 0.f ? v : 0.f) : (v >= 1.f ? 1.f : 0.f);
    }
    // No spread to draw from (T <= 0, NaN), or none left: the first of the largest.
    __device__ __forceinline__ bool greedy() const {
        return !(temperature > 0.f) || min_p > 1.f || top_k == 1;
    }
    __device__ __forceinline__ bool by_count() const { return top_k > 0; }
    __device__ __forceinline__ bool by_mass() const { return top_k == 0 && top_p < 1.f; }
    __device__ __forceinline__ bool all() const { return top_k == 0 && !(top_p < 1.f) && !(min_p > 0.f); }
    __device__ __forceinline__ Weight weight(uint32_t top_key, const double* table) const {
        return Weight{(double)fminf(value_of(top_key), 3.402823466e38f),
                      1.4426950408889634074 / (double)temperature, table};
    }
};

__device__ __forceinline__ uint32_t row_top(const Params& p, const Record& rec) {
    uint32_t k = 0;
    for (int i = 0; i < p.slices; ++i) k = max(k, rec.slice_top[i]);
    return k;
}

// f(i0, words) for the blocks of this slice and wave.
template <typename T, typename F>
__device__ __forceinline__ void each_block(const Params& p, const Row<T>& row, F f) {
    const int end = min(((int)blockIdx.x + 1) * p.per, p.blocks);
    for (int b = (int)blockIdx.x * p.per + (int)(threadIdx.x >> 6); b < end; b += kWaves) {
        const int i0 = b * kBlock + (int)(threadIdx.x & 63) * kVec;
        uint32_t w[Row<T>::kWords];
        row.bits(i0, w);
        f(b, i0, w);
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void top_kernel(Params p) {
    __shared__ float wave_top[kWaves];
    const Row<T> row(p, blockIdx.y);
    Record& rec = p.records[blockIdx.y];
    for (int i = blockIdx.x * kThreads + threadIdx.x; i < kHist; i += gridDim.x * kThreads) {
        rec.mass[i] = 0;
        rec.count[i] = 0;
        if (i < kBlocks) rec.block[i] = 0;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        rec.rest = 0;
        rec.listed = 0;
    }
    float top = -INFINITY;
    each_block(p, row, [&](int, int, const uint32_t (&w)[Row<T>::kWords]) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) top = fmaxf(top, Row<T>::value(w, e));
    });
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) wave_top[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kWaves; ++i) top = fmaxf(top, wave_top[i]);
        rec.slice_top[blockIdx.x] = key_of(top);
    }
}

// Values that a bin of 2^16 of fp32's bits holds: bfloat16 1, fp16 8 (fp32: weights are summed).
template <typename T>
constexpr int kFine = std::is_same<T, half_t>::value ? 8 : 1;

template <typename T>
__global__ __launch_bounds__(kThreads) void hist_kernel(Params p) {
    constexpr bool kSums = sizeof(T) == 4;
    __shared__ uint64_t mass[kSums ? kHist : 1];
    __shared__ uint32_t count[kHist * kFine<T>];
    __shared__ double table[kTable];
    const Settings o(p, blockIdx.y);
    Record& rec = p.records[blockIdx.y];
    const uint32_t top_key = row_top(p, rec);
    const bool by_count = o.by_count(), by_mass = o.by_mass();
    if (top_key == kNoKey || o.greedy() || !(by_count || by_mass || o.all())) return;
    const Row<T> row(p, blockIdx.y);
    const Weight w = o.weight(top_key, table);
    const Bins bins(top_key);
    fill_table(table);
    if (!by_count && !by_mass) {
        __syncthreads();
        each_block(p, row, [&](int b, int, const uint32_t (&v)[Row<T>::kWords]) {
            uint64_t m = 0;
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                const float x = Row<T>::value(v, e);
                m += x > -INFINITY ? w.units(x) : 0;
            }
            m = wave_sum_u64(m);
            if ((threadIdx.x & 63) == 0) rec.block[b] = m;
        });
        return;
    }
    const int fine = by_mass ? kFine<T> : 1;
    for (int i = threadIdx.x; i < kHist * fine; i += kThreads) count[i] = 0;
    if (kSums && by_mass)
        for (int i = threadIdx.x; i < kHist; i += kThreads) mass[i] = 0;
    __syncthreads();
    if (by_count) {
        each_block(p, row, [&](int, int, const uint32_t (&v)[Row<T>::kWords]) {
            float x = -INFINITY;
#pragma unroll
            for (int e = 0; e < kVec; ++e) x = fmaxf(x, Row<T>::value(v, e));
            const uint32_t d = bins.of(x);
            if (d != kOver) atomicAdd(&count[d], 1u);
        });
        __syncthreads();
        for (int i = threadIdx.x; i < kHist; i += kThreads)
            if (count[i]) atomicAdd(&rec.count[i], count[i]);
        return;
    }
    uint64_t rest = 0;
    each_block(p, row, [&](int, int, const uint32_t (&v)[Row<T>::kWords]) {
        uint32_t out = 0;  // elements without a bin
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const float x = Row<T>::value(v, e);
            const uint32_t d = bins.of(x);
            // 16-bit values without a bin of their own share one: their weights are summed.
            const bool sums = kSums || d == bins.between();
            if (d != kOver) {
                if (kFine<T> == 1 || sums) atomicAdd(&count[d * kFine<T>], 1u);
                else atomicAdd(&count[d * kFine<T> + ((__float_as_uint(x) >> 13) & 7u)], 1u);
                if constexpr (kSums)
                    atomicAdd(reinterpret_cast<unsigned long long*>(&mass[d]), (unsigned long long)w.units(x));
            }
            out |= (!kSums && d != kOver && sums) || (d == kOver && x > -INFINITY) ? 1u << e : 0u;
        }
        while (__any(out != 0)) {  // few: one a lane and turn
            if (out) {
                const int e = __builtin_ctz(out);
                out &= out - 1;
                float x = 0.f;
#pragma unroll
                for (int j = 0; j < kVec; ++j) x = j == e ? Row<T>::value(v, j) : x;
                const uint32_t d = bins.of(x);
                const uint64_t m = w.units(x);
                if (d == kOver) rest += m;
                else atomicAdd(&rec.mass[bins.between()], (unsigned long long)m);
            }
        }
    });
    rest = wave_sum_u64(rest);
    if ((threadIdx.x & 63) == 0 && rest) atomicAdd(&rec.rest, (unsigned long long)rest);
    __syncthreads();
    for (int d = threadIdx.x; d < kHist; d += kThreads) {
        uint32_t n = 0;
        uint64_t m = 0;
        if constexpr (kSums) {
            n = count[d];
            m = mass[d];
        } else if (d == (int)bins.between()) {
            n = count[d * kFine<T>];
        } else {
            // The bin's values, from bits whose upper half is the same.
            uint32_t first, last;
            bins.keys(d, first, last);
            const uint32_t bits = __float_as_uint(value_of(first)) & 0xFFFF0000u;
#pragma unroll
            for (int j = 0; j < kFine<T>; ++j) {
                const uint32_t c = count[d * kFine<T> + j];
                if (c) m += c * w.units(__uint_as_float(bits | ((uint32_t)j << 13)));
                n += c;
            }
        }
        if (n) {
            atomicAdd(&rec.count[d], n);
            if (m) atomicAdd(&rec.mass[d], (unsigned long long)m);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void list_kernel(Params p) {
    __shared__ Shared sh;
    __shared__ double table[kTable];
    const Settings o(p, blockIdx.y);
    Record& rec = p.records[blockIdx.y];
    const uint32_t top_key = row_top(p, rec);
    if (top_key == kNoKey || (o.all() && !o.greedy())) return;
    fill_table(table);
    __syncthreads();
    const int tid = threadIdx.x;
    const bool by_mass = !o.greedy() && o.by_mass();
    uint32_t low = top_key, high = kOver;  // keys low .. high are listed
    bool over = false;
    uint64_t all = 0, mass_above = 0;
    if (!o.greedy() && (o.by_count() || by_mass)) {
        constexpr int kPer = kHist / kThreads;
        uint32_t n[kPer], c = 0, call;
        uint64_t v[kPer], m = 0, mall;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            n[i] = rec.count[kPer * tid + i];
            v[i] = by_mass ? rec.mass[kPer * tid + i] : 0;
            c += n[i];
            m += v[i];
        }
        if (tid == 0) sh.bin = kOver;
        block_scan(sh, c, m, call, mall);
        all = mall + rec.rest;
        // The bin in which the k-th lies, or the last entry of the prefix.
        const double target = (double)o.top_p * (double)all;
        auto reached = [&](uint32_t cc, uint64_t mm) {
            return by_mass ? cc > 0 && (double)mm >= target : cc >= (uint32_t)o.top_k;
        };
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (!reached(c, m) && reached(c + n[i], m + v[i])) {
                sh.bin = kPer * tid + i;
                sh.mass_above = m;
            }
            c += n[i];
            m += v[i];
        }
        __syncthreads();
        over = sh.bin == kOver;
        mass_above = sh.mass_above;
        uint32_t last = kOver;
        if (!over) Bins(top_key).keys((int)sh.bin, low, last);
        low = max(low, kNoKey + 1);
        if (by_mass) high = last;
    } else if (!o.greedy()) {
        // Above the border of min-p, a little lowered: the weights decide.
        const double t = (double)value_of(top_key) +
                         log((double)o.min_p) * (double)o.temperature * 1.000001;
        const float f = (float)t;
        low = max(key_of(f - fabsf(f) * 1e-6f - 1e-30f), kNoKey + 1);
        if (value_of(top_key) == INFINITY) low = top_key;
    }
    if (blockIdx.x == 0 && tid == 0) {
        rec.all = all;
        rec.mass_above = mass_above;
        rec.high = high;
        if (over) rec.listed = kOver;
    }
    if (over) return;
    const Row<T> row(p, blockIdx.y);
    const Weight w = o.weight(top_key, table);
    const double min_p = o.min_p > 0.f ? (double)o.min_p : 0.0;
    each_block(p, row, [&](int b, int i0, const uint32_t (&v)[Row<T>::kWords]) {
        uint32_t in = 0, above = 0;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const uint32_t k = key_of(Row<T>::value(v, e));
            in |= ((k >= low) & (k <= high)) ? 1u << e : 0u;
            above |= k > high ? 1u << e : 0u;
        }
        if (__any(in != 0)) {
            if (in) {
                uint32_t at = atomicAdd(&rec.listed, (uint32_t)__popc(in));
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    if (in >> e & 1u) {
                        if (at < kList)
                            rec.list[at] = Entry{key_of(Row<T>::value(v, e)), (uint32_t)(i0 + e)};
                        ++at;
                    }
            }
        }
        if (by_mass) {  // kept for sure, but for min-p: their weight
            uint64_t m = 0;
            while (__any(above != 0)) {
                if (above) {
                    const int e = __builtin_ctz(above);
                    above &= above - 1;
                    float x = 0.f;
#pragma unroll
                    for (int j = 0; j < kVec; ++j) x = j == e ? Row<T>::value(v, j) : x;
                    const double d = w.of(x);
                    m += d >= min_p ? Weight::units_of(d) : 0;
                }
            }
            m = wave_sum_u64(m);
            if ((tid & 63) == 0) rec.block[b] = m;
        }
    });
}

// The borders of the kept entries over `acc`, which has every entry that may be kept (and, for
// `bin`, those of the border's bin alone): keys above `key`, and of the equal ones those up to
// the index `last`. `all`: the weight that top-p refers to without top-k (0: that of acc).
struct Kept {
    uint32_t key;
    int last;
};
template <typename A>
__device__ __forceinline__ Kept borders(const A& acc, const Settings& o, const Weight& w,
                                        Shared& sh, uint64_t all, uint64_t mass_above, int cols) {
    uint32_t key = kNoKey + 1, above = 0, ties = kOver;  // ties: how many of the equal ones
    if (o.by_count()) {
        uint64_t none = 0;
        key = select<false>(acc, w, sh, (uint32_t)o.top_k, 0.0, 0u, above, none);
        const uint32_t equal = sh.in_bin;
        ties = (uint32_t)o.top_k - above < equal ? (uint32_t)o.top_k - above : kOver;
    }
    if (o.top_p < 1.f) {
        if (!all) {  // the weight of the kept entries
            uint32_t c = 0, call;
            uint64_t m = 0, mall;
            acc.each([&](uint32_t k, int) {
                m += k > key ? w.units(value_of(k)) : 0;
                c += k == key ? 1u : 0u;
            });
            block_scan(sh, c, m, call, mall);
            all = mall + (key > kNoKey + 1 ? w.units(value_of(key)) * min(call, ties) : 0);
        }
        const double target = (double)o.top_p * (double)all;
        const uint32_t kp = select<true>(acc, w, sh, 0u, target, key, above, mass_above);
        const uint32_t equal = kp == key ? min(sh.in_bin, ties) : sh.in_bin;
        key = kp;
        // The first t with mass_above + t each >= target, at least one.
        const double each = (double)w.units(value_of(key));
        const double t = each > 0.0 ? ceil((target - (double)mass_above) / each) : (double)equal;
        uint32_t n = t < 1.0 ? 1u : (t > (double)equal ? equal : (uint32_t)t);
        while (n > 1 && each > 0.0 && (double)mass_above + (n - 1) * each >= target) --n;
        while (n < equal && (double)mass_above + n * each < target) ++n;
        ties = n;
    }
    int last = cols;
    if (ties != kOver) {
        locate(acc, sh, -1.0, (double)(ties - 1), [&](uint32_t k, int) -> uint64_t { return k == key ? 1 : 0; });
        last = (int)sh.index;
    }
    return Kept{key, last};
}

// The weight that an entry adds: its own where it is kept.
struct Part {
    Weight w;
    Kept kept;
    double min_p;  // (the largest weighs 1: it passes)
    __device__ __forceinline__ uint64_t operator()(uint32_t k, int i) const {
        const bool in = (k > kept.key) | ((k == kept.key) & (i <= kept.last));
        if (!in) return 0;
        const double v = w.of(value_of(k));
        return v >= min_p ? Weight::units_of(v) : 0;
    }
};

// Top-p without top-k: what lies above the border's bin is summed by 512 indices already, the
// bin's entries are listed, and the row has the one block that is looked at in the end.
template <typename T>
struct Above {
    const Row<T>& row;
    const List& list;
    const Record& rec;
    template <typename F>
    __device__ __forceinline__ void sum_blocks(uint64_t* block, F part) const {
        if (threadIdx.x < kBlocks) block[threadIdx.x] = rec.block[threadIdx.x];
        __syncthreads();
        list.sum_blocks(block, part);
    }
    template <typename F>
    __device__ __forceinline__ void fill_block(uint32_t b, uint64_t* inside, F part) const {
        row.fill_block(b, inside, part);
    }
};

__device__ __forceinline__ uint64_t add_xor(uint64_t v, int x) {
    const uint32_t lo = __shfl_xor((uint32_t)v, x, 64), hi = __shfl_xor((uint32_t)(v >> 32), x, 64);
    return v + (((uint64_t)hi << 32) | lo);
}

// Lists of at most 256 entries, four threads an entry: its rank and the weight before it by
// comparison with every other. Leaves the kept entries' weights in sh.mass[entry] (0: not
// kept) and returns their sum. The weight before the first is mass_above; `all` as in borders.
__device__ __forceinline__ uint64_t keep_small(const List& list, const Settings& o, const Weight& w,
                                               Shared& sh, uint64_t all, uint64_t mass_above) {
    const int a = threadIdx.x >> 2, part = threadIdx.x & 3, n = list.n;
    const bool have = a < n;
    const Entry me = list.e[have ? a : 0];
    const double weight = have ? w.of(value_of(me.key)) : 0.0;
    const uint64_t units = Weight::units_of(weight);
    __syncthreads();
    if (part == 0) sh.mass[a] = units;
    __syncthreads();
    uint32_t rank = 0;
    uint64_t before = 0;
    for (int i = part; i < n; i += 4) {
        const Entry b = list.e[i];
        const bool first = (b.key > me.key) | ((b.key == me.key) & (b.index < me.index));
        rank += first ? 1u : 0u;
        before += first ? sh.mass[i] : 0;
    }
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
        rank += __shfl_xor(rank, x, 64);
        before = add_xor(before, x);
    }
    const bool own = have & (part == 0);  // one thread of an entry's four counts it
    const uint32_t k = o.top_k > 0 ? (uint32_t)o.top_k : kOver;
    if (!all) all = block_sum(sh, (own & (rank < k)) ? units : 0);
    before += mass_above;
    // Selects, no branches: the compiler has lost the zero of an `if (!keep) units = 0` here.
    const bool in_p = !(o.top_p < 1.f) | ((double)before < (double)o.top_p * (double)all);
    const bool in_m = !(o.min_p > 0.f) | (weight >= (double)o.min_p);
    const bool keep = own & (rank < k) & (((rank == 0) & (mass_above == 0)) | (in_p & in_m));
    const uint64_t kept = keep ? units : 0;
    const uint64_t total = block_sum(sh, kept);  // its barriers end the reading of sh.mass
    if (part == 0) sh.mass[a] = kept;
    __syncthreads();
    return total;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void pick_kernel(Params p) {
    __shared__ Shared sh;
    __shared__ Entry entries[kList];
    __shared__ double table[kTable];
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const Settings o(p, r);
    const Record& rec = p.records[r];
    const Row<T> row(p, r);
    const uint32_t top_key = row_top(p, rec);
    if (top_key == kNoKey) {  // nothing to take
        if (tid == 0) {
            p.ids[p.row0 + r] = -1;
            if (p.logprobs) p.logprobs[p.row0 + r] = -INFINITY;
        }
        return;
    }
    const bool greedy = o.greedy(), by_mass = !greedy && o.by_mass();
    const Weight w = o.weight(top_key, table);
    fill_table(table);
    const bool listed = (greedy || !o.all()) && rec.listed <= kList;
    const List list{entries, listed ? (int)rec.listed : 0};
    for (int i = tid; i < list.n; i += kThreads) entries[i] = rec.list[i];
    if (tid == 0) sh.index = -1;
    __syncthreads();
    const double min_p = o.min_p > 0.f ? (double)o.min_p : 0.0;
    uint64_t total = 0;
    if (greedy) {
        auto first = [&](uint32_t k, int) -> uint64_t { return k == top_key ? 1 : 0; };
        if (listed) locate(list, sh, -1.0, 0.0, first);
        else locate(row, sh, -1.0, 0.0, first);
    } else if (o.all()) {
        const List none{entries, 0};
        total = locate(Above<T>{row, none, rec}, sh, (double)o.u, 0.0,
                       Part{w, Kept{kNoKey + 1, row.cols}, 0.0});
    } else if (listed && list.n <= kSmall) {
        const uint64_t kept = keep_small(list, o, w, sh, rec.all, by_mass ? rec.mass_above : 0);
        if (!by_mass) {
            // Cumulative weights in index order, by comparison.
            total = kept;
            const int a = tid >> 2, part = tid & 3;
            const uint64_t own = sh.mass[a];
            const uint32_t index = entries[a < list.n ? a : 0].index;
            uint64_t cum = 0;
            for (int i = part; i < list.n; i += 4) cum += entries[i].index < index ? sh.mass[i] : 0;
            cum = add_xor(add_xor(cum, 1), 2);
            if (part == 0 && a < list.n && falls_on(cum, own, (double)o.u * (double)total, total))
                sh.index = index;
        } else {
            // The last kept of the bin, in order: the border for the one block that is read.
            __shared__ uint32_t low_key;
            __shared__ int last;
            if (tid == 0) {
                low_key = kOver;
                last = -1;
            }
            __syncthreads();
            const bool mine = tid < list.n && sh.mass[tid] != 0;
            const Entry e = entries[tid < list.n ? tid : 0];
            if (mine) atomicMin(&low_key, e.key);
            __syncthreads();
            if (mine && e.key == low_key) atomicMax(&last, (int)e.index);
            __syncthreads();
            const Kept border{low_key == kOver ? rec.high : low_key, low_key == kOver ? -1 : last};
            total = locate(Above<T>{row, list, rec}, sh, (double)o.u, 0.0, Part{w, border, min_p});
        }
    } else if (listed) {
        const Kept border = borders(list, o, w, sh, rec.all, by_mass ? rec.mass_above : 0, row.cols);
        const Part part{w, border, min_p};
        if (by_mass) total = locate(Above<T>{row, list, rec}, sh, (double)o.u, 0.0, part);
        else total = locate(list, sh, (double)o.u, 0.0, part);
    } else {
        const Kept border = borders(row, o, w, sh, 0, 0, row.cols);
        total = locate(row, sh, (double)o.u, 0.0, Part{w, border, min_p});
    }
    __syncthreads();
    if (tid == 0) {
        const int64_t i = sh.index;
        p.ids[p.row0 + r] = i;
        if (p.logprobs)
            p.logprobs[p.row0 + r] =
                greedy ? 0.f : (float)log(w.of(to_f32(row.x[i])) * kUnit / (double)total);
    }
}

// Rows at a time: what bounds the workspace (117 KB a row).
constexpr int64_t kRows = 1024;

}  // namespace sample
}  // namespace ortmi

using namespace ortmi;

extern "C" size_t ortmi_sample_rows_workspace_size(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return (size_t)std::min(rows, sample::kRows) * sizeof(sample::Record);
}

template <typename T>
static int sample_rows(sample::Params p, int64_t rows, hipStream_t st) {
    p.blocks = (int)((p.cols + sample::kBlock - 1) / sample::kBlock);
    for (int64_t r0 = 0; r0 < rows; r0 += sample::kRows) {
        const int64_t n = std::min(sample::kRows, rows - r0);
        // Slices of a row, whole rounds of a workgroup's 16 waves: two workgroups a CU, and four
        // a row, so that rows whose settings ask for more work do not hold up the others.
        const int64_t rounds = (p.blocks + sample::kWaves - 1) / sample::kWaves;
        const int64_t want = std::min<int64_t>(std::max<int64_t>(4, 2 * device_cu_count() / n), rounds);
        const int64_t each = (rounds + want - 1) / want;
        p.per = (int)each * sample::kWaves;
        p.slices = (int)((rounds + each - 1) / each);
        p.row0 = r0;
        const dim3 grid((unsigned)p.slices, (unsigned)n), block(sample::kThreads);
        hipLaunchKernelGGL(sample::top_kernel<T>, grid, block, 0, st, p);
        hipLaunchKernelGGL(sample::hist_kernel<T>, grid, block, 0, st, p);
        hipLaunchKernelGGL(sample::list_kernel<T>, grid, block, 0, st, p);
        hipLaunchKernelGGL(sample::pick_kernel<T>, dim3((unsigned)n), block, 0, st, p);
        if (int rc = check_launch("sample")) return rc;
    }
    return ORTMI_OK;
}

extern "C" int ortmi_sample_rows(const void* logits, const float* uniform, const float* temperature,
                                 const int32_t* top_k, const float* top_p, const float* min_p,
                                 float temperature_value, int32_t top_k_value, float top_p_value,
                                 float min_p_value, int64_t* ids, float* logprobs, int64_t rows,
                                 int64_t cols, int32_t dtype, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    ORTMI_REQUIRE(dtype == ORTMI_F32 || dtype == ORTMI_F16 || dtype == ORTMI_BF16,
                  "Sample: dtype must be fp32, fp16 or bf16");
    ORTMI_REQUIRE(rows >= 0 && rows < (1LL << 31), "Sample: bad row count");
    // 2^18 entries of weight 1 sum to 2^62 units.
    ORTMI_REQUIRE(cols > 0 && cols <= (1LL << 18), "Sample: 1 to 262144 columns");
    if (rows == 0) return ORTMI_OK;
    ORTMI_REQUIRE(logits && uniform && ids, "Sample: null tensor");
    if (!workspace || workspace_bytes < ortmi_sample_rows_workspace_size(rows, cols))
        return fail(ORTMI_E_WORKSPACE, "Sample: workspace too small");
    ORTMI_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
                  "Sample: workspace must be 16-byte aligned");
    sample::Params p{};
    p.x = logits;
    p.uniform = uniform;
    p.temperature = temperature;
    p.top_p = top_p;
    p.min_p = min_p;
    p.top_k = top_k;
    p.temperature_value = temperature_value;
    p.top_p_value = top_p_value;
    p.min_p_value = min_p_value;
    p.top_k_value = top_k_value;
    p.ids = ids;
    p.logprobs = logprobs;
    p.cols = cols;
    p.records = static_cast<sample::Record*>(workspace);
    hipStream_t st = as_stream(stream);
    if (dtype == ORTMI_F32) return sample_rows<float>(p, rows, st);
    if (dtype == ORTMI_F16) return sample_rows<half_t>(p, rows, st);
    return sample_rows<uint16_t>(p, rows, st);
}
