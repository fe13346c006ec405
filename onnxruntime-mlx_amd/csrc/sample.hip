// Sampling of one token per row of logits: temperature, top-k, top-p, min-p and one given
// uniform number per row.
//
// w_i = exp((x_i - max) / T). In the order of falling logits, ties by rising index, the kept
// entries are the first k (top-k), of those the shortest prefix that holds p of their weight
// (top-p), of those the entries with w >= min_p (min-p; max w is 1). The token is the first,
// in index order, at which the kept weight exceeds u times all of it. Borders decide, so
// weights are computed in 64 bits (2e-13 relative) and summed as integers in units of 2^-44:
// a sum is then the same in whatever order its parts arrive.
//
// Four launches, the first three with several workgroups a row where rows are few:
//   top_kernel   the largest logit of each slice of a row;
//   hist_kernel  top-k: a histogram of the largest of every eight logits, over keys relative
//                to the row's largest: k of those are above a border, so at least k logits
//                are, and few more. Top-p without top-k: histograms of all logits' weights
//                and counts. Neither, nor min-p: the weight of every 512 logits;
//   list_kernel  the entries above the border that the histogram gives go to a list (8192 at
//                most; of a wider nucleus the entries of the border's bin);
//   pick_kernel  one workgroup a row: the exact borders by radix selection over ordered
//                32-bit keys (11 + 11 + 10 bits) on the list, then the token by the kept
//                weight of every 512 indices and, in the 512 that pass u, of every one.
// A row whose border lies too low for the list has its selection over all of the row.
#include <algorithm>
#include <cmath>

#include "common.h"

namespace ortmi {
namespace sample {

constexpr int kThreads = 1024, kWaves = 16, kBins = 2048, kVec = 8;
constexpr int kBlock = 512, kBlocks = 512;  // indices summed together; 262144 columns
constexpr int kList = 8192, kSlices = 32;
constexpr int kBinShift = 16;  // of keys: 128 bins an octave, 16 octaves below the largest
constexpr double kUnit = 17592186044416.0;  // 2^44
constexpr uint32_t kNoKey = 0;              // -inf and NaN: never taken

struct Entry {
    uint32_t key, index;
};

// What the launches leave for each other, one for each row.
struct Record {
    uint32_t slice_top[kSlices];  // keys
    unsigned long long mass[kBins];
    uint32_t count[kBins];
    unsigned long long rest;      // weight below the bins
    unsigned long long block[kBlocks];
    unsigned long long mass_above, all;
    uint32_t listed;              // kOver: the list does not have what the row needs
    uint32_t bin_only;            // the list holds the border's bin, mass_above lies above it
    Entry list[kList];
};
constexpr uint32_t kOver = 0xFFFFFFFFu;

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

// 2^z for z <= 0, within 2e-13 of it: the power series of exp to the tenth term on half a unit
// around the next integer.
__device__ __forceinline__ double exp2_64(double z) {
    const double n = rint(z), t = (z - n) * 0.69314718055994530942;
    double r = 1.0 / 3628800.0;
    r = fma(r, t, 1.0 / 362880.0);
    r = fma(r, t, 1.0 / 40320.0);
    r = fma(r, t, 1.0 / 5040.0);
    r = fma(r, t, 1.0 / 720.0);
    r = fma(r, t, 1.0 / 120.0);
    r = fma(r, t, 1.0 / 24.0);
    r = fma(r, t, 1.0 / 6.0);
    r = fma(r, t, 0.5);
    r = fma(r, t, 1.0);
    r = fma(r, t, 1.0);
    return ldexp(r, (int)n);
}

struct Weight {
    double top, c;  // the row's maximum, log2(e) / T
    // The largest weighs 1 (also an infinity, beside which all else weighs 0).
    __device__ __forceinline__ double of(float x) const {
        const double z = ((double)x - top) * c;
        return (double)x == top ? 1.0 : (z > -1000.0 ? exp2_64(z) : 0.0);
    }
    __device__ static __forceinline__ uint64_t units_of(double w) {  // at most 2^44: exact in 2^52
        const double v = w * kUnit + 4503599627370496.0;
        return __builtin_bit_cast(uint64_t, v) & 0xFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ uint64_t units(float x) const { return units_of(of(x)); }
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
    __device__ __forceinline__ Weight weight(uint32_t top_key) const {
        return Weight{(double)value_of(top_key), 1.4426950408889634074 / (double)temperature};
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
#pragma unroll 2
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
    for (int i = blockIdx.x * kThreads + threadIdx.x; i < kBins; i += gridDim.x * kThreads) {
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

template <typename T>
__global__ __launch_bounds__(kThreads) void hist_kernel(Params p) {
    __shared__ uint64_t mass[kBins];
    __shared__ uint32_t count[kBins];
    __shared__ uint64_t wave_rest[kWaves];
    const Settings o(p, blockIdx.y);
    Record& rec = p.records[blockIdx.y];
    const uint32_t top_key = row_top(p, rec);
    const bool by_count = o.by_count(), by_mass = o.by_mass();
    if (top_key == kNoKey || o.greedy() || !(by_count || by_mass || o.all())) return;
    const Row<T> row(p, blockIdx.y);
    const Weight w = o.weight(top_key);
    if (!by_count && !by_mass) {
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
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        mass[i] = 0;
        count[i] = 0;
    }
    __syncthreads();
    uint64_t rest = 0;
    if (by_count) {
        each_block(p, row, [&](int, int, const uint32_t (&v)[Row<T>::kWords]) {
            float x = -INFINITY;
#pragma unroll
            for (int e = 0; e < kVec; ++e) x = fmaxf(x, Row<T>::value(v, e));
            const uint32_t d = (top_key - key_of(x)) >> kBinShift;
            if (d < kBins) atomicAdd(&count[d], 1u);
        });
    } else {
        each_block(p, row, [&](int, int, const uint32_t (&v)[Row<T>::kWords]) {
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                const float x = Row<T>::value(v, e);
                const uint32_t k = key_of(x), d = (top_key - k) >> kBinShift;
                const uint64_t m = k == kNoKey ? 0 : w.units(x);
                rest += d < kBins ? 0 : m;
                if (d < kBins) {
                    atomicAdd(&count[d], 1u);
                    atomicAdd(reinterpret_cast<unsigned long long*>(&mass[d]), (unsigned long long)m);
                }
            }
        });
        rest = wave_sum_u64(rest);
        if ((threadIdx.x & 63) == 0) wave_rest[threadIdx.x >> 6] = rest;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads)
        if (count[i]) {
            atomicAdd(&rec.count[i], count[i]);
            if (by_mass) atomicAdd(&rec.mass[i], (unsigned long long)mass[i]);
        }
    if (by_mass && threadIdx.x == 0) {
        rest = 0;
        for (int i = 0; i < kWaves; ++i) rest += wave_rest[i];
        if (rest) atomicAdd(&rec.rest, (unsigned long long)rest);
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void list_kernel(Params p) {
    __shared__ Shared sh;
    const Settings o(p, blockIdx.y);
    Record& rec = p.records[blockIdx.y];
    const uint32_t top_key = row_top(p, rec);
    if (top_key == kNoKey || (o.all() && !o.greedy())) return;
    const int tid = threadIdx.x;
    uint32_t low = top_key, high = 0xFFFFFFFFu, bin_only = 0;  // keys low .. high are listed
    bool over = false;
    uint64_t all = 0, mass_above = 0;
    if (!o.greedy() && (o.by_count() || o.by_mass())) {
        const bool by_mass = o.by_mass();
        const uint32_t c0 = rec.count[2 * tid], c1 = rec.count[2 * tid + 1];
        const uint64_t m0 = by_mass ? rec.mass[2 * tid] : 0, m1 = by_mass ? rec.mass[2 * tid + 1] : 0;
        uint32_t c = c0 + c1, call;
        uint64_t m = m0 + m1, mall;
        if (tid == 0) sh.bin = kOver;
        block_scan(sh, c, m, call, mall);
        all = mall + rec.rest;
        // The bin in which the k-th lies, or the last entry of the prefix.
        const double target = (double)o.top_p * (double)all;
        auto reached = [&](uint32_t cc, uint64_t mm) {
            return by_mass ? cc > 0 && (double)mm >= target : cc >= (uint32_t)o.top_k;
        };
        if (!reached(c, m) && reached(c + c0 + c1, m + m0 + m1)) {
            const bool second = !reached(c + c0, m + m0);
            sh.bin = 2 * tid + (second ? 1 : 0);
            sh.mass_above = second ? m + m0 : m;
            sh.above = c + c0 + (second ? c1 : 0);
        }
        __syncthreads();
        const uint32_t bin = sh.bin;
        over = bin == kOver;
        mass_above = sh.mass_above;
        const uint64_t down = ((uint64_t)bin + 1) << kBinShift;
        low = top_key >= down ? top_key - (uint32_t)down + 1 : kNoKey + 1;
        if (by_mass && !over && sh.above > kList) {
            bin_only = 1;
            high = top_key - (bin << kBinShift);
        }
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
        rec.bin_only = bin_only;
        if (over) rec.listed = kOver;
    }
    if (over) return;
    const Row<T> row(p, blockIdx.y);
    each_block(p, row, [&](int, int i0, const uint32_t (&v)[Row<T>::kWords]) {
        uint32_t k[kVec], n = 0;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            k[e] = key_of(Row<T>::value(v, e));
            n += k[e] >= low && k[e] <= high ? 1u : 0u;
        }
        if (__any(n > 0)) {
            if (n > 0) {
                uint32_t at = atomicAdd(&rec.listed, n);
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    if (k[e] >= low && k[e] <= high) {
                        if (at < kList) rec.list[at] = Entry{k[e], (uint32_t)(i0 + e)};
                        ++at;
                    }
            }
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

// The token over `acc`; the kept weight is returned, the index left in sh.index.
template <typename A>
__device__ __forceinline__ uint64_t draw(const A& acc, const Settings& o, const Weight& w,
                                         Shared& sh, const Kept& kept) {
    const bool floor = o.min_p > 0.f;
    const double min_p = (double)o.min_p;
    return locate(acc, sh, (double)o.u, 0.0, [&](uint32_t k, int i) -> uint64_t {
        const bool in = (k > kept.key) | ((k == kept.key) & (i <= kept.last));
        if (!in) return 0;
        const double v = w.of(value_of(k));  // (min_p keeps the largest: its weight is 1)
        return floor & !(v >= min_p) ? 0 : Weight::units_of(v);
    });
}

template <typename T>
__global__ __launch_bounds__(kThreads) void pick_kernel(Params p) {
    __shared__ Shared sh;
    __shared__ Entry entries[kList];
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
    const bool greedy = o.greedy();
    const Weight w = o.weight(top_key);
    const bool listed = (greedy || !o.all()) && rec.listed <= kList;
    List list{entries, listed ? (int)rec.listed : 0};
    for (int i = tid; i < list.n; i += kThreads) entries[i] = rec.list[i];
    uint64_t total = 0;
    if (greedy) {
        auto first = [&](uint32_t k, int) -> uint64_t { return k == top_key ? 1 : 0; };
        if (listed) locate(list, sh, -1.0, 0.0, first);
        else locate(row, sh, -1.0, 0.0, first);
    } else if (o.all()) {
        // The blocks' weights are there.
        __syncthreads();
        if (tid < kBlocks) {
            sh.block[tid] = rec.block[tid];
            sh.inside[tid] = 0;
        }
        __syncthreads();
        double want = 0.0;
        total = find_part(sh, sh.block, (double)o.u, 0, 0, true, want);
        const uint32_t b = sh.hit;
        const uint64_t before = sh.before;
        row.fill_block(b, sh.inside, [&](uint32_t k, int) -> uint64_t {
            return k == kNoKey ? 0 : w.units(value_of(k));
        });
        __syncthreads();
        find_part(sh, sh.inside, 0.0, before, total, false, want);
        if (tid == 0) sh.index = (int64_t)b * kBlock + sh.hit;
    } else if (listed && !rec.bin_only) {
        total = draw(list, o, w, sh, borders(list, o, w, sh, rec.all, 0, row.cols));
    } else if (listed) {
        total = draw(row, o, w, sh, borders(list, o, w, sh, rec.all, rec.mass_above, row.cols));
    } else {
        total = draw(row, o, w, sh, borders(row, o, w, sh, 0, 0, row.cols));
    }
    if (tid == 0) {
        const int64_t i = sh.index;
        p.ids[p.row0 + r] = i;
        if (p.logprobs)
            p.logprobs[p.row0 + r] =
                greedy ? 0.f : (float)log(w.of(to_f32(row.x[i])) * kUnit / (double)total);
    }
}

// Rows at a time: what bounds the workspace (95 KB a row).
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
        // Slices of a row, whole rounds of a workgroup's 16 waves: one workgroup a CU in all.
        const int64_t rounds = (p.blocks + sample::kWaves - 1) / sample::kWaves;
        const int64_t want = std::max<int64_t>(1, std::min<int64_t>(device_cu_count() / n, rounds));
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
