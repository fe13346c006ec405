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
// One workgroup of 16 waves has a row. The k-th largest logit, and the one at which the
// prefix of p ends, are found by radix selection over ordered 32-bit keys (11 + 11 + 10 bits)
// with histograms of counts and of weights in LDS.
#include <cmath>

#include "common.h"

namespace ortmi {
namespace sample {

constexpr int kThreads = 1024, kWaves = 16, kBins = 2048, kVec = 8;
constexpr double kUnit = 17592186044416.0;  // 2^44
constexpr uint32_t kNoKey = 0;              // -inf and NaN: never taken

struct Params {
    const void* x;
    const float* uniform;
    const float *temperature, *top_p, *min_p;  // per row, or null: the values below
    const int32_t* top_k;
    float temperature_value, top_p_value, min_p_value;
    int32_t top_k_value;
    int64_t* ids;
    float* logprobs;
    int64_t cols;
    int dtype;
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
    __device__ __forceinline__ uint64_t units(float x) const {  // at most 2^44: exact in 2^52
        const double v = of(x) * kUnit + 4503599627370496.0;
        return __builtin_bit_cast(uint64_t, v) & 0xFFFFFFFFFFFFFull;
    }
};

struct Shared {
    uint64_t mass[kBins];
    uint32_t count[kBins];
    uint64_t wave_mass[kWaves];
    uint32_t wave_count[kWaves];
    float wave_max[kWaves];
    // What one thread finds for all.
    uint32_t bin, above, in_bin;
    uint64_t mass_above, mass_in;
    int64_t index;
    double weight;
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

// A row's elements in index order, eight a thread and step.
template <typename T>
struct Row {
    const T* x;
    int64_t cols;
    int steps;
    __device__ __forceinline__ Row(const Params& p, int64_t row)
        : x(static_cast<const T*>(p.x) + row * p.cols), cols(p.cols),
          steps((int)((p.cols + kThreads * kVec - 1) / (kThreads * kVec))) {}
    __device__ __forceinline__ int64_t first(int j) const {
        return ((int64_t)j * kThreads + threadIdx.x) * kVec;
    }
    __device__ __forceinline__ void keys(int j, uint32_t (&k)[kVec]) const {
        const int64_t i0 = first(j);
#pragma unroll
        for (int e = 0; e < kVec; ++e) k[e] = i0 + e < cols ? key_of(to_f32(x[i0 + e])) : kNoKey;
    }
};

// Radix selection from the largest key down. By count: the key at which `need` keys are
// reached. By weight (MASS): the key at which the weight of the keys >= floor_key reaches
// `target` units. Gives the key, and of the keys above it the number and the weight; of the
// equal ones sh.in_bin and sh.mass_in.
template <bool MASS, typename R>
__device__ __forceinline__ uint32_t select(const R& row, const Weight& w, Shared& sh,
                                           uint32_t need, double target, uint32_t floor_key,
                                           uint32_t& above, uint64_t& mass_above) {
    uint32_t prefix = 0;
    above = 0;
    mass_above = 0;
    for (int level = 0; level < 3; ++level) {
        const int shift = level == 0 ? 21 : (level == 1 ? 10 : 0), bits = level == 2 ? 10 : 11;
        for (int i = threadIdx.x; i < kBins; i += kThreads) {
            sh.count[i] = 0;
            sh.mass[i] = 0;
        }
        __syncthreads();
        for (int j = 0; j < row.steps; ++j) {
            uint32_t k[kVec];
            row.keys(j, k);
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                const bool in = k[e] > kNoKey && k[e] >= floor_key &&
                                (level == 0 || k[e] >> (shift + bits) == prefix);
                if (in) {
                    const uint32_t bin = (k[e] >> shift) & ((1u << bits) - 1);
                    atomicAdd(&sh.count[bin], 1u);
                    if constexpr (MASS)
                        atomicAdd(reinterpret_cast<unsigned long long*>(&sh.mass[bin]),
                                  (unsigned long long)w.units(value_of(k[e])));
                }
            }
        }
        __syncthreads();
        // Bins from the top, two a thread.
        const int b0 = kBins - 1 - 2 * threadIdx.x, b1 = b0 - 1;
        const uint32_t c0 = sh.count[b0], c1 = sh.count[b1];
        const uint64_t m0 = sh.mass[b0], m1 = sh.mass[b1];
        uint32_t c = c0 + c1, call;
        uint64_t m = m0 + m1, mall;
        block_scan(sh, c, m, call, mall);
        if (threadIdx.x == 0) sh.bin = 0xFFFFFFFFu;
        __syncthreads();
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
        __syncthreads();
    }
    return prefix;
}

// The index of the `rank`-th (from 0) element for which `take` holds, in index order. Every
// thread's steps are counted a wave at a time; the segment that has it is gone through once.
template <typename R, typename F>
__device__ __forceinline__ int64_t index_of_rank(const R& row, Shared& sh, uint32_t rank, F take) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t before = 0;
    for (int j = 0; j < row.steps; ++j) {
        uint32_t k[kVec], n = 0;
        row.keys(j, k);
#pragma unroll
        for (int e = 0; e < kVec; ++e) n += take(k[e]) ? 1u : 0u;
        uint32_t incl = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t v = __shfl_up(incl, o, 64);
            if (lane >= o) incl += v;
        }
        __syncthreads();
        if (lane == 63) sh.wave_count[wave] = incl;
        __syncthreads();
        uint32_t mine = before, all = 0;
        for (int i = 0; i < kWaves; ++i) {
            if (i < wave) mine += sh.wave_count[i];
            all += sh.wave_count[i];
        }
        mine += incl - n;
        if (rank >= mine && rank < mine + n) {
            uint32_t at = mine;
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                if (take(k[e])) {
                    if (at == rank) sh.index = row.first(j) + e;
                    ++at;
                }
        }
        before += all;
        if (rank < before) break;
    }
    __syncthreads();
    const int64_t r = sh.index;
    __syncthreads();
    return r;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(Params p) {
    __shared__ Shared sh;
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Row<T> row(p, r);
    const float temperature = p.temperature ? p.temperature[r] : p.temperature_value;
    const float top_p = p.top_p ? p.top_p[r] : p.top_p_value;
    const float min_p = p.min_p ? p.min_p[r] : p.min_p_value;
    const int top_k = p.top_k ? p.top_k[r] : p.top_k_value;
    const float u = p.uniform[r];

    float top = -INFINITY;
    for (int j = 0; j < row.steps; ++j) {
        uint32_t k[kVec];
        row.keys(j, k);
#pragma unroll
        for (int e = 0; e < kVec; ++e) top = fmaxf(top, k[e] ? value_of(k[e]) : -INFINITY);
    }
    top = wave_max(top);
    if (lane == 0) sh.wave_max[wave] = top;
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) top = fmaxf(top, sh.wave_max[i]);
    if (!(top > -INFINITY)) {  // nothing to take
        if (threadIdx.x == 0) {
            p.ids[r] = -1;
            if (p.logprobs) p.logprobs[r] = -INFINITY;
        }
        return;
    }
    const uint32_t top_key = key_of(top);
    // No spread to draw from (T <= 0, NaN), or none left: the first of the largest.
    if (!(temperature > 0.f) || min_p > 1.f || top_k == 1) {
        const int64_t i = index_of_rank(row, sh, 0, [&](uint32_t k) { return k == top_key; });
        if (threadIdx.x == 0) {
            p.ids[r] = i;
            if (p.logprobs) p.logprobs[r] = 0.f;
        }
        return;
    }
    const Weight w{(double)top, 1.4426950408889634074 / (double)temperature};

    // The kept entries: keys above `key`, and of those equal to it the ones up to `last`.
    uint32_t key = kNoKey + 1, above = 0;
    uint64_t mass_above = 0;
    int64_t last = p.cols;
    uint32_t ties = 0xFFFFFFFFu;  // how many of the equal ones
    if (top_k > 0 && top_k < p.cols) {
        key = select<false>(row, w, sh, (uint32_t)top_k, 0.0, 0u, above, mass_above);
        const uint32_t equal = sh.in_bin;
        __syncthreads();
        if ((uint32_t)top_k - above < equal) ties = (uint32_t)top_k - above;
    }
    if (top_p < 1.f) {
        // The weight of the kept entries, then the key at which p of it is reached.
        uint32_t c = 0, call;
        uint64_t m = 0, mall;
        for (int j = 0; j < row.steps; ++j) {
            uint32_t k[kVec];
            row.keys(j, k);
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                if (k[e] > key) m += w.units(value_of(k[e]));
                else if (k[e] == key) ++c;
        }
        block_scan(sh, c, m, call, mall);
        const uint64_t unit = key > kNoKey ? w.units(value_of(key)) : 0;
        mall += unit * min(call, ties);
        const double target = (double)top_p * (double)mall;
        const uint32_t kp = select<true>(row, w, sh, 0u, target, key, above, mass_above);
        const uint32_t equal = kp == key ? min(sh.in_bin, ties) : sh.in_bin;
        __syncthreads();
        key = kp;
        // The first t with mass_above + t unit >= target, at least one.
        const double each = (double)w.units(value_of(key));
        uint32_t t = equal;
        if (each > 0.0) {
            const double q = ceil((target - (double)mass_above) / each);
            t = q < 1.0 ? 1u : (q > (double)equal ? equal : (uint32_t)q);
            while (t > 1 && (double)mass_above + (t - 1) * each >= target) --t;
            while (t < equal && (double)mass_above + t * each < target) ++t;
        }
        ties = t;
    }
    if (ties != 0xFFFFFFFFu)
        last = index_of_rank(row, sh, ties - 1, [&](uint32_t k) { return k == key; });

    // Kept weight by wave and step, in index order; then the segment that passes u of it.
    // (min_p keeps the largest: its weight is 1.)
    auto kept = [&](uint32_t k, int64_t i) -> uint64_t {
        if (k < key || k == kNoKey || (k == key && i > last)) return 0;
        const float x = value_of(k);
        if (min_p > 0.f && !(w.of(x) >= (double)min_p)) return 0;
        return w.units(x);
    };
    uint64_t total = 0;
    for (int pass = 0; pass < 2; ++pass) {
        const double want = pass ? (u < 1.f ? (u > 0.f ? (double)u : 0.0) : 1.0) * (double)total : 0.0;
        uint64_t before = 0;
        if (pass && threadIdx.x == 0) sh.index = -1;
        for (int j = 0; j < row.steps; ++j) {
            uint32_t k[kVec];
            row.keys(j, k);
            uint64_t m = 0;
#pragma unroll
            for (int e = 0; e < kVec; ++e) m += kept(k[e], row.first(j) + e);
            const uint64_t own = m;
            uint32_t c = 0, call;
            uint64_t mall;
            block_scan(sh, c, m, call, mall);
            if (pass) {
                // The first entry whose cumulative weight exceeds `want`; the last one of all
                // where rounding (or u = 1) leaves none.
                const uint64_t at = before + m;
                const bool here = own && !((double)at > want) &&
                                  ((double)(at + own) > want || at + own == total);
                if (here) {
                    uint64_t cum = at;
#pragma unroll
                    for (int e = 0; e < kVec; ++e) {
                        const uint64_t v = kept(k[e], row.first(j) + e);
                        if (v && !((double)cum > want) &&
                            ((double)(cum + v) > want || cum + v == total)) {
                            sh.index = row.first(j) + e;
                            sh.weight = w.of(value_of(k[e]));
                        }
                        cum += v;
                    }
                }
            }
            before += mall;
        }
        total = before;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        p.ids[r] = sh.index;
        if (p.logprobs) p.logprobs[r] = (float)log(sh.weight * kUnit / (double)total);
    }
}

}  // namespace sample
}  // namespace ortmi

using namespace ortmi;

extern "C" size_t ortmi_sample_rows_workspace_size(int64_t rows, int64_t cols) {
    (void)rows, (void)cols;
    return 0;
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
    (void)workspace, (void)workspace_bytes;
    const sample::Params p{logits, uniform, temperature, top_p, min_p, top_k, temperature_value,
                           top_p_value, min_p_value, top_k_value, ids, logprobs, cols, dtype};
    const dim3 grid((unsigned)rows), block(sample::kThreads);
    hipStream_t st = as_stream(stream);
    if (dtype == ORTMI_F32)
        hipLaunchKernelGGL(sample::sample_kernel<float>, grid, block, 0, st, p);
    else if (dtype == ORTMI_F16)
        hipLaunchKernelGGL(sample::sample_kernel<half_t>, grid, block, 0, st, p);
    else
        hipLaunchKernelGGL(sample::sample_kernel<uint16_t>, grid, block, 0, st, p);
    return check_launch("sample");
}
