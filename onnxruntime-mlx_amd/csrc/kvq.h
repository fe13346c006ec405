// Attention over quantised key-value caches: what its kernels share (kvq*.hip).
//
// A cache row (one key or value of one head) holds codes: int8, int4 (two per byte, the
// even channel in the low nibble, stored as code + 8) or fp8 e4m3. A code stands for
// code * scale, scale one fp32 number for the tensor or one per (kv head, channel). A new
// row is rotated (keys), divided by the scale and rounded to the nearest code, all in
// 64 bits: fp16, bf16 and fp32 products are exact there, so the code is that of the exact
// row whatever the order of the operations, save at borders 2^-53 wide. Codes outside the
// range are clamped to it and NaN is stored as 0, so a new row never holds NaN.
#pragma once

#include "common.h"

namespace ortmi {
namespace kvq {

enum Code { kInt8, kInt4, kFp8 };

// Everything a call's kernels read; by value in the launch.
struct Params {
    const void *q, *k, *v;      // new rows [token][head][hd], tokens q_tok / kv_tok elements apart
    int64_t q_tok, kv_tok;
    uint8_t *kc, *vc;           // the cache after the call: [B, KV, cap, hd] or pages
    int64_t cap;                // rows of a slab (0: pages)
    const int32_t* bt;          // pages: block table [B, maxb] of blocks of blk rows
    int64_t nblk;
    int blk, maxb;
    const int32_t* lens;        // slabs: tokens of a sequence less one [B], or null
    const int32_t *cum, *past;  // pages: cumulative new tokens [B + 1], cached tokens [B]
    int vpast, S, B, H, KV, hd, T;
    int limit;                  // keys at or past it are not attended
    const void *cos, *sin;      // [max_pos, half], or null
    int half, interleaved;
    int64_t max_pos;
    const void *qw, *kw;        // RMS norm weights of query and key heads, or null
    float eps;
    const float *ks, *vs;
    int k_chan, v_chan;         // scales per (kv head, channel)
    float scale;                // of the scores, times log2(e)
    const void* sink;           // [H], or null
    int dtype, code;
    void* out;                  // [T, H * hd]
    // Keys are taken in ranges of whole 128s. A unit is one range of one tile of columns and kv
    // head; units of tiles with more than one range leave outputs part [unit][columns][hd],
    // maxima and sums ml [unit][columns][2], unscaled.
    float *part, *ml;           // of token tiles, and of slabs' prompt tiles
    int tcols;                  // columns of a token tile's unit there
    int titems, tmin;           // token tiles: units over KV to come near, least keys of a range
    int ntile, nsplit, chunk;   // slabs: tiles of a sequence, ranges of `chunk` keys at most
    int planned;                // slabs, token tiles: ranges from the sequences' lengths
    float *ppart, *pml;         // pages: of prompt tiles
    int pparts, pmin;           // prompt tiles: units over KV in ppart, least keys of a range
    int4* plan;                 // pages: plan_units()
    int tgrid, pgrid;           // units over KV at most
    int fused;                  // slabs: the tiles write the new rows themselves
    int pieces;                 // new rows come in 16-byte pieces, rotated over the whole head
    uint32_t blk_mul;           // pages of whole key tiles: division by blk (Source)
    int blk_shift;
};

__device__ __forceinline__ float load_elem(const void* p, int64_t i, int dtype) {
    if (dtype == ORTMI_F32) return static_cast<const float*>(p)[i];
    if (dtype == ORTMI_F16) return (float)static_cast<const half_t*>(p)[i];
    return to_f32(static_cast<const uint16_t*>(p)[i]);
}

__device__ __forceinline__ void store_elem(void* p, int64_t i, float x, int dtype) {
    if (dtype == ORTMI_F32) static_cast<float*>(p)[i] = x;
    else if (dtype == ORTMI_F16) static_cast<half_t*>(p)[i] = (half_t)x;
    else static_cast<uint16_t*>(p)[i] = from_f32<uint16_t>(x);
}

__host__ __device__ constexpr int row_bytes(int code, int hd) {
    return code == kInt4 ? hd / 2 : hd;
}

// One sequence of the call: its rows are tokens tok0 .. tok0 + rows - 1, at positions past,
// past + 1, ...; the first `real` of them exist, the others pad a batch.
struct Seq {
    int tok0, rows, real, past;
    // Keys that the rows up to row r attend to.
    __device__ __forceinline__ int keys_to(int r, int limit) const {
        return min(past + min(r + 1, real), limit);
    }
};

template <bool PAGED>
__device__ __forceinline__ Seq sequence(const Params& p, int b) {
    Seq s;
    if constexpr (PAGED) {
        s.tok0 = min(max(p.cum[b], 0), p.T);
        s.rows = min(max(p.cum[b + 1], s.tok0), p.T) - s.tok0;
        s.real = s.rows;
        s.past = min(max(p.past[b], 0), INT32_MAX - p.T);  // positions stay below 2^31
    } else {
        const int full = p.vpast + p.S;
        const int n = p.lens ? min(max(p.lens[b], -1), full - 1) + 1 : full;
        s.tok0 = b * p.S;
        s.rows = p.S;
        s.past = max(n - p.S, 0);
        s.real = min(n, p.S);
    }
    return s;
}

// Cache row index of position `pos` of sequence b, kv head h, or -1 where the block table
// holds no block of the cache. Row r starts at byte r * row_bytes.
template <bool PAGED>
__device__ __forceinline__ int64_t cache_row(const Params& p, int b, int h, int pos) {
    if constexpr (PAGED) {
        const int lb = pos / p.blk;
        if (lb >= p.maxb) return -1;
        const int id = p.bt[(int64_t)b * p.maxb + lb];
        if (id < 0 || id >= p.nblk) return -1;
        return ((int64_t)id * p.blk + pos % p.blk) * p.KV + h;
    } else {
        return ((int64_t)b * p.KV + h) * p.cap + pos;
    }
}

// ------------------------------------------------------------------- new rows --
__device__ __forceinline__ int encode_int(double r, int lo, int hi) {
    if (!(r == r)) return 0;
    r = rint(r);
    return r < lo ? lo : (r > hi ? hi : (int)r);
}

__device__ __forceinline__ uint32_t encode_e4m3(double r) {
    if (!(r == r)) return 0;
    const uint32_t sign = signbit(r) ? 0x80u : 0u;
    const double a = fabs(r);
    if (a >= 448.0) return sign | 0x7Eu;
    if (a < 0.015625) return sign | (uint32_t)rint(a * 512.0);  // below 2^-6: steps of 2^-9
    const int e = ilogb(a);
    // 8 .. 16 eighths of 2^e; 16 carries into the exponent. At most 0x7E, as a < 448.
    return sign | (uint32_t)(((e + 7) << 3) + (int)rint(ldexp(a, 3 - e)) - 8);
}

// The stored code (int4: with its offset) of x / scale.
__device__ __forceinline__ uint32_t encode(double x, float scale, int code) {
    const double r = x / (double)scale;
    if (code == kInt8) return (uint32_t)encode_int(r, -128, 127) & 0xFFu;
    if (code == kFp8) return encode_e4m3(r);
    return (uint32_t)(encode_int(r, -8, 7) + 8);
}

// One new row, key or value, of kv head h by 16 lanes (`lane` of them), two channels a step.
template <bool PAGED>
__device__ __forceinline__ void append_row(const Params& p, int b, const Seq& s, int r, int h,
                                           bool is_v, int lane) {
    const int hd = p.hd, pos = s.past + r;
    const int64_t row = cache_row<PAGED>(p, b, h, pos);
    const void* src = is_v ? p.v : p.k;
    const int64_t x0 = (int64_t)(s.tok0 + r) * p.kv_tok + (int64_t)h * hd;
    const void* w = is_v ? nullptr : p.kw;
    double rinv = 1.0;
    if (p.kw) {  // (a value row's lanes go along)
        double ss = 0;
        for (int c = lane; c < hd; c += 16) {
            const double x = load_elem(src, x0 + c, p.dtype);
            ss += x * x;
        }
#pragma unroll
        for (int o = 8; o; o >>= 1) ss += __shfl_xor(ss, o, 64);
        rinv = 1.0 / sqrt(ss / hd + (double)p.eps);
    }
    if (row < 0) return;
    const bool rope = !is_v && p.cos;
    const int64_t prow = min((int64_t)pos, p.max_pos - 1) * p.half;
    const float* sc = is_v ? p.vs : p.ks;
    const bool chan = is_v ? p.v_chan : p.k_chan;
    uint8_t* dst = (is_v ? p.vc : p.kc) + row * row_bytes(p.code, hd);
    auto elem = [&](int c) -> double {
        const double x = load_elem(src, x0 + c, p.dtype);
        return w ? x * rinv * (double)load_elem(w, c, p.dtype) : x;
    };
    for (int c0 = 2 * lane; c0 < hd; c0 += 32) {
        uint32_t u[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = c0 + i;
            double x = elem(c);
            if (rope && c < 2 * p.half) {
                const bool second = p.interleaved ? (c & 1) : c >= p.half;
                const int f = p.interleaved ? c >> 1 : (second ? c - p.half : c);
                const double part = elem(p.interleaved ? c ^ 1 : (second ? c - p.half : c + p.half));
                const double co = load_elem(p.cos, prow + f, p.dtype);
                const double si = load_elem(p.sin, prow + f, p.dtype);
                x = second ? x * co + part * si : x * co - part * si;
            }
            u[i] = encode(x, sc[chan ? h * hd + c : 0], p.code);
        }
        if (p.code == kInt4) {
            dst[c0 >> 1] = (uint8_t)(u[0] | (u[1] << 4));
        } else {
            dst[c0] = (uint8_t)u[0];
            dst[c0 + 1] = (uint8_t)u[1];
        }
    }
}

// ------------------------------------------------------------------ query rows --
// Channel c of a query row, normalised and rotated, in 32 bits.
__device__ __forceinline__ float query_elem(const Params& p, int64_t x0, int64_t prow, float rinv,
                                            int c) {
    auto elem = [&](int i) {
        float x = load_elem(p.q, x0 + i, p.dtype);
        if (p.qw) x = x * rinv * load_elem(p.qw, i, p.dtype);
        return x;
    };
    const float self = elem(c);
    if (!p.cos || c >= 2 * p.half) return self;
    const bool second = p.interleaved ? (c & 1) : c >= p.half;
    const int f = p.interleaved ? c >> 1 : (second ? c - p.half : c);
    const float part = elem(p.interleaved ? c ^ 1 : (second ? c - p.half : c + p.half));
    const float co = load_elem(p.cos, prow + f, p.dtype), si = load_elem(p.sin, prow + f, p.dtype);
    return second ? self * co + part * si : self * co - part * si;
}

// 32-bit value of code `c` of a cache row (any code, any head size).
__device__ __forceinline__ float code_value(const uint8_t* row, int c, int code) {
    if (code == kInt8) return (float)(int8_t)row[c];
    if (code == kInt4) return (float)(int)((row[c >> 1] >> (4 * (c & 1))) & 15) - 8.f;
    const uint32_t u = row[c], e = (u >> 3) & 15u, m = u & 7u;
    if ((u & 0x7Fu) == 0x7Fu) return NAN;
    const float mag = e ? ldexpf((float)(8u + m), (int)e - 10) : (float)m * 0.001953125f;
    return u & 0x80u ? -mag : mag;
}

}  // namespace kvq
}  // namespace ortmi
