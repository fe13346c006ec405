// Attention over quantised key-value caches on the matrix cores (head sizes 64, 96, 128).
//
// A workgroup of 4 waves takes 16 NT columns, a column being one query row of one head of a
// group (all heads of the group read the same keys), over a range of keys; its waves take
// every fourth block of 32 keys and are joined at the end, ranges by merge_kernel. Scores are
// computed transposed, S^T = K Q^T, with v_mfma_f32_16x16x32_f16: a lane then holds column
// lane % 16 and, of a block's two key tiles, keys 4 (lane / 16) + i. That is already the order
// in which the second product O^T = V^T P^T takes P as its right operand (the 8 keys of a
// lane's k slots are those), so P never leaves its registers, and V is read with lane % 16
// running over channels, 8 keys of a lane's own channels at a time, which byte permutes turn
// into the left operand. Neither K nor V passes through LDS.
//
// Codes are exact in fp16 (int8 and int4 by putting the byte under the exponent of 1024, fp8
// by the conversion instruction). The key scales are folded into the query row, which is
// rounded to fp16 after a power of two has brought its largest element to [2^10, 2^11): one
// rounding of 2^-11 of an element, no range to leave. The probabilities are rounded to fp16
// at up to 2^14 (2^6 where a row's running maximum is exact), 2^-11 of each and 2^-31 of the
// largest at worst. fp32 tensors take both as two fp16 halves (22 bits) and twice the
// products. Sums, maxima and outputs are fp32. The value scales are applied to the output.
#pragma once

#include "kvq.h"

namespace ortmi {
namespace kvq {

// The reference point of a column's exponentials follows its maximum only where that has
// grown by more than 2^kSlack: most blocks then rescale nothing.
constexpr float kSlack = 8.f, kPBase = 6.f, kNone = -1e30f;

// Columns of a tile for a sequence with `cols` columns in all. fp32 holds twice the query
// registers: 64 columns of it do not fit.
__host__ __device__ constexpr int tile_width(int cols, int dtype) {
    return cols <= 16 ? 16 : (cols <= 32 || dtype == ORTMI_F32 ? 32 : 64);
}
// Pages: of a sequence with more than 16.
__host__ __device__ constexpr int page_width(int dtype) { return dtype == ORTMI_F32 ? 32 : 64; }

__device__ __forceinline__ half2_t as_half2(uint32_t u) { return __builtin_bit_cast(half2_t, u); }

// Four int8 or fp8 codes of a word as fp16: (0, 1), (2, 3).
template <int CODE>
__device__ __forceinline__ void halves4(uint32_t w, half2_t& a, half2_t& b) {
    if constexpr (CODE == kFp8) {
        a = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
        b = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    } else {
        const half2_t off = {(half_t)1152.f, (half_t)1152.f};
        const uint32_t u = w ^ 0x80808080u;
        a = as_half2(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
        b = as_half2(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
    }
}

// Two 4-bit codes at bits 0..3 and 16..19 of a word.
__device__ __forceinline__ half2_t nibbles2(uint32_t w) {
    const half2_t off = {(half_t)1032.f, (half_t)1032.f};
    return as_half2((w & 0x000F000Fu) | 0x64006400u) - off;
}

template <int CODE, int HD>
struct Layout {
    static constexpr bool kNib = CODE == kInt4;
    static constexpr int RB = row_bytes(CODE, HD);
    static constexpr int KS = HD / 32;      // k steps of a score
    static constexpr int MT = HD / 16;      // channel tiles of an output
    static constexpr int KW = RB / 16;      // words of a key row per lane
    static constexpr int VW = HD == 96 ? 2 : (RB == 128 ? 2 : 1);  // words of a value row per lane

    // Channel of element j of k step ks in the lanes of quarter q.
    __device__ static __forceinline__ int key_channel(int q, int ks, int j) {
        const int jj = kNib ? (j >> 1) + 4 * (j & 1) : j;
        if constexpr (HD == 128)
            return kNib ? 32 * q + 8 * ks + jj : 64 * (ks >> 1) + 16 * q + 8 * (ks & 1) + jj;
        else
            return ks < 2 ? 16 * q + 8 * ks + jj : 64 + 8 * q + jj;
    }
    // Byte at which the lanes of quarter q begin in a key row (and, HD 96, in its last third).
    static constexpr int kKeyStep = RB == 48 || RB == 32 ? 8 : 16;
    __device__ static __forceinline__ void load_key(__amdgpu_buffer_rsrc_t r, uint32_t at,
                                                    uint32_t at2, uint32_t (&w)[KW]) {
        if constexpr (kKeyStep == 16) {
            put(__builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0), &w[0]);
            if constexpr (RB == 128) put(__builtin_amdgcn_raw_buffer_load_b128(r, at + 64, 0, 0), &w[4]);
            if constexpr (RB == 96) put(__builtin_amdgcn_raw_buffer_load_b64(r, at2 + 64, 0, 0), &w[4]);
        } else {
            put(__builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0), &w[0]);
            if constexpr (RB == 48) w[2] = __builtin_amdgcn_raw_buffer_load_b32(r, at2 + 32, 0, 0);
        }
    }
    template <typename V>
    __device__ static __forceinline__ void put(V v, uint32_t* w) {
#pragma unroll
        for (unsigned i = 0; i < sizeof(V) / 4; ++i) w[i] = v[i];
    }
    __device__ static __forceinline__ half8_t key_step(const uint32_t (&w)[KW], int ks) {
        half2_t h[4];
        if constexpr (kNib) {
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = nibbles2(w[ks] >> (4 * i));
        } else {
            halves4<CODE>(w[2 * ks], h[0], h[1]);
            halves4<CODE>(w[2 * ks + 1], h[2], h[3]);
        }
        return __builtin_bit_cast(half8_t, h);
    }

    // Channel of row m of channel tile t: a lane's channels are neighbours in memory.
    __device__ static __forceinline__ int value_channel(int m, int t) {
        if constexpr (HD == 128) return 8 * m + t;
        else if constexpr (HD == 64) return 4 * m + t;
        else return t < 4 ? 4 * m + t : 64 + 2 * m + (t - 4);
    }
    // Bytes of a lane's first channels in a value row (HD 96: of its last third).
    static constexpr int kValStep = HD == 128 ? RB / 16 : RB * 4 / HD;
    __device__ static __forceinline__ void load_value(__amdgpu_buffer_rsrc_t r, uint32_t at,
                                                      uint32_t at2, uint32_t (&w)[VW]) {
        if constexpr (kValStep == 8) put(__builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0), &w[0]);
        else if constexpr (kValStep == 4) w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0);
        else w[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0);
        if constexpr (RB == 96)
            w[1] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at2 + 64, 0, 0);
        if constexpr (RB == 48)
            w[1] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, at2 + 32, 0, 0);
    }
    // Left operands of channel tiles 2u and 2u + 1 from a lane's 8 value rows.
    __device__ static __forceinline__ void value_steps(const uint32_t (&w)[8][VW], int u, half8_t& a, half8_t& b) {
        half2_t ha[4], hb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (kNib) {
                const int word = HD == 96 ? u / 2 : 0, byte = HD == 96 ? u % 2 : u;
                const uint32_t sel = 0x0C000C00u | (uint32_t)byte | ((uint32_t)(4 + byte) << 16);
                const uint32_t x = __builtin_amdgcn_perm(w[2 * i + 1][word], w[2 * i][word], sel);
                ha[i] = nibbles2(x);
                hb[i] = nibbles2(x >> 4);
            } else {
                const int word = u / 2, byte = 2 * (u % 2);
                const uint32_t sel = (uint32_t)byte | ((uint32_t)(4 + byte) << 8) |
                                     ((uint32_t)(byte + 1) << 16) | ((uint32_t)(5 + byte) << 24);
                halves4<CODE>(__builtin_amdgcn_perm(w[2 * i + 1][word], w[2 * i][word], sel),
                              ha[i], hb[i]);
            }
        }
        a = __builtin_bit_cast(half8_t, ha);
        b = __builtin_bit_cast(half8_t, hb);
    }
};

// A lane's share of a block of 32 keys: of both key tiles the row lane % 16, and its 8 value
// rows 4 (lane / 16) + i of both.
template <int CODE, int HD>
struct Block {
    uint32_t k[2][Layout<CODE, HD>::KW];
    uint32_t v[8][Layout<CODE, HD>::VW];
};

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// Where a wave finds the keys and values of a range [k0, k1) of one sequence and kv head.
// Loads go through buffer resources whose size ends with the last key, so that what lies
// behind it reads as zeros (0 times a stray NaN code would be NaN). Slabs: one resource each
// for the range. Pages, multiples of 16 keys: a tile of 16 keys lies in one page; its
// resources are made from the block table, of size 0 where the table holds no block.
template <int CODE, int HD, bool PAGED>
struct Source {
    using L = Layout<CODE, HD>;
    const Params& p;
    const uint8_t *kbase, *vbase;
    int b, k0, k1;
    uint32_t stride, kat, kat2, vat, vat2;

    __device__ __forceinline__ Source(const Params& p_, int b_, int h, int k0_, int k1_)
        : p(p_), b(b_), k0(k0_), k1(k1_) {
        const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
        stride = (uint32_t)(PAGED ? p.KV * L::RB : L::RB);
        const int64_t at = (PAGED ? (int64_t)h : cache_row<false>(p, b, h, k0)) * L::RB;
        kbase = p.kc + at;
        vbase = p.vc + at;
        kat = m * stride + q * L::kKeyStep;
        kat2 = m * stride + q * (L::kKeyStep / 2);
        vat = 4 * q * stride + m * L::kValStep;
        vat2 = 4 * q * stride + m * (L::kValStep / 2);
    }
    // Slots of the two key tiles of block kb: -1 behind the end and where there is no block.
    __device__ __forceinline__ int2 slots(int kb) const {
        int s[2] = {-1, -1};
        if constexpr (PAGED) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int key = kb + 16 * t;
                if (key < k1) {
                    const int lb = p.blk_shift >= 0 ? key >> p.blk_shift : key / p.blk;
                    const int id = lb < p.maxb ? p.bt[(int64_t)b * p.maxb + lb] : -1;
                    if (id >= 0 && id < p.nblk) s[t] = id * p.blk + (key - lb * p.blk);
                }
            }
        }
        return make_int2(s[0], s[1]);
    }
    __device__ __forceinline__ void load(int kb, int2 sl, Block<CODE, HD>& o) const {
        if constexpr (!PAGED) {
            const uint32_t bytes = (uint32_t)(k1 - k0) * L::RB;
            const __amdgpu_buffer_rsrc_t kr = buffer_rsrc(kbase, bytes);
            const __amdgpu_buffer_rsrc_t vr = buffer_rsrc(vbase, bytes);
            const uint32_t off = (uint32_t)(kb - k0) * L::RB;
#pragma unroll
            for (int t = 0; t < 2; ++t)
                L::load_key(kr, off + kat + 16 * t * L::RB, off + kat2 + 16 * t * L::RB, o.k[t]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t r = ((j & 3) + 16 * (j >> 2)) * L::RB;
                L::load_value(vr, off + vat + r, off + vat2 + r, o.v[j]);
            }
        } else {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int slot = t ? sl.y : sl.x;
                const int rows = min(16, k1 - kb - 16 * t);
                const uint32_t bytes = slot < 0 ? 0u : (uint32_t)(rows - 1) * stride + L::RB;
                const int64_t at = (int64_t)max(slot, 0) * stride;
                const __amdgpu_buffer_rsrc_t kr = buffer_rsrc(kbase + at, bytes);
                const __amdgpu_buffer_rsrc_t vr = buffer_rsrc(vbase + at, bytes);
                L::load_key(kr, kat, kat2, o.k[t]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    L::load_value(vr, vat + j * stride, vat2 + j * stride, o.v[4 * t + j]);
            }
        }
    }
};

template <int HD, int NT, bool F32>
struct TileShared {
    static constexpr int kCols = 16 * NT;
    static constexpr int kRow = HD + 4;  // floats of a row, four more than a multiple of the banks
    // Raw query rows and their cos/sin; then two waves' outputs; then the tile's output rows.
    static constexpr int kFloats = 2 * kCols * kRow;
    __align__(16) float rows[kFloats];
    __align__(16) half_t q[(F32 ? 2 : 1) * kCols * HD];
    float f[kCols], inv[kCols];
    int pos[kCols];
    float m[4][kCols], l[4][kCols];
};

// N consecutive elements of a 16-byte aligned row as fp32.
template <int N, bool F32>
__device__ __forceinline__ void load_piece(const void* base, int64_t at, int dtype, float (&x)[N]) {
    if constexpr (F32) {
        const float* s = static_cast<const float*>(base) + at;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 v = *reinterpret_cast<const float2*>(s + i);
            x[i] = v.x;
            x[i + 1] = v.y;
        }
    } else {
        const uint32_t* s = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(base) + at);
        uint32_t w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = s[i];
        if (dtype == ORTMI_F16) {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = (float)as_half2(w[i / 2])[i & 1];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = to_f32((uint16_t)(w[i / 2] >> (16 * (i & 1))));
        }
    }
}

template <bool F32>
__device__ __forceinline__ float load_one(const void* base, int64_t at, int dtype) {
    if constexpr (F32) return static_cast<const float*>(base)[at];
    const uint16_t u = static_cast<const uint16_t*>(base)[at];
    return dtype == ORTMI_F16 ? (float)__builtin_bit_cast(half_t, u) : to_f32(u);
}

// The query rows of columns c0 .. c0 + 16 NT - 1 into LDS, 16 lanes a column: (normalised and)
// rotated, times the key scales, brought to [2^10, 2^11) and rounded to fp16, in the order
// [column][k step][quarter][8] of the right operand (fp32: the second halves behind).
template <int CODE, int HD, int NT, bool F32>
__device__ __forceinline__ void stage_queries(const Params& p, const Seq& s, int h, int c0,
                                              TileShared<HD, NT, F32>& sh) {
    using L = Layout<CODE, HD>;
    using SH = TileShared<HD, NT, F32>;
    constexpr int N = HD / 16;
    const int G = p.H / p.KV, tid = threadIdx.x, lane = tid & 15;
    float x[NT][N];
    const bool rope = p.cos != nullptr;
#pragma unroll
    for (int cc = 0; cc < NT; ++cc) {
        const int c = 16 * cc + (tid >> 4), r = (c0 + c) / G, g = (c0 + c) - r * G;
        const bool live = r < s.real;
        const int tok = s.tok0 + (live ? r : 0), pos = s.past + (live ? r : 0);
        load_piece<N, F32>(p.q, (int64_t)tok * p.q_tok + (int64_t)(h * G + g) * HD + lane * N,
                           p.dtype, x[cc]);
        if (rope) {
            const int64_t prow = min((int64_t)pos, p.max_pos - 1) * p.half;
            float* cs = sh.rows + (SH::kCols + c) * SH::kRow;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
                const int f = lane + 16 * i;
                if (f < p.half) {
                    cs[2 * f] = load_one<F32>(p.cos, prow + f, p.dtype);
                    cs[2 * f + 1] = load_one<F32>(p.sin, prow + f, p.dtype);
                }
            }
        }
        if (lane == 0) sh.pos[c] = live ? pos : -1;
    }
    if (p.qw) {
        float w[N];
        load_piece<N, F32>(p.qw, lane * N, p.dtype, w);
#pragma unroll
        for (int cc = 0; cc < NT; ++cc) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) ss += x[cc][i] * x[cc][i];
            const float rinv = 1.f / sqrtf(group_sum<16>(ss) / (float)HD + p.eps);
#pragma unroll
            for (int i = 0; i < N; ++i) x[cc][i] = x[cc][i] * rinv * w[i];
        }
    }
#pragma unroll
    for (int cc = 0; cc < NT; ++cc) {
        float* row = sh.rows + (16 * cc + (tid >> 4)) * SH::kRow + lane * N;
#pragma unroll
        for (int i = 0; i < N; ++i) row[i] = x[cc][i];
    }
    __syncthreads();
    // Element e of a column is channel ch[e]; the channels and scales serve every column.
    int ch[N];
    float sc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = lane * N + i;
        ch[i] = L::key_channel((e >> 3) & 3, e >> 5, e & 7);
        sc[i] = p.ks[p.k_chan ? h * HD + ch[i] : 0];
    }
#pragma unroll
    for (int cc = 0; cc < NT; ++cc) {
        const int c = 16 * cc + (tid >> 4);
        const float* row = sh.rows + c * SH::kRow;
        const float* cs = sh.rows + (SH::kCols + c) * SH::kRow;
        float y[N], top = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int k = ch[i];
            float v = row[k];
            if (rope && k < 2 * p.half) {
                const bool second = p.interleaved ? (k & 1) : k >= p.half;
                const int f = p.interleaved ? k >> 1 : (second ? k - p.half : k);
                const float o = row[p.interleaved ? k ^ 1 : (second ? k - p.half : k + p.half)];
                const float co = cs[2 * f], si = cs[2 * f + 1];
                v = second ? v * co + o * si : v * co - o * si;
            }
            y[i] = v * sc[i];
            top = fmaxf(top, fabsf(y[i]));
        }
        top = group_max<16>(top);
        // A row of zeros, or with an infinity, is taken as it is.
        const int ex = top > 0.f && top < INFINITY ? max(-100, min(ilogbf(top), 116)) : 10;
        const bool live = sh.pos[c] >= 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float z = live ? ldexpf(y[i], 10 - ex) : 0.f;
            const half_t hi = (half_t)z;
            sh.q[c * HD + lane * N + i] = hi;
            if constexpr (F32) sh.q[(16 * NT + c) * HD + lane * N + i] = (half_t)(z - (float)hi);
        }
        if (lane == 0) sh.f[c] = ldexpf(p.scale, ex - 10);
    }
}

__device__ __forceinline__ half8_t pack_p(const float (&a)[4], const float (&b)[4]) {
    half8_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[i] = (half_t)a[i];
        r[4 + i] = (half_t)b[i];
    }
    return r;
}

// One tile of columns c0 .. over keys [k0, k1) of sequence s: range `split` of `nsplit`.
template <int CODE, int HD, int NT, bool F32, bool PAGED>
__device__ __forceinline__ void attend_tile(const Params& p, const Seq& s, int b, int h, int c0,
                                            int k0, int k1, int split, int nsplit,
                                            TileShared<HD, NT, F32>& sh) {
    using L = Layout<CODE, HD>;
    using SH = TileShared<HD, NT, F32>;
    constexpr int KS = L::KS, MT = L::MT;
    const int lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
    const int wave = uniform(threadIdx.x >> 6);
    const int G = p.H / p.KV;

    stage_queries<CODE, HD, NT, F32>(p, s, h, c0, sh);
    __syncthreads();
    const half8_t* sq = reinterpret_cast<const half8_t*>(sh.q);
    half8_t Q[NT][KS], QL[F32 ? NT : 1][KS];
    float f[NT];
    int pos[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            Q[t][ks] = sq[((16 * t + n) * KS + ks) * 4 + q];
            if constexpr (F32) QL[t][ks] = sq[((16 * (NT + t) + n) * KS + ks) * 4 + q];
        }
        f[t] = sh.f[16 * t + n];
        pos[t] = sh.pos[16 * t + n];
    }
    const int first = s.past + c0 / G;  // the lowest position of the tile

    float4_t O[MT][NT];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = kNone;
        l[t] = 0.f;
#pragma unroll
        for (int d = 0; d < MT; ++d) O[d][t] = float4_t{0.f, 0.f, 0.f, 0.f};
    }

    const Source<CODE, HD, PAGED> src(p, b, h, k0, k1);
    int kb = k0 + 32 * wave;
    int2 sl = src.slots(kb), sl_n = src.slots(kb + 128);
    Block<CODE, HD> cur, nxt;
    if (kb < k1) src.load(kb, sl, cur);
    for (; kb < k1; kb += 128) {
        const int2 sl_c = sl;
        if (kb + 128 < k1) {
            src.load(kb + 128, sl_n, nxt);
            sl = sl_n;
            sl_n = src.slots(kb + 256);
        }
        float4_t S[2][NT];
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
#pragma unroll
            for (int t = 0; t < NT; ++t) S[t2][t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const half8_t a = L::key_step(cur.k[t2], ks);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    S[t2][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, Q[t][ks], S[t2][t], 0, 0, 0);
                    if constexpr (F32)
                        S[t2][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, QL[t][ks], S[t2][t], 0, 0, 0);
                }
            }
        }
        // Keys that a column does not attend: later ones, behind the end, of no page.
        const bool masked = kb + 31 > first || kb + 32 > k1 ||
                            (PAGED && (sl_c.x < 0 || sl_c.y < 0));
        float x[NT][2][4];
        bool grow = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[t][t2][i] = S[t2][t][i] * f[t];
            if (masked) {
#pragma unroll
                for (int t2 = 0; t2 < 2; ++t2) {
                    const bool none = PAGED && (t2 ? sl_c.y : sl_c.x) < 0;
                    const int end = none ? -1 : min(pos[t], k1 - 1);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        x[t][t2][i] = kb + 16 * t2 + 4 * q + i > end ? -INFINITY : x[t][t2][i];
                }
            }
            const float top =
                fmaxf(fmaxf(fmaxf(x[t][0][0], x[t][0][1]), fmaxf(x[t][0][2], x[t][0][3])),
                      fmaxf(fmaxf(x[t][1][0], x[t][1][1]), fmaxf(x[t][1][2], x[t][1][3])));
            grow |= top > m[t] + kSlack;
        }
        if (__any(grow)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float top = kNone;
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(x[t][0][i], x[t][1][i]));
                LanePair pr = swap16(top);
                pr = swap32(fmaxf(pr.a, pr.b));
                const float mm = fmaxf(m[t], fmaxf(pr.a, pr.b));
                const float a = __builtin_amdgcn_exp2f(m[t] - mm);
                m[t] = mm;
                l[t] *= a;
#pragma unroll
                for (int d = 0; d < MT; ++d) O[d][t] *= a;
            }
        }
        half8_t P[NT], PL[F32 ? NT : 1];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float ref = m[t] - kPBase;
            float e[2][4];
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[t2][i] = __builtin_amdgcn_exp2f(x[t][t2][i] - ref);
                    l[t] += e[t2][i];
                }
            P[t] = pack_p(e[0], e[1]);
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[0][i] -= (float)P[t][i];
                    e[1][i] -= (float)P[t][4 + i];
                }
                PL[t] = pack_p(e[0], e[1]);
            }
        }
#pragma unroll
        for (int u = 0; u < MT / 2; ++u) {
            half8_t a[2];
            L::value_steps(cur.v, u, a[0], a[1]);
#pragma unroll
            for (int d = 0; d < 2; ++d)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float4_t& o = O[2 * u + d][t];
                    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[d], P[t], o, 0, 0, 0);
                    if constexpr (F32)
                        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[d], PL[t], o, 0, 0, 0);
                }
        }
        cur = nxt;
    }

    // The four waves: maxima and sums, then outputs in two steps through LDS.
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        LanePair pr = swap16(l[t]);
        pr = swap32(pr.a + pr.b);
        l[t] = pr.a + pr.b;
        if (q == 0) {
            sh.m[wave][16 * t + n] = m[t];
            sh.l[wave][16 * t + n] = l[t];
        }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float mm = kNone, sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sh.m[w][16 * t + n]);
#pragma unroll
        for (int w = 0; w < 4; ++w)
            sum += sh.l[w][16 * t + n] * __builtin_amdgcn_exp2f(sh.m[w][16 * t + n] - mm);
        const float a = __builtin_amdgcn_exp2f(m[t] - mm);
#pragma unroll
        for (int d = 0; d < MT; ++d) O[d][t] *= a;
        m[t] = mm;
        l[t] = sum;
    }
    float4_t* so = reinterpret_cast<float4_t*>(sh.rows);
    constexpr int kSlotVecs = MT * NT * 64;
#pragma unroll
    for (int step = 2; step; step >>= 1) {
        if (wave >= step && wave < 2 * step) {
#pragma unroll
            for (int d = 0; d < MT; ++d)
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    so[(wave - step) * kSlotVecs + (d * NT + t) * 64 + lane] = O[d][t];
        }
        __syncthreads();
        if (wave < step) {
#pragma unroll
            for (int d = 0; d < MT; ++d)
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    O[d][t] += so[wave * kSlotVecs + (d * NT + t) * 64 + lane];
        }
        __syncthreads();
    }
    // Output rows by all waves. A partial row stays unscaled, with its maximum and sum.
    if (wave == 0) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float* row = sh.rows + (16 * t + n) * SH::kRow;
#pragma unroll
            for (int d = 0; d < MT; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) row[L::value_channel(4 * q + i, d)] = O[d][t][i];
            const int c = c0 + 16 * t + n, r = c / G, head = h * G + (c - r * G);
            if (q == 0 && r < s.real) {
                const int64_t orow = (int64_t)(s.tok0 + r) * p.H + head;
                if (nsplit > 1) {
                    p.ml[(orow * p.nsplit + split) * 2] = m[t];
                    p.ml[(orow * p.nsplit + split) * 2 + 1] = l[t];
                } else {
                    float a = 1.f, sum = l[t];
                    if (PAGED && p.sink) {
                        const float sk = load_one<F32>(p.sink, head, p.dtype) * 1.44269504088896341f;
                        const float mm = fmaxf(m[t], sk);
                        a = __builtin_amdgcn_exp2f(m[t] - mm);
                        sum = sum * a + __builtin_amdgcn_exp2f(sk - mm + kPBase);
                    }
                    sh.inv[16 * t + n] = sum != 0.f ? a / sum : 0.f;
                }
            }
        }
    }
    __syncthreads();
    constexpr int kPieces = HD / 4;  // of a row: four channels a thread and step
    for (int i = threadIdx.x; i < SH::kCols * kPieces; i += 256) {
        const int c = i / kPieces, ch = 4 * (i % kPieces), r = (c0 + c) / G;
        if (r >= s.rows) break;
        const int64_t orow = (int64_t)(s.tok0 + r) * p.H + h * G + (c0 + c - r * G);
        float4_t v = *reinterpret_cast<const float4_t*>(sh.rows + c * SH::kRow + ch);
        if (nsplit > 1) {
            if (r < s.real)
                *reinterpret_cast<float4_t*>(p.part + (orow * p.nsplit + split) * HD + ch) = v;
            continue;
        }
        const float inv = r < s.real ? sh.inv[c] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[j] = inv != 0.f ? v[j] * inv * p.vs[p.v_chan ? h * HD + ch + j : 0] : 0.f;
        if constexpr (F32) {
            *reinterpret_cast<float4_t*>(static_cast<float*>(p.out) + orow * HD + ch) = v;
        } else {
            uint16_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                o[j] = p.dtype == ORTMI_F16 ? __builtin_bit_cast(uint16_t, (half_t)v[j])
                                            : from_f32<uint16_t>(v[j]);
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + orow * HD + ch) =
                *reinterpret_cast<const uint2*>(o);
        }
    }
}

// A tile that attends nothing: padded rows.
template <int HD, bool F32>
__device__ __forceinline__ void zero_rows(const Params& p, const Seq& s, int h, int c0, int cols) {
    const int G = p.H / p.KV;
    for (int i = threadIdx.x; i < cols * HD; i += 256) {
        const int c = c0 + i / HD, r = c / G;
        if (r >= s.rows) break;
        const int64_t o = ((int64_t)(s.tok0 + r) * p.H + h * G + (c - r * G)) * HD + i % HD;
        if constexpr (F32) static_cast<float*>(p.out)[o] = 0.f;
        else static_cast<uint16_t*>(p.out)[o] = 0;
    }
}

// Slabs. Workgroups: (range, tile, slab), the slab running fastest (slabs of one residue
// modulo 8 then stay on one XCD) and later tiles, which see more keys, first. Where a
// sequence's columns are one tile, the workgroup whose range holds the new rows writes them
// to the cache itself.
template <int CODE, int HD, int NT, bool F32>
__global__ __launch_bounds__(256, NT == 1 ? 2 : 1) void tile_kernel(Params p) {
    __shared__ TileShared<HD, NT, F32> sh;
    const int slabs = p.B * p.KV;
    const int split = blockIdx.x / (slabs * p.ntile), rem = blockIdx.x % (slabs * p.ntile);
    const int tile = p.ntile - 1 - rem / slabs, slab = rem % slabs, b = slab / p.KV, h = slab % p.KV;
    const Seq s = sequence<false>(p, b);
    const int G = p.H / p.KV, c0 = tile * 16 * NT;
    if (c0 / G >= s.real) {
        if (split == 0) zero_rows<HD, F32>(p, s, h, c0, 16 * NT);
        return;
    }
    const int kend = s.keys_to((min(c0 + 16 * NT, s.rows * G) - 1) / G, p.limit);
    const int k0 = split * p.chunk, k1 = min(k0 + p.chunk, kend);
    if (k0 >= kend) {  // not the range that writes the rows past the sequence's end
        return;
    }
    if (p.fused) {
        const int r0 = max(k0 - s.past, 0), r1 = min(k1 - s.past, s.real);
        for (int i = 2 * r0 + uniform(threadIdx.x >> 6); i < 2 * r1; i += 4)
            append_row<false>(p, b, s, i >> 1, h, i & 1);
        __syncthreads();
    }
    const int nsplit = (kend + p.chunk - 1) / p.chunk;
    attend_tile<CODE, HD, NT, F32, false>(p, s, b, h, c0, k0, k1, split, nsplit, sh);
    if (nsplit > 1 && split == 0 && s.real < s.rows)  // rows of the tile that only pad
        zero_rows<HD, F32>(p, s, h, max(c0, s.real * G), c0 + 16 * NT - max(c0, s.real * G));
}

// Pages, sequences of at most 16 columns: workgroups (range, sequence, kv head).
template <int CODE, int HD, bool F32>
__global__ __launch_bounds__(256, 2) void page_token_kernel(Params p) {
    __shared__ TileShared<HD, 1, F32> sh;
    const int slabs = p.B * p.KV, split = blockIdx.x / slabs, slab = blockIdx.x % slabs;
    const int b = slab / p.KV, h = slab % p.KV, G = p.H / p.KV;
    const Seq s = sequence<true>(p, b);
    if (s.rows == 0 || s.rows * G > 16) return;
    const int kend = s.keys_to(s.rows - 1, p.limit);
    const int k0 = split * p.chunk, k1 = min(k0 + p.chunk, kend);
    if (k0 >= kend) return;
    attend_tile<CODE, HD, 1, F32, true>(p, s, b, h, 0, k0, k1, split,
                                        (kend + p.chunk - 1) / p.chunk, sh);
}

// Pages, the other sequences: a workgroup for each (range, listed tile, kv head), those past
// the list's end with nothing to do.
template <int CODE, int HD, bool F32>
__global__ __launch_bounds__(256, 1) void page_tile_kernel(Params p) {
    constexpr int NT = page_width(F32 ? ORTMI_F32 : ORTMI_F16) / 16;
    __shared__ TileShared<HD, NT, F32> sh;
    const int G = p.H / p.KV, per = p.max_tiles * p.KV;
    const int split = blockIdx.x / per, rem = blockIdx.x % per, h = rem % p.KV, i = rem / p.KV;
    if (i >= *p.tile_count) return;
    const int2 tl = p.tiles[i];
    const int b = tl.x, c0 = tl.y;
    const Seq s = sequence<true>(p, b);
    const int kend = s.keys_to((min(c0 + 16 * NT, s.rows * G) - 1) / G, p.limit);
    const int k0 = split * p.tile_chunk, k1 = min(k0 + p.tile_chunk, kend);
    if (k0 >= kend) return;
    attend_tile<CODE, HD, NT, F32, true>(p, s, b, h, c0, k0, k1, split,
                                        (kend + p.tile_chunk - 1) / p.tile_chunk, sh);
}

// Launches for one code; in kvq_int8.hip, kvq_int4.hip and kvq_fp8.hip.
int tiles_int8(const Params& p, bool paged, hipStream_t st);
int tiles_int4(const Params& p, bool paged, hipStream_t st);
int tiles_fp8(const Params& p, bool paged, hipStream_t st);

template <int CODE, int HD, bool F32>
int launch_tiles(const Params& p, bool paged, hipStream_t st) {
    if (!paged) {
        const dim3 grid((unsigned)(p.B * p.KV * p.ntile * p.nsplit));
        const int w = tile_width(p.S * (p.H / p.KV), p.dtype);
        if (w == 16) hipLaunchKernelGGL((tile_kernel<CODE, HD, 1, F32>), grid, dim3(256), 0, st, p);
        else if (w == 32) hipLaunchKernelGGL((tile_kernel<CODE, HD, 2, F32>), grid, dim3(256), 0, st, p);
        else if constexpr (!F32) hipLaunchKernelGGL((tile_kernel<CODE, HD, 4, F32>), grid, dim3(256), 0, st, p);
        return check_launch("kv tiles");
    }
    const int G = p.H / p.KV;
    if (G <= 16) {
        hipLaunchKernelGGL((page_token_kernel<CODE, HD, F32>),
                           dim3((unsigned)(p.B * p.KV * p.nsplit)), dim3(256), 0, st, p);
        if (int rc = check_launch("kv page tokens")) return rc;
    }
    if ((int64_t)p.T * G <= 16) return ORTMI_OK;  // no sequence has more than 16 columns
    hipLaunchKernelGGL((page_tile_kernel<CODE, HD, F32>),
                       dim3((unsigned)(p.max_tiles * p.KV * p.tile_nsplit)), dim3(256), 0, st, p);
    return check_launch("kv page tiles");
}

template <int CODE>
int launch_code(const Params& p, bool paged, hipStream_t st) {
    const bool f32 = p.dtype == ORTMI_F32;
    switch (p.hd) {
        case 64: return f32 ? launch_tiles<CODE, 64, true>(p, paged, st) : launch_tiles<CODE, 64, false>(p, paged, st);
        case 96: return f32 ? launch_tiles<CODE, 96, true>(p, paged, st) : launch_tiles<CODE, 96, false>(p, paged, st);
        default: return f32 ? launch_tiles<CODE, 128, true>(p, paged, st) : launch_tiles<CODE, 128, false>(p, paged, st);
    }
}

}  // namespace kvq
}  // namespace ortmi
