// Attention over quantised key-value caches on the matrix cores (head sizes 64, 96, 128).
//
// A column is one query row of one head of a group: all heads of a group read the same keys.
// Scores are computed transposed, S^T = K Q^T, with v_mfma_f32_16x16x32_f16: a lane then holds
// column lane % 16 and, of a tile of 16 keys, keys 4 (lane / 16) + i. Two tiles are already the
// order in which the second product O^T = V^T P^T takes P as its right operand (the 8 keys of
// a lane's k slots are those), so P never leaves its registers, and V is read with lane % 16
// running over channels, 8 keys of a lane's own channels at a time, which byte permutes turn
// into the left operand.
//
// Codes are exact in fp16 (int8 and int4 by putting the byte under the exponent of 1024, fp8
// by the conversion instruction). The key scales are folded into the query row, which is
// rounded to fp16 after a power of two has brought its largest element to [2^10, 2^11): one
// rounding of 2^-11 of an element, no range to leave. The probabilities are rounded to fp16
// at up to 2^14 (2^6 where a row's running maximum is exact), 2^-11 of each and 2^-31 of the
// largest at worst. Sums, maxima and outputs are fp32. The value scales are applied to the
// output. Where few columns leave the matrix cores idle (token tiles), the query row is taken
// as two fp16 halves, 22 bits; fp32 tensors take the probabilities as two halves too.
//
// Token tiles: 16 columns. A workgroup's 4 waves take every fourth block of 32 keys of its
// range and are joined at the end; keys and values go from memory into registers, where each
// wave decodes its own. Memory binds it: 4 sequences of 131072 int8 keys, 8 heads of 128, 190
// us, 5.65 TB/s.
//
// Prompt tiles: 128 columns (fp32 64), 32 a wave, by two teams of 4 waves that take every other
// block of 64 keys and are joined at the end. A team decodes its block together into LDS, a
// quarter each, in the order that the products read: decoded once for 128 columns. Two buffers
// a team, so that one barrier for two blocks suffices; the second team fills the waits of the
// first, which the registers (200 of 256 at two waves a SIMD) leave no other wave for.
#pragma once

#include "kvq.h"

namespace ortmi {
namespace kvq {

// The reference point of a column's exponentials follows its maximum only where that has
// grown by more than 2^kSlack: most blocks then rescale nothing.
constexpr float kSlack = 8.f, kPBase = 6.f, kNone = -1e30f;

// Columns of a tile for a sequence with `cols` columns in all: 16, or those of a prompt tile
// (fp32 holds twice the operands).
__host__ __device__ constexpr int prompt_width(int dtype) { return dtype == ORTMI_F32 ? 64 : 128; }
__host__ __device__ constexpr int tile_width(int cols, int dtype) {
    return cols <= 16 ? 16 : prompt_width(dtype);
}

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

    // Channel jj (of 8) of k step ks in the lanes of quarter q: HD 128, codes of a byte: 64
    // (ks / 2) + 16 q + 8 (ks % 2) + jj; of a nibble: 32 q + 8 ks + jj; else 16 q + 8 ks + jj,
    // and 64 + 8 q + jj in the third step of 96. A word of nibbles gives jj in the order 0, 4,
    // 1, 5, 2, 6, 3, 7.
    // The place of channel c in a column's [k step][quarter][8] operand.
    __device__ static __forceinline__ int key_slot(int c) {
        int q, ks;
        const int jj = c & 7;
        if constexpr (HD == 128) {
            q = kNib ? c >> 5 : (c >> 4) & 3;
            ks = kNib ? (c >> 3) & 3 : 2 * (c >> 6) + ((c >> 3) & 1);
        } else {
            q = c < 64 ? c >> 4 : (c - 64) >> 3;
            ks = c < 64 ? (c >> 3) & 1 : 2;
        }
        const int j = kNib ? ((jj & 3) << 1) | (jj >> 2) : jj;
        return (ks * 4 + q) * 8 + j;
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
    // Slot of the key tile at `key`: -1 behind the end and where there is no block.
    __device__ __forceinline__ int slot(int key) const {
        int s = -1;
        if constexpr (PAGED) {
            if (key < k1) {
                const int lb = p.blk_shift >= 0 ? key >> p.blk_shift : key / p.blk;
                const int id = lb < p.maxb ? p.bt[(int64_t)b * p.maxb + lb] : -1;
                s = id >= 0 && id < p.nblk ? id * p.blk + (key - lb * p.blk) : -1;
            }
        }
        return s;
    }
    // The resource of the cache rows of a tile in a page.
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t page(const uint8_t* base, int key, int slot) const {
        const int rows = min(16, k1 - key);
        const uint32_t bytes = slot < 0 ? 0u : (uint32_t)(rows - 1) * stride + L::RB;
        return buffer_rsrc(base + (int64_t)max(slot, 0) * stride, bytes);
    }
    // A lane's share of the key tile at `key`.
    __device__ __forceinline__ void keys(int key, int slot, uint32_t (&w)[L::KW]) const {
        if constexpr (PAGED) {
            L::load_key(page(kbase, key, slot), kat, kat2, w);
        } else {
            const uint32_t off = (uint32_t)(key - k0) * L::RB;
            L::load_key(buffer_rsrc(kbase, (uint32_t)(k1 - k0) * L::RB), off + kat, off + kat2, w);
        }
    }
    // Its 8 value rows of the two tiles at `key`.
    __device__ __forceinline__ void values(int key, int slot0, int slot1, uint32_t (&w)[8][L::VW]) const {
        if constexpr (PAGED) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const __amdgpu_buffer_rsrc_t r = page(vbase, key + 16 * t, t ? slot1 : slot0);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    L::load_value(r, vat + j * stride, vat2 + j * stride, w[4 * t + j]);
            }
        } else {
            const uint32_t off = (uint32_t)(key - k0) * L::RB;
            const __amdgpu_buffer_rsrc_t r = buffer_rsrc(vbase, (uint32_t)(k1 - k0) * L::RB);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t at = ((j & 3) + 16 * (j >> 2)) * L::RB;
                L::load_value(r, off + vat + at, off + vat2 + at, w[j]);
            }
        }
    }
    __device__ __forceinline__ int2 slots(int kb) const { return make_int2(slot(kb), slot(kb + 16)); }
    __device__ __forceinline__ void load(int kb, int2 sl, Block<CODE, HD>& o) const {
        keys(kb, sl.x, o.k[0]);
        keys(kb + 16, sl.y, o.k[1]);
        values(kb, sl.x, sl.y, o.v);
    }
};

template <int HD>
constexpr int kRowFloats = HD + 4;  // of a row in LDS: four more than a multiple of the banks

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

// The query rows of columns c0 .. c0 + GR NC - 1 into LDS, 16 lanes a column, each a sixteenth
// of its channels: (normalised and) rotated, times the key scales, brought to [2^10, 2^11) and
// rounded to fp16, in the order [column][k step][quarter][8] of the right operand (SPLIT: the
// second halves behind). f: what a product is to be multiplied by; pos: the column's position,
// -1 for none. The code is kept short: a workgroup runs it once, from a cold cache.
template <int CODE, int HD, int GR, int NC, bool F32, bool SPLIT>
__device__ __forceinline__ void stage_queries(const Params& p, const Seq& s, int h, int c0,
                                              half_t* sq, float* f, int* pos) {
    using L = Layout<CODE, HD>;
    constexpr int N = HD / 16;
    const int G = p.H / p.KV, tid = threadIdx.x, lane = tid & 15, group = tid >> 4;
    const int ch = lane * N;
    const bool second = ch >= HD / 2;
    const int other = second ? ch - HD / 2 : ch + HD / 2;
    float x[NC][N], o[NC][N], co[NC][N], si[NC][N];
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
        const int c = GR * cc + group, r = (c0 + c) / G, g = (c0 + c) - r * G;
        const bool live = r < s.real;
        const int tok = s.tok0 + (live ? r : 0), at = s.past + (live ? r : 0);
        const int64_t x0 = (int64_t)tok * p.q_tok + (int64_t)(h * G + g) * HD;
        load_piece<N, F32>(p.q, x0 + ch, p.dtype, x[cc]);
        if (p.cos && p.pieces) {
            const int64_t k = min((int64_t)at, p.max_pos - 1) * (HD / 2) + (second ? other : ch);
            load_piece<N, F32>(p.q, x0 + other, p.dtype, o[cc]);
            load_piece<N, F32>(p.cos, k, p.dtype, co[cc]);
            load_piece<N, F32>(p.sin, k, p.dtype, si[cc]);
        }
        if (lane == 0) pos[c] = live ? at : -1;
    }
    float sc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sc[i] = p.ks[p.k_chan ? h * HD + ch + i : 0];
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
        const int c = GR * cc + group, r = (c0 + c) / G, g = (c0 + c) - r * G;
        const bool live = r < s.real;
        float rinv = 1.f;
        if (p.qw) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) ss += x[cc][i] * x[cc][i];
            rinv = 1.f / sqrtf(group_sum<16>(ss) / (float)HD + p.eps);
        }
        if (p.pieces) {
            if (p.qw) {
                float w[N];
                load_piece<N, F32>(p.qw, ch, p.dtype, w);
#pragma unroll
                for (int i = 0; i < N; ++i) x[cc][i] = x[cc][i] * rinv * w[i];
                if (p.cos) {
                    load_piece<N, F32>(p.qw, other, p.dtype, w);
#pragma unroll
                    for (int i = 0; i < N; ++i) o[cc][i] = o[cc][i] * rinv * w[i];
                }
            }
            if (p.cos) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    x[cc][i] = x[cc][i] * co[cc][i] + (second ? o[cc][i] : -o[cc][i]) * si[cc][i];
            }
        } else {  // any rotation: element by element
            const int at = s.past + (live ? r : 0);
            const int64_t x0 = (int64_t)(s.tok0 + (live ? r : 0)) * p.q_tok + (int64_t)(h * G + g) * HD;
            const int64_t prow = min((int64_t)at, p.max_pos - 1) * p.half;
            for (int i = 0; i < N; ++i) {
                const float v = query_elem(p, x0, prow, rinv, ch + i);
#pragma unroll
                for (int j = 0; j < N; ++j) x[cc][j] = j == i ? v : x[cc][j];
            }
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[cc][i] *= sc[i];
            top = fmaxf(top, fabsf(x[cc][i]));
        }
        top = group_max<16>(top);
        // A row of zeros, or with an infinity, is taken as it is.
        const int ex = top > 0.f && top < INFINITY ? max(-100, min(ilogbf(top), 116)) : 10;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float z = live ? ldexpf(x[cc][i], 10 - ex) : 0.f;
            const half_t hi = (half_t)z;
            const int at = c * HD + L::key_slot(ch + i);
            sq[at] = hi;
            if constexpr (SPLIT) sq[GR * NC * HD + at] = (half_t)(z - (float)hi);
        }
        if (lane == 0) f[c] = ldexpf(p.scale, ex - 10);
    }
    __syncthreads();
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

// Scores of the lane's 4 keys of a tile at `key` for a column at position pos, in units of
// log2(e): -inf where the column does not attend the key (later ones, behind the end, no page).
__device__ __forceinline__ void mask_scores(float (&x)[4], int key, int end) {
    const int q = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = key + 4 * q + i > end ? -INFINITY : x[i];
}

// exp2 of the scores about the column's reference, rounded to fp16 as the second product's
// operand (and, SPLIT, what the rounding left), added to the lane's sum.
template <bool SPLIT>
__device__ __forceinline__ void probabilities(const float (&x0)[4], const float (&x1)[4], float m,
                                              float& l, half8_t& p, half8_t& rest) {
    const float ref = m - kPBase;
    float a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = __builtin_amdgcn_exp2f(x0[i] - ref);
        b[i] = __builtin_amdgcn_exp2f(x1[i] - ref);
        l += a[i] + b[i];
    }
    p = pack_p(a, b);
    if constexpr (SPLIT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] -= (float)p[i];
            b[i] -= (float)p[4 + i];
        }
        rest = pack_p(a, b);
    }
}

__device__ __forceinline__ float max4(const float (&x)[4]) {
    return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
}
// Maximum and sum over the four quarters that share a column.
__device__ __forceinline__ float quarters_max(float v) {
    LanePair pr = swap16(v);
    pr = swap32(fmaxf(pr.a, pr.b));
    return fmaxf(pr.a, pr.b);
}
__device__ __forceinline__ float quarters_sum(float v) {
    LanePair pr = swap16(v);
    pr = swap32(pr.a + pr.b);
    return pr.a + pr.b;
}

#define ORTMI_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0)

// What a column's output is multiplied by, from its maximum and sum and the sink of its head.
template <bool F32, bool PAGED>
__device__ __forceinline__ float output_factor(const Params& p, int head, float m, float l) {
    float a = 1.f;
    if (PAGED && p.sink) {
        const float sk = load_one<F32>(p.sink, head, p.dtype) * 1.44269504088896341f;
        const float mm = fmaxf(m, sk);
        a = __builtin_amdgcn_exp2f(m - mm);
        l = l * a + __builtin_amdgcn_exp2f(sk - mm + kPBase);
    }
    return l != 0.f ? a / l : 0.f;
}

// N (2, 4 or 8) neighbouring channels of an output row, times their value scales vs; a factor
// of 0 gives zeros whatever they are.
template <int N, bool F32>
__device__ __forceinline__ void store_piece(const Params& p, int64_t at, const float (&v)[N],
                                            const float (&vs)[N], float inv) {
    float y[N];
#pragma unroll
    for (int j = 0; j < N; ++j) y[j] = inv != 0.f ? v[j] * inv * vs[j] : 0.f;
    if constexpr (F32) {
        float* o = static_cast<float*>(p.out) + at;
#pragma unroll
        for (int j = 0; j < N; j += 2) *reinterpret_cast<float2*>(o + j) = make_float2(y[j], y[j + 1]);
    } else {
        uint32_t w[N / 2];
        if (p.dtype == ORTMI_F16) {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                const half2_t z = {(half_t)y[2 * j], (half_t)y[2 * j + 1]};
                w[j] = __builtin_bit_cast(uint32_t, z);
            }
        } else {
#pragma unroll
            for (int j = 0; j < N / 2; ++j)
                w[j] = from_f32<uint16_t>(y[2 * j]) | ((uint32_t)from_f32<uint16_t>(y[2 * j + 1]) << 16);
        }
        uint16_t* o = static_cast<uint16_t*>(p.out) + at;
        if constexpr (N == 8) *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (N == 4) *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(o) = w[0];
    }
}
template <int N>
__device__ __forceinline__ void value_scales(const Params& p, int at, float (&vs)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) vs[j] = p.vs[p.v_chan ? at + j : 0];
}

// ----------------------------------------------------------------- token tiles --
template <int HD, bool F32>
struct TokenShared {
    union {
        __align__(16) half_t queries[2 * 16 * HD];
        __align__(16) float4_t out[2][HD / 16][64];    // two waves' outputs
        __align__(16) float rows[16 * kRowFloats<HD>];  // the tile's output
    };
    float f[16], inv[16];
    int pos[16];
    float m[4][16], l[4][16];
};

// One tile of columns 0 .. 15 over keys [k0, k1) of sequence s: range `split` of `nsplit`.
template <int CODE, int HD, bool F32, bool PAGED>
__device__ __forceinline__ void token_tile(const Params& p, const Seq& s, int b, int h, int k0,
                                           int k1, int split, int nsplit, TokenShared<HD, F32>& sh) {
    using L = Layout<CODE, HD>;
    constexpr int KS = L::KS, MT = L::MT;
    const int lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
    const int wave = uniform(threadIdx.x >> 6);
    const int G = p.H / p.KV;

    // The first block's rows are on their way while the queries are staged.
    const Source<CODE, HD, PAGED> src(p, b, h, k0, k1);
    int kb = k0 + 32 * wave;
    int2 sl = src.slots(kb), sl_n = src.slots(kb + 128);
    Block<CODE, HD> cur, nxt;
    if (kb < k1) src.load(kb, sl, cur);
    stage_queries<CODE, HD, 16, 1, F32, true>(p, s, h, 0, sh.queries, sh.f, sh.pos);
    const half8_t* sq = reinterpret_cast<const half8_t*>(sh.queries);
    half8_t Q[KS], QL[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        Q[ks] = sq[(n * KS + ks) * 4 + q];
        QL[ks] = sq[((16 + n) * KS + ks) * 4 + q];
    }
    const float f = sh.f[n];
    const int pos = sh.pos[n];
    const int first = s.past;  // the lowest position of the tile

    float4_t O[MT];
    float m = kNone, l = 0.f;
#pragma unroll
    for (int d = 0; d < MT; ++d) O[d] = float4_t{0.f, 0.f, 0.f, 0.f};
    for (; kb < k1; kb += 128) {
        const int2 sl_c = sl;
        if (kb + 128 < k1) {
            src.load(kb + 128, sl_n, nxt);
            sl = sl_n;
            sl_n = src.slots(kb + 256);
        }
        float x[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float4_t S{0.f, 0.f, 0.f, 0.f}, SL{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const half8_t a = L::key_step(cur.k[t], ks);
                S = ORTMI_MFMA(a, Q[ks], S);
                SL = ORTMI_MFMA(a, QL[ks], SL);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) x[t][i] = (S[i] + SL[i]) * f;
        }
        if (kb + 31 > first || kb + 32 > k1 || (PAGED && (sl_c.x < 0 || sl_c.y < 0))) {
            const int end = min(pos, k1 - 1);
            mask_scores(x[0], kb, PAGED && sl_c.x < 0 ? -1 : end);
            mask_scores(x[1], kb + 16, PAGED && sl_c.y < 0 ? -1 : end);
        }
        const float top = fmaxf(max4(x[0]), max4(x[1]));
        if (__any(top > m + kSlack)) {
            const float mm = fmaxf(m, quarters_max(fmaxf(top, kNone)));
            const float a = __builtin_amdgcn_exp2f(m - mm);
            m = mm;
            l *= a;
#pragma unroll
            for (int d = 0; d < MT; ++d) O[d] *= a;
        }
        half8_t P, PL;
        probabilities<F32>(x[0], x[1], m, l, P, PL);
#pragma unroll
        for (int u = 0; u < MT / 2; ++u) {
            half8_t a[2];
            L::value_steps(cur.v, u, a[0], a[1]);
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                O[2 * u + d] = ORTMI_MFMA(a[d], P, O[2 * u + d]);
                if constexpr (F32) O[2 * u + d] = ORTMI_MFMA(a[d], PL, O[2 * u + d]);
            }
        }
        cur = nxt;
    }

    // The four waves: maxima and sums, then outputs in two steps through LDS.
    l = quarters_sum(l);
    if (q == 0) {
        sh.m[wave][n] = m;
        sh.l[wave][n] = l;
    }
    __syncthreads();
    float mm = kNone, sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sh.m[w][n]);
#pragma unroll
    for (int w = 0; w < 4; ++w) sum += sh.l[w][n] * __builtin_amdgcn_exp2f(sh.m[w][n] - mm);
    const float a = __builtin_amdgcn_exp2f(m - mm);
#pragma unroll
    for (int d = 0; d < MT; ++d) O[d] *= a;
#pragma unroll
    for (int step = 2; step; step >>= 1) {
        if (wave >= step && wave < 2 * step) {
#pragma unroll
            for (int d = 0; d < MT; ++d) sh.out[wave - step][d][lane] = O[d];
        }
        __syncthreads();
        if (wave < step) {
#pragma unroll
            for (int d = 0; d < MT; ++d) O[d] += sh.out[wave][d][lane];
        }
        __syncthreads();
    }
    // Output rows by all waves. A partial row stays unscaled, with its maximum and sum.
    if (wave == 0) {
        float* row = sh.rows + n * kRowFloats<HD>;
#pragma unroll
        for (int d = 0; d < MT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) row[L::value_channel(4 * q + i, d)] = O[d][i];
        const int r = n / G, head = h * G + (n - r * G);
        if (q == 0 && r < s.real) {
            const int64_t orow = (int64_t)(s.tok0 + r) * p.H + head;
            if (nsplit > 1) {
                p.ml[(orow * p.nsplit + split) * 2] = mm;
                p.ml[(orow * p.nsplit + split) * 2 + 1] = sum;
            } else {
                sh.inv[n] = output_factor<F32, PAGED>(p, head, mm, sum);
            }
        }
    }
    __syncthreads();
    constexpr int kPieces = HD / 4;  // of a row: four channels a thread and step
    for (int i = threadIdx.x; i < 16 * kPieces; i += 256) {
        const int c = i / kPieces, ch = 4 * (i % kPieces), r = c / G;
        if (r >= s.rows) break;
        const int64_t orow = (int64_t)(s.tok0 + r) * p.H + h * G + (c - r * G);
        const float4_t v = *reinterpret_cast<const float4_t*>(sh.rows + c * kRowFloats<HD> + ch);
        if (nsplit > 1 && r < s.real) {
            *reinterpret_cast<float4_t*>(p.part + (orow * p.nsplit + split) * HD + ch) = v;
        } else if (nsplit <= 1 || split == 0) {
            const float y[4] = {v[0], v[1], v[2], v[3]};
            float vs[4];
            value_scales(p, h * HD + ch, vs);
            store_piece<4, F32>(p, orow * HD + ch, y, vs, r < s.real ? sh.inv[c] : 0.f);
        }
    }
}

// ---------------------------------------------------------------- prompt tiles --
template <int CODE, int HD, bool F32>
struct PromptShared {
    static constexpr int kNT = F32 ? 1 : 2, kCols = 64 * kNT;
    struct Blocks {  // two blocks of 64 keys: [key tile][k step], [half][channel tile], by lane
        half8_t k[2][4][HD / 32][64], v[2][2][HD / 16][64];
    };
    union {
        __align__(16) half_t queries[(F32 ? 2 : 1) * kCols * HD];
        Blocks team[2];
        __align__(16) float4_t out[4][HD / 16][kNT][64];  // the second team's outputs
    };
    float f[kCols], m[kCols], l[kCols];
    int pos[kCols];
};

// One tile of columns c0 .. over keys [k0, k1) of sequence s: range `split` of `nsplit`.
template <int CODE, int HD, bool F32, bool PAGED>
__device__ __forceinline__ void prompt_tile(const Params& p, const Seq& s, int b, int h, int c0,
                                            int k0, int k1, int split, int nsplit,
                                            PromptShared<CODE, HD, F32>& sh) {
    using L = Layout<CODE, HD>;
    using SH = PromptShared<CODE, HD, F32>;
    constexpr int KS = L::KS, MT = L::MT, NT = SH::kNT, UH = (MT / 2 + 1) / 2;
    const int lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
    const int team = uniform(threadIdx.x >> 8), wave = uniform(threadIdx.x >> 6) & 3;
    const int G = p.H / p.KV;
    const Source<CODE, HD, PAGED> src(p, b, h, k0, k1);
    auto& blocks = sh.team[team];

    // Of a block at kb a wave decodes key tile `wave`, and of the values of its half of the
    // keys (wave / 2) half of the channel tiles.
    uint32_t rk[L::KW], rv[8][L::VW];
    int slot[4], slot_n[4];
    auto slots = [&](int kb, int (&sl)[4]) {
#pragma unroll
        for (int t = 0; t < 4; ++t) sl[t] = src.slot(kb + 16 * t);
    };
    auto load = [&](int kb, const int (&sl)[4]) {
        const int s0 = sl[0], s1 = sl[1], s2 = sl[2], s3 = sl[3];
        const int a = wave & 2 ? s2 : s0, c = wave & 2 ? s3 : s1;
        src.keys(kb + 16 * wave, wave & 1 ? c : a, rk);
        src.values(kb + 32 * (wave >> 1), a, c, rv);
    };
    auto decode = [&](int buf) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) blocks.k[buf][wave][ks][lane] = L::key_step(rk, ks);
#pragma unroll
        for (int u = 0; u < MT / 2; ++u)
            if ((u < UH) == !(wave & 1)) {
                half8_t a, c;
                L::value_steps(rv, u, a, c);
                blocks.v[buf][wave >> 1][2 * u][lane] = a;
                blocks.v[buf][wave >> 1][2 * u + 1][lane] = c;
            }
    };

    int kb = k0 + 64 * team;
    slots(kb, slot);
    if (kb < k1) load(kb, slot);
    stage_queries<CODE, HD, 32, 2 * NT, F32, F32>(p, s, h, c0, sh.queries, sh.f, sh.pos);
    const half8_t* sq = reinterpret_cast<const half8_t*>(sh.queries);
    half8_t Q[NT][KS], QL[F32 ? NT : 1][KS];
    float f[NT];
    int pos[NT];
    const int cw = 16 * NT * wave;  // the wave's columns
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            Q[t][ks] = sq[((cw + 16 * t + n) * KS + ks) * 4 + q];
            if constexpr (F32) QL[t][ks] = sq[((SH::kCols + cw + 16 * t + n) * KS + ks) * 4 + q];
        }
        f[t] = sh.f[cw + 16 * t + n];
        pos[t] = sh.pos[cw + 16 * t + n];
    }
    // The lowest and the highest position of the wave's columns (none: the latter is -1).
    const int first = s.past + (c0 + cw) / G;
    const int last = (c0 + cw) / G < s.real
                         ? s.past + min((c0 + cw + 16 * NT - 1) / G, s.real - 1) : -1;

    float4_t O[MT][NT];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = kNone;
        l[t] = 0.f;
#pragma unroll
        for (int d = 0; d < MT; ++d) O[d][t] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    __syncthreads();  // the queries are read: the blocks take their place
    if (kb < k1) decode(0);
    slots(kb + 128, slot_n);
    if (kb + 128 < k1) load(kb + 128, slot_n);
    __syncthreads();
    int buf = 0;
    for (int first_kb = k0; first_kb < k1; first_kb += 128, kb += 128, buf ^= 1) {
        const int sl[4] = {slot[0], slot[1], slot[2], slot[3]};
        if (kb + 128 < k1) {
            decode(buf ^ 1);
#pragma unroll
            for (int t = 0; t < 4; ++t) slot[t] = slot_n[t];
            slots(kb + 256, slot_n);
            if (kb + 256 < k1) load(kb + 256, slot_n);
        }
        if (kb <= last && kb < k1) {
            float x[NT][4][4];
#pragma unroll
            for (int t4 = 0; t4 < 4; ++t4) {
                float4_t S[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) S[t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const half8_t a = blocks.k[buf][t4][ks][lane];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        S[t] = ORTMI_MFMA(a, Q[t][ks], S[t]);
                        if constexpr (F32) S[t] = ORTMI_MFMA(a, QL[t][ks], S[t]);
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[t][t4][i] = S[t][i] * f[t];
            }
            const bool gone = PAGED && (sl[0] < 0 || sl[1] < 0 || sl[2] < 0 || sl[3] < 0);
            if (kb + 63 > first || kb + 64 > k1 || gone) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int t4 = 0; t4 < 4; ++t4)
                        mask_scores(x[t][t4], kb + 16 * t4,
                                    PAGED && sl[t4] < 0 ? -1 : min(pos[t], k1 - 1));
            }
            bool grow = false;
            float top[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                top[t] = fmaxf(fmaxf(max4(x[t][0]), max4(x[t][1])), fmaxf(max4(x[t][2]), max4(x[t][3])));
                grow |= top[t] > m[t] + kSlack;
            }
            if (__any(grow)) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const float mm = fmaxf(m[t], quarters_max(fmaxf(top[t], kNone)));
                    const float a = __builtin_amdgcn_exp2f(m[t] - mm);
                    m[t] = mm;
                    l[t] *= a;
#pragma unroll
                    for (int d = 0; d < MT; ++d) O[d][t] *= a;
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                half8_t P[NT], PL[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    probabilities<F32>(x[t][2 * j], x[t][2 * j + 1], m[t], l[t], P[t], PL[t]);
#pragma unroll
                for (int d = 0; d < MT; ++d) {
                    const half8_t a = blocks.v[buf][j][d][lane];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        O[d][t] = ORTMI_MFMA(a, P[t], O[d][t]);
                        if constexpr (F32) O[d][t] = ORTMI_MFMA(a, PL[t], O[d][t]);
                    }
                }
            }
        }
        __syncthreads();
    }

    // The second team's outputs to the first, which writes them: a lane's neighbouring channels
    // at once.
    if (team) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float sum = quarters_sum(l[t]);
            if (q == 0) {
                sh.m[cw + 16 * t + n] = m[t];
                sh.l[cw + 16 * t + n] = sum;
            }
#pragma unroll
            for (int d = 0; d < MT; ++d) sh.out[wave][d][t][lane] = O[d][t];
        }
    }
    __syncthreads();
    if (team) return;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float m1 = sh.m[cw + 16 * t + n], mm = fmaxf(m[t], m1);
        const float a0 = __builtin_amdgcn_exp2f(m[t] - mm), a1 = __builtin_amdgcn_exp2f(m1 - mm);
        m[t] = mm;
        l[t] = quarters_sum(l[t]) * a0 + sh.l[cw + 16 * t + n] * a1;
#pragma unroll
        for (int d = 0; d < MT; ++d) O[d][t] = O[d][t] * a0 + sh.out[wave][d][t][lane] * a1;
    }
    constexpr int W = HD == 128 ? 8 : 4;  // (HD 96: and two of the last third)
    int64_t row[NT];
    float inv[NT];
    bool live[NT], partial[NT], any[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int c = c0 + cw + 16 * t + n, r = c / G, head = h * G + (c - r * G);
        row[t] = (int64_t)(s.tok0 + r) * p.H + head;
        live[t] = r < s.real;
        partial[t] = nsplit > 1 && live[t];
        any[t] = r < s.rows && (live[t] || nsplit <= 1 || split == 0);
        if (partial[t] && q == 0) {
            p.ml[(row[t] * p.nsplit + split) * 2] = m[t];
            p.ml[(row[t] * p.nsplit + split) * 2 + 1] = l[t];
        }
        inv[t] = live[t] ? output_factor<F32, PAGED>(p, head, m[t], l[t]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int ch = L::value_channel(4 * q + i, 0), ch2 = L::value_channel(4 * q + i, MT - 2);
        float vs[W], vs2[2];
        value_scales(p, h * HD + ch, vs);
        if constexpr (HD == 96) value_scales(p, h * HD + ch2, vs2);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (!any[t]) continue;
            float v[W];
#pragma unroll
            for (int j = 0; j < W; ++j) v[j] = O[j][t][i];
            const float z[2] = {O[MT - 2][t][i], O[MT - 1][t][i]};
            if (partial[t]) {
                float* part = p.part + (row[t] * p.nsplit + split) * HD;
#pragma unroll
                for (int j = 0; j < W; j += 4)
                    *reinterpret_cast<float4_t*>(part + ch + j) = float4_t{v[j], v[j + 1], v[j + 2], v[j + 3]};
                if constexpr (HD == 96)
                    *reinterpret_cast<float2*>(part + ch2) = make_float2(z[0], z[1]);
            } else {
                store_piece<W, F32>(p, row[t] * HD + ch, v, vs, inv[t]);
                if constexpr (HD == 96) store_piece<2, F32>(p, row[t] * HD + ch2, z, vs2, inv[t]);
            }
        }
    }
}

// -------------------------------------------------------------------- new rows --
// append_row in pieces: 16 lanes a row, each a sixteenth of its channels, which lie side by
// side as their partners in the rotation do.
template <int CODE, int HD, bool F32, bool PAGED>
__device__ __forceinline__ void append_piece(const Params& p, int b, const Seq& s, int r, int h,
                                             bool is_v, int lane) {
    constexpr int N = HD / 16, RB = row_bytes(CODE, HD);
    const int pos = s.past + r, c0 = lane * N;
    const int64_t row = cache_row<PAGED>(p, b, h, pos);
    const int64_t x0 = (int64_t)(s.tok0 + r) * p.kv_tok + (int64_t)h * HD;
    const void* src = is_v ? p.v : p.k;
    const bool rope = !is_v && p.cos, second = c0 >= HD / 2;
    float x[N], o[N], co[N], si[N], w[N], wo[N];
    load_piece<N, F32>(src, x0 + c0, p.dtype, x);
    const int c1 = second ? c0 - HD / 2 : c0 + HD / 2;  // of the partners
    if (rope) {
        const int64_t at = min((int64_t)pos, p.max_pos - 1) * (HD / 2) + (second ? c1 : c0);
        load_piece<N, F32>(src, x0 + c1, p.dtype, o);
        load_piece<N, F32>(p.cos, at, p.dtype, co);
        load_piece<N, F32>(p.sin, at, p.dtype, si);
    }
    double rinv = 1.0;
    const bool norm = p.kw && !is_v;
    if (p.kw) {  // (a value row's lanes go along)
        double ss = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) ss += (double)x[i] * (double)x[i];
#pragma unroll
        for (int k = 8; k; k >>= 1) ss += __shfl_xor(ss, k, 64);
        rinv = 1.0 / sqrt(ss / HD + (double)p.eps);
        load_piece<N, F32>(p.kw, c0, p.dtype, w);
        load_piece<N, F32>(p.kw, c1, p.dtype, wo);
    }
    if (row < 0) return;
    const float* sc = (is_v ? p.vs : p.ks);
    const bool chan = is_v ? p.v_chan : p.k_chan;
    uint32_t u[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        double a = x[i];
        if (norm) a = a * rinv * (double)w[i];
        if (rope) {
            double e = o[i];
            if (norm) e = e * rinv * (double)wo[i];
            const double f = a * (double)co[i], g = e * (double)si[i];
            a = second ? f + g : f - g;
        }
        u[i] = encode(a, sc[chan ? h * HD + c0 + i : 0], CODE);
    }
    uint8_t* dst = (is_v ? p.vc : p.kc) + row * RB + (CODE == kInt4 ? c0 / 2 : c0);
    if constexpr (CODE == kInt4) {
        uint32_t v = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) v |= u[i] << (4 * i);
        if constexpr (N == 8) *reinterpret_cast<uint32_t*>(dst) = v;
        else if constexpr (N == 4) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)v;
        else
#pragma unroll
            for (int i = 0; i < N / 2; ++i) dst[i] = (uint8_t)(v >> (8 * i));
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2)
            *reinterpret_cast<uint16_t*>(dst + i) = (uint16_t)(u[i] | (u[i + 1] << 8));
    }
}

// Rows r0 .. r1 - 1 of sequence s, key and value of one kv head, by the workgroup.
template <int CODE, int HD, bool F32, bool PAGED>
__device__ __forceinline__ void append_rows(const Params& p, int b, const Seq& s, int r0, int r1,
                                            int h) {
    const int lane = threadIdx.x & 15;
    for (int i = 2 * r0 + (int)(threadIdx.x >> 4); i < 2 * r1; i += (int)(blockDim.x >> 4)) {
        if (p.pieces) append_piece<CODE, HD, F32, PAGED>(p, b, s, i >> 1, h, i & 1, lane);
        else append_row<PAGED>(p, b, s, i >> 1, h, i & 1, lane);
    }
}

// The last sequence that starts at or before token `tok`, and whether it has the token.
__device__ __forceinline__ bool sequence_of_token(const Params& p, int tok, int& b, Seq& s) {
    int lo = 0, hi = p.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p.cum[mid] <= tok) lo = mid;
        else hi = mid;
    }
    b = lo;
    s = sequence<true>(p, lo);
    return tok >= s.tok0 && tok < s.tok0 + s.rows;
}

// The prompt tiles of the sequences with more than 16 columns, in order, by one wave. Ranges
// of tokens are clamped to the call's (sequence()), and at most max_tiles are written.
__device__ __forceinline__ void list_tiles(const Params& p) {
    const int lane = threadIdx.x & 63, G = p.H / p.KV, w = prompt_width(p.dtype);
    int base = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        const int b = b0 + lane;
        const int cols = b < p.B ? sequence<true>(p, b).rows * G : 0;
        const int n = cols > 16 ? (cols + w - 1) / w : 0;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(incl, o, 64);
            if (lane >= o) incl += v;
        }
        const int first = base + incl - n;
        for (int i = 0; i < n && first + i < p.max_tiles; ++i) p.tiles[first + i] = make_int2(b, w * i);
        base += __shfl(incl, 63, 64);
    }
    if (lane == 0) *p.tile_count = min(base, p.max_tiles);
}

// New keys and values into the cache: 16 lanes per (token, kv head, key or value). Pages: the
// first workgroup lists the tiles.
template <int CODE, int HD, bool F32, bool PAGED>  // HD 0: any
__global__ __launch_bounds__(256) void append_kernel(Params p) {
    int64_t item = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if constexpr (PAGED) {
        if (blockIdx.x == 0) {
            if (threadIdx.x < 64 && p.tiles) list_tiles(p);
            return;
        }
        item -= 16;
    }
    const int per = 2 * p.KV;
    const int64_t tok = item / per;
    if (tok >= p.T) return;
    const int hv = (int)(item % per);
    int b;
    Seq s;
    if constexpr (PAGED) {
        if (!sequence_of_token(p, (int)tok, b, s)) return;
    } else {
        b = (int)(tok / p.S);
        s = sequence<false>(p, b);
    }
    const int r = (int)tok - s.tok0;
    if (r >= s.real) return;
    if constexpr (HD > 0)
        append_piece<CODE, HD, F32, PAGED>(p, b, s, r, hv % p.KV, hv >= p.KV, threadIdx.x & 15);
    else
        append_row<PAGED>(p, b, s, r, hv % p.KV, hv >= p.KV, threadIdx.x & 15);
}

// A tile that attends nothing: padded rows.
template <int HD, bool F32>
__device__ __forceinline__ void zero_rows(const Params& p, const Seq& s, int h, int c0, int cols) {
    const int G = p.H / p.KV;
    for (int i = threadIdx.x; i < cols * HD; i += blockDim.x) {
        const int c = c0 + i / HD, r = c / G;
        if (r >= s.rows) break;
        const int64_t o = ((int64_t)(s.tok0 + r) * p.H + h * G + (c - r * G)) * HD + i % HD;
        if constexpr (F32) static_cast<float*>(p.out)[o] = 0.f;
        else static_cast<uint16_t*>(p.out)[o] = 0;
    }
}

// Slabs. Workgroups: (range, tile, slab), the slab running fastest (slabs of one residue
// modulo 8 then stay on one XCD). Later tiles, which see more keys, come first. Where a
// sequence's columns are one tile, the workgroup whose range holds the new rows writes them to
// the cache itself.
template <int CODE, int HD, bool F32, bool PROMPT>
__global__ __launch_bounds__(PROMPT ? 512 : 256, 2) void tile_kernel(Params p) {
    using SH = std::conditional_t<PROMPT, PromptShared<CODE, HD, F32>, TokenShared<HD, F32>>;
    __shared__ SH sh;
    constexpr int kCols = PROMPT ? prompt_width(F32 ? ORTMI_F32 : ORTMI_F16) : 16;
    const int slabs = p.B * p.KV;
    const int split = blockIdx.x / (slabs * p.ntile), rem = blockIdx.x % (slabs * p.ntile);
    const int tile = p.ntile - 1 - rem / slabs, slab = rem % slabs, b = slab / p.KV, h = slab % p.KV;
    const Seq s = sequence<false>(p, b);
    const int G = p.H / p.KV, c0 = tile * kCols;
    if (c0 / G >= s.real) {
        if (split == 0) zero_rows<HD, F32>(p, s, h, c0, kCols);
        return;
    }
    const int kend = s.keys_to((min(c0 + kCols, s.rows * G) - 1) / G, p.limit);
    const int k0 = split * p.chunk, k1 = min(k0 + p.chunk, kend);
    if (k0 >= kend) return;
    if (p.fused) {
        append_rows<CODE, HD, F32, false>(p, b, s, max(k0 - s.past, 0), min(k1 - s.past, s.real), h);
        __syncthreads();
    }
    const int nsplit = (kend + p.chunk - 1) / p.chunk;
    if constexpr (PROMPT)
        prompt_tile<CODE, HD, F32, false>(p, s, b, h, c0, k0, k1, split, nsplit, sh);
    else
        token_tile<CODE, HD, F32, false>(p, s, b, h, k0, k1, split, nsplit, sh);
}

// Pages, sequences of at most 16 columns: workgroups (range, sequence, kv head).
template <int CODE, int HD, bool F32>
__global__ __launch_bounds__(256, 2) void page_token_kernel(Params p) {
    __shared__ TokenShared<HD, F32> sh;
    const int slabs = p.B * p.KV, split = blockIdx.x / slabs, slab = blockIdx.x % slabs;
    const int b = slab / p.KV, h = slab % p.KV, G = p.H / p.KV;
    const Seq s = sequence<true>(p, b);
    if (s.rows == 0 || s.rows * G > 16) return;
    const int kend = s.keys_to(s.rows - 1, p.limit);
    const int k0 = split * p.chunk, k1 = min(k0 + p.chunk, kend);
    if (k0 >= kend) return;
    token_tile<CODE, HD, F32, true>(p, s, b, h, k0, k1, split, (kend + p.chunk - 1) / p.chunk, sh);
}

// Pages, the other sequences: a workgroup for each (range, listed tile, kv head), those past
// the list's end with nothing to do.
template <int CODE, int HD, bool F32>
__global__ __launch_bounds__(512, 2) void page_tile_kernel(Params p) {
    constexpr int kCols = prompt_width(F32 ? ORTMI_F32 : ORTMI_F16);
    __shared__ PromptShared<CODE, HD, F32> sh;
    const int G = p.H / p.KV, per = p.max_tiles * p.KV;
    const int split = blockIdx.x / per, rem = blockIdx.x % per, h = rem % p.KV, i = rem / p.KV;
    if (i >= *p.tile_count) return;
    const int2 tl = p.tiles[i];
    const int b = tl.x, c0 = tl.y;
    const Seq s = sequence<true>(p, b);
    const int kend = s.keys_to((min(c0 + kCols, s.rows * G) - 1) / G, p.limit);
    const int k0 = split * p.tile_chunk, k1 = min(k0 + p.tile_chunk, kend);
    if (k0 >= kend) return;
    prompt_tile<CODE, HD, F32, true>(p, s, b, h, c0, k0, k1, split,
                                     (kend + p.tile_chunk - 1) / p.tile_chunk, sh);
}

// New rows and attention for one code; in kvq_int8.hip, kvq_int4.hip and kvq_fp8.hip.
int tiles_int8(const Params& p, bool paged, hipStream_t st);
int tiles_int4(const Params& p, bool paged, hipStream_t st);
int tiles_fp8(const Params& p, bool paged, hipStream_t st);

template <int CODE, int HD, bool F32>
int launch_tiles(const Params& p, bool paged, hipStream_t st) {
    const int G = p.H / p.KV;
    const dim3 rows((unsigned)(((int64_t)p.T * 2 * p.KV + 15) / 16 + (paged ? 1 : 0)));
    if (p.pieces && !p.fused) {
        if (paged) hipLaunchKernelGGL((append_kernel<CODE, HD, F32, true>), rows, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((append_kernel<CODE, HD, F32, false>), rows, dim3(256), 0, st, p);
        if (int rc = check_launch("kv append")) return rc;
    }
    if (!paged) {
        const dim3 grid((unsigned)(p.B * p.KV * p.ntile * p.nsplit));
        if (p.S * G <= 16)
            hipLaunchKernelGGL((tile_kernel<CODE, HD, F32, false>), grid, dim3(256), 0, st, p);
        else
            hipLaunchKernelGGL((tile_kernel<CODE, HD, F32, true>), grid, dim3(512), 0, st, p);
        return check_launch("kv tiles");
    }
    if (G <= 16) {
        hipLaunchKernelGGL((page_token_kernel<CODE, HD, F32>),
                           dim3((unsigned)(p.B * p.KV * p.nsplit)), dim3(256), 0, st, p);
        if (int rc = check_launch("kv page tokens")) return rc;
    }
    if ((int64_t)p.T * G <= 16) return ORTMI_OK;  // no sequence has more than 16 columns
    hipLaunchKernelGGL((page_tile_kernel<CODE, HD, F32>),
                       dim3((unsigned)(p.max_tiles * p.KV * p.tile_nsplit)), dim3(512), 0, st, p);
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
