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
// output. Except in prompt tiles of head size 128, the query row is taken as two fp16 halves, 22
// bits; fp32 tensors take the probabilities as two halves too.
//
// Token tiles: 16 columns. A workgroup's 4 waves take every fourth block of 32 keys of its
// range and are joined at the end; keys and values go from memory into registers, where each
// wave decodes its own. Memory binds it: 4 sequences of 131072 int8 keys, 8 heads of 128, 190
// us, 5.65 TB/s; 32 of 256 to 8192 in pages 64 us, 4.2 TB/s. A unit has about 8 us around its
// loop (its place 2.5, rotated queries 2.3, the first loads, the join 1.3), which is all of a
// short call: 512 keys, 12 us.
//
// Prompt tiles: 128 columns (fp32 64), 32 a wave, by two teams of 4 waves that take every other
// block of 64 keys and are joined at the end. A team decodes its block together into LDS, a
// quarter each, in the order that the products read: decoded once for 128 columns. Two buffers
// a team, so that one barrier for two blocks suffices; the second team fills the waits of the
// first, which the registers (220 of 256 at two waves a SIMD) leave no other wave for. One team
// a workgroup and two workgroups a CU instead: a 2048-token prompt 76 us, not 71 (34.4 GFLOP,
// 485 TFLOP/s; at 8160 keys before it 676). 128 keys take 2.1 to 2.7 us of a CU, issued vector
// instructions beside matrix cores 24 % busy, and a unit has 12 us around its loop.
#pragma once

#include <algorithm>

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
    const int32_t* table;
    int k0, k1;
    uint32_t stride, kat, kat2, vat, vat2;

    __device__ __forceinline__ Source(const Params& p_, int b, int h, int k0_, int k1_)
        : p(p_), table(p_.bt + (PAGED ? (int64_t)b * p_.maxb : 0)), k0(k0_), k1(k1_) {
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
    // Logical block of a key: key / blk, both in units of 16 (blk_mul is 2^blk_shift / (blk / 16),
    // rounded up: exact for 27 bits).
    __device__ __forceinline__ uint32_t logical(int key) const {
        return (uint32_t)(((uint64_t)((uint32_t)key >> 4) * p.blk_mul) >> p.blk_shift);
    }
    // The block table's entry for the key tile at `key`, its last one behind the table's end: a
    // load nothing waits for until the entry is used.
    __device__ __forceinline__ int entry(int key) const {
        if constexpr (!PAGED) return 0;
        return table[min(logical(key), (uint32_t)p.maxb - 1)];
    }
    // Whether a key tile with this entry has no block.
    __device__ __forceinline__ bool gone(int key, int id) const {
        if constexpr (!PAGED) return false;
        return (logical(key) >= (uint32_t)p.maxb) | ((uint32_t)id >= (uint32_t)p.nblk);
    }
    // Slot of the key tile at `key`: -1 behind the end and where there is no block.
    __device__ __forceinline__ int slot(int key, int id) const {
        if constexpr (!PAGED) return -1;
        const bool is = (key < k1) & !gone(key, id);
        return is ? id * p.blk + (key - (int)logical(key) * p.blk) : -1;
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
    __device__ __forceinline__ int2 ids(int kb) const { return make_int2(entry(kb), entry(kb + 16)); }
    __device__ __forceinline__ int2 slots(int kb, int2 id) const {
        return make_int2(slot(kb, id.x), slot(kb + 16, id.y));
    }
    __device__ __forceinline__ void load(int kb, int2 sl, Block<CODE, HD>& o) const {
        keys(kb, sl.x, o.k[0]);
        keys(kb + 16, sl.y, o.k[1]);
        values(kb, sl.x, sl.y, o.v);
    }
};

template <int HD>
constexpr int kRowFloats = HD + 4;  // of a row in LDS: four more than a multiple of the banks

// Four consecutive elements of a row, 8-byte aligned (fp32: 16). Loads and conversions are
// apart: the conversion's branch on the type would otherwise wait for each load before the next
// is issued.
template <bool F32>
struct Piece {
    std::conditional_t<F32, uint4, uint2> w;
    __device__ __forceinline__ void load(const void* base, int64_t at) {
        w = *reinterpret_cast<const decltype(w)*>(static_cast<const uint8_t*>(base) + at * (F32 ? 4 : 2));
    }
    template <bool HALF>
    __device__ __forceinline__ float get(int i) const {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&w);
        if constexpr (F32) return __builtin_bit_cast(float, u[i]);
        else if constexpr (HALF) return (float)as_half2(u[i / 2])[i & 1];
        else return to_f32((uint16_t)(u[i / 2] >> (16 * (i & 1))));
    }
};
// New rows are taken by groups of lanes, each with four channels of the first half of the row
// and their partners in the rotation, four of the second: 8 lanes at head size 64, 16 at 128,
// 12 of 16 at 96.
template <int HD>
constexpr int kRowLanes = HD == 64 ? 8 : 16;
// N scales from element `at` on, or one.
template <int N>
__device__ __forceinline__ void load_scales(const float* base, bool chan, int at, float (&x)[N]) {
    if (chan) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = base[at + i];
    } else {
        const float one = base[0];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = one;
    }
}

template <bool F32>
__device__ __forceinline__ float load_one(const void* base, int64_t at, int dtype) {
    if constexpr (F32) return static_cast<const float*>(base)[at];
    const uint16_t u = static_cast<const uint16_t*>(base)[at];
    return dtype == ORTMI_F16 ? (float)__builtin_bit_cast(half_t, u) : to_f32(u);
}

// The query rows of columns c0 .. c0 + COLS - 1 into LDS: (normalised and) rotated, times the key
// scales, brought to [2^10, 2^11) and rounded to fp16, in the order [column][k step][quarter][8]
// of the right operand (SPLIT: the second halves behind). f: what a product is to be multiplied
// by; pos: the column's position, -1 for none. Behind sq's rows is room for as many of fp32.
template <int CODE, int HD, int COLS, int THREADS, bool F32, bool SPLIT>
__device__ __forceinline__ void stage_queries(const Params& p, const Seq& s, int h, int c0,
                                              half_t* sq, float* f, int* pos) {
    using L = Layout<CODE, HD>;
    constexpr int W = kRowLanes<HD>, GR = std::min(COLS, THREADS / W), NC = COLS / GR;
    const int G = p.H / p.KV, lane = threadIdx.x % W;
    const int group = min((int)threadIdx.x / W, GR - 1);
    const bool on = lane < HD / 8 && (int)threadIdx.x < GR * W;
    const int ch = lane < HD / 8 ? 4 * lane : 0, hi = ch + HD / 2;
    Piece<F32> x0[NC], x1[NC], co[NC], si[NC], w0, w1;
    const bool rope = p.cos && p.pieces;
    if (p.qw && p.pieces) {
        w0.load(p.qw, ch);
        w1.load(p.qw, hi);
    }
    float s0[4], s1[4];
    load_scales<4>(p.ks, p.k_chan, h * HD + ch, s0);
    load_scales<4>(p.ks, p.k_chan, h * HD + hi, s1);
    // Column GR cc + group is head g of the group, row r; -1: a row that does not exist.
    int g = (c0 + group) % G, r = (c0 + group) / G;
    const int dg = GR % G, dr = GR / G;
    int64_t from[NC];
    int at[NC];
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
        const int row = r < s.real ? r : 0;
        at[cc] = s.past + row;
        from[cc] = (int64_t)(s.tok0 + row) * p.q_tok + (int64_t)(h * G + g) * HD;
        x0[cc].load(p.q, from[cc] + ch);
        x1[cc].load(p.q, from[cc] + hi);
        if (rope) {
            const int64_t k = min((int64_t)at[cc], p.max_pos - 1) * (HD / 2) + ch;
            co[cc].load(p.cos, k);
            si[cc].load(p.sin, k);
        }
        if (r >= s.real) at[cc] = -1;
        r += dr;
        g += dg;
        if (g >= G) {
            g -= G;
            ++r;
        }
    }
    auto stage = [&](auto half) {
        constexpr bool HALF = decltype(half)::value;
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) {
            const int c = GR * cc + group;
            float x[8], rinv = 1.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = x0[cc].template get<HALF>(i);
                x[4 + i] = x1[cc].template get<HALF>(i);
            }
            if (p.qw) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
                ss = group_sum<W>(lane < HD / 8 ? ss : 0.f);
                rinv = 1.f / sqrtf(ss / (float)HD + p.eps);
            }
            if (p.pieces) {
                if (p.qw) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[i] = x[i] * rinv * w0.template get<HALF>(i);
                        x[4 + i] = x[4 + i] * rinv * w1.template get<HALF>(i);
                    }
                }
                if (rope) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float a = x[i], b = x[4 + i];
                        const float cv = co[cc].template get<HALF>(i), sv = si[cc].template get<HALF>(i);
                        x[i] = a * cv - b * sv;
                        x[4 + i] = b * cv + a * sv;
                    }
                }
            } else if (on) {  // any rotation: element by element, by way of LDS (a register has no index)
                const int64_t prow = min((int64_t)max(at[cc], 0), p.max_pos - 1) * p.half;
                float* own = reinterpret_cast<float*>(sq + (SPLIT ? 2 : 1) * COLS * HD) + c * HD + 8 * lane;
#pragma unroll 1
                for (int i = 0; i < 8; ++i)
                    own[i] = query_elem(p, from[cc], prow, rinv, (i < 4 ? ch : hi - 4) + i);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = own[i];
            }
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] *= i < 4 ? s0[i] : s1[i - 4];
                top = fmaxf(top, fabsf(x[i]));
            }
            top = group_max<W>(top);
            // A row of zeros, or with an infinity, is taken as it is.
            const int ex = top > 0.f && top < INFINITY ? max(-100, min(ilogbf(top), 116)) : 10;
            if (on) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    half_t* to = sq + c * HD + L::key_slot(b ? hi : ch);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float z = at[cc] >= 0 ? ldexpf(x[4 * b + i], 10 - ex) : 0.f;
                        const half_t y = (half_t)z;
                        constexpr int kStep = CODE == kInt4 ? 2 : 1;
                        to[kStep * i] = y;
                        if constexpr (SPLIT) to[COLS * HD + kStep * i] = (half_t)(z - (float)y);
                    }
                }
                if (lane == 0) {
                    f[c] = ldexpf(p.scale, ex - 10);
                    pos[c] = at[cc];
                }
            }
        }
    };
    if (F32 || p.dtype == ORTMI_F16) stage(std::true_type{});
    else stage(std::false_type{});
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

// x[0] + .. + x[7] + s, the sums in fp32.
__device__ __forceinline__ float sum8(half8_t x, float s) {
    const half2_t one = {(half_t)1.f, (half_t)1.f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) s = __builtin_amdgcn_fdot2(half2_t{x[i], x[i + 1]}, one, s, false);
    return s;
}

// exp2 of the scores about the column's reference, rounded to fp16 as the second product's
// operand (and, SPLIT, what the rounding left), added to the lane's sum as rounded: a weight's
// rounding then counts with the value's distance from the mean, and a lone key's not at all.
template <bool SPLIT>
__device__ __forceinline__ void probabilities(const float (&x0)[4], const float (&x1)[4], float m,
                                              float& l, half8_t& p, half8_t& rest) {
    const float ref = m - kPBase;
    float a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = __builtin_amdgcn_exp2f(x0[i] - ref);
        b[i] = __builtin_amdgcn_exp2f(x1[i] - ref);
    }
    p = pack_p(a, b);
    if constexpr (SPLIT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] -= (float)p[i];
            b[i] -= (float)p[4 + i];
        }
        rest = pack_p(a, b);
        l = sum8(rest, l);
    }
    l = sum8(p, l);
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

// One unit: a range of keys [k0, k1), `split` of `n`, for the tile of columns c0 .. of sequence
// b and kv head h. The tile's units are first, first + step, ... in part and ml.
struct Unit {
    int b, h, c0, split, n, k0, k1, step;
    int64_t first;
    float *part, *ml;
    __device__ __forceinline__ int64_t row(int i, int cols, int c) const {
        return (first + (int64_t)i * step) * cols + c;
    }
};

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
// A unit's columns from LDS rows, eight channels a thread and step, all of a row side by side:
// as output times inv, or (one range of several) unscaled into part. Padded rows are zeros.
// The scales are on their way while the rows are written: this waits for the other threads.
template <int HD, bool F32, int COLS, int THREADS>
__device__ __forceinline__ void write_rows(const Params& p, const Seq& s, const Unit& un,
                                           const float* rows, const float* inv, int part_cols) {
    constexpr int kPieces = HD / 8, kRows = THREADS / kPieces;
    const int G = p.H / p.KV, ch = 8 * (threadIdx.x % kPieces);
    float vs[8];
    load_scales<8>(p.vs, p.v_chan, un.h * HD + ch, vs);
    __syncthreads();
#pragma unroll 1
    for (int c = threadIdx.x / kPieces; c < COLS; c += kRows) {
        const int r = (un.c0 + c) / G;
        if (r >= s.rows || threadIdx.x >= kRows * kPieces) break;
        const float* x = rows + c * kRowFloats<HD> + ch;
        const float4_t a = *reinterpret_cast<const float4_t*>(x), b = *reinterpret_cast<const float4_t*>(x + 4);
        if (un.n > 1 && r < s.real) {
            float* o = un.part + un.row(un.split, part_cols, c) * HD + ch;
            *reinterpret_cast<float4_t*>(o) = a;
            *reinterpret_cast<float4_t*>(o + 4) = b;
        } else if (un.n <= 1 || un.split == 0) {
            const int64_t row = (int64_t)(s.tok0 + r) * p.H + un.h * G + (un.c0 + c - r * G);
            const float y[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
            store_piece<8, F32>(p, row * HD + ch, y, vs, r < s.real ? inv[c] : 0.f);
        }
    }
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

// A unit of columns 0 .. 15 of sequence s.
template <int CODE, int HD, bool F32, bool PAGED>
__device__ __forceinline__ void token_tile(const Params& p, const Seq& s, const Unit& un,
                                           TokenShared<HD, F32>& sh) {
    const int b = un.b, h = un.h, k0 = un.k0, k1 = un.k1;
    using L = Layout<CODE, HD>;
    constexpr int KS = L::KS, MT = L::MT;
    const int lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
    const int wave = uniform(threadIdx.x >> 6);
    const int G = p.H / p.KV;

    // The first block's rows are on their way while the queries are staged.
    const Source<CODE, HD, PAGED> src(p, b, h, k0, k1);
    int kb = k0 + 32 * wave;
    int2 id = src.ids(kb), id_n = src.ids(kb + 128), sl = src.slots(kb, id);
    Block<CODE, HD> cur, nxt;
    if (kb < k1) src.load(kb, sl, cur);
    stage_queries<CODE, HD, 16, 256, F32, true>(p, s, h, 0, sh.queries, sh.f, sh.pos);
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
            sl = src.slots(kb + 128, id_n);
            id_n = src.ids(kb + 256);
            src.load(kb + 128, sl, nxt);
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
            if (un.n > 1)
                reinterpret_cast<float2*>(un.ml)[un.row(un.split, p.tcols, n)] = make_float2(mm, sum);
            else
                sh.inv[n] = output_factor<F32, PAGED>(p, head, mm, sum);
        }
    }
    write_rows<HD, F32, 16, 256>(p, s, un, sh.rows, sh.inv, p.tcols);
}

// ---------------------------------------------------------------- prompt tiles --
template <int CODE, int HD, bool F32>
struct PromptShared {
    static constexpr int kNT = F32 ? 1 : 2, kCols = 64 * kNT;
    // Query rows as two fp16 halves where registers and time allow: at head size 128 the second
    // products would take a 2048-token prompt from 71 to 82 us and the output's error from
    // 3.1e-4 to 2.9e-4, 2.1e-4 of it the output's own rounding.
    static constexpr bool kSplit = F32 || HD < 128;
    struct Blocks {  // two blocks of 64 keys: [key tile][k step], [half][channel tile], by lane
        half8_t k[2][4][HD / 32][64], v[2][2][HD / 16][64];
    };
    union {
        __align__(16) half_t queries[(kSplit ? 2 : 1) * kCols * HD];
        Blocks team[2];
        struct {
            __align__(16) float4_t out[4][HD / 16][kNT][64];  // the second team's outputs
            __align__(16) float rows[kCols * kRowFloats<HD>];  // the tile's
        };
    };
    float f[kCols], m[kCols], l[kCols], inv[kCols];
    int pos[kCols];
};

// A unit of columns c0 .. c0 + 127 (fp32: 63) of sequence s.
template <int CODE, int HD, bool F32, bool PAGED>
__device__ __forceinline__ void prompt_tile(const Params& p, const Seq& s, const Unit& un,
                                            PromptShared<CODE, HD, F32>& sh) {
    const int b = un.b, h = un.h, c0 = un.c0, k0 = un.k0, k1 = un.k1;
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
    // Entries of the block of keys to be loaded next, and the key tiles without a block (bits) of
    // this one and the next.
    int id[4];
    uint32_t gone = 0, gone_n = 0;
    auto ids = [&](int kb) {
#pragma unroll
        for (int t = 0; t < 4; ++t) id[t] = src.entry(kb + 16 * t);
    };
    auto load = [&](int kb) {
        gone_n = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t) gone_n |= (uint32_t)src.gone(kb + 16 * t, id[t]) << t;
        const int a0 = id[0], a1 = id[1], a2 = id[2], a3 = id[3], kv = kb + 32 * (wave >> 1);
        const int a = src.slot(kv, wave & 2 ? a2 : a0), c = src.slot(kv + 16, wave & 2 ? a3 : a1);
        src.keys(kb + 16 * wave, wave & 1 ? c : a, rk);
        src.values(kv, a, c, rv);
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
    ids(kb);
    if (kb < k1) load(kb);
    ids(kb + 128);
    stage_queries<CODE, HD, SH::kCols, 512, F32, SH::kSplit>(p, s, h, c0, sh.queries, sh.f, sh.pos);
    const half8_t* sq = reinterpret_cast<const half8_t*>(sh.queries);
    half8_t Q[NT][KS], QL[SH::kSplit ? NT : 1][KS];
    float f[NT];
    int pos[NT];
    const int cw = 16 * NT * wave;  // the wave's columns
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            Q[t][ks] = sq[((cw + 16 * t + n) * KS + ks) * 4 + q];
            if constexpr (SH::kSplit) QL[t][ks] = sq[((SH::kCols + cw + 16 * t + n) * KS + ks) * 4 + q];
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
    gone = gone_n;
    if (kb + 128 < k1) load(kb + 128);
    ids(kb + 256);
    __syncthreads();
    int buf = 0;
    for (int first_kb = k0; first_kb < k1; first_kb += 128, kb += 128, buf ^= 1) {
        const uint32_t out = gone;
        if (kb + 128 < k1) {
            decode(buf ^ 1);
            gone = gone_n;
            if (kb + 256 < k1) load(kb + 256);
            ids(kb + 384);
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
                        if constexpr (SH::kSplit) S[t] = ORTMI_MFMA(a, QL[t][ks], S[t]);
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[t][t4][i] = S[t][i] * f[t];
            }
            if (kb + 63 > first || kb + 64 > k1 || (PAGED && out)) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int t4 = 0; t4 < 4; ++t4)
                        mask_scores(x[t][t4], kb + 16 * t4,
                                    PAGED && (out >> t4 & 1) ? -1 : min(pos[t], k1 - 1));
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

    // The second team's outputs to the first, which adds its own.
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
    if (!team) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int c = cw + 16 * t + n, r = (c0 + c) / G;
            const float m1 = sh.m[c], mm = fmaxf(m[t], m1);
            const float a0 = __builtin_amdgcn_exp2f(m[t] - mm), a1 = __builtin_amdgcn_exp2f(m1 - mm);
            const float sum = quarters_sum(l[t]) * a0 + sh.l[c] * a1;
            float* row = sh.rows + c * kRowFloats<HD>;
#pragma unroll
            for (int d = 0; d < MT; ++d) O[d][t] = O[d][t] * a0 + sh.out[wave][d][t][lane] * a1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // a lane's neighbouring channels at once
                const int ch = L::value_channel(4 * q + i, 0);
#pragma unroll
                for (int d = 0; d < (HD == 96 ? 4 : MT); d += 4)
                    *reinterpret_cast<float4_t*>(row + ch + d) =
                        float4_t{O[d][t][i], O[d + 1][t][i], O[d + 2][t][i], O[d + 3][t][i]};
                if constexpr (HD == 96)
                    *reinterpret_cast<float2*>(row + L::value_channel(4 * q + i, 4)) =
                        make_float2(O[4][t][i], O[5][t][i]);
            }
            if (q == 0 && r < s.real) {
                if (un.n > 1)
                    reinterpret_cast<float2*>(un.ml)[un.row(un.split, SH::kCols, c)] = make_float2(mm, sum);
                else
                    sh.inv[c] = output_factor<F32, PAGED>(p, h * G + (c0 + c - r * G), mm, sum);
            }
        }
    }
    write_rows<HD, F32, SH::kCols, 512>(p, s, un, sh.rows, sh.inv, SH::kCols);
}

// -------------------------------------------------------------------- new rows --
// append_row in pieces.
template <int CODE, int HD, bool F32, bool PAGED>
__device__ __forceinline__ void append_piece(const Params& p, int b, const Seq& s, int r, int h,
                                             bool is_v, int lane) {
    constexpr int RB = row_bytes(CODE, HD);
    const int pos = s.past + r, c0 = lane < HD / 8 ? 4 * lane : 0, c1 = c0 + HD / 2;
    const int64_t row = cache_row<PAGED>(p, b, h, pos);
    const int64_t from = (int64_t)(s.tok0 + r) * p.kv_tok + (int64_t)h * HD;
    const void* src = is_v ? p.v : p.k;
    const bool rope = !is_v && p.cos, norm = p.kw && !is_v;
    Piece<F32> x0, x1, co, si, w0, w1;
    float sc[2][4];
    x0.load(src, from + c0);
    x1.load(src, from + c1);
    load_scales<4>(is_v ? p.vs : p.ks, is_v ? p.v_chan : p.k_chan, h * HD + c0, sc[0]);
    load_scales<4>(is_v ? p.vs : p.ks, is_v ? p.v_chan : p.k_chan, h * HD + c1, sc[1]);
    if (rope) {
        const int64_t at = min((int64_t)pos, p.max_pos - 1) * (HD / 2) + c0;
        co.load(p.cos, at);
        si.load(p.sin, at);
    }
    if (p.kw) {
        w0.load(p.kw, c0);
        w1.load(p.kw, c1);
    }
    auto codes = [&](auto half) {
        constexpr bool HALF = decltype(half)::value;
        double x[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[0][i] = x0.template get<HALF>(i);
            x[1][i] = x1.template get<HALF>(i);
        }
        if (p.kw) {  // (a value row's lanes go along)
            double ss = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) ss += x[0][i] * x[0][i] + x[1][i] * x[1][i];
            ss = lane < HD / 8 ? ss : 0.0;
#pragma unroll
            for (int k = kRowLanes<HD> / 2; k; k >>= 1) ss += __shfl_xor(ss, k, 64);
            const double rinv = norm ? 1.0 / sqrt(ss / HD + (double)p.eps) : 1.0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[0][i] = norm ? x[0][i] * rinv * (double)w0.template get<HALF>(i) : x[0][i];
                x[1][i] = norm ? x[1][i] * rinv * (double)w1.template get<HALF>(i) : x[1][i];
            }
        }
        if (row < 0 || lane >= HD / 8) return;
        uint8_t* dst = (is_v ? p.vc : p.kc) + row * RB;
        if (rope) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const double a = x[0][i], e = x[1][i];
                const double c = co.template get<HALF>(i), d = si.template get<HALF>(i);
                x[0][i] = a * c - e * d;
                x[1][i] = e * c + a * d;
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t u = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                u |= encode(x[j][i], sc[j][i], CODE) << ((CODE == kInt4 ? 4 : 8) * i);
            const int ch = j ? c1 : c0;
            if constexpr (CODE == kInt4) *reinterpret_cast<uint16_t*>(dst + ch / 2) = (uint16_t)u;
            else *reinterpret_cast<uint32_t*>(dst + ch) = u;
        }
    };
    if (F32 || p.dtype == ORTMI_F16) codes(std::true_type{});
    else codes(std::false_type{});
}

// Rows r0 .. r1 - 1 of sequence s, key and value of one kv head, by the workgroup.
template <int CODE, int HD, bool F32, bool PAGED>
__device__ __forceinline__ void append_rows(const Params& p, int b, const Seq& s, int r0, int r1,
                                            int h) {
    const int w = p.pieces ? kRowLanes<HD> : 16, lane = threadIdx.x % w;
    for (int i = 2 * r0 + (int)threadIdx.x / w; i < 2 * r1; i += (int)blockDim.x / w) {
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

// Keys of a range where `total` keys are to be taken in about `items` ranges.
constexpr int kMostKeys = 1 << 24;  // a range's bytes stay below 2^32
__device__ __forceinline__ int range_keys(int64_t total, int items, int least) {
    const int64_t per = (total / items + 128) & ~127LL;  // above total / items
    return (int)max((int64_t)least, min(per, (int64_t)kMostKeys));
}
// Keys of each of n ranges of equal size: n stays the least number of ranges of at most the
// keys it was found with.
__device__ __forceinline__ int even_keys(int keys, int n) { return ((keys + n - 1) / n + 127) & ~127; }
// Units that n of a sequence's ranges put into part and ml: with one range, none.
__device__ __forceinline__ int64_t parts_of(int64_t n, int64_t tiles) { return n > 1 ? n * tiles : 0; }

__device__ __forceinline__ int64_t scan64(int64_t x, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t v = __shfl_up(x, o, 64);
        x += lane >= o ? v : 0;
    }
    return x;
}

// Keys of a range of prompt tiles, for `seqs` sequences of which the longest has `most` keys;
// shape(b, keys, tiles) gives each. A workgroup of prompt tiles has a CU of its own and kAround
// keys' time around its loop, so that r rounds of ranges of c keys take about r (c + kAround): a
// lane prices a number of ranges for the longest sequence. Workgroups start in order and wait for
// the engine whose turn it is: short ranges between long ones do not fill gaps (four prompts of
// 256 rows over 2200 to 5500 keys in ranges of 3584 and what remained: 160 us for 106 of work).
template <typename F>
__device__ __forceinline__ int prompt_keys(const Params& p, int seqs, int most, F shape) {
    constexpr int kAround = 570, kCus = 256;
    const int lane = threadIdx.x & 63;
    int c = max(p.pmin, (most + 127) & ~127);
    if (seqs > kCus) return c;  // enough of them
    c = max(p.pmin, even_keys(most, lane + 1));
    int64_t units = 0, parts = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        int keys, tiles;
        shape(b0 + lane, keys, tiles);
        for (uint64_t left = __ballot(tiles > 0); left; left &= left - 1) {
            const int j = __builtin_ctzll(left);
            const int k = __shfl(keys, j, 64), t = __shfl(tiles, j, 64);
            const int n = (k + c - 1) / c;
            units += (int64_t)n * t;
            parts += parts_of(n, t);
        }
    }
    const int64_t rounds = (units * p.KV + kCus - 1) / kCus;
    const float cost = parts <= p.pparts ? (float)rounds * (float)(c + kAround) : INFINITY;
    const uint64_t best = __ballot(cost == -wave_max(-cost));  // (lane 0: no parts)
    return __shfl(c, __builtin_ctzll(best), 64);
}

// Pages: the ranges, by one wave. Token tiles are those of sequences with at most 16 columns;
// the others have prompt tiles, all over the ranges of the sequence's last. plan[b]: the units
// (over KV) in front of sequence b, of token tiles x (in part: y), of prompt tiles z (in ppart:
// w); plan[B]: all units x, z and the most keys of a range y, w. Ranges of near equal size,
// whatever the sequences' lengths, keep the GPU evenly filled. Of token tiles, units that are not
// their tile's only one are at most twice those aimed at: n ranges for one of c keys, n > 1, lie
// over more than n c / 2 keys.
template <bool F32>
__device__ __forceinline__ void plan_units(const Params& p) {
    constexpr int kW = prompt_width(F32 ? ORTMI_F32 : ORTMI_F16);
    const int lane = threadIdx.x & 63, G = p.H / p.KV;
    auto shape = [&](int b, int& kend, int& tiles) {
        kend = tiles = 0;
        if (b >= p.B) return;
        const Seq s = sequence<true>(p, b);
        const int64_t cols = (int64_t)s.rows * G;
        if (s.rows > 0) kend = s.keys_to(s.rows - 1, p.limit);
        tiles = cols > 16 ? (int)((cols + kW - 1) / kW) : 0;
    };
    int64_t total = 0;
    int most = 0, seqs = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        int kend, tiles;
        shape(b0 + lane, kend, tiles);
        total += tiles ? 0 : kend;
        most = max(most, tiles ? kend : 0);
        seqs += __popcll(__ballot(tiles > 0));
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        total += __shfl_xor(total, o, 64);
        most = max(most, __shfl_xor(most, o, 64));
    }
    const int chunk[2] = {range_keys(total, p.titems, p.tmin), seqs ? prompt_keys(p, seqs, most, shape) : 128};
    int64_t base[4] = {0, 0, 0, 0};
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        int kend, tiles, at[4];
        shape(b0 + lane, kend, tiles);
        const int64_t nt = tiles ? 0 : (kend + chunk[0] - 1) / chunk[0];
        const int64_t np = tiles ? (kend + chunk[1] - 1) / chunk[1] : 0;
        const int64_t x[4] = {nt, parts_of(nt, 1), np * tiles, parts_of(np, tiles)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t incl = scan64(x[i], lane);
            at[i] = (int)min(base[i] + incl - x[i], (int64_t)1 << 30);
            base[i] += __shfl(incl, 63, 64);
        }
        if (b0 + lane < p.B) p.plan[b0 + lane] = make_int4(at[0], at[1], at[2], at[3]);
    }
    if (lane == 0)
        p.plan[p.B] = make_int4((int)min(base[0], (int64_t)1 << 30), chunk[0],
                                (int)min(base[2], (int64_t)1 << 30), chunk[1]);
}

// Pages: unit `i` (over KV) and kv head h of the token or prompt tiles; false: none.
template <bool F32, bool PROMPT>
__device__ __forceinline__ bool page_unit(const Params& p, int i, int h, Unit& un, Seq& s) {
    constexpr int kW = PROMPT ? prompt_width(F32 ? ORTMI_F32 : ORTMI_F16) : 16;
    const int lane = threadIdx.x & 63;
    const int4 all = p.plan[p.B];
    if (i >= (PROMPT ? all.z : all.x)) return false;
    // The last sequence with at most i units in front, 64 places at a time.
    int lo = 0, len = p.B;
    while (len > 1) {
        const int step = (len + 63) / 64, at = lane * step;
        const int4 e = p.plan[lo + min(at, len - 1)];
        const uint64_t le = __ballot(at < len && (PROMPT ? e.z : e.x) <= i);
        const int skip = max(__popcll(le) - 1, 0) * step;
        lo = uniform(lo + skip);
        len = uniform(min(step, len - skip));
    }
    const int4 e = p.plan[lo];
    s = sequence<true>(p, lo);
    const int G = p.H / p.KV, most = PROMPT ? all.w : all.y, j = i - (PROMPT ? e.z : e.x);
    int first = PROMPT ? e.w : e.y, tile = 0;
    un.split = j;
    const int keys = s.keys_to(s.rows - 1, p.limit), n = (keys + most - 1) / most;
    const int chunk = even_keys(keys, n);
    if constexpr (PROMPT) {
        tile = j / n;
        un.split = j - tile * n;
        first += tile * n;
    }
    un.b = lo;
    un.h = h;
    un.c0 = tile * kW;
    const int kend = s.keys_to((min(un.c0 + kW, s.rows * G) - 1) / G, p.limit);
    un.n = (kend + chunk - 1) / chunk;
    un.k0 = un.split * chunk;
    un.k1 = min(un.k0 + chunk, kend);
    un.first = (int64_t)first * p.KV + h;
    un.step = p.KV;
    un.part = PROMPT ? p.ppart : p.part;
    un.ml = PROMPT ? p.pml : p.ml;
    return un.split < un.n;
}

// Slabs: unit `i` of the tile and its sequence, also of tiles whose rows are all padding (k0 =
// k1 = 0, one range).
template <bool F32, bool PROMPT>
__device__ __forceinline__ bool slab_unit(const Params& p, int i, Unit& un, Seq& s) {
    constexpr int kW = PROMPT ? prompt_width(F32 ? ORTMI_F32 : ORTMI_F16) : 16;
    const int G = p.H / p.KV;
    int chunk = p.chunk, tile = 0;
    un.part = p.part;
    un.ml = p.ml;
    if (PROMPT || !p.planned) {
        // (range, tile, slab), the slab running fastest (slabs of one residue modulo 8 stay on
        // one XCD). Later tiles, which see more keys, come first.
        const int slabs = p.B * p.KV, rem = i % (slabs * p.ntile), slab = rem % slabs;
        tile = p.ntile - 1 - rem / slabs;
        un.b = slab / p.KV;
        un.h = slab % p.KV;
        un.split = i / (slabs * p.ntile);
        un.first = ((int64_t)slab * p.ntile + tile) * p.nsplit;
        un.step = 1;
    } else {
        // At most 64 sequences, a lane each: ranges of equal size (plan_units()).
        const int lane = threadIdx.x & 63, item = i / p.KV;
        const int kend = lane < p.B ? sequence<false>(p, lane).keys_to(p.S - 1, p.limit) : 0;
        int64_t total = kend;
#pragma unroll
        for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o, 64);
        chunk = uniform(range_keys(total, p.titems, p.tmin));
        const int n = lane < p.B ? max(1, (kend + chunk - 1) / chunk) : 0;
        int at = n, part = n > 1 ? n : 0;
        const int own = part;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(at, o, 64), v = __shfl_up(part, o, 64);
            at += lane >= o ? u : 0;
            part += lane >= o ? v : 0;
        }
        const int b = uniform(__popcll(__ballot(at <= item)));  // sequences that end before it
        if (b >= p.B) return false;
        un.b = b;
        un.h = i % p.KV;
        chunk = uniform(__shfl(even_keys(kend, max(n, 1)), b, 64));
        un.split = item - uniform(__shfl(at - n, b, 64));
        un.first = (int64_t)uniform(__shfl(part - own, b, 64)) * p.KV + un.h;
        un.step = p.KV;
    }
    s = sequence<false>(p, un.b);
    un.c0 = tile * kW;
    un.k0 = un.k1 = 0;
    un.n = 1;
    if (un.c0 / G >= s.real) return un.split == 0;
    const int kend = s.keys_to((min(un.c0 + kW, s.rows * G) - 1) / G, p.limit);
    un.n = (kend + chunk - 1) / chunk;
    un.k0 = un.split * chunk;
    un.k1 = min(un.k0 + chunk, kend);
    return un.split < un.n;
}

// New keys and values into the cache: a group of lanes per (token, kv head, key or value). 2048
// tokens of 8 heads of 128: 9 us, the 64-bit divisions' instructions. Pages: the
// first workgroup plans the units.
template <int CODE, int HD, bool F32, bool PAGED>  // HD 0: any
__global__ __launch_bounds__(256) void append_kernel(Params p) {
    constexpr int W = kRowLanes<HD>;
    int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / W;
    if constexpr (PAGED) {
        if (blockIdx.x == 0) {
            if (threadIdx.x < 64 && p.plan) {
                if (p.dtype == ORTMI_F32) plan_units<true>(p);
                else plan_units<false>(p);
            }
            return;
        }
        item -= 256 / W;
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
        append_piece<CODE, HD, F32, PAGED>(p, b, s, r, hv % p.KV, hv >= p.KV, threadIdx.x % W);
    else
        append_row<PAGED>(p, b, s, r, hv % p.KV, hv >= p.KV, threadIdx.x % W);
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

// Slabs, a workgroup for each unit. Where a sequence's columns are one tile, the workgroup whose
// range holds the new rows writes them to the cache itself.
template <int CODE, int HD, bool F32, bool PROMPT>
__global__ __launch_bounds__(PROMPT ? 512 : 256, 2) void tile_kernel(Params p) {
    using SH = std::conditional_t<PROMPT, PromptShared<CODE, HD, F32>, TokenShared<HD, F32>>;
    __shared__ SH sh;
    Unit un;
    Seq s;
    if (!slab_unit<F32, PROMPT>(p, blockIdx.x, un, s)) return;
    if (un.k0 == un.k1) {
        zero_rows<HD, F32>(p, s, un.h, un.c0, PROMPT ? prompt_width(F32 ? ORTMI_F32 : ORTMI_F16) : 16);
        return;
    }
    if (p.fused) {
        append_rows<CODE, HD, F32, false>(p, un.b, s, max(un.k0 - s.past, 0),
                                          min(un.k1 - s.past, s.real), un.h);
        __syncthreads();
    }
    if constexpr (PROMPT) prompt_tile<CODE, HD, F32, false>(p, s, un, sh);
    else token_tile<CODE, HD, F32, false>(p, s, un, sh);
}

// Pages, the same, of sequences with at most 16 columns (token tiles) and with more.
template <int CODE, int HD, bool F32, bool PROMPT>
__global__ __launch_bounds__(PROMPT ? 512 : 256, 2) void page_kernel(Params p) {
    using SH = std::conditional_t<PROMPT, PromptShared<CODE, HD, F32>, TokenShared<HD, F32>>;
    __shared__ SH sh;
    Unit un;
    Seq s;
    if (!page_unit<F32, PROMPT>(p, blockIdx.x / p.KV, blockIdx.x % p.KV, un, s)) return;
    if constexpr (PROMPT) prompt_tile<CODE, HD, F32, true>(p, s, un, sh);
    else token_tile<CODE, HD, F32, true>(p, s, un, sh);
}

// New rows and attention for one code; in kvq_int8.hip, kvq_int4.hip and kvq_fp8.hip.
int tiles_int8(const Params& p, bool paged, hipStream_t st);
int tiles_int4(const Params& p, bool paged, hipStream_t st);
int tiles_fp8(const Params& p, bool paged, hipStream_t st);

inline int64_t slab_units(const Params& p) {
    return p.planned ? (int64_t)p.tgrid * p.KV : (int64_t)p.B * p.KV * p.ntile * p.nsplit;
}

template <int CODE, int HD, bool F32>
int launch_tiles(const Params& p, bool paged, hipStream_t st) {
    const int G = p.H / p.KV;
    constexpr int kItems = 256 / kRowLanes<HD>;
    const dim3 rows((unsigned)(((int64_t)p.T * 2 * p.KV + kItems - 1) / kItems + (paged ? 1 : 0)));
    if (p.pieces && !p.fused) {
        if (paged) hipLaunchKernelGGL((append_kernel<CODE, HD, F32, true>), rows, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((append_kernel<CODE, HD, F32, false>), rows, dim3(256), 0, st, p);
        if (int rc = check_launch("kv append")) return rc;
    }
    if (!paged) {
        if (p.S * G <= 16)
            hipLaunchKernelGGL((tile_kernel<CODE, HD, F32, false>), dim3((unsigned)slab_units(p)),
                               dim3(256), 0, st, p);
        else
            hipLaunchKernelGGL((tile_kernel<CODE, HD, F32, true>), dim3((unsigned)slab_units(p)),
                               dim3(512), 0, st, p);
        return check_launch("kv tiles");
    }
    if (p.tgrid) {
        hipLaunchKernelGGL((page_kernel<CODE, HD, F32, false>), dim3((unsigned)((int64_t)p.tgrid * p.KV)),
                           dim3(256), 0, st, p);
        if (int rc = check_launch("kv page tokens")) return rc;
    }
    if (!p.pgrid) return ORTMI_OK;
    hipLaunchKernelGGL((page_kernel<CODE, HD, F32, true>), dim3((unsigned)((int64_t)p.pgrid * p.KV)),
                       dim3(512), 0, st, p);
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
