// GroupQueryAttention and PagedAttention over quantised key-value caches: new rows into the
// cache, attention for any head size, entry points.
#include <algorithm>
#include <cmath>

#include "kvq_tile.h"

namespace ortmi {
namespace kvq {

// Joins the ranges of tiles that have more than one: a workgroup for each unit, which takes its
// share of the tile's columns (of prompt tiles, eight for each unit). A column's ranges are read
// by 2, 4 or 8 half-waves, float4 a lane, and joined through LDS: many ranges of few columns and
// few of many keep all lanes busy. Latency binds it: 32 sequences of 2 to 11 ranges 7 us, a prompt
// piece of 2 x 333 rows of 14 heads over 3 ranges 11 us.
constexpr int kShares = 8;
template <bool F32, bool PAGED>
__global__ __launch_bounds__(256) void merge_kernel(Params p) {
    __shared__ float4_t acc_s[8][32];
    constexpr int kW = prompt_width(F32 ? ORTMI_F32 : ORTMI_F16);
    const int G = p.H / p.KV;
    Unit un;
    Seq s;
    int cols = p.tcols, shares = 1, share = 0;  // (cols: of a unit in part and ml)
    bool any;
    if constexpr (PAGED) {
        const int i = (int)blockIdx.x / p.KV, h = (int)blockIdx.x % p.KV;
        if (i < p.tgrid) {
            any = page_unit<F32, false>(p, i, h, un, s);
        } else {
            share = (i - p.tgrid) % kShares;
            shares = kShares;
            any = page_unit<F32, true>(p, (i - p.tgrid) / kShares, h, un, s);
        }
    } else if (p.S * G <= 16) {
        any = slab_unit<F32, false>(p, blockIdx.x, un, s);
    } else {
        share = blockIdx.x % kShares;
        shares = kShares;
        any = slab_unit<F32, true>(p, blockIdx.x / kShares, un, s);
    }
    if (!any || un.n <= 1) return;
    if (shares > 1) cols = kW;
    const int n = un.n, live = min(cols, s.real * G - un.c0);
    // Of the columns, part `at` of n * shares.
    const int at = un.split * shares + share;
    const int end = (int)((int64_t)live * (at + 1) / (n * shares));
    const int per = n > 16 ? 8 : n > 4 ? 4 : 2;  // half-waves a column
    const int hw = threadIdx.x >> 5, lane = threadIdx.x & 31, ch = 4 * lane;
    for (int c0 = (int)((int64_t)live * at / (n * shares)); c0 < end; c0 += 8 / per) {
        const int c = min(c0 + hw / per, end - 1), sub = hw % per;
        float top = kNone;
        for (int i = lane; i < n; i += 32) top = fmaxf(top, un.ml[un.row(i, cols, c) * 2]);
        top = group_max<32>(top);
        float sum = 0.f;
        float4_t acc{0.f, 0.f, 0.f, 0.f};
        for (int i0 = 0; i0 < n; i0 += 32) {
            float w = 0.f;
            if (i0 + lane < n) {
                const float2 ml = reinterpret_cast<const float2*>(un.ml)[un.row(i0 + lane, cols, c)];
                w = __builtin_amdgcn_exp2f(ml.x - top);
                sum += w * ml.y;
            }
            const int m = min(32, n - i0);
            for (int j = 0; j < m; j += per) {
                const int i = j + sub;  // (at most 31)
                const float e = __shfl(w, i, 32);
                if (ch < p.hd && i < m)
                    acc += e * *reinterpret_cast<const float4_t*>(
                                   un.part + un.row(i0 + i, cols, c) * p.hd + ch);
            }
        }
        sum = group_sum<32>(sum);
        __syncthreads();
        acc_s[hw][lane] = acc;
        __syncthreads();
        const int col = un.c0 + c, r = col / G, head = un.h * G + (col - r * G);
        if (sub == 0 && ch < p.hd && c0 + hw / per < end) {
            for (int i = 1; i < per; ++i) acc += acc_s[hw + i][lane];
            float vs[4];
            load_scales<4>(p.vs, p.v_chan, un.h * p.hd + ch, vs);
            const float y[4] = {acc[0], acc[1], acc[2], acc[3]};
            store_piece<4, F32>(p, ((int64_t)(s.tok0 + r) * p.H + head) * p.hd + ch, y, vs,
                                output_factor<F32, PAGED>(p, head, top, sum));
        }
    }
}

// Attention of one query row and head per workgroup, any head size that is a multiple of 16
// up to 256: 16 teams of 16 lanes take every 16th key, a lane 1/16 of the channels; each
// team keeps a running maximum and sum, joined at the end. The key scales are folded into
// the query row and the value scales into the output, so the loop multiplies codes. Only for
// shapes and alignments that tiles do not take: latency of one key after another binds it (a
// token of 12 heads of 128 over 512 keys 91 us, in tiles 12).
constexpr int kTeams = 16, kMaxPerLane = 16;
template <bool PAGED>
__global__ __launch_bounds__(256) void row_kernel(Params p) {
    __shared__ float sq[256];
    __shared__ float so[kTeams][256];
    __shared__ float sm[kTeams], sl[kTeams];
    const int tok = blockIdx.x, head = blockIdx.y, hd = p.hd, tid = threadIdx.x;
    const int h = head / (p.H / p.KV);
    int b;
    Seq s;
    if constexpr (PAGED) {
        if (!sequence_of_token(p, tok, b, s)) return;
    } else {
        b = tok / p.S;
        s = sequence<false>(p, b);
    }
    const int r = tok - s.tok0;
    const int64_t o0 = ((int64_t)tok * p.H + head) * hd;
    if (r >= s.real) {  // a padded row
        if (tid < hd) store_elem(p.out, o0 + tid, 0.f, p.dtype);
        return;
    }
    const int64_t x0 = (int64_t)tok * p.q_tok + (int64_t)head * hd;
    float rinv = 1.f;
    if (p.qw) {
        __shared__ float ssum[4];
        float ss = 0.f;
        if (tid < hd) {
            const float x = load_elem(p.q, x0 + tid, p.dtype);
            ss = x * x;
        }
        ss = wave_sum(ss);
        if ((tid & 63) == 0) ssum[tid >> 6] = ss;
        __syncthreads();
        rinv = 1.f / sqrtf((ssum[0] + ssum[1] + ssum[2] + ssum[3]) / (float)hd + p.eps);
    }
    if (tid < hd) {
        const int64_t prow = min((int64_t)(s.past + r), p.max_pos - 1) * p.half;
        sq[tid] = query_elem(p, x0, prow, rinv, tid) * p.ks[p.k_chan ? h * hd + tid : 0] * p.scale;
    }
    __syncthreads();
    const int team = tid >> 4, lane = tid & 15, per = hd / 16, c0 = lane * per;
    float o[kMaxPerLane];
    for (int i = 0; i < kMaxPerLane; ++i) o[i] = 0.f;
    float m = -1e30f, l = 0.f;
    const int rb = row_bytes(p.code, hd);
    const int kend = s.keys_to(r, p.limit);
    for (int j = team; j < kend; j += kTeams) {
        const int64_t row = cache_row<PAGED>(p, b, h, j);
        if (row < 0) continue;
        const uint8_t* kr = p.kc + row * rb;
        const uint8_t* vr = p.vc + row * rb;
        float x = 0.f;
        for (int i = 0; i < per; ++i) x += sq[c0 + i] * code_value(kr, c0 + i, p.code);
        x = group_sum<16>(x);
        const float mm = fmaxf(m, x), a = exp2f(m - mm), e = exp2f(x - mm);
        l = l * a + e;
        for (int i = 0; i < kMaxPerLane; ++i)
            if (i < per) o[i] = o[i] * a + e * code_value(vr, c0 + i, p.code);
        m = mm;
    }
    for (int i = 0; i < kMaxPerLane; ++i)
        if (i < per) so[team][c0 + i] = o[i];
    if (lane == 0) {
        sm[team] = m;
        sl[team] = l;
    }
    __syncthreads();
    if (tid >= hd) return;
    float mm = -1e30f;
    if (p.sink) mm = load_elem(p.sink, head, p.dtype) * 1.44269504088896341f;
    const float ms = mm;
    for (int t = 0; t < kTeams; ++t) mm = fmaxf(mm, sm[t]);
    float sum = p.sink ? exp2f(ms - mm) : 0.f, acc = 0.f;
    for (int t = 0; t < kTeams; ++t) {
        const float a = exp2f(sm[t] - mm);
        sum += a * sl[t];
        acc += a * so[t][tid];
    }
    const float v = sum != 0.f ? acc / sum * p.vs[p.v_chan ? h * hd + tid : 0] : 0.f;
    store_elem(p.out, o0 + tid, v, p.dtype);
}

// Rows of the past into a present that is another buffer: `bytes` of each slab.
__global__ __launch_bounds__(256) void copy_slabs_kernel(const uint8_t* __restrict__ src,
                                                         uint8_t* __restrict__ dst,
                                                         int64_t src_pitch, int64_t dst_pitch,
                                                         int64_t bytes) {
    const uint8_t* s = src + blockIdx.y * src_pitch;
    uint8_t* d = dst + blockIdx.y * dst_pitch;
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 16;
    if (i >= bytes) return;
    if (i + 16 <= bytes &&
        ((reinterpret_cast<uintptr_t>(s) | reinterpret_cast<uintptr_t>(d)) & 15) == 0) {
        *reinterpret_cast<uint4*>(d + i) = *reinterpret_cast<const uint4*>(s + i);
    } else {
        for (int64_t j = i; j < min(i + 16, bytes); ++j) d[j] = s[j];
    }
}

static int copy_slabs(const void* src, void* dst, int64_t slabs, int64_t src_pitch,
                      int64_t dst_pitch, int64_t bytes, hipStream_t st) {
    if (slabs == 0 || bytes == 0) return ORTMI_OK;
    const int64_t gx = (bytes + 4095) / 4096;
    for (int64_t s0 = 0; s0 < slabs; s0 += 65535) {
        const int64_t n = std::min<int64_t>(65535, slabs - s0);
        hipLaunchKernelGGL(copy_slabs_kernel, dim3((unsigned)gx, (unsigned)n), dim3(256), 0, st,
                           static_cast<const uint8_t*>(src) + s0 * src_pitch,
                           static_cast<uint8_t*>(dst) + s0 * dst_pitch, src_pitch, dst_pitch,
                           bytes);
        if (int rc = check_launch("kv copy")) return rc;
    }
    return ORTMI_OK;
}

// Ranges of keys for `wgs` workgroups each over n keys: enough to fill the GPU, each a
// multiple of 128 keys (a block of 32 for each wave).
static void plan_ranges(int64_t wgs, int64_t n, int64_t target, int& nsplit, int& chunk) {
    const int64_t blocks = std::max<int64_t>(1, (n + 127) / 128);
    const int64_t want = std::min<int64_t>(blocks, std::max<int64_t>(1, target / std::max<int64_t>(1, wgs)));
    // At most 2^22 keys: a range's bytes stay below 2^31.
    const int64_t per = std::min<int64_t>((blocks + want - 1) / want, 1 << 15);
    chunk = (int)per * 128;
    nsplit = (int)((blocks + per - 1) / per);
}

static bool tile_head(int64_t hd) { return hd == 64 || hd == 96 || hd == 128; }
static size_t align_up(size_t x) { return (x + 255) & ~(size_t)255; }

// Units that token and prompt tiles are cut into, where there are keys enough: three workgroups
// of token tiles fit on a CU, and two rounds of them even out what differs (32 int8 sequences of
// 256 to 8192 keys: 512 units 78 us, 768 72, 1536 64; 16 int4 ones of up to 32768: 124, 120,
// 102), but a range of fewer than 512 keys is mostly start and end (eight of 4096: 512 keys 21
// us, 171 27), and a lone sequence that short needs no join. One workgroup of prompt tiles fills
// a CU: as many units as CUs, since each has about 12 us around its loop.
constexpr int64_t kTokenUnits = 1536, kPromptUnits = 256;
constexpr int kTokenLeast = 512, kPromptLeast = 256;

// The ranges' part of the workspace, from byte `ws` of it; returns what lies behind it.
static size_t place_parts(float*& part, float*& ml, char* ws, size_t at, int64_t rows, int64_t hd) {
    part = reinterpret_cast<float*>(ws + at);
    at += align_up((size_t)rows * hd * 4);
    ml = reinterpret_cast<float*>(ws + at);
    return at + align_up((size_t)rows * 8);
}

// Slabs: the plan of a call, and its workspace from ws on; returns the bytes.
static size_t plan_slabs(Params& p, int64_t n, char* ws) {
    const int64_t cols = (int64_t)p.S * (p.H / p.KV), slabs = (int64_t)p.B * p.KV;
    const int w = tile_width((int)std::min<int64_t>(cols, 1 << 20), p.dtype);
    p.ntile = (int)((cols + w - 1) / w);
    p.planned = w == 16 && p.B <= 64;
    p.tcols = (int)cols;
    p.tmin = kTokenLeast;
    plan_ranges(slabs * p.ntile, n, w == 16 ? kTokenUnits : kPromptUnits, p.nsplit, p.chunk);
    if (!tile_head(p.hd)) p.planned = 0, p.nsplit = 1;
    int64_t units = slabs * p.ntile * p.nsplit;
    if (p.planned) {
        const int64_t most = (n + p.tmin - 1) / p.tmin;  // ranges of a sequence
        p.titems = (int)std::max<int64_t>(1, kTokenUnits / p.KV);
        p.tgrid = (int)std::min<int64_t>(p.titems + p.B, p.B * std::max<int64_t>(1, most));
        p.nsplit = most > 1 ? 2 : 1;  // (more than one, or one)
        units = std::min<int64_t>(p.tgrid, 2 * p.titems) * p.KV;
    }
    if (p.nsplit == 1) return 0;
    return place_parts(p.part, p.ml, ws, 0, units * (w == 16 ? cols : w), p.hd);
}

// Pages: the same.
static size_t plan_pages(Params& p, char* ws) {
    const int64_t G = p.H / p.KV, cols = p.T * G, w = prompt_width(p.dtype);
    const int64_t seqs = std::min<int64_t>(p.B, p.T);
    p.titems = (int)std::max<int64_t>(1, kTokenUnits / p.KV);
    p.tmin = kTokenLeast;
    p.pmin = kPromptLeast;
    p.tcols = (int)std::min<int64_t>(16, cols);
    p.tgrid = G > 16 ? 0 : (int)(p.titems + seqs);
    // Sequences with prompt tiles have 17 columns or more.
    const int64_t tiles = cols / w + std::min<int64_t>(seqs, cols / 17);
    p.pparts = (int)std::min<int64_t>(std::max<int64_t>(1, 2 * kPromptUnits / p.KV),
                                      tiles * ((p.limit + (int64_t)p.pmin - 1) / p.pmin));
    p.pgrid = tiles ? (int)(p.pparts + tiles) : 0;
    size_t at = align_up((size_t)(p.B + 1) * sizeof(int4));
    p.plan = reinterpret_cast<int4*>(ws);
    p.nsplit = p.limit > std::min(p.tmin, kPromptLeast) ? 2 : 1;
    if (p.nsplit == 1) return at;
    at = place_parts(p.part, p.ml, ws, at, std::min(p.tgrid, 2 * p.titems) * (int64_t)p.KV * p.tcols, p.hd);
    return place_parts(p.ppart, p.pml, ws, at, (int64_t)p.pparts * p.KV * w, p.hd);
}

// On the matrix cores where head size and alignment allow 16-byte loads and pages are whole
// numbers of key tiles, otherwise a workgroup per row.
template <bool PAGED>
static int attend(Params& p, hipStream_t st) {
    uintptr_t bits = 0;
    for (const void* x : {(const void*)p.kc, (const void*)p.vc, p.q, (const void*)p.out, p.qw})
        bits |= reinterpret_cast<uintptr_t>(x);
    const bool tiles = tile_head(p.hd) && (bits & 15) == 0 &&
                       (!PAGED || (p.blk % 16 == 0 && p.nblk <= INT32_MAX / p.blk));
    if (!tiles) p.plan = nullptr;
    p.fused = !PAGED && tiles && p.ntile == 1;
    for (const void* x : {p.k, p.v, p.cos, p.sin, p.kw}) bits |= reinterpret_cast<uintptr_t>(x);
    p.pieces = tiles && (bits & 15) == 0 && (!p.cos || (2 * p.half == p.hd && !p.interleaved));
    if (!p.fused && !p.pieces) {
        const int64_t items = (int64_t)p.T * 2 * p.KV;
        hipLaunchKernelGGL((append_kernel<kInt8, 0, false, PAGED>),
                           dim3((unsigned)((items + 15) / 16 + (PAGED ? 1 : 0))), dim3(256), 0, st,
                           p);
        if (int rc = check_launch("kv append")) return rc;
    }
    if (!tiles) {
        hipLaunchKernelGGL((row_kernel<PAGED>), dim3((unsigned)p.T, (unsigned)p.H), dim3(256), 0,
                           st, p);
        return check_launch("kv rows");
    }
    int rc;
    if (p.code == kInt8) rc = tiles_int8(p, PAGED, st);
    else if (p.code == kInt4) rc = tiles_int4(p, PAGED, st);
    else rc = tiles_fp8(p, PAGED, st);
    if (rc || p.nsplit == 1) return rc;
    const int64_t shares = p.S * (p.H / p.KV) > 16 ? kShares : 1;
    const dim3 units((unsigned)(PAGED ? (p.tgrid + (int64_t)kShares * p.pgrid) * p.KV : shares * slab_units(p)));
    if (p.dtype == ORTMI_F32)
        hipLaunchKernelGGL((merge_kernel<true, PAGED>), units, dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL((merge_kernel<false, PAGED>), units, dim3(256), 0, st, p);
    return check_launch("kv merge");
}

static bool code_of(int32_t cache_type, int& code) {
    if (cache_type == ORTMI_INT8) code = kInt8;
    else if (cache_type == ORTMI_INT4) code = kInt4;
    else if (cache_type == ORTMI_F8E4M3) code = kFp8;
    else return false;
    return true;
}

}  // namespace kvq
}  // namespace ortmi

using namespace ortmi;

// The checks that both operators share; `what` begins their messages.
static int check_common(const std::string& what, int64_t num_heads, int64_t kv_num_heads,
                        int64_t head_size, const void* cos_cache, const void* sin_cache,
                        int64_t rotary_half, int64_t max_pos, const void* q_norm_weight,
                        const void* k_norm_weight, const float* k_scale, const float* v_scale,
                        int32_t cache_type, int32_t dtype) {
    int code;
    ORTMI_REQUIRE(num_heads > 0 && kv_num_heads > 0 && num_heads % kv_num_heads == 0 &&
                      num_heads <= 65535,
                  what + ": bad num_heads/kv_num_heads");
    ORTMI_REQUIRE(head_size > 0 && head_size % 16 == 0 && head_size <= 256,
                  what + ": head_size must be a multiple of 16 up to 256");
    ORTMI_REQUIRE(dtype == ORTMI_F32 || dtype == ORTMI_F16 || dtype == ORTMI_BF16,
                  what + ": dtype must be fp32, fp16 or bf16");
    ORTMI_REQUIRE(kvq::code_of(cache_type, code), what + ": cache must be int8, int4 or fp8 e4m3");
    ORTMI_REQUIRE(k_scale && v_scale, what + ": k_scale and v_scale must both be given");
    ORTMI_REQUIRE((cos_cache != nullptr) == (sin_cache != nullptr),
                  what + ": cos_cache and sin_cache must both be given");
    ORTMI_REQUIRE(!cos_cache || (rotary_half > 0 && 2 * rotary_half <= head_size && max_pos > 0),
                  what + ": rotary dims exceed head_size");
    ORTMI_REQUIRE((q_norm_weight != nullptr) == (k_norm_weight != nullptr),
                  what + ": q/k norm weights must both be given");
    return ORTMI_OK;
}

extern "C" size_t ortmi_group_query_attention_quantized_workspace_size(
    int64_t batch, int64_t seq_len, int64_t num_heads, int64_t kv_num_heads, int64_t head_size,
    int64_t total_kv) {
    if (batch <= 0 || seq_len <= 0 || kv_num_heads <= 0 || num_heads < kv_num_heads ||
        std::max({batch, seq_len, num_heads}) > INT32_MAX || !kvq::tile_head(head_size))
        return 0;
    size_t most = 0;  // over the types: fp32 has tiles of its own
    for (int dtype : {ORTMI_F32, ORTMI_F16}) {
        kvq::Params p{};
        p.B = (int)batch;
        p.S = (int)seq_len;
        p.H = (int)num_heads;
        p.KV = (int)kv_num_heads;
        p.hd = (int)head_size;
        p.dtype = dtype;
        most = std::max(most, kvq::plan_slabs(p, total_kv, nullptr));
    }
    return most;
}

extern "C" int ortmi_group_query_attention_quantized(
    const void* query, const void* key, const void* value, const void* past_key,
    const void* past_value, int64_t past_cap, int32_t total_sequence_length,
    const int32_t* seqlens_k, const void* cos_cache, const void* sin_cache, int64_t rotary_half,
    int64_t max_pos, const void* q_norm_weight, const void* k_norm_weight, float qk_norm_epsilon,
    const float* k_scale, const float* v_scale, int32_t k_per_channel, int32_t v_per_channel,
    int32_t cache_type, void* output, void* present_key, void* present_value, int64_t batch,
    int64_t seq_len, int64_t num_heads, int64_t kv_num_heads, int64_t head_size, float scale,
    int32_t rotary_interleaved, int32_t dtype, void* workspace, size_t workspace_bytes,
    void* stream) {
    const std::string what = "GroupQueryAttention (quantized)";
    if (int rc = check_common(what, num_heads, kv_num_heads, head_size, cos_cache, sin_cache,
                              rotary_half, max_pos, q_norm_weight, k_norm_weight, k_scale, v_scale,
                              cache_type, dtype))
        return rc;
    ORTMI_REQUIRE(batch >= 0 && seq_len >= 0 && past_cap >= 0, what + ": negative size");
    ORTMI_REQUIRE(batch < (1LL << 31) && seq_len < (1LL << 31) && past_cap < (1LL << 31) &&
                      batch * seq_len < (1LL << 31) && batch * seq_len * num_heads < (1LL << 31) && past_cap + seq_len < (1LL << 31) - 4096 &&
                      batch * kv_num_heads < (1LL << 31),
                  what + ": too many rows");
    if (batch == 0 || seq_len == 0) return ORTMI_OK;
    ORTMI_REQUIRE((key == nullptr) == (value == nullptr),
                  what + ": key and value must both be given (or both absent, packed QKV)");
    ORTMI_REQUIRE(query && output && present_key && present_value, what + ": null tensor");
    // The KV contract of GroupQueryAttention (rust/src/ops/attention.rs:636-651).
    int64_t vpast = (int64_t)total_sequence_length - seq_len;
    bool shared = false;
    if (vpast < 0 || vpast > past_cap) vpast = past_cap;
    else shared = past_cap > vpast;
    const int64_t pcap = shared ? past_cap : past_cap + seq_len;
    ORTMI_REQUIRE(!shared || vpast + seq_len <= past_cap,
                  what + ": total_sequence_length exceeds the KV buffer capacity");
    ORTMI_REQUIRE(vpast == 0 || (past_key && past_value), what + ": null past");
    ORTMI_REQUIRE(shared || past_cap == 0 ||
                      (present_key != past_key && present_value != past_value),
                  what + ": a growing cache needs present buffers of its own");
    ORTMI_REQUIRE(!cos_cache || vpast + seq_len <= max_pos,
                  what + ": position exceeds the cos/sin cache");
    const int64_t hd = head_size;
    hipStream_t st = as_stream(stream);
    kvq::Params p{};
    kvq::code_of(cache_type, p.code);
    const size_t esize = dtype == ORTMI_F32 ? 4 : 2;
    p.q = query;
    if (key) {
        p.k = key;
        p.v = value;
        p.q_tok = num_heads * hd;
        p.kv_tok = kv_num_heads * hd;
    } else {
        p.k = static_cast<const char*>(query) + (size_t)(num_heads * hd) * esize;
        p.v = static_cast<const char*>(p.k) + (size_t)(kv_num_heads * hd) * esize;
        p.q_tok = p.kv_tok = (num_heads + 2 * kv_num_heads) * hd;
    }
    p.kc = static_cast<uint8_t*>(present_key);
    p.vc = static_cast<uint8_t*>(present_value);
    p.cap = pcap;
    p.lens = seqlens_k;
    p.vpast = (int)vpast;
    p.S = (int)seq_len;
    p.B = (int)batch;
    p.H = (int)num_heads;
    p.KV = (int)kv_num_heads;
    p.hd = (int)hd;
    p.T = (int)(batch * seq_len);
    p.limit = (int)(vpast + seq_len);
    p.cos = cos_cache;
    p.sin = sin_cache;
    p.half = (int)rotary_half;
    p.interleaved = rotary_interleaved;
    p.max_pos = max_pos;
    p.qw = q_norm_weight;
    p.kw = k_norm_weight;
    p.eps = qk_norm_epsilon;
    p.ks = k_scale;
    p.vs = v_scale;
    p.k_chan = k_per_channel;
    p.v_chan = v_per_channel;
    p.scale = (scale != 0.f ? scale : 1.0f / sqrtf((float)hd)) * 1.44269504088896341f;
    p.dtype = dtype;
    p.out = output;
    const size_t need = kvq::plan_slabs(p, vpast + seq_len, static_cast<char*>(workspace));
    if (need && (!workspace || workspace_bytes < need))
        return fail(ORTMI_E_WORKSPACE, what + ": workspace too small");
    ORTMI_REQUIRE(!need || (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
                  what + ": workspace must be 16-byte aligned");
    const int64_t rb = kvq::row_bytes(p.code, (int)hd), slabs = batch * kv_num_heads;
    const int64_t kept = shared ? past_cap : vpast;  // rows of a past that is another buffer
    const void* past[2] = {past_key, past_value};
    void* present[2] = {present_key, present_value};
    for (int i = 0; i < 2; ++i)
        if (past[i] && present[i] != past[i])
            if (int rc = kvq::copy_slabs(past[i], present[i], slabs, past_cap * rb, pcap * rb,
                                         kept * rb, st))
                return rc;
    return kvq::attend<false>(p, st);
}

extern "C" size_t ortmi_paged_attention_quantized_workspace_size(
    int64_t num_tokens, int64_t batch, int64_t num_heads, int64_t kv_num_heads, int64_t head_size,
    int64_t max_context) {
    if (num_tokens <= 0 || batch <= 0 || kv_num_heads <= 0 || num_heads < kv_num_heads ||
        std::max({num_tokens, batch, num_heads}) > INT32_MAX || !kvq::tile_head(head_size))
        return 0;
    size_t most = 0;  // over the types: fp32 has tiles of its own
    for (int dtype : {ORTMI_F32, ORTMI_F16}) {
        kvq::Params p{};
        p.B = (int)batch;
        p.T = (int)num_tokens;
        p.H = (int)num_heads;
        p.KV = (int)kv_num_heads;
        p.hd = (int)head_size;
        p.limit = (int)std::min<int64_t>(max_context, INT32_MAX);
        p.dtype = dtype;
        most = std::max(most, kvq::plan_pages(p, nullptr));
    }
    return most;
}

extern "C" int ortmi_paged_attention_quantized(
    const void* query, const void* key, const void* value, void* key_cache, void* value_cache,
    int64_t num_blocks, int64_t block_size, const int32_t* cum_seqlens,
    const int32_t* past_seqlens, const int32_t* block_table, int64_t batch, int64_t max_blocks,
    int64_t num_tokens, int64_t max_context, const void* cos_cache, const void* sin_cache,
    int64_t rotary_half, int64_t max_pos, int32_t rotary_interleaved, const void* head_sink,
    const void* q_norm_weight, const void* k_norm_weight, float qk_norm_epsilon,
    const float* k_scale, const float* v_scale, int32_t k_per_channel, int32_t v_per_channel,
    int32_t cache_type, void* output, int64_t num_heads, int64_t kv_num_heads, int64_t head_size,
    float scale, int32_t dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const std::string what = "PagedAttention (quantized)";
    if (int rc = check_common(what, num_heads, kv_num_heads, head_size, cos_cache, sin_cache,
                              rotary_half, max_pos, q_norm_weight, k_norm_weight, k_scale, v_scale,
                              cache_type, dtype))
        return rc;
    ORTMI_REQUIRE(batch > 0 && block_size > 0 && num_blocks > 0 && max_blocks > 0,
                  what + ": bad cache or batch shape");
    ORTMI_REQUIRE(num_tokens >= 0 && num_tokens < (1LL << 31), what + ": bad token count");
    ORTMI_REQUIRE(batch < (1LL << 31) && block_size < (1LL << 31) && max_blocks < (1LL << 31),
                  what + ": bad cache or batch shape");
    ORTMI_REQUIRE(max_context > 0, what + ": max_context must be positive");
    ORTMI_REQUIRE(num_tokens * num_heads + 64 * batch < (1LL << 31), what + ": too many rows");
    ORTMI_REQUIRE(std::min<int64_t>(max_context, max_blocks * block_size) < (1LL << 31) - 4096,
                  what + ": too many keys");
    if (num_tokens == 0) return ORTMI_OK;
    ORTMI_REQUIRE(query && key && value && key_cache && value_cache && cum_seqlens &&
                      past_seqlens && block_table && output,
                  what + ": null tensor");
    kvq::Params p{};
    kvq::code_of(cache_type, p.code);
    p.q = query;
    p.k = key;
    p.v = value;
    p.q_tok = num_heads * head_size;
    p.kv_tok = kv_num_heads * head_size;
    p.kc = static_cast<uint8_t*>(key_cache);
    p.vc = static_cast<uint8_t*>(value_cache);
    p.bt = block_table;
    p.nblk = num_blocks;
    p.blk = (int)block_size;
    p.maxb = (int)max_blocks;
    p.cum = cum_seqlens;
    p.past = past_seqlens;
    p.B = (int)batch;
    p.H = (int)num_heads;
    p.KV = (int)kv_num_heads;
    p.hd = (int)head_size;
    p.T = (int)num_tokens;
    p.limit = (int)std::min<int64_t>(max_context, max_blocks * block_size);
    p.cos = cos_cache;
    p.sin = sin_cache;
    p.half = (int)rotary_half;
    p.interleaved = rotary_interleaved;
    p.max_pos = max_pos;
    p.qw = q_norm_weight;
    p.kw = k_norm_weight;
    p.eps = qk_norm_epsilon;
    p.ks = k_scale;
    p.vs = v_scale;
    p.k_chan = k_per_channel;
    p.v_chan = v_per_channel;
    p.scale = (scale != 0.f ? scale : 1.0f / sqrtf((float)head_size)) * 1.44269504088896341f;
    p.sink = head_sink;
    p.dtype = dtype;
    p.out = output;
    if (const uint32_t d = (uint32_t)(block_size / 16)) {
        p.blk_shift = 27;
        while (p.blk_shift < 58 && (1u << (p.blk_shift - 27)) < d) ++p.blk_shift;
        p.blk_mul = (uint32_t)(((1ULL << p.blk_shift) + d - 1) / d);
    }
    p.nsplit = 1;
    if (kvq::tile_head(head_size)) {
        const size_t need = kvq::plan_pages(p, static_cast<char*>(workspace));
        if (!workspace || workspace_bytes < need)
            return fail(ORTMI_E_WORKSPACE, what + ": workspace too small");
        ORTMI_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
                      what + ": workspace must be 16-byte aligned");
    }
    return kvq::attend<true>(p, as_stream(stream));
}
