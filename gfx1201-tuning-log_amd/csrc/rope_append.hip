// Position rotation and KV-cache append in one pass for gfx950: queries are rotated, new keys are
// rotated and, with the new values, written into the paged cache that the attention kernels read.
//
// Mathematics.  With R = rotary_dim and the table row of the token's position p holding
// cos(p f_i) (i < R / 2) and then sin(p f_i), a pair (a, b) of one head becomes
//   a' = a cos - b sin,  b' = b cos + a sin,
// (a, b) = (x[i], x[i + R / 2]), or (x[2 i], x[2 i + 1]) with `interleaved`; elements from R on are
// unchanged.  fp32 without contraction, so the results are those of the formula written out, and ONE
// rounding at the end: to bf16 (q_out, bf16 caches) or of y / scale to e4m3 (a rotation kernel before
// the cache write rounds keys to bf16 in between).  The table is an input: made once in 64 bits, it
// has no error that grows with the position.  A position outside the table gives NaN and reads nothing.
//
// Caches: e4m3 with one scale per tensor, bf16, or e4m3 with a power-of-two scale per 16 tokens and
// kv head ("block-scaled", below).
//
// What bounds it: bytes (q read and written, K and V read, codes written) for prompts, the chain of
// dependent loads for single tokens.  One thread takes 16 elements of one head as two pieces of
// 8 that hold whole pairs of either kind: (8 u, 8 u + R / 2) where halves are paired, else
// (16 u, 16 u + 8); each piece is one 16-byte load, and both table rows are read at 8 u.  Measured in a graph:
// 4096 tokens of 28 + 4 heads, bf16, 15.9 us (4.8 TB/s; a large copy 5.5), six prompts of 37..900, block-scaled, 10.7
// (4.2 TB/s), one token 3.3, 64 tokens block-scaled 4.7, 2048 tokens of 24 + 4 heads, e4m3, 9.8 (3.3 TB/s).  Four heads
// per thread, which read the table once, are no faster (15.6 and 10.9) and 7.5 for one token.
#include "fp8kv_common.h"
#include "fp8kv_status.h"
#include "e4m3_store.h"

namespace fp8kv {
namespace rope_append_detail {

constexpr int kThreads = 256;
constexpr int kGroup = 16;            // tokens that share a scale in a block-scaled cache
constexpr int kScaleMinExp = -100;    // smallest exponent of such a scale
constexpr int kBlkHead = 128;         // head size of a block-scaled cache

enum CacheKind { kE4m3 = 0, kBf16 = 1, kBlk = 2 };

struct Params {
    const uint16_t* q;          // bf16 bits; null: no queries
    uint16_t* q_out;
    const uint16_t* key;
    const uint16_t* value;
    uint8_t* kc;
    uint8_t* vc;
    int64_t q_stride, qo_stride, key_stride, value_stride;   // elements per token row
    int64_t sk0, sk1, sk2, sv0, sv1, sv2;                    // bytes
    const int64_t* positions;
    const void* table;          // null: no rotation
    int64_t table_stride;       // elements per position
    int64_t table_rows;
    int rot, interleaved;
    const int64_t* slots;       // per-tensor and bf16 caches
    const float* k_scale;
    const float* v_scale;
    uint8_t* kv_scales;         // block-scaled caches: [num_blocks][block_size / 16][hkv][2]
    const int32_t* qsl;
    const int32_t* seq_lens;
    const int32_t* bt;
    int64_t bt_stride, max_blocks, num_blocks;
    int num_tokens, num_seqs, hq, hkv, units, pblk, pshift;  // units: 16-element units per head
    int kv_wgs;                 // block-scaled: workgroups of cache items, ahead of those of queries
};

// Two pieces of 8 elements of one head, as fp32.
struct Unit {
    float x[2][8];
};

__device__ __forceinline__ void unpack8(const u32x4_t w, float (&x)[8])
{
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[2 * j] = __uint_as_float(w[j] << 16);
        x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
}

__device__ __forceinline__ u32x4_t pack8(const float (&x)[8])
{
    return (u32x4_t){pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
}

// Eight table entries from element i of row `row`.
template <bool TB16>
__device__ __forceinline__ void load_table(const Params& P, int64_t row, int i, float (&t)[8])
{
    if constexpr (TB16) {
        unpack8(load_16(static_cast<const uint16_t*>(P.table) + row * P.table_stride + i), t);
    } else {
        const float* p = static_cast<const float*>(P.table) + row * P.table_stride + i;
        const u32x4_t a = load_16(p), b = load_16(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            t[j] = __uint_as_float(a[j]);
            t[4 + j] = __uint_as_float(b[j]);
        }
    }
}

// First elements of unit u's two pieces within a head.
__device__ __forceinline__ void unit_places(const Params& P, bool rotated, int u, int& d0, int& d1)
{
    const bool halves = rotated && !P.interleaved;
    d0 = halves ? 8 * u : 16 * u;
    d1 = halves ? 8 * u + (P.rot >> 1) : 16 * u + 8;
}

// Rotates unit u (u < rot / 16) of a head to position pos.
template <bool TB16>
__device__ __forceinline__ void rotate(const Params& P, int64_t pos, int u, Unit& v)
{
#pragma clang fp contract(off)
    float c[8], s[8];
    if (pos >= 0 && pos < P.table_rows) {
        load_table<TB16>(P, pos, 8 * u, c);
        load_table<TB16>(P, pos, (P.rot >> 1) + 8 * u, s);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = s[j] = __builtin_nanf("");
    }
    if (P.interleaved) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float& a = v.x[j >> 2][2 * (j & 3)];
            float& b = v.x[j >> 2][2 * (j & 3) + 1];
            const float y = a * c[j] - b * s[j], z = b * c[j] + a * s[j];
            a = y;
            b = z;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float a = v.x[0][j], b = v.x[1][j];
            v.x[0][j] = a * c[j] - b * s[j];
            v.x[1][j] = b * c[j] + a * s[j];
        }
    }
}

// Query unit u of head h of token tok.
template <bool TB16>
__device__ __forceinline__ void query_unit(const Params& P, int tok, int h, int u)
{
    const bool rotated = 16 * u < P.rot;
    int d0, d1;
    unit_places(P, rotated, u, d0, d1);
    const int64_t e = (int64_t)h * (16 * P.units);
    const uint16_t* src = P.q + (int64_t)tok * P.q_stride + e;
    Unit v;
    unpack8(load_16(src + d0), v.x[0]);
    unpack8(load_16(src + d1), v.x[1]);
    if (rotated) rotate<TB16>(P, P.positions[tok], u, v);
    uint16_t* dst = P.q_out + (int64_t)tok * P.qo_stride + e;
    *reinterpret_cast<u32x4_t*>(dst + d0) = pack8(v.x[0]);
    *reinterpret_cast<u32x4_t*>(dst + d1) = pack8(v.x[1]);
}

// e4m3 codes of eight values.
__device__ __forceinline__ u32x2_t codes8(const float (&x)[8])
{
    return (u32x2_t){e4m3_pair(x[0], x[1]) | (e4m3_pair(x[2], x[3]) << 16),
                     e4m3_pair(x[4], x[5]) | (e4m3_pair(x[6], x[7]) << 16)};
}

// ---- caches with one scale per tensor, and bf16 caches -------------------------------------------
// Items are (token, head row, unit), head rows counting queries, then keys, then values.
template <int KIND, bool TB16>
__global__ void __launch_bounds__(kThreads)
rope_append_kernel(Params P)
{
    const int rows = (P.q ? P.hq : 0) + 2 * P.hkv;
    const int per_tok = rows * P.units;
    const int n_items = P.num_tokens * per_tok;
    for (int it = blockIdx.x * kThreads + threadIdx.x; it < n_items; it += gridDim.x * kThreads) {
        const int tok = it / per_tok;
        const int r = it - tok * per_tok;
        int h = r / P.units;
        const int u = r - h * P.units;
        if (P.q) {
            if (h < P.hq) {
                query_unit<TB16>(P, tok, h, u);
                continue;
            }
            h -= P.hq;
        }
        const bool isv = h >= P.hkv;
        if (isv) h -= P.hkv;
        const int64_t s = P.slots[tok];
        const int64_t blk = s >> P.pshift, slot = s & (P.pblk - 1);
        if (s < 0 || blk >= P.num_blocks) continue;
        const bool rotated = !isv && 16 * u < P.rot;
        int d0, d1;
        unit_places(P, rotated, u, d0, d1);
        const int64_t e = (int64_t)h * (16 * P.units);
        const uint16_t* src = (isv ? P.value + (int64_t)tok * P.value_stride : P.key + (int64_t)tok * P.key_stride) + e;
        Unit v;
        unpack8(load_16(src + d0), v.x[0]);
        unpack8(load_16(src + d1), v.x[1]);
        if (rotated) rotate<TB16>(P, P.positions[tok], u, v);
        uint8_t* dst = isv ? P.vc + blk * P.sv0 + slot * P.sv1 + (int64_t)h * P.sv2
                           : P.kc + blk * P.sk0 + slot * P.sk1 + (int64_t)h * P.sk2;
        if constexpr (KIND == kBf16) {
            *reinterpret_cast<u32x4_t*>(dst + 2 * d0) = pack8(v.x[0]);
            *reinterpret_cast<u32x4_t*>(dst + 2 * d1) = pack8(v.x[1]);
        } else {
            const float scale = isv ? P.v_scale[0] : P.k_scale[0];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v.x[0][j] /= scale;
                v.x[1][j] /= scale;
            }
            *reinterpret_cast<u32x2_t*>(dst + d0) = codes8(v.x[0]);
            *reinterpret_cast<u32x2_t*>(dst + d1) = codes8(v.x[1]);
        }
    }
}

// ---- block-scaled caches -------------------------------------------------------------------------
// A group of 16 consecutive tokens of a sequence (always inside one cache block) has, per kv head and
// for K and V apart, one power-of-two scale, kept as an e8m0 byte.  A wave owns one group of one head
// of K or V, so nobody else reads or writes its bytes: the new rows' largest finite |y| gives the
// exponent they need, ceil(log2(amax / 448)) (at least -100); tokens that were in the group before
// keep their scale unless the new rows need a larger one, and then their codes are re-rounded once, by
// an exact power of two (only codes that become subnormal change); a group whose first token is
// new takes the exponent its new rows need.  A power of two costs up to a factor of two of the range, where
// e4m3's relative precision does not depend on the scale, and makes growing a scale nearly lossless.
//
// Sequence of cache item `idx`: sequence s has the items from qsl[s] / 16 + 2 s on, at least as many
// as the groups its new tokens can touch ((n + 30) / 16 at most).  64 lanes probe 64 sequences at once.
__device__ __forceinline__ int find_sequence(const Params& P, int idx, int lane)
{
    int lo = 0, step = 1;
    while (step * 64 < P.num_seqs) step *= 64;
    for (;; step >>= 6) {
        const int s = lo + lane * step;
        const bool below = s < P.num_seqs && (P.qsl[s] >> 4) + 2 * s <= idx;
        const int n = __popcll(__ballot(below));            // the probes ascend: the first n are at or below idx
        if (n == 0) return -1;
        lo += (n - 1) * step;
        if (step == 1) return lo;
    }
}

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}

// Exponent of the smallest power of two s with amax / s <= 448 = 1.75 * 2^8, for a finite amax.
__device__ __forceinline__ int needed_exp(float amax)
{
    const uint32_t b = __float_as_uint(amax);
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return e < kScaleMinExp ? kScaleMinExp : e;
}

template <bool TB16>
__device__ void blk_item(const Params& P, int item, int lane)
{
    const int x = item & 1;
    int idx = (item >> 1) / P.hkv;
    const int h = (item >> 1) - idx * P.hkv;
    const int seq = find_sequence(P, idx, lane);
    if (seq < 0) return;
    const int start = P.qsl[seq], n = P.qsl[seq + 1] - start;
    const int len = P.seq_lens[seq], first = len - n;        // position of the sequence's first new token
    const int g = (first >> 4) + idx - ((start >> 4) + 2 * seq);
    const int t0 = kGroup * g;                               // the group's first token
    if (start < 0 || n <= 0 || start + n > P.num_tokens || g < 0 || t0 >= len) return;
    const int64_t col = t0 >> P.pshift;
    if (col >= P.max_blocks) return;
    const int64_t blk = P.bt[(int64_t)seq * P.bt_stride + col];
    if (blk < 0 || blk >= P.num_blocks) return;
    const int slot0 = t0 & (P.pblk - 1);
    uint8_t* const scale = P.kv_scales + ((blk * (P.pblk / kGroup) + slot0 / kGroup) * P.hkv + h) * 2 + x;
    uint8_t* const rows = x ? P.vc + blk * P.sv0 + slot0 * P.sv1 + (int64_t)h * P.sv2
                            : P.kc + blk * P.sk0 + slot0 * P.sk1 + (int64_t)h * P.sk2;
    const int64_t row_stride = x ? P.sv1 : P.sk1;

    const int u = lane & 7;
    const bool rotated = x == 0 && 16 * u < P.rot;
    int d0, d1;
    unit_places(P, rotated, u, d0, d1);
    const bool has_old = t0 < first;
    const uint32_t before = has_old ? *scale : 0u;
    // lane (token lane / 8 + 8 j, unit lane % 8)
    Unit v[2];
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int pos = t0 + (lane >> 3) + 8 * j;
        if (pos < first || pos >= len) continue;
        const int64_t tok = start + (pos - first);
        const uint16_t* src = (x ? P.value + tok * P.value_stride : P.key + tok * P.key_stride) + h * kBlkHead;
        unpack8(load_16(src + d0), v[j].x[0]);
        unpack8(load_16(src + d1), v[j].x[1]);
        if (rotated) rotate<TB16>(P, P.positions[tok], u, v[j]);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float a = fabsf(v[j].x[i >> 3][i & 7]);
            amax = fmaxf(amax, a <= 3.4028235e38f ? a : 0.f);
        }
    }
    uint32_t now = (uint32_t)(needed_exp(wave_max(amax)) + 127);
    if (has_old && before > now) now = before;
    const float inv = e8m0_to_f32(now == 255u ? 255u : 254u - now);
    const bool grown = has_old && now != before;
    const int diff = (int)before - (int)now;                 // factor of the old codes, 2^diff
    const float shrink = __uint_as_float((uint32_t)(127 + (diff < -100 ? -100 : diff)) << 23);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int row = (lane >> 3) + 8 * j, pos = t0 + row;
        uint8_t* dst = rows + row * row_stride;
        if (pos >= first && pos < len) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[j].x[i >> 3][i & 7] *= inv;
            *reinterpret_cast<u32x2_t*>(dst + d0) = codes8(v[j].x[0]);
            *reinterpret_cast<u32x2_t*>(dst + d1) = codes8(v[j].x[1]);
        } else if (grown && pos < first) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                u32x2_t* p = reinterpret_cast<u32x2_t*>(dst + (half ? d1 : d0));
                const u32x2_t w = *p;
                float y[8];
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[d], false);
                    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[d], true);
                    y[4 * d] = a[0] * shrink;
                    y[4 * d + 1] = a[1] * shrink;
                    y[4 * d + 2] = b[0] * shrink;
                    y[4 * d + 3] = b[1] * shrink;
                }
                *p = codes8(y);
            }
        }
    }
    if (lane == 0 && (!has_old || grown)) *scale = (uint8_t)now;
}

template <bool TB16>
__global__ void __launch_bounds__(kThreads)
rope_append_blk_kernel(Params P)
{
    const int lane = threadIdx.x & 63;
    if ((int)blockIdx.x < P.kv_wgs) {
        const int item = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        blk_item<TB16>(P, item, lane);               // items past the last sequence's find no group
        return;
    }
    // query units; rows behind the last sequence are left as they are
    const int tokens = min(P.num_tokens, P.qsl[P.num_seqs]);
    const int per_tok = P.hq * P.units;
    const int n_items = tokens * per_tok;
    const int stride = (gridDim.x - P.kv_wgs) * kThreads;
    for (int it = (blockIdx.x - P.kv_wgs) * kThreads + threadIdx.x; it < n_items; it += stride) {
        const int tok = it / per_tok;
        const int r = it - tok * per_tok;
        const int h = r / P.units;
        query_unit<TB16>(P, tok, h, r - h * P.units);
    }
}

constexpr int kMaxWgs = 4096;        // grid-stride beyond: 16 waves per CU

// What every entry point checks; strides in elements of elem_bytes bytes.  Fills P.
int setup(Params& P, const void* q, int64_t q_row_stride, void* q_out, int64_t q_out_row_stride, const void* key,
          int64_t key_row_stride, const void* value, int64_t value_row_stride, void* k_cache, void* v_cache, int64_t sk0,
          int64_t sk1, int64_t sk2, int64_t sv0, int64_t sv1, int64_t sv2, const int64_t* positions, const void* cos_sin,
          int64_t cos_sin_row_stride, int cos_sin_bf16, int64_t num_positions, int rotary_dim, int interleaved, int num_tokens,
          int num_q_heads, int num_kv_heads, int head_size, int block_size, int64_t num_blocks, int elem_bytes)
{
    if (!key || !value || !k_cache || !v_cache) return FP8KV_ERR_ARG;
    if (num_tokens < 0 || num_kv_heads < 1 || head_size < 1 || block_size < 1 || num_blocks < 0) return FP8KV_ERR_ARG;
    if (q && (!q_out || num_q_heads < 1)) return FP8KV_ERR_ARG;
    if (cos_sin && (!positions || num_positions < 1 || rotary_dim < 1)) return FP8KV_ERR_ARG;
    if (head_size % 16 != 0 || (block_size & (block_size - 1)) != 0) return FP8KV_ERR_SHAPE;
    if (cos_sin && (rotary_dim % 16 != 0 || rotary_dim > head_size)) return FP8KV_ERR_SHAPE;
    const int64_t rows = (q ? num_q_heads : 0) + 2 * (int64_t)num_kv_heads;
    if (num_tokens * rows * (head_size / 16) + (int64_t)kMaxWgs * kThreads >= ((int64_t)1 << 31)) return FP8KV_ERR_SHAPE;
    if (!aligned(key, 16) || !aligned(value, 16) || ((key_row_stride | value_row_stride) & 7)) return FP8KV_ERR_ALIGN;
    if (q && (!aligned(q, 16) || !aligned(q_out, 16) || ((q_row_stride | q_out_row_stride) & 7))) return FP8KV_ERR_ALIGN;
    if (cos_sin && (!aligned(cos_sin, 16) || (cos_sin_row_stride & (cos_sin_bf16 ? 7 : 3)))) return FP8KV_ERR_ALIGN;
    const int64_t kv_row = (int64_t)num_kv_heads * head_size, q_row = (int64_t)num_q_heads * head_size;
    if (key_row_stride < kv_row || value_row_stride < kv_row) return FP8KV_ERR_ARG;
    if (q && (q_row_stride < q_row || q_out_row_stride < q_row)) return FP8KV_ERR_ARG;
    if (cos_sin && cos_sin_row_stride < rotary_dim) return FP8KV_ERR_ARG;
    sk0 *= elem_bytes; sk1 *= elem_bytes; sk2 *= elem_bytes;
    sv0 *= elem_bytes; sv1 *= elem_bytes; sv2 *= elem_bytes;
    if (!aligned(k_cache, 16) || ((sk0 | sk1 | sk2) & 15)) return FP8KV_ERR_ALIGN;
    const int64_t vmask = 8 * elem_bytes - 1;
    if (!aligned(v_cache, (uintptr_t)vmask + 1) || ((sv0 | sv1 | sv2) & vmask)) return FP8KV_ERR_ALIGN;

    P = Params{};
    P.q = static_cast<const uint16_t*>(q);
    P.q_out = static_cast<uint16_t*>(q_out);
    P.key = static_cast<const uint16_t*>(key);
    P.value = static_cast<const uint16_t*>(value);
    P.kc = static_cast<uint8_t*>(k_cache);
    P.vc = static_cast<uint8_t*>(v_cache);
    P.q_stride = q_row_stride;
    P.qo_stride = q_out_row_stride;
    P.key_stride = key_row_stride;
    P.value_stride = value_row_stride;
    P.sk0 = sk0; P.sk1 = sk1; P.sk2 = sk2;
    P.sv0 = sv0; P.sv1 = sv1; P.sv2 = sv2;
    P.positions = positions;
    P.table = cos_sin;
    P.table_stride = cos_sin_row_stride;
    P.table_rows = num_positions;
    P.rot = cos_sin ? rotary_dim : 0;
    P.interleaved = interleaved ? 1 : 0;
    P.num_blocks = num_blocks;
    P.num_tokens = num_tokens;
    P.hq = q ? num_q_heads : 0;
    P.hkv = num_kv_heads;
    P.units = head_size / 16;
    P.pblk = block_size;
    P.pshift = __builtin_ctz((unsigned)block_size);
    return FP8KV_OK;
}

inline unsigned wgs_for(int64_t items)
{
    const int64_t n = (items + kThreads - 1) / kThreads;
    return (unsigned)(n < kMaxWgs ? n : kMaxWgs);
}

template <int KIND>
int launch(const Params& P, bool table_bf16, hipStream_t stream)
{
    const dim3 grid(wgs_for((int64_t)P.num_tokens * (P.hq + 2 * P.hkv) * P.units));
    begin_launch();
    if (table_bf16) launch_kernel(rope_append_kernel<KIND, true>, grid, dim3(kThreads), 0, stream, P);
    else launch_kernel(rope_append_kernel<KIND, false>, grid, dim3(kThreads), 0, stream, P);
    return finish_launch();
}

}  // namespace rope_append_detail
}  // namespace fp8kv

using namespace fp8kv;
using namespace fp8kv::rope_append_detail;

extern "C" int fp8kv_rope_append(const void* q, int64_t q_row_stride, void* q_out, int64_t q_out_row_stride,
                                 const void* key, int64_t key_row_stride, const void* value, int64_t value_row_stride,
                                 void* k_cache, void* v_cache, int64_t sk0, int64_t sk1, int64_t sk2, int64_t sv0,
                                 int64_t sv1, int64_t sv2, const int64_t* positions, const void* cos_sin,
                                 int64_t cos_sin_row_stride, int cos_sin_bf16, int64_t num_positions, int rotary_dim,
                                 int interleaved, const int64_t* slot_mapping, const float* k_scale, const float* v_scale,
                                 int num_tokens, int num_q_heads, int num_kv_heads, int head_size, int block_size,
                                 int64_t num_blocks, void* stream)
{
    if (!slot_mapping || !k_scale || !v_scale) return FP8KV_ERR_ARG;
    Params P;
    const int st = setup(P, q, q_row_stride, q_out, q_out_row_stride, key, key_row_stride, value, value_row_stride, k_cache,
                         v_cache, sk0, sk1, sk2, sv0, sv1, sv2, positions, cos_sin, cos_sin_row_stride, cos_sin_bf16,
                         num_positions, rotary_dim, interleaved, num_tokens, num_q_heads, num_kv_heads, head_size, block_size,
                         num_blocks, 1);
    if (st != FP8KV_OK || num_tokens == 0) return st;
    P.slots = slot_mapping;
    P.k_scale = k_scale;
    P.v_scale = v_scale;
    return launch<kE4m3>(P, cos_sin_bf16 != 0, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int fp8kv_rope_append_bf16(const void* q, int64_t q_row_stride, void* q_out, int64_t q_out_row_stride,
                                      const void* key, int64_t key_row_stride, const void* value, int64_t value_row_stride,
                                      void* k_cache, void* v_cache, int64_t sk0, int64_t sk1, int64_t sk2, int64_t sv0,
                                      int64_t sv1, int64_t sv2, const int64_t* positions, const void* cos_sin,
                                      int64_t cos_sin_row_stride, int cos_sin_bf16, int64_t num_positions, int rotary_dim,
                                      int interleaved, const int64_t* slot_mapping, int num_tokens, int num_q_heads,
                                      int num_kv_heads, int head_size, int block_size, int64_t num_blocks, void* stream)
{
    if (!slot_mapping) return FP8KV_ERR_ARG;
    Params P;
    const int st = setup(P, q, q_row_stride, q_out, q_out_row_stride, key, key_row_stride, value, value_row_stride, k_cache,
                         v_cache, sk0, sk1, sk2, sv0, sv1, sv2, positions, cos_sin, cos_sin_row_stride, cos_sin_bf16,
                         num_positions, rotary_dim, interleaved, num_tokens, num_q_heads, num_kv_heads, head_size, block_size,
                         num_blocks, 2);
    if (st != FP8KV_OK || num_tokens == 0) return st;
    P.slots = slot_mapping;
    return launch<kBf16>(P, cos_sin_bf16 != 0, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int fp8kv_rope_append_blk(const void* q, int64_t q_row_stride, void* q_out, int64_t q_out_row_stride,
                                     const void* key, int64_t key_row_stride, const void* value, int64_t value_row_stride,
                                     void* k_cache, void* v_cache, int64_t sk0, int64_t sk1, int64_t sk2, int64_t sv0,
                                     int64_t sv1, int64_t sv2, const int64_t* positions, const void* cos_sin,
                                     int64_t cos_sin_row_stride, int cos_sin_bf16, int64_t num_positions, int rotary_dim,
                                     int interleaved, void* kv_scales, const int32_t* query_start_loc,
                                     const int32_t* seq_lens, const int32_t* block_table, int64_t bt_stride, int max_blocks,
                                     int num_seqs, int num_tokens, int num_q_heads, int num_kv_heads, int head_size,
                                     int block_size, int64_t num_blocks, void* stream)
{
    if (!kv_scales || !query_start_loc || !seq_lens || !block_table) return FP8KV_ERR_ARG;
    if (num_seqs < 0 || max_blocks < 0 || bt_stride < 0) return FP8KV_ERR_ARG;
    Params P;
    const int st = setup(P, q, q_row_stride, q_out, q_out_row_stride, key, key_row_stride, value, value_row_stride, k_cache,
                         v_cache, sk0, sk1, sk2, sv0, sv1, sv2, positions, cos_sin, cos_sin_row_stride, cos_sin_bf16,
                         num_positions, rotary_dim, interleaved, num_tokens, num_q_heads, num_kv_heads, head_size, block_size,
                         num_blocks, 1);
    if (st != FP8KV_OK) return st;
    if (head_size != kBlkHead || block_size < kGroup) return FP8KV_ERR_SHAPE;
    if (num_tokens == 0 || num_seqs == 0) return FP8KV_OK;
    P.kv_scales = static_cast<uint8_t*>(kv_scales);
    P.qsl = query_start_loc;
    P.seq_lens = seq_lens;
    P.bt = block_table;
    P.bt_stride = bt_stride;
    P.max_blocks = max_blocks;
    P.num_seqs = num_seqs;
    const int64_t items = ((int64_t)(num_tokens / 16) + 2 * (int64_t)num_seqs) * num_kv_heads * 2;
    if (items >= ((int64_t)1 << 31)) return FP8KV_ERR_SHAPE;
    P.kv_wgs = (int)((items + kThreads / 64 - 1) / (kThreads / 64));
    const dim3 grid((unsigned)P.kv_wgs + wgs_for((int64_t)num_tokens * P.hq * P.units));
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    begin_launch();
    if (cos_sin_bf16) launch_kernel(rope_append_blk_kernel<true>, grid, dim3(kThreads), 0, hs, P);
    else launch_kernel(rope_append_blk_kernel<false>, grid, dim3(kThreads), 0, hs, P);
    return finish_launch();
}
