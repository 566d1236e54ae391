// What the key-split prefill kernels share (prefill_attn.hip, prefill_visible.hip): the launch parameters, the
// placement of raw K/V tiles in the LDS ring and the copies into it, the lazily rescaled softmax
// state, and the shapes by GQA.
#pragma once
#include "fp8kv_common.h"
#include "attn_common.h"
#include "fp8kv_status.h"

namespace fp8kv {
namespace prefill_detail {

constexpr int kD = 128;
constexpr int kBN = 32;                       // keys per tile
constexpr int kMaxGqa = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleSlack = 8.f;          // log2 growth of a row max tolerated before rescaling
constexpr int kTileBytes = 8192;              // raw fp8 tile: K rows 0..31 (4 KB), then V rows (4 KB)

struct Params {
    const __bf16* q;
    const uint8_t* k;
    const uint8_t* v;
    __bf16* out;
    const int32_t* cu_q;        // [NS + 1] or null (single sequence: q0_host / qlen_host)
    const int32_t* seq_lens;    // [NS] total context of each sequence (new tokens included)
    const int32_t* bt;
    const float* k_scale;
    const float* v_scale;
    int64_t q_stride, o_stride, bt_stride;
    int64_t sk0, sk1, sk2, sv0, sv1, sv2;
    float sm_scale;
    int hkv, gqa, pblk, pshift, nb;
    int paired;                 // 1: nb == 2 and the two 16-token blocks are r and n16 - 1 - r
    int ntb_grid;               // token blocks per (sequence, kv head) the grid covers
    int xcd_map;                // 1: kv head from the XCD index (8 % HKV == 0), see kernel
    int q0_host, qlen_host;
};

// ---- raw fp8 tile placement in LDS ---------------------------------------------------------------
// The tile is copied by eight 1 KB global_load_lds_dwordx4 instructions: I = 0..3 carry K rows
// 8I .. 8I+7, I = 4..7 carry V rows 8(I-4) .. +7; lane l of an instruction lands at 16 l.  Which
// (row, 16-byte chunk) a lane fetches is chosen so that the fragment reads below are free of bank
// conflicts:
//   K: row r (0..7), chunk c at slot 8 r + (c ^ (r >> 1)) - the 16 rows one fragment read touches
//      (same chunk) fall in 16 distinct 16-byte bank groups;
//   V: row r at slot 8 rho(r) + c with rho(r) = 2 (r & 3) + (r >> 2) - the rows 4p + j one
//      transposing read touches (p = 0..3) alternate between the two bank halves.
__host__ __device__ inline int k_slot(int r, int c) { return 8 * r + (c ^ (r >> 1)); }
__host__ __device__ inline int v_slot(int r, int c) { return 8 * (2 * (r & 3) + (r >> 2)) + c; }

// (row within the 8-row group, chunk) lane l of a K or V copy instruction fetches.
__device__ __forceinline__ void dma_lane_rc(bool is_v, int lane, int& r, int& c)
{
    if (!is_v) {
        r = lane >> 3;
        c = (lane & 7) ^ (r >> 1);
    } else {
        const int rho = lane >> 3;
        c = lane & 7;
        r = (rho >> 1) + 4 * (rho & 1);
    }
}

// global_load_lds_dwordx4 issued as inline assembly, in its scalar-base form: lane i's 16 bytes
// from sbase + voff (sbase a wave-uniform 64-bit address, voff this lane's 32-bit offset, so no
// 64-bit address arithmetic per lane) land at lds_dst + 16 i.  The compiler does not see this
// copy, so it inserts no wait for it: in particular no vmcnt(0) before LDS reads it cannot prove
// disjoint from the copy's destination, which would drain the whole prefetch ring each tile.
// Completion is tracked only by the kernel's explicit vmcnt waits (vmcnt counts in issue order,
// so the compiler's own waits for its loads stay correct - at worst they wait longer).  lds_dst
// must be wave-uniform.
__device__ __forceinline__ void dma16_saddr(const void* sbase, uint32_t voff, unsigned char* lds_dst)
{
    const uint32_t lds_addr = (uint32_t)(uintptr_t)(lds_void_t*)lds_dst;
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(lds_addr), "v"(voff), "s"(sbase) : "memory", "m0");
}

// Workgroup barrier that orders LDS only.  __syncthreads() carries a workgroup-scope release
// fence, which on gfx950 waits for every outstanding vector-memory operation - including the
// async tile copies still in flight for later tiles.  Here each wave has already waited for its
// own copies of the tile it is about to read (vmcnt), so the barrier only needs this wave's LDS
// reads of the previous tile to have completed (lgkmcnt) before the slot is overwritten; the
// "memory" clobber keeps the compiler from moving LDS accesses across it.
__device__ __forceinline__ void lds_barrier()
{
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

constexpr int kSplitWaves = 8;

constexpr int kStageFloats = 8 * 64 * 4 + 64;        // one row-set: o [n][lane][4], then l [lane]

// Running-max floor of the key-split kernel: finite, so that no -inf ever enters the softmax
// arithmetic (exp2(kMaxFloor - m) is 0 for any real row max m, and a row that has seen no key
// keeps l = 0 and o = 0).
constexpr float kMaxFloor = -3e38f;
// Smallest softmax factor of a row, so that -inf * factor stays -inf where a scale is 0: times any score it
// is applied to, it is 0 to exp2.
constexpr float kMinFactor16 = 1.4e-45f;

// max without the NaN-quieting canonicalisation the compiler adds to fmaxf of values that come
// from MFMA results or lane swaps (finite K and Q give no NaN score; that of a scale joins at the output).
__device__ __forceinline__ float max_raw(float a, float b)
{
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ float max3_raw(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float max_xor16_32_raw(float v)
{
    const uint32_t b = __float_as_uint(v);
    const auto r16 = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    const float m = max_raw(__uint_as_float(r16[0]), __uint_as_float(r16[1]));
    const uint32_t c = __float_as_uint(m);
    const auto r32 = __builtin_amdgcn_permlane32_swap(c, c, false, false);
    return max_raw(__uint_as_float(r32[0]), __uint_as_float(r32[1]));
}

// Lazy rescale of RS row-sets for one tile of raw scores sc (-inf where masked), whose factor to log2 units is
// qkr > 0: the accumulators move to a new reference max only when a row's max grew by more than kRescaleSlack.
template <int RS>
__device__ __forceinline__ void rescale_rows(const f32x4_t (&sc)[RS][2], float (&m_run)[RS], float (&l_run)[RS],
                                             f32x4_t (&o)[RS][8], const float (&qkr)[RS])
{
    float m8[RS];
    bool any_need = false;
#pragma unroll
    for (int j = 0; j < RS; ++j) {
        float m = max3_raw(sc[j][0][0], sc[j][0][1], sc[j][0][2]);
        m = max3_raw(m, sc[j][0][3], sc[j][1][0]);
        m = max3_raw(m, sc[j][1][1], sc[j][1][2]);
        m8[j] = max_raw(m, sc[j][1][3]);
        any_need |= m8[j] * qkr[j] > m_run[j] + kRescaleSlack;
    }
    if (__any(any_need)) {
#pragma unroll
        for (int j = 0; j < RS; ++j) {
            const float mc = max_xor16_32_raw(m8[j]) * qkr[j];    // -inf for a fully masked row
            const bool need = mc > m_run[j] + kRescaleSlack;
            const float m_new = need ? mc : m_run[j];
            const float alpha = __builtin_amdgcn_exp2f(m_run[j] - m_new);
            l_run[j] *= alpha;
#pragma unroll
            for (int n = 0; n < 8; ++n) o[j][n] *= alpha;
            m_run[j] = m_new;
        }
    }
}

constexpr int kTileBytes16 = 16384;
__device__ __forceinline__ int b16_slot(int row, int c) { return row * 256 + 16 * (c ^ (row & 15)); }

// Key-split shapes (RS row-sets per wave, NG head groups) for gqa = RS * NG.
struct SplitShape {
    int rs, ng;
};
constexpr SplitShape kSplitShapes[] = {{3, 2}, {3, 4}, {2, 2}, {2, 4}, {2, 8}};
constexpr int kNumSplitShapes = sizeof(kSplitShapes) / sizeof(kSplitShapes[0]);

// Key-split shape of a GQA: its own, or the smallest that holds its heads (with row-sets repeated, or
// two or four token blocks per workgroup at GQA 2 and 1).
inline int split_shape_for(int gqa)
{
    return gqa <= 4 ? 2 : gqa <= 6 ? 0 : gqa <= 8 ? 3 : gqa <= 12 ? 1 : 4;
}
inline bool split_shape_exact(int gqa)
{
    const SplitShape s = kSplitShapes[split_shape_for(gqa)];
    return s.rs * s.ng == gqa;
}
inline int split_blocks(int gqa) { return gqa <= 2 ? 4 / gqa : 1; }

// Workgroups of the key-split kernel resident at once on a gfx950 part (256 CUs, one each).
constexpr int kSplitRoundWorkgroups = 256;

// Token-block ranks per (sequence, kv head) padded for the XCD-aware grid (8 % HKV == 0).
inline int split_xcd_per(int hkv) { return (hkv <= 8 && 8 % hkv == 0) ? 8 / hkv : 1; }

// Workgroups of a grid of n ranks per sequence and kv head, and whether the key-split kernel runs them in
// one round: with one 16-token block each, n blocks, or with pairs of them, (n + 1) / 2.
inline int64_t split_workgroups(int n, int hkv, int num_seqs)
{
    const int per = split_xcd_per(hkv);
    return (int64_t)((n + per - 1) / per * per) * hkv * num_seqs;
}
inline bool split_single_blocks_fit(int n16, int hkv, int num_seqs)
{
    return split_workgroups(n16, hkv, num_seqs) <= kSplitRoundWorkgroups;
}
inline bool split_pairs_fit(int n16, int hkv, int num_seqs)
{
    return split_workgroups((n16 + 1) / 2, hkv, num_seqs) <= kSplitRoundWorkgroups;
}

// What every prefill entry point checks (cache strides in bytes).
inline int check_common(const void* q, const void* k_cache, const void* v_cache, void* out,
                 int64_t q_row_stride, int64_t sk0, int64_t sk1, int64_t sk2, int64_t sv0,
                 int64_t sv1, int64_t sv2, const int32_t* block_table, int64_t bt_stride,
                 const float* k_scale, const float* v_scale, int num_q_heads, int num_kv_heads,
                 int head_size, int block_size, int64_t out_row_stride)
{
    if (!q || !k_cache || !v_cache || !out || !block_table || !k_scale || !v_scale) return FP8KV_ERR_ARG;
    if (num_kv_heads < 1 || num_q_heads < 1 || block_size < 1 || bt_stride < 0) return FP8KV_ERR_ARG;
    if (num_kv_heads > 65535) return FP8KV_ERR_SHAPE;
    if (head_size != kD || num_q_heads % num_kv_heads != 0) return FP8KV_ERR_SHAPE;
    if (num_q_heads / num_kv_heads > kMaxGqa) return FP8KV_ERR_SHAPE;
    if (block_size < 16 || (block_size & (block_size - 1)) != 0) return FP8KV_ERR_SHAPE;
    if (!aligned(k_cache, 16) || !aligned(v_cache, 8) || !aligned(q, 16) || !aligned(out, 16))
        return FP8KV_ERR_ALIGN;
    if ((sk0 | sk1 | sk2) & 15) return FP8KV_ERR_ALIGN;
    if ((sv0 | sv1 | sv2) & 7) return FP8KV_ERR_ALIGN;
    if ((q_row_stride & 7) || (out_row_stride & 7)) return FP8KV_ERR_ALIGN;
    // The tile copies address a row within its cache block with a 32-bit offset.
    if (sk1 < 0 || sv1 < 0 || (int64_t)(block_size - 1) * (sk1 > sv1 ? sk1 : sv1) + 128 >= ((int64_t)1 << 32))
        return FP8KV_ERR_SHAPE;
    return FP8KV_OK;
}

inline Params make_params(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                   int64_t sk0, int64_t sk1, int64_t sk2, int64_t sv0, int64_t sv1, int64_t sv2,
                   void* out, int64_t out_row_stride, const int32_t* block_table, int64_t bt_stride,
                   const float* k_scale, const float* v_scale, float sm_scale, int num_q_heads,
                   int num_kv_heads, int block_size)
{
    Params P;
    P.q = static_cast<const __bf16*>(q);
    P.k = static_cast<const uint8_t*>(k_cache);
    P.v = static_cast<const uint8_t*>(v_cache);
    P.out = static_cast<__bf16*>(out);
    P.cu_q = nullptr;
    P.seq_lens = nullptr;
    P.bt = block_table;
    P.k_scale = k_scale;
    P.v_scale = v_scale;
    P.q_stride = q_row_stride;
    P.o_stride = out_row_stride;
    P.bt_stride = bt_stride;
    P.sk0 = sk0; P.sk1 = sk1; P.sk2 = sk2;
    P.sv0 = sv0; P.sv1 = sv1; P.sv2 = sv2;
    P.sm_scale = sm_scale;
    P.hkv = num_kv_heads;
    P.gqa = num_q_heads / num_kv_heads;
    P.pblk = block_size;
    P.pshift = __builtin_ctz((unsigned)block_size);
    P.nb = 1;
    P.paired = 0;
    P.ntb_grid = 0;
    P.xcd_map = 0;
    P.q0_host = 0;
    P.qlen_host = 0;
    return P;
}

}  // namespace prefill_detail
}  // namespace fp8kv
