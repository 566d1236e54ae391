// Causal prefill attention over the visible keys of each query (a sliding window and the first tokens, or
// everything before it), on e4m3 caches with one scale per tensor, block-scaled e4m3 caches and bf16
// caches, for gfx950.
//
// Mathematics.  Query i of a sequence is token p = seq_len - qlen + i.  It sees the keys t <= p with
// t > p - window or t < sinks (window 0: all t <= p), and with g(t) the 16-token group of t
//   out = sum_t w_t 2^ev(g) V_t / sum_t w_t,   w_t = exp(sm_scale (q . 2^ek(g) K_t) - max)
// (per-tensor scales: k_scale joins sm_scale and v_scale the result; bf16: no scales).  Rows that see
// nothing (p < 0) are zeros.
//
// What bounds it: the matrix units and the softmax's exponentials; the keys of a token block are read
// from L2 by its workgroup alone.  The shape is the key-split one of prefill_attn.hip: a workgroup of 8 waves
// owns some blocks of 16 tokens (the launch plan says how many) of one kv head's query heads, or a pair of such
// sets where all of a causal context is seen; wave w takes row-set group w / NR, RS sets of 16 (token, head) rows,
// and of every ring window the key tiles of residue w % NR.  Raw rows stream through an LDS ring of two windows.  Here:
//   * a block walks the 32-key tiles that hold a visible key: those of the sinks, then those from
//     the first query's window on.  A 16-key group inside them that holds none is not read (nor its
//     block-table entry): its rows are copied from the window's first group and masked.
//   * masks are applied only on tiles that some row of the block does not see whole.
//   * block scales (SC) are powers of two.  K's byte is the A scale of the block-scaled MFMA that forms the scores
//     anyway, V's the scale operand of the conversion that widens its codes to bf16, where they stay exact; neither
//     costs an instruction per element.  A group's pair of bytes is loaded with the window's copies and passed
//     through LDS.
//   * the weights are rounded to bf16 for P.V, which has the range for any score and any block scale, and the sum
//     that divides the result is that of the ROUNDED weights, so that they add up to one (v_dot2_f32_bf16 with ones:
//     four instructions for a row-set's eight weights).  Outputs are 0.0018 of their norm off those of 64 bits, with weights
//     in 32 bits 0.0016 (most of it their own rounding to bf16); a second part of each weight would double P.V's products.
//   * a masked key's V must not reach a row through 0 * NaN: on masked tiles that hold a non-finite V
//     (one test of the raw words, with block scales of the range that each group's scale leaves its codes), it is zeroed
//     for the product and added afterwards to the rows that see it.
// Measured in a graph: 2048 block-scaled tokens after 2048, 24 / 4 heads, 91.6 us (844 Tflop/s of visible work; a large bf16
// product 1117), 4096 e4m3 tokens with a window of 1024 63.6, six block-scaled prompts of 37..900 47.0, five bf16
// prompts of 100..1500 with a window of 512, 32 / 8 heads, 62.4.  The matrix units are busy 36 % of the time, the vector units
// 53 % (the six prompts: 25 and 50, the five: 26 and 51).  At an earlier step, when the first took 104 us, it was 10
// faster without the exponentials, 7 without the second part of Q and 7 without widening V.
#include "fp8kv_common.h"
#include "fp8kv_status.h"
#include "fp8kv_diag.h"
#include "attn_common.h"
#include "prefill_tiles.h"

#include <type_traits>

namespace fp8kv {
namespace prefill_detail {

struct VisibleParams : Params {
    const uint16_t* kv_scales;      // [blocks][block_size / 16][hkv] pairs of e8m0 bytes (K low), or null
    int window, sinks;
    int gqa_inverse;                // 1024 / GQA, rounded up
};

// Scores of one 16-key group: K codes times the group's scale (byte KG * 2 of `scales`) against a split
// query row.
template <int KG, bool LO>
__device__ __forceinline__ f32x4_t score_mfma(const v8i& k, const v8i& q, f32x4_t c, uint32_t scales)
{
    constexpr int qs = 127 | (127 + kQLoExp) << 8;
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q, c, 0, 0, 2 * KG, (int)scales, LO ? 1 : 0, qs);
}

// Any non-finite element among the e4m3 codes (bf16 values) of a word: its field's top bit.  `past` (past_range) lets codes
// count whose value leaves the range of 32 bits with their group's scale.
constexpr uint32_t kNanCodes = 0x01010101u;           // NaN alone
template <bool B16>
__device__ __forceinline__ uint32_t non_finite(uint32_t w, uint32_t past = kNanCodes)
{
    return B16 ? ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u : ((w & 0x7F7F7F7Fu) + past) & 0x80808080u;
}
// What lifts the magnitude of such a code to its field's top bit.  |code| 2^(byte - 127) >= 2^128, which the widening to bf16
// makes infinite, from byte 247 on (448 * 2^119 is below): the least such code is 2^(255 - byte), whose bits are
// (262 - byte) << 3.
__device__ __forceinline__ uint32_t past_range(uint32_t byte)
{
    return byte < 247u ? kNanCodes : (0x80u - ((262u - byte) << 3)) * 0x01010101u;
}
// The word with its non-finite elements zeroed.
template <bool B16>
__device__ __forceinline__ uint32_t finite_only(uint32_t w, uint32_t past = kNanCodes)
{
    const uint32_t bad = non_finite<B16>(w, past);    // the top bit of each bad element's field
    const uint32_t mask = B16 ? (bad << 1) - (bad >> 15) : (bad << 1) - (bad >> 7);
    return w & ~mask;
}

// l plus the two bf16 values of w.
__device__ __forceinline__ float add_bf16x2(uint32_t w, float l)
{
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), __builtin_bit_cast(bf16x2_t, 0x3F803F80u), l, false);
}

// What a weight may grow to before its row's reference moves, and how far above the row's max it moves then, in log2: a
// row whose max then grows by less than the sum of the two is left alone, at weights between 2^-kLift and 2^kCeil.
constexpr float kCeil = 256.f, kLift = 8.f;
// References from here on are spaced so widely that the exact difference to one can leave a weight's range.
constexpr float kFar = 0x1p28f;

// The difference of a score, rounded, and a reference.
__device__ __forceinline__ float rounded_difference(float x, float factor, float m)
{
#pragma clang fp contract(off)
    const float s = x * factor;
    return s - m;
}

// New references and accumulators of RS row-sets after a weight past kCeil, from the tile's raw scores.  Returns the
// lanes where the reference of a row that has seen a key is past kFar.
template <int RS>
__device__ __forceinline__ uint64_t lift_rows(const f32x4_t (&sc)[RS][2], float (&m_run)[RS], float (&l_run)[RS],
                                              f32x4_t (&o)[RS][8], const float (&qkr)[RS])
{
#pragma clang fp contract(off)                  // the max is rounded as the scores are
    bool far = false;
#pragma unroll
    for (int j = 0; j < RS; ++j) {
        float m = max3_raw(sc[j][0][0], sc[j][0][1], sc[j][0][2]);
        m = max3_raw(m, sc[j][0][3], sc[j][1][0]);
        m = max3_raw(m, sc[j][1][1], sc[j][1][2]);
        const float mc = max_xor16_32_raw(max_raw(m, sc[j][1][3])) * qkr[j];      // -inf for a fully masked row
        const float m_new = mc > m_run[j] ? mc + kLift : m_run[j];
        const float alpha = __builtin_amdgcn_exp2f(m_run[j] - m_new);
        l_run[j] *= alpha;
#pragma unroll
        for (int n = 0; n < 8; ++n) o[j][n] *= alpha;
        m_run[j] = m_new;
        far |= fabsf(m_new) >= kFar && m_new > kMaxFloor;
    }
    return __ballot(far);
}

// SC: block-scaled e4m3 caches.
template <int RS, int NG, int TPW, bool B16, bool SC>
__global__ void __launch_bounds__(kSplitWaves * 64)
prefill_visible_kernel(VisibleParams P)
{
    constexpr int W = kSplitWaves;
    constexpr int TILE = B16 ? kTileBytes16 : kTileBytes;
    constexpr int NR = W / NG;
    constexpr int NT = NR * TPW;                           // tiles per window
    constexpr int UNROLL = TPW <= 2 ? TPW : 1;
    static_assert(NG * NR == W && RS >= 1 && NT <= 64, "split shape");
    constexpr int kWinBytes = NT * TILE;
    constexpr int kRingBytes = 2 * kWinBytes;
    constexpr int kStageBytes = NG * RS * (NR - 1) * kStageFloats * 4;
    // the query rows' hand-over, from the ring's second window on: that is written only after the first barrier of the
    // key loop
    constexpr int kSetBytes = 4 * 1024 + 256;
    constexpr int kExch = kWinBytes;
    constexpr int kExchEnd = B16 || NR == 1 ? 0 : kExch + NG * RS * kSetBytes;
    constexpr int kLoopBytes = kRingBytes > kExchEnd ? kRingBytes : kExchEnd;
    __shared__ __align__(16) unsigned char ring[kLoopBytes > kStageBytes ? kLoopBytes : kStageBytes];
    __shared__ float stage_m[NR > 1 ? NG * NR * RS * 16 : 4];
    static_assert(!(B16 && SC), "block scales belong to e4m3 caches");
    __shared__ __align__(4) uint16_t lds_scales[2][SC ? NT : 1][2];
    float* const stage = reinterpret_cast<float*>(ring);

    const int lin = blockIdx.x, seq = blockIdx.z;
    int kh, rank;
    if (P.xcd_map) {
        const int xcd = lin & 7, per = 8 / P.hkv;
        kh = xcd % P.hkv;
        rank = (lin >> 3) * per + xcd / P.hkv;
    } else {
        kh = lin % P.hkv;
        rank = lin / P.hkv;
    }
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = wave / NR;
    const int res = wave % NR;
    const int lr = lane & 15;
    const int lp = lane >> 4;

    const int q_begin = P.cu_q[seq], qlen = P.cu_q[seq + 1] - q_begin;
    const int q0 = P.seq_lens[seq] - qlen;                         // may be negative: those rows see nothing
    const int nbt = P.nb;                                          // token blocks of 16 per workgroup
    const int n16 = (qlen + 16 * nbt - 1) / (16 * nbt);
    const int tb = P.ntb_grid - 1 - rank;
    const int nwg = P.paired ? (n16 + 1) >> 1 : n16;              // workgroups this sequence needs
    if (tb < 0 || tb >= nwg) return;                              // whole workgroup, before any barrier
    const int blk_a = tb, blk_b = P.paired ? n16 - 1 - tb : tb;
    const int nphase = blk_b > blk_a ? 2 : 1;
    const int32_t* btrow = P.bt + (int64_t)seq * P.bt_stride;
    const float qk_signed = B16 || SC ? P.sm_scale * kLog2e : P.sm_scale * P.k_scale[0] * kLog2e;
    auto uniform = [](float f) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(f))); };
    const float qk = uniform(fabsf(qk_signed));                // a NaN reaches the output through vs
    const uint32_t qflip = qk_signed < 0.f ? (B16 ? 0x80008000u : 0x80808080u) : 0u;   // negate Q (exact)
    const float vs = uniform((B16 || SC ? 1.f : P.v_scale[0]) + (qk_signed == qk_signed ? 0.f : qk_signed));
    const int window = P.window > 0 ? P.window : 1 << 30;
    const int sinks = P.sinks;

    // This wave's copies of every tile, lane (row, chunk), as in prefill_attn.hip: e4m3 one, of K rows (waves 0-3)
    // or V rows (waves 4-7) 8 (wave & 3) .. +7; bf16 two, of K and V rows 4 wave .. +3.  Its rows lie in one
    // 16-key group, hence in one cache block.
    const bool dma_v = !B16 && wave >= 4;
    int dma_r, dma_c;
    if constexpr (B16) {
        dma_r = lane >> 4;
        dma_c = (lane & 15) ^ ((4 * wave + dma_r) & 15);
    } else {
        dma_lane_rc(dma_v, lane, dma_r, dma_c);
    }
    const int dma_row0 = B16 ? 4 * wave : 8 * (wave & 3);
    const uint8_t* dma_base = dma_v ? P.v + (int64_t)kh * P.sv2 : P.k + (int64_t)kh * P.sk2;
    const int64_t dma_s0 = dma_v ? P.sv0 : P.sk0;
    const uint32_t dma_s1 = (uint32_t)(dma_v ? P.sv1 : P.sk1);    // < 2^32 / block size (host check)
    const uint32_t voff_lane = (uint32_t)dma_r * dma_s1 + 16u * (uint32_t)dma_c;
    const uint8_t* const dma_base_v = P.v + (int64_t)kh * P.sv2;   // bf16: the second copy
    const uint32_t voff_lane_v = (uint32_t)dma_r * (uint32_t)P.sv1 + 16u * (uint32_t)dma_c;

    // Byte offsets in an e4m3 tile of this lane's fragments: K row lr, chunk lp (k_slot; chunk 4 + lp lies 64 away), and
    // V row 4 lp, d = 8 lr (v_slot; row 4 lp + j lies 256 j behind, 16 rows further 2048).
    const int k_lane = 1024 * (lr >> 3) + 16 * k_slot(lr & 7, lp);
    const int v_lane = TILE / 2 + 1024 * (lp >> 1) + 16 * v_slot(4 * (lp & 1), lr >> 1) + 8 * (lr & 1);

    // head, and block within the workgroup, of row-set rset (those past the last repeat it)
    const int last_set = nbt * P.gqa - 1;
    // (row-sets are below 64 and GQA at most 16, for which 1024 / GQA rounded up divides exactly)
    auto block_of = [&](int rset) { return min(rset, last_set) * P.gqa_inverse >> 10; };
    auto head_of = [&](int rset) { return min(rset, last_set) - block_of(rset) * P.gqa; };
    int my_block[RS];                                              // block of this wave's row-sets
#pragma unroll
    for (int j = 0; j < RS; ++j) my_block[j] = block_of(grp * RS + j);

    for (int ph = 0; ph < nphase; ++ph) {
        const int blk = ph == 0 ? blk_b : blk_a;
        const int tok0 = 16 * nbt * blk;                          // first token of the block(s)
        const int qfirst = q0 + tok0;
        const int qlast = q0 + min(tok0 + 16 * nbt, qlen) - 1;
        const int k_hi = max(qlast + 1, 0);                       // keys [0, k_hi)
        // Tiles walked: `head` ones that hold sinks, then, `jump` further, those from the window of the first query on.
        const int low = max(qfirst - window + 1, 0);              // first key of that window
        const int head = (min(sinks, low) + kBN - 1) / kBN;
        const int jump = max(low / kBN - head, 0);
        const int ntiles = (k_hi + kBN - 1) / kBN - jump;
        const int nwin = (ntiles + NT - 1) / NT;
        const int first_group = low >> 4;
        auto tile_at = [&](int t) { return t + (t >= head ? jump : 0); };
        // First key that this wave's copy of walked tile t reads: of its own 16-key group, or, where nobody sees a key
        // of that, of one that is there: the window's first, and behind the last key the last.  Slots of a group behind
        // the last key are read as they are: masks and the test for non-finite V take care of what they hold.
        const int last_group = (k_hi - 1) >> 4;
        auto copy_key = [&](int t) {
            int g = 2 * tile_at(t) + (dma_row0 >> 4);
            g = (g >= first_group) | (16 * g < sinks) ? g : first_group;
            return 16 * min(g, last_group) + (dma_row0 & 15);
        };
        auto token_of = [&](int j) { return tok0 + 16 * my_block[j] + lr; };
        // Tiles past this wave's last row, and below its first row's window, are left out.
        const int my_hi = qfirst + 16 * my_block[RS - 1] + 15;
        const int my_low = qfirst + 16 * my_block[0] - window + 1;

        // A window's copies are prepared by lane: lane u holds the block id, then the address, of tile u's first row, and
        // a copy takes it from there with two readlanes (formed by scalar instructions, copy by copy, addresses were
        // most of a tile's instructions).  Scale bytes of the window's groups come along in the two waves whose K copies
        // are those of a tile's groups (rows 0 and 16).
        int bids = 0;
        uint64_t src = 0;
        [[maybe_unused]] uint64_t src_v = 0;
        [[maybe_unused]] uint32_t sc_next = 0;
        auto load_bids = [&](int wi) { bids = lane < NT ? btrow[copy_key(wi * NT + lane) >> P.pshift] : 0; };
        auto place_window = [&](int wi) {
            const uint32_t slot = (uint32_t)(copy_key(wi * NT + lane) & (P.pblk - 1));
            src = (uint64_t)dma_base + (int64_t)bids * dma_s0 + (uint64_t)slot * dma_s1;
            if constexpr (B16) src_v = (uint64_t)dma_base_v + (int64_t)bids * P.sv0 + (uint64_t)slot * (uint32_t)P.sv1;
            if constexpr (SC) {
                if ((wave == 0 || wave == 2) && lane < NT)
                    sc_next = P.kv_scales[((int64_t)bids * (P.pblk >> 4) + (slot >> 4)) * P.hkv + kh];
            }
        };
        auto lane_address = [&](uint64_t a, int u) -> const uint8_t* {
            const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)a, u), hi = __builtin_amdgcn_readlane((uint32_t)(a >> 32), u);
            return reinterpret_cast<const uint8_t*>((uint64_t)hi << 32 | lo);
        };
        // Copies of part v of window wi: tiles NR v .. NR v + NR - 1.
        auto issue_part = [&](int wi, int v) {
#pragma unroll
            for (int k = 0; k < NR; ++k) {
                const int u = NR * v + k;
                if (wi * NT + u < ntiles) {
                    unsigned char* dst = ring + (wi & 1) * kWinBytes + u * TILE + wave * 1024;
                    dma16_saddr(lane_address(src, u), voff_lane, dst);
                    if constexpr (B16) dma16_saddr(lane_address(src_v, u), voff_lane_v, dst + TILE / 2);
                }
            }
        };
        auto first_window = [&]() {
            place_window(0);
#pragma unroll UNROLL
            for (int v = 0; v < TPW; ++v) issue_part(0, v);
            if (1 < nwin) load_bids(1);
        };
        // Q as the B operand of S^T = K.Q^T: see prefill_attn.hip.  e4m3 caches: hi + lo parts, split by one wave per row-set
        // and handed over through the LDS; bf16 caches: the four fragments, loaded by each wave.
        auto load_query = [&](u32x4_t (&qf)[4], int tok, int head) {
            const u32x4_t zero = {0u, 0u, 0u, 0u};
            const bool ok = tok < qlen;
            const __bf16* qrow = P.q + (int64_t)(q_begin + (ok ? tok : 0)) * P.q_stride + (int64_t)(kh * P.gqa + head) * kD;
            qf[0] = ok ? load_16(qrow + 16 * lp) : zero;
            qf[1] = ok ? load_16(qrow + 16 * lp + 8) : zero;
            qf[2] = ok ? load_16(qrow + 64 + 16 * lp) : zero;
            qf[3] = ok ? load_16(qrow + 64 + 16 * lp + 8) : zero;
        };
        v8i qhi[RS], qlo[RS];
        float qkr[RS];
        if (ntiles > 0) load_bids(0);
        if constexpr (B16) {
            u32x4_t qf[RS][4];
#pragma unroll
            for (int j = 0; j < RS; ++j) load_query(qf[j], token_of(j), head_of(grp * RS + j));
#pragma unroll
            for (int j = 0; j < RS; ++j) {
                asm volatile("" : "+v"(qf[j][0]), "+v"(qf[j][1]), "+v"(qf[j][2]), "+v"(qf[j][3]));
                qkr[j] = fmaxf(qk, kMinFactor16);
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    qhi[j][d] = (int)(qf[j][0][d] ^ qflip);
                    qhi[j][4 + d] = (int)(qf[j][1][d] ^ qflip);
                    qlo[j][d] = (int)(qf[j][2][d] ^ qflip);
                    qlo[j][4 + d] = (int)(qf[j][3][d] ^ qflip);
                }
            }
            first_window();
        } else if constexpr (NR == 1) {
            // every wave has row-sets of its own
            u32x4_t qf[RS][4];
#pragma unroll
            for (int j = 0; j < RS; ++j) load_query(qf[j], token_of(j), head_of(grp * RS + j));
#pragma unroll
            for (int j = 0; j < RS; ++j)
                asm volatile("" : "+v"(qf[j][0]), "+v"(qf[j][1]), "+v"(qf[j][2]), "+v"(qf[j][3]));
            first_window();
#pragma unroll
            for (int j = 0; j < RS; ++j) qkr[j] = fmaxf(qk * q_fp8_split(qf[j], qflip, qhi[j], qlo[j]), kMinFactor16);
        } else {
            constexpr int SETS = NG * RS, PER = (SETS + W - 1) / W;        // row-sets, and splits per wave at most
            unsigned char* const exch = ring + kExch;
            int ln = lane;                             // opaque: its addresses stay out of the key loop's registers
            asm volatile("" : "+v"(ln));
            u32x4_t qf[PER][4];
#pragma unroll
            for (int u = 0; u < PER; ++u) {
                const int rset = wave + W * u;
                load_query(qf[u], tok0 + 16 * block_of(rset) + lr, head_of(rset));
            }
#pragma unroll
            for (int u = 0; u < PER; ++u)
                asm volatile("" : "+v"(qf[u][0]), "+v"(qf[u][1]), "+v"(qf[u][2]), "+v"(qf[u][3]));
            first_window();
#pragma unroll
            for (int u = 0; u < PER; ++u) {
                const int rset = wave + W * u;
                if (rset < SETS) {
                    v8i hi, lo;
                    const float inv = q_fp8_split(qf[u], qflip, hi, lo);
                    unsigned char* x = exch + rset * kSetBytes + 16 * ln;
                    *reinterpret_cast<u32x4_t*>(x) = (u32x4_t){(uint32_t)hi[0], (uint32_t)hi[1], (uint32_t)hi[2], (uint32_t)hi[3]};
                    *reinterpret_cast<u32x4_t*>(x + 1024) = (u32x4_t){(uint32_t)hi[4], (uint32_t)hi[5], (uint32_t)hi[6], (uint32_t)hi[7]};
                    *reinterpret_cast<u32x4_t*>(x + 2 * 1024) = (u32x4_t){(uint32_t)lo[0], (uint32_t)lo[1], (uint32_t)lo[2], (uint32_t)lo[3]};
                    *reinterpret_cast<u32x4_t*>(x + 3 * 1024) = (u32x4_t){(uint32_t)lo[4], (uint32_t)lo[5], (uint32_t)lo[6], (uint32_t)lo[7]};
                    *reinterpret_cast<float*>(exch + rset * kSetBytes + 4096 + 4 * ln) = fmaxf(qk * inv, kMinFactor16);
                }
            }
            lds_barrier();
#pragma unroll
            for (int j = 0; j < RS; ++j) {
                const unsigned char* x = exch + (grp * RS + j) * kSetBytes + 16 * ln;
                u32x4_t v[4];
#pragma unroll
                for (int d = 0; d < 4; ++d) v[d] = *reinterpret_cast<const u32x4_t*>(x + 1024 * d);
                qhi[j] = (v8i){(int)v[0][0], (int)v[0][1], (int)v[0][2], (int)v[0][3],
                               (int)v[1][0], (int)v[1][1], (int)v[1][2], (int)v[1][3]};
                qlo[j] = (v8i){(int)v[2][0], (int)v[2][1], (int)v[2][2], (int)v[2][3],
                               (int)v[3][0], (int)v[3][1], (int)v[3][2], (int)v[3][3]};
                qkr[j] = *reinterpret_cast<const float*>(exch + (grp * RS + j) * kSetBytes + 4096 + 4 * ln);
            }
        }

        float m_run[RS], l_run[RS];
        f32x4_t o[RS][8];
        uint64_t far = 0;                                          // lanes with a reference past kFar
#pragma unroll
        for (int j = 0; j < RS; ++j) {
            m_run[j] = kMaxFloor;
            l_run[j] = 0.f;
#pragma unroll
            for (int n = 0; n < 8; ++n) o[j][n] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        }

        for (int i = 0; i < nwin; ++i) {
            // Everything this wave has in flight: window i's copies and scales, the block ids of window i + 1.  The
            // barrier then publishes window i and frees window i - 1's slot.
            wait_vmcnt<0>();
            if constexpr (SC) {
                if ((wave == 0 || wave == 2) && lane < NT) lds_scales[i & 1][lane][wave >> 1] = (uint16_t)sc_next;
            }
            lds_barrier();
            const bool more = i + 1 < nwin;
            if (more) place_window(i + 1);

#pragma unroll UNROLL
            for (int v = 0; v < TPW; ++v) {
                // The next window's copies go out in TPW parts, one before each tile.
                if (more) issue_part(i + 1, v);
                const int tw = NR * v + res;                     // tile within the window, in the order of the copies
                const int t = i * NT + tw;
                const int k0 = kBN * tile_at(t);
                if (t >= ntiles || k0 > my_hi || (k0 + kBN <= my_low && k0 >= sinks)) continue;
                const unsigned char* buf = ring + (i & 1) * kWinBytes + tw * TILE;
                // Some row of this wave does not see some key: past its first query, or below its last one's window and no sink.
                const bool masked = k0 + kBN - 1 > qfirst + 16 * my_block[0] ||
                                    (k0 <= min(qlast, my_hi) - window && k0 + kBN > sinks);
                f32x4_t sc[RS][2];
                bool poisoned = false;
                if constexpr (B16) {
                    if (masked) {
                        int ln = lane;                 // opaque, as above
                        asm volatile("" : "+v"(ln));
                        uint32_t bad = 0;
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            const u32x4_t w = *reinterpret_cast<const u32x4_t*>(buf + TILE / 2 + 1024 * c + 16 * ln);
#pragma unroll
                            for (int d = 0; d < 4; ++d) bad |= non_finite<true>(w[d]);
                        }
                        poisoned = __any(bad != 0);
                    }
#pragma unroll
                    for (int kg = 0; kg < 2; ++kg) {
                        const int row = 16 * kg + lr;
                        u32x4_t kf[4];
#pragma unroll
                        for (int f = 0; f < 4; ++f)
                            kf[f] = *reinterpret_cast<const u32x4_t*>(buf + b16_slot(row, 8 * (f >> 1) + 2 * lp + (f & 1)));
#pragma unroll
                        for (int j = 0; j < RS; ++j) {
                            f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int f = 0; f < 4; ++f) {
                                const v8i& qq = f < 2 ? qhi[j] : qlo[j];
                                const int h = 4 * (f & 1);
                                const u32x4_t qv = {(uint32_t)qq[h], (uint32_t)qq[h + 1], (uint32_t)qq[h + 2],
                                                    (uint32_t)qq[h + 3]};
                                acc = mfma16x16x32_bf16(as_bf16x8(kf[f]), as_bf16x8(qv), acc);
                            }
                            sc[j][kg] = acc;
                        }
                    }
                }
                [[maybe_unused]] u32x4_t vf[8];
                [[maybe_unused]] u32x2_t vr[8];
                [[maybe_unused]] float vsc[2] = {1.f, 1.f};
                // past_range of group g of the tile
                [[maybe_unused]] auto past_of = [&](int g) {
                    if constexpr (SC) return past_range((uint32_t)__builtin_amdgcn_readfirstlane(lds_scales[i & 1][tw][g]) >> 8);
                    else return kNanCodes;
                };
                // V^T fragments 4 w .. 4 w + 3 (d = 8c + 4w ..) from word w of the raw rows, as v_fragments
                auto widen = [&](int w) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t x = __builtin_amdgcn_perm(vr[2 * k + 1][w], vr[2 * k][w], 0x05010400u);   // a0 b0 a1 b1
                        const uint32_t y = __builtin_amdgcn_perm(vr[2 * k + 1][w], vr[2 * k][w], 0x07030602u);   // a2 b2 a3 b3
                        const float f = vsc[k >> 1];
                        vf[4 * w + 0][k] = bf16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, f, false));
                        vf[4 * w + 1][k] = bf16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, f, true));
                        vf[4 * w + 2][k] = bf16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, f, false));
                        vf[4 * w + 3][k] = bf16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, f, true));
                    }
                };
                if constexpr (!B16) {
                    v8i kf[2];
#pragma unroll
                    for (int kg = 0; kg < 2; ++kg) {
                        const u32x4_t lo = *reinterpret_cast<const u32x4_t*>(buf + k_lane + 2048 * kg);
                        const u32x4_t hi = *reinterpret_cast<const u32x4_t*>(buf + (k_lane ^ 64) + 2048 * kg);
                        kf[kg] = (v8i){(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3],
                                       (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
                    }
                    uint32_t scales = 127 | 127 << 16;
                    [[maybe_unused]] uint32_t tile_scales = 0;
                    if constexpr (SC) {
                        scales = *reinterpret_cast<const uint32_t*>(lds_scales[i & 1][tw]);
                        const uint32_t u = __builtin_amdgcn_readfirstlane(scales);
                        tile_scales = u;
                        vsc[0] = __uint_as_float((u & 0xFF00u) << 15);         // bytes 1 .. 254 are exponents as they are
                        vsc[1] = __uint_as_float((u & 0xFF000000u) >> 1);
                    }
                    // V^T raw rows (lane (c, p) transposes d = 8c .. 8c+7) and the widening of their first half go along
                    // with S^T = K.Q^T
#pragma unroll
                    for (int jj = 0; jj < 8; ++jj) {
                        vr[jj] = *reinterpret_cast<const u32x2_t*>(buf + v_lane + 256 * (jj & 3) + (jj < 4 ? 0 : 2048));
                    }
                    if (masked) {
                        uint32_t bad = 0;
                        asm volatile("" : "+v"(bad));  // a branch: nothing of the test runs on other tiles
#pragma unroll
                        for (int jj = 0; jj < 8; ++jj) bad |= non_finite<false>(vr[jj][0]) | non_finite<false>(vr[jj][1]);
                        poisoned = __any(bad != 0);
                        if constexpr (SC) poisoned |= (tile_scales & 0xFF00u) >= 247u << 8 || tile_scales >> 24 >= 247u;
                        if (poisoned) {
                            const uint32_t past[2] = {past_of(0), past_of(1)};
#pragma unroll
                            for (int jj = 0; jj < 8; ++jj) {
                                vr[jj][0] = finite_only<false>(vr[jj][0], past[jj >> 2]);
                                vr[jj][1] = finite_only<false>(vr[jj][1], past[jj >> 2]);
                            }
                        }
                    }
                    widen(0);
#pragma unroll
                    for (int j = 0; j < RS; ++j) {
                        const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
                        f32x4_t acc = score_mfma<0, false>(kf[0], qhi[j], zero, scales);
                        sc[j][0] = score_mfma<0, true>(kf[0], qlo[j], acc, scales);
                        acc = score_mfma<1, false>(kf[1], qhi[j], zero, scales);
                        sc[j][1] = score_mfma<1, true>(kf[1], qlo[j], acc, scales);
                    }
                    // pinned here, where the vector units would wait: one MFMA, then two or three of its 24 instructions
#pragma unroll
                    for (int n = 0; n < 4; ++n) asm volatile("" : "+v"(vf[n]));
#pragma unroll
                    for (int g = 0; g < 4 * RS; ++g) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x002, 24 / (4 * RS), 0);
                    }
                }
                if (masked) {
                    int lm = lane;                     // opaque, as above
                    asm volatile("" : "+v"(lm));
#pragma unroll
                    for (int j = 0; j < RS; ++j) {
                        const int qpos = q0 + tok0 + 16 * my_block[j] + (lm & 15);
#pragma unroll
                        for (int kg = 0; kg < 2; ++kg)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int key = k0 + 16 * kg + 4 * (lm >> 4) + e;
                                const bool hidden = (key > qpos) | ((key <= qpos - window) & (key >= sinks));
                                sc[j][kg][e] = hidden ? neg_inf() : sc[j][kg][e];
                            }
                    }
                }
                // Weights of row-set j in bf16 (the P^T operand) and their sum: of the exact difference of score and
                // reference, which takes one instruction, or of the rounded product's, which is never above 2^-kLift for a
                // reference that has moved.
                u32x4_t pb[RS];
                float ps[RS];
                auto row_weights = [&](int j, auto rounded) {
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        float w[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float x = sc[j][d >> 1][2 * (d & 1) + e];
                            w[e] = __builtin_amdgcn_exp2f(rounded ? rounded_difference(x, qkr[j], m_run[j])
                                                                  : __builtin_fmaf(x, qkr[j], -m_run[j]));
                        }
                        pb[j][d] = pack_bf16x2(w[0], w[1]);
                    }
                    ps[j] = add_bf16x2(pb[j][3], add_bf16x2(pb[j][2], add_bf16x2(pb[j][1], add_bf16x2(pb[j][0], 0.f))));
                };
                // The sums tell whether a weight grew past kCeil (or eight of them together): then the references move and the
                // weights are formed again.  Looking for the row maxima first costs 24 instructions a tile and one more
                // dependent step, for something that happens at the start of a row and hardly ever after.
                bool over = false;
#pragma unroll
                for (int j = 0; j < RS; ++j) {
                    row_weights(j, std::false_type{});
                    over |= ps[j] > kCeil;
                }
                if (__builtin_expect((__ballot(over) | far) != 0, 0)) {
                    far = lift_rows<RS>(sc, m_run, l_run, o, qkr);
#pragma unroll
                    for (int j = 0; j < RS; ++j) row_weights(j, std::true_type{});
                }
#pragma unroll
                for (int j = 0; j < RS; ++j) l_run[j] += ps[j];
                if constexpr (!B16) {
                    // the first half of d, and the second half's widening beside it
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int j = 0; j < RS; ++j) o[j][n] = mfma16x16x32_bf16(as_bf16x8(vf[n]), as_bf16x8(pb[j]), o[j][n]);
                    widen(1);
#pragma unroll
                    for (int n = 4; n < 8; ++n)
#pragma unroll
                        for (int j = 0; j < RS; ++j) o[j][n] = mfma16x16x32_bf16(as_bf16x8(vf[n]), as_bf16x8(pb[j]), o[j][n]);
#pragma unroll
                    for (int g = 0; g < 4 * RS; ++g) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x002, 24 / (4 * RS), 0);
                    }
                } else {
                    // Half of a V row's 16 bytes at a time: half h is d = 8c + 4h .. + 3.
                    auto read_half = [&](int h) {
#pragma unroll
                        for (int jj = 0; jj < 8; ++jj) {
                            const int row = (jj < 4 ? 0 : 16) + 4 * lp + (jj & 3);
                            vr[jj] = *reinterpret_cast<const u32x2_t*>(buf + TILE / 2 + b16_slot(row, lr) + 8 * h);
                        }
                        if (poisoned) {
#pragma unroll
                            for (int jj = 0; jj < 8; ++jj) {
                                vr[jj][0] = finite_only<true>(vr[jj][0]);
                                vr[jj][1] = finite_only<true>(vr[jj][1]);
                            }
                        }
                    };
                    read_half(0);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        u32x4_t va[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int w = 0; w < 2; ++w) {
                                va[2 * w][k] = __builtin_amdgcn_perm(vr[2 * k + 1][w], vr[2 * k][w], 0x05040100u);
                                va[2 * w + 1][k] = __builtin_amdgcn_perm(vr[2 * k + 1][w], vr[2 * k][w], 0x07060302u);
                            }
                        if (h == 0) read_half(1);
#pragma unroll
                        for (int n = 0; n < 4; ++n)
#pragma unroll
                            for (int j = 0; j < RS; ++j)
                                o[j][4 * h + n] = mfma16x16x32_bf16(as_bf16x8(va[n]), as_bf16x8(pb[j]), o[j][4 * h + n]);
                    }
                }
                if (poisoned) {
                    // The non-finite V elements of the tile, key by key, to the rows that see them: lane (q, p) holds
                    // d = 32 p + 8 i + n.
                    int ln = lane;                     // opaque: nothing of this stays in registers through the key loop
                    asm volatile("" : "+v"(ln));
                    const int part = ln >> 4;
                    for (int row = 0; row < kBN; ++row) {
                        const int key = k0 + row;
                        const uint32_t past = past_of(row >> 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int d = 0; d < (B16 ? 4 : 2); ++d) {
                                const unsigned char* src = B16 ? buf + TILE / 2 + b16_slot(row, 4 * part + e)
                                    : buf + TILE / 2 + (row >> 3) * 1024 + 16 * v_slot(row & 7, 2 * part + (e >> 1)) + 8 * (e & 1);
                                const uint32_t w = reinterpret_cast<const uint32_t*>(src)[d];
                                const uint32_t bad = non_finite<B16>(w, past);
                                if (!__any(bad != 0)) continue;
#pragma unroll
                                for (int j = 0; j < RS; ++j) {
                                    const int qpos = q0 + tok0 + 16 * my_block[j] + (ln & 15);
                                    const bool sees = key <= qpos && (key > qpos - window || key < sinks);
                                    constexpr int per = B16 ? 2 : 4;               // elements of a word
#pragma unroll
                                    for (int h = 0; h < per; ++h) {
                                        float x;
                                        if constexpr (B16) {
                                            const uint32_t bits = h ? w & 0xFFFF0000u : w << 16;
                                            x = (bits & 0x7F800000u) == 0x7F800000u ? __uint_as_float(bits) : 0.f;
                                        } else {
                                            const uint32_t code = w >> (8 * h);
                                            const float inf = code & 0x80u ? neg_inf() : -neg_inf();
                                            x = (code & 0x7Fu) == 0x7Fu ? __builtin_nanf("") : bad >> (8 * h) & 0x80u ? inf : 0.f;
                                        }
                                        o[j][per * d + h][e] += sees ? x : 0.f;
                                    }
                                }
                            }
                    }
                }
            }
            // Block ids for the next window's copies, after this iteration's LDS reads.
            if (i + 2 < nwin) load_bids(i + 2);
        }

        int ln = lane;                                 // opaque, as above
        asm volatile("" : "+v"(ln));
        const int er = ln & 15, ep = ln >> 4;
        // ---- merge the NR partial states of each head group, then normalise and store ----------
        if constexpr (NR > 1) {
            // m_run is the same in the four lane groups of a query row: lanes 0..15 publish it.
            if (ep == 0) {
#pragma unroll
                for (int j = 0; j < RS; ++j) stage_m[((grp * NR + res) * RS + j) * 16 + er] = m_run[j];
            }
            lds_barrier();
#pragma unroll
            for (int j = 0; j < RS; ++j) {
                float mg = kMaxFloor;
#pragma unroll
                for (int r = 0; r < NR; ++r) mg = fmaxf(mg, stage_m[((grp * NR + r) * RS + j) * 16 + er]);
                const float f = __builtin_amdgcn_exp2f(m_run[j] - mg);
                l_run[j] *= f;
#pragma unroll
                for (int n = 0; n < 8; ++n) o[j][n] *= f;
            }
            // Row-set j is summed and written by residue j % NR, in the order of the residues behind it.
#pragma unroll
            for (int j = 0; j < RS; ++j) {
                if (res == j % NR) continue;
                const int slot = (res - j % NR + NR) % NR - 1;
                float* s = stage + (((grp * RS + j) * (NR - 1)) + slot) * kStageFloats;
#pragma unroll
                for (int n = 0; n < 8; ++n) *reinterpret_cast<f32x4_t*>(s + (n * 64 + ln) * 4) = o[j][n];
                s[8 * 64 * 4 + ln] = l_run[j];
            }
            lds_barrier();
#pragma unroll
            for (int j = 0; j < RS; ++j) {
                if (res != j % NR) continue;
#pragma unroll
                for (int r = 0; r < NR - 1; ++r) {
                    const float* s = stage + ((grp * RS + j) * (NR - 1) + r) * kStageFloats;
#pragma unroll
                    for (int n = 0; n < 8; ++n) o[j][n] += *reinterpret_cast<const f32x4_t*>(s + (n * 64 + ln) * 4);
                    l_run[j] += s[8 * 64 * 4 + ln];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < RS; ++j) {
            if (res != j % NR) continue;
            const float l = sum_xor16_32(l_run[j]);
            const int tok = tok0 + 16 * my_block[j] + er;
            if (tok >= qlen || grp * RS + j >= nbt * P.gqa) continue;
            // a row that sees no key has l = 0 and is written as zeros; NaN in l reaches the output
            const float f = l == 0.f ? 0.f : vs / l;
            __bf16* orow = P.out + (int64_t)(q_begin + tok) * P.o_stride +
                           (int64_t)(kh * P.gqa + head_of(grp * RS + j)) * kD + 32 * ep;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                u32x4_t w;
                w[0] = pack_bf16x2(o[j][0][e] * f, o[j][1][e] * f);
                w[1] = pack_bf16x2(o[j][2][e] * f, o[j][3][e] * f);
                w[2] = pack_bf16x2(o[j][4][e] * f, o[j][5][e] * f);
                w[3] = pack_bf16x2(o[j][6][e] * f, o[j][7][e] * f);
                *reinterpret_cast<u32x4_t*>(orow + 8 * e) = w;
            }
        }
        // The next block's copies overwrite the ring, which holds the stage: every wave must be
        // done with its final stage reads above.
        if (ph + 1 < nphase) lds_barrier();
    }
}

// ---- launch plan ----------------------------------------------------------------------------------
// A workgroup takes nb token blocks of 16, whose nb * GQA row-sets fill a shape.  More blocks share the copies of their
// keys, start and end once, and leave fewer partial states to merge; fewer blocks split the keys over more waves, so the
// GPU is full with fewer tokens.  The shape follows from the time that each would take, in us, fitted to 100 batches
// (1 to 16 sequences of 100..4000, GQA 4 to 10, either cache width) at every shape; the one taken is 1.1 % slower than
// the best on average, 32 % at most.  Outside of them, 24 batches of 300..4000 each: GQA 1 7.6 % on average and 40 % at most
// (16 of 30..300: 42.0 us in blocks of 256 tokens, 30.0 in 384), 2 and 3 3 % and 13 %, 11 to 16 1.5 % and 14 %.  The terms:
//   a workgroup   9.5 (three row-sets a wave: 9.6), and per key tile 0.2 (bf16: 0.3) for its copies and 0.65 (two row-sets
//                 a wave) or 1.2 (three) times the filled part of its eight waves, where a wave without rows still costs
//                 three quarters;
//   the grid      its rounds of 256 workgroups and 0.4 for the end; where the blocks cost alike (a window, pairs) half
//                 of a last round that is not full.  Not less than the longest workgroup.
// The host knows the queries and not the context: 192 more keys than them stand for it, and a block of a whole context
// sees 0.45 of its longest.  Measured, us with two / three row-sets of 2, 4 and 8 groups: GQA 4, 16 of 30..300, 71 / 60,
// 49 / 51, 39 / 49; one of 4000, window 400, 83 / 85, 64 / 70, 55 / 64; 4 of 30..300 21 / 24, 17 / 22, 24 / 33.
struct VisibleShape {
    int rs, ng;
};
constexpr VisibleShape kVisibleShapes[] = {{2, 2}, {3, 2}, {2, 4}, {3, 4}, {2, 8}, {3, 8}};       // by row-sets

struct VisiblePlan {
    VisibleShape shape;
    int nb, paired, ranks;             // ranks: workgroups per (sequence, kv head) of the longest sequence
};

// num_tokens: queries of all sequences, 0 where the caller did not say.
VisiblePlan plan_visible(bool b16, int gqa, int hkv, int num_seqs, int max_query_len, int num_tokens, int window, int sinks)
{
    const double all = num_tokens > 0 ? num_tokens : (double)num_seqs * max_query_len;
    const bool limited = window > 0 && window < max_query_len;
    const double longest = max_query_len + 192.0;
    VisiblePlan best{};
    double best_time = 1e300;
    for (const VisibleShape s : kVisibleShapes) {
        const int nb = s.rs * s.ng / gqa;
        if (nb < 1) continue;
        const int block = 16 * nb, used = (nb * gqa + s.rs - 1) / s.rs;
        const double tile = (b16 ? 0.3 : 0.2) + (s.rs == 2 ? 0.65 : 1.2) * (0.75 * s.ng + 0.25 * used) / kSplitWaves;
        const double seen = (double)window + sinks + block;
        const double fixed = s.rs == 2 ? 9.5 : 9.6;
        const double most = fixed + tile / kBN * (limited && seen < longest ? seen : longest);
        const double mean = limited ? most : fixed + tile / kBN * (0.45 * max_query_len + 192);
        const int n = (max_query_len + block - 1) / block;
        const double blocks = num_seqs == 1 ? n : all / block + num_seqs / 2.0;
        for (int paired = 0; paired < (limited ? 1 : 2); ++paired) {
            // a sequence's last workgroup is half empty, or its only one
            const double some = paired ? (num_seqs == 1 ? (n + 1) / 2 : (blocks + num_seqs / 2.0) / 2) : blocks;
            const double x = hkv * (some > num_seqs ? some : num_seqs) / kSplitRoundWorkgroups;
            const double one = paired ? 2 * mean : mean, least = paired ? 2 * mean : most;
            double time = x <= 1 ? 0 : one * (limited || paired ? 0.5 * (x + 0.4 + ceil(x - 0.05)) : x + 0.4);
            if (time < least) time = least;
            if (time < best_time) {
                best_time = time;
                best = VisiblePlan{s, nb, paired, paired ? (n + 1) / 2 : n};
            }
        }
    }
    return best;
}

template <bool B16, bool SC>
void launch_shape(const VisibleParams& P, VisibleShape s, dim3 grid, dim3 block, hipStream_t stream)
{
    constexpr int T = B16 ? 1 : 2;                     // tiles per wave and window, for windows of 64 KB
    if (s.rs == 2) {
        if (s.ng == 2) launch_kernel(prefill_visible_kernel<2, 2, T, B16, SC>, grid, block, 0, stream, P);
        else if (s.ng == 4) launch_kernel(prefill_visible_kernel<2, 4, 2 * T, B16, SC>, grid, block, 0, stream, P);
        else launch_kernel(prefill_visible_kernel<2, 8, 4 * T, B16, SC>, grid, block, 0, stream, P);
    } else {
        if (s.ng == 2) launch_kernel(prefill_visible_kernel<3, 2, T, B16, SC>, grid, block, 0, stream, P);
        else if (s.ng == 4) launch_kernel(prefill_visible_kernel<3, 4, 2 * T, B16, SC>, grid, block, 0, stream, P);
        else launch_kernel(prefill_visible_kernel<3, 8, 4 * T, B16, SC>, grid, block, 0, stream, P);
    }
}

int launch_visible(const VisibleParams& P0, bool b16, int num_seqs, int max_query_len, int num_tokens, hipStream_t stream)
{
    VisibleParams P = P0;
    const VisiblePlan L = plan_visible(b16, P.gqa, P.hkv, num_seqs, max_query_len, num_tokens, P.window, P.sinks);
    P.nb = L.nb;
    P.paired = L.paired;
    P.xcd_map = (P.hkv <= 8 && 8 % P.hkv == 0) ? 1 : 0;
    const int per = split_xcd_per(P.hkv);
    P.ntb_grid = (L.ranks + per - 1) / per * per;
    const dim3 grid((unsigned)(P.ntb_grid * P.hkv), 1u, (unsigned)num_seqs), block(64 * kSplitWaves);
    begin_launch();
    if (b16) launch_shape<true, false>(P, L.shape, grid, block, stream);
    else if (P.kv_scales) launch_shape<false, true>(P, L.shape, grid, block, stream);
    else launch_shape<false, false>(P, L.shape, grid, block, stream);
    return finish_launch();
}

enum CacheKind { kE4m3 = 0, kBf16 = 1, kBlk = 2 };

template <int KIND>
int prefill_visible(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache, int64_t sk0, int64_t sk1,
                    int64_t sk2, int64_t sv0, int64_t sv1, int64_t sv2, void* out, int64_t out_row_stride,
                    const int32_t* cu_seqlens_q, const int32_t* seq_lens, const int32_t* block_table, int64_t bt_stride,
                    const float* k_scale, const float* v_scale, const void* kv_scales, float sm_scale, int num_seqs,
                    int num_q_heads, int num_kv_heads, int head_size, int block_size, int window, int sinks,
                    int max_query_len, int num_tokens, void* stream)
{
    if (!cu_seqlens_q || !seq_lens || num_seqs < 1 || max_query_len < 0 || num_tokens < 0 || window < 0 || sinks < 0)
        return FP8KV_ERR_ARG;
    if (KIND == kBlk && !kv_scales) return FP8KV_ERR_ARG;
    if (num_seqs > 65535) return FP8KV_ERR_SHAPE;
    const int64_t elem = KIND == kBf16 ? 2 : 1;
    sk0 *= elem; sk1 *= elem; sk2 *= elem;
    sv0 *= elem; sv1 *= elem; sv2 *= elem;
    const float* any = reinterpret_cast<const float*>(q);           // scales that only the kE4m3 kernels read
    const int st = check_common(q, k_cache, v_cache, out, q_row_stride, sk0, sk1, sk2, sv0, sv1, sv2, block_table, bt_stride,
                                KIND == kE4m3 ? k_scale : any, KIND == kE4m3 ? v_scale : any, num_q_heads, num_kv_heads,
                                head_size, block_size, out_row_stride);
    if (st != FP8KV_OK) return st;
    if (KIND == kBf16 && (!aligned(v_cache, 16) || ((sv0 | sv1 | sv2) & 15))) return FP8KV_ERR_ALIGN;
    if (KIND == kBlk && !aligned(kv_scales, 2)) return FP8KV_ERR_ALIGN;
    if (max_query_len == 0) return FP8KV_OK;
    VisibleParams P;
    static_cast<Params&>(P) = make_params(q, q_row_stride, k_cache, v_cache, sk0, sk1, sk2, sv0, sv1, sv2, out, out_row_stride,
                                          block_table, bt_stride, k_scale, v_scale, sm_scale, num_q_heads, num_kv_heads,
                                          block_size);
    P.cu_q = cu_seqlens_q;
    P.seq_lens = seq_lens;
    P.kv_scales = static_cast<const uint16_t*>(kv_scales);
    P.window = window < 1 << 30 ? window : 1 << 30;     // positions less a window stay within 32 bits
    P.sinks = sinks;
    P.gqa_inverse = (1024 + P.gqa - 1) / P.gqa;
    return launch_visible(P, KIND == kBf16, num_seqs, max_query_len, num_tokens, reinterpret_cast<hipStream_t>(stream));
}

}  // namespace prefill_detail
}  // namespace fp8kv

using namespace fp8kv::prefill_detail;

extern "C" int fp8kv_prefill_attn_window(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                                         int64_t sk0, int64_t sk1, int64_t sk2, int64_t sv0, int64_t sv1, int64_t sv2,
                                         void* out, int64_t out_row_stride, const int32_t* cu_seqlens_q,
                                         const int32_t* seq_lens, const int32_t* block_table, int64_t bt_stride,
                                         const float* k_scale, const float* v_scale, float sm_scale, int num_seqs,
                                         int num_q_heads, int num_kv_heads, int head_size, int block_size, int window,
                                         int sinks, int max_query_len, int num_tokens, void* stream)
{
    return prefill_visible<kE4m3>(q, q_row_stride, k_cache, v_cache, sk0, sk1, sk2, sv0, sv1, sv2, out, out_row_stride,
                                  cu_seqlens_q, seq_lens, block_table, bt_stride, k_scale, v_scale, nullptr, sm_scale, num_seqs,
                                  num_q_heads, num_kv_heads, head_size, block_size, window, sinks, max_query_len, num_tokens,
                                  stream);
}

extern "C" int fp8kv_prefill_attn_window_bf16(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                                              int64_t sk0, int64_t sk1, int64_t sk2, int64_t sv0, int64_t sv1, int64_t sv2,
                                              void* out, int64_t out_row_stride, const int32_t* cu_seqlens_q,
                                              const int32_t* seq_lens, const int32_t* block_table, int64_t bt_stride,
                                              float sm_scale, int num_seqs, int num_q_heads, int num_kv_heads, int head_size,
                                              int block_size, int window, int sinks, int max_query_len, int num_tokens, void* stream)
{
    return prefill_visible<kBf16>(q, q_row_stride, k_cache, v_cache, sk0, sk1, sk2, sv0, sv1, sv2, out, out_row_stride,
                                  cu_seqlens_q, seq_lens, block_table, bt_stride, nullptr, nullptr, nullptr, sm_scale, num_seqs,
                                  num_q_heads, num_kv_heads, head_size, block_size, window, sinks, max_query_len, num_tokens,
                                  stream);
}

extern "C" int fp8kv_prefill_attn_blk(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                                      int64_t sk0, int64_t sk1, int64_t sk2, int64_t sv0, int64_t sv1, int64_t sv2,
                                      void* out, int64_t out_row_stride, const int32_t* cu_seqlens_q, const int32_t* seq_lens,
                                      const int32_t* block_table, int64_t bt_stride, const void* kv_scales, float sm_scale,
                                      int num_seqs, int num_q_heads, int num_kv_heads, int head_size, int block_size,
                                      int window, int sinks, int max_query_len, int num_tokens, void* stream)
{
    return prefill_visible<kBlk>(q, q_row_stride, k_cache, v_cache, sk0, sk1, sk2, sv0, sv1, sv2, out, out_row_stride,
                                 cu_seqlens_q, seq_lens, block_table, bt_stride, nullptr, nullptr, kv_scales, sm_scale, num_seqs,
                                 num_q_heads, num_kv_heads, head_size, block_size, window, sinks, max_query_len, num_tokens,
                                  stream);
}

extern "C" int fp8kv_prefill_visible_plan(int num_q_heads, int num_kv_heads, int num_seqs, int max_query_len, int num_tokens,
                                          int window, int sinks, int bf16, int* out)
{
    if (!out || num_q_heads < 1 || num_kv_heads < 1 || num_seqs < 1 || max_query_len < 0 || num_tokens < 0 || window < 0 || sinks < 0)
        return FP8KV_ERR_ARG;
    if (num_q_heads % num_kv_heads != 0 || num_q_heads / num_kv_heads > kMaxGqa) return FP8KV_ERR_SHAPE;
    const VisiblePlan L = plan_visible(bf16 != 0, num_q_heads / num_kv_heads, num_kv_heads, num_seqs, max_query_len, num_tokens, window, sinks);
    const int v[5] = {L.shape.rs, L.shape.ng, L.nb, L.paired, L.ranks};
    for (int i = 0; i < 5; ++i) out[i] = v[i];
    return FP8KV_OK;
}
