// The walk over the visible keys of one decode query, and what it does with a chunk of them (kv_chunk.h).
//
// Visible to the query of a sequence of `len` tokens (its position is len - 1): the keys t < len with
// t >= len - window or t < sinks; window 0: all.  In 16-token groups that is a run from token 0, which
// holds the sinks, and a run that ends with the sequence; where they touch there is one.  The walk
// counts the tokens of both runs through, so splits, waves and chunks take their spans of it as of a whole
// context, and only the place of a group (its block and slot) and the masks know about the gap.
// Groups without a visible key are never read, nor are their block-table entries.
//
// KIND: e4m3 caches with one scale per tensor, bf16 caches, or block-scaled e4m3 caches (a power of
// two per 16 tokens, kv head and tensor as an e8m0 byte).  K's scale joins the factor that its group's
// scores are multiplied by anyway; V's goes into its widening to bf16, which stays exact.
//
// The probabilities enter P.V as bf16 hi + lo parts (error at most 2^-16 of each; of one rounded bf16 2^-8): one token's
// worth of queries leaves the matrix units idle most of the time, so the second MFMA costs nothing.  hi is cut off,
// not rounded, and the last bit of the fp32 weight is set (2^-23 of it), so that lo has the weight's sign and is
// not 0: an infinite V is then infinite in both products.  (Rounded to nearest, lo is 0 or negative for half of the
// weights, and 0 * inf or inf - inf is NaN.)  Where a weight is next to nothing (below 2^-100) the product may be NaN.
#pragma once
#include "kv_chunk.h"

namespace fp8kv {
namespace kv_chunk {

enum CacheKind { kE4m3 = 0, kBf16 = 1, kBlk = 2 };

struct Walk {
    int nv;             // tokens walked
    int head;           // of them, tokens of the run that holds the sinks
    int jump;           // tokens left out behind it
    int sinks, low, len;
    __device__ __forceinline__ int operator()(int t0) const { return t0 + (t0 >= head ? jump : 0); }
    // Chunks that start below this walked token may hold a key that is not visible (the end apart).
    __device__ __forceinline__ int ragged() const { return low > 0 ? head + 16 : 0; }
};

__device__ __forceinline__ Walk make_walk(int len, int window, int sinks)
{
    Walk w;
    w.len = len > 0 ? len : 0;
    w.low = window > 0 && w.len > window ? w.len - window : 0;
    w.sinks = sinks;
    const int s = sinks < w.low ? sinks : w.low;
    w.head = (s + 15) & ~15;
    const int start = w.low & ~15;
    w.jump = start > w.head ? start - w.head : 0;
    w.nv = w.len - w.jump;
    return w;
}

// The walks of a batch, end to end in groups of 16 tokens and at least one group per sequence, cut into equal parts: one
// for each workgroup of a kv head, which takes the segments of the sequences in it one after another.  Where every
// sequence has as many workgroups as any other, a ragged batch ends with a few of them on its longest sequence.  (32 x
// 8 pairs of 512..8192 tokens, one split 68.8 us, four 60.4, 32 parts per kv head 55.1; of 4096 each 46.1 and 44.3.)
// Every wave finds its part from all the lengths, which stay on the device.
constexpr int kMaxShared = 256;      // sequences: four per lane
constexpr int kMaxRecords = 256;     // segments of a sequence, as many as a call can have splits

struct Part {
    int size;           // groups of every part; 0: the parts before this one hold everything
    int seq, len;       // the first sequence, its tokens
    int start;          // where the part starts in the batch,
    int base;           // and where its first sequence does
};

// Groups of a sequence's walk.
__device__ __forceinline__ int walk_groups(int nv) { return nv > 0 ? (int)(((unsigned)nv + 15u) >> 4) : 1; }

// Inclusive scan of numbers >= 0 over the lanes of a wave, by addition or max.
template <typename F>
__device__ __forceinline__ int wave_scan(int x, F op)
{
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));      // row_shr:1, 2, 4, 8
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));      // row_bcast:15 to rows 1 and 3
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));      // row_bcast:31 to rows 2 and 3
    return x;
}

template <int K>
__device__ __forceinline__ Part find_part_k(const int32_t* seq_lens, int ns, int parts, int w, int window, int sinks, int lane)
{
    int len[K], g[K], own = 0, most = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) len[i] = seq_lens[K * lane + i < ns ? K * lane + i : ns - 1];
#pragma unroll
    for (int i = 0; i < K; ++i) {
        g[i] = K * lane + i < ns ? walk_groups(make_walk(len[i], window, sinks).nv) : 0;
        own += g[i];
        most = g[i] > most ? g[i] : most;
    }
    const int upto = wave_scan(own, [](int a, int b) { return a + b; });
    const unsigned total = (unsigned)__builtin_amdgcn_readlane(upto, 63);
    most = __builtin_amdgcn_readlane(wave_scan(most, [](int a, int b) { return a > b ? a : b; }), 63);
    // a sequence of m groups lies in m / size + 2 parts at the most
    const unsigned even = (total + (unsigned)parts - 1) / (unsigned)parts, least = (unsigned)most / (kMaxRecords - 2) + 1;
    Part r = {(int)(even > least ? even : least), 0, 0, 0, 0};
    if ((int64_t)w * r.size >= (int64_t)total) {
        r.size = 0;
        return r;
    }
    r.start = w * r.size;
    const int at = __builtin_ctzll(__ballot(r.start < upto));
    r.base = at > 0 ? __builtin_amdgcn_readlane(upto, at - 1) : 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const int gi = __builtin_amdgcn_readlane(g[i], at);
        if (!found) {
            found = r.start < r.base + gi;
            r.seq = K * at + i;
            r.len = __builtin_amdgcn_readlane(len[i], at);
            r.base += found ? 0 : gi;
        }
    }
    return r;
}

// Part w of the ns <= kMaxShared sequences.
__device__ __forceinline__ Part find_part(const int32_t* seq_lens, int ns, int parts, int w, int window, int sinks, int lane)
{
    return ns <= 64 ? find_part_k<1>(seq_lens, ns, parts, w, window, sinks, lane)
                    : find_part_k<4>(seq_lens, ns, parts, w, window, sinks, lane);
}

// A chunk's scale bytes (K low, V high), one pair per group.
template <int NG>
struct ChunkScales {
    uint32_t kv[NG];
};

template <int NG, typename PT>
__device__ __forceinline__ void issue_scales(ChunkScales<NG>& c, const PT& P, const ChunkIds<NG>& ids, int kh, int c0,
                                             int last, const Walk& w)
{
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const int t0 = c0 + 16 * g;
        const int part = (w(t0 < last ? t0 : last) & (P.pblk - 1)) >> 4;
        c.kv[g] = P.kv_scales[((int64_t)ids.blk[g] * (P.pblk >> 4) + part) * P.hkv + kh];
    }
}

// consume_chunk for a walk: keys c0 .. c0 + 16 NG of it, of which those below hi are used.
template <int NG, int KIND>
__device__ __forceinline__ void consume_visible(const ChunkRegs<NG, KIND == kBf16>& c, const ChunkScales<NG>& scales,
                                                WaveState& st, const u32x4_t (&qf)[4], float qk_scale, int c0, int hi,
                                                const Walk& w, int lp)
{
    constexpr bool B16 = KIND == kBf16;
    const bool masked = c0 + 16 * NG > hi || c0 < w.ragged();
    // of the walked token tv in the group that starts at walked token t0
    auto visible = [&](int t0, int tv) {
        const int t = w(t0) + (tv - t0);
        return tv < hi && (t >= w.low || t < w.sinks);
    };
    f32x4_t s[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < 4; ++f) acc = mfma16x16x32_bf16(k_fragment(c, g, f), as_bf16x8(qf[f]), acc);
        const float factor = KIND == kBlk ? qk_scale * e8m0_to_f32(scales.kv[g] & 0xFFu) : qk_scale;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[g][i] = acc[i] * factor;
    }
    if (masked) {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!visible(c0 + 16 * g, c0 + 16 * g + 4 * lp + i)) s[g][i] = neg_inf();
    }
    float mc = neg_inf();
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) mc = fmaxf(mc, s[g][i]);
    mc = max_xor16_32(mc);
    const float m_new = fmaxf(st.m_run, mc);
    const float m_use = m_new == neg_inf() ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(st.m_run - m_use);
    float psum = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float pv = __builtin_amdgcn_exp2f(s[g][i] - m_use);
            s[g][i] = pv;
            psum += pv;
        }
    st.l_run = st.l_run * alpha + psum;
    st.m_run = m_new;
#pragma unroll
    for (int n = 0; n < 8; ++n) st.o[n] *= alpha;
#pragma unroll
    for (int G = 0; G < NG / 2; ++G) {
        u32x4_t hi4, lo4;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const uint32_t a = __float_as_uint(s[2 * G + (d >> 1)][2 * (d & 1)]) | 1u;
            const uint32_t b = __float_as_uint(s[2 * G + (d >> 1)][2 * (d & 1) + 1]) | 1u;
            hi4[d] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            lo4[d] = pack_bf16x2(__uint_as_float(a) - __uint_as_float(a & 0xFFFF0000u),
                                 __uint_as_float(b) - __uint_as_float(b & 0xFFFF0000u));
        }
        typename VRow<B16>::type vv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) vv[j] = c.vr[G][j];
        if (masked) {                                    // 0 * NaN of a key that is not visible must not reach O
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int t0 = c0 + 32 * G + (j < 4 ? 0 : 16);
                if (!visible(t0, t0 + 4 * lp + (j & 3))) vv[j] = typename VRow<B16>::type{};
            }
        }
        u32x4_t va[8];
        if constexpr (KIND == kBf16)
            v_fragments_b16(vv, va);
        else if constexpr (KIND == kBlk)
            v_fragments(vv, va, e8m0_to_f32(scales.kv[2 * G] >> 8), e8m0_to_f32(scales.kv[2 * G + 1] >> 8));
        else
            v_fragments(vv, va);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            st.o[n] = mfma16x16x32_bf16(as_bf16x8(va[n]), as_bf16x8(hi4), st.o[n]);
            st.o[n] = mfma16x16x32_bf16(as_bf16x8(va[n]), as_bf16x8(lo4), st.o[n]);
        }
    }
}

}  // namespace kv_chunk
}  // namespace fp8kv
