// Split-KV paged GQA decode over an MXFP4 cache, matrix-core path, gfx950.
//
// The same contract, pieces, work distribution and partial rows as fdk_splitkv_mfma.h, for a cache of 4-bit rows (counterpart
// in the reference: kernel_gqa_fwd_batch_decode_split_kv, python/triton_dist/kernels/nvidia/flash_decode.py:129-239, which
// knows 16-bit caches only).  A workgroup works on one kv head and a tile of 16 q heads; its wavefronts interleave steps
// of 32 tokens and are merged through LDS at the end of the piece.
//
// A row of 128 values is 64 bytes, so nothing goes through LDS on the way: K and V are loaded in the layout of the MFMA
// operands, and converted in registers.
//   K   lane (c, a) loads the a-th quarter of token c's row.  The k index of an MFMA is only a summation index: step ks of
//       S^T = K Q^T multiplies values (D/4) a + 8 ks .. + 7, and Q^T is held in the same order.  A quarter row of 128
//       values is one block of 32: one scale per lane and tile, applied by the conversion.
//   V   lane (c, a) loads values (D/16) c .. + D/16 - 1 of the tokens whose probabilities the lane group a holds, converts
//       them (again with the scale of its own block) and pairs the tokens up with byte permutes: operand A of
//       O^T += V^T P^T, row m = c of column block db being value (D/16) c + db.
//   P   in two 16-bit parts, straight from the softmax registers: lane (h, a) holds the logits of head h for tokens a, a + 4, a + 8, a + 12 of both
//       halves of the step (K rows are assigned to the rows of S^T that way, so that one V load instruction reads four
//       consecutive tokens).
// The 64-byte rows of two kv heads share a 128-byte line, and so do the scales of four tokens and all heads: every unit of a
// (sequence, split) runs on one XCD, with loads that leave the lines in its L2 (tiles_on_one_xcd).  Pairs of 64-byte rows with
// pages of 16 << n tokens go through LDS instead (fdk_splitkv_mx4_staged.hip).
//
// Bound by the bytes of the rows, laid out by head: 4 sequences x 8 kv heads x 131072 tokens (570 MB) in 97 us, 5.9 TB/s; 32 x 8 x 4096
// (143 MB) in 27 us, 5.2 TB/s, fill and drain included; calls without the arithmetic take 87 and 24.  The arithmetic (96 conversions
// and permutes, 16 MFMAs, a softmax and the splitting of the probabilities per step of 32 tokens) is somewhat more than half of
// that time by its instructions' rates, and runs beside the loads.
#pragma once

#include "fdk_mxfp4.h"
#include "fdk_splitkv_mfma.h"

namespace fdk {

namespace {

constexpr int kWaves = 8;                  // wavefronts of a workgroup
constexpr int kStep = 32;                  // tokens per wavefront and step: two tiles of 16 rows, one k-step of P V

template <int D>
struct Mx4Tile {                           // one step in registers, as loaded
    static constexpr int KW = D / 32;      // dwords of a quarter K row
    static constexpr int VW = D >= 128 ? D / 128 : 1;     // dwords of a sixteenth of a V row (D = 64: half of one)
    static constexpr int KS = D == 256 ? 2 : 1;           // blocks a quarter K row touches
    uint32_t k[2][KW];
    uint32_t ks[2][KS];
    uint32_t v[8][VW];
    static constexpr int VS = D == 256 ? 2 : 1;           // V scales a lane loads per tile (of the four tokens of a lane group)
    uint32_t vs[2][VS];
};

// What a wavefront does with a step of 32 tokens of one kv head, and how the wavefronts of a head are merged.  Lane (c, a):
// q head c of the tile, tokens 16 hf + a + 4 i of the step.
template <int QDT, int D, bool FOLDED>
struct Mx4Math {
    using P2 = Pack2<QDT>;
    using T = Mx4Tile<D>;
    static constexpr int DB = D / 16;          // column blocks of O^T, values of a V row per lane
    static constexpr int KSTEPS = D / 32;      // MFMA steps of a K row

    static __device__ __forceinline__ f32x4_t mma(uint4 a, uint4 b, f32x4_t c) { return Mma<QDT>::qk(a, b, c); }     // 16 x 16 x 32

    // the scales of the lane group's four tokens, from the four lanes (two pairs of lanes) that loaded them
    static __device__ __forceinline__ void v_scales(const uint32_t (&in)[T::VS], float* sc) {
        if constexpr (T::VS == 1) {
            const float x0 = mx_scale(in[0]);
            sc[0] = dpp_mov<0x00>(x0);                         // quad_perm [0,0,0,0] ...
            sc[1] = dpp_mov<0x55>(x0);
            sc[2] = dpp_mov<0xAA>(x0);
            sc[3] = dpp_mov<0xFF>(x0);
        } else {
            const float x0 = mx_scale(in[0]), x1 = mx_scale(in[1]);
            sc[0] = dpp_mov<0xA0>(x0);                         // quad_perm [0,0,2,2]
            sc[1] = dpp_mov<0xF5>(x0);                         // quad_perm [1,1,3,3]
            sc[2] = dpp_mov<0xA0>(x1);
            sc[3] = dpp_mov<0xF5>(x1);
        }
    }

    // ---- S^T[token][head] = K Q^T, two tiles of 16 tokens: sv[4 hf + i] is token 16 hf + a + 4 i ----
    static __device__ __forceinline__ void scores(const T& r, const uint4 (&q)[KSTEPS], float (&sv)[8]) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks) {
                const float sc = mx_scale(r.ks[hf][T::KS == 2 ? ks / 4 : 0]);
                const uint32_t w = r.k[hf][ks];
                s = mma(make_uint4(mx_unpack2<QDT, 0>(w, sc), mx_unpack2<QDT, 1>(w, sc), mx_unpack2<QDT, 2>(w, sc),
                                   mx_unpack2<QDT, 3>(w, sc)), q[ks], s);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sv[4 * hf + i] = s[i];
        }
    }

    // Eight probabilities as operand B of P V: rounded to 16 bits, and what that left over, rounded in turn: together within 2^-16
    // (fp16: 2^-22) of them, so that the result is rounded once, when it is stored.  (The rounded ones alone are off by half a
    // step of 16 bits, as much as the result's own rounding.)  FOLDED (groups of at most eight q heads): the columns c + 8 of
    // every operand, which would be empty, stand for the heads c once more and take the second part: no matrix instruction is
    // added, and O is the sum of columns c and c + 8 (leave_part).  Larger groups multiply V twice.  In us, the rounded ones
    // alone / folded / V twice: 4 x 8 kv heads x 131072 tokens in token layout 105.7 / 106.8 / 110.4, by head 94.0 / 97.1 /
    // 101.2; 32 x 8 x 4096 35.7 / 37.1 / 37.8, by head 27.2 / 27.4 / 28.8.
    struct Probs {
        uint4 hi, lo;
    };
    // the q head of the tile that column c stands for (columns without one repeat the last, and are not stored)
    static __device__ __forceinline__ int head_of(int c, int heads_here) { return min(FOLDED ? c & 7 : c, heads_here - 1); }

    // ---- online softmax for head c over this lane group's eight tokens.  MASKED: only
    // the first `left` tokens of the step (at least one) take part ----
    template <typename MaskedTag>
    static __device__ __forceinline__ Probs softmax(float (&sv)[8], float& m_run, float& l_run, f32x4_t (&acc)[DB], const SplitParams& p,
                                                    float inv_cap, int a, int c, int left, MaskedTag) {
        if (p.soft_cap > 0.f) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sv[i] = soft_cap_fn(sv[i] * p.sm_scale, p.soft_cap, inv_cap) * kLog2e;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) sv[i] *= p.scale_log2;
        }
        if (MaskedTag::value) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (16 * (i >> 2) + a + 4 * (i & 3) >= left) sv[i] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3])), fmaxf(fmaxf(sv[4], sv[5]), fmaxf(sv[6], sv[7])));
        mx = max_across_rows(mx);
        // The running maximum moves only when a step exceeds it by more than 2^8: probabilities of up to 256 are as exact
        // in 16 bits and in the fp32 sums as those below 1, and the accumulators are rescaled a few times per piece.
        // (fp16: the reference stays 2^7 below the maximum, so that probabilities down to 2^-21 of the largest are normal fp16
        // values; the largest is then at most 2^15.)
        constexpr float kBelow = QDT == FDK_FP16 ? 7.0f : 0.0f;
        if (__builtin_amdgcn_ballot_w64(mx > m_run + (8.0f + kBelow)) != 0) {
            const float m_new = fmaxf(m_run, mx - kBelow);
            const float alpha = fast_exp2(m_run - m_new);
            l_run *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] *= alpha;
            m_run = m_new;
        }
        float pr[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) pr[i] = fast_exp2(sv[i] - m_run);
        l_run += ((pr[0] + pr[1]) + (pr[2] + pr[3])) + ((pr[4] + pr[5]) + (pr[6] + pr[7]));
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            hi[i] = P2::pack(pr[2 * i], pr[2 * i + 1]);
            lo[i] = P2::pack(pr[2 * i] - P2::lo(hi[i]), pr[2 * i + 1] - P2::hi(hi[i]));
        }
        if constexpr (FOLDED) {
#pragma unroll
            for (int i = 0; i < 4; ++i) hi[i] = c >= 8 ? lo[i] : hi[i];
        }
        return Probs{make_uint4(hi[0], hi[1], hi[2], hi[3]), make_uint4(lo[0], lo[1], lo[2], lo[3])};
    }

    // ---- O^T[value][head] += V^T P^T ----
    static __device__ __forceinline__ void values(const T& r, const Probs& pv, f32x4_t (&o)[DB]) {
        float sc[8];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) v_scales(r.vs[hf], sc + 4 * hf);
        auto pair = [&](auto byte_tag, int w, int db) {        // column blocks db, db + 1: byte `byte_tag` of the V words
            constexpr int BY = decltype(byte_tag)::value;
            uint32_t u[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = mx_unpack2<QDT, BY>(r.v[j][w], sc[j]);
            uint32_t lo[4], hi[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                lo[j] = __builtin_amdgcn_perm(u[2 * j + 1], u[2 * j], 0x05040100u);
                hi[j] = __builtin_amdgcn_perm(u[2 * j + 1], u[2 * j], 0x07060302u);
            }
            const uint4 v0 = make_uint4(lo[0], lo[1], lo[2], lo[3]), v1 = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            o[db] = mma(v0, pv.hi, o[db]);
            o[db + 1] = mma(v1, pv.hi, o[db + 1]);
            if constexpr (!FOLDED) {
                o[db] = mma(v0, pv.lo, o[db]);
                o[db + 1] = mma(v1, pv.lo, o[db + 1]);
            }
        };
#pragma unroll
        for (int w = 0; w < T::VW; ++w) {
            pair(IntTag<0>(), w, 8 * w);
            pair(IntTag<1>(), w, 8 * w + 2);
            if constexpr (D >= 128) {
                pair(IntTag<2>(), w, 8 * w + 4);
                pair(IntTag<3>(), w, 8 * w + 6);
            }
        }
    }

    // A wavefront's part of the merge: block e = i (DB / 4) + q of its D * 64 bytes holds, per lane, the values
    // DB (4 a + i) + 4 q .. + 3 of head c - every LDS instruction touches one contiguous kilobyte, and a merging lane stores
    // four consecutive values -; m and l: [16]
    static __device__ __forceinline__ void leave_part(f32x4_t (&acc)[DB], float m_run, float l_run, char* part, float* m, float* l,
                                                      int heads_here, int lane) {
        const bool live = (lane & 15) < heads_here;
        if constexpr (FOLDED) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[db][i] += dpp_mov<0x128>(acc[db][i]);              // row_ror:8: the lane of column c + 8
        }
        l_run += __shfl_xor(l_run, 16, 64);
        l_run += __shfl_xor(l_run, 32, 64);
        if (!live) return;
        float4* o = reinterpret_cast<float4*>(part);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int q = 0; q < DB / 4; ++q)
                o[(i * (DB / 4) + q) * 64 + lane] = make_float4(acc[4 * q][i], acc[4 * q + 1][i], acc[4 * q + 2][i], acc[4 * q + 3][i]);
        if (lane < 16) {
            m[lane] = m_run;
            l[lane] = l_run;
        }
    }
    // TI parts of one kv head, `stride` bytes apart (m, l: ml_stride values apart), by the TI wavefronts that left them: this one
    // takes the blocks e = first, first + TI ...  Row: q head hq of the result, or partial row prow.
    template <int TI>
    static __device__ __forceinline__ void merge_parts(const SplitParams& p, const char* parts, int stride, const float* m, const float* l,
                                                       int ml_stride, int first, int b, int hq, int64_t prow, int lane) {
        const int a = lane >> 4, c = lane & 15;
        float mw[TI], lw[TI];
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < TI; ++t) {
            mw[t] = m[t * ml_stride + c];
            lw[t] = l[t * ml_stride + c];
            mx = fmaxf(mx, mw[t]);
        }
        float sc[TI], sum = 0.f;
#pragma unroll
        for (int t = 0; t < TI; ++t) {
            sc[t] = fast_exp2(mw[t] - mx);               // mx is finite: the piece holds a token
            sum += lw[t] * sc[t];
        }
        const float norm = fast_rcp(sum);
        const float lse_nat = (mx + fast_log2(sum)) * kLn2;
#pragma unroll
        for (int t = 0; t < TI; ++t) sc[t] *= norm;
        for (int e = first; e < DB; e += TI) {
            float4 xw[TI];
#pragma unroll
            for (int t = 0; t < TI; ++t) xw[t] = reinterpret_cast<const float4*>(parts + t * stride)[e * 64 + lane];
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int t = 0; t < TI; ++t) {
                o.x += xw[t].x * sc[t];
                o.y += xw[t].y * sc[t];
                o.z += xw[t].z * sc[t];
                o.w += xw[t].w * sc[t];
            }
            const int d0 = DB * (4 * a + e / (DB / 4)) + 4 * (e % (DB / 4));
            if (p.direct) store_out4(p.out, (int64_t)b * p.out_sb + (int64_t)hq * p.out_sh + d0, o, p.out_dtype);
            else *reinterpret_cast<float4*>(p.part_o + prow * D + d0) = o;
        }
        if (first == 0 && a == 0) {
            if (p.direct) {
                if (p.lse) p.lse[(int64_t)b * p.lse_sb + hq] = lse_nat;
                if (p.pack_lse) store_out(p.out, (int64_t)b * p.out_sb + (int64_t)hq * p.out_sh + D, lse_nat, p.out_dtype);
            } else {
                p.part_lse[prow] = lse_nat;
            }
        }
    }
    // out = 0, lse = -inf for the q heads [head0, head0 + heads_here) of an empty sequence; one wavefront
    static __device__ __forceinline__ void write_empty_rows(const SplitParams& p, int b, int head0, int heads_here, int lane) {
        for (int idx = lane; idx < heads_here * D; idx += 64) {
            const int g = idx / D, d = idx % D;
            const int64_t ob = (int64_t)b * p.out_sb + (int64_t)(head0 + g) * p.out_sh;
            store_out(p.out, ob + d, 0.f, p.out_dtype);
            if (d == 0) {
                if (p.lse) p.lse[(int64_t)b * p.lse_sb + head0 + g] = -INFINITY;
                if (p.pack_lse) store_out(p.out, ob + D, -INFINITY, p.out_dtype);
            }
        }
    }
};

// NH: kv heads of a workgroup (neighbours in memory: their rows share lines).  STREAM: every line is one workgroup's alone, and
// is loaded with the non-temporal hint; otherwise plain loads leave the lines in the L2 for the next reader.  FOLDED: see
// Mx4Math::Probs.
template <int QDT, int PM, int D, int MODE, int NH, bool STREAM, bool FOLDED>
__global__ __launch_bounds__(512) void splitkv_mx4_kernel(const SplitParams p, const Mx4Scales x) {
    static_assert(PM == PM_TILE || PM == PM_ROW, "page numbers per tile of 16 tokens, or per row");
    static_assert(!STREAM || NH == 1, "two buffers of one kv head's rows");
    using T = Mx4Tile<D>;
    using Math = Mx4Math<QDT, D, FOLDED>;
    constexpr int DB = D / 16;                 // column blocks of O^T, values of a V row per lane
    constexpr int KSTEPS = D / 32;             // MFMA steps of a K row
    constexpr int kTileHeads = 16;
    constexpr bool kOneSegment = false;        // (fdk_splitkv_mfma_work.h: no single-launch form, units mapped to XCDs)
    constexpr bool kRowsShareLines = true, kScalesShareLines = true;
    constexpr bool kFirstPieceStraight = true;
    extern __shared__ __attribute__((aligned(16))) char lds[];      // [nw][NH][D * 64] then m[nw][NH][16], l[nw][NH][16], s_next

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int a = lane >> 4;
    const int c = lane & 15;
    const int nw = p.wavefronts;
    const int nh = NH, hl = 0;                 // kv heads of a workgroup: every wavefront works on all of them
    const int tix = wave;
    constexpr int kScratch = D * 64;           // 16 output rows in fp32: a wavefront's for one kv head
    float* sm_m = reinterpret_cast<float*>(lds + nw * NH * kScratch);
    float* sm_l = sm_m + nw * NH * 16;
    int* const s_next = reinterpret_cast<int*>(sm_l + nw * NH * 16);

    auto write_empty_rows = [&](const int b, const int head0, const int heads_here) {
        Math::write_empty_rows(p, b, head0, heads_here, lane);
    };

    // One piece: tokens [c_start, min(c_limit, kv_len)) of sequence b for kv heads NH hgb .. NH hgb + NH - 1 and q-head tile ht;
    // c_start is a multiple of 16.  Partial results of head g of the tile go to row prow0 + g * prow_step of the workspace,
    // those of the next kv head to the rows kv_step further on.
    const int64_t kv_step = MODE == WM_SHARES ? p.heads_per_tile : (int64_t)p.group * p.num_splits;
    auto run_piece = [&](const int b, const int hgb, const int ht, const int c_start, const int c_limit, const int64_t prow0,
                         const int prow_step, MergeRows) {
    const int kvh = hgb * NH;
    const int head0 = kvh * p.group + ht * kTileHeads;                     // + h * group for kv head kvh + h
    const int heads_here = min(kTileHeads, p.group - ht * kTileHeads);
    // Q^T: lane (h = c, a) holds q[h][(D/4) a + 8 ks .. + 7] (head_of)
    uint4 qb[NH][KSTEPS];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
        const uint16_t* qp = reinterpret_cast<const uint16_t*>(p.q) + (int64_t)b * p.q_sb +
                             (int64_t)(head0 + h * p.group + Math::head_of(c, heads_here)) * p.q_sh + (D / 4) * a;
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) qb[h][ks] = *reinterpret_cast<const uint4*>(qp + 8 * ks);
    }
    const ConstI32 tbl = as_const(p.block_table + (int64_t)b * p.tbl_sb);
    const int pmask = p.page_size - 1;
    // Page numbers of a step: one per 16 tokens, wave-uniform; or (any page size) lane l has the one of token l mod 32.
    struct Pages { int32_t pg[PM == PM_TILE ? 2 : 1]; };
    auto page_of_token = [&](int n) { return tbl[p.page_shift < 0 ? n / p.page_size : n >> p.page_shift]; };
    auto fetch_pages = [&](int t, int last, Pages& pi) {     // positions clamped to `last`
        const int tok0 = c_start + t * kStep;
        if constexpr (PM == PM_TILE) {
            pi.pg[0] = tbl[min(tok0, last) >> p.page_shift];
            pi.pg[1] = tbl[min(tok0 + 16, last) >> p.page_shift];
        } else {
            pi.pg[0] = page_of_token(min(tok0 + (lane & 31), last));
        }
    };
    // (ahead of kv_len: clamped to the table, the entries behind the sequence's end are fetched but never used)
    Pages pa, pb;
    fetch_pages(tix, p.max_tokens - 1, pa);
    fetch_pages(tix + nw, p.max_tokens - 1, pb);
    const int kv_len = min(as_const(p.kv_lens)[b], p.max_tokens);
    if (c_start >= kv_len) {
        if (p.direct && tix == 0) {
#pragma unroll
            for (int h = 0; h < NH; ++h) write_empty_rows(b, head0 + h * p.group, heads_here);
        }
        return;
    }
    const int c_end = min(c_limit, kv_len);
    const float inv_cap = p.soft_cap > 0.f ? 1.0f / p.soft_cap : 0.f;

    const char* kplane = reinterpret_cast<const char*>(p.k) + (int64_t)kvh * p.k_sh;
    const char* vplane = reinterpret_cast<const char*>(p.v) + (int64_t)kvh * p.v_sh;
    const char* ksplane = reinterpret_cast<const char*>(x.k) + (int64_t)kvh * x.k_sh;
    const char* vsplane = reinterpret_cast<const char*>(x.v) + (int64_t)kvh * x.v_sh;
    const int krow = (c >> 2) + 4 * (c & 3);                  // the token (of 16) that row c of S^T belongs to
    const uint32_t kbyte = (uint32_t)(a * (D / 8)), vbyte = (uint32_t)(c * (D / 32));
    const uint32_t ksbyte = (uint32_t)((D / 4) * a / kMxBlock), vsbyte = (uint32_t)(DB * c / kMxBlock);
    // V scales: four neighbouring lanes hold values of one block (D = 256: two lanes) and need the scales of the same four
    // tokens of each tile; each lane loads one token's (two tokens') and they exchange (v_scales).
    const int vstok = a + 4 * (T::VS == 1 ? c & 3 : c & 1);               // + 8 g: the token of scale g

    auto load = [&](auto type_tag, const char* at) {
        using V = decltype(type_tag);
        if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const V*>(at));
        else return *reinterpret_cast<const V*>(at);
    };
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
    auto load_k = [&](const char* at, uint32_t (&dst)[T::KW]) {
        if constexpr (D == 64) {
            const u32x2_t w = load(u32x2_t(), at);
            dst[0] = w.x; dst[1] = w.y;
        } else {
#pragma unroll
            for (int j = 0; j < T::KW; j += 4) {
                const u32x4_t w = load(u32x4_t(), at + 4 * j);
                dst[j] = w.x; dst[j + 1] = w.y; dst[j + 2] = w.z; dst[j + 3] = w.w;
            }
        }
    };
    auto load_v = [&](const char* at, uint32_t (&dst)[T::VW]) {
        if constexpr (D == 64) {
            dst[0] = load(uint16_t(), at);
        } else if constexpr (D == 128) {
            dst[0] = load(uint32_t(), at);
        } else {
            const u32x2_t w = load(u32x2_t(), at);
            dst[0] = w.x; dst[1] = w.y;
        }
    };
    auto load_byte = [&](const char* at) { return (uint32_t) * reinterpret_cast<const uint8_t*>(at); };
    // per-lane byte offsets of a tile's rows from its first row (PM_TILE)
    uint32_t voff[4];
    const uint32_t vsoff = (uint32_t)(vstok * x.v_st) + vsbyte;
    const uint32_t koff = (uint32_t)(krow * p.k_st) + kbyte;
    const uint32_t ksoff = (uint32_t)(krow * x.k_st) + ksbyte;
#pragma unroll
    for (int i = 0; i < 4; ++i) voff[i] = (uint32_t)((a + 4 * i) * p.v_st) + vbyte;
    // byte offset of a row: page strides and in-page offsets are below 4 GiB, one 32 x 32 -> 64 bit multiply-add
    auto offset = [&](int64_t sp, int64_t st, uint32_t pg, uint32_t slot) {
        return (uint64_t)pg * (uint32_t)sp + (uint64_t)(slot * (uint32_t)st);
    };
    // page and slot of row 0 .. 31 of step t; CLAMP: positions past c_end repeat the last token (the partial last step)
    auto place = [&](int t, const Pages& pi, int row, auto clamp_tag, uint32_t& pg, uint32_t& slot) {
        int n = c_start + t * kStep + row;
        if (decltype(clamp_tag)::value) n = min(n, c_end - 1);
        slot = (uint32_t)(p.page_shift < 0 ? n % p.page_size : (n & pmask));
        if constexpr (PM == PM_TILE) pg = (uint32_t)(row < 16 ? pi.pg[0] : pi.pg[PM == PM_TILE ? 1 : 0]);
        else pg = (uint32_t)__shfl(pi.pg[0], row, 64);
    };
    // The rows of step t.  The kv heads of a workgroup are neighbours: their rows are parts of the same lines, requested one
    // right after the other.
    auto issue_k = [&](int t, const Pages& pi, T (&r)[NH], auto clamp_tag) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            uint32_t pg, slot;
            if constexpr (PM == PM_TILE && !decltype(clamp_tag)::value) {
                pg = (uint32_t)pi.pg[hf];                                     // (wave-uniform: the lanes' part is an offset)
                slot = (uint32_t)((c_start + t * kStep + 16 * hf) & pmask);
            } else {
                place(t, pi, 16 * hf + krow, clamp_tag, pg, slot);
            }
            constexpr bool UNIFORM = PM == PM_TILE && !decltype(clamp_tag)::value;
            const char* kp = kplane + offset(p.k_sp, p.k_st, pg, slot);
            const char* ksp = ksplane + offset(x.k_sp, x.k_st, pg, slot);
#pragma unroll
            for (int h = 0; h < NH; ++h) load_k(kp + h * p.k_sh + (UNIFORM ? koff : kbyte), r[h].k[hf]);
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int g = 0; g < T::KS; ++g) r[h].ks[hf][g] = load_byte(ksp + h * x.k_sh + (UNIFORM ? ksoff : ksbyte) + g);
        }
    };
    auto issue_v = [&](int t, const Pages& pi, T (&r)[NH], auto clamp_tag) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            if constexpr (PM == PM_TILE && !decltype(clamp_tag)::value) {
                const uint32_t pg = (uint32_t)pi.pg[hf], slot = (uint32_t)((c_start + t * kStep + 16 * hf) & pmask);
                const char* vp = vplane + offset(p.v_sp, p.v_st, pg, slot);
                const char* vsp = vsplane + offset(x.v_sp, x.v_st, pg, slot);
#pragma unroll
                for (int g = 0; g < T::VS; ++g)
#pragma unroll
                    for (int h = 0; h < NH; ++h) r[h].vs[hf][g] = load_byte(vsp + h * x.v_sh + (uint32_t)(8 * g * x.v_st) + vsoff);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int h = 0; h < NH; ++h) load_v(vp + h * p.v_sh + voff[i], r[h].v[4 * hf + i]);
            } else {
#pragma unroll
                for (int g = 0; g < T::VS; ++g) {
                    uint32_t pg, slot;
                    place(t, pi, 16 * hf + vstok + 8 * g, clamp_tag, pg, slot);
                    const char* vsp = vsplane + offset(x.v_sp, x.v_st, pg, slot) + vsbyte;
#pragma unroll
                    for (int h = 0; h < NH; ++h) r[h].vs[hf][g] = load_byte(vsp + h * x.v_sh);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t pg, slot;
                    place(t, pi, 16 * hf + a + 4 * i, clamp_tag, pg, slot);
                    const char* vp = vplane + offset(p.v_sp, p.v_st, pg, slot) + vbyte;
#pragma unroll
                    for (int h = 0; h < NH; ++h) load_v(vp + h * p.v_sh, r[h].v[4 * hf + i]);
                }
            }
        }
    };

    float m_run[NH], l_run[NH];                  // for head c; l_run is this lane group's share of the sum
    f32x4_t acc[NH][DB];                         // acc[h][db][i] = O[head c of kv head h][DB (4 a + i) + db]
#pragma unroll
    for (int h = 0; h < NH; ++h) {
        m_run[h] = -INFINITY;
        l_run[h] = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[h][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    auto softmax = [&](int t, float (&sv)[8], int h, auto masked_tag) {
        return Math::softmax(sv, m_run[h], l_run[h], acc[h], p, inv_cap, a, c, c_end - (c_start + t * kStep), masked_tag);
    };

    // ---- pipeline ----
    // Streamed rows: two register buffers, a step's rows are requested a whole step ahead.  Rows shared through the L2: one
    // buffer, the K registers take the next step's rows as soon as the logits are there, the V registers after P V (batch 32 x
    // 8 kv heads x 4096 tokens in a single pass, before the probabilities had a second part: 36 us against 38 us with two).  Page numbers run a step further ahead: vector
    // loads of them in front of the rows, scalar ones behind (see fdk_splitkv_mfma_body.h).
    const int n_full = (c_end - c_start) / kStep;
    {
        T r[NH];
        int t = tix;
        const int st = nw;
        if (t < n_full) {
            issue_k(t, pa, r, BoolTag<false>());
            issue_v(t, pa, r, BoolTag<false>());
        }
        if constexpr (STREAM) {
            T r2[NH];
            auto work = [&](int tw, const T (&rw)[NH]) {
                float sv[8];
                Math::scores(rw[0], qb[0], sv);
                Math::values(rw[0], softmax(tw, sv, 0, BoolTag<false>()), acc[0]);
            };
            while (t + 2 * st < n_full) {
                fetch_pages(t + 2 * st, p.max_tokens - 1, pa);
                issue_k(t + st, pb, r2, BoolTag<false>());
                issue_v(t + st, pb, r2, BoolTag<false>());
                work(t, r);
                fetch_pages(t + 3 * st, p.max_tokens - 1, pb);
                issue_k(t + 2 * st, pa, r, BoolTag<false>());
                issue_v(t + 2 * st, pa, r, BoolTag<false>());
                work(t + st, r2);
                t += 2 * st;
            }
            if (t + st < n_full) {
                issue_k(t + st, pb, r2, BoolTag<false>());
                issue_v(t + st, pb, r2, BoolTag<false>());
                work(t, r);
                work(t + st, r2);
            } else if (t < n_full) {
                work(t, r);
            }
        } else {
            constexpr bool kIdsFirst = PM == PM_ROW;
            while (t < n_full) {
                const int tn = t + st;
                const bool more = tn < n_full;
                if (kIdsFirst) fetch_pages(tn + st, p.max_tokens - 1, pa);
                float sv[NH][8];
#pragma unroll
                for (int h = 0; h < NH; ++h) Math::scores(r[h], qb[h], sv[h]);
                if (more) issue_k(tn, pb, r, BoolTag<false>());
                typename Math::Probs pv[NH];
#pragma unroll
                for (int h = 0; h < NH; ++h) pv[h] = softmax(t, sv[h], h, BoolTag<false>());
#pragma unroll
                for (int h = 0; h < NH; ++h) Math::values(r[h], pv[h], acc[h]);
                if (more) issue_v(tn, pb, r, BoolTag<false>());
                if (!kIdsFirst) fetch_pages(tn + st, p.max_tokens - 1, pa);
                pb = pa;
                t = tn;
            }
        }
        if (n_full * kStep < c_end - c_start && n_full % nw == tix) {
            fetch_pages(n_full, c_end - 1, pa);
            issue_k(n_full, pa, r, BoolTag<true>());
            issue_v(n_full, pa, r, BoolTag<true>());
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                float sv[8];
                Math::scores(r[h], qb[h], sv);
                Math::values(r[h], softmax(n_full, sv, h, BoolTag<true>()), acc[h]);
            }
        }
    }

    // ---- merge of the wavefronts through LDS ----
    const bool live = c < heads_here;
#pragma unroll
    for (int h = 0; h < NH; ++h)
        Math::leave_part(acc[h], m_run[h], l_run[h], lds + (wave * NH + h) * kScratch, sm_m + (wave * NH + h) * 16, sm_l + (wave * NH + h) * 16,
                         heads_here, lane);
    __syncthreads();
    if (live) {
#pragma unroll
        for (int h = 0; h < NH; ++h)
            Math::template merge_parts<kWaves>(p, lds + h * kScratch, NH * kScratch, sm_m + h * 16, sm_l + h * 16, NH * 16, wave, b,
                                               head0 + h * p.group + c, prow0 + h * kv_step + (int64_t)c * prow_step, lane);
    }
    };   // run_piece
#include "fdk_splitkv_mfma_work.h"
}

// (one piece per workgroup or equal shares: a call with counters runs one workgroup per piece, too)
template <int QDT, int D>
int launch_mx4(const SplitParams& p_in, const Mx4Scales& x, hipStream_t stream) {
    SplitParams p = p_in;
    if (p.fused || p.probe || p.hkv % p.hg_per_wg) return (int)hipErrorInvalidValue;
    p.head_tiles = (p.group + 15) / 16;
    p.hg_blocks = p.hkv / p.hg_per_wg;
    p.persistent = 0;
    const unsigned units = (unsigned)(p.hg_blocks * p.head_tiles);
    const dim3 grid = p.balanced ? dim3(units, (unsigned)p.workgroups / units) : dim3(units, (unsigned)p.num_splits, (unsigned)p.batch);
    p.shares = (int32_t)grid.y;
    p.grid_x = (int32_t)grid.x;
    p.wavefronts = kWaves;
    const size_t lds_bytes = (size_t)kWaves * p.hg_per_wg * (D * 64 + 2 * 16 * sizeof(float)) + 16;
    const bool tile = p.page_shift >= 0 && p.page_size % 16 == 0;
#define FDK_MX4_LAUNCH_OF(PMV, MODEV, NHV, STV, FV)                                                                                           \
    do {                                                                                                                               \
        if (lds_bytes > 64 * 1024) {                                                                                                   \
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&splitkv_mx4_kernel<QDT, PMV, D, MODEV, NHV, STV, FV>), \
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_bytes);                      \
            if (e != hipSuccess) return (int)e;                                                                                        \
        }                                                                                                                              \
        hipLaunchKernelGGL((splitkv_mx4_kernel<QDT, PMV, D, MODEV, NHV, STV, FV>), grid, dim3(64 * kWaves), lds_bytes, stream, p, x);      \
    } while (0)
#define FDK_MX4_LAUNCH(PMV, MODEV, NHV, STV)                               \
    do {                                                                   \
        if (p.group <= 8) FDK_MX4_LAUNCH_OF(PMV, MODEV, NHV, STV, true);   \
        else FDK_MX4_LAUNCH_OF(PMV, MODEV, NHV, STV, false);               \
    } while (0)
#define FDK_MX4_LAUNCH_NH(NHV, STV)                                 \
    do {                                                            \
        if (p.balanced) {                                           \
            if (tile) FDK_MX4_LAUNCH(PM_TILE, WM_SHARES, NHV, STV); \
            else FDK_MX4_LAUNCH(PM_ROW, WM_SHARES, NHV, STV);       \
        } else {                                                    \
            if (tile) FDK_MX4_LAUNCH(PM_TILE, WM_ONE, NHV, STV);    \
            else FDK_MX4_LAUNCH(PM_ROW, WM_ONE, NHV, STV);          \
        }                                                           \
    } while (0)
    // Lines that no other workgroup reads: one q-head tile, and rows of whole lines or no neighbour within the line
    const bool stream_rows = p.head_tiles == 1 && (D >= 256 || p.hkv == 1 || (p.k_sh > D / 2 && p.v_sh > D / 2));
    if (p.hg_per_wg == 1) {
        if (stream_rows) FDK_MX4_LAUNCH_NH(1, true);
        else FDK_MX4_LAUNCH_NH(1, false);
    } else {
        if constexpr (D <= 128) {
            // (D = 128, pages of 16 << n tokens: fdk_splitkv_mx4_staged.hip)
            if (p.hg_per_wg != 2 || (D == 128 && tile)) return (int)hipErrorInvalidValue;
            if constexpr (D == 64) {
                FDK_MX4_LAUNCH_NH(2, false);
            } else if (p.balanced) {
                FDK_MX4_LAUNCH(PM_ROW, WM_SHARES, 2, false);
            } else {
                FDK_MX4_LAUNCH(PM_ROW, WM_ONE, 2, false);
            }
        } else {
            return (int)hipErrorInvalidValue;
        }
    }
#undef FDK_MX4_LAUNCH_NH
#undef FDK_MX4_LAUNCH
#undef FDK_MX4_LAUNCH_OF
    return (int)hipGetLastError();
}

}  // namespace

}  // namespace fdk
