// Split-KV paged GQA decode over an MXFP4 cache, pairs of 64-byte rows staged through LDS.
//
// The rows (128 values) of two neighbouring kv heads of a token are one 128-byte line, so a workgroup takes two heads and every
// wavefront reads whole lines: the rows of a step of 32 tokens (K, V and their scales, 8.5 KB) go from memory straight into LDS -
// global_load_lds, no registers in between.  Each wavefront has two such places of its own and needs no barrier: it reads a
// step's rows into registers in the layout of the MFMA operands (fdk_splitkv_mx4.h), requests the step after next into the place
// just read, and works on the heads one by one; up to 136 KB are under way per compute unit.
//
// A load instruction fills 64 consecutive 16-byte pieces of LDS, eight tokens.  The eight pieces of token t's rows are stored in
// the order s -> s ^ swizzle(t), applied on the memory side (the lane whose bytes land in piece s fetches piece s ^ swizzle(t)):
// the 16 tokens of a K tile, and the four tokens of a V load, then sit in different banks.  The loads are issued from inline asm
// and waited for by count (loads return in order, every step issues the same number), as in fdk_splitkv_mfma_shared.h; the
// compiler sees no other vector loads in that loop: page numbers come as scalar loads (pages of 16 << n tokens).
//
// Measured, whole calls, 4 sequences x 8 kv heads x 131072 tokens (570 MB): 106 us, 5.4 TB/s; without the arithmetic 98; the same
// rows laid out by head stream at 97 (fdk_splitkv_mx4.h).  With probabilities of one part, which took 104: pairs loaded into
// registers (one buffer, L2) 116, eight heads per workgroup sharing four staged places behind a barrier 111; and, for rows of 32
// bytes, which are not staged, four heads of a line per wavefront 94 where pairs in registers took 70 (now 73; 64 sequences x 8
// kv heads x 8192 tokens).

#include "fdk_splitkv_mx4.h"

namespace fdk {

namespace {

constexpr int kMx4Place = 2 * (32 * 128 + 32 * 2 * 4);      // bytes of a step's rows and scales

template <int QDT, int MODE, bool FOLDED>
__global__ __launch_bounds__(512) void splitkv_mx4_staged_kernel(const SplitParams p, const Mx4Scales x) {
    constexpr int D = 128, NH = 2;             // values of a row, kv heads of a workgroup
    using T = Mx4Tile<D>;
    using Math = Mx4Math<QDT, D, FOLDED>;
    constexpr int KSTEPS = D / 32, DB = D / 16;
    constexpr int kTileHeads = 16;
    constexpr bool kOneSegment = false;        // (fdk_splitkv_mfma_work.h: no single-launch form, units mapped to XCDs)
    constexpr bool kRowsShareLines = true, kScalesShareLines = true;
    constexpr bool kFirstPieceStraight = true;
    constexpr int RB = D / 2;                  // bytes of a row
    constexpr int RU = NH * RB / 16;           // 16-byte pieces of a token's rows
    static_assert(RU == 8, "the rows of a token are one line");
    constexpr int kRowBytes = kStep * RU * 16; // K rows of a step
    constexpr int kScaleBytes = kStep * NH * 4;          // K scales of a step: a dword per row
    constexpr int kPlace = 2 * (kRowBytes + kScaleBytes);
    static_assert(kPlace == kMx4Place, "K rows, V rows, K scales, V scales");
    constexpr int kLoads = 10;                 // of a step

    extern __shared__ __attribute__((aligned(16))) char lds[];      // [kWaves][2 places]; then, for the merge, as in splitkv_mx4_kernel
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int a = lane >> 4, c = lane & 15;
    const int nh = NH, hl = 0;                 // kv heads of a workgroup: every wavefront works on all of them
    const int tix = wave;
    constexpr int kScratch = D * 64;
    float* sm_m = reinterpret_cast<float*>(lds + kWaves * NH * kScratch);
    float* sm_l = sm_m + kWaves * NH * 16;
    int* const s_next = reinterpret_cast<int*>(sm_l + kWaves * NH * 16);

    auto write_empty_rows = [&](const int b, const int head0, const int heads_here) {
        Math::write_empty_rows(p, b, head0, heads_here, lane);
    };
    auto swizzle = [](int t) { return ((t >> 1) & 1) << 2 | ((t >> 2) & 3); };

    // ---- the loads: row instruction j fetches tokens 8 j .. 8 j + 7 of the step, this lane piece lane % 8 of token 8 j + lane / 8 ----
    const int tok8 = lane >> 3;
    uint32_t piece[2];                         // the byte of the token's rows that goes there, for even and odd j
#pragma unroll
    for (int j = 0; j < 2; ++j) piece[j] = (uint32_t)(((lane & 7) ^ swizzle(8 * j + tok8)) * 16);
    // the scale instructions: row (token, head) of the step
    const int sc_tok = lane / NH, sc_head = lane % NH;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds + (uint32_t)(wave * 2 * kPlace);
    // ---- and this lane's operands in a place, of kv head h ----
    const int krow = (c >> 2) + 4 * (c & 3);                  // the token (of 16) that row c of S^T belongs to
    auto k_at = [&](int h) { return (krow * RU + ((h * (RB / 16) + a) ^ swizzle(krow))) * 16; };
    auto v_at = [&](int h, int i) {
        const int t = a + 4 * i, byte = h * RB + c * (D / 32);
        return kRowBytes + (t * RU + ((byte >> 4) ^ swizzle(t))) * 16 + (byte & 15);
    };
    const int ks_at = 2 * kRowBytes + krow * NH * 4 + (D / 4) * a / kMxBlock;
    const int vs_at = 2 * kRowBytes + kScaleBytes + (a + 4 * (c & 3)) * NH * 4 + DB * c / kMxBlock;

    // One piece, as in splitkv_mx4_kernel
    const int64_t kv_step = MODE == WM_SHARES ? p.heads_per_tile : (int64_t)p.group * p.num_splits;
    auto run_piece = [&](const int b, const int hgb, const int ht, const int c_start, const int c_limit, const int64_t prow0,
                         const int prow_step, MergeRows) {
    const int kvh0 = hgb * NH;
    const int head0 = kvh0 * p.group + ht * kTileHeads;
    const int heads_here = min(kTileHeads, p.group - ht * kTileHeads);
    uint4 qb[NH][KSTEPS];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
        const uint16_t* qp = reinterpret_cast<const uint16_t*>(p.q) + (int64_t)b * p.q_sb +
                             (int64_t)(head0 + h * p.group + Math::head_of(c, heads_here)) * p.q_sh + (D / 4) * a;
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) qb[h][ks] = *reinterpret_cast<const uint4*>(qp + 8 * ks);
    }
    const ConstI32 tbl = as_const(p.block_table + (int64_t)b * p.tbl_sb);
    const int kv_len = min(as_const(p.kv_lens)[b], p.max_tokens);
    if (c_start >= kv_len) {
        if (p.direct && tix == 0) {
#pragma unroll
            for (int h = 0; h < NH; ++h) write_empty_rows(b, head0 + h * p.group, heads_here);
        }
        return;
    }
    const int c_end = min(c_limit, kv_len);
    const int last = c_end - 1;
    const int pmask = p.page_size - 1;
    const float inv_cap = p.soft_cap > 0.f ? 1.0f / p.soft_cap : 0.f;
    const char* kplane = reinterpret_cast<const char*>(p.k) + (int64_t)kvh0 * p.k_sh;
    const char* vplane = reinterpret_cast<const char*>(p.v) + (int64_t)kvh0 * p.v_sh;
    const char* ksplane = reinterpret_cast<const char*>(x.k) + (int64_t)(kvh0 + sc_head) * x.k_sh;      // (of this lane's head)
    const char* vsplane = reinterpret_cast<const char*>(x.v) + (int64_t)(kvh0 + sc_head) * x.v_sh;
    // this lane's byte offsets from the first token of an instruction
    const uint32_t krows = (uint32_t)tok8 * (uint32_t)p.k_st, vrows = (uint32_t)tok8 * (uint32_t)p.v_st;
    const uint32_t kscales = (uint32_t)(sc_tok & 15) * (uint32_t)x.k_st;
    const uint32_t vscales = (uint32_t)(sc_tok & 15) * (uint32_t)x.v_st;

    struct Pages { int32_t pg[2]; };           // of a step's two tiles of 16 tokens; positions past the piece stand for its last
    auto fetch_pages = [&](int t, Pages& pi) {
        const int tok0 = c_start + t * kStep;
        pi.pg[0] = tbl[min(tok0, last) >> p.page_shift];
        pi.pg[1] = tbl[min(tok0 + 16, last) >> p.page_shift];
    };
    // (several q-head tiles read the same rows: those run on one XCD, and plain loads leave the lines in its L2)
    auto row_load = [&](const char* base, uint32_t off, uint32_t dst, auto shared_tag) {
        if constexpr (decltype(shared_tag)::value)
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(dst) : "memory");
        else
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(base), "s"(dst) : "memory");
    };
    auto scale_load = [&](const char* at, uint32_t dst) {
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(at), "s"(dst) : "memory");
    };
    // byte offset of a row: page strides and in-page offsets are below 4 GiB
    auto offset = [&](int64_t sp, int64_t st, int32_t pg, int slot) {
        return (uint64_t)(uint32_t)pg * (uint32_t)sp + (uint64_t)((uint32_t)slot * (uint32_t)st);
    };
    // The rows and scales of step t, into the LDS bytes from dst.  CLAMP: positions past the piece repeat its last token.
    auto issue = [&](int t, const Pages& pi, uint32_t dst, auto clamp_tag, auto shared_tag) {
        constexpr bool CLAMP = decltype(clamp_tag)::value;
        const int tok0 = c_start + t * kStep;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const int first = CLAMP ? min(tok0 + 16 * hf, last) : tok0 + 16 * hf;
            const char* kp = kplane + offset(p.k_sp, p.k_st, pi.pg[hf], first & pmask);
            const char* vp = vplane + offset(p.v_sp, p.v_st, pi.pg[hf], first & pmask);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t to = dst + 1024 * (2 * hf + j);
                if constexpr (CLAMP) {
                    const uint32_t mine = (uint32_t)min(8 * j + tok8, last - first);
                    row_load(kp, mine * (uint32_t)p.k_st + piece[j], to, shared_tag);
                    row_load(vp, mine * (uint32_t)p.v_st + piece[j], to + kRowBytes, shared_tag);
                } else {
                    row_load(kp + 8 * j * (uint32_t)p.k_st, krows + piece[j], to, shared_tag);
                    row_load(vp + 8 * j * (uint32_t)p.v_st, vrows + piece[j], to + kRowBytes, shared_tag);
                }
            }
        }
        const uint32_t kd = dst + 2 * kRowBytes, vd = kd + kScaleBytes;
        const bool second = sc_tok >= 16;                             // the tile of this lane's token
        if constexpr (CLAMP) {
            const int n = min(tok0 + sc_tok, last), pg = second ? pi.pg[1] : pi.pg[0];
            scale_load(ksplane + offset(x.k_sp, x.k_st, pg, n & pmask), kd);
            scale_load(vsplane + offset(x.v_sp, x.v_st, pg, n & pmask), vd);
        } else {
            const uint64_t k0 = offset(x.k_sp, x.k_st, pi.pg[0], tok0 & pmask), k1 = offset(x.k_sp, x.k_st, pi.pg[1], (tok0 + 16) & pmask);
            const uint64_t v0 = offset(x.v_sp, x.v_st, pi.pg[0], tok0 & pmask), v1 = offset(x.v_sp, x.v_st, pi.pg[1], (tok0 + 16) & pmask);
            scale_load(ksplane + (second ? k1 : k0) + kscales, kd);
            scale_load(vsplane + (second ? v1 : v0) + vscales, vd);
        }
    };

    float m_run[NH], l_run[NH];
    f32x4_t acc[NH][DB];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
        m_run[h] = -INFINITY;
        l_run[h] = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[h][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    // q is waited for before the first direct load: the compiler counts only the loads it knows
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) asm volatile("" : "+v"(qb[h][ks].x), "+v"(qb[h][ks].y), "+v"(qb[h][ks].z), "+v"(qb[h][ks].w));

    // ---- the steps of this wavefront: tix, tix + kWaves ... ----
    const int n_steps = (c_end - c_start + kStep - 1) / kStep, n_full = (c_end - c_start) / kStep;
    auto request = [&](int t, const Pages& pi, uint32_t dst) {
        if (t >= n_steps) return;
        if (t < n_full && p.head_tiles == 1) issue(t, pi, dst, BoolTag<false>(), BoolTag<false>());
        else if (t < n_full) issue(t, pi, dst, BoolTag<false>(), BoolTag<true>());
        else issue(t, pi, dst, BoolTag<true>(), BoolTag<true>());
    };
    Pages pa, pb;
    fetch_pages(tix, pa);
    fetch_pages(tix + kWaves, pb);
    request(tix, pa, lds0);
    request(tix + kWaves, pb, lds0 + kPlace);
    fetch_pages(tix + 2 * kWaves, pa);
    int at = 0;
    for (int t = tix; t < n_steps; t += kWaves) {
        if (t + kWaves < n_steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const char* place = lds + wave * 2 * kPlace + at;
        T r[NH];
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const char* kp = place + k_at(h) + hf * 16 * RU * 16;
                const uint4 w = *reinterpret_cast<const uint4*>(kp);
                r[h].k[hf][0] = w.x; r[h].k[hf][1] = w.y; r[h].k[hf][2] = w.z; r[h].k[hf][3] = w.w;
                r[h].ks[hf][0] = *reinterpret_cast<const uint8_t*>(place + ks_at + (hf * 16 * NH + h) * 4);
                r[h].vs[hf][0] = *reinterpret_cast<const uint8_t*>(place + vs_at + (hf * 16 * NH + h) * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) r[h].v[4 * hf + i][0] = *reinterpret_cast<const uint32_t*>(place + v_at(h, i) + hf * 16 * RU * 16);
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");               // everything is read: the place takes the step after next
        request(t + 2 * kWaves, pa, lds0 + at);
        fetch_pages(t + 3 * kWaves, pa);
        at = kPlace - at;
        const int left = c_end - (c_start + t * kStep);
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            float sv[8];
            Math::scores(r[h], qb[h], sv);
            if (left >= kStep) Math::values(r[h], Math::softmax(sv, m_run[h], l_run[h], acc[h], p, inv_cap, a, c, left, BoolTag<false>()), acc[h]);
            else Math::values(r[h], Math::softmax(sv, m_run[h], l_run[h], acc[h], p, inv_cap, a, c, left, BoolTag<true>()), acc[h]);
        }
    }

    // ---- merge of the wavefronts through LDS (the places of all of them) ----
    __syncthreads();
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

template <int QDT>
int launch_staged(const SplitParams& p_in, const Mx4Scales& x, hipStream_t stream) {
    SplitParams p = p_in;
    if (p.fused || p.probe || p.head_dim != 128 || p.hg_per_wg != 2 || p.hkv % 2 || p.page_shift < 4) return (int)hipErrorInvalidValue;
    p.head_tiles = (p.group + 15) / 16;
    p.hg_blocks = p.hkv / 2;
    p.persistent = 0;
    const unsigned units = (unsigned)(p.hg_blocks * p.head_tiles);
    const dim3 grid = p.balanced ? dim3(units, (unsigned)p.workgroups / units) : dim3(units, (unsigned)p.num_splits, (unsigned)p.batch);
    p.shares = (int32_t)grid.y;
    p.grid_x = (int32_t)grid.x;
    p.wavefronts = kWaves;
    // the places of all wavefronts; the merge needs 16 fp32 rows per wavefront and head, and m and l
    constexpr int kLds = kWaves * 2 * kMx4Place;
    static_assert(kLds >= kWaves * 2 * (128 * 64 + 2 * 16 * (int)sizeof(float)) + 16, "the merge");
    auto* kernel = p.group <= 8 ? (p.balanced ? &splitkv_mx4_staged_kernel<QDT, WM_SHARES, true> : &splitkv_mx4_staged_kernel<QDT, WM_ONE, true>)
                                : (p.balanced ? &splitkv_mx4_staged_kernel<QDT, WM_SHARES, false> : &splitkv_mx4_staged_kernel<QDT, WM_ONE, false>);
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), kLds, stream, p, x);
    return (int)hipGetLastError();
}

}  // namespace

int launch_splitkv_mx4_staged(const SplitParams& p, const Mx4Scales& x, int q_dtype, hipStream_t stream) {
    return q_dtype == FDK_BF16 ? launch_staged<FDK_BF16>(p, x, stream) : launch_staged<FDK_FP16>(p, x, stream);
}

}  // namespace fdk
