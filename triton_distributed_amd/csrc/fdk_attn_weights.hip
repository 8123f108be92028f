// weights[b, kvh, n] += sum over the q heads of the group of exp(logit(b, h, n) - lse[b, h]): what each cached token receives
// from the query's attention, given the log-sum-exp that the decode returns.  gfx950.
//
// One pass over the K rows, no softmax of its own: the logits of 16 tokens x 16 q heads are S = Q K^T by MFMA with both
// operands loaded straight in their layouts, K as operand B (lane (c, a): token c, its a-th piece of every 64 bytes), so that
// lane (c, a) holds token c's logits of heads 4a .. 4a + 3 and the sum over the heads is three additions and two exchanges.
// Every weight belongs to one wavefront: no atomics, the same bits on every run.  Bound by the bytes of the K rows: 32
// sequences x 8 kv heads x 4096 tokens x 256 bytes in 51 us, 5.4 TB/s (one head a workgroup: 59 us); an fp8 cache 30 us.
#include "fdk_kv_evict.h"

namespace fdk {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4;                  // wavefronts of a workgroup
constexpr int kWorkgroupsPerCu = 4;

enum KeyKind { KEY_16BIT = 0, KEY_FP8 = 1, KEY_MX4 = 2 };

template <int QDT>
__device__ __forceinline__ f32x4_t mma16(uint4 a, uint4 b, f32x4_t c) {
    if constexpr (QDT == FDK_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// (the sum over lanes l, l ^ 16, l ^ 32, l ^ 48, see max_across_rows in fdk_splitkv_mfma.h)
__device__ __forceinline__ float sum_across_rows(float x) {
    float a = x, b = x;
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    a += b;
    b = a;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    return a + b;
}

// How lane group a's pieces of a K row feed the D / 32 MFMA steps: the k index is a summation index, so any order of the
// values does that Q is held in, too.  16 bit: step s takes values 32 s + 8 a .. + 7 (a load instruction reads 64 contiguous
// bytes of each row).  fp8: a 16-byte piece 64 j + 16 a .. + 15 feeds steps 2 j and 2 j + 1.  MXFP4: the a-th quarter of the row.
template <int KIND, int D>
__device__ __forceinline__ constexpr int first_value(int step, int a) {
    return KIND == KEY_16BIT ? 32 * step + 8 * a : KIND == KEY_FP8 ? 64 * (step / 2) + 16 * a + 8 * (step % 2) : (D / 4) * a + 8 * step;
}

// MANY: more than 16 q heads per kv head - their fragments are read again for every step (from the L1) instead of being held
// TILE: pages of a power of two and at least 16 tokens - one page number per tile of 16, wave-uniform addresses
template <int QDT, int KIND, int D, bool MANY, bool TILE>
__global__ __launch_bounds__(64 * kWaves) void attn_weights_kernel(const AttnWeightsParams p) {
    using P2 = Pack2<QDT>;
    constexpr int STEPS = D / 32;
    // tiles of 16 tokens whose rows are under way together (four, where rows are short, measured 30-40 % slower: the shares of
    // ragged batches are cut into longer steps)
    constexpr int TILES = KIND == KEY_16BIT ? (D <= 128 ? 2 : 1) : KIND == KEY_FP8 ? (D <= 256 ? 2 : 1) : 2;
    constexpr bool kWholeLines = (KIND == KEY_16BIT ? 2 * D : KIND == KEY_FP8 ? D : D / 2) % 128 == 0;
    constexpr int LOADS = KIND == KEY_16BIT ? STEPS : KIND == KEY_FP8 ? D / 64 : D > 64 ? D / 128 : 1;     // 16-byte pieces
    constexpr int MXS = KIND == KEY_MX4 && D == 256 ? 2 : 1;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int a = lane >> 4, c = lane & 15;
    // A unit of work: a share of a sequence for a block of nh neighbouring kv heads, one to a wavefront (the wavefronts of a head
    // interleave steps): together they read longer runs of every token, and rows below 128 bytes share their lines within the
    // workgroup; all blocks of a (sequence, share) run on one XCD, whose L2 then serves what blocks share.
    const int nh = p.heads_per_wg, blocks = p.hkv / nh;
    int unit, row;
    {
        const int id = (int)blockIdx.x, rows = p.batch * p.shares, T = blocks;
        const int full = rows & ~7;
        if (id < full * T) {
            const int blk = id / (8 * T), in = id - blk * 8 * T;
            unit = in >> 3;
            row = blk * 8 + (in & 7);
        } else {
            const int rest = id - full * T;
            row = full + rest / T;
            unit = rest % T;
        }
    }
    const int kvh = unit * nh + wave % nh;
    const int wg_step = kWaves / nh * 16 * TILES;
    int b, share, per = 0;                                     // per: tokens of a share, in the balanced form
    if (p.balanced) {
        // Shares of one size for the whole batch, counted in steps: as small as the workgroups allow (or, where the remainders of
        // the sequences do not fit, what surely fits: sum of ceil(steps / size) <= steps / size + batch).  Every wavefront finds
        // the same sizes and its own place, 64 sequences at a time.
        const int rows = p.batch * p.shares;
        auto steps_of = [&](int i) { return i < p.batch ? (max(min(p.kv_lens[i], p.max_tokens), 0) + wg_step - 1) / wg_step : 0; };
        const int mine = steps_of(lane);
        int total = mine;
        for (int i = 64 + lane; i - lane < p.batch; i += 64) total += steps_of(i);
        total = wave_sum_i32(total);
        int size = max((total + rows - 1) / rows, 1);
        int need = (mine + size - 1) / size;
        for (int i = 64 + lane; i - lane < p.batch; i += 64) need += (steps_of(i) + size - 1) / size;
        if (wave_sum_i32(need) > rows) size = (total + rows - p.batch - 1) / (rows - p.batch);
        int before = 0;                                        // shares of the sequences before the 64 looked at
        b = -1;
        share = 0;
        for (int i = lane; i - lane < p.batch; i += 64) {
            const int n = ((i < 64 ? mine : steps_of(i)) + size - 1) / size, incl = before + wave_scan_i32(n);
            const uint64_t past = __builtin_amdgcn_ballot_w64(incl > row);
            if (past) {
                const int at = __builtin_ctzll(past);
                b = i - lane + at;
                share = row - (__builtin_amdgcn_readlane(incl, at) - __builtin_amdgcn_readlane(n, at));
                break;
            }
            before = __builtin_amdgcn_readlane(incl, 63);
        }
        b = __builtin_amdgcn_readfirstlane(b);
        if (b < 0) return;
        per = size * wg_step;
    } else {
        b = row / p.shares;
        share = row - b * p.shares;
    }
    // (what does not depend on the length is requested before it)
    const uint16_t* qrow = reinterpret_cast<const uint16_t*>(p.q) + (int64_t)b * p.q_sb;
    const float* lse_row = p.lse + (int64_t)b * p.lse_sb;
    const int head_tiles = MANY ? (p.group + 15) / 16 : 1;
    uint4 qf[STEPS];
    float lse2[4];
    auto load_q = [&](int ht) {
        const uint16_t* qp = qrow + (int64_t)(kvh * p.group + min(ht * 16 + c, p.group - 1)) * p.q_sh;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) qf[s] = *reinterpret_cast<const uint4*>(qp + first_value<KIND, D>(s, a));
#pragma unroll
        for (int i = 0; i < 4; ++i) lse2[i] = lse_row[kvh * p.group + min(ht * 16 + 4 * a + i, p.group - 1)] * kLog2e;
    };
    if (!MANY) load_q(0);
    typedef const __attribute__((address_space(4))) int32_t* ConstI32;     // read-only for the whole kernel: scalar loads
    const int kv_len = min(((ConstI32)(uintptr_t)p.kv_lens)[b], p.max_tokens);
    // equal shares of the sequence's own length
    if (!p.balanced) per = max(((kv_len + p.shares - 1) / p.shares + wg_step - 1) / wg_step, 1) * wg_step;
    const int64_t begin64 = (int64_t)share * per;
    if (begin64 >= kv_len) return;
    const int begin = (int)begin64, end = (int)min(begin64 + per, (int64_t)kv_len);

    const ConstI32 tbl = (ConstI32)(uintptr_t)(p.block_table + (int64_t)b * p.tbl_sb);
    const char* kplane = reinterpret_cast<const char*>(p.k) + (int64_t)kvh * p.k_sh;
    const uint8_t* splane = p.k_block_scale + (int64_t)kvh * p.bs_sh;
    float* wrow = p.weights + (int64_t)b * p.w_sb + (int64_t)kvh * p.w_sh;
    float kscale = 1.f;
    if (KIND == KEY_FP8 && p.k_scale) kscale = p.k_scale[kvh];
    const bool softcap = p.soft_cap > 0.f;
    const float inv_cap = softcap ? 1.0f / p.soft_cap : 0.f;

    auto page_of = [&](int n) { return tbl[p.page_shift < 0 ? n / p.page_size : n >> p.page_shift]; };
    struct Step {
        uint4 raw[TILES][LOADS];
        uint32_t sc[TILES][MXS];
        float old;
    };
    struct Pages { int32_t pg[TILES]; };
    // (positions past the end: the last token's page)
    auto first_of = [&](int tok, int t) { return min(tok + 16 * t, (end - 1) & ~15); };       // TILE
    auto fetch_pages = [&](int tok, Pages& pi) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
            pi.pg[t] = TILE ? tbl[first_of(tok, t) >> p.page_shift] : page_of(min(tok + 16 * t + c, end - 1));
    };
    // byte offset of a row: page strides and in-page offsets are below 4 GiB, one 32 x 32 -> 64 bit multiply-add
    auto offset = [&](int64_t sp, int64_t st, uint32_t pg, uint32_t slot) {
        return (uint64_t)pg * (uint32_t)sp + (uint64_t)(slot * (uint32_t)st);
    };
    // rows past the end repeat the last one; lane 16 t + c keeps the weight of token c of tile t
    auto issue = [&](int tok, const Pages& pi, Step& r) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const char *kp, *sp;
            if constexpr (TILE) {
                const int first = first_of(tok, t);
                const uint32_t slot = (uint32_t)(first & (p.page_size - 1)), mine = (uint32_t)min(c, end - 1 - first);
                kp = kplane + offset(p.k_sp, p.k_st, (uint32_t)pi.pg[t], slot) + (uint32_t)(mine * (uint32_t)p.k_st);
                sp = reinterpret_cast<const char*>(splane) + offset(p.bs_sp, p.bs_st, (uint32_t)pi.pg[t], slot) + (uint32_t)(mine * (uint32_t)p.bs_st);
            } else {
                const int n = min(tok + 16 * t + c, end - 1);
                const uint32_t slot = (uint32_t)(p.page_shift < 0 ? n % p.page_size : (n & (p.page_size - 1)));
                kp = kplane + offset(p.k_sp, p.k_st, (uint32_t)pi.pg[t], slot);
                sp = reinterpret_cast<const char*>(splane) + offset(p.bs_sp, p.bs_st, (uint32_t)pi.pg[t], slot);
            }
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                if constexpr (KIND == KEY_MX4 && D == 64) {
                    const uint2 w = *reinterpret_cast<const uint2*>(kp + 8 * a);
                    r.raw[t][j] = make_uint4(w.x, w.y, 0, 0);
                } else if constexpr (KIND == KEY_MX4) {
                    r.raw[t][j] = *reinterpret_cast<const uint4*>(kp + (D / 8) * a + 16 * j);
                } else {
                    // (rows of whole lines are read by one wavefront once: past the caches)
                    const char* at = kp + 64 * j + 16 * a;
                    r.raw[t][j] = kWholeLines ? load_stream16(at) : *reinterpret_cast<const uint4*>(at);
                }
            }
            if constexpr (KIND == KEY_MX4) {
#pragma unroll
                for (int g = 0; g < MXS; ++g) r.sc[t][g] = *reinterpret_cast<const uint8_t*>(sp + (D / 4) * a / kMxBlock + g);
            }
        }
        const int mine = tok + (lane & (16 * TILES - 1));
        r.old = lane < 16 * TILES && mine < end ? wrow[mine] : 0.f;
    };
    auto work = [&](int tok, const Step& r) {
        float sum[TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t) sum[t] = 0.f;
        for (int ht = 0; ht < head_tiles; ++ht) {
            if (MANY) load_q(ht);
            f32x4_t s[TILES];
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                s[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    uint4 kf;
                    if constexpr (KIND == KEY_16BIT) {
                        kf = r.raw[t][st];
                    } else if constexpr (KIND == KEY_FP8) {
                        // (k8 * scale) rounded to the q dtype, as the decode does by default
                        const uint4 w = r.raw[t][st / 2];
                        const uint32_t two[2] = {st % 2 ? w.z : w.x, st % 2 ? w.w : w.y};
                        uint32_t o[4];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const f32x2_t k01 = __builtin_amdgcn_cvt_pk_f32_fp8(two[i], false);
                            const f32x2_t k23 = __builtin_amdgcn_cvt_pk_f32_fp8(two[i], true);
                            o[2 * i] = P2::pack(k01.x * kscale, k01.y * kscale);
                            o[2 * i + 1] = P2::pack(k23.x * kscale, k23.y * kscale);
                        }
                        kf = make_uint4(o[0], o[1], o[2], o[3]);
                    } else {
                        const uint4 w4 = r.raw[t][st / 4];
                        const uint32_t w = st % 4 == 0 ? w4.x : st % 4 == 1 ? w4.y : st % 4 == 2 ? w4.z : w4.w;
                        const float f = mx_scale(r.sc[t][MXS == 2 ? st / 4 : 0]);
                        kf = make_uint4(mx_unpack2<QDT, 0>(w, f), mx_unpack2<QDT, 1>(w, f), mx_unpack2<QDT, 2>(w, f), mx_unpack2<QDT, 3>(w, f));
                    }
                    s[t] = mma16<QDT>(qf[st], kf, s[t]);
                }
            }
            if (softcap) {
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t][i] = soft_cap_fn(s[t][i] * p.sm_scale, p.soft_cap, inv_cap) * kLog2e;
            } else {
#pragma unroll
                for (int t = 0; t < TILES; ++t) s[t] *= p.scale_log2;
            }
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = fast_exp2(s[t][i] - lse2[i]);
                    sum[t] += ht * 16 + 4 * a + i < p.group ? e : 0.f;
                }
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t) sum[t] = sum_across_rows(sum[t]);
        const int mine = tok + (lane & (16 * TILES - 1));
        if (lane < 16 * TILES && mine < end) {
            float x = sum[0];
            if (TILES >= 2 && a == 1) x = sum[TILES >= 2 ? 1 : 0];
            wrow[mine] = r.old + x;
        }
    };
    // two register buffers (long rows: one): the next step's rows are requested before a step is worked on, page numbers a step
    // further ahead
    int tok = begin + wave / nh * 16 * TILES;
    if (tok >= end) return;
    Pages pa, pb;
    fetch_pages(tok, pa);
    if constexpr (D <= 256) {
        Step ra, rb;
        fetch_pages(tok + wg_step, pb);
        issue(tok, pa, ra);
        for (;;) {
            const int next = tok + wg_step, after = next + wg_step;
            fetch_pages(after, pa);
            if (next < end) issue(next, pb, rb);
            work(tok, ra);
            if (next >= end) return;
            fetch_pages(after + wg_step, pb);
            if (after < end) issue(after, pa, ra);
            work(next, rb);
            if (after >= end) return;
            tok = after;
        }
    } else {
        Step r;
        for (; tok < end; tok += wg_step) {
            issue(tok, pa, r);
            fetch_pages(tok + wg_step, pa);
            work(tok, r);
        }
    }
}

template <int QDT, int KIND, int D>
int launch_d(const AttnWeightsParams& p, dim3 grid, hipStream_t stream) {
    const bool tile = p.page_shift >= 4;
#define FDK_WEIGHTS_LAUNCH(MANY, TILE) \
    hipLaunchKernelGGL((attn_weights_kernel<QDT, KIND, D, MANY, TILE>), grid, dim3(64 * kWaves), 0, stream, p)
    if (p.group > 16) {
        if (tile) FDK_WEIGHTS_LAUNCH(true, true);
        else FDK_WEIGHTS_LAUNCH(true, false);
    } else {
        if (tile) FDK_WEIGHTS_LAUNCH(false, true);
        else FDK_WEIGHTS_LAUNCH(false, false);
    }
#undef FDK_WEIGHTS_LAUNCH
    return (int)hipGetLastError();
}

template <int QDT, int KIND>
int launch_kind(const AttnWeightsParams& p, int head_dim, dim3 grid, hipStream_t stream) {
    switch (head_dim) {
        case 64: return launch_d<QDT, KIND, 64>(p, grid, stream);
        case 128: return launch_d<QDT, KIND, 128>(p, grid, stream);
        case 256: return launch_d<QDT, KIND, 256>(p, grid, stream);
        default: break;
    }
    if constexpr (KIND != KEY_MX4) {
        if (head_dim == 192) return launch_d<QDT, KIND, 192>(p, grid, stream);
        if (head_dim == 576) return launch_d<QDT, KIND, 576>(p, grid, stream);
    }
    return (int)hipErrorInvalidValue;
}

}  // namespace

int launch_attn_weights(const AttnWeightsParams& p_in, int head_dim, int q_dtype, int kv_dtype, int num_cus, hipStream_t stream) {
    AttnWeightsParams p = p_in;
    p.heads_per_wg = p.hkv % 4 == 0 ? 4 : p.hkv % 2 == 0 ? 2 : 1;
    // Shares of a sequence per block of heads: enough workgroups for a few to a compute unit (they need no merge, so cutting a
    // sequence finer costs only the loads of q again), at most one per step.
    const int64_t units = (int64_t)p.batch * (p.hkv / p.heads_per_wg);
    int64_t shares = (kWorkgroupsPerCu * (int64_t)num_cus + units - 1) / units;
    const int64_t most = ((int64_t)p.max_tokens + 31) / 32;
    if (shares > most) shares = most;
    if (shares < 1) shares = 1;
    p.shares = (int32_t)shares;
    // Long tables may hold sequences of very different lengths: the workgroups then go to the sequences by their lengths, for the
    // price of kv_lens before anything else (16 sequences x 8 heads of 100 .. 16384 tokens, 64-byte rows: 22.8 us against 26.5;
    // 32 of 4096 each, 256-byte rows: 51.5 against 51.2).  (Steps are counted in 32 bits.)
    p.balanced = shares > 1 && p.batch > 1 && p.max_tokens >= 2048 && (int64_t)p.batch * p.max_tokens < ((int64_t)1 << 35);
    const dim3 grid((unsigned)(units * shares));
    const bool bf16 = q_dtype == FDK_BF16;
    if (kv_dtype == FDK_MXFP4)
        return bf16 ? launch_kind<FDK_BF16, KEY_MX4>(p, head_dim, grid, stream) : launch_kind<FDK_FP16, KEY_MX4>(p, head_dim, grid, stream);
    if (kv_dtype == FDK_FP8_E4M3)
        return bf16 ? launch_kind<FDK_BF16, KEY_FP8>(p, head_dim, grid, stream) : launch_kind<FDK_FP16, KEY_FP8>(p, head_dim, grid, stream);
    return bf16 ? launch_kind<FDK_BF16, KEY_16BIT>(p, head_dim, grid, stream) : launch_kind<FDK_FP16, KEY_16BIT>(p, head_dim, grid, stream);
}

}  // namespace fdk
