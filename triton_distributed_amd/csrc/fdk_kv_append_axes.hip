// Per-head RMSNorm, rotary embedding and cache append of the new tokens for explicit positions - of one or several axes (time,
// height, width ...), each turning its own rotary pairs - and for MXFP4 caches.  gfx950.
//
// The same operator as fdk_kv_append.hip (counterpart in the reference: rmsnorm_rope_update_kv_cache_task_compute,
// python/triton_dist/mega_triton_kernel/kernels/norm.py:32-190) with the angle of pair i taken from row
// positions[axis(i), b, t] of the cos / sin tables:  y = w x rsqrt(mean(x^2) + eps), halves rounded to 16 bits, then
// (y0, y1) -> (y0 cos - y1 sin, y1 cos + y0 sin).
//
// A lane owns four pairs - values 4s .. 4s + 3 of both halves of a row, 8-byte loads -, D / 8 lanes a row, a wavefront 512 / D
// rows at a time.  All rows of a wavefront belong to one token, whose position, page and angles are looked up once and serve R
// rounds of rows: prompts, whose rows outnumber the resident wavefronts, take four rounds (the loads of all of them are
// requested together), single tokens one, which is the most wavefronts for the least latency.  A block of an MXFP4 row is the
// values of eight neighbouring lanes.
//
// Prompts are bound by the bytes moved: 2 x 2041 tokens of 64 q and 8 kv heads, D = 128, into MXFP4 in 37 us (157 MB, 4.2 TB/s;
// a large copy reaches 4.9); single tokens by launch and latency: 32 of them in 4.7 us, a smallest launch takes 4.4.
#include "fdk_mxfp4.h"

namespace fdk {

namespace {

enum CacheKind { KV_16BIT = 0, KV_FP8 = 1, KV_MX4 = 2 };

template <int QDT> struct Elem16;
template <> struct Elem16<FDK_BF16> {
    using T = __bf16;
};
template <> struct Elem16<FDK_FP16> {
    using T = _Float16;
};

__device__ __forceinline__ uint32_t to_e4m3(float x) {
    x = __builtin_fminf(__builtin_fmaxf(x, -448.0f), 448.0f);      // NaN stays NaN
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false) & 0xFFu;
}

// the largest of eight neighbouring lanes
__device__ __forceinline__ float max_of_eight(float x) {
    x = fmaxf(x, dpp_mov<0xB1>(x));
    x = fmaxf(x, dpp_mov<0x4E>(x));
    return fmaxf(x, dpp_mov<0x141>(x));
}

template <int QDT, int KV, int D, int R>
__global__ __launch_bounds__(256) void kv_append_axes_kernel(const KvAppendParams p, const KvAppendAxes m) {
    using T = typename Elem16<QDT>::T;
    using P2 = Pack2<QDT>;
    constexpr int HALF = D / 2;
    constexpr int LPR = D / 8;                  // lanes per row
    constexpr int RPW = 64 / LPR;               // rows of a wavefront and round
    const int lane = threadIdx.x & 63;
    const int sub = lane % LPR, slot_of_wave = lane / LPR;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads = p.hq + 2 * p.hkv;
    const int groups = (heads + RPW * R - 1) / (RPW * R);
    const int64_t w = (int64_t)blockIdx.x * 4 + wave;
    const int64_t token = w / groups;
    if (token >= (int64_t)p.batch * p.new_tokens) return;
    const int head0 = (int)(w - token * groups) * (RPW * R) + slot_of_wave;
    const int b = (int)(token / p.new_tokens), t = (int)(token - (int64_t)b * p.new_tokens);

    // four 16-bit values from `x`: one load where everything is aligned for it
    auto load4 = [&](const uint16_t* x) {
        if (m.aligned) return *reinterpret_cast<const uint2*>(x);
        return make_uint2(x[0] | ((uint32_t)x[1] << 16), x[2] | ((uint32_t)x[3] << 16));
    };
    auto store4 = [&](uint16_t* x, uint2 v) {
        if (m.aligned) {
            *reinterpret_cast<uint2*>(x) = v;
        } else {
            x[0] = (uint16_t)v.x; x[1] = (uint16_t)(v.x >> 16); x[2] = (uint16_t)v.y; x[3] = (uint16_t)(v.y >> 16);
        }
    };
    uint2 in0[R], in1[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int h = min(head0 + r * RPW, heads - 1);
        const uint16_t* x = reinterpret_cast<const uint16_t*>(p.qkv) + b * p.qkv_sb + t * p.qkv_st + h * p.qkv_sh + 4 * sub;
        in0[r] = load4(x);
        in1[r] = load4(x + HALF);
    }
    // the token's place in the cache, and its angles
    const int at = p.kv_lens[b] - p.new_tokens + t;
    bool writable = at >= 0 && at < (int64_t)p.max_pages * p.page_size;
    int64_t page = 0;
    int in_page = 0;
    if (writable) {
        page = p.block_table[b * p.tbl_sb + at / p.page_size];
        in_page = at % p.page_size;
        writable = page >= 0 && page < p.num_pages;
    }
    int pos[4] = {at, at, at, at};
    if (m.positions) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (x < m.num_axes) pos[x] = m.positions[x * m.pos_sa + b * m.pos_sb + t * m.pos_st];
    }
    float c[4], s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i = 4 * sub + j;
        int axis = (i >= m.section_end[0] ? 1 : 0) + (i >= m.section_end[1] ? 1 : 0) + (i >= m.section_end[2] ? 1 : 0);
        if (m.interleaved) {
            axis = i % m.num_axes;
            const int first = axis == 0 ? 0 : m.section_end[axis - 1];
            if (i / m.num_axes >= m.section_end[axis] - first) axis = 0;
        }
        const int x = axis == 0 ? pos[0] : axis == 1 ? pos[1] : axis == 2 ? pos[2] : pos[3];
        const int64_t row = b * p.cs_sb + (int64_t)min(max(x, 0), p.max_positions - 1) * p.cs_sp + i;
        c[j] = p.cos[row];
        s[j] = p.sin[row];
    }

#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int h = head0 + r * RPW;
        if (h >= heads) break;                                        // (whole rows of lanes; nothing below crosses rows)
        const bool is_q = h < p.hq, is_k = !is_q && h < p.hq + p.hkv;
        uint2 out0 = in0[r], out1 = in1[r];
        if (is_q || is_k) {
            const float x0[4] = {P2::lo(in0[r].x), P2::hi(in0[r].x), P2::lo(in0[r].y), P2::hi(in0[r].y)};
            const float x1[4] = {P2::lo(in1[r].x), P2::hi(in1[r].x), P2::lo(in1[r].y), P2::hi(in1[r].y)};
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) ss += x0[j] * x0[j] + x1[j] * x1[j];
            ss = group_sum<(LPR < 16 ? LPR : 16)>(ss);
            if constexpr (LPR == 32) ss += __shfl_xor(ss, 16, 64);
            const float rms = 1.0f / sqrtf(ss / (float)D + (is_q ? p.q_eps : p.k_eps));
            const T* wt = reinterpret_cast<const T*>(is_q ? p.q_weight : p.k_weight) + 4 * sub;
            float o0[4], o1[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // halves rounded to the 16-bit dtype before the rotation, as the reference does (norm.py:168-171)
                const float y0 = (float)(T)((float)wt[j] * (x0[j] * rms));
                const float y1 = (float)(T)((float)wt[j + HALF] * (x1[j] * rms));
                o0[j] = y0 * c[j] - y1 * s[j];
                o1[j] = y1 * c[j] + y0 * s[j];
            }
            out0 = make_uint2(P2::pack(o0[0], o0[1]), P2::pack(o0[2], o0[3]));
            out1 = make_uint2(P2::pack(o1[0], o1[1]), P2::pack(o1[2], o1[3]));
        }
        if (is_q) {
            uint16_t* q = reinterpret_cast<uint16_t*>(p.q_out) + b * p.qo_sb + t * p.qo_st + h * p.qo_sh + 4 * sub;
            store4(q, out0);
            store4(q + HALF, out1);
            continue;
        }
        if (!writable) continue;
        const int kvh = h - p.hq - (is_k ? 0 : p.hkv);
        const int64_t row = is_k ? page * p.k_sp + in_page * p.k_st + kvh * p.k_sh : page * p.v_sp + in_page * p.v_st + kvh * p.v_sh;
        char* const pool = reinterpret_cast<char*>(is_k ? p.k_cache : p.v_cache);
        if constexpr (KV == KV_16BIT) {
            uint16_t* x = reinterpret_cast<uint16_t*>(pool) + row + 4 * sub;
            store4(x, out0);
            store4(x + HALF, out1);
            continue;
        }
        // one- and half-byte rows: from the 16-bit values that a 16-bit cache would have received
        const float v[8] = {P2::lo(out0.x), P2::hi(out0.x), P2::lo(out0.y), P2::hi(out0.y),
                            P2::lo(out1.x), P2::hi(out1.x), P2::lo(out1.y), P2::hi(out1.y)};
        if constexpr (KV == KV_FP8) {
            const float scale = is_k ? p.k_scale[kvh] : p.v_scale[kvh];
            uint8_t* x = reinterpret_cast<uint8_t*>(pool) + row + 4 * sub;
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                uint32_t bytes = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) bytes |= to_e4m3(v[4 * hf + j] / scale) << (8 * j);
                uint8_t* to = x + hf * HALF;
                if (m.aligned) {
                    *reinterpret_cast<uint32_t*>(to) = bytes;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) to[j] = (uint8_t)(bytes >> (8 * j));
                }
            }
        }
        if constexpr (KV == KV_MX4) {
            char* const x = pool + row + 2 * sub;
            uint8_t* const sc = const_cast<uint8_t*>(is_k ? m.scales.k + page * m.scales.k_sp + in_page * m.scales.k_st + kvh * m.scales.k_sh
                                                          : m.scales.v + page * m.scales.v_sp + in_page * m.scales.v_st + kvh * m.scales.v_sh);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const float* y = v + 4 * hf;
                float amax = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
                if (y[0] != y[0] || y[1] != y[1] || y[2] != y[2] || y[3] != y[3]) amax = INFINITY;     // (fmaxf passes over a NaN)
                const uint32_t byte = mx_scale_byte(max_of_eight(amax), mx_max_exp<QDT>());
                const float scale = mx_scale(byte);
                uint32_t codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], scale, 0);
                codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[2], y[3], scale, 1);
                *reinterpret_cast<uint16_t*>(x + hf * (HALF / 2)) = (uint16_t)codes;
                if (sub % 8 == 0) sc[hf * (HALF / kMxBlock) + sub / 8] = (uint8_t)byte;
            }
        }
    }
}

template <int QDT, int KV, int D>
int launch_rows(const KvAppendParams& p, const KvAppendAxes& m, hipStream_t stream) {
    constexpr int RPW = 512 / D;
    const int64_t tokens = (int64_t)p.batch * p.new_tokens, heads = p.hq + 2 * p.hkv;
    constexpr int64_t kResidentWaves = 256 * 32;
    const bool one_round = tokens * ((heads + RPW - 1) / RPW) <= kResidentWaves;
    const int64_t waves = tokens * ((heads + RPW * (one_round ? 1 : 4) - 1) / (RPW * (one_round ? 1 : 4)));
    const dim3 grid((unsigned)((waves + 3) / 4)), block(256);
    if (one_round) hipLaunchKernelGGL((kv_append_axes_kernel<QDT, KV, D, 1>), grid, block, 0, stream, p, m);
    else hipLaunchKernelGGL((kv_append_axes_kernel<QDT, KV, D, 4>), grid, block, 0, stream, p, m);
    return (int)hipGetLastError();
}

template <int QDT, int KV>
int launch_kind(const KvAppendParams& p, const KvAppendAxes& m, hipStream_t stream) {
    switch (p.head_dim) {
        case 64: return launch_rows<QDT, KV, 64>(p, m, stream);
        case 128: return launch_rows<QDT, KV, 128>(p, m, stream);
        case 256: return launch_rows<QDT, KV, 256>(p, m, stream);
        default: return (int)hipErrorInvalidValue;
    }
}

}  // namespace

int launch_kv_append_axes(const KvAppendParams& p, const KvAppendAxes& m, int qkv_dtype, int kv_dtype, hipStream_t stream) {
    if ((int64_t)p.batch * p.new_tokens * (p.hq + 2 * p.hkv) == 0) return 0;
    const bool bf16 = qkv_dtype == FDK_BF16;
    if (kv_dtype == FDK_MXFP4) return bf16 ? launch_kind<FDK_BF16, KV_MX4>(p, m, stream) : launch_kind<FDK_FP16, KV_MX4>(p, m, stream);
    if (kv_dtype == FDK_FP8_E4M3) return bf16 ? launch_kind<FDK_BF16, KV_FP8>(p, m, stream) : launch_kind<FDK_FP16, KV_FP8>(p, m, stream);
    return bf16 ? launch_kind<FDK_BF16, KV_16BIT>(p, m, stream) : launch_kind<FDK_FP16, KV_16BIT>(p, m, stream);
}

}  // namespace fdk
