// MXFP4 rows: dispatch of the decode kernels over the head dimension, and the conversion between 16-bit rows and MXFP4 rows.
#include "fdk_mxfp4.h"

namespace fdk {

#define FDK_DECLARE_MX4(D) int launch_splitkv_mx4_d##D(const SplitParams& p, const Mx4Scales& x, int q_dtype, hipStream_t stream);
FDK_DECLARE_MX4(64)
FDK_DECLARE_MX4(128)
FDK_DECLARE_MX4(256)
#undef FDK_DECLARE_MX4
int launch_splitkv_mx4_staged(const SplitParams& p, const Mx4Scales& x, int q_dtype, hipStream_t stream);

int launch_splitkv_mx4(const SplitParams& p, const Mx4Scales& x, int q_dtype, hipStream_t stream) {
    // pairs of 64-byte rows (one line), pages of 16 << n tokens: through LDS
    if (p.head_dim == 128 && p.hg_per_wg == 2 && p.page_shift >= 4) return launch_splitkv_mx4_staged(p, x, q_dtype, stream);
    switch (p.head_dim) {
        case 64: return launch_splitkv_mx4_d64(p, x, q_dtype, stream);
        case 128: return launch_splitkv_mx4_d128(p, x, q_dtype, stream);
        case 256: return launch_splitkv_mx4_d256(p, x, q_dtype, stream);
        default: return (int)hipErrorInvalidValue;
    }
}

namespace {

// A thread converts eight values: 16 bytes of x, four bytes of codes; the four threads of a block share its maximum.  The
// grid covers rows x (values / 8) such pieces.  Bound by the bytes moved: 131072 x 8 rows of 128
// (340 MB) in 85 us to MXFP4 (4.0 TB/s), in 76 us back (4.5).
template <int QDT, bool QUANTIZE>
__global__ __launch_bounds__(256) void mxfp4_kernel(const fdk_mxfp4_args a) {
    const int per_row = a.num_values >> 3;                           // a multiple of four
    const uint64_t first = (uint64_t)blockIdx.x * 256;
    const uint32_t in = (uint32_t)(first % (uint32_t)per_row) + threadIdx.x;
    const uint64_t row = first / (uint32_t)per_row + in / (uint32_t)per_row;
    const uint32_t piece = in % (uint32_t)per_row;
    // (whole blocks of four threads are inside or outside)
    if (row >= (uint64_t)a.n[0] * a.n[1] * a.n[2]) return;
    int64_t i0 = 0, i1 = 0, i2 = (int64_t)row;
    if (a.n[0] > 1 || a.n[1] > 1) {
        i2 = (int64_t)(row % (uint32_t)a.n[2]);
        const uint64_t up = row / (uint32_t)a.n[2];
        i1 = (int64_t)(up % (uint32_t)a.n[1]);
        i0 = (int64_t)(up / (uint32_t)a.n[1]);
    }
    uint16_t* x = reinterpret_cast<uint16_t*>(a.x) + i0 * a.x_stride[0] + i1 * a.x_stride[1] + i2 * a.x_stride[2] + 8 * piece;
    uint32_t* codes = reinterpret_cast<uint32_t*>(a.codes + i0 * a.codes_stride[0] + i1 * a.codes_stride[1] + i2 * a.codes_stride[2]) + piece;
    uint8_t* scale = a.scales + i0 * a.scales_stride[0] + i1 * a.scales_stride[1] + i2 * a.scales_stride[2] + (piece >> 2);
    if constexpr (QUANTIZE) {
        const uint4 w = *reinterpret_cast<const uint4*>(x);
        const uint32_t in2[4] = {w.x, w.y, w.z, w.w};
        float v[8], amax = 0.f;
        uint32_t nan = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = Pack2<QDT>::lo(in2[i]);
            v[2 * i + 1] = Pack2<QDT>::hi(in2[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            amax = fmaxf(amax, fabsf(v[i]));                          // (fmaxf passes over a NaN)
            nan |= v[i] != v[i];
        }
        if (nan) amax = INFINITY;
        amax = fmaxf(amax, dpp_mov<0xB1>(amax));
        amax = fmaxf(amax, dpp_mov<0x4E>(amax));
        const uint32_t byte = mx_scale_byte(amax, mx_max_exp<QDT>());
        const float sc = mx_scale(byte);
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], sc, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], sc, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], sc, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], sc, 3);
        *codes = c;
        if ((piece & 3) == 0) *scale = (uint8_t)byte;
    } else {
        const uint32_t c = *codes;
        const float sc = mx_scale(*scale);
        *reinterpret_cast<uint4*>(x) = make_uint4(mx_unpack2<QDT, 0>(c, sc), mx_unpack2<QDT, 1>(c, sc), mx_unpack2<QDT, 2>(c, sc),
                                                  mx_unpack2<QDT, 3>(c, sc));
    }
}

}  // namespace

int launch_mxfp4(const fdk_mxfp4_args& a, bool quantize, hipStream_t stream) {
    const uint64_t pieces = (uint64_t)a.n[0] * a.n[1] * a.n[2] * (uint64_t)(a.num_values / 8);
    const dim3 grid((unsigned)((pieces + 255) / 256)), block(256);
    const bool bf16 = a.x_dtype == FDK_BF16;
    if (quantize) {
        if (bf16) hipLaunchKernelGGL((mxfp4_kernel<FDK_BF16, true>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((mxfp4_kernel<FDK_FP16, true>), grid, block, 0, stream, a);
    } else {
        if (bf16) hipLaunchKernelGGL((mxfp4_kernel<FDK_BF16, false>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((mxfp4_kernel<FDK_FP16, false>), grid, block, 0, stream, a);
    }
    return (int)hipGetLastError();
}

}  // namespace fdk
