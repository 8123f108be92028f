// MXFP4 rows of a paged cache on gfx950: the OCP microscaling format with 4-bit elements.
//
// A row of D values is D / 2 bytes of e2m1 codes (value 2i in the low four bits of byte i) and, in a pool of its own,
// D / 32 e8m0 bytes, one per block of 32 consecutive values:  value = code * 2^(byte - 127), byte 255: NaN.  Both
// conversions are instructions of gfx950 that take the block's power of two as an exponent operand: two values per
// instruction, exact on the way to bf16 / fp16 (three significant bits), rounded to nearest even and saturating at 6 on
// the way back (checked against the format's definition over all 256 bytes x 256 scales, and over all 65536 bf16 values x
// 252 scales).
#pragma once

#include "fdk_device.h"

namespace fdk {

constexpr int kMxBlock = 32;               // values that share a scale

// Where the scale bytes of an MXFP4 cache are: [num_pages, P, Hkv, D / 32], byte strides of the page, token and head axes.
struct Mx4Scales {
    const uint8_t* k;
    const uint8_t* v;
    int64_t k_sp, k_st, k_sh;
    int64_t v_sp, v_st, v_sh;
};

// Explicit positions of an append (several axes: each turns its own section of the rotary pairs) and the scales of an MXFP4
// cache, beside KvAppendParams.
struct KvAppendAxes {
    const int32_t* positions;                // [axes, B, T]; null: every pair turns by the token's place in the cache
    int64_t pos_sa, pos_sb, pos_st;
    int32_t num_axes, interleaved;
    int32_t section_end[4];                  // pairs of axes 0 .. x together (INT32_MAX from the last axis on)
    int32_t aligned;                         // rows may be read and written four values at a time
    Mx4Scales scales;
};

// Launchers; return hipError_t as int.
int launch_kv_append_axes(const KvAppendParams& p, const KvAppendAxes& m, int qkv_dtype, int kv_dtype, hipStream_t stream);
int launch_splitkv_mx4(const SplitParams& p, const Mx4Scales& x, int q_dtype, hipStream_t stream);
int launch_mxfp4(const fdk_mxfp4_args& a, bool quantize, hipStream_t stream);

#if defined(__HIPCC__)

// the scale byte as the float whose exponent the conversion instructions use (byte 0 stands for 2^-127: its exponent field
// is 0, which the instructions read as just that; byte 255 makes every value a NaN)
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// byte `BYTE` of eight e2m1 codes -> two 16-bit values
template <int QDT, int BYTE>
__device__ __forceinline__ uint32_t mx_unpack2(uint32_t codes, float scale) {
    if constexpr (QDT == FDK_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, BYTE));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, BYTE));
}

// The scale byte of a block from the largest magnitude in it: the smallest power of two with amax <= 7 scales, within
// [2^-126, 2^max_exp].  Values in (6, 7] scales round down to 6, the largest code, and lose no more than values between
// two codes do; with the bound at 6 half of the blocks would be given twice the scale instead (mean square error of
// Gaussian blocks: 0.0125 against 0.0133 of the variance; at 8, the format's floor(log2 amax) rule, 0.0132).
// max_exp (125 for bf16, 13 for fp16) keeps 6 scales finite in the 16-bit type the cache is decoded in.
// A block that holds an infinity or a NaN gets byte 255.
__device__ __forceinline__ uint32_t mx_scale_byte(float amax, int max_exp) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, amax);        // (amax >= 0; subnormal: exponent field 0)
    if (bits >= 0x7f800000u) return 255u;
    const int e = (int)(bits >> 23) - 127 - 2 + ((bits & 0x007fffffu) > 0x00600000u ? 1 : 0);
    return (uint32_t)(min(max(e, -126), max_exp) + 127);
}
template <int QDT> __device__ __forceinline__ constexpr int mx_max_exp() { return QDT == FDK_BF16 ? 125 : 13; }

#endif  // __HIPCC__

}  // namespace fdk
