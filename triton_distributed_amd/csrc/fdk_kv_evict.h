// Bounding a paged KV cache: attention weights accumulated per cached token, and the eviction of the tokens with the least of
// it.  Kernel arguments and launchers (fdk_attn_weights.hip, fdk_kv_evict.hip).
#pragma once

#include "fdk_device.h"
#include "fdk_mxfp4.h"

namespace fdk {

struct AttnWeightsParams {
    const void* q;
    const void* k;
    const uint8_t* k_block_scale;            // MXFP4 caches
    const float* k_scale;                    // fp8 caches: [Hkv] or null
    const int32_t* block_table;
    const int32_t* kv_lens;
    const float* lse;
    float* weights;
    int64_t q_sb, q_sh;
    int64_t k_sp, k_st, k_sh;                // bytes
    int64_t bs_sp, bs_st, bs_sh;             // bytes
    int64_t tbl_sb, lse_sb;
    int64_t w_sb, w_sh;
    int32_t batch, hkv, group;
    int32_t page_size, page_shift;           // page_shift = log2(page_size) or -1
    int32_t max_tokens;                      // min(table capacity, weights_len)
    int32_t shares, heads_per_wg;            // workgroups per (sequence, block of kv heads); heads of a block
    int32_t balanced;                        // workgroups go to the sequences by their lengths: shares is the average
    float scale_log2, sm_scale, soft_cap;
};

// rows of one tensor of the cache: `cols` pieces of 16 bytes (or single bytes: the block scales); none where another tensor's
// rows hold them
struct EvictRows {
    char* pool;
    int64_t sp, st, sh;                      // byte strides of the page, token and head axes
    int32_t cols, bytes;                     // bytes: 16 or 1 per piece
};

struct EvictParams {
    EvictRows rows[4];
    const int32_t* block_table;
    const int32_t* kv_lens;
    const float* weights;
    float* weights_out;
    int32_t* kept;                           // [B, Hkv, keep]
    int32_t* plan;                           // [B, Hkv, 4]: first row that moves, first row from outside, new length, unused
    int32_t* kv_lens_out;
    int64_t tbl_sb, w_sb, w_sh, wo_sb, wo_sh;
    int32_t batch, hkv, keep, recent;
    int32_t weights_len, max_tokens;
    int32_t page_size, page_shift;
    int32_t num_tensors, num_pages;
    // rows whose weights are spread over several workgroups (parts of the workspace)
    int32_t segments;
    int2* row_state;                         // [rows][2]: leading bits of the last survivor's weight, survivors left to find
    int32_t* seg_gt;                         // [rows][segments]: weights known to be above them
    uint16_t* seg_hist;                      // [3][rows][segments][2048]
    float* stash;                            // [rows][keep]: the survivors' weights
};

int launch_attn_weights(const AttnWeightsParams& p, int head_dim, int q_dtype, int kv_dtype, int num_cus, hipStream_t stream);
int evict_segments(int batch, int hkv, int max_tokens, int num_cus);
size_t evict_workspace_bytes(int batch, int hkv, int max_tokens, int keep, int num_cus);
int launch_kv_evict(const EvictParams& p, int num_cus, hipStream_t stream);

}  // namespace fdk
