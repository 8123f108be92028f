// Eviction from a paged KV cache by accumulated attention weight.  gfx950.
//
// Of a sequence's n tokens the last `recent` stay, and of the rest those with the largest weights, up to `keep` in all; the
// survivors move to the front in their order, for every kv head on its own.  Two steps:
//
//   select   one workgroup per (sequence, kv head).  The weight that the last survivor has is found by three counting passes
//            over the weights' bits, most significant first; ties go to the lowest slot.  Every wavefront then owns a
//            contiguous range: it counts, and with the other wavefronts' counts writes its survivors to their places.
//   move     row j of the result is row kept[j] >= j of the cache.  Rows [first, outside) come from inside the first `keep`
//            slots: they are moved in ascending chunks, a chunk read whole before it is written (a later chunk reads only
//            slots behind this one's).  Rows [outside, keep) come from behind them and are never overwritten: any order will
//            do, once the first part is done.  The columns of a row do not depend on each other: a workgroup takes a slice of
//            128 bytes of the rows, so that few sequences still fill the GPU.
#include "fdk_kv_evict.h"

namespace fdk {

namespace {

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kBins = 2048;

// weights as integers of the same order: -0 as +0, NaN above everything
__device__ __forceinline__ uint32_t order_key(float w) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
    if (w != w) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const EvictParams p) {
    __shared__ int hist[kBins];
    __shared__ int wave_sum_[kSelectWaves], wave_eq[kSelectWaves], wave_gt[kSelectWaves];
    __shared__ int s_bin, s_above, s_first, s_inside;
    const int h = blockIdx.x, b = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* w = p.weights + b * p.w_sb + h * p.w_sh;
    float* wo = p.weights_out + b * p.wo_sb + h * p.wo_sh;
    int32_t* kept = p.kept + ((int64_t)b * p.hkv + h) * p.keep;
    const int n = max(min(p.kv_lens[b], p.max_tokens), 0);
    const int new_len = min(n, p.keep);
    int first = n, outside = n;                            // n <= keep: everything stays where it is
    if (n <= p.keep) {
        for (int j = tid; j < p.keep; j += kSelectThreads) kept[j] = j < n ? j : -1;
    } else {
        const int old = n - p.recent, need = p.keep - p.recent;      // need < old
        uint32_t bits = 0, mask = 0;
        int remaining = need;
        if (need > 0) {
            for (int pass = 0; pass < 3; ++pass) {
                const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
                const int bins = pass == 2 ? 1024 : 2048;
                for (int i = tid; i < kBins; i += kSelectThreads) hist[i] = 0;
                __syncthreads();
                for (int i = tid; i < old; i += kSelectThreads) {
                    const uint32_t key = order_key(w[i]);
                    if ((key & mask) == bits) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1);
                }
                __syncthreads();
                // the bin that holds the remaining-th largest: thread t has the bins 2t and 2t + 1 from the top
                const int top = bins - 1 - 2 * tid;
                const int c0 = top >= 0 ? hist[top] : 0, c1 = top >= 1 ? hist[top - 1] : 0;
                const int incl = wave_scan_i32(c0 + c1);
                if (lane == 63) wave_sum_[wave] = incl;
                __syncthreads();
                int above = incl - c0 - c1;
                for (int i = 0; i < wave; ++i) above += wave_sum_[i];
                if (above < remaining && remaining <= above + c0) {
                    s_bin = top;
                    s_above = above;
                } else if (above + c0 < remaining && remaining <= above + c0 + c1) {
                    s_bin = top - 1;
                    s_above = above + c0;
                }
                __syncthreads();
                bits |= (uint32_t)s_bin << shift;
                mask |= (uint32_t)(bins - 1) << shift;
                remaining -= s_above;
            }
        }
        // survivors: keys above `bits`, and the first `remaining` of those equal to it
        const int range = ((old + kSelectWaves - 1) / kSelectWaves + 63) / 64 * 64;
        const int64_t from64 = (int64_t)wave * range;
        const int from = (int)min(from64, (int64_t)old), to = (int)min(from64 + range, (int64_t)old);
        int gt = 0, eq = 0;
        if (need > 0) {
            for (int i = from + lane; __builtin_amdgcn_ballot_w64(i < to) != 0; i += 64) {
                const uint32_t key = i < to ? order_key(w[i]) : 0;
                gt += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < to && key > bits));
                eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < to && key == bits));
            }
        }
        if (lane == 0) {
            wave_gt[wave] = gt;
            wave_eq[wave] = eq;
        }
        if (tid == 0) {
            s_first = old;
            s_inside = 0;
        }
        __syncthreads();
        int at = 0, quota = remaining;                     // survivors before this wavefront's, equal ones left to take
        for (int i = 0; i < wave; ++i) {
            const int e = min(wave_eq[i], quota);
            at += wave_gt[i] + e;
            quota -= e;
        }
        int hole = old, inside = 0;                        // first slot that does not stay; survivors in the first `keep` slots
        for (int i = from + lane; __builtin_amdgcn_ballot_w64(i < to) != 0; i += 64) {
            const uint32_t key = i < to ? order_key(w[i]) : 0;
            const uint64_t is_eq = need > 0 ? __builtin_amdgcn_ballot_w64(i < to && key == bits) : 0;
            const uint64_t below = (1ull << lane) - 1;
            const bool stays = need > 0 && i < to && (key > bits || (key == bits && __builtin_popcountll(is_eq & below) < quota));
            const uint64_t sel = __builtin_amdgcn_ballot_w64(stays);
            if (stays) kept[at + __builtin_popcountll(sel & below)] = i;
            at += __builtin_popcountll(sel);
            quota -= min(quota, __builtin_popcountll(is_eq));
            inside += __builtin_popcountll(__builtin_amdgcn_ballot_w64(stays && i < p.keep));
            const uint64_t gone = __builtin_amdgcn_ballot_w64(i < to && !stays);
            if (gone && hole == old) hole = i - lane + __builtin_ctzll(gone);
        }
        if (lane == 0) {
            atomicMin(&s_first, hole);
            atomicAdd(&s_inside, inside);
        }
        for (int i = tid; i < p.recent; i += kSelectThreads) kept[need + i] = old + i;
        __syncthreads();
        first = s_first;
        outside = s_inside + max(min(p.keep, n) - old, 0);           // (the recent ones among the first `keep` slots)
    }
    __syncthreads();                                       // kept is whole
    if (tid == 0) *reinterpret_cast<int4*>(p.plan + ((int64_t)b * p.hkv + h) * 4) = make_int4(first, outside, new_len, 0);
    // the weights move as the rows do; a chunk is read before it is written, so weights_out may be weights
    for (int j0 = 0; j0 < new_len; j0 += kSelectThreads) {
        const int j = j0 + tid;
        const float x = j < new_len ? w[kept[j]] : 0.f;
        __syncthreads();
        if (j < new_len) wo[j] = x;
    }
    __syncthreads();
    for (int j = new_len + tid; j < p.weights_len; j += kSelectThreads) wo[j] = 0.f;      // behind them: tokens to come
}

struct MoveParams {
    EvictParams e;
    int32_t lanes[4], slices[4], slice0[4];  // lanes per row of a slice, slices of each tensor, the first one's index
    int32_t serial, parallel, parts;         // which rows this launch moves; workgroups per slice for the parallel ones
};

template <typename V>
__device__ __forceinline__ void move_rows(const MoveParams& m, const EvictRows& r, const int lanes, const int slice, const int b,
                                          const int h, const int part) {
    constexpr int U = 8;                                   // rows of a thread that are under way together
    const EvictParams& p = m.e;
    const int32_t* kept = p.kept + ((int64_t)b * p.hkv + h) * p.keep;
    const int4 plan = *reinterpret_cast<const int4*>(p.plan + ((int64_t)b * p.hkv + h) * 4);
    const int32_t* tbl = p.block_table + b * p.tbl_sb;
    char* base = r.pool + h * r.sh + ((int64_t)slice * lanes + threadIdx.x % lanes) * (int64_t)sizeof(V);
    const int row = threadIdx.x / lanes, rows = 256 / lanes;
    auto at = [&](int n) {
        const int64_t page = tbl[p.page_shift < 0 ? n / p.page_size : n >> p.page_shift];
        const int64_t slot = p.page_shift < 0 ? n % p.page_size : (n & (p.page_size - 1));
        return reinterpret_cast<V*>(base + page * r.sp + slot * r.st);
    };
    const int chunk = rows * U;
    if (m.serial) {
        for (int j0 = plan.x; j0 < plan.y; j0 += chunk) {
            V x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + u * rows + row;
                if (j < plan.y) x[u] = *at(kept[j]);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + u * rows + row;
                if (j < plan.y) *at(j) = x[u];
            }
        }
        if (m.parallel) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
    }
    if (m.parallel) {
        for (int j0 = plan.y + part * chunk; j0 < plan.z; j0 += m.parts * chunk) {
            V x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + u * rows + row;
                if (j < plan.z) x[u] = *at(kept[j]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + u * rows + row;
                if (j < plan.z) *at(j) = x[u];
            }
        }
    }
}

__global__ __launch_bounds__(256) void evict_move_kernel(const MoveParams m) {
    const int part = blockIdx.x % m.parts, slice = blockIdx.x / m.parts;
    const int h = blockIdx.y, b = blockIdx.z;
    // (written here, by the last launch, so that kv_lens_out may be kv_lens)
    if (m.parallel && blockIdx.x == 0 && h == 0 && threadIdx.x == 0)
        m.e.kv_lens_out[b] = m.e.plan[(int64_t)b * m.e.hkv * 4 + 2];
    int t = 0;
    while (t + 1 < m.e.num_tensors && slice >= m.slice0[t + 1]) ++t;
    if (m.e.rows[t].bytes == 16) move_rows<uint4>(m, m.e.rows[t], m.lanes[t], slice - m.slice0[t], b, h, part);
    else move_rows<uint8_t>(m, m.e.rows[t], m.lanes[t], slice - m.slice0[t], b, h, part);
}

}  // namespace

int launch_kv_evict(const EvictParams& p, int num_cus, hipStream_t stream) {
    hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)p.hkv, (unsigned)p.batch), dim3(kSelectThreads), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    MoveParams m;
    m.e = p;
    int slices = 0;
    for (int t = 0; t < p.num_tensors; ++t) {
        int lanes = 8;
        while (p.rows[t].cols % lanes) lanes >>= 1;
        m.lanes[t] = lanes;
        m.slices[t] = p.rows[t].cols / lanes;
        m.slice0[t] = slices;
        slices += m.slices[t];
    }
    for (int t = p.num_tensors; t < 4; ++t) m.lanes[t] = m.slices[t] = m.slice0[t] = 0;
    // Enough slices for four workgroups per compute unit: one launch, each workgroup first the rows that depend on each other,
    // then the rest.  Fewer: the rest gets a launch with more workgroups to a slice.
    const int64_t wgs = (int64_t)slices * p.hkv * p.batch;
    const bool one = wgs >= 4 * (int64_t)num_cus;
    m.serial = 1;
    m.parallel = one ? 1 : 0;
    m.parts = 1;
    hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)slices, (unsigned)p.hkv, (unsigned)p.batch), dim3(256), 0, stream, m);
    e = hipGetLastError();
    if (e != hipSuccess || one) return (int)e;
    m.serial = 0;
    m.parallel = 1;
    m.parts = (int32_t)((4 * (int64_t)num_cus + wgs - 1) / wgs);
    hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)(slices * m.parts), (unsigned)p.hkv, (unsigned)p.batch), dim3(256), 0, stream, m);
    return (int)hipGetLastError();
}

}  // namespace fdk
