// Eviction from a paged KV cache by accumulated attention weight.  gfx950.
//
// Of a sequence's n tokens the last `recent` stay, and of the rest those with the largest weights, up to `keep` in all; the
// survivors move to the front in their order, for every kv head on its own.  Two steps:
//
//   select   one workgroup per (sequence, kv head), or several (evict_segment_kernel).  The weight that the last survivor has is found by three counting passes
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
constexpr int kMaxSegments = 64;

// weights as integers of the same order: -0 as +0, NaN above everything
__device__ __forceinline__ uint32_t order_key(float w) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
    if (w != w) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Add one per active lane to hist[bin]: the lanes that share the first active lane's bin add their number at once (sums of
// weights hold many equal values, zeros among them; a bin that all lanes hit one by one is 64 times slower).
__device__ __forceinline__ void count_bin(int* hist, int bin, bool active, int lane) {
    uint64_t rest = __builtin_amdgcn_ballot_w64(active);
    if (rest == 0) return;
    const int lead = __builtin_amdgcn_readlane(bin, __builtin_ctzll(rest));
    const uint64_t same = __builtin_amdgcn_ballot_w64(active && bin == lead);
    if (lane == __builtin_ctzll(rest)) atomicAdd(&hist[lead], __builtin_popcountll(same));
    if (active && bin != lead) atomicAdd(&hist[bin], 1);
}

// KPT > 0: a thread holds up to KPT weights in registers, the workgroup reads each of them once (rows of up to 1024 KPT
// tokens; one wavefront's are consecutive).  KPT = 0: any length, the weights are read again in each pass.
template <int KPT>
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const EvictParams p) {
    __shared__ int hist[kBins];
    __shared__ int wave_sum_[kSelectWaves], wave_eq[kSelectWaves], wave_gt[kSelectWaves];
    __shared__ int s_bin, s_above, s_first, s_inside;
    const int h = blockIdx.x, b = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float* w = p.weights + b * p.w_sb + h * p.w_sh;
    float* wo = p.weights_out + b * p.wo_sb + h * p.wo_sh;
    int32_t* kept = p.kept + ((int64_t)b * p.hkv + h) * p.keep;
    const int n = max(min(p.kv_lens[b], p.max_tokens), 0);
    const int new_len = min(n, p.keep);
    int first = n, outside = n;                            // n <= keep: everything stays where it is
    int copied = 0;                                        // weights of the result that are in place already
    if (n <= p.keep) {
        for (int j = tid; j < p.keep; j += kSelectThreads) kept[j] = j < n ? j : -1;
    } else {
        const int old = n - p.recent, need = p.keep - p.recent;      // need < old
        const int range = ((old + kSelectWaves - 1) / kSelectWaves + 63) / 64 * 64;
        const int64_t from64 = (int64_t)wave * range;
        const int from = (int)min(from64, (int64_t)old), to = (int)min(from64 + range, (int64_t)old);
        float mine[KPT > 0 ? KPT : 1];
        // every weight of this wavefront's range, 64 at a time: f(index, weight), inactive lanes with index >= to
        auto each = [&](auto&& f) {
            if constexpr (KPT > 0) {
#pragma unroll
                for (int r = 0; r < KPT; ++r) {
                    if (from + 64 * r >= to) break;
                    f(from + 64 * r + lane, mine[r]);
                }
            } else {
#pragma unroll 4
                for (int i = from + lane; __builtin_amdgcn_ballot_w64(i < to) != 0; i += 64) f(i, i < to ? w[i] : 0.f);
            }
        };
        if constexpr (KPT > 0) {
#pragma unroll
            for (int r = 0; r < KPT; ++r) {
                const int i = from + 64 * r + lane;
                mine[r] = i < to ? w[i] : 0.f;
            }
        }
        uint32_t bits = 0, mask = 0;
        int remaining = need;
        if (need > 0) {
            for (int pass = 0; pass < 3; ++pass) {
                const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
                const int bins = pass == 2 ? 1024 : 2048;
                for (int i = tid; i < kBins; i += kSelectThreads) hist[i] = 0;
                __syncthreads();
                each([&](int i, float x) {
                    const uint32_t key = order_key(x);
                    count_bin(hist, (int)((key >> shift) & (uint32_t)(bins - 1)), i < to && (key & mask) == bits, lane);
                });
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
        int gt = 0, eq = 0;
        if (need > 0) {
            each([&](int i, float x) {
                const uint32_t key = order_key(x);
                gt += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < to && key > bits));
                eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < to && key == bits));
            });
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
        const uint64_t below = (1ull << lane) - 1;
        each([&](int i, float x) {
            const uint32_t key = order_key(x);
            const uint64_t is_eq = need > 0 ? __builtin_amdgcn_ballot_w64(i < to && key == bits) : 0;
            const bool stays = need > 0 && i < to && (key > bits || (key == bits && __builtin_popcountll(is_eq & below) < quota));
            const uint64_t sel = __builtin_amdgcn_ballot_w64(stays);
            if (stays) {
                const int j = at + __builtin_popcountll(sel & below);
                kept[j] = i;
                if (KPT > 0) wo[j] = x;                    // (all weights of the range have been read: also where wo is w)
            }
            at += __builtin_popcountll(sel);
            quota -= min(quota, __builtin_popcountll(is_eq));
            inside += __builtin_popcountll(__builtin_amdgcn_ballot_w64(stays && i < p.keep));
            const uint64_t gone = __builtin_amdgcn_ballot_w64(i < to && !stays);
            if (gone && hole == old) hole = i - lane + __builtin_ctzll(gone);
        });
        if (lane == 0) {
            atomicMin(&s_first, hole);
            atomicAdd(&s_inside, inside);
        }
        for (int i = tid; i < p.recent; i += kSelectThreads) kept[need + i] = old + i;
        if (KPT > 0) copied = need;
        __syncthreads();
        first = s_first;
        outside = s_inside + max(min(p.keep, n) - old, 0);           // (the recent ones among the first `keep` slots)
    }
    __syncthreads();                                       // kept is whole
    if (tid == 0) *reinterpret_cast<int4*>(p.plan + ((int64_t)b * p.hkv + h) * 4) = make_int4(first, outside, new_len, 0);
    // the other weights move as the rows do; a chunk is read before it is written, so weights_out may be weights
    for (int j0 = copied; j0 < new_len; j0 += kSelectThreads) {
        const int j = j0 + tid;
        const float x = j < new_len ? w[kept[j]] : 0.f;
        __syncthreads();
        if (j < new_len) wo[j] = x;
    }
    __syncthreads();
    for (int j = new_len + tid; j < p.weights_len; j += kSelectThreads) wo[j] = 0.f;      // behind them: tokens to come
}

// ---- long rows and few of them: a row's weights over several workgroups ----
// The counting passes become launches: every workgroup (segment g of a row) writes the histogram of its own segment, plain
// stores of 16-bit counts (a segment has fewer than 65536 weights), and the next launch's workgroups all derive the same bin
// from the sum of the row's histograms.  The last launch knows from them how many survivors the earlier segments have, and
// writes its own to their places; the weights go through the workspace, since another segment may not have been read yet
// where weights_out is weights.

// counts of segment `seg` (of all rows' segments) at level 0, 1 or 2
__device__ __forceinline__ uint32_t* segment_hist(const EvictParams& p, int level, int64_t seg) {
    return reinterpret_cast<uint32_t*>(p.seg_hist) + (level * (int64_t)p.batch * p.hkv * p.segments + seg) * (kBins / 2);
}

struct Level {                                             // what a level's counts say, uniform over the workgroup
    int bin, above;                                        // the bin that holds the `remaining`-th largest; weights in higher bins
    int mine_above;                                        // ... of this workgroup's segment
};

// all threads of the workgroup; scratch: kSelectWaves + 3 ints
__device__ __forceinline__ Level read_level(const EvictParams& p, int level, int64_t seg0, int g, int remaining, int* scratch) {
    const int bins = level == 2 ? 1024 : kBins;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int word = bins / 2 - 1 - tid, top = 2 * word + 1;          // this thread's bins: top, top - 1
    int c0 = 0, c1 = 0, m0 = 0, m1 = 0;
    if (word >= 0) {
#pragma unroll 16
        for (int s = 0; s < p.segments; ++s) {
            const uint32_t x = segment_hist(p, level, seg0 + s)[word];
            c0 += (int)(x >> 16);
            c1 += (int)(x & 0xffffu);
            if (s == g) {
                m0 = (int)(x >> 16);
                m1 = (int)(x & 0xffffu);
            }
        }
    }
    const int incl = wave_scan_i32(c0 + c1);
    if (lane == 63) scratch[wave] = incl;
    if (tid == 0) scratch[kSelectWaves + 2] = 0;
    __syncthreads();
    int above = incl - c0 - c1;
    for (int i = 0; i < wave; ++i) above += scratch[i];
    if (above < remaining && remaining <= above + c0) {
        scratch[kSelectWaves] = top;
        scratch[kSelectWaves + 1] = above;
    } else if (above + c0 < remaining && remaining <= above + c0 + c1) {
        scratch[kSelectWaves] = top - 1;
        scratch[kSelectWaves + 1] = above + c0;
    }
    __syncthreads();
    Level l;
    l.bin = scratch[kSelectWaves];
    l.above = scratch[kSelectWaves + 1];
    const int part = wave_sum_i32((top > l.bin ? m0 : 0) + (top - 1 > l.bin ? m1 : 0));
    if (lane == 0) atomicAdd(&scratch[kSelectWaves + 2], part);
    __syncthreads();
    l.mine_above = scratch[kSelectWaves + 2];
    __syncthreads();
    return l;
}

// the weights of a wavefront's part of a segment, 64 at a time (see evict_select_kernel)
template <int KPT>
struct SegmentWeights {
    float mine[KPT > 0 ? KPT : 1];
    const float* w;
    int from, to, lane;
    __device__ __forceinline__ void load(const float* w_, int seg_from, int seg_to, int wave, int lane_) {
        w = w_;
        lane = lane_;
        const int len = seg_to - seg_from, range = ((len + kSelectWaves - 1) / kSelectWaves + 63) / 64 * 64;
        from = min(seg_from + wave * range, seg_to);
        to = min(from + range, seg_to);
        if constexpr (KPT > 0) {
#pragma unroll
            for (int r = 0; r < KPT; ++r) {
                const int i = from + 64 * r + lane;
                mine[r] = i < to ? w[i] : 0.f;
            }
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(F&& f) {
        if constexpr (KPT > 0) {
#pragma unroll
            for (int r = 0; r < KPT; ++r) {
                if (from + 64 * r >= to) break;
                f(from + 64 * r + lane, mine[r]);
            }
        } else {
#pragma unroll 4
            for (int i = from + lane; __builtin_amdgcn_ballot_w64(i < to) != 0; i += 64) f(i, i < to ? w[i] : 0.f);
        }
    }
};

// LEVEL 0, 1, 2: count; 3: write the survivors.
template <int KPT, int LEVEL>
__global__ __launch_bounds__(kSelectThreads) void evict_segment_kernel(const EvictParams p) {
    __shared__ int hist[kBins];
    __shared__ int scratch[kSelectWaves + 3];
    __shared__ int wave_eq[kSelectWaves], wave_gt[kSelectWaves], seg_gt[kMaxSegments], seg_eq[kMaxSegments];
    __shared__ int s_first, s_inside;
    const int g = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = (int64_t)b * p.hkv + h, seg0 = row * p.segments;
    const float* w = p.weights + b * p.w_sb + h * p.w_sh;
    int32_t* plan = p.plan + row * 4;
    const int n = max(min(p.kv_lens[b], p.max_tokens), 0);
    const int old = max(n - p.recent, 0), need = p.keep - p.recent;
    const int new_len = min(n, p.keep);
    if (LEVEL == 0 && g == 0 && tid == 0)
        *reinterpret_cast<int4*>(plan) = n <= p.keep ? make_int4(n, n, new_len, 0) : make_int4(old, max(p.keep - old, 0), new_len, 0);
    int32_t* kept = p.kept + row * p.keep;
    float* stash = p.stash + row * p.keep;
    if (n <= p.keep || need == 0) {
        if (LEVEL < 3) return;
        // everything stays where it is, or only the recent ones do
        for (int j = g * kSelectThreads + tid; j < p.keep; j += p.segments * kSelectThreads) {
            const int src = n <= p.keep ? (j < n ? j : -1) : old + j;
            kept[j] = src;
            if (src >= 0) stash[j] = w[src];
        }
        if (n > p.keep && g == 0 && tid == 0) plan[0] = 0;                 // (plan[1]: set at level 0)
        return;
    }
    const int per = ((old + p.segments - 1) / p.segments + 63) / 64 * 64;
    const int seg_from = (int)min((int64_t)g * per, (int64_t)old), seg_to = (int)min((int64_t)seg_from + per, (int64_t)old);
    SegmentWeights<KPT> mine;
    mine.load(w, seg_from, seg_to, wave, lane);
    uint32_t bits = 0, mask = 0;
    int remaining = need, mine_gt = 0;
    if constexpr (LEVEL >= 2) {                            // what the launch before found out about the levels before its own
        const int2 st = p.row_state[row * 2 + (LEVEL - 2)];
        bits = (uint32_t)st.x;
        remaining = st.y;
        mask = LEVEL == 2 ? 0x7ffu << 21 : 0xfffffc00u;
        mine_gt = p.seg_gt[seg0 + g];
    }
    if constexpr (LEVEL >= 1) {
        const int shift = LEVEL == 1 ? 21 : LEVEL == 2 ? 10 : 0;
        const Level l = read_level(p, LEVEL - 1, seg0, g, remaining, scratch);
        bits |= (uint32_t)l.bin << shift;
        mask |= (uint32_t)(LEVEL == 3 ? 1023 : 2047) << shift;
        remaining -= l.above;
        if constexpr (LEVEL < 3) {
            if (tid == 0) {
                p.seg_gt[seg0 + g] = mine_gt + l.mine_above;
                if (g == 0) p.row_state[row * 2 + (LEVEL - 1)] = make_int2((int)bits, remaining);
            }
        }
    }
    if constexpr (LEVEL < 3) {
        const int shift = LEVEL == 0 ? 21 : LEVEL == 1 ? 10 : 0, bins = LEVEL == 2 ? 1024 : kBins;
        for (int i = tid; i < kBins; i += kSelectThreads) hist[i] = 0;
        __syncthreads();
        mine.each([&](int i, float x) {
            const uint32_t key = order_key(x);
            count_bin(hist, (int)((key >> shift) & (uint32_t)(bins - 1)), i < mine.to && (key & mask) == bits, lane);
        });
        __syncthreads();
        if (tid < bins / 2) segment_hist(p, LEVEL, seg0 + g)[tid] = (uint32_t)hist[2 * tid] | ((uint32_t)hist[2 * tid + 1] << 16);
    } else {
        // survivors and equal weights of every segment of the row
        const int bin = (int)(bits & 1023u);
        for (int s = wave; s < p.segments; s += kSelectWaves) {
            int above = 0;
#pragma unroll
            for (int i = lane; i < 512; i += 64) {
                const uint32_t x = segment_hist(p, 2, seg0 + s)[i];
                above += (2 * i + 1 > bin ? (int)(x >> 16) : 0) + (2 * i > bin ? (int)(x & 0xffffu) : 0);
            }
            above = wave_sum_i32(above);
            if (lane == 0) {
                const uint32_t x = segment_hist(p, 2, seg0 + s)[bin >> 1];
                seg_gt[s] = p.seg_gt[seg0 + s] + above;
                seg_eq[s] = (int)(bin & 1 ? x >> 16 : x & 0xffffu);
            }
        }
        int gt = 0, eq = 0;
        mine.each([&](int i, float x) {
            const uint32_t key = order_key(x);
            gt += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < mine.to && key > bits));
            eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < mine.to && key == bits));
        });
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
        for (int s = 0; s < g; ++s) {
            const int e = min(seg_eq[s], quota);
            at += seg_gt[s] + e;
            quota -= e;
        }
        for (int i = 0; i < wave; ++i) {
            const int e = min(wave_eq[i], quota);
            at += wave_gt[i] + e;
            quota -= e;
        }
        int hole = old, inside = 0;
        const uint64_t below = (1ull << lane) - 1;
        mine.each([&](int i, float x) {
            const uint32_t key = order_key(x);
            const uint64_t is_eq = __builtin_amdgcn_ballot_w64(i < mine.to && key == bits);
            const bool stays = i < mine.to && (key > bits || (key == bits && __builtin_popcountll(is_eq & below) < quota));
            const uint64_t sel = __builtin_amdgcn_ballot_w64(stays);
            if (stays) {
                const int j = at + __builtin_popcountll(sel & below);
                kept[j] = i;
                stash[j] = x;
            }
            at += __builtin_popcountll(sel);
            quota -= min(quota, __builtin_popcountll(is_eq));
            inside += __builtin_popcountll(__builtin_amdgcn_ballot_w64(stays && i < p.keep));
            const uint64_t gone = __builtin_amdgcn_ballot_w64(i < mine.to && !stays);
            if (gone && hole == old) hole = i - lane + __builtin_ctzll(gone);
        });
        if (lane == 0) {
            atomicMin(&s_first, hole);
            atomicAdd(&s_inside, inside);
        }
        for (int i = g * kSelectThreads + tid; i < p.recent; i += p.segments * kSelectThreads) {
            kept[need + i] = old + i;
            stash[need + i] = w[old + i];
        }
        __syncthreads();
        if (tid == 0) {                                    // (whole numbers: the order of these does not matter)
            atomicMin(&plan[0], s_first);
            atomicAdd(&plan[1], s_inside);
        }
    }
}

struct MoveParams {
    EvictParams e;
    int32_t lanes[4], slices[4];             // lanes per row of a slice, slices of each tensor
    int32_t serial, parallel, parts;         // which rows this launch moves; workgroups per slice for the parallel ones
    int32_t row_blocks;                      // workgroups that move rows; behind them, of weights from the workspace
};

// rows are read once and written once: the non-temporal hint keeps them out of the caches' replacement order
__device__ __forceinline__ uint4 load_row(const uint4* p) { return load_stream16(p); }
__device__ __forceinline__ uint8_t load_row(const uint8_t* p) { return *p; }
__device__ __forceinline__ void store_row(uint4* p, uint4 v) {
    __builtin_nontemporal_store(u32x4_t{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4_t*>(p));
}
__device__ __forceinline__ void store_row(uint8_t* p, uint8_t v) { *p = v; }

template <int THREADS, typename V>
__device__ __forceinline__ void move_rows(const MoveParams& m, const EvictRows& r, const int lanes, const int slice, const int b,
                                          const int h, const int part) {
    constexpr int U = 8;                                   // rows of a thread that are under way together
    const EvictParams& p = m.e;
    const int32_t* kept = p.kept + ((int64_t)b * p.hkv + h) * p.keep;
    const int4 plan = *reinterpret_cast<const int4*>(p.plan + ((int64_t)b * p.hkv + h) * 4);
    const int32_t* tbl = p.block_table + b * p.tbl_sb;
    char* base = r.pool + h * r.sh + ((int64_t)slice * lanes + threadIdx.x % lanes) * (int64_t)sizeof(V);
    const int row = threadIdx.x / lanes, rows = THREADS / lanes;
    // Rows j0 + row, j0 + rows + row ... of a chunk, as far as they are below `end`.  In stages - slots, pages, rows - so that
    // each stage's loads are under way together; rows past the end repeat the last one and are not stored.
    const int chunk = rows * U;
    V x[U];
    char* to[U];
    auto place = [&](int n) { return p.page_shift < 0 ? n / p.page_size : n >> p.page_shift; };
    auto slot = [&](int n) { return (int64_t)(p.page_shift < 0 ? n % p.page_size : (n & (p.page_size - 1))); };
    auto read = [&](int j0, int end) {
        int src[U];
        int32_t pg[U], pg_to[U];
#pragma unroll
        for (int u = 0; u < U; ++u) src[u] = kept[min(j0 + u * rows + row, end - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u) pg_to[u] = tbl[place(min(j0 + u * rows + row, end - 1))];
#pragma unroll
        for (int u = 0; u < U; ++u) pg[u] = tbl[place(src[u])];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool inside = (uint32_t)pg[u] < (uint32_t)p.num_pages && (uint32_t)pg_to[u] < (uint32_t)p.num_pages;
            if (!inside) pg[u] = 0;
            if (!inside) pg_to[u] = -1;                    // (not stored)
            x[u] = load_row(reinterpret_cast<const V*>(base + pg[u] * r.sp + slot(src[u]) * r.st));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) to[u] = pg_to[u] < 0 ? nullptr : base + pg_to[u] * r.sp + slot(min(j0 + u * rows + row, end - 1)) * r.st;
    };
    auto write = [&](int j0, int end) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j0 + u * rows + row < end && to[u]) store_row(reinterpret_cast<V*>(to[u]), x[u]);
    };
    if (m.serial) {
        for (int j0 = plan.x; j0 < plan.y; j0 += chunk) {
            read(j0, plan.y);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            write(j0, plan.y);
        }
        if (m.parallel) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
    }
    if (m.parallel) {
        for (int j0 = plan.y + part * chunk; j0 < plan.z; j0 += m.parts * chunk) {
            read(j0, plan.z);
            write(j0, plan.z);
        }
    }
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void evict_move_kernel(const MoveParams m) {
    const int part = blockIdx.x % m.parts, slice = blockIdx.x / m.parts;
    const int h = blockIdx.y, b = blockIdx.z;
    if ((int)blockIdx.x >= m.row_blocks) {                // (rows of several segments) the survivors' weights
        const int64_t row = (int64_t)b * m.e.hkv + h;
        const int new_len = m.e.plan[row * 4 + 2], blocks = (int)gridDim.x - m.row_blocks;
        float* wo = m.e.weights_out + b * m.e.wo_sb + h * m.e.wo_sh;
        for (int j = ((int)blockIdx.x - m.row_blocks) * THREADS + (int)threadIdx.x; j < m.e.weights_len; j += blocks * THREADS)
            wo[j] = j < new_len ? m.e.stash[row * m.e.keep + j] : 0.f;
        return;
    }
    // (written here, by the last launch, so that kv_lens_out may be kv_lens)
    if (m.parallel && blockIdx.x == 0 && h == 0 && threadIdx.x == 0)
        m.e.kv_lens_out[b] = m.e.plan[(int64_t)b * m.e.hkv * 4 + 2];
    // (written out: an index into the arrays of the argument block would put them into scratch memory)
    if (slice < m.slices[0]) move_rows<THREADS, uint4>(m, m.e.rows[0], m.lanes[0], slice, b, h, part);
    else if (slice < m.slices[0] + m.slices[1]) move_rows<THREADS, uint4>(m, m.e.rows[1], m.lanes[1], slice - m.slices[0], b, h, part);
    else if (slice < m.slices[0] + m.slices[1] + m.slices[2])
        move_rows<THREADS, uint8_t>(m, m.e.rows[2], m.lanes[2], slice - m.slices[0] - m.slices[1], b, h, part);
    else move_rows<THREADS, uint8_t>(m, m.e.rows[3], m.lanes[3], slice - m.slices[0] - m.slices[1] - m.slices[2], b, h, part);
}

}  // namespace

// Segments of a row (of its capacity: the lengths are on the device): as many as give two workgroups to a compute unit, of about
// 4096 weights or more.  One workgroup does it in one launch instead of four, up to 16384 weights out of registers; more are for
// longer rows, and for few of them: whole calls in a graph, a quarter kept, in us, one workgroup to a row against several (rows of 256 bytes)
// 8 rows of 4097 / 8192 / 16384 tokens 25 / 28 / 42 against 32 / 32 / 42, 256 rows 72 / 134 / 257 against 113 / 195 / 385; (rows of
// 128 bytes) 8 rows of 16400 / 65536 tokens 49 / 140 against 39 / 67, 64 rows (eight segments) 78 / 258 against 79 / 190, 128 rows
// (four) 108 / 389 against 127 / 376, 256 rows (two) 177 / 653 against 229 / 890.
int evict_segments(int batch, int hkv, int max_tokens, int num_cus) {
    int64_t s = 2 * (int64_t)num_cus / ((int64_t)batch * hkv);
    if (max_tokens <= 16 * kSelectThreads || s < 8) return 1;
    const int64_t most = ((int64_t)max_tokens + 4095) / 4096;
    if (s > most) s = most;
    if (s > kMaxSegments) s = kMaxSegments;
    // (16-bit counts; a segment is rounded up to a multiple of 64)
    constexpr int64_t kLargest = 65535 - 64;
    const int64_t least = (max_tokens + kLargest - 1) / kLargest;
    return s < least ? 1 : (int)s;
}

size_t evict_workspace_bytes(int batch, int hkv, int max_tokens, int keep, int num_cus) {
    const size_t rows = (size_t)batch * hkv;
    const int segments = evict_segments(batch, hkv, max_tokens, num_cus);
    size_t bytes = rows * 16;                                                // plan
    if (segments > 1)                                                        // row state, counts per segment, histograms, weights
        bytes += rows * 16 + (rows * segments * 4 + 15) / 16 * 16 + 3 * rows * segments * kBins * 2 + rows * (size_t)keep * 4;
    return bytes;
}

template <int KPT>
static int launch_segments(const EvictParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)p.segments, (unsigned)p.hkv, (unsigned)p.batch), threads(kSelectThreads);
    hipLaunchKernelGGL((evict_segment_kernel<KPT, 0>), grid, threads, 0, stream, p);
    hipLaunchKernelGGL((evict_segment_kernel<KPT, 1>), grid, threads, 0, stream, p);
    hipLaunchKernelGGL((evict_segment_kernel<KPT, 2>), grid, threads, 0, stream, p);
    hipLaunchKernelGGL((evict_segment_kernel<KPT, 3>), grid, threads, 0, stream, p);
    return (int)hipGetLastError();
}

int launch_kv_evict(const EvictParams& p_in, int num_cus, hipStream_t stream) {
    EvictParams p = p_in;
    p.segments = evict_segments(p.batch, p.hkv, p.max_tokens, num_cus);
    if (p.segments > 1) {
        const int64_t rows = (int64_t)p.batch * p.hkv;
        char* at = reinterpret_cast<char*>(p.plan) + rows * 16;
        p.row_state = reinterpret_cast<int2*>(at);
        at += rows * 16;
        p.seg_gt = reinterpret_cast<int32_t*>(at);
        at += (rows * p.segments * 4 + 15) / 16 * 16;
        p.seg_hist = reinterpret_cast<uint16_t*>(at);
        at += 3 * rows * p.segments * kBins * 2;
        p.stash = reinterpret_cast<float*>(at);
        const int per = (p.max_tokens + p.segments - 1) / p.segments;         // (+ up to 63: ranges are multiples of 64)
        const int rc = per <= 4 * kSelectThreads ? launch_segments<4>(p, stream)
                     : per <= 16 * kSelectThreads ? launch_segments<16>(p, stream)
                                                  : launch_segments<0>(p, stream);
        if (rc) return rc;
    } else {
        const dim3 units((unsigned)p.hkv, (unsigned)p.batch), threads(kSelectThreads);
        if (p.max_tokens <= 4 * kSelectThreads) hipLaunchKernelGGL(evict_select_kernel<4>, units, threads, 0, stream, p);
        else if (p.max_tokens <= 16 * kSelectThreads) hipLaunchKernelGGL(evict_select_kernel<16>, units, threads, 0, stream, p);
        else hipLaunchKernelGGL(evict_select_kernel<0>, units, threads, 0, stream, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
    }
    MoveParams m;
    m.e = p;
    // Slices of the rows: 256 bytes, if that gives two workgroups to a compute unit - then one launch does it, each workgroup
    // first the rows that depend on each other, then the rest (32 x 8 kv heads, 2048 rows of K and V kept: 114 us, with slices of
    // 128 bytes 126 us: the rate of a large copy).  Otherwise 128 bytes, and the rest in a launch of its own with more
    // workgroups to a slice; short results stay one launch, which costs less than the few chunks it would spread.  The launch of
    // the dependent rows alone has workgroups of 1024 threads, a quarter of the chunks that wait for one another (8 heads, 1024 such
    // rows: 8.5 us, with 256 threads 12.7; one launch for 256 rows: 7.9 us, with 256 threads 6.1).
    const int64_t rows = (int64_t)p.batch * p.hkv;
    int slices = 0;
    bool one = false;
    for (int widest = 16; widest >= 8 && !one; widest >>= 1) {
        slices = 0;
        for (int t = 0; t < 4; ++t) {
            m.lanes[t] = 1;
            m.slices[t] = 0;
            if (t >= p.num_tensors) continue;
            int lanes = widest;
            while (p.rows[t].cols % lanes) lanes >>= 1;
            m.lanes[t] = lanes;
            m.slices[t] = p.rows[t].cols / lanes;
            slices += m.slices[t];
        }
        one = widest == 16 && slices * rows >= 2 * (int64_t)num_cus;
    }
    const int weight_blocks = p.segments > 1 ? 8 : 0;
    one = one || p.keep <= 1024;
    m.serial = 1;
    m.parallel = one ? 1 : 0;
    m.parts = 1;
    m.row_blocks = slices;
    const dim3 grid((unsigned)(slices + (one ? weight_blocks : 0)), (unsigned)p.hkv, (unsigned)p.batch);
    if (one) hipLaunchKernelGGL(evict_move_kernel<256>, grid, dim3(256), 0, stream, m);
    else hipLaunchKernelGGL(evict_move_kernel<1024>, grid, dim3(1024), 0, stream, m);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || one) return (int)e;
    m.serial = 0;
    m.parallel = 1;
    m.parts = (int32_t)((4 * (int64_t)num_cus + slices * rows - 1) / (slices * rows));
    m.row_blocks = slices * m.parts;
    hipLaunchKernelGGL(evict_move_kernel<256>, dim3((unsigned)(m.row_blocks + weight_blocks), (unsigned)p.hkv, (unsigned)p.batch), dim3(256),
                       0, stream, m);
    return (int)hipGetLastError();
}

}  // namespace fdk
