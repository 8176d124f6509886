// Eviction from a paged cache by accumulated attention weight (gfx950): which keys every (sequence, KV head) keeps, and the
// move of their rows to new pages.
//
// A sequence of L keys keeps n = min(L, budget) of them.  All, when L <= budget; else its first `sinks`, its last `recent`
// and, of the keys between, those with the largest weights; equal weights go to the lower position, a NaN counts as -inf.
// The kept positions stay in order.  Rows are copied to the pages of new_block_table and never within the pages that are
// read: other sequences may share those.
#include "common.hpp"
#include "kernels.hpp"

namespace fck {
namespace {

constexpr int kThreads = 1024;
constexpr int kSelectWaves = kThreads / 64;

// order-preserving map of a weight to an unsigned key; -0 and +0 are equal, NaN is -inf
__device__ __forceinline__ uint32_t weight_key(float w)
{
    if (w != w) w = -INFINITY;
    if (w == 0.f) w = 0.f;
    const uint32_t u = __builtin_bit_cast(uint32_t, w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One workgroup per (sequence, KV head).  The k-th largest key of the middle is found 8 bits at a time from a histogram in
// LDS; then one ordered pass over the positions writes the kept ones (ranks by ballot and a prefix sum over the waves).
__global__ __launch_bounds__(kThreads) void evict_select_kernel(const CacheEvictArgs a)
{
    __shared__ int hist[256];
    __shared__ int chosen[2];
    __shared__ int wave_count[2][kSelectWaves];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hkv = blockIdx.x % a.hk, b = blockIdx.x / a.hk;
    const int64_t cap = (int64_t)a.block_table_stride * a.page_size;
    const int len = (int)min((int64_t)max(a.seqlen_k[b], 0), cap);
    const int n_keep = min(len, a.budget);
    const float* w = a.weights + ((int64_t)b * a.hk + hkv) * a.cols;
    float* nw = a.new_weights + ((int64_t)b * a.hk + hkv) * a.cols;
    int32_t* kept = a.kept + ((int64_t)b * a.hk + hkv) * a.budget;
    // a position the weights have no column for has received nothing
    auto weight = [&](int t) { return t < a.cols ? w[t] : 0.f; };

    // positions [0, lo) and [hi, len) are kept anyway, `want` of [lo, hi) by weight
    const bool all = len <= a.budget;
    const int lo = all ? len : a.sinks, hi = all ? len : len - a.recent;
    const int want = all ? 0 : a.budget - a.sinks - a.recent;
    uint32_t threshold = 0;  // the want-th largest key
    int equal_wanted = 0;    // how many of the positions whose key equals it are kept
    if (want > 0) {
        uint32_t mask = 0;
        int left = want;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int t = lo + tid; t < hi; t += kThreads) {
                const uint32_t key = weight_key(weight(t));
                if ((key & mask) == threshold) atomicAdd(&hist[key >> shift & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int digit = 255, above = 0;
                while (digit > 0 && above + hist[digit] < left) above += hist[digit--];
                chosen[0] = digit;
                chosen[1] = left - above;
            }
            __syncthreads();
            threshold |= (uint32_t)chosen[0] << shift;
            left = chosen[1];
            mask |= 255u << shift;
            __syncthreads();
        }
        equal_wanted = left;
    }

    int n_before = 0, eq_before = 0;  // kept positions and equal keys ahead of this chunk
    for (int t0 = 0; t0 < len; t0 += kThreads) {
        const int t = t0 + tid;
        const float wt = t < len ? weight(t) : 0.f;
        const bool middle = t >= lo && t < hi;
        const uint32_t key = weight_key(wt);
        const bool equal = middle && want > 0 && key == threshold;
        const uint64_t eq_mask = __builtin_amdgcn_ballot_w64(equal);
        const uint64_t below = ((uint64_t)1 << lane) - 1;
        if (lane == 0) wave_count[0][wave] = __builtin_popcountll(eq_mask);
        __syncthreads();
        int eq_rank = eq_before + __builtin_popcountll(eq_mask & below), eq_total = 0;
        for (int v = 0; v < kSelectWaves; ++v) {
            if (v < wave) eq_rank += wave_count[0][v];
            eq_total += wave_count[0][v];
        }
        const bool keep = t < len && (!middle || (want > 0 && (key > threshold || (equal && eq_rank < equal_wanted))));
        const uint64_t keep_mask = __builtin_amdgcn_ballot_w64(keep);
        if (lane == 0) wave_count[1][wave] = __builtin_popcountll(keep_mask);
        __syncthreads();
        int rank = n_before + __builtin_popcountll(keep_mask & below), total = 0;
        for (int v = 0; v < kSelectWaves; ++v) {
            if (v < wave) rank += wave_count[1][v];
            total += wave_count[1][v];
        }
        if (keep && rank < n_keep) {
            kept[rank] = t;
            if (rank < a.cols) nw[rank] = wt;
        }
        n_before += total;
        eq_before += eq_total;
    }
    for (int j = n_keep + tid; j < a.budget; j += kThreads) kept[j] = -1;
    for (int64_t j = n_keep + tid; j < a.cols; j += kThreads) nw[j] = 0.f;
    if (hkv == 0 && tid == 0) a.new_seqlen[b] = n_keep;
}

// Copies the kept rows.  Unit: one 8-byte or 16-byte piece of K or V of one (slot, KV head).
template <typename Piece>
__global__ __launch_bounds__(256) void evict_move_kernel(const CacheEvictArgs a)
{
    const int kp = a.k_row / (int)sizeof(Piece), vp = a.v_row / (int)sizeof(Piece);
    const int per_head = kp + vp;
    const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int piece = (int)(item % per_head);
    const int hkv = (int)(item / per_head % a.hk);
    const int64_t s = item / per_head / a.hk;
    const int slot = (int)(s % a.budget);
    const int64_t b = s / a.budget;
    if (b >= a.batch) return;
    const int t = a.kept[(b * a.hk + hkv) * a.budget + slot];
    if (t < 0) return;
    const int64_t src = (int64_t)a.block_table[b * a.block_table_stride + t / a.page_size] * a.page_size + t % a.page_size;
    const int64_t dst = (int64_t)a.new_block_table[b * a.new_block_table_stride + slot / a.new_page_size] * a.new_page_size + slot % a.new_page_size;
    if (piece < kp)
        ((Piece*)a.new_k)[(dst * a.hk + hkv) * kp + piece] = ((const Piece*)a.k)[(src * a.hk + hkv) * kp + piece];
    else
        ((Piece*)a.new_v)[(dst * a.hk + hkv) * vp + piece - kp] = ((const Piece*)a.v)[(src * a.hk + hkv) * vp + piece - kp];
}

template <typename Piece>
hipError_t launch_move(const CacheEvictArgs& a, hipStream_t st)
{
    const int64_t items = (int64_t)a.batch * a.budget * a.hk * ((a.k_row + a.v_row) / (int)sizeof(Piece));
    const int64_t grid = (items + 255) / 256;
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((evict_move_kernel<Piece>), dim3((unsigned)grid), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_evict(const CacheEvictArgs& a, hipStream_t st)
{
    if ((int64_t)a.batch * a.hk > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)(a.batch * a.hk)), dim3(kThreads), 0, st, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    // rows of an odd number of 8-byte pieces (an e4m3 cache with such a head dim) are moved 8 bytes at a time
    return a.k_row % 16 == 0 && a.v_row % 16 == 0 ? launch_move<u32x4_t>(a, st) : launch_move<u32x2_t>(a, st);
}

}  // namespace fck
