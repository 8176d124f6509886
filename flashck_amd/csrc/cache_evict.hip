// Eviction from a paged cache by accumulated attention weight (gfx950): which keys every (sequence, KV head) keeps, and the
// move of their rows to new pages.
//
// A sequence of L keys keeps n = min(L, budget) of them.  All, when L <= budget; else its first `sinks`, its last `recent`
// and, of the keys between, those with the largest weights; equal weights go to the lower position, a NaN counts as -inf.
// The kept positions stay in order.  Rows are copied to the pages of new_block_table and never within the pages that are
// read: other sequences may share those.
#include "common.hpp"
#include "kernels.hpp"

#include <type_traits>

namespace fck {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;

// order-preserving map of a weight to an unsigned key; -0 and +0 are equal, NaN is -inf
__device__ __forceinline__ uint32_t weight_key(float w)
{
    const float x = fmaxf(w + 0.f, -INFINITY);  // the sum turns -0 into +0, the maximum a NaN into -inf
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// The histogram of one digit: kBins counters in kColumns copies, a lane adds to copy lane % kColumns.
constexpr int kBits = 11, kBins = 1 << kBits, kColumns = 8;

// One workgroup per (sequence, KV head); bound by the walks over its weights (L2 round trips), so they are few and wide: a wave
// owns a contiguous sixteenth of the row and reads 4 weights per lane and load.
//   1. The want-th largest key of the middle, 11 bits per walk, from a histogram in LDS with a copy for every 8th lane, so
//      that equal weights, zeros above all, meet at an address seldom (one copy and 8 bits per walk: 369 us for a sequence of
//      131072 keys and 8 heads; a copy per lane: 154 us).
//   2. A walk that counts what each wave keeps, and one that writes it from the wave's first rank on: ranks are ballots, and
//      no barrier lies inside a walk.
__global__ __launch_bounds__(kThreads) void evict_select_kernel(const CacheEvictArgs a)
{
    __shared__ int hist[kBins * kColumns];  // [digit][copy]
    __shared__ __align__(16) int digits[kBins], groups[kBins / 64];
    __shared__ int chosen[3];
    __shared__ int counts[2][kWaves];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hkv = blockIdx.x % a.hk, b = blockIdx.x / a.hk;
    const int64_t cap = (int64_t)a.block_table_stride * a.page_size;
    const int len = __builtin_amdgcn_readfirstlane((int)min((int64_t)max(a.seqlen_k[b], 0), cap));
    const int n_keep = min(len, a.budget);
    const float* const w = a.weights + ((int64_t)b * a.hk + hkv) * a.cols;
    float* const nw = a.new_weights + ((int64_t)b * a.hk + hkv) * a.cols;
    int32_t* const kept = a.kept + ((int64_t)b * a.hk + hkv) * a.budget;
    const bool vec = a.cols % 4 == 0 && (reinterpret_cast<uintptr_t>(a.weights) & 15) == 0;

    // positions [0, lo) and [hi, len) are kept anyway, `want` of [lo, hi) by weight
    const bool all = len <= a.budget;
    const int lo = all ? len : a.sinks, hi = all ? len : len - a.recent;
    const int want = all ? 0 : a.budget - a.sinks - a.recent;

    const int seg = ((len + kWaves - 1) / kWaves + 255) / 256 * 256;
    const int seg0 = (int)min((int64_t)wave * seg, (int64_t)len), seg1 = (int)min((int64_t)(wave + 1) * seg, (int64_t)len);
    // the 4 weights from position t on; a position the weights have no column for has received nothing
    auto load4 = [&](int t) -> f32x4_t {
        if (vec && t + 4 <= a.cols) return *reinterpret_cast<const f32x4_t*>(w + t);
        f32x4_t x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = t + e < a.cols ? w[t + e] : 0.f;
        return x;
    };
    // calls f(position of the lane's first weight, its 4 weights, whether all of the wave's 256 lie in the middle) for the
    // wave's segment; other positions may lie behind the row, which is f's to leave out.  Four loads are in flight per lane.
    auto walk = [&](auto f) {
        auto call = [&](int t0, const f32x4_t& x) {
            if (t0 >= lo && t0 + 256 <= hi)
                f(t0 + lane * 4, x, std::true_type{});
            else
                f(t0 + lane * 4, x, std::false_type{});
        };
        int t0 = seg0;
        for (; t0 + 1024 <= seg1; t0 += 1024) {
            f32x4_t x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = load4(t0 + u * 256 + lane * 4);
#pragma unroll
            for (int u = 0; u < 4; ++u) call(t0 + u * 256, x[u]);
        }
        for (; t0 < seg1; t0 += 256) call(t0, load4(t0 + lane * 4));
    };

    uint32_t threshold = 0;  // the want-th largest key, in the digits that decide
    int equal_wanted = 0;    // how many of the positions whose key equals it are kept
    if (want > 0) {
        uint32_t mask = 0;
        int left = want;
        for (int shift = 32 - kBits; mask != 0xffffffffu; shift = max(shift - kBits, 0)) {
            const uint32_t digit_mask = (kBins - 1u) << shift & ~mask;
            for (int e = tid; e < kBins * kColumns; e += kThreads) hist[e] = 0;
            __syncthreads();
            walk([&](int t, const f32x4_t& x, auto middle) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t key = weight_key(x[e]);
                    const bool in = decltype(middle)::value || (t + e >= lo && t + e < hi);
                    if (in && (key & mask) == threshold) atomicAdd(&hist[((key & digit_mask) >> shift) * kColumns + lane % kColumns], 1);
                }
            });
            __syncthreads();
            // the digit of the left-th largest: by groups of 64 digits first
            for (int d = tid; d < kBins; d += kThreads) {
                int sum = 0;
#pragma unroll
                for (int c = 0; c < kColumns; ++c) sum += hist[d * kColumns + ((c + d) & (kColumns - 1))];
                digits[d] = sum;
            }
            __syncthreads();
            if (tid < kBins / 64) {
                int sum = 0;
                for (int d = 0; d < 64; ++d) sum += digits[tid * 64 + ((d + tid) & 63)];
                groups[tid] = sum;
            }
            __syncthreads();
            if (tid < kBins / 64) {
                int above = 0;
                for (int j = 0; j < kBins / 64; ++j) above += j > tid ? groups[j] : 0;
                if (above < left && left <= above + groups[tid]) {  // exactly one thread
                    chosen[0] = tid * 64;
                    chosen[1] = left - above;
                }
            }
            __syncthreads();
            const int first = chosen[0], in_group = chosen[1];
            __syncthreads();
            if (tid < 64) {
                int above = 0;
                for (int j = 0; j < 64; j += 4) {
                    const u32x4_t n = *reinterpret_cast<const u32x4_t*>(&digits[first + j]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) above += j + e > tid ? (int)n[e] : 0;
                }
                const int here = digits[first + tid];
                if (above < in_group && in_group <= above + here) {  // exactly one thread
                    chosen[0] = first + tid;
                    chosen[1] = in_group - above;
                    chosen[2] = here;
                }
            }
            __syncthreads();
            threshold |= (uint32_t)chosen[0] << shift;
            left = chosen[1];
            mask |= digit_mask;
            if (chosen[2] == left) break;  // every key that begins like this is kept: the digits behind do not matter
            __syncthreads();
        }
        equal_wanted = left;
        const uint32_t m = mask;
        int sure = 0, equal = 0;
        walk([&](int t, const f32x4_t& x, auto in) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int p = t + e;
                const uint32_t key = weight_key(x[e]) & m;
                const bool middle = decltype(in)::value || (p >= lo && p < hi);
                sure += __builtin_popcountll(__builtin_amdgcn_ballot_w64(p < len && (!middle || key > threshold)));
                equal += __builtin_popcountll(__builtin_amdgcn_ballot_w64(middle && key == threshold));
            }
        });
        if (lane == 0) {
            counts[0][wave] = sure;
            counts[1][wave] = equal;
        }
        __syncthreads();
        int rank = 0, equal_left = equal_wanted;
        for (int v = 0; v < wave; ++v) {
            const int eq = min(counts[1][v], equal_left);
            rank += counts[0][v] + eq;
            equal_left -= eq;
        }
        walk([&](int t, const f32x4_t& x, auto in) {
            // per element: kept without question, or equal to the threshold and early enough
            uint64_t keep_mask[4], eq_mask[4];
            bool mine[4], eq[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int p = t + e;
                const uint32_t key = weight_key(x[e]) & m;
                const bool middle = decltype(in)::value || (p >= lo && p < hi);
                mine[e] = p < len && (!middle || key > threshold);
                eq[e] = middle && key == threshold;
                eq_mask[e] = __builtin_amdgcn_ballot_w64(eq[e]);
            }
            const uint64_t below = ((uint64_t)1 << lane) - 1;
            int eq_rank = 0, eq_total = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                eq_rank += __builtin_popcountll(eq_mask[e] & below);
                eq_total += __builtin_popcountll(eq_mask[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (eq[e] && eq_rank < equal_left) mine[e] = true;
                eq_rank += eq[e] ? 1 : 0;
            }
            equal_left = max(equal_left - eq_total, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) keep_mask[e] = __builtin_amdgcn_ballot_w64(mine[e]);
            int at = rank;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                at += __builtin_popcountll(keep_mask[e] & below);
                rank += __builtin_popcountll(keep_mask[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (mine[e]) {
                    if (at < n_keep) {
                        kept[at] = t + e;
                        if (at < a.cols) nw[at] = x[e];
                    }
                    ++at;
                }
        });
    } else {
        // all of them, or the sinks and the most recent ones
        for (int j = tid; j < n_keep; j += kThreads) {
            const int t = all || j < a.sinks ? j : len - n_keep + j;
            kept[j] = t;
            if (j < a.cols) nw[j] = t < a.cols ? w[t] : 0.f;
        }
    }
    for (int j = n_keep + tid; j < a.budget; j += kThreads) kept[j] = -1;
    int64_t z = min(((int64_t)n_keep + 3) / 4 * 4, a.cols);
    if (n_keep + tid < z) nw[n_keep + tid] = 0.f;
    if (vec && (reinterpret_cast<uintptr_t>(a.new_weights) & 15) == 0)
        for (z += tid * 4; z < a.cols; z += kThreads * 4) *reinterpret_cast<f32x4_t*>(nw + z) = f32x4_t{0.f, 0.f, 0.f, 0.f};
    else
        for (z += tid; z < a.cols; z += kThreads) nw[z] = 0.f;
    if (hkv == 0 && tid == 0) a.new_seqlen[b] = n_keep;
}

// Copies the kept rows.  A thread moves one 8- or 16-byte piece of K and of V of one KV head for kSlots consecutive slots, so
// that the chain position -> page -> row is walked for all of them at once and 2 kSlots loads are in flight; consecutive
// threads write consecutive pieces of a slot's row.
constexpr int kSlots = 4;
template <typename Piece>
__global__ __launch_bounds__(256) void evict_move_kernel(const CacheEvictArgs a)
{
    const uint32_t kp = a.k_row / (uint32_t)sizeof(Piece), vp = a.v_row / (uint32_t)sizeof(Piece);
    const uint32_t pieces = max(kp, vp), per_seq = (uint32_t)(a.budget + kSlots - 1) / kSlots;
    uint32_t id = blockIdx.x * 256u + threadIdx.x;
    const uint32_t piece = id % pieces;
    id /= pieces;
    const uint32_t hkv = id % (uint32_t)a.hk;
    id /= (uint32_t)a.hk;
    const int slot0 = (int)(id % per_seq) * kSlots;
    const int64_t b = id / per_seq;
    if (b >= a.batch) return;
    const int32_t* const kept = a.kept + (b * a.hk + hkv) * a.budget;
    int t[kSlots];
#pragma unroll
    for (int s = 0; s < kSlots; ++s) t[s] = slot0 + s < a.budget ? kept[slot0 + s] : -1;
    auto locate = [](const int32_t* table, int pos, int page, int shift) -> int64_t {
        const int pi = shift >= 0 ? pos >> shift : pos / page;
        return (int64_t)table[pi] * page + (pos - pi * page);
    };
    int64_t src[kSlots], dst[kSlots];
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
        src[s] = dst[s] = 0;
        if (t[s] >= 0) {
            src[s] = locate(a.block_table + b * a.block_table_stride, t[s], a.page_size, a.page_shift) * a.hk + hkv;
            dst[s] = locate(a.new_block_table + b * a.new_block_table_stride, slot0 + s, a.new_page_size, a.new_page_shift) * a.hk + hkv;
        }
    }
    Piece k[kSlots], v[kSlots];
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
        if (t[s] >= 0 && piece < kp) k[s] = __builtin_nontemporal_load((const Piece*)a.k + src[s] * kp + piece);
        if (t[s] >= 0 && piece < vp) v[s] = __builtin_nontemporal_load((const Piece*)a.v + src[s] * vp + piece);
    }
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
        if (t[s] >= 0 && piece < kp) ((Piece*)a.new_k)[dst[s] * kp + piece] = k[s];
        if (t[s] >= 0 && piece < vp) ((Piece*)a.new_v)[dst[s] * vp + piece] = v[s];
    }
}

template <typename Piece>
hipError_t launch_move(const CacheEvictArgs& a, hipStream_t st)
{
    const int64_t pieces = (a.k_row > a.v_row ? a.k_row : a.v_row) / (int)sizeof(Piece);
    const int64_t items = (int64_t)a.batch * ((a.budget + kSlots - 1) / kSlots) * a.hk * pieces;
    if (items > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((evict_move_kernel<Piece>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, st, a);
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
