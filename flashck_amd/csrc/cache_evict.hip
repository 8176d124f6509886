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

constexpr int kEvictParts = 8;           // workgroups per row of the wide choice
// columns from which it is taken: one sequence, 8 heads, choice and move, with one and with 8 workgroups per row: 45 and 49 us
// at 32768 keys, 90 and 49 us at 131072
constexpr int64_t kEvictWideCols = 65536;
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

// The choice of one (sequence, KV head), by `parts` workgroups of 16 waves.  Bound by the walks over its weights (L2 round
// trips and some 20 instructions per weight), so they are few and wide: a wave owns a contiguous part of the row and reads 4
// weights per lane and load.
//   1. The want-th largest key of the middle, 11 bits per walk, from a histogram in LDS with a copy for every 8th lane, so
//      that equal weights, zeros above all, meet at an address seldom (one copy and 8 bits per walk: 369 us for a sequence of
//      131072 keys and 8 heads; a copy per lane: 154 us; so: 107 us).
//   2. A walk that counts what each wave keeps, and one that writes it from the wave's first rank on: ranks are ballots, and
//      no barrier lies inside a walk.
struct SelectLds {
    int hist[kBins * kColumns];  // [digit][copy]
    __align__(16) int digits[kBins];
    int groups[kBins / 64];
    int chosen[3];
    int counts[2][kWaves];
};

struct Select {
    const CacheEvictArgs& a;
    SelectLds& lds;
    int tid, lane, wave, hkv, b, part, parts;
    int len, n_keep, lo, hi, want, seg0, seg1;
    bool all, vec;
    const float* w;
    float* nw;
    int32_t* kept;
    // the want-th largest key in the digits of `mask`, and how many of the positions whose key equals it are kept
    uint32_t threshold = 0, mask = 0;
    int left = 0;

    __device__ __forceinline__ Select(const CacheEvictArgs& a_, SelectLds& lds_, int row, int part_, int parts_) : a(a_), lds(lds_)
    {
        tid = threadIdx.x;
        lane = tid & 63;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        hkv = row % a.hk;
        b = row / a.hk;
        part = part_;
        parts = parts_;
        const int64_t cap = (int64_t)a.block_table_stride * a.page_size;
        len = __builtin_amdgcn_readfirstlane((int)min((int64_t)max(a.seqlen_k[b], 0), cap));
        n_keep = min(len, a.budget);
        w = a.weights + (int64_t)row * a.cols;
        nw = a.new_weights + (int64_t)row * a.cols;
        kept = a.kept + (int64_t)row * a.budget;
        vec = a.cols % 4 == 0 && (reinterpret_cast<uintptr_t>(a.weights) & 15) == 0;
        // positions [0, lo) and [hi, len) are kept anyway, `want` of [lo, hi) by weight
        all = len <= a.budget;
        lo = all ? len : a.sinks;
        hi = all ? len : len - a.recent;
        want = all ? 0 : a.budget - a.sinks - a.recent;
        left = want;
        const int waves = parts * kWaves;
        const int64_t seg = ((len + waves - 1) / waves + 255) / 256 * 256;
        seg0 = (int)min((part * kWaves + wave) * seg, (int64_t)len);
        seg1 = (int)min((part * kWaves + wave + 1) * seg, (int64_t)len);
    }

    // the 4 weights from position t on; a position the weights have no column for has received nothing
    __device__ __forceinline__ f32x4_t load4(int t) const
    {
        if (vec && t + 4 <= a.cols) return *reinterpret_cast<const f32x4_t*>(w + t);
        f32x4_t x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = t + e < a.cols ? w[t + e] : 0.f;
        return x;
    }

    // calls f(position of the lane's first weight, its 4 weights, whether all of the wave's 256 lie in the middle) for the
    // wave's part; other positions may lie behind the row, which is f's to leave out.  Four loads are in flight per lane.
    template <typename F>
    __device__ __forceinline__ void walk(F f) const
    {
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
    }

    __device__ __forceinline__ static int shift_of(int digit) { return max(32 - kBits * (digit + 1), 0); }
    __device__ __forceinline__ uint32_t digit_bits(int digit) const { return (kBins - 1u) << shift_of(digit) & ~mask; }

    // counts the digit of the keys that begin like the threshold: lds.digits
    __device__ __forceinline__ void histogram(int digit)
    {
        const int shift = shift_of(digit);
        const uint32_t bits = digit_bits(digit);
        for (int e = tid; e < kBins * kColumns; e += kThreads) lds.hist[e] = 0;
        __syncthreads();
        walk([&](int t, const f32x4_t& x, auto middle) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t key = weight_key(x[e]);
                const bool in = decltype(middle)::value || (t + e >= lo && t + e < hi);
                if (in && (key & mask) == threshold) atomicAdd(&lds.hist[((key & bits) >> shift) * kColumns + lane % kColumns], 1);
            }
        });
        __syncthreads();
        for (int d = tid; d < kBins; d += kThreads) {
            int sum = 0;
#pragma unroll
            for (int c = 0; c < kColumns; ++c) sum += lds.hist[d * kColumns + ((c + d) & (kColumns - 1))];
            lds.digits[d] = sum;
        }
        __syncthreads();
    }

    // the digit of the left-th largest from lds.digits, by groups of 64 digits first; true when no further digit matters
    __device__ __forceinline__ bool take_digit(int digit)
    {
        if (tid < kBins / 64) {
            int sum = 0;
            for (int d = 0; d < 64; ++d) sum += lds.digits[tid * 64 + ((d + tid) & 63)];
            lds.groups[tid] = sum;
        }
        __syncthreads();
        if (tid < kBins / 64) {
            int above = 0;
            for (int j = 0; j < kBins / 64; ++j) above += j > tid ? lds.groups[j] : 0;
            if (above < left && left <= above + lds.groups[tid]) {  // exactly one thread
                lds.chosen[0] = tid * 64;
                lds.chosen[1] = left - above;
            }
        }
        __syncthreads();
        const int first = lds.chosen[0], in_group = lds.chosen[1];
        __syncthreads();
        if (tid < 64) {
            int above = 0;
            for (int j = 0; j < 64; j += 4) {
                const u32x4_t n = *reinterpret_cast<const u32x4_t*>(&lds.digits[first + j]);
#pragma unroll
                for (int e = 0; e < 4; ++e) above += j + e > tid ? (int)n[e] : 0;
            }
            const int here = lds.digits[first + tid];
            if (above < in_group && in_group <= above + here) {  // exactly one thread
                lds.chosen[0] = first + tid;
                lds.chosen[1] = in_group - above;
                lds.chosen[2] = here;
            }
        }
        __syncthreads();
        const uint32_t bits = digit_bits(digit);
        threshold |= (uint32_t)lds.chosen[0] << shift_of(digit);
        left = lds.chosen[1];
        mask |= bits;
        const bool done = mask == 0xffffffffu || lds.chosen[2] == left;  // every key that begins like this is kept
        __syncthreads();
        return done;
    }

    // (kept without question, equal to the threshold) of the wave's part
    __device__ __forceinline__ void count(int& sure, int& equal) const
    {
        int s = 0, q = 0;
        walk([&](int t, const f32x4_t& x, auto in) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int p = t + e;
                const uint32_t key = weight_key(x[e]) & mask;
                const bool middle = decltype(in)::value || (p >= lo && p < hi);
                s += __builtin_popcountll(__builtin_amdgcn_ballot_w64(p < len && (!middle || key > threshold)));
                q += __builtin_popcountll(__builtin_amdgcn_ballot_w64(middle && key == threshold));
            }
        });
        sure = s;
        equal = q;
    }

    // writes what the wave's part keeps from `rank` on; equal_left of the keys that equal the threshold are still wanted
    __device__ __forceinline__ void write(int rank, int equal_left) const
    {
        walk([&](int t, const f32x4_t& x, auto in) {
            // per element: kept without question, or equal to the threshold and early enough
            uint64_t keep_mask[4], eq_mask[4];
            bool mine[4], eq[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int p = t + e;
                const uint32_t key = weight_key(x[e]) & mask;
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
    }

    // a row whose weights do not matter: all of it, or the sinks and the most recent ones
    __device__ __forceinline__ void write_fixed() const
    {
        for (int j = part * kThreads + tid; j < n_keep; j += parts * kThreads) {
            const int t = all || j < a.sinks ? j : len - n_keep + j;
            kept[j] = t;
            if (j < a.cols) nw[j] = t < a.cols ? w[t] : 0.f;
        }
    }

    // what lies behind the kept keys
    __device__ __forceinline__ void write_tail() const
    {
        const int me = part * kThreads + tid, step = parts * kThreads;
        for (int j = n_keep + me; j < a.budget; j += step) kept[j] = -1;
        int64_t z = min(((int64_t)n_keep + 3) / 4 * 4, a.cols);
        if (n_keep + me < z) nw[n_keep + me] = 0.f;
        if (vec && (reinterpret_cast<uintptr_t>(a.new_weights) & 15) == 0)
            for (z += (int64_t)me * 4; z < a.cols; z += (int64_t)step * 4) *reinterpret_cast<f32x4_t*>(nw + z) = f32x4_t{0.f, 0.f, 0.f, 0.f};
        else
            for (z += me; z < a.cols; z += step) nw[z] = 0.f;
        if (hkv == 0 && me == 0) a.new_seqlen[b] = n_keep;
    }
};

// one workgroup per row
__global__ __launch_bounds__(kThreads) void evict_select_kernel(const CacheEvictArgs a)
{
    __shared__ SelectLds lds;
    Select s(a, lds, blockIdx.x, 0, 1);
    if (s.want > 0) {
        for (int digit = 0;; ++digit) {
            s.histogram(digit);
            if (s.take_digit(digit)) break;
        }
        int sure, equal;
        s.count(sure, equal);
        if (s.lane == 0) {
            lds.counts[0][s.wave] = sure;
            lds.counts[1][s.wave] = equal;
        }
        __syncthreads();
        int rank = 0, equal_left = s.left;
        for (int v = 0; v < s.wave; ++v) {
            const int eq = min(lds.counts[1][v], equal_left);
            rank += lds.counts[0][v] + eq;
            equal_left -= eq;
        }
        s.write(rank, equal_left);
    } else {
        s.write_fixed();
    }
    s.write_tail();
}

// kEvictParts workgroups per row, one launch per step, for few long rows: the steps hand each other their sums through the
// workspace.  Step d = 0, 1, 2 takes the digit before (d > 0) and counts digit d of its part; step 3 takes the last digit and
// counts what each wave keeps; step 4 writes.
struct WideRow {
    int hist[3][kEvictParts][kBins];
    uint32_t state[3][4];  // after digit d: threshold, mask, left, done
    int counts[kEvictParts * kWaves][2];
};

template <int kStep>
__global__ __launch_bounds__(kThreads) void evict_select_wide_kernel(const CacheEvictArgs a)
{
    __shared__ SelectLds lds;
    const int row = blockIdx.x / kEvictParts;
    Select s(a, lds, row, blockIdx.x % kEvictParts, kEvictParts);
    WideRow& ws = reinterpret_cast<WideRow*>(a.workspace)[row];
    if (s.want == 0) {  // uniform
        if (kStep == 4) {
            s.write_fixed();
            s.write_tail();
        }
        return;
    }
    bool done = false;
    if constexpr (kStep >= 2) {
        const uint32_t* st = ws.state[kStep == 4 ? 2 : kStep - 2];
        s.threshold = st[0];
        s.mask = st[1];
        s.left = (int)st[2];
        done = st[3] != 0;
    }
    if constexpr (kStep >= 1 && kStep <= 3) {
        if (!done) {
            for (int d = s.tid; d < kBins; d += kThreads) {
                int sum = 0;
#pragma unroll
                for (int p = 0; p < kEvictParts; ++p) sum += ws.hist[kStep - 1][p][d];
                lds.digits[d] = sum;
            }
            __syncthreads();
            done = s.take_digit(kStep - 1);
        }
        if (s.part == 0 && s.tid == 0) {
            uint32_t* st = ws.state[kStep - 1];
            st[0] = s.threshold;
            st[1] = s.mask;
            st[2] = (uint32_t)s.left;
            st[3] = done;
        }
    }
    if constexpr (kStep <= 2) {
        if (done) return;
        s.histogram(kStep);
        for (int d = s.tid; d < kBins; d += kThreads) ws.hist[kStep][s.part][d] = lds.digits[d];
    } else if constexpr (kStep == 3) {
        int sure, equal;
        s.count(sure, equal);
        if (s.lane == 0) {
            ws.counts[s.part * kWaves + s.wave][0] = sure;
            ws.counts[s.part * kWaves + s.wave][1] = equal;
        }
    } else {
        // the counts of all waves of the row through LDS: read one by one they are a chain of round trips
        if (s.tid < kEvictParts * kWaves * 2) lds.digits[s.tid] = ws.counts[s.tid / 2][s.tid & 1];
        __syncthreads();
        int rank = 0, equal_left = s.left;
        for (int v = 0; v < s.part * kWaves + s.wave; ++v) {
            const int eq = min(lds.digits[2 * v + 1], equal_left);
            rank += lds.digits[2 * v] + eq;
            equal_left -= eq;
        }
        s.write(rank, equal_left);
        s.write_tail();
    }
}

// Copies the kept rows.  A thread moves one 8- or 16-byte piece of K and of V of one KV head for kSlots consecutive slots, so
// that the chain position -> page -> row is walked for all of them at once and 2 kSlots loads are in flight; consecutive
// threads write consecutive pieces of a slot's row.
constexpr int kSlots = 4;

// rows of an odd number of 8-byte pieces (an e4m3 cache with such a head dim) are moved 8 bytes at a time
int move_piece(const CacheEvictArgs& a) { return a.k_row % 16 == 0 && a.v_row % 16 == 0 ? 16 : 8; }

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
    const int64_t items = cache_evict_move_items(a);
    hipLaunchKernelGGL((evict_move_kernel<Piece>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

int64_t cache_evict_move_items(const CacheEvictArgs& a)
{
    const int64_t pieces = (a.k_row > a.v_row ? a.k_row : a.v_row) / move_piece(a);
    const int64_t groups = ((int64_t)a.budget + kSlots - 1) / kSlots * pieces, rows = (int64_t)a.batch * a.hk;
    return rows > INT32_MAX / groups ? -1 : rows * groups;  // the kernel counts in 32 bits
}

size_t cache_evict_workspace_bytes(int64_t rows, int64_t cols, int num_cu)
{
    // several workgroups per row where one per row leaves most of the chip idle and the walks outweigh the extra launches
    return rows * kEvictParts <= num_cu && cols >= kEvictWideCols ? (size_t)rows * sizeof(WideRow) : 0;
}

hipError_t launch_cache_evict(const CacheEvictArgs& a, hipStream_t st)
{
    if ((int64_t)a.batch * a.hk > INT32_MAX) return hipErrorInvalidValue;
    const dim3 rows((unsigned)(a.batch * a.hk)), parts((unsigned)(a.batch * a.hk * kEvictParts)), threads(kThreads);
    if (a.workspace) {
        hipLaunchKernelGGL((evict_select_wide_kernel<0>), parts, threads, 0, st, a);
        hipLaunchKernelGGL((evict_select_wide_kernel<1>), parts, threads, 0, st, a);
        hipLaunchKernelGGL((evict_select_wide_kernel<2>), parts, threads, 0, st, a);
        hipLaunchKernelGGL((evict_select_wide_kernel<3>), parts, threads, 0, st, a);
        hipLaunchKernelGGL((evict_select_wide_kernel<4>), parts, threads, 0, st, a);
    } else {
        hipLaunchKernelGGL(evict_select_kernel, rows, threads, 0, st, a);
    }
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    return move_piece(a) == 16 ? launch_move<u32x4_t>(a, st) : launch_move<u32x2_t>(a, st);
}

}  // namespace fck
