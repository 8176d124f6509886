// Attention weight that every key of a cache receives (gfx950):
//   out[b, hk, t] = weights[b, hk, t] + sum over the query heads h of KV head hk and the rows i that see t of exp(s_ih(t) - lse_ih)
// with s = mod(scale * q.k) and lse the log-sum-exp the attention over the same keys returned.  Entries at and behind a
// sequence's key count are written as zeros, so that a key appended later starts from nothing.
//
// Work decomposition
//   A wave owns 32 keys: their K rows sit in its registers as the A operand of S^T = K . Q^T (v_mfma_f32_32x32x16) while it
//   walks the query rows that see them, 32 at a time, as the B operand.  Each accumulator element (key, row) is one
//   exponential added to a running sum of its own; the 32 row columns are added up once at the end.  No two waves write the
//   same key, so there are no atomics and the order of the sums is fixed.
// The contraction index of both operands is permuted the same way (lane half `half` of step t holds chunk half * D/16 + t):
// the product does not change, and a lane reads contiguous 16-byte chunks of one row.
#include "common.hpp"
#include "kernels.hpp"

namespace fck {
namespace {

constexpr int kWaves = 4;
constexpr int kKeysPerWave = 32;
constexpr int kKeysPerWg = kWaves * kKeysPerWave;

// kMod: ALiBi / soft cap.  kKv8: e4m3 keys, widened to T; always with kMod.  The stored head dim a.d may be smaller than D
// (missing chunks are zeros).
template <typename T, int D, bool kMod, bool kKv8>
__global__ __launch_bounds__(kWaves * 64) void key_weights_kernel(const KeyWeightsArgs a)
{
    typedef typename T::vec8 vec8;
    constexpr int KT = D / 16;
    __shared__ float sums[kWaves][kKeysPerWave][33];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, half = lane >> 5;
    const int g = a.hq / a.hk;
    const int hkv = blockIdx.x % a.hk;
    const int b = blockIdx.x / a.hk % a.batch;
    const int64_t key0 = (int64_t)(blockIdx.x / a.hk / a.batch) * kKeysPerWg + wave * kKeysPerWave;

    const KvSeq ks = kv_seq(a.kv, b);
    const int sk = max(ks.len, 0);
    const int tok0 = a.seqstart_q ? a.seqstart_q[b] : b * a.sq;
    const int sq = a.seqstart_q ? a.seqstart_q[b + 1] - tok0 : a.sq;
    const MaskYX mk = make_mask(a.mask_type, a.window_left, a.window_right, sq, sk);

    f32x16_t acc;
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] = 0.f;

    if (key0 < sk) {  // uniform per wave
        u32x4_t kf[KT];
        {
            const int key = (int)min(key0 + l32, (int64_t)sk - 1);  // keys past the end repeat the last one, and are not stored
            const int64_t row = (kv_row(a.kv, ks, key) * a.hk + hkv) * a.d;
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const int chunk = half * KT + t;
                kf[t] = u32x4_t{0u, 0u, 0u, 0u};
                if (chunk * 8 < a.d) {
                    if constexpr (kKv8) {
                        const u32x2_t v = ldg8_stream((const uint8_t*)a.k + row + chunk * 8);
                        kf[t] = fp8x8_to_t<T>(u32x4_t{v[0], v[1], 0u, 0u});
                    } else {
                        kf[t] = ldg16_stream((const uint16_t*)a.k + row + chunk * 8);
                    }
                }
            }
        }
        // rows r = head in group * sq + i
        const int64_t R = (int64_t)g * sq;
        for (int64_t r0 = 0; r0 < R; r0 += 32) {
            const int64_t r = r0 + l32;
            const bool row_ok = r < R;
            const int hl = row_ok ? (int)(r / sq) : 0, i = row_ok ? (int)(r % sq) : 0;
            const int h = hkv * g + hl;
            const int lo = row_ok ? mask_lo(mk, i) : 0, hi = row_ok ? mask_hi(mk, i, sk) : 0;
            // nothing of this tile sees one of the wave's keys
            if (__builtin_amdgcn_ballot_w64(hi > key0 && lo < key0 + kKeysPerWave) == 0) continue;
            const float lse = row_ok ? a.lse[((int64_t)(a.seqstart_q ? 0 : b) * a.hq + h) * a.lse_sq + (a.seqstart_q ? tok0 : 0) + i] : -INFINITY;
            // a row that saw no key has lse = -inf and gives nothing
            const float lse2 = lse * kLog2e;
            const bool row_in = row_ok && lse != -INFINITY;
            ArithMod amod;
            if constexpr (kMod) amod.init(a.mod, b, h, i, sq, sk, a.mask_type, a.window_left, a.window_right);
            f32x16_t s;
#pragma unroll
            for (int j = 0; j < 16; ++j) s[j] = 0.f;
            const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + ((int64_t)(tok0 + i) * a.hq + h) * a.d + half * KT * 8;
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                u32x4_t qv = {0u, 0u, 0u, 0u};
                if (row_ok && (half * KT + t) * 8 < a.d) qv = ldg16(qp + t * 8);
                s = T::mfma32(as_vec8<vec8>(kf[t]), as_vec8<vec8>(qv), s);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int key = (int)key0 + (j >> 2) * 8 + half * 4 + (j & 3);
                float e;
                if constexpr (kMod)
                    e = fast_exp2(amod.score(s[j], key) - lse2);
                else
                    e = fast_exp2(__builtin_fmaf(s[j], a.scale_log2, -lse2));
                acc[j] += row_in && key >= lo && key < hi ? e : 0.f;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) sums[wave][(j >> 2) * 8 + half * 4 + (j & 3)][l32] = acc[j];
    __syncthreads();
    // one thread per key
    const int64_t key = key0 + l32;
    if (lane >= 32 || key >= a.cols) return;
    float total = 0.f;
    if (key < sk) {
        for (int n = 0; n < 32; ++n) total += sums[wave][l32][n];
        if (a.weights) total += a.weights[((int64_t)b * a.hk + hkv) * a.cols + key];
    }
    a.out[((int64_t)b * a.hk + hkv) * a.cols + key] = total;
}

template <typename T, int D>
hipError_t launch_d(const KeyWeightsArgs& a, hipStream_t st)
{
    const int64_t grid = (a.cols + kKeysPerWg - 1) / kKeysPerWg * a.batch * a.hk;
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    const dim3 blocks((unsigned)grid), threads(kWaves * 64);
    if (a.kv8)
        hipLaunchKernelGGL((key_weights_kernel<T, D, true, true>), blocks, threads, 0, st, a);
    else if (a.mod.active())
        hipLaunchKernelGGL((key_weights_kernel<T, D, true, false>), blocks, threads, 0, st, a);
    else
        hipLaunchKernelGGL((key_weights_kernel<T, D, false, false>), blocks, threads, 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_key_weights(const KeyWeightsArgs& a, int d, int dtype, hipStream_t st)
{
    switch (d) {
    case 64: return dtype == 4 ? launch_d<BF16, 64>(a, st) : launch_d<FP16, 64>(a, st);
    case 128: return dtype == 4 ? launch_d<BF16, 128>(a, st) : launch_d<FP16, 128>(a, st);
    case 256: return dtype == 4 ? launch_d<BF16, 256>(a, st) : launch_d<FP16, 256>(a, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace fck
