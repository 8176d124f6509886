// Attention weight that every key of a cache receives (gfx950):
//   out[b, hk, t] = weights[b, hk, t] + sum over the query heads h of KV head hk and the rows i that see t of exp(s_ih(t) - lse_ih)
// with s = mod(scale * q.k) and lse the log-sum-exp the attention over the same keys returned.  Entries at and behind a
// sequence's key count are written as zeros, so that a key appended later starts from nothing.
//
// All kernels compute S = Q . K^T with the keys as the columns of the matrix instruction: a lane owns one key per block and
// its accumulator registers are query rows, so the sum over rows is an addition in the lane and only the few lanes that
// hold the same key are added up at the end.  No two workgroups write the same key: there are no atomics and the order of
// every sum is fixed.
#include "common.hpp"
#include "kernels.hpp"

#include <type_traits>

namespace fck {
namespace {

// keys of a sequence: its count, cut to what its table row (without a table: its row of the cache) holds
__device__ __forceinline__ int key_count(const KvAddr& a, const KvSeq& s)
{
    const int64_t cap = s.table ? (int64_t)a.block_table_stride * a.page_size : a.seqlen_k;
    const int n = max(s.len, 0);
    return n < cap ? n : (int)cap;
}

// K (and Q) tiles are staged in LDS as they lie in memory, rows of ROWB bytes, with the 16-byte chunk index XOR-swizzled by
// the row so that lanes reading one logical chunk of consecutive rows spread over the banks.
template <int CH>
__device__ __forceinline__ int chunk_swizzle(int row)
{
    if constexpr (CH >= 16)
        return row & 15;
    else if constexpr (CH == 8)
        return ((row & 7) + ((row >> 3) & 1)) & 7;
    else
        return (row ^ (row >> 2)) & (CH - 1);
}

// 8 consecutive elements of a staged row, as T: elements 8c .. 8c+7
template <typename T, bool kKv8, int CH>
__device__ __forceinline__ u32x4_t staged8(const char FCK_LDS* row_p, int row, int c)
{
    if constexpr (kKv8) {
        const u32x2_t v = *(const u32x2_t FCK_LDS*)(row_p + ((((c >> 1) ^ chunk_swizzle<CH>(row)) << 4) | ((c & 1) << 3)));
        return fp8x8_to_t<T>(u32x4_t{v[0], v[1], 0u, 0u});
    } else {
        return *(const u32x4_t FCK_LDS*)(row_p + ((c ^ chunk_swizzle<CH>(row)) << 4));
    }
}

// ---- few query rows: decode steps --------------------------------------------------------------------------------------------
//
// Bound by reading K once.  A wave owns NT tiles of 32 keys and streams them through an LDS buffer of its own (global -> LDS
// copies with the non-temporal hint, no workgroup barrier): a tile goes to registers as soon as it has landed and the next
// one is requested into the same buffer, so that small buffers leave room for many waves, each with a tile in flight.  The
// 16 MB query rows sit in registers as the A operand of v_mfma_f32_16x16x32.  One token of 16 sequences of up to 32768 keys
// (8 KV heads of 8 query heads, D 128, bf16): 126 us, 5.0 TB/s; the first version, through a tile shared by the workgroup
// behind barriers, 718 us.
template <int D, bool kKv8>
struct StepShape {
    static constexpr int ROWB = D * (kKv8 ? 1 : 2);
    static constexpr int CH = ROWB / 16;
    static constexpr int TILEB = 32 * ROWB;
    static constexpr int LD = TILEB / 1024;  // 1 KiB copies per tile
    static constexpr int KT = D / 32;
};

// requests the 32 keys from kb on, whose rows hold row_bytes of S::ROWB, into the calling wave's tile
template <typename S>
__device__ __forceinline__ void request_keys(const KeyWeightsArgs& a, const KvSeq& ks, bool uniform, int sk, int hkv, int row_bytes,
                                             char FCK_LDS* tile, int kb)
{
    const int lane = threadIdx.x & 63;
    int64_t row0 = ks.base_row + kb;
    if (uniform && ks.table) {
        const int pi = a.kv.page_shift >= 0 ? kb >> a.kv.page_shift : kb / a.kv.page_size;
        row0 = (int64_t)const_load(ks.table, pi) * a.kv.page_size + (kb - pi * a.kv.page_size);
    }
#pragma unroll
    for (int u = 0; u < S::LD; ++u) {
        const int off = u * 1024 + lane * 16;
        const int row = off / S::ROWB;
        const int chunk = (off % S::ROWB / 16) ^ chunk_swizzle<S::CH>(row);
        const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_address(tile + u * 1024));
        if (chunk * 16 >= row_bytes) {  // the stored row is shorter than D: these places were zeroed once
            FCK_LOAD_TO_LDS_MASKED();
            continue;
        }
        const int in = min(row, sk - 1 - kb);  // rows past the last key repeat it, and are not stored
        const int64_t cr = uniform ? row0 + in : kv_row(a.kv, ks, kb + in);
        load_to_lds_stream(dst, (const char*)a.k + (cr * a.hk + hkv) * row_bytes + chunk * 16);
    }
}

// zeroes the places of a tile that no request fills
template <typename S>
__device__ __forceinline__ void clear_missing(char FCK_LDS* tile, int row_bytes)
{
    if (row_bytes >= S::ROWB) return;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < S::LD; ++u) {
        const int off = u * 1024 + lane * 16;
        const int row = off / S::ROWB;
        if (((off % S::ROWB / 16) ^ chunk_swizzle<S::CH>(row)) * 16 >= row_bytes) *(u32x4_t FCK_LDS*)(tile + off) = u32x4_t{0u, 0u, 0u, 0u};
    }
}

template <typename T, int D, int MB, int NT, bool kMod, bool kKv8>
__global__ __launch_bounds__(256) void key_weights_step_kernel(const KeyWeightsArgs a)
{
    typedef StepShape<D, kKv8> S;
    typedef typename T::vec8 vec8;
    FCK_DYNAMIC_LDS(smem);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, kg = lane >> 4;
    char FCK_LDS* const tiles = (char FCK_LDS*)smem + wave * S::TILEB;
    float FCK_LDS* const before = (float FCK_LDS*)((char FCK_LDS*)smem + 4 * S::TILEB) + wave * NT * 32;

    const int g = a.hq / a.hk;
    // the sequence last: workgroups that run at the same time read neighbouring rows of one cache (136 us with the key range
    // last, 125 us so; a ragged batch of 16, up to 32768 keys, 8 KV heads of 128)
    const int ranges = (int)((a.cols + 4 * NT * 32 - 1) / (4 * NT * 32));
    const int hkv = blockIdx.x % a.hk;
    const int b = blockIdx.x / a.hk / ranges;
    const int64_t key0 = (int64_t)(blockIdx.x / a.hk % ranges) * (4 * NT * 32) + wave * (NT * 32);
    if (key0 >= a.cols) return;
    const KvSeq ks = kv_seq(a.kv, b);
    const int sk = __builtin_amdgcn_readfirstlane(key_count(a.kv, ks));
    const int64_t row_out = ((int64_t)b * a.hk + hkv) * a.cols;
    // tiles that hold keys with a column: what is requested is waited for before the wave ends
    const int64_t key1 = min((int64_t)sk, a.cols);
    const int n = key0 < key1 ? (int)min((int64_t)NT, (key1 - key0 + 31) / 32) : 0;

    const bool uniform = ks.table == nullptr || a.kv.page_size % 32 == 0;  // a tile never straddles a page
    const int row_bytes = a.d * (kKv8 ? 1 : 2);
    auto request = [&](int c) __attribute__((always_inline)) { request_keys<S>(a, ks, uniform, sk, hkv, row_bytes, tiles, (int)key0 + c * 32); };
    clear_missing<S>(tiles, row_bytes);
    if (n > 0) request(0);

    const int tok0 = __builtin_amdgcn_readfirstlane(a.seqstart_q ? a.seqstart_q[b] : b * a.sq);
    const int sq = __builtin_amdgcn_readfirstlane(a.seqstart_q ? a.seqstart_q[b + 1] - tok0 : a.sq);
    const MaskYX mk = make_mask(a.mask_type, a.window_left, a.window_right, sq, sk);
    const int R = sq * g;
    // rows r = i * g + head of the group; this lane's accumulator registers are rows mb * 16 + kg * 4 + v
    float lse2[MB][4];
    int lo[MB][4], hi[MB][4];
    ArithMod amod[MB][4];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int r = mb * 16 + kg * 4 + v;
            const int i = r < R ? r / g : 0, h = hkv * g + (r < R ? r % g : 0);
            // a row that does not exist, or that saw no key, adds nothing: lse2 = +inf gives exp2(-inf) = 0 for a finite score, and the
            // terms of scores that are not (a key with an infinite element) are left out by selection
            lse2[mb][v] = INFINITY;
            if (r < R) {
                const float l = a.lse[((int64_t)(a.seqstart_q ? 0 : b) * a.hq + h) * a.lse_sq + (a.seqstart_q ? tok0 : 0) + i];
                if (l != -INFINITY) lse2[mb][v] = l * kLog2e;
            }
            lo[mb][v] = mask_lo(mk, i);
            hi[mb][v] = r < R ? mask_hi(mk, i, sk) : 0;
            if constexpr (kMod) amod[mb][v].init(a.mod, b, h, i, sq, sk, a.mask_type, a.window_left, a.window_right);
        }
    // keys in [all_lo, all_hi) are visible to every row
    const int all_lo = sq > 0 ? mask_lo(mk, sq - 1) : 0, all_hi = sq > 0 ? mask_hi(mk, 0, sk) : 0;
    vec8 qf[MB][S::KT];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
        const int r = mb * 16 + l16;
        const uint16_t* qp = (const uint16_t*)a.q + ((int64_t)(tok0 + (r < R ? r / g : 0)) * a.hq + hkv * g + (r < R ? r % g : 0)) * a.d + kg * 8;
#pragma unroll
        for (int t = 0; t < S::KT; ++t) {
            u32x4_t v = {0u, 0u, 0u, 0u};
            if (r < R && t * 32 + kg * 8 < a.d) v = ldg16(qp + t * 32);
            qf[mb][t] = as_vec8<vec8>(v);
        }
    }
    // what is there already, read up front: a load inside the loop would wait for the copies in flight
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) {
        const int64_t key = key0 + j * 64 + lane;
        before[j * 64 + lane] = a.weights && key < sk && key < a.cols ? a.weights[row_out + key] : 0.f;
    }

    auto tile = [&](int c, float (&sum)[2]) __attribute__((always_inline)) {
        wait_vm<0>();
        FCK_WAVE_LDS_ORDER();
        u32x4_t kf[2][S::KT];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
            const int row = nb * 16 + l16;
#pragma unroll
            for (int t = 0; t < S::KT; ++t) kf[nb][t] = staged8<T, kKv8, S::CH>(tiles + row * S::ROWB, row, t * 4 + kg);
        }
        wait_lds();
        if (c + 1 < n) request(c + 1);
        f32x4_t s[2][MB];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
                s[nb][mb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int t = 0; t < S::KT; ++t) s[nb][mb] = T::mfma16(qf[mb][t], as_vec8<vec8>(kf[nb][t]), s[nb][mb]);
            }
        const int kb = (int)key0 + c * 32;
        const bool all = kb >= all_lo && min(kb + 32, sk) <= all_hi;  // uniform
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
            const int key = kb + nb * 16 + l16;
            float x = 0.f;
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    float e;
                    if constexpr (kMod)
                        e = fast_exp2(amod[mb][v].score(s[nb][mb][v], key) - lse2[mb][v]);
                    else
                        e = fast_exp2(__builtin_fmaf(s[nb][mb][v], a.scale_log2, -lse2[mb][v]));
                    x += (all || (key >= lo[mb][v] && key < hi[mb][v])) && lse2[mb][v] != INFINITY ? e : 0.f;
                }
            sum[nb] = quad16_sum(x);
        }
    };
#pragma unroll 1
    for (int p = 0; p < NT / 2; ++p) {
        const int64_t key = key0 + p * 64 + lane;  // lane = (tile parity, block, l16) of the pair's sums
        if (key0 + p * 64 >= a.cols) break;
        float even[2] = {0.f, 0.f}, odd[2] = {0.f, 0.f};
        if (2 * p < n) tile(2 * p, even);
        if (2 * p + 1 < n) tile(2 * p + 1, odd);
        const float x = kg == 0 ? even[0] : kg == 1 ? even[1] : kg == 2 ? odd[0] : odd[1];
        if (key < a.cols) a.out[row_out + key] = key < sk ? before[p * 64 + lane] + x : 0.f;
    }
}

// ---- observation windows -----------------------------------------------------------------------------------------------------
//
// More query rows than registers hold, few enough for LDS: still bound by reading K once.  All query rows of the KV head are
// staged once per workgroup; each of its 8 waves streams its own tiles of 32 keys as above and holds a tile in registers as
// the B operand of v_mfma_f32_32x32x16 while it walks the rows.
template <int D, bool kKv8>
struct WindowShape {
    static constexpr int ROWB = D * (kKv8 ? 1 : 2), CH = ROWB / 16;
    static constexpr int QB = D * 2, QCH = QB / 16;
    static constexpr int TILEB = 32 * ROWB;
    static constexpr int LD = TILEB / 1024;
    static constexpr int KT = D / 16;
    static constexpr int NT = 4;  // key tiles per wave
    static constexpr int KEYS = 8 * NT * 32;
    static constexpr int MAX_ROWS = 65536 / QB;
    static constexpr size_t lds(int rows32) { return 8 * TILEB + 8 * NT * 32 * 4 + (size_t)rows32 * (QB + 8) + rows32 / 32 * 4; }
};

// Tokens [first, end) see key `key`: the mask [mask_lo, mask_hi) of a token, solved for the token.  A row that does not exist,
// or whose lse is -inf, has token INT32_MAX, which no range holds: it adds nothing whatever its scores are.
struct Seen {
    int32_t first, end;
};
__device__ __forceinline__ Seen seen_by(const MaskYX& mk, int key)
{
    if (!mk.masking) return Seen{0, INT32_MAX};
    return Seen{key - mk.x + 1, (int32_t)min((int64_t)key + mk.y, (int64_t)INT32_MAX)};
}

// accumulates one 32-row block against NB 32-key blocks: acc[nb] += sum over the lane's rows of exp2(s * scale - lse2);
// lp / tp: lse2 and token of the lane's first row (rows (j >> 2) * 8 + (j & 3) from there), rs its number, key0 the lane's first key
template <typename T, bool kMod, int NB>
__device__ __forceinline__ void add_block(const KeyWeightsArgs& a, const MaskYX& mk, float (&acc)[NB], const f32x16_t (&s)[NB], const float FCK_LDS* lp,
                                          const int FCK_LDS* tp, bool all, int rs, int key0, int b, int h0, int g, int sq, int sk)
{
    if (!kMod && all) {
#pragma unroll
        for (int j4 = 0; j4 < 4; ++j4) {
            const f32x4_t l = *(const f32x4_t FCK_LDS*)(lp + j4 * 8);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float x = 0.f;
#pragma unroll
                for (int v = 0; v < 4; ++v) x += fast_exp2(__builtin_fmaf(s[nb][j4 * 4 + v], a.scale_log2, -l[v]));
                acc[nb] += x;
            }
        }
    } else {
        Seen seen[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) seen[nb] = seen_by(mk, key0 + nb * 32);
#pragma unroll
        for (int j4 = 0; j4 < 4; ++j4) {
            const f32x4_t l = *(const f32x4_t FCK_LDS*)(lp + j4 * 8);
            const u32x4_t tok = *(const u32x4_t FCK_LDS*)(tp + j4 * 8);
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int i = (int)tok[v];
                ArithMod amod;
                if constexpr (kMod) {
                    const bool row_ok = i != INT32_MAX;
                    amod.init(a.mod, b, h0 + (row_ok ? (rs + j4 * 8 + v) % g : 0), row_ok ? i : 0, sq, sk, a.mask_type, a.window_left, a.window_right);
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float e;
                    if constexpr (kMod)
                        e = fast_exp2(amod.score(s[nb][j4 * 4 + v], key0 + nb * 32) - l[v]);
                    else
                        e = fast_exp2(__builtin_fmaf(s[nb][j4 * 4 + v], a.scale_log2, -l[v]));
                    acc[nb] += i >= seen[nb].first && i < seen[nb].end ? e : 0.f;
                }
                if constexpr (kMod) __builtin_amdgcn_sched_barrier(0);  // one row at a time: their modifiers do not fit the registers together
            }
        }
    }
}

template <typename T, int D, bool kMod, bool kKv8>
__global__ __launch_bounds__(512) void key_weights_window_kernel(const KeyWeightsArgs a)
{
    typedef WindowShape<D, kKv8> S;
    typedef typename T::vec8 vec8;
    FCK_DYNAMIC_LDS(smem);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, half = lane >> 5;
    const int g = a.hq / a.hk;
    const int hkv = blockIdx.x % a.hk;
    const int ranges = (int)((a.cols + S::KEYS - 1) / S::KEYS);
    const int b = blockIdx.x / a.hk / ranges;
    const int64_t key0 = (int64_t)(blockIdx.x / a.hk % ranges) * S::KEYS + wave * (S::NT * 32);
    const int rows32 = (a.rows_max + 31) / 32 * 32;
    char FCK_LDS* const tile = (char FCK_LDS*)smem + wave * S::TILEB;
    float FCK_LDS* const before = (float FCK_LDS*)((char FCK_LDS*)smem + 8 * S::TILEB) + wave * S::NT * 32;
    char FCK_LDS* const qs = (char FCK_LDS*)smem + 8 * S::TILEB + 8 * S::NT * 32 * 4;
    float FCK_LDS* const row_lse = (float FCK_LDS*)(qs + rows32 * S::QB);
    int FCK_LDS* const row_tok = (int FCK_LDS*)(row_lse + rows32);
    int FCK_LDS* const block_full = row_tok + rows32;  // every row of the 32-row block adds something

    const KvSeq ks = kv_seq(a.kv, b);
    const int sk = __builtin_amdgcn_readfirstlane(key_count(a.kv, ks));
    const int tok0 = __builtin_amdgcn_readfirstlane(a.seqstart_q ? a.seqstart_q[b] : b * a.sq);
    const int sq = __builtin_amdgcn_readfirstlane(a.seqstart_q ? a.seqstart_q[b + 1] - tok0 : a.sq);
    const MaskYX mk = make_mask(a.mask_type, a.window_left, a.window_right, sq, sk);
    const int64_t row_out = ((int64_t)b * a.hk + hkv) * a.cols;
    const int64_t key1 = min((int64_t)sk, a.cols);  // tiles that hold keys with a column, as above
    const int n = key0 < key1 ? (int)min((int64_t)S::NT, (key1 - key0 + 31) / 32) : 0;
    const int R = min(sq * g, rows32);
    const int q_bytes = a.d * 2, k_bytes = a.d * (kKv8 ? 1 : 2);

    const bool uniform = ks.table == nullptr || a.kv.page_size % 32 == 0;  // a tile never straddles a page
    auto request = [&](int c) __attribute__((always_inline)) { request_keys<S>(a, ks, uniform, sk, hkv, k_bytes, tile, (int)key0 + c * 32); };
    clear_missing<S>(tile, k_bytes);
    if (n > 0) request(0);
#pragma unroll
    for (int j = 0; j < S::NT / 2; ++j) {
        const int64_t key = key0 + j * 64 + lane;
        before[j * 64 + lane] = a.weights && key < sk && key < a.cols ? a.weights[row_out + key] : 0.f;
    }
    // all query rows r = i * g + head of the group, through registers (they stay for the whole workgroup)
    for (int e = tid; e < rows32 * S::QCH; e += 512) {
        const int row = e / S::QCH, chunk = e % S::QCH;
        u32x4_t v = {0u, 0u, 0u, 0u};
        if (row < R && chunk * 16 < q_bytes)
            v = ldg16((const char*)a.q + ((int64_t)(tok0 + row / g) * a.hq + hkv * g + row % g) * q_bytes + chunk * 16);
        *(u32x4_t FCK_LDS*)(qs + row * S::QB + ((chunk ^ chunk_swizzle<S::QCH>(row)) << 4)) = v;
    }
    for (int row0 = wave * 64; row0 < rows32; row0 += 512) {  // whole waves: two blocks
        const int row = row0 + lane;
        float l = -INFINITY;
        if (row < R) l = a.lse[((int64_t)(a.seqstart_q ? 0 : b) * a.hq + hkv * g + row % g) * a.lse_sq + (a.seqstart_q ? tok0 : 0) + row / g];
        // a row that does not exist, or that saw no key, adds nothing
        const bool none = l == -INFINITY;
        const uint64_t nones = __builtin_amdgcn_ballot_w64(none);
        if (row < rows32) {
            row_lse[row] = none ? INFINITY : l * kLog2e;
            row_tok[row] = none ? INT32_MAX : row / g;
            if (l32 == 0) block_full[row / 32] = (uint32_t)(nones >> (half * 32)) == 0;
        }
    }
    __syncthreads();

    auto sum_tile = [&](int c) __attribute__((always_inline)) -> float {
        wait_vm<0>();
        FCK_WAVE_LDS_ORDER();
        u32x4_t kf[S::KT];
#pragma unroll
        for (int t = 0; t < S::KT; ++t) kf[t] = staged8<T, kKv8, S::CH>(tile + l32 * S::ROWB, l32, t * 2 + half);
        wait_lds();
        if (c + 1 < n) request(c + 1);
        const int kb = (int)key0 + c * 32;
        float acc[1] = {0.f};
        for (int rs = 0; rs < R; rs += 32) {
            const int i_first = rs / g, i_last = min(rs + 31, R - 1) / g;
            if (mask_hi(mk, i_last, sk) <= kb || mask_lo(mk, i_first) >= kb + 32) continue;
            f32x16_t s[1];
#pragma unroll
            for (int j = 0; j < 16; ++j) s[0][j] = 0.f;
#pragma unroll
            for (int t = 0; t < S::KT; ++t)
                s[0] = T::mfma32(as_vec8<vec8>(staged8<T, false, S::QCH>(qs + (rs + l32) * S::QB, rs + l32, t * 2 + half)), as_vec8<vec8>(kf[t]), s[0]);
            const bool all = __builtin_amdgcn_readfirstlane(block_full[rs / 32]) != 0 && mask_lo(mk, i_last) <= kb && mask_hi(mk, i_first, sk) >= min(kb + 32, sk);
            add_block<T, kMod, 1>(a, mk, acc, s, row_lse + rs + half * 4, row_tok + rs + half * 4, all, rs + half * 4, kb + l32, b, hkv * g, g, sq, sk);
        }
        return pair32_sum(acc[0]);
    };
#pragma unroll 1
    for (int p = 0; p < S::NT / 2; ++p) {
        const int64_t key = key0 + p * 64 + lane;
        if (key0 + p * 64 >= a.cols) break;
        float even = 0.f, odd = 0.f;
        if (2 * p < n) even = sum_tile(2 * p);
        if (2 * p + 1 < n) odd = sum_tile(2 * p + 1);
        if (key < a.cols) a.out[row_out + key] = key < sk ? before[p * 64 + lane] + (half == 0 ? even : odd) : 0.f;
    }
}

// ---- many query rows: prompts ------------------------------------------------------------------------------------------------
//
// Bound by the matrix product and one exponential per (row, key).  A workgroup of 8 waves owns KEYS = 4 NB 32 keys, four waves
// side by side with NB blocks of 32 keys each in registers as the B operand of v_mfma_f32_32x32x16 (two blocks, so that
// every Q fragment read from LDS feeds two instructions; one at head dim 256, where two do not fit the registers); the two
// wave rows take different rows of the queries that see the keys, SUB blocks of 32 per stage, which are staged through two
// LDS buffers by global -> LDS copies.  The partial sums of the wave rows are added up at the end.
//   The query tokens are cut into row_splits equal runs and a workgroup handles one run: the runs fill the chip when there
// are few keys, and under a causal mask they make the items equal (a run is either seen whole, or crossed by the diagonal,
// or skipped).  A run's sums go to a slice of the workspace, key_weights_sum_kernel adds the slices in order.
//   A prompt of 8192 tokens, 32 query heads, D 128, bf16, causal: 333 us, 830 TFLOP/s of visible pairs (without a mask
// 950 to 1036); the first version 2213 us.
template <int D, bool kKv8>
struct RowsShape {
    static constexpr int KW = 4, RW = 2;
    static constexpr int NB = D == 256 ? 1 : 2;
    static constexpr int SUB = D == 256 ? 2 : 4;
    static constexpr int KEYS = KW * NB * 32, ROWS = RW * SUB * 32;  // per workgroup, per stage
    static constexpr int QB = D * 2, QCH = QB / 16;                  // staged query row
    static constexpr int KB = D * (kKv8 ? 1 : 2), KCH = KB / 16;
    static constexpr int STAGEB = ROWS * QB;
    static constexpr int LDQ = STAGEB / 8192, LDK = KEYS * KB / 8192;  // copies per wave
    static constexpr int RPL = 1024 / QB;                              // query rows per copy
    static constexpr int KT = D / 16;
    static constexpr size_t lds = 2 * STAGEB + 2 * ROWS * 12 + RW * KEYS * 4 + 2 * (ROWS / 64) * 4;
    static_assert(KEYS * KB <= 2 * STAGEB && KEYS * KB % 8192 == 0 && STAGEB % 8192 == 0, "the key tile passes through the stage buffers");
    static_assert(ROWS <= 512, "one thread per staged row");
};

template <typename T, int D, bool kMod, bool kKv8>
__global__ __launch_bounds__(512) void key_weights_rows_kernel(const KeyWeightsArgs a)
{
    typedef RowsShape<D, kKv8> S;
    typedef typename T::vec8 vec8;
    FCK_DYNAMIC_LDS(smem);
    char FCK_LDS* const lds = (char FCK_LDS*)smem;  // two stages (or the key tile) | of their rows: lse, token, -lse / scale | sums | pairs of row blocks
    float FCK_LDS* const row_lse = (float FCK_LDS*)(lds + 2 * S::STAGEB);
    int FCK_LDS* const row_tok = (int FCK_LDS*)(row_lse + 2 * S::ROWS);
    float FCK_LDS* const row_init = (float FCK_LDS*)(row_tok + 2 * S::ROWS);
    float FCK_LDS* const sums = row_init + 2 * S::ROWS;
    int FCK_LDS* const pair_none = (int FCK_LDS*)(sums + S::RW * S::KEYS);  // some of the 64 rows adds nothing

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kw = wave % S::KW, rw = wave / S::KW;
    const int l32 = lane & 31, half = lane >> 5;
    const int g = a.hq / a.hk;
    // The key tiles are taken in row_splits parts, like the query tokens.  ids: KV head, tile of the part, (run, part), sequence,
    // with the pairs in order of decreasing run - part: under a causal mask the items whose rows see every key come first,
    // then those that the diagonal crosses, then the empty ones, so that the short items fill in behind the long ones.
    // Workgroups that run at the same time mostly read the same query rows, those of one KV head from one XCD's L2.
    const int tiles = (int)((a.cols + S::KEYS - 1) / S::KEYS);
    const int per_part = (tiles + a.row_splits - 1) / a.row_splits;
    int id = blockIdx.x;
    const int hkv = id % a.hk;
    id /= a.hk;
    const int in_part = id % per_part;
    id /= per_part;
    int pair_id = id % (a.row_splits * a.row_splits);
    const int b = id / (a.row_splits * a.row_splits);
    int ahead = a.row_splits - 1;  // run - part of the pair
    for (int n = 1; pair_id >= n; n = a.row_splits - (ahead < 0 ? -ahead : ahead)) {
        pair_id -= n;
        --ahead;
    }
    const int part = (ahead < 0 ? -ahead : 0) + pair_id, split = part + ahead;
    if (part * per_part + in_part >= tiles) return;
    const int64_t k0 = (int64_t)(part * per_part + in_part) * S::KEYS;

    const KvSeq ks = kv_seq(a.kv, b);
    const int sk = __builtin_amdgcn_readfirstlane(key_count(a.kv, ks));
    const int tok0 = __builtin_amdgcn_readfirstlane(a.seqstart_q ? a.seqstart_q[b] : b * a.sq);
    const int sq = __builtin_amdgcn_readfirstlane(a.seqstart_q ? a.seqstart_q[b + 1] - tok0 : a.sq);
    const MaskYX mk = make_mask(a.mask_type, a.window_left, a.window_right, sq, sk);
    const int q_bytes = a.d * 2, k_bytes = a.d * (kKv8 ? 1 : 2);
    const int64_t tok_bytes = (int64_t)a.hq * q_bytes;

    float acc[S::NB] = {};
    // tokens of the run whose range [mask_lo, mask_hi) meets the workgroup's keys: mask_hi and mask_lo grow with the token
    const int k_end = (int)min(k0 + S::KEYS, (int64_t)sk);
    const int run = (sq + a.row_splits - 1) / a.row_splits;
    int i_begin = min((int64_t)run * split, (int64_t)sq), i_end = k0 < sk ? (int)min((int64_t)run * (split + 1), (int64_t)sq) : 0;
    if (mk.masking) {
        i_begin = (int)max((int64_t)i_begin, k0 + 1 - mk.x);
        i_end = (int)min((int64_t)i_end, (int64_t)k_end - 1 + mk.y);
    }
    if (i_begin < i_end) {  // uniform
        const int kwave0 = (int)k0 + kw * S::NB * 32;
        u32x4_t kf[S::NB][S::KT];
        if (q_bytes < S::QB) {  // stored rows shorter than D: the places no copy fills
            for (int off = tid * 16; off < 2 * S::STAGEB; off += 512 * 16) {
                const int row = off / S::QB;
                if (((off % S::QB / 16) ^ chunk_swizzle<S::QCH>(row)) * 16 >= q_bytes) *(u32x4_t FCK_LDS*)(lds + off) = u32x4_t{0u, 0u, 0u, 0u};
            }
        }
#pragma unroll
        for (int u = 0; u < S::LDK; ++u) {
            const int off = (wave + 8 * u) * 1024 + lane * 16;
            const int row = off / S::KB;
            const int chunk = (off % S::KB / 16) ^ chunk_swizzle<S::KCH>(row);
            const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_address(lds + (wave + 8 * u) * 1024));
            if (chunk * 16 >= k_bytes) {
                FCK_LOAD_TO_LDS_MASKED();
                continue;
            }
            const int key = (int)min(k0 + row, (int64_t)sk - 1);  // keys past the end repeat the last one, and are not stored
            load_to_lds(dst, (const char*)a.k + (kv_row(a.kv, ks, key) * a.hk + hkv) * k_bytes + chunk * 16);
        }
        wait_vm<0>();
        __syncthreads();
#pragma unroll
        for (int nb = 0; nb < S::NB; ++nb) {
            const int row = kw * S::NB * 32 + nb * 32 + l32;
#pragma unroll
            for (int t = 0; t < S::KT; ++t) kf[nb][t] = staged8<T, kKv8, S::KCH>(lds + row * S::KB, row, t * 2 + half);
        }
        __syncthreads();

        // rows r = i * g + head of the group, from the first to the last token of the run that sees a key of the tile
        const int r_begin = i_begin * g, r_end = i_end * g;
        const int stages = (r_end - r_begin + S::ROWS - 1) / S::ROWS;
        // rows [vis_lo, vis_hi) see some of this wave's keys, rows [all_lo, all_hi) all of them
        int vis_lo = r_begin, vis_hi = kwave0 < sk ? r_end : 0, all_lo = r_begin, all_hi = r_end;
        if (mk.masking) {
            const int64_t ke = min(kwave0 + S::NB * 32, sk);
            vis_lo = (int)max((int64_t)vis_lo, ((int64_t)kwave0 + 1 - mk.x) * g);
            vis_hi = (int)min((int64_t)vis_hi, (ke - 1 + mk.y) * g);
            all_lo = (int)min(max((int64_t)all_lo, (ke - mk.x) * g), (int64_t)r_end);
            all_hi = (int)max(min((int64_t)all_hi, ((int64_t)kwave0 + mk.y) * g), (int64_t)r_begin);
        }
        const char* const q_first = (const char*)a.q + ((int64_t)(tok0 + i_begin) * a.hq + hkv * g) * q_bytes;
        const float* const lse_first = a.lse + ((int64_t)(a.seqstart_q ? 0 : b) * a.hq + hkv * g) * a.lse_sq + (a.seqstart_q ? tok0 : 0) + i_begin;
        // Copy u of a wave moves the rows (wave + 8 u) * RPL .. of a stage.  When the group size divides the distance 8 RPL
        // between two copies, the tokens of a copy follow from its number alone: the address is a uniform base plus an
        // offset that a lane computes once (dividing for every copy cost as much as a third of the exponentials).
        const int copy_row = wave * S::RPL + lane * 16 / S::QB;
        const int copy_chunk = (lane * 16 % S::QB / 16) ^ chunk_swizzle<S::QCH>(copy_row);  // 8 RPL is a multiple of the swizzle's period
        const bool strided = 8 * S::RPL % g == 0 && (int64_t)8 * S::RPL * tok_bytes < ((int64_t)1 << 31);
        const uint32_t copy_off = (uint32_t)(copy_row / g * (int)tok_bytes + copy_row % g * q_bytes + copy_chunk * 16);
        float lse_next = 0.f;
        int tok_next = 0;
        auto request = [&](int st) __attribute__((always_inline)) {
            const int at = st * S::ROWS;  // first row of the stage, from r_begin
            const bool fast = strided && at + S::ROWS <= r_end - r_begin;
            const char* const base = q_first + at / g * tok_bytes;
#pragma unroll
            for (int u = 0; u < S::LDQ; ++u) {
                const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_address(lds + (st & 1) * S::STAGEB + (wave + 8 * u) * 1024));
                if (copy_chunk * 16 >= q_bytes) {
                    FCK_LOAD_TO_LDS_MASKED();
                    continue;
                }
                if (fast) {
                    load_to_lds(dst, base + u * (8 * S::RPL / g) * tok_bytes, copy_off);
                } else {
                    const int r = min(at + copy_row + 8 * S::RPL * u, r_end - r_begin - 1);  // rows past the last repeat it, and are masked
                    load_to_lds(dst, q_first + r / g * tok_bytes + r % g * q_bytes + copy_chunk * 16);
                }
            }
            if (tid < S::ROWS) {
                const int r = min(at + tid, r_end - r_begin - 1);
                tok_next = at + tid < r_end - r_begin ? i_begin + r / g : INT32_MAX;
                lse_next = lse_first[r % g * a.lse_sq + r / g];
            }
        };
        auto publish = [&](int st) __attribute__((always_inline)) {
            if (tid < S::ROWS) {
                // a row that saw no key adds nothing: the pair of row blocks it lies in takes the path that selects by token
                const bool none = lse_next == -INFINITY;
                const float l = none ? INFINITY : lse_next * kLog2e;
                row_lse[(st & 1) * S::ROWS + tid] = l;
                row_init[(st & 1) * S::ROWS + tid] = -l / a.scale_log2;
                row_tok[(st & 1) * S::ROWS + tid] = none ? INT32_MAX : tok_next;
                const uint64_t nones = __builtin_amdgcn_ballot_w64(none);
                if (lane == 0) pair_none[(st & 1) * (S::ROWS / 64) + wave] = nones != 0;
            }
        };
        // The block pipeline of the tiles every row sees: while the matrix instructions of a block run, the exponentials of
        // the block before it (its scores in the other of two register sets) fill the vector ALU, two per matrix instruction
        // at head dim 128: 32 cycles of either.  The accumulators start at -lse / scale instead of 0 (a rounding of 2^-24 lse
        // per step of the product), so that no register holds an lse while a block waits and an exponential needs one multiply.
        f32x16_t s[2][S::NB];
        bool pending = false;  // s[1] waits for its exponentials
        auto exps = [&](int set, int e0, int n, float (&part)[S::NB]) __attribute__((always_inline)) {
#pragma unroll
            for (int e = e0; e < e0 + n; ++e) {
                const int j = e / S::NB, nb = e % S::NB;
                part[nb] += fast_exp2(s[set][nb][j] * a.scale_log2);
            }
        };
        auto drain = [&]() __attribute__((always_inline)) {
            float part[S::NB] = {};
            exps(1, 0, 16 * S::NB, part);
#pragma unroll
            for (int nb = 0; nb < S::NB; ++nb) acc[nb] += part[nb];
            pending = false;
        };
        auto block = [&](int set, const char FCK_LDS* q0, const float FCK_LDS* lp, auto kAll, auto kExps) __attribute__((always_inline)) {
            constexpr int kPer = 16 / S::KT;  // exponentials per matrix instruction
            constexpr int kAhead = S::NB == 2 ? 4 : 6;  // steps between an LDS read of Q and its use
            f32x16_t init;
#pragma unroll
            for (int j = 0; j < 16; ++j) init[j] = 0.f;
            float part[S::NB] = {};
            u32x4_t qf[kAhead + 1];
            auto fetch = [&](int t) __attribute__((always_inline)) { return staged8<T, false, S::QCH>(q0, l32, t * 2 + half); };
            if constexpr (decltype(kAll)::value) {
#pragma unroll
                for (int j4 = 0; j4 < 4; ++j4) {
                    const f32x4_t l = *(const f32x4_t FCK_LDS*)(lp + j4 * 8);
#pragma unroll
                    for (int v = 0; v < 4; ++v) init[j4 * 4 + v] = l[v];
                }
            }
#pragma unroll
            for (int t = 0; t < kAhead && t < S::KT; ++t) qf[t] = fetch(t);
#pragma unroll
            for (int t = 0; t < S::KT; ++t) {
                if (t + kAhead < S::KT) qf[(t + kAhead) % (kAhead + 1)] = fetch(t + kAhead);
#pragma unroll
                for (int nb = 0; nb < S::NB; ++nb) {
                    s[set][nb] = T::mfma32(as_vec8<vec8>(qf[t % (kAhead + 1)]), as_vec8<vec8>(kf[nb][t]), t == 0 ? init : s[set][nb]);
                    if constexpr (decltype(kExps)::value) {
                        exps(set ^ 1, (t * S::NB + nb) * kPer, kPer, part);
                        // without a use here the exponentials are sunk behind the last matrix instruction
#pragma unroll
                        for (int p = 0; p < S::NB; ++p) FCK_PIN_VGPR(part[p]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if constexpr (decltype(kExps)::value) {
#pragma unroll
                for (int nb = 0; nb < S::NB; ++nb) acc[nb] += part[nb];
            }
        };
        request(0);
        for (int st = 0; st < stages; ++st) {
            wait_vm<0>();
            publish(st);
            __syncthreads();
            if (st + 1 < stages) request(st + 1);
            uint32_t none = 0;  // bit p: pair p of this wave's rows
#pragma unroll
            for (int p = 0; p < S::SUB / 2; ++p) none |= (uint32_t)pair_none[(st & 1) * (S::ROWS / 64) + rw * (S::SUB / 2) + p] << p;
            none = __builtin_amdgcn_readfirstlane(none);
#pragma unroll 1
            for (int pair = 0; pair < S::SUB / 2; ++pair) {
                const int rl = (rw * S::SUB + pair * 2) * 32;  // this wave's rows in the stage, 64 at a time
                const int rs = r_begin + st * S::ROWS + rl;
                if (rs >= vis_hi || rs + 64 <= vis_lo) continue;
                const char FCK_LDS* q0 = lds + (st & 1) * S::STAGEB + (rl + l32) * S::QB;
                const float FCK_LDS* lp = row_lse + (st & 1) * S::ROWS + rl + half * 4;
                const float FCK_LDS* ip = row_init + (st & 1) * S::ROWS + rl + half * 4;
                const int FCK_LDS* tp = row_tok + (st & 1) * S::ROWS + rl + half * 4;
                if (!kMod && (none >> pair & 1) == 0 && rs >= all_lo && rs + 64 <= all_hi) {
                    if (pending)
                        block(0, q0, ip, std::true_type{}, std::true_type{});
                    else
                        block(0, q0, ip, std::true_type{}, std::false_type{});
                    block(1, q0 + 32 * S::QB, ip + 32, std::true_type{}, std::true_type{});
                    pending = true;
                } else {
                    if (pending) drain();
#pragma unroll 1
                    for (int sub = 0; sub < 2; ++sub) {
                        block(0, q0 + sub * 32 * S::QB, lp + sub * 32, std::false_type{}, std::false_type{});
                        add_block<T, kMod, S::NB>(a, mk, acc, s[0], lp + sub * 32, tp + sub * 32, false, rs + sub * 32 + half * 4, kwave0 + l32, b, hkv * g, g, sq, sk);
                    }
                }
            }
        }
        if (pending) drain();
    }
#pragma unroll
    for (int nb = 0; nb < S::NB; ++nb) {
        const float x = pair32_sum(acc[nb]);
        if (half == 0) sums[rw * S::KEYS + kw * S::NB * 32 + nb * 32 + l32] = x;
    }
    __syncthreads();
    const int64_t key = k0 + tid;
    if (tid < S::KEYS && key < a.cols) {
        const int64_t at = ((int64_t)b * a.hk + hkv) * a.cols + key;
        float x = 0.f;
        if (key < sk) {
#pragma unroll
            for (int w = 0; w < S::RW; ++w) x += sums[w * S::KEYS + tid];
        }
        if (a.row_splits > 1)
            a.partial[(int64_t)split * a.batch * a.hk * a.cols + at] = x;
        else
            a.out[at] = key < sk && a.weights ? a.weights[at] + x : x;
    }
}

// out = weights + the slices of the workspace, in order
__global__ __launch_bounds__(256) void key_weights_sum_kernel(const KeyWeightsArgs a)
{
    const int64_t per = (int64_t)a.batch * a.hk * a.cols;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= per) return;
    float x = 0.f;
    for (int s = 0; s < a.row_splits; ++s) x += a.partial[s * per + at];
    if (a.weights) {
        const int b = (int)(at / (a.hk * a.cols));
        if (at % a.cols < key_count(a.kv, kv_seq(a.kv, b))) x += a.weights[at];
    }
    a.out[at] = x;
}

template <typename T, int D, int MB, int NT>
hipError_t launch_step(const KeyWeightsArgs& a, hipStream_t st)
{
    const int64_t grid = (a.cols + 4 * NT * 32 - 1) / (4 * NT * 32) * a.batch * a.hk;
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    const dim3 blocks((unsigned)grid), threads(256);
    constexpr size_t extra = 4 * NT * 32 * 4;
    if (a.kv8) return launch_with_lds<key_weights_step_kernel<T, D, MB, NT, true, true>>(blocks, threads, 4 * StepShape<D, true>::TILEB + extra, st, a);
    if (a.mod.active())
        return launch_with_lds<key_weights_step_kernel<T, D, MB, NT, true, false>>(blocks, threads, 4 * StepShape<D, false>::TILEB + extra, st, a);
    return launch_with_lds<key_weights_step_kernel<T, D, MB, NT, false, false>>(blocks, threads, 4 * StepShape<D, false>::TILEB + extra, st, a);
}

template <typename T, int D>
hipError_t launch_window(const KeyWeightsArgs& a, hipStream_t st)
{
    constexpr int KEYS = WindowShape<D, false>::KEYS;
    const int64_t grid = (a.cols + KEYS - 1) / KEYS * a.batch * a.hk;
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    const dim3 blocks((unsigned)grid), threads(512);
    const int rows32 = (a.rows_max + 31) / 32 * 32;
    // the most a call can ask for is what the kernel is opted in for (once per kernel and device)
    if (a.kv8)
        return launch_with_lds<key_weights_window_kernel<T, D, true, true>>(blocks, threads, WindowShape<D, true>::lds(rows32), st, a, WindowShape<D, true>::lds(WindowShape<D, true>::MAX_ROWS));
    if (a.mod.active())
        return launch_with_lds<key_weights_window_kernel<T, D, true, false>>(blocks, threads, WindowShape<D, false>::lds(rows32), st, a, WindowShape<D, false>::lds(WindowShape<D, false>::MAX_ROWS));
    return launch_with_lds<key_weights_window_kernel<T, D, false, false>>(blocks, threads, WindowShape<D, false>::lds(rows32), st, a, WindowShape<D, false>::lds(WindowShape<D, false>::MAX_ROWS));
}

template <typename T, int D>
hipError_t launch_rows(const KeyWeightsArgs& a, hipStream_t st)
{
    constexpr int KEYS = RowsShape<D, false>::KEYS;
    const int64_t tiles = (a.cols + KEYS - 1) / KEYS;
    const int64_t grid = (tiles + a.row_splits - 1) / a.row_splits * a.row_splits * a.row_splits * a.batch * a.hk;
    const int64_t sum_grid = ((int64_t)a.batch * a.hk * a.cols + 255) / 256;
    if (grid > INT32_MAX || sum_grid > INT32_MAX) return hipErrorInvalidValue;
    const dim3 blocks((unsigned)grid), threads(512);
    hipError_t e;
    if (a.kv8)
        e = launch_with_lds<key_weights_rows_kernel<T, D, true, true>>(blocks, threads, RowsShape<D, true>::lds, st, a);
    else if (a.mod.active())
        e = launch_with_lds<key_weights_rows_kernel<T, D, true, false>>(blocks, threads, RowsShape<D, false>::lds, st, a);
    else
        e = launch_with_lds<key_weights_rows_kernel<T, D, false, false>>(blocks, threads, RowsShape<D, false>::lds, st, a);
    if (e != hipSuccess || a.row_splits == 1) return e;
    hipLaunchKernelGGL(key_weights_sum_kernel, dim3((unsigned)sum_grid), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <typename T, int D>
hipError_t launch_d(const KeyWeightsArgs& a, hipStream_t st)
{
    if (a.rows_max <= 32) {
        // 8 tiles a wave when that still gives every CU two workgroups
        const bool many = (a.cols + 1023) / 1024 * a.batch * a.hk >= 2 * (int64_t)a.num_cu;
        if (a.rows_max <= 16) return many ? launch_step<T, D, 1, 8>(a, st) : launch_step<T, D, 1, 2>(a, st);
        return many ? launch_step<T, D, 2, 8>(a, st) : launch_step<T, D, 2, 2>(a, st);
    }
    // at head dim 256 the key buffers of the 8 waves leave no room for the rows
    if constexpr (D <= 128)
        if (a.rows_max <= WindowShape<D, false>::MAX_ROWS) return launch_window<T, D>(a, st);
    return launch_rows<T, D>(a, st);
}

}  // namespace

int key_weights_row_splits(int d, int64_t batch, int64_t hk, int64_t g, int64_t sq, int64_t cols, bool masked, int num_cu)
{
    if (sq * g <= 32 || (d <= 128 && sq * g * d * 2 <= 65536)) return 1;  // the kernels that hold all rows
    const int64_t keys = d == 256 ? 128 : 256;
    const int64_t items = (cols + keys - 1) / keys * batch * hk;
    // One item per CU, two under a mask, which makes them unequal (a causal prompt of 8192 tokens, 32 / 8 heads of 128: 485,
    // 338, 388 and 346 us with 1, 2, 4 and 8 runs; without a mask and with 8 heads: 135, 141, 151 and 164 us); but runs of 4
    // stages of 256 rows at least, since a run starts with a round trip for its keys.
    const int64_t want = ((masked ? 2 : 1) * (int64_t)num_cu + items - 1) / items, most = sq * g / 1024;
    const int64_t n = want < most ? want : most;
    return (int)(n < 1 ? 1 : n > 16 ? 16 : n);
}

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
