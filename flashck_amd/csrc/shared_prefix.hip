// Decode attention of a batch whose sequences share prefixes (gfx950).
//
// The sequences [c_g, c_{g+1}) of group g begin with the same P_g tokens.  Softmax attention over a union of disjoint key
// sets is the merge of the attentions over each of them,
//   LSE = log(sum_s exp(LSE_s)),  O = sum_s exp(LSE_s - LSE) O_s,
// so the keys of a prefix are attended to by the query rows of the whole group at once (they are read once, through the
// pages of the group's first sequence) and the keys behind it by the rows of each sequence alone.  One launch does both,
// a second one merges the partial results.
//
// Work decomposition
//   An item = a tile of packed query rows (token, head of the KV head's group) x one split of a key range: of a prefix with
//   the rows of its group, or of a sequence's own keys with the rows of that sequence.  Which keys a row sees is a range
//   [lo, hi) of its own (its sequence's length and mask decide), so an item never has to know where its rows come from
//   after it has set them up.
//   Prefix items come first (they are the long ones); those that stream the same keys get ids congruent modulo 8, i.e. one
//   XCD and one L2.  Groups take equally many row tiles each when the caller bounds their size; otherwise the tiles of all
//   groups are numbered in one row, tile floor(first row / BM) + g being the first of group g: ceil(x - y) <= floor(x) -
//   floor(y) + 1, so every group has the tiles it needs, and there is one idle tile per group at most.
//   Every slot of every row is written (an empty one as lse = -inf), so the merge reads no lengths and no groups.
//
// What bounds it: a small group reads its keys (32 sequences on 4096 shared and up to 1024 own keys, 8 KV heads of 4 query
// heads, D 128, bf16: 22 + 4 us, 3.1 TB/s), a large one multiplies (64 sequences x 8 heads on 32768 keys: 115 + 8 us,
// 600 TFLOP/s: two products a tile with the softmax of 128 rows between them, and two waves per SIMD to overlap the two).
#include "common.hpp"
#include "kernels.hpp"

namespace fck {
namespace {

struct SharedGroup {
    int first, count, prefix;
};

__device__ __forceinline__ int shared_len(const SharedPrefixArgs& a, int b)
{
    const int64_t cap = (int64_t)a.block_table_stride * a.page_size;
    const int n = max(a.seqlen_k[b], 0);
    return n < cap ? n : (int)cap;
}

// sequences [first, first + count) of group g share their first `prefix` tokens (never more than the first of them has)
__device__ __forceinline__ SharedGroup shared_group(const SharedPrefixArgs& a, int g)
{
    SharedGroup s;
    s.first = a.cu_groups ? min(max(a.cu_groups[g], 0), a.batch) : 0;
    const int end = a.cu_groups ? min(max(a.cu_groups[g + 1], s.first), a.batch) : a.batch;
    s.count = min(end - s.first, a.max_group);
    s.prefix = s.count > 0 ? min(max(a.prefix_lens[g], 0), shared_len(a, s.first)) : 0;
    return s;
}

// number of entries of the non-decreasing starts[0..n] that are <= x, minus one: the interval x lies in
__device__ __forceinline__ int interval_of(const int32_t* starts, int n, int x)
{
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (starts[mid] <= x)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// first key of sequence b that is not part of its group's prefix
__device__ __forceinline__ int own_begin(const SharedPrefixArgs& a, int b)
{
    const SharedGroup s = shared_group(a, a.cu_groups ? interval_of(a.cu_groups, a.groups, b) : 0);
    return b >= s.first && b < s.first + s.count ? s.prefix : 0;
}

// first row tile of group i when the tiles of all groups are numbered in one row; g packed rows per query token
template <int BM>
__device__ __forceinline__ int first_tile(const SharedPrefixArgs& a, int i, int g)
{
    const int b = a.cu_groups ? min(max(a.cu_groups[i], 0), a.batch) : 0;
    return (a.seqstart_q ? a.seqstart_q[b] : b * a.sq) * g / BM + i;
}

// the last group whose first tile is at or before t
template <int BM>
__device__ __forceinline__ int group_of_tile(const SharedPrefixArgs& a, int t, int g)
{
    int lo = 0, hi = a.groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first_tile<BM>(a, mid, g) <= t)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

template <int D, int MB>
struct SharedShape {
    static constexpr int TK = D == 256 ? 32 : 64;  // keys per tile
    static constexpr int BM = 64 * MB;             // query rows per workgroup, 16 MB per wave
    static constexpr int NBK = TK / 16;            // 16-key blocks per tile
    static constexpr int KT = D / 32;              // MFMA k-steps of the QK product
    static constexpr int DB = D / 16;              // 16-column blocks of the output
    static constexpr int CH = D / 8;               // 16-byte chunks per staged row
    static constexpr int ROWB = D * 2;
    static constexpr int TILEB = TK * ROWB;
    static constexpr int LD = TK * CH / 256;  // chunks per thread and operand
};

// waves per SIMD (= workgroups per CU) the registers leave
template <int D, int MB>
constexpr int kSharedWaves = MB == 2 || D == 256 ? 2 : 3;

template <int D>
__device__ __forceinline__ int shared_v_swizzle(int key)
{
    return ((key & 7) << 1) & (D / 8 - 1);
}

// 4 waves of 16 MB rows.  A K/V tile goes through registers into one LDS buffer that all waves read; the next tile is in
// flight in the registers meanwhile.  One buffer and not two: three small workgroups per CU hide the latencies of short items
// better than two large ones.
// MB = 2 (groups of more than 128 rows, head dim <= 128): every fragment read from LDS feeds two matrix instructions, which
// is what bounds the product of a large group with its prefix.
// kUniform: pages are a multiple of the key tile.  kMod: ALiBi / soft cap.  kPad: stored head dims smaller than D (missing
// chunks are zeros).  kKv8: e4m3 caches, widened to T on their way into LDS; always with kMod.
template <typename T, int D, int MB, bool kUniform, bool kMod, bool kPad, bool kKv8>
__global__ __launch_bounds__(256, (kSharedWaves<D, MB>)) void shared_prefix_kernel(const SharedPrefixArgs a)
{
    typedef SharedShape<D, MB> S;
    typedef typename T::vec8 vec8;
    FCK_DYNAMIC_LDS(smem);
    char FCK_LDS* const lds = (char FCK_LDS*)smem;  // K | V | visible range
    int FCK_LDS* const range = (int FCK_LDS*)(lds + 2 * S::TILEB);

    const int dq = kPad ? a.d : D, dvs = kPad ? a.dv : D;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, kg = lane >> 4;
    const int g = a.hq / a.hk;

    // ---- the item (uniform) ----------------------------------------------------------------------------------------------
    int id = blockIdx.x;
    const bool prefix = id < a.prefix_items;
    int hkv, split, ns, slot, mt, leader, key_lo, key_hi, tok0, tok1;
    if (prefix) {
        constexpr int kXcd = 8;
        const int s = id / kXcd, per = max(a.prefix_tiles, 1);
        mt = s % per;
        int stream = s / per * kXcd + id % kXcd;
        if (a.prefix_tiles > 0) {
            if (stream >= a.groups * a.ns_prefix * a.hk) return;
        } else {
            const int combos = a.ns_prefix * a.hk;
            const int group = group_of_tile<S::BM>(a, id / combos, g);
            mt = id / combos - first_tile<S::BM>(a, group, g);
            if (mt < 0) return;  // rows of sequences before the first group
            stream = group * combos + id % combos;
        }
        hkv = stream % a.hk;
        split = slot = stream / a.hk % a.ns_prefix;
        ns = a.ns_prefix;
        const SharedGroup sg = shared_group(a, stream / (a.hk * a.ns_prefix));
        leader = sg.first;
        key_lo = 0;
        key_hi = sg.prefix;
        if (key_hi <= 0) return;  // the own items of its sequences write these slots
        tok0 = a.seqstart_q ? a.seqstart_q[sg.first] : sg.first * a.sq;
        tok1 = a.seqstart_q ? a.seqstart_q[sg.first + sg.count] : (sg.first + sg.count) * a.sq;
    } else {
        id -= a.prefix_items;
        hkv = id % a.hk;
        id /= a.hk;
        split = id % a.ns_own;
        id /= a.ns_own;
        mt = id % a.own_tiles;
        const int b = leader = id / a.own_tiles;
        ns = a.ns_own;
        slot = a.ns_prefix + split;
        key_lo = own_begin(a, b);
        key_hi = max(shared_len(a, b), key_lo);
        tok0 = a.seqstart_q ? a.seqstart_q[b] : b * a.sq;
        tok1 = a.seqstart_q ? a.seqstart_q[b + 1] : tok0 + a.sq;
    }
    const int64_t R = (int64_t)(tok1 - tok0) * g;
    const int64_t r0 = (int64_t)mt * S::BM;
    if (r0 >= R) return;
    // A split is an equal part of the keys there are, in whole tiles, and no smaller than the caller's least chunk (which leaves
    // the last splits of a short range empty).  Parts sized from host bounds alone put a range beyond its bound into the last
    // split, and everything into the first when the bound is loose: 32 sequences on 4096 shared keys with bounds of 32768 took
    // 96 us (32 us so; with exact bounds 25 us either way).
    const int base = key_lo / S::TK * S::TK;
    const int64_t part = ((int64_t)key_hi - base + ns - 1) / ns;
    const int64_t per = max((int64_t)(prefix ? a.prefix_chunk : a.own_chunk), (part + 63) / 64 * 64);
    const int k0 = (int)min(max((int64_t)key_lo, base + per * split), (int64_t)key_hi);
    const int k1 = split == ns - 1 ? key_hi : (int)min((int64_t)key_hi, base + per * (split + 1));

    const bool wave_rows = r0 + wave * 16 * MB < R;  // uniform per wave

    // ---- this lane's rows, one per 16-row block -----------------------------------------------------------------------------
    bool row_ok[MB];
    int tok[MB], h[MB], lo[MB], hi[MB];
    int64_t wofs[MB];  // places of the rows' partial results
    ArithMod amod[MB];
    const int slots = a.ns_prefix + a.ns_own;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
        const int64_t r = r0 + (wave * MB + mb) * 16 + l16;
        row_ok[mb] = r < R;
        tok[mb] = tok0 + (row_ok[mb] ? (int)(r / g) : 0);
        h[mb] = hkv * g + (row_ok[mb] ? (int)(r % g) : 0);
        const int b = !prefix ? leader : a.seqstart_q ? interval_of(a.seqstart_q, a.batch, tok[mb]) : tok[mb] / a.sq;
        const int first_tok = a.seqstart_q ? a.seqstart_q[b] : b * a.sq;
        const int sq_b = a.seqstart_q ? a.seqstart_q[b + 1] - first_tok : a.sq;
        const int i = tok[mb] - first_tok;
        const int sk_b = shared_len(a, b);
        const MaskYX mk = make_mask(a.mask_type, a.window_left, a.window_right, sq_b, sk_b);
        lo[mb] = row_ok[mb] ? max(mask_lo(mk, i), k0) : 0;
        hi[mb] = row_ok[mb] ? min(mask_hi(mk, i, sk_b), k1) : 0;
        if constexpr (kMod) amod[mb].init(a.mod, b, h[mb], i, sq_b, sk_b, a.mask_type, a.window_left, a.window_right);
        const int64_t head = (int64_t)(a.seqstart_q ? 0 : b) * a.hq + h[mb];
        wofs[mb] = (head * slots + slot) * a.shape_sq + (a.seqstart_q ? tok[mb] : i);
        // a sequence without a shared prefix has no prefix item
        if (!prefix && split == 0 && key_lo == 0 && row_ok[mb] && kg == 0)
            for (int e = 0; e < a.ns_prefix; ++e) a.lse_acc[wofs[mb] - (int64_t)(slot - e) * a.shape_sq] = -INFINITY;
    }
    // Keys the item walks.  A mask can leave out whole tiles at either end; where it can leave out many (a window on the
    // left, or a diagonal that does not end at the last key) the range that any row of the workgroup sees is found first.
    int vis_lo = k0, vis_hi = k1;
    if (a.mask_type != 0 && (a.window_left >= 0 || a.mask_type == 1)) {
        if (tid == 0) {
            range[0] = INT32_MAX;
            range[1] = 0;
        }
        __syncthreads();
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
            if (lo[mb] < hi[mb] && kg == 0) {
                atomicMin((int*)&range[0], lo[mb]);
                atomicMin((int*)&range[1], -hi[mb]);
            }
        __syncthreads();
        vis_lo = range[0];
        vis_hi = -range[1];
    }
    if (vis_lo >= vis_hi) {  // an empty split, or one that every row's mask leaves out
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
            if (row_ok[mb] && kg == 0) a.lse_acc[wofs[mb]] = -INFINITY;
        return;
    }
    const int t_begin = vis_lo / S::TK;
    const int n = (vis_hi + S::TK - 1) / S::TK - t_begin;

    // ---- K/V tiles ----------------------------------------------------------------------------------------------------------
    const int32_t* table = a.block_table + (int64_t)leader * a.block_table_stride;
    auto page_of = [&](int key) { return a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size; };
    auto cache_row = [&](int key) -> int64_t {
        const int pi = page_of(key);
        return (int64_t)table[pi] * a.page_size + (key - pi * a.page_size);
    };
    constexpr int kElem = kKv8 ? 1 : 2;
    auto fetch = [&](const void* base_p, int64_t row, int chunk, int dim) -> u32x4_t {
        if (kPad && chunk * 8 >= dim) return u32x4_t{0u, 0u, 0u, 0u};
        const char* p = (const char*)base_p + ((row * a.hk + hkv) * dim + chunk * 8) * kElem;
        if constexpr (kKv8) {
            const u32x2_t v = *reinterpret_cast<const u32x2_t*>(p);
            return u32x4_t{v[0], v[1], 0u, 0u};
        } else {
            // own keys have one reader; with the non-temporal hint they leave the prefix in the L2s (the group of 512 rows over
            // 32768 keys: 127 us without, 117 us with the hint)
            return prefix ? ldg16(p) : ldg16_stream(p);
        }
    };
    auto staged = [](u32x4_t v) -> u32x4_t {
        if constexpr (kKv8)
            return fp8x8_to_t<T>(v);
        else
            return v;
    };
    u32x4_t kreg[S::LD], vreg[S::LD];
    auto load_tile = [&](int c) {
        const int kb = (t_begin + c) * S::TK;
        int64_t row0 = 0;
        if constexpr (kUniform) row0 = cache_row(kb);
#pragma unroll
        for (int u = 0; u < S::LD; ++u) {
            const int row = (u * 256 + tid) / S::CH, chunk = (u * 256 + tid) % S::CH;
            // Rows outside the walked keys repeat the first or last of them: their scores are masked, but a probability of 0 times
            // an infinite or NaN value is NaN, so a key that no row of the workgroup sees must not be read either.
            const int key = min(max(kb + row, vis_lo), vis_hi - 1);
            const int64_t cr = kUniform ? row0 + (key - kb) : cache_row(key);
            kreg[u] = fetch(a.k, cr, chunk, dq);
            vreg[u] = fetch(a.v, cr, chunk, dvs);
        }
    };
    auto store_tile = [&]() {
#pragma unroll
        for (int u = 0; u < S::LD; ++u) {
            const int row = (u * 256 + tid) / S::CH, chunk = (u * 256 + tid) % S::CH;
            *(u32x4_t FCK_LDS*)(lds + row * S::ROWB + ((chunk ^ (row & 7)) << 4)) = staged(kreg[u]);
            *(u32x4_t FCK_LDS*)(lds + S::TILEB + row * S::ROWB + ((chunk ^ shared_v_swizzle<D>(row)) << 4)) = staged(vreg[u]);
        }
    };

    load_tile(0);
    vec8 qf[MB][S::KT];
    float m_run[MB], l_run[MB];
    f32x4_t oacc[MB][S::DB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
        const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + ((int64_t)tok[mb] * a.hq + h[mb]) * dq + kg * 8;
#pragma unroll
        for (int t = 0; t < S::KT; ++t) {
            u32x4_t v = {0u, 0u, 0u, 0u};
            if (row_ok[mb] && (!kPad || t * 32 + kg * 8 < dq)) v = ldg16(qp + t * 32);
            qf[mb][t] = as_vec8<vec8>(v);
        }
        m_run[mb] = -INFINITY;
        l_run[mb] = 0.f;
#pragma unroll
        for (int db = 0; db < S::DB; ++db) oacc[mb][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    const int tr_key = kg * 4 + (l16 >> 2);
    const int tr_sw = shared_v_swizzle<D>(tr_key);
    const char FCK_LDS* const kt = lds + l16 * S::ROWB;
    const char FCK_LDS* const vt = lds + S::TILEB + tr_key * S::ROWB + ((l16 & 2) << 3) + ((l16 & 1) << 3);
    auto compute = [&](int c) {
        const int kb = (t_begin + c) * S::TK;
        // S^T[key][row] = K . Q^T
        f32x4_t s[MB][S::NBK];
#pragma unroll
        for (int nb = 0; nb < S::NBK; ++nb) {
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) s[mb][nb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < S::KT; ++t) {
                const u32x4_t kf = *(const u32x4_t FCK_LDS*)(kt + nb * 16 * S::ROWB + (((t * 4 + kg) ^ (l16 & 7)) << 4));
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) s[mb][nb] = T::mfma16(as_vec8<vec8>(kf), qf[mb][t], s[mb][nb]);
            }
        }
        uint32_t pk[MB][2 * S::NBK];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
            // scores stay raw and the scale goes into the exponent's fused multiply-add; modified scores are in the log2 domain
            const float scale = kMod ? 1.f : a.scale_log2;
            if constexpr (kMod) {
#pragma unroll
                for (int nb = 0; nb < S::NBK; ++nb)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[mb][nb][j] = amod[mb].score(s[mb][nb][j], kb + nb * 16 + kg * 4 + j);
            }
            // a row that does not exist (lo = hi = 0) computes along on zeros
            if (__builtin_amdgcn_ballot_w64(row_ok[mb] && (lo[mb] > kb || hi[mb] < kb + S::TK)) != 0) {
#pragma unroll
                for (int nb = 0; nb < S::NBK; ++nb)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int key = kb + nb * 16 + kg * 4 + j;
                        s[mb][nb][j] = key >= lo[mb] && key < hi[mb] ? s[mb][nb][j] : -INFINITY;
                    }
            }
            float tmax = -INFINITY;
#pragma unroll
            for (int nb = 0; nb < S::NBK; ++nb)
#pragma unroll
                for (int j = 0; j < 4; ++j) tmax = fmaxf(tmax, s[mb][nb][j]);
            tmax = quad16_max(tmax) * scale;  // scale > 0
            // The reference of the exponentials moves only when some row outgrows it by 2^8: softmax is shift invariant, so an
            // older one is exact (a group of 512 rows over 32768 keys: 127 us with a reference that follows, 117 us so).
            constexpr float kLazy = 8.f;
            float alpha = 1.f;
            if (__builtin_amdgcn_ballot_w64(tmax > m_run[mb] + kLazy) != 0) {
                const float m_new = fmaxf(m_run[mb], tmax);
                alpha = fast_exp2(m_run[mb] - (m_new == -INFINITY ? 0.f : m_new));
                m_run[mb] = m_new;
            }
            const float m_use = m_run[mb] == -INFINITY ? 0.f : m_run[mb];
            float psum = 0.f;
#pragma unroll
            for (int e = 0; e < 2 * S::NBK; ++e) {
                const float p0 = fast_exp2(__builtin_fmaf(s[mb][e >> 1][(e & 1) * 2], scale, -m_use));
                const float p1 = fast_exp2(__builtin_fmaf(s[mb][e >> 1][(e & 1) * 2 + 1], scale, -m_use));
                psum += p0 + p1;
                // P feeds the 16-bit matrix instructions like K and V do; the row sum keeps the unrounded values
                pk[mb][e] = T::pack2(p0, p1);
            }
            l_run[mb] = l_run[mb] * alpha + psum;
            if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0) {
#pragma unroll
                for (int db = 0; db < S::DB; ++db) oacc[mb][db] *= alpha;
            }
        }
        // O^T[dv][row] += V^T . P^T
#pragma unroll
        for (int kk = 0; kk < S::NBK / 2; ++kk)
#pragma unroll
            for (int db = 0; db < S::DB; ++db) {
                const char FCK_LDS* p = vt + kk * 32 * S::ROWB + (((db * 2) ^ tr_sw) << 4);
                const u32x2_t lo4 = lds_read_tr16(p), hi4 = lds_read_tr16(p + 16 * S::ROWB);
                const u32x4_t av = {lo4[0], lo4[1], hi4[0], hi4[1]};
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) {
                    const u32x4_t pv = {pk[mb][kk * 4], pk[mb][kk * 4 + 1], pk[mb][kk * 4 + 2], pk[mb][kk * 4 + 3]};
                    oacc[mb][db] = T::mfma16(as_vec8<vec8>(av), as_vec8<vec8>(pv), oacc[mb][db]);
                }
            }
    };

    // tile c is in LDS between the two barriers of iteration c, tile c + 1 in flight
    for (int c = 0; c < n; ++c) {
        store_tile();
        __syncthreads();
        if (c + 1 < n) load_tile(c + 1);
        if (wave_rows) compute(c);
        __syncthreads();
    }

#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
        l_run[mb] = quad16_sum(l_run[mb]);
        if (!row_ok[mb]) continue;
        const float inv = l_run[mb] == 0.f ? 0.f : a.v_descale / l_run[mb];
        float* op = a.o_acc + wofs[mb] * dvs + kg * 4;
#pragma unroll
        for (int db = 0; db < S::DB; ++db) {
            if (kPad && db * 16 + kg * 4 >= dvs) continue;
            *reinterpret_cast<f32x4_t*>(op + db * 16) = oacc[mb][db] * inv;
        }
        if (kg == 0) a.lse_acc[wofs[mb]] = l_run[mb] == 0.f ? -INFINITY : (m_run[mb] + fast_log2(l_run[mb])) * kLn2;
    }
}

// Merge of a row's partial results.  Dv/4 lanes per row, 4 columns each; the work is a chain of round trips, so the rows are
// spread over one-wave workgroups while there are few.
template <typename T, int DV, int NT>
__global__ __launch_bounds__(NT) void shared_prefix_combine_kernel(const SharedPrefixArgs a)
{
    constexpr int TPR = DV / 4;
    const int64_t item = (int64_t)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;  // (row, head)
    const int c = threadIdx.x % TPR * 4;
    const int64_t rows = a.seqstart_q ? a.shape_sq : (int64_t)a.batch * a.sq;
    if (item >= rows * a.hq || c >= a.dv) return;
    const int tok = (int)(item / a.hq), h = (int)(item % a.hq);
    if (a.seqstart_q && tok >= a.seqstart_q[a.batch]) return;  // a row behind the last sequence stays as it was
    const int b = a.seqstart_q ? 0 : tok / a.sq, i = a.seqstart_q ? tok : tok - b * a.sq;
    const int slots = a.ns_prefix + a.ns_own;
    const int64_t row = (int64_t)b * a.hq + h, w0 = row * slots * a.shape_sq + i;
    float lse;
    const f32x4_t acc = combine_splits<DV>(a.lse_acc, a.o_acc, w0, a.shape_sq, slots, c, a.dv, &lse);
    u32x2_t out;
    out[0] = T::pack2(acc[0], acc[1]);
    out[1] = T::pack2(acc[2], acc[3]);
    *reinterpret_cast<u32x2_t*>(reinterpret_cast<uint16_t*>(a.o) + item * a.dv + c) = out;
    if (a.lse && c == 0) a.lse[row * a.shape_sq + i] = lse;
}

template <typename T, int D, int MB>
hipError_t launch_general(const SharedPrefixArgs& a, bool uniform, int64_t grid, hipStream_t st)
{
    constexpr size_t lds = (size_t)2 * SharedShape<D, MB>::TILEB + 16;
    const dim3 blocks((unsigned)grid), threads(256);
    if (a.kv8) {
        if (uniform) return launch_with_lds<shared_prefix_kernel<T, D, MB, true, true, false, true>>(blocks, threads, lds, st, a);
        return launch_with_lds<shared_prefix_kernel<T, D, MB, false, true, false, true>>(blocks, threads, lds, st, a);
    }
    if (a.d != D || a.dv != D) {
        if (uniform) return launch_with_lds<shared_prefix_kernel<T, D, MB, true, true, true, false>>(blocks, threads, lds, st, a);
        return launch_with_lds<shared_prefix_kernel<T, D, MB, false, true, true, false>>(blocks, threads, lds, st, a);
    }
    if (a.mod.active()) {
        if (uniform) return launch_with_lds<shared_prefix_kernel<T, D, MB, true, true, false, false>>(blocks, threads, lds, st, a);
        return launch_with_lds<shared_prefix_kernel<T, D, MB, false, true, false, false>>(blocks, threads, lds, st, a);
    }
    if (uniform) return launch_with_lds<shared_prefix_kernel<T, D, MB, true, false, false, false>>(blocks, threads, lds, st, a);
    return launch_with_lds<shared_prefix_kernel<T, D, MB, false, false, false, false>>(blocks, threads, lds, st, a);
}

template <typename T, int DV>
hipError_t launch_combine(const SharedPrefixArgs& a, hipStream_t st)
{
    const int64_t items = (a.seqstart_q ? a.shape_sq : (int64_t)a.batch * a.sq) * a.hq;
    constexpr int per_wg = 256 / (DV / 4), per_wave = 64 / (DV / 4);
    const int64_t wide = (items + per_wg - 1) / per_wg;
    if (wide > INT32_MAX) return hipErrorInvalidValue;
    if (wide < 4 * (int64_t)a.num_cu)
        hipLaunchKernelGGL((shared_prefix_combine_kernel<T, DV, 64>), dim3((unsigned)((items + per_wave - 1) / per_wave)), dim3(64), 0, st, a);
    else
        hipLaunchKernelGGL((shared_prefix_combine_kernel<T, DV, 256>), dim3((unsigned)wide), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <typename T, int D, int MB>
hipError_t launch_mb(SharedPrefixArgs& a, const SharedPrefixRows& rows, hipStream_t st)
{
    constexpr int BM = SharedShape<D, MB>::BM;
    const int64_t p_tiles = (rows.group + BM - 1) / BM, o_tiles = (rows.own + BM - 1) / BM;
    const int64_t streams = ((int64_t)a.groups * a.ns_prefix * a.hk + 7) / 8 * 8;
    // Equally many tiles per group, unless the bound on their size makes that more than twice what all rows can need (256
    // sequences in 64 groups without a bound: 213 us so, 94 us with the tiles in one row, 92 us with an exact bound).
    const int64_t all_tiles = rows.all / BM + a.groups;
    const bool equal = p_tiles * a.groups <= 2 * all_tiles;
    const int64_t prefix_items = equal ? streams * p_tiles : (int64_t)a.ns_prefix * a.hk * all_tiles;
    const int64_t grid = prefix_items + (int64_t)a.hk * a.ns_own * o_tiles * a.batch;
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    a.prefix_tiles = equal ? (int32_t)p_tiles : 0;
    a.own_tiles = (int32_t)o_tiles;
    a.prefix_items = (int32_t)prefix_items;
    // a key tile then never straddles a page
    const bool uniform = a.page_size % SharedShape<D, MB>::TK == 0;
    if (hipError_t e = launch_general<T, D, MB>(a, uniform, grid, st); e != hipSuccess) return e;
    if (a.dv <= 64) return launch_combine<T, 64>(a, st);
    if (a.dv <= 128) return launch_combine<T, 128>(a, st);
    return launch_combine<T, 256>(a, st);
}

template <typename T, int D>
hipError_t launch_d(SharedPrefixArgs& a, const SharedPrefixRows& rows, hipStream_t st)
{
    if constexpr (D <= 128)
        if (shared_prefix_blocks(D, rows.typical) == 2) return launch_mb<T, D, 2>(a, rows, st);
    return launch_mb<T, D, 1>(a, rows, st);
}

}  // namespace

// Two row blocks per wave: 512 rows over 32768 keys take 117 us instead of 126; 128 rows over 4096 keys 32.8 us instead of 31.2
// (half as many items then share out the keys).
int shared_prefix_blocks(int d, int64_t rows_prefix) { return d <= 128 && rows_prefix > 128 ? 2 : 1; }

hipError_t launch_shared_prefix(SharedPrefixArgs a, int d, int dtype, const SharedPrefixRows& rows, hipStream_t st)
{
    switch (d) {
    case 64: return dtype == 4 ? launch_d<BF16, 64>(a, rows, st) : launch_d<FP16, 64>(a, rows, st);
    case 128: return dtype == 4 ? launch_d<BF16, 128>(a, rows, st) : launch_d<FP16, 128>(a, rows, st);
    case 256: return dtype == 4 ? launch_d<BF16, 256>(a, rows, st) : launch_d<FP16, 256>(a, rows, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace fck
