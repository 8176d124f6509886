"""Functional FMHA operators: the `flash_ck.ops.fmha` surface FlashCK declares but leaves empty
(flash_ck/utils/utils.py:49-58; tests/pytorch/fmha/test_{fmha_fwd,fmha_fwd_var_len,fmha_fwd_append_kv,
batch_prefill}.py are 0-byte files), backed by the gfx950 kernels through the C ABI.

The wrappers follow flash_ck/ops/norm/layer_norm.py:61-116 for validation (TypeError / ValueError before any
launch).  Unlike that operator there is no PyTorch fallback: a missing library or a rejected call raises.

Tensor conventions (T = torch.float16 | torch.bfloat16, contiguous, on the GPU):
    q, o         [B, sq, Hq, D]  or packed [total_q, Hq, D] with cu_seqlens_q (int32 [B+1])
    k, v         [B, sk, Hk, D]  or packed [total_k, Hk, D] with cu_seqlens_k
    k/v_cache    paged [num_pages, page_size, Hk, D] with block_table int32 [B, max_pages_per_seq]
    seqlen_k     int32 [B] valid keys per sequence
"""
import contextlib
import ctypes
import functools
import math
from typing import Optional, Tuple

import torch

from ... import _lib
from ...utils import FlashCKOperationType, flags, register_flashck_functions, tuning

__all__ = [
    "MASK_NONE", "MASK_TOP_LEFT", "MASK_BOTTOM_RIGHT", "MASK_GENERIC", "ROPE_NONE", "ROPE_INTERLEAVED",
    "ROPE_HALF_ROTATED", "fmha_fwd", "fmha_fwd_varlen", "fmha_fwd_splitkv", "fmha_fwd_splitkv_combine",
    "fmha_fwd_splitkv_fused", "fused_splitkv_fits",
    "fmha_fwd_appendkv", "fmha_batch_prefill", "fmha_fwd_pagedkv", "fmha_decode_paged", "fmha_decode_step",
    "tune_decode_num_splits", "tune_prefill_variant", "DecodeWorkspace", "num_splits_heuristic", "splitkv_workspace", "validate_paged", "fused_reset",
    "fmha_decode_shared_prefix", "fmha_key_weights", "fmha_cache_evict", "shared_prefix_splits",
]

# GenericAttentionMaskEnum / RopeEnum, core/profiling/attention/fmha_library.h:81-87,195-200
MASK_NONE, MASK_TOP_LEFT, MASK_BOTTOM_RIGHT, MASK_GENERIC = 0, 1, 2, 3
ROPE_NONE, ROPE_INTERLEAVED, ROPE_HALF_ROTATED = 0, 1, 2

# flashck::DataType, core/utils/dtype.h:16-28.  float8_e4m3fn queries select the all-fp8 roles (Q, K, V, P and O in e4m3,
# FmhaFwdTypeConfig<fp8_t>, core/module/kernels/attention_kernels/fmha_common_jinja.h:157-171).
_DTYPE_ID = {torch.float8_e4m3fn: 1, torch.float16: 3, torch.bfloat16: 4}


# Host-side tests of the validation code switch this off (and replace _call); nothing else may.
_REQUIRE_GPU_TENSORS = True


def _dtype_id(t: torch.Tensor) -> int:
    if t.dtype not in _DTYPE_ID:
        raise TypeError(f"FMHA supports torch.float16, torch.bfloat16 and torch.float8_e4m3fn, got {t.dtype}")
    return _DTYPE_ID[t.dtype]


def _check_tensor(name, t, dtype=None, ndim=None, optional=False):
    if t is None:
        if optional:
            return
        raise TypeError(f"{name} must be a torch.Tensor, got None")
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"Expected {name} to be a torch.Tensor, got {type(t)}")
    if _REQUIRE_GPU_TENSORS and not t.is_cuda:
        raise ValueError(f"{name} must live on the GPU (got device {t.device})")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must have dtype {dtype}, got {t.dtype}")
    if ndim is not None and t.dim() not in (ndim if isinstance(ndim, tuple) else (ndim,)):
        raise ValueError(f"{name} must have {ndim} dimensions, got shape {tuple(t.shape)}")


def _check_shape(name, t, shape, like):
    """A caller-supplied buffer (workspace or output) must be exactly what the kernel is about to write: the C ABI
    only sees a pointer, so a wrong size here would be an out-of-bounds write on the GPU."""
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, the inputs are on {like.device}")


def _out(name, out, shape, dtype, like):
    """`out` validated against (shape, dtype, device of `like`), or a new tensor when it is None."""
    if out is None:
        return torch.empty(*shape, dtype=dtype, device=like.device)
    _check_tensor(name, out, dtype=dtype)
    _check_shape(name, out, shape, like)
    return out


def _check_kv(q, k, v, ndim):
    """k and v against q: same rank, k's head dim is q's, v agrees with k on everything but the head dim."""
    if k.dim() != ndim or v.dim() != ndim:
        raise ValueError(f"k {tuple(k.shape)} / v {tuple(v.shape)} must have {ndim} dimensions")
    if k.shape[-1] != q.shape[-1]:
        raise ValueError(f"k head dim {k.shape[-1]} != q head dim {q.shape[-1]}")
    if v.shape[:-1] != k.shape[:-1]:
        raise ValueError(f"v {tuple(v.shape)} does not match k {tuple(k.shape)}")
    if k.shape[-2] <= 0 or q.shape[-2] % k.shape[-2]:
        raise ValueError(f"q heads {q.shape[-2]} must be a multiple of kv heads {k.shape[-2]}")


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    # the handle alone: building a torch.cuda.Stream object costs as much as the rest of a small call's host side
    return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(torch.cuda.current_device()))


def _call(name, *args):
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    if rc != 0:
        msg = lib.fck_last_error().decode()
        if rc == -2:
            raise NotImplementedError(f"{name}: {msg}")
        if rc == -1:
            raise ValueError(f"{name}: {msg}")
        raise RuntimeError(f"{name} failed ({rc}): {msg}")


def _scale(scale, d):
    # scale == 0 selects 1/sqrt(head_dim), as the FlashCK harness does (fmha_fwd_split_kv_jinja.h:60-62)
    return float(scale) if scale else 1.0 / math.sqrt(d)


def _window(window):
    wl, wr = window
    return int(wl), int(wr)


def _attrs(q, bias, alibi_slopes, logits_soft_cap, group, batch, rows, min_cols, kv_fp8=False, k_descale=1.0, v_descale=1.0,
           decode_variant=0, prefill_variant=0, max_seqlen_k=0, o_scale=1.0, lse=None):
    """fck_fmha_attrs for a call, or None when no score modifier is asked for.

    o_scale (float8_e4m3fn queries on the dense / paged / page-list prefill calls): the output is
    saturate(o_scale * o) in e4m3.
    lse: fp32 [B, Hq, sq] (group mode [Hq, total_q]) that receives the log-sum-exp of every row, on the prefill-family calls.
    bias (elementwise, BiasEnum ELEMENTWISE_BIAS): q's dtype (float32 for float8_e4m3fn queries), last dim contiguous; batch mode [1|B, 1|Hq, sq, >= sk],
    group mode [1|Hq, total_q, >= max sk]; size-1 dims are shared (the reference's rank 0 / 1 / 2).
    alibi_slopes (ALIBI): fp32 [Hq] or [B, Hq].  logits_soft_cap > 0: s = cap * tanh(scale * qk / cap).
    Returns (pointer argument, object to keep alive until the call has been made)."""
    cap = float(logits_soft_cap)
    if not (cap >= 0.0) or math.isinf(cap):
        raise ValueError("logits_soft_cap must be finite and >= 0")
    if int(decode_variant) not in (0, 1, 2, 3, 4):
        raise ValueError("decode_variant must be 0 (library's choice), 1 (one KV head per workgroup), 2 (head pairs), or 3 / 4 (the same "
                         "with splits of equal size in keys)")
    if int(prefill_variant) not in (0, 1, 2, 3, 4):
        raise ValueError("prefill_variant must be 0 (library's choice) or 1..4 (see fck_fmha_attrs.prefill_variant)")
    if bias is None and alibi_slopes is None and cap == 0.0 and not kv_fp8 and not decode_variant and not prefill_variant and lse is None:
        return None, None
    if bias is not None and alibi_slopes is not None:
        raise ValueError("bias and alibi_slopes are exclusive (one BiasEnum per call)")
    a = _lib.Attrs()
    a.size = ctypes.sizeof(_lib.Attrs)
    a.logits_soft_cap = cap
    a.decode_variant = int(decode_variant)
    a.max_seqlen_k = max(int(max_seqlen_k), 0)
    a.prefill_variant = int(prefill_variant)
    if kv_fp8:
        if not (float(k_descale) > 0.0 and float(v_descale) > 0.0 and math.isfinite(k_descale) and math.isfinite(v_descale)):
            raise ValueError("k_descale and v_descale must be positive and finite")
        a.kv_dtype, a.k_descale, a.v_descale = 1, float(k_descale), float(v_descale)  # flashck::DataType FLOAT8
    if not (float(o_scale) > 0.0 and math.isfinite(o_scale)):
        raise ValueError("o_scale must be positive and finite")
    a.o_scale = float(o_scale)
    Hq = q.shape[-2]
    if lse is not None:
        _check_tensor("lse", lse, dtype=torch.float32)
        _check_shape("lse", lse, (Hq, rows) if group else (batch, Hq, rows), q)
        a.lse, a.lse_head_stride = lse.data_ptr(), rows
    if bias is not None:
        if not isinstance(bias, torch.Tensor):
            raise TypeError(f"Expected bias to be a torch.Tensor, got {type(bias)}")
        if _REQUIRE_GPU_TENSORS and not bias.is_cuda:
            raise ValueError(f"bias must live on the GPU (got device {bias.device})")
        want = torch.float32 if q.dtype == torch.float8_e4m3fn else q.dtype   # BiasDataType of the e4m3 roles is float
        if bias.dtype != want:
            raise TypeError(f"bias must have dtype {want} for {q.dtype} queries, got {bias.dtype}")
        if bias.dim() != (3 if group else 4) or bias.stride(-1) != 1:
            raise ValueError(f"bias must be {'[1|Hq, total_q, sk]' if group else '[1|B, 1|Hq, sq, sk]'} with a contiguous last dim, "
                             f"got shape {tuple(bias.shape)} strides {bias.stride()}")
        if bias.shape[-3] not in (1, Hq) or (not group and bias.shape[0] not in (1, batch)):
            raise ValueError(f"bias {tuple(bias.shape)}: head dim must be 1 or {Hq}" + ("" if group else f", batch dim 1 or {batch}"))
        if bias.shape[-2] != rows or bias.shape[-1] < min_cols:
            raise ValueError(f"bias {tuple(bias.shape)} must have {rows} rows and at least {min_cols} columns")
        a.bias_type = 1
        a.bias_cols = bias.shape[-1]
        a.bias = bias.data_ptr()
        a.bias_row_stride = bias.stride(-2)
        a.bias_head_stride = bias.stride(-3) if bias.shape[-3] > 1 else 0
        a.bias_batch_stride = 0 if group or bias.shape[0] == 1 else bias.stride(0)
    elif alibi_slopes is not None:
        _check_tensor("alibi_slopes", alibi_slopes, dtype=torch.float32, ndim=(1, 2))
        if alibi_slopes.shape[-1] != Hq or (alibi_slopes.dim() == 2 and alibi_slopes.shape[0] != batch):
            raise ValueError(f"alibi_slopes must be [{Hq}] or [{batch}, {Hq}], got {tuple(alibi_slopes.shape)}")
        a.bias_type = 2
        a.bias = alibi_slopes.data_ptr()
        a.bias_batch_stride = Hq if alibi_slopes.dim() == 2 else 0
    return ctypes.byref(a), (a, bias, alibi_slopes, lse)


def validate_paged(*, seqlen_k=None, block_table=None, kv_indptr=None, kv_page_indices=None, kv_last_page_lens=None,
                   num_total_pages: int, page_size: int, out=None, check: bool = False):
    """Debug aid: checks on the GPU what the paged kernels trust - key counts against what the block-table row / page
    list can address, page ids against the pool - without allocating when `out` (int32[4] on the device) is given.
    Returns the counters tensor [sequences with a bad length, page ids out of range, malformed page lists, first
    offending sequence or -1]; nothing is read back unless check=True, which synchronises and raises ValueError when a
    counter is non-zero.  The operators call it with check=True before every paged launch while the flag
    FC_DEBUG_KERNEL_INSTANCE is on (core/utils/flags.cc:169)."""
    paged = block_table is not None
    ref = block_table if paged else kv_indptr
    _check_tensor("block_table" if paged else "kv_indptr", ref, dtype=torch.int32, ndim=2 if paged else 1)
    if paged:
        _check_tensor("seqlen_k", seqlen_k, dtype=torch.int32, ndim=1)
        if kv_indptr is not None or kv_page_indices is not None:
            raise ValueError("give a block table or a page list, not both")
        B, stride = block_table.shape
        if seqlen_k.numel() != B:
            raise ValueError(f"seqlen_k has {seqlen_k.numel()} entries, the block table {B} rows")
    else:
        _check_tensor("kv_page_indices", kv_page_indices, dtype=torch.int32, ndim=1)
        _check_tensor("kv_last_page_lens", kv_last_page_lens, dtype=torch.int32, ndim=1, optional=True)
        B, stride = kv_indptr.numel() - 1, 0
    counts = _out("out", out, (4,), torch.int32, ref)
    _call("fck_fmha_validate_paged", _ptr(seqlen_k), _ptr(block_table), stride, _ptr(kv_indptr), _ptr(kv_page_indices),
          _ptr(kv_last_page_lens), B, int(num_total_pages), int(page_size), _ptr(counts), _stream())
    if check:
        bad_len, bad_page, bad_list, first = counts.tolist()
        if bad_len or bad_page or bad_list:
            raise ValueError(f"paged-cache arguments are inconsistent: {bad_len} sequence(s) longer than their table can address, "
                             f"{bad_page} page id(s) outside the pool of {num_total_pages}, {bad_list} malformed page list(s); "
                             f"first offending sequence: {first}")
    return counts


def _debug_validate(**kw):
    if flags.flag("FC_DEBUG_KERNEL_INSTANCE"):
        validate_paged(check=True, **kw)


def _read_entries(block_table, seqlen_k, prefix_lens, cu_groups, max_group_size, page, append=False):
    """The table a step over shared prefixes uses, for the debug flag's check (synchronises): whole pages of a prefix come from the
    row of the group's first sequence, whatever the other rows hold there.  append: seqlen_k are the lengths before an append, which
    goes to the pages of a sequence's own row."""
    table, lens, B = block_table.clone(), seqlen_k.tolist(), seqlen_k.numel()
    cu = [0, B] if cu_groups is None else [min(max(x, 0), B) for x in cu_groups.tolist()]
    for first, end, prefix in zip(cu, cu[1:], prefix_lens.tolist()):
        end = min(end, first + max_group_size) if max_group_size > 0 else end
        if first < end:
            whole = min(max(prefix, 0), max(lens[first], 0), table.shape[1] * page) // page
            for b in range(first + 1, end):
                n = min(whole, max(lens[b], 0) // page) if append else whole
                table[b, :n] = block_table[first, :n]
    return table


def fused_reset() -> None:
    """Zero the arrival tickets of fmha_fwd_splitkv_fused on the current device and forget which stream owns which slice
    of the library's array (after a fused launch that did not run to completion, or to serve other streams; only while
    no fused call is in flight; see fck_fmha_fused_reset)."""
    _call("fck_fmha_fused_reset", _stream())


def num_splits_heuristic(batch, q_num_heads, kv_num_heads, seqlen_q, max_seqlen_k, head_dim, num_cu=0) -> int:
    """Split count chosen from the CU count and the KV length."""
    return int(_lib.load().fck_fmha_num_splits_heuristic(batch, q_num_heads, kv_num_heads, seqlen_q, max_seqlen_k,
                                                         head_dim, num_cu))


def splitkv_workspace(shape_batch, q_num_heads, shape_seqlen_q, v_head_dim, num_splits, device) -> Tuple[torch.Tensor, torch.Tensor]:
    """(o_acc fp32 [Bs,Hq,ns,Sq,Dv], lse_acc fp32 [Bs,Hq,ns,Sq]) - fmha_fwd_split_kv_jinja.h:543-547."""
    o_acc = torch.empty(shape_batch, q_num_heads, num_splits, shape_seqlen_q, v_head_dim, dtype=torch.float32, device=device)
    lse_acc = torch.empty(shape_batch, q_num_heads, num_splits, shape_seqlen_q, dtype=torch.float32, device=device)
    return o_acc, lse_acc


def fmha_fwd(q, k, v, scale: float = 0.0, mask_type: int = MASK_NONE, window: Tuple[int, int] = (-1, -1),
             seqlen_k: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, *, bias=None, alibi_slopes=None,
             logits_soft_cap: float = 0.0, k_descale: float = 1.0, v_descale: float = 1.0, o_scale: float = 1.0, lse=None) -> torch.Tensor:
    """Dense attention, batch mode: q [B,sq,Hq,D], k/v [B,sk,Hk,D] -> o [B,sq,Hq,D].
    bias / alibi_slopes / logits_soft_cap: see _attrs.  float8_e4m3fn tensors: the all-fp8 roles, with k = k_descale *
    stored, v = v_descale * stored, o = saturate(o_scale * result).  lse (fp32 [B,Hq,sq], optional) receives the log-sum-exp
    of every row."""
    _check_tensor("q", q, ndim=4)
    _check_tensor("k", k, dtype=q.dtype, ndim=4)
    _check_tensor("v", v, dtype=q.dtype, ndim=4)
    _check_tensor("seqlen_k", seqlen_k, dtype=torch.int32, ndim=1, optional=True)
    B, sq, Hq, D = q.shape
    _check_kv(q, k, v, 4)
    if k.shape[0] != B:
        raise ValueError(f"k {tuple(k.shape)} / v {tuple(v.shape)} do not match q {tuple(q.shape)}")
    if q.numel() == 0:
        raise ValueError("Input tensor cannot be empty")
    if seqlen_k is not None and seqlen_k.numel() != B:
        raise ValueError(f"seqlen_k must have {B} entries, got {seqlen_k.numel()}")
    sk, Hk, Dv = k.shape[1], k.shape[2], v.shape[3]
    o = _out("out", out, (B, sq, Hq, Dv), q.dtype, q)
    wl, wr = _window(window)
    at, keep = _attrs(q, bias, alibi_slopes, logits_soft_cap, False, B, sq, sk, q.dtype == torch.float8_e4m3fn, k_descale, v_descale,
                      o_scale=o_scale, lse=lse)
    if at is None:
        _call("fck_fmha_fwd", _ptr(q), _ptr(k), _ptr(v), None, _ptr(o), None, None, _ptr(seqlen_k), B, sq, sk, Hq, Hk, D, Dv,
              sq, _scale(scale, D), wl, wr, mask_type, _dtype_id(q), _stream())
    else:
        _call("fck_fmha_fwd_attrs", _ptr(q), _ptr(k), _ptr(v), None, _ptr(o), None, None, _ptr(seqlen_k), B, sq, sk, Hq, Hk, D, Dv,
              sq, _scale(scale, D), wl, wr, mask_type, _dtype_id(q), at, _stream())
    del keep
    return o


def fmha_fwd_varlen(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q: int, scale: float = 0.0,
                    mask_type: int = MASK_NONE, window=(-1, -1), seqlen_k=None, out=None, *, bias=None, alibi_slopes=None,
                    logits_soft_cap: float = 0.0, k_descale: float = 1.0, v_descale: float = 1.0, o_scale: float = 1.0, lse=None) -> torch.Tensor:
    """Dense attention, group mode: q [total_q,Hq,D], k/v [total_k,Hk,D] packed by cu_seqlens.
    bias / alibi_slopes / logits_soft_cap: see _attrs; float8_e4m3fn tensors and their scales: see fmha_fwd.
    lse (fp32 [Hq,total_q], optional) receives the log-sum-exp of every row.

    seqlen_k (int32 [B], optional): logical key counts when the packed K/V slots hold padding behind the keys."""
    _check_tensor("q", q, ndim=3)
    _check_tensor("k", k, dtype=q.dtype, ndim=3)
    _check_tensor("v", v, dtype=q.dtype, ndim=3)
    _check_tensor("cu_seqlens_q", cu_seqlens_q, dtype=torch.int32, ndim=1)
    _check_tensor("cu_seqlens_k", cu_seqlens_k, dtype=torch.int32, ndim=1)
    if cu_seqlens_q.numel() != cu_seqlens_k.numel() or cu_seqlens_q.numel() < 2:
        raise ValueError("cu_seqlens_q and cu_seqlens_k must both have batch + 1 entries")
    B = cu_seqlens_q.numel() - 1
    tq, Hq, D = q.shape
    _check_kv(q, k, v, 3)
    _check_tensor("seqlen_k", seqlen_k, dtype=torch.int32, ndim=1, optional=True)
    if seqlen_k is not None and seqlen_k.numel() != B:
        raise ValueError(f"seqlen_k must have {B} entries, got {seqlen_k.numel()}")
    Hk, Dv = k.shape[1], v.shape[2]
    o = _out("out", out, (tq, Hq, Dv), q.dtype, q)
    wl, wr = _window(window)
    at, keep = _attrs(q, bias, alibi_slopes, logits_soft_cap, True, B, tq, 1, q.dtype == torch.float8_e4m3fn, k_descale, v_descale,
                      o_scale=o_scale, lse=lse)
    if at is None:
        _call("fck_fmha_fwd", _ptr(q), _ptr(k), _ptr(v), None, _ptr(o), _ptr(cu_seqlens_q), _ptr(cu_seqlens_k), _ptr(seqlen_k), B, tq,
              k.shape[0], Hq, Hk, D, Dv, max_seqlen_q, _scale(scale, D), wl, wr, mask_type, _dtype_id(q), _stream())
    else:
        _call("fck_fmha_fwd_attrs", _ptr(q), _ptr(k), _ptr(v), None, _ptr(o), _ptr(cu_seqlens_q), _ptr(cu_seqlens_k), _ptr(seqlen_k),
              B, tq, k.shape[0], Hq, Hk, D, Dv, max_seqlen_q, _scale(scale, D), wl, wr, mask_type, _dtype_id(q), at, _stream())
    del keep
    return o


def fmha_fwd_splitkv(q, k, v, num_splits: int, *, seqlen_k=None, block_table=None, cache_batch_idx=None,
                     cu_seqlens_q=None, cu_seqlens_k=None, max_seqlen_q: int = 0, scale: float = 0.0,
                     mask_type: int = MASK_NONE, window=(-1, -1), o_acc=None, lse_acc=None, bias=None, alibi_slopes=None,
                     logits_soft_cap: float = 0.0, k_descale: float = 1.0, v_descale: float = 1.0, decode_variant: int = 0,
                     max_seqlen_k: int = 0):
    """Split-KV forward: returns the per-split partials (o_acc, lse_acc), to be merged by fmha_fwd_splitkv_combine.
    decode_variant: 0 = the library picks the kernel variant, 1 / 2 force it (what the tuner records, see
    tune_decode_num_splits); 3 / 4 = 1 / 2 with splits of equal size in keys (chunks of ceil(max_seqlen_k / num_splits)
    keys, the same for every sequence: even work items for a ragged batch; max_seqlen_k = 0 takes the block table's
    capacity).
    bias / alibi_slopes / logits_soft_cap: see _attrs.  k and v may be torch.float8_e4m3fn (a quantised cache with the
    static per-tensor scales k_descale, v_descale: value = descale * stored); q and the output keep q's dtype.

    k/v are a paged cache when block_table is given, packed when cu_seqlens_k is given, else [B*, sk, Hk, D].
    """
    group = cu_seqlens_q is not None
    _check_tensor("q", q, ndim=3 if group else 4)
    kv_fp8 = isinstance(k, torch.Tensor) and k.dtype == torch.float8_e4m3fn
    _check_tensor("k", k, dtype=torch.float8_e4m3fn if kv_fp8 else q.dtype)
    _check_tensor("v", v, dtype=torch.float8_e4m3fn if kv_fp8 else q.dtype)
    for name, t in (("seqlen_k", seqlen_k), ("block_table", block_table), ("cache_batch_idx", cache_batch_idx),
                    ("cu_seqlens_q", cu_seqlens_q), ("cu_seqlens_k", cu_seqlens_k)):
        _check_tensor(name, t, dtype=torch.int32, optional=True)
    if int(num_splits) < 1:
        raise ValueError("num_splits must be >= 1")
    Hq, D = q.shape[-2], q.shape[-1]
    _check_kv(q, k, v, 3 if (cu_seqlens_k is not None and block_table is None) else 4)
    Hk, Dv = k.shape[-2], v.shape[-1]
    if group:
        B, sq, bs = cu_seqlens_q.numel() - 1, q.shape[0], 1
        if max_seqlen_q <= 0:
            raise ValueError("group mode needs max_seqlen_q")
    else:
        B, sq, bs = q.shape[0], q.shape[1], q.shape[0]
        max_seqlen_q = sq
    if seqlen_k is not None and seqlen_k.numel() != B:
        raise ValueError(f"seqlen_k must have {B} entries, got {seqlen_k.numel()}")
    if block_table is not None:
        if seqlen_k is None:
            raise ValueError("a paged cache needs seqlen_k")
        if block_table.dim() != 2 or block_table.shape[0] != B:
            raise ValueError(f"block_table must be [batch, max_pages_per_seq], got {tuple(block_table.shape)}")
        page, sk, max_blocks = k.shape[1], 0, block_table.numel()
        _debug_validate(seqlen_k=seqlen_k, block_table=block_table, num_total_pages=k.shape[0], page_size=page)
    else:
        page, max_blocks = 0, 0
        sk = k.shape[0] if cu_seqlens_k is not None else k.shape[1]
    if (o_acc is None) != (lse_acc is None):
        raise ValueError("o_acc and lse_acc must be given together")
    if o_acc is None:
        o_acc, lse_acc = splitkv_workspace(bs, Hq, sq, Dv, num_splits, q.device)
    else:
        # the kernel writes with the strides of THIS split count
        _check_tensor("o_acc", o_acc, dtype=torch.float32)
        _check_tensor("lse_acc", lse_acc, dtype=torch.float32)
        _check_shape("o_acc", o_acc, (bs, Hq, int(num_splits), sq, Dv), q)
        _check_shape("lse_acc", lse_acc, (bs, Hq, int(num_splits), sq), q)
    wl, wr = _window(window)
    at, keep = _attrs(q, bias, alibi_slopes, logits_soft_cap, group, B, sq, 1 if (group or block_table is not None) else sk,
                      kv_fp8, k_descale, v_descale, decode_variant, max_seqlen_k=max_seqlen_k)
    if at is None:
        _call("fck_fmha_fwd_splitkv", _ptr(q), _ptr(k), _ptr(v), None, _ptr(lse_acc), _ptr(o_acc), _ptr(cu_seqlens_q),
              _ptr(cu_seqlens_k), _ptr(seqlen_k), _ptr(block_table), _ptr(cache_batch_idx), B, sq, sk, Hq, Hk, D, Dv,
              max_seqlen_q, int(num_splits), max_blocks, page, _scale(scale, D), wl, wr, mask_type, _dtype_id(q), _stream())
    else:
        _call("fck_fmha_fwd_splitkv_attrs", _ptr(q), _ptr(k), _ptr(v), None, _ptr(lse_acc), _ptr(o_acc), _ptr(cu_seqlens_q),
              _ptr(cu_seqlens_k), _ptr(seqlen_k), _ptr(block_table), _ptr(cache_batch_idx), B, sq, sk, Hq, Hk, D, Dv,
              max_seqlen_q, int(num_splits), max_blocks, page, _scale(scale, D), wl, wr, mask_type, _dtype_id(q), at, _stream())
    del keep
    return o_acc, lse_acc


# limits of the fused entry point's fixed device array (fmha_c_api.h, fck_fmha_fwd_splitkv_fused)
_FUSED_MAX_PARTIAL_FLOATS = 4 << 20
_FUSED_MAX_TICKETS = 16384
_FUSED_MAX_AUTO_SPLITS = 128


def fused_splitkv_fits(shape_batch, batch, q_num_heads, kv_num_heads, shape_seqlen_q, max_seqlen_q, v_head_dim, num_splits) -> bool:
    """Whether fmha_fwd_splitkv_fused can hold this problem's partial results (num_splits = 0: worst case of the
    library's own choice)."""
    ns = num_splits if num_splits > 0 else _FUSED_MAX_AUTO_SPLITS
    rows = max_seqlen_q * (q_num_heads // max(kv_num_heads, 1))
    m_tiles = 1 if rows <= 32 else (rows + 31) // 32
    return (shape_batch * q_num_heads * ns * shape_seqlen_q * (v_head_dim + 1) <= _FUSED_MAX_PARTIAL_FLOATS
            and batch * kv_num_heads * m_tiles <= _FUSED_MAX_TICKETS)


def fmha_fwd_splitkv_fused(q, k, v, num_splits: int = 0, *, seqlen_k=None, block_table=None, cache_batch_idx=None,
                           cu_seqlens_q=None, cu_seqlens_k=None, max_seqlen_q: int = 0, scale: float = 0.0,
                           mask_type: int = MASK_NONE, window=(-1, -1), out=None) -> torch.Tensor:
    """Split-KV forward + LSE combine in one launch that allocates nothing on the GPU side: the partial results live in
    a fixed device array of the library (limits: see fused_splitkv_fits; beyond them NotImplementedError).

    num_splits = 0 lets the library take its heuristic split count for the CU count and the longest possible KV length.
    Each stream owns a slice of that array from its first call on; at most 4 streams per GPU (then NotImplementedError
    until fused_reset()).
    Arguments as fmha_fwd_splitkv; returns o [B,sq,Hq,Dv] (or [total_q,Hq,Dv] in group mode).
    """
    group = cu_seqlens_q is not None
    _check_tensor("q", q, ndim=3 if group else 4)
    _check_tensor("k", k, dtype=q.dtype)
    _check_tensor("v", v, dtype=q.dtype)
    for name, t in (("seqlen_k", seqlen_k), ("block_table", block_table), ("cache_batch_idx", cache_batch_idx),
                    ("cu_seqlens_q", cu_seqlens_q), ("cu_seqlens_k", cu_seqlens_k)):
        _check_tensor(name, t, dtype=torch.int32, optional=True)
    if int(num_splits) < 0:
        raise ValueError("num_splits must be >= 0")
    Hq, D = q.shape[-2], q.shape[-1]
    _check_kv(q, k, v, 3 if (cu_seqlens_k is not None and block_table is None) else 4)
    Hk, Dv = k.shape[-2], v.shape[-1]
    if group:
        B, sq = cu_seqlens_q.numel() - 1, q.shape[0]
        if max_seqlen_q <= 0:
            raise ValueError("group mode needs max_seqlen_q")
    else:
        B, sq = q.shape[0], q.shape[1]
        max_seqlen_q = sq
    if seqlen_k is not None and seqlen_k.numel() != B:
        raise ValueError(f"seqlen_k must have {B} entries, got {seqlen_k.numel()}")
    if block_table is not None:
        if seqlen_k is None:
            raise ValueError("a paged cache needs seqlen_k")
        if block_table.dim() != 2 or block_table.shape[0] != B:
            raise ValueError(f"block_table must be [batch, max_pages_per_seq], got {tuple(block_table.shape)}")
        page, sk, max_blocks = k.shape[1], 0, block_table.numel()
        _debug_validate(seqlen_k=seqlen_k, block_table=block_table, num_total_pages=k.shape[0], page_size=page)
    else:
        page, max_blocks = 0, 0
        sk = k.shape[0] if cu_seqlens_k is not None else k.shape[1]
    o = _out("out", out, (*q.shape[:-1], Dv), q.dtype, q)
    wl, wr = _window(window)
    _call("fck_fmha_fwd_splitkv_fused", _ptr(q), _ptr(k), _ptr(v), None, _ptr(o), _ptr(cu_seqlens_q), _ptr(cu_seqlens_k),
          _ptr(seqlen_k), _ptr(block_table), _ptr(cache_batch_idx), B, sq, sk, Hq, Hk, D, Dv, max_seqlen_q, int(num_splits),
          max_blocks, page, _scale(scale, D), wl, wr, mask_type, _dtype_id(q), _stream())
    return o


def fmha_fwd_splitkv_combine(lse_acc, o_acc, dtype, cu_seqlens_q=None, max_seqlen_q: int = 0, out=None, lse=None) -> torch.Tensor:
    """LSE combine of split-KV partials -> o [B,sq,Hq,Dv] (or [total_q,Hq,Dv] in group mode).  lse (fp32 [B,Hq,sq] or
    [Hq,total_q], optional) receives the merged log-sum-exp of every row."""
    if dtype not in _DTYPE_ID:
        raise TypeError(f"FMHA supports torch.float16, torch.bfloat16 and torch.float8_e4m3fn, got {dtype}")
    _check_tensor("lse_acc", lse_acc, dtype=torch.float32, ndim=4)
    _check_tensor("o_acc", o_acc, dtype=torch.float32, ndim=5)
    _check_tensor("cu_seqlens_q", cu_seqlens_q, dtype=torch.int32, optional=True)
    bs, Hq, ns, sq, Dv = o_acc.shape
    if tuple(lse_acc.shape) != (bs, Hq, ns, sq):
        raise ValueError(f"lse_acc {tuple(lse_acc.shape)} does not match o_acc {tuple(o_acc.shape)}")
    if lse_acc.device != o_acc.device:
        raise ValueError(f"lse_acc is on {lse_acc.device}, o_acc on {o_acc.device}")
    if cu_seqlens_q is not None:
        if bs != 1:
            raise ValueError(f"group mode partials have shape batch 1, got {bs}")
        B = cu_seqlens_q.numel() - 1
        o = _out("out", out, (sq, Hq, Dv), dtype, o_acc)
    else:
        B = bs
        o = _out("out", out, (bs, sq, Hq, Dv), dtype, o_acc)
    if lse is None:
        _call("fck_fmha_fwd_splitkv_combine", _ptr(lse_acc), _ptr(o_acc), _ptr(o), _ptr(cu_seqlens_q), B, sq, Hq, Dv,
              max_seqlen_q or sq, ns, _DTYPE_ID[dtype], _stream())
    else:
        _check_tensor("lse", lse, dtype=torch.float32)
        _check_shape("lse", lse, (Hq, sq) if cu_seqlens_q is not None else (bs, Hq, sq), o_acc)
        _call("fck_fmha_fwd_splitkv_combine_lse", _ptr(lse_acc), _ptr(o_acc), _ptr(o), _ptr(lse), _ptr(cu_seqlens_q), B, sq, Hq, Dv,
              max_seqlen_q or sq, ns, _DTYPE_ID[dtype], _stream())
    return o


def fmha_fwd_appendkv(q, k_cache, v_cache, knew, vnew, seqlen_k, *, cu_seqlens_knew=None, max_seqlen_knew: int = 0,
                      rotary_cos=None, rotary_sin=None, rope_mode: int = ROPE_NONE, has_mask: bool = True,
                      block_table=None, cache_batch_idx=None, k_descale: float = 1.0, v_descale: float = 1.0,
                      _read_table=None) -> None:
    """Rotate knew (and q, in place) and append knew/vnew to the cache behind seqlen_k[b] tokens; in place.

    knew/vnew/q are packed [total_new, H, D] with cu_seqlens_knew, or [B, n, H, D] with n new tokens everywhere.
    seqlen_k is NOT advanced: the caller adds the new counts, as with the ck_tile kernel.
    torch.float8_e4m3fn caches are written quantised with the static scales: cache = fp8(x / descale), saturating.
    _read_table: what the debug flag's check walks in place of block_table (see _read_entries).
    """
    packed = cu_seqlens_knew is not None
    _check_tensor("knew", knew, ndim=3 if packed else 4)
    _check_tensor("vnew", vnew, dtype=knew.dtype, ndim=3 if packed else 4)
    _check_tensor("q", q, dtype=knew.dtype, ndim=3 if packed else 4, optional=True)
    kv_fp8 = isinstance(k_cache, torch.Tensor) and k_cache.dtype == torch.float8_e4m3fn
    _check_tensor("k_cache", k_cache, dtype=torch.float8_e4m3fn if kv_fp8 else knew.dtype, ndim=4)
    _check_tensor("v_cache", v_cache, dtype=torch.float8_e4m3fn if kv_fp8 else knew.dtype, ndim=4)
    _check_tensor("seqlen_k", seqlen_k, dtype=torch.int32, ndim=1)
    for name, t in (("cu_seqlens_knew", cu_seqlens_knew), ("block_table", block_table), ("cache_batch_idx", cache_batch_idx)):
        _check_tensor(name, t, dtype=torch.int32, optional=True)
    _check_tensor("rotary_cos", rotary_cos, dtype=knew.dtype, ndim=2, optional=True)
    _check_tensor("rotary_sin", rotary_sin, dtype=knew.dtype, ndim=2, optional=True)
    B = seqlen_k.numel()
    Hk, D, Dv = knew.shape[-2], knew.shape[-1], vnew.shape[-1]
    Hq = q.shape[-2] if q is not None else 0
    if k_cache.shape[2:] != (Hk, D) or v_cache.shape[2:] != (Hk, Dv) or v_cache.shape[:2] != k_cache.shape[:2]:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} / v_cache {tuple(v_cache.shape)} do not match knew "
                         f"{tuple(knew.shape)} / vnew {tuple(vnew.shape)}")
    if vnew.shape[:-1] != knew.shape[:-1]:
        raise ValueError(f"vnew {tuple(vnew.shape)} does not match knew {tuple(knew.shape)}")
    if q is not None and (q.shape[-1] != D or q.shape[:-2] != knew.shape[:-2] or Hq % Hk):
        raise ValueError(f"q {tuple(q.shape)} does not match knew {tuple(knew.shape)}")
    if packed and cu_seqlens_knew.numel() != B + 1:
        raise ValueError(f"cu_seqlens_knew must have {B + 1} entries, got {cu_seqlens_knew.numel()}")
    if not packed and knew.shape[0] != B:
        raise ValueError(f"knew batch {knew.shape[0]} != number of sequences {B}")
    if block_table is not None and (block_table.dim() != 2 or block_table.shape[0] != B):
        raise ValueError(f"block_table must be [batch, max_pages_per_seq] with batch {B}, got {tuple(block_table.shape)}")
    if rope_mode != ROPE_NONE and rotary_cos is not None and rotary_sin is not None and rotary_cos.shape != rotary_sin.shape:
        raise ValueError("rotary_cos and rotary_sin must have the same shape")
    if packed:
        if max_seqlen_knew <= 0:
            raise ValueError("packed new tokens need max_seqlen_knew")
        n = max_seqlen_knew
    else:
        n = knew.shape[1]
    if rope_mode != ROPE_NONE:
        if rotary_cos is None or rotary_sin is None:
            raise ValueError("rope_mode != ROPE_NONE needs rotary_cos and rotary_sin")
        rotary_dim = rotary_cos.shape[1] * 2
    else:
        rotary_dim = 0
    if block_table is not None:
        stride, page, rows = block_table.shape[1], k_cache.shape[1], 0
        if flags.flag("FC_DEBUG_KERNEL_INSTANCE"):  # the table must hold the sequences WITH their new tokens
            grown = seqlen_k + ((cu_seqlens_knew[1:] - cu_seqlens_knew[:-1]) if packed else n)
            validate_paged(seqlen_k=grown.to(torch.int32), block_table=block_table if _read_table is None else _read_table,
                           num_total_pages=k_cache.shape[0], page_size=page, check=True)
    else:
        stride, page, rows = 0, 0, k_cache.shape[1]
    args = (_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(knew), _ptr(vnew), _ptr(seqlen_k), _ptr(cu_seqlens_knew), n,
            _ptr(rotary_cos), _ptr(rotary_sin), rotary_dim, rope_mode, int(bool(has_mask)), _ptr(block_table), stride, page,
            _ptr(cache_batch_idx), rows, B, Hq, Hk, D, Dv, _dtype_id(knew))
    if kv_fp8:
        if not (float(k_descale) > 0.0 and float(v_descale) > 0.0 and math.isfinite(k_descale) and math.isfinite(v_descale)):
            raise ValueError("k_descale and v_descale must be positive and finite")
        at = _lib.Attrs()
        at.size = ctypes.sizeof(_lib.Attrs)
        at.kv_dtype, at.k_descale, at.v_descale = 1, float(k_descale), float(v_descale)  # flashck::DataType FLOAT8
        _call("fck_fmha_fwd_appendkv_attrs", *args, ctypes.byref(at), _stream())
    else:
        _call("fck_fmha_fwd_appendkv", *args, _stream())


def _usable_prefill_variant(variant, head_dim, v_head_dim, max_seqlen_q, page_size):
    """A cached tile variant is a hint (the problem class is coarser than the variant's preconditions): variants 2..4
    need the ping-pong kernel, i.e. equal head dims of 64 or 128, query runs longer than 128 and pages a multiple of 64."""
    variant = int(variant)
    if variant in (2, 3, 4):
        ok = head_dim == v_head_dim and head_dim in (64, 128) and max_seqlen_q > 128 and page_size % 64 == 0
        return variant if ok else 0
    return variant if variant == 1 else 0


def tune_prefill_variant(q, k_cache, v_cache, cu_seqlens_q, kv_indptr, kv_page_indices, kv_last_page_lens=None, *, max_seqlen_q: int,
                         variants=(1, 2, 3, 4), cache=None, **kwargs) -> dict:
    """Time fmha_batch_prefill with each tile variant on these tensors and record the fastest for the problem class (see
    utils/tuning.py); later calls on problems of that class with prefill_variant = 0 use it.  Returns the record."""
    tq, Hq, D = q.shape
    _, page, Hk, Dv = v_cache.shape
    mask_type = kwargs.get("mask_type", MASK_BOTTOM_RIGHT)
    problem = tuning.prefill_problem(Hq, Hk, D, max_seqlen_q, tq, page, "fp16" if q.dtype == torch.float16 else "bf16", mask_type)
    out = torch.empty(tq, Hq, Dv, dtype=q.dtype, device=q.device)

    def run(variant):
        fmha_batch_prefill(q, k_cache, v_cache, cu_seqlens_q, kv_indptr, kv_page_indices, kv_last_page_lens, max_seqlen_q=max_seqlen_q,
                           out=out, prefill_variant=variant, **kwargs)
        return _lib.load().fck_fmha_last_kernel().decode()

    return tuning.tune_prefill_variant(run, tuning.gpu_timer, variants, problem, cache=cache)


def fmha_batch_prefill(q, k_cache, v_cache, cu_seqlens_q, kv_indptr, kv_page_indices, kv_last_page_lens=None, *,
                       max_seqlen_q: int, scale: float = 0.0, mask_type: int = MASK_BOTTOM_RIGHT, window=(-1, 0),
                       out=None, bias=None, alibi_slopes=None, logits_soft_cap: float = 0.0, k_descale: float = 1.0,
                       v_descale: float = 1.0, prefill_variant: int = 0, o_scale: float = 1.0, lse=None) -> torch.Tensor:
    """Varlen prefill over a page list: q [total_q,Hq,D]; sequence b owns pages
    kv_page_indices[kv_indptr[b]:kv_indptr[b+1]] of the cache [num_pages, page_size, Hk, D].  The caches may be
    torch.float8_e4m3fn with the static scales k_descale / v_descale (value = descale * stored); with float8_e4m3fn
    queries as well (the all-fp8 roles) the output is float8_e4m3fn, saturate(o_scale * result)."""
    _check_tensor("q", q, ndim=3)
    kv_fp8 = isinstance(k_cache, torch.Tensor) and k_cache.dtype == torch.float8_e4m3fn
    _check_tensor("k_cache", k_cache, dtype=torch.float8_e4m3fn if kv_fp8 else q.dtype, ndim=4)
    _check_tensor("v_cache", v_cache, dtype=torch.float8_e4m3fn if kv_fp8 else q.dtype, ndim=4)
    for name, t in (("cu_seqlens_q", cu_seqlens_q), ("kv_indptr", kv_indptr), ("kv_page_indices", kv_page_indices)):
        _check_tensor(name, t, dtype=torch.int32, ndim=1)
    _check_tensor("kv_last_page_lens", kv_last_page_lens, dtype=torch.int32, ndim=1, optional=True)
    B = cu_seqlens_q.numel() - 1
    if kv_indptr.numel() != B + 1:
        raise ValueError("kv_indptr must have batch + 1 entries")
    tq, Hq, D = q.shape
    _check_kv(q, k_cache, v_cache, 4)
    if kv_last_page_lens is not None and kv_last_page_lens.numel() != B:
        raise ValueError(f"kv_last_page_lens must have {B} entries, got {kv_last_page_lens.numel()}")
    num_pages, page, Hk, Dv = v_cache.shape
    o = _out("out", out, (tq, Hq, Dv), q.dtype, q)
    wl, wr = _window(window)
    _debug_validate(kv_indptr=kv_indptr, kv_page_indices=kv_page_indices, kv_last_page_lens=kv_last_page_lens,
                    num_total_pages=num_pages, page_size=page)
    plain = bias is None and alibi_slopes is None and not logits_soft_cap and not kv_fp8
    if not prefill_variant and plain:   # a tuned tile variant for this class of problems, if one is recorded and fits
        prefill_variant = _usable_prefill_variant(tuning.choose_prefill_variant(tuning.prefill_problem(
            Hq, Hk, D, max_seqlen_q, tq, page, "fp16" if q.dtype == torch.float16 else "bf16", mask_type)), D, Dv, max_seqlen_q, page)
    at, keep = _attrs(q, bias, alibi_slopes, logits_soft_cap, True, B, tq, 1, kv_fp8, k_descale, v_descale,
                      prefill_variant=prefill_variant, o_scale=o_scale, lse=lse)
    if at is None:
        _call("fck_fmha_batch_prefill", _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(o), _ptr(cu_seqlens_q), _ptr(kv_indptr),
              _ptr(kv_page_indices), _ptr(kv_last_page_lens), num_pages, page, B, Hq, Hk, D, Dv, max_seqlen_q,
              _scale(scale, D), wl, wr, mask_type, _dtype_id(q), _stream())
    else:
        _call("fck_fmha_batch_prefill_attrs", _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(o), _ptr(cu_seqlens_q), _ptr(kv_indptr),
              _ptr(kv_page_indices), _ptr(kv_last_page_lens), num_pages, page, B, Hq, Hk, D, Dv, max_seqlen_q,
              _scale(scale, D), wl, wr, mask_type, _dtype_id(q), at, _stream())
    del keep
    return o


def fmha_fwd_pagedkv(q, k_cache, v_cache, seqlen_k, block_table, *, cu_seqlens_q=None, max_seqlen_q: int = 0,
                     scale: float = 0.0, mask_type: int = MASK_BOTTOM_RIGHT, window=(-1, 0), out=None, bias=None,
                     alibi_slopes=None, logits_soft_cap: float = 0.0, k_descale: float = 1.0, v_descale: float = 1.0,
                     prefill_variant: int = 0, o_scale: float = 1.0, lse=None) -> torch.Tensor:
    """Prefill over a block table (no splits): q [B,sq,Hq,D] or packed [total_q,Hq,D].  The caches may be
    torch.float8_e4m3fn with the static scales k_descale / v_descale (value = descale * stored); float8_e4m3fn queries
    and o_scale: see fmha_batch_prefill."""
    group = cu_seqlens_q is not None
    _check_tensor("q", q, ndim=3 if group else 4)
    kv_fp8 = isinstance(k_cache, torch.Tensor) and k_cache.dtype == torch.float8_e4m3fn
    _check_tensor("k_cache", k_cache, dtype=torch.float8_e4m3fn if kv_fp8 else q.dtype, ndim=4)
    _check_tensor("v_cache", v_cache, dtype=torch.float8_e4m3fn if kv_fp8 else q.dtype, ndim=4)
    _check_tensor("seqlen_k", seqlen_k, dtype=torch.int32, ndim=1)
    _check_tensor("block_table", block_table, dtype=torch.int32, ndim=2)
    _check_tensor("cu_seqlens_q", cu_seqlens_q, dtype=torch.int32, ndim=1, optional=True)
    B = seqlen_k.numel()
    Hq, D = q.shape[-2], q.shape[-1]
    _check_kv(q, k_cache, v_cache, 4)
    if block_table.shape[0] != B:
        raise ValueError(f"block_table must be [batch, max_pages_per_seq] with batch {B}, got {tuple(block_table.shape)}")
    if (cu_seqlens_q.numel() - 1 if group else q.shape[0]) != B:
        raise ValueError("seqlen_k must have one entry per sequence of q")
    _, page, Hk, Dv = v_cache.shape
    sq = 0 if group else q.shape[1]
    if group and max_seqlen_q <= 0:
        raise ValueError("group mode needs max_seqlen_q")
    o = _out("out", out, (*q.shape[:-1], Dv), q.dtype, q)
    wl, wr = _window(window)
    _debug_validate(seqlen_k=seqlen_k, block_table=block_table, num_total_pages=k_cache.shape[0], page_size=page)
    at, keep = _attrs(q, bias, alibi_slopes, logits_soft_cap, group, B, q.shape[0] if group else sq, 1, kv_fp8, k_descale, v_descale,
                      prefill_variant=prefill_variant, o_scale=o_scale, lse=lse)
    if at is None:
        _call("fck_fmha_fwd_pagedkv", _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(o), _ptr(cu_seqlens_q), _ptr(seqlen_k),
              _ptr(block_table), block_table.shape[1], page, B, sq, Hq, Hk, D, Dv, max_seqlen_q or sq, _scale(scale, D), wl, wr,
              mask_type, _dtype_id(q), _stream())
    else:
        _call("fck_fmha_fwd_pagedkv_attrs", _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(o), _ptr(cu_seqlens_q), _ptr(seqlen_k),
              _ptr(block_table), block_table.shape[1], page, B, sq, Hq, Hk, D, Dv, max_seqlen_q or sq, _scale(scale, D), wl, wr,
              mask_type, _dtype_id(q), at, _stream())
    del keep
    return o


def _auto_num_splits(batch, q_num_heads, kv_num_heads, seqlen_q, max_seqlen_k, head_dim, page_size, dtype):
    """(split count, kernel variant): the tuned pair recorded for this class of problems if there is one, else the
    heuristic split count and variant 0 (the library's choice)."""
    return tuning.choose_splitkv(
        lambda: num_splits_heuristic(batch, q_num_heads, kv_num_heads, seqlen_q, max_seqlen_k, head_dim),
        batch, q_num_heads, kv_num_heads, seqlen_q, max_seqlen_k, head_dim, page_size,
        "fp16" if dtype == torch.float16 else "bf16")


def _usable_variant(variant, q_num_heads, kv_num_heads, rows, head_dim, v_head_dim, plain=True, page_size=128):
    """A kernel variant from the tuning cache is a hint: the record's problem class is coarser than what the variant
    needs (query counts are bucketed, v_head_dim is not part of the key), so its preconditions are checked again for
    this call, and 0 (the library's choice) is returned when one fails.  Head pairs (2) need an even number of KV heads,
    equal head dims of 64 or 128 and at most 16 packed query rows (queries x heads per KV head); a record is only served to
    the kind of call it was measured with (plain: no score modifier, 16-bit cache); one head per workgroup (1) fits
    every call.  Variants 3 / 4 (splits of equal size) are 1 / 2 for plain calls with at most 16 packed rows, head dim 64
    or 128 and pages a multiple of 32 keys."""
    variant = int(variant)
    g = q_num_heads // max(kv_num_heads, 1)
    small = plain and head_dim == v_head_dim and head_dim in (64, 128) and rows * g <= 16
    if variant in (2, 4):
        return variant if small and kv_num_heads % 2 == 0 and (variant == 2 or page_size % 32 == 0) else 0
    if variant == 3:
        return 3 if small and page_size % 32 == 0 else 0
    return variant if variant == 1 else 0


def fmha_decode_paged(q, k_cache, v_cache, seqlen_k, block_table, *, num_splits: int = 0, max_seqlen_k: int = 0,
                      cu_seqlens_q=None, max_seqlen_q: int = 0, scale: float = 0.0, mask_type: int = MASK_NONE,
                      window=(-1, -1), workspace=None, out=None, fused: bool = False, bias=None, alibi_slopes=None,
                      logits_soft_cap: float = 0.0, k_descale: float = 1.0, v_descale: float = 1.0,
                      decode_variant: int = 0, lse=None) -> torch.Tensor:
    """Paged decode = split-KV forward + LSE combine; num_splits = 0 asks the tuning cache, then the heuristic (needs
    max_seqlen_k); a cached record also brings the kernel variant it was measured with.  bias / alibi_slopes /
    logits_soft_cap / fp8 caches with k_descale, v_descale: as fmha_fwd_splitkv (not with fused = True).  lse: see
    fmha_fwd_splitkv_combine (not with fused = True either).

    fused = True runs both in one launch that allocates nothing (fmha_fwd_splitkv_fused; the partial results then live
    in the library's fixed device array, `workspace` is not used, and problems beyond its limits raise)."""
    group = cu_seqlens_q is not None
    _check_tensor("q", q, ndim=3 if group else 4)
    kv_fp8 = isinstance(k_cache, torch.Tensor) and k_cache.dtype == torch.float8_e4m3fn
    _check_tensor("k_cache", k_cache, dtype=torch.float8_e4m3fn if kv_fp8 else q.dtype, ndim=4)
    _check_tensor("v_cache", v_cache, dtype=torch.float8_e4m3fn if kv_fp8 else q.dtype, ndim=4)
    _check_tensor("seqlen_k", seqlen_k, dtype=torch.int32, ndim=1)
    _check_tensor("block_table", block_table, dtype=torch.int32, ndim=2)
    Hq, D = q.shape[-2], q.shape[-1]
    Hk = k_cache.shape[2]
    B = seqlen_k.numel()
    sq = max_seqlen_q if group else q.shape[1]
    plain = bias is None and alibi_slopes is None and not logits_soft_cap and not kv_fp8
    if workspace is not None and num_splits <= 0:
        # the partials are laid out for one split count: with a caller-owned workspace that count is the workspace's
        num_splits = int(workspace[0].shape[2]) if workspace[0].dim() == 5 else 0
        if num_splits <= 0:
            raise ValueError("workspace must be (o_acc [Bs,Hq,ns,Sq,Dv], lse_acc [Bs,Hq,ns,Sq])")
    if num_splits <= 0:
        if max_seqlen_k <= 0:
            max_seqlen_k = block_table.shape[1] * k_cache.shape[1]
        num_splits, cached_variant = _auto_num_splits(B, Hq, Hk, sq, max_seqlen_k, D, k_cache.shape[1], q.dtype)
        if not decode_variant:
            decode_variant = _usable_variant(cached_variant, Hq, Hk, sq, D, v_cache.shape[3], plain, k_cache.shape[1])
    if fused:
        if not plain or decode_variant or lse is not None:
            raise NotImplementedError("the fused launch takes no bias / soft cap / fp8 cache / kernel variant / lse")
        return fmha_fwd_splitkv_fused(q, k_cache, v_cache, num_splits, seqlen_k=seqlen_k, block_table=block_table,
                                      cu_seqlens_q=cu_seqlens_q, max_seqlen_q=max_seqlen_q, scale=scale,
                                      mask_type=mask_type, window=window, out=out)
    o_acc, lse_acc = workspace if workspace is not None else (None, None)
    o_acc, lse_acc = fmha_fwd_splitkv(q, k_cache, v_cache, num_splits, seqlen_k=seqlen_k, block_table=block_table,
                                      cu_seqlens_q=cu_seqlens_q, max_seqlen_q=max_seqlen_q, scale=scale,
                                      mask_type=mask_type, window=window, o_acc=o_acc, lse_acc=lse_acc, bias=bias,
                                      alibi_slopes=alibi_slopes, logits_soft_cap=logits_soft_cap, k_descale=k_descale,
                                      v_descale=v_descale, decode_variant=decode_variant, max_seqlen_k=max_seqlen_k)
    return fmha_fwd_splitkv_combine(lse_acc, o_acc, q.dtype, cu_seqlens_q=cu_seqlens_q, max_seqlen_q=max_seqlen_q, out=out, lse=lse)


def tune_decode_num_splits(q, k_cache, v_cache, seqlen_k, block_table, *, max_seqlen_k: int,
                           candidates=(1, 2, 4, 8, 16, 32, 64), variants=(0,), cache=None, **kwargs) -> dict:
    """Time `fmha_decode_paged` with each candidate (split count, kernel variant) on these tensors and record the
    fastest for the problem class (see utils/tuning.py); later calls with num_splits = 0 on problems of that class use
    both.  variants: 0 = the library's own choice, 1 = one KV head per workgroup, 2 = head pairs (skipped where the
    problem cannot take it).  cache: the tuning.TuningCache to record into (default: the process-wide one).  Returns
    the record ({"num_splits", "variant", "kernel", "latency_us", "tried_us", ...})."""
    Hq, D = q.shape[-2], q.shape[-1]
    Hk, page = k_cache.shape[2], k_cache.shape[1]
    B = seqlen_k.numel()
    sq = kwargs.get("max_seqlen_q", 0) or (q.shape[1] if q.dim() == 4 else 1)
    problem = tuning.splitkv_problem(B, Hq, Hk, sq, max_seqlen_k, D, page, "fp16" if q.dtype == torch.float16 else "bf16")
    ws = {}

    def run(ns, variant=0):
        if ns not in ws:
            shape_batch, shape_sq = (1, q.shape[0]) if q.dim() == 3 else (q.shape[0], q.shape[1])
            ws[ns] = splitkv_workspace(shape_batch, Hq, shape_sq, v_cache.shape[3], ns, q.device)
        fmha_decode_paged(q, k_cache, v_cache, seqlen_k, block_table, num_splits=ns, max_seqlen_k=max_seqlen_k,
                          workspace=ws[ns], decode_variant=variant, **kwargs)
        return _lib.load().fck_fmha_last_kernel().decode()

    return tuning.tune_num_splits(run, tuning.gpu_timer, candidates, problem, cache=cache, variants=variants)


class DecodeWorkspace:
    """Buffers a decode step needs besides its inputs and outputs, kept between steps.

    Holds the split-KV partials (o_acc, lse_acc) and the advanced key counts.  Buffers are only reallocated when a
    step needs a larger one, so a serving loop with a fixed batch allocates on its first step only.  A buffer that was outgrown
    stays allocated as long as the workspace: a graph captured with it writes to it at every replay.  One workspace serves one
    stream at a time.
    """

    def __init__(self):
        self._outgrown = []
        self._o_acc = None
        self._lse_acc = None
        self._seqlen = None
        self._counts = None

    def _fit(self, buf, numel, dtype, device):
        fits = lambda x: x.numel() >= numel and x.dtype == dtype and x.device == device
        if buf is None:
            return torch.empty(numel, dtype=dtype, device=device)
        if fits(buf):
            return buf
        self._outgrown.append(buf)
        for i, old in enumerate(self._outgrown):
            if fits(old):
                return self._outgrown.pop(i)
        # half as much again at least: what was outgrown then adds up to less than twice the buffer in use
        if buf.dtype == dtype and buf.device == device:
            numel = max(numel, buf.numel() * 3 // 2)
        return torch.empty(numel, dtype=dtype, device=device)

    def partials(self, shape_batch, q_num_heads, num_splits, shape_seqlen_q, v_head_dim, device):
        n_lse = shape_batch * q_num_heads * num_splits * shape_seqlen_q
        self._o_acc = self._fit(self._o_acc, n_lse * v_head_dim, torch.float32, device)
        self._lse_acc = self._fit(self._lse_acc, n_lse, torch.float32, device)
        o_acc = self._o_acc[:n_lse * v_head_dim].view(shape_batch, q_num_heads, num_splits, shape_seqlen_q, v_head_dim)
        lse_acc = self._lse_acc[:n_lse].view(shape_batch, q_num_heads, num_splits, shape_seqlen_q)
        return o_acc, lse_acc

    def lengths(self, batch, device):
        self._seqlen = self._fit(self._seqlen, batch, torch.int32, device)
        self._counts = self._fit(self._counts, batch, torch.int32, device)
        return self._seqlen[:batch], self._counts[:batch]


def fmha_decode_step(q, knew, vnew, k_cache, v_cache, seqlen_k, block_table, *, cu_seqlens_knew=None,
                     max_seqlen_knew: int = 0, rotary_cos=None, rotary_sin=None, rope_mode: int = ROPE_NONE,
                     num_splits: int = 0, max_seqlen_k: int = 0, scale: float = 0.0, window_left: int = -1,
                     workspace: Optional[DecodeWorkspace] = None, out=None, k_descale: float = 1.0, v_descale: float = 1.0,
                     prefix_lens=None, cu_groups=None, max_group_size: int = 0, max_prefix_len: int = 0, lse=None):
    """One serving step over a paged cache: append the new tokens, then attend from them.

    The caller side of the split-KV path, FmhaKind::FwdAppendKV -> FwdSplitKV -> FwdSplitKVCombine
    (core/profiling/attention/fmha_library.h:17-25), with the argument set of AttentionLayer
    (core/module/layers/attention_layers/attention_layer.h:13-35):
      1. knew is rotated and knew/vnew are written behind the seqlen_k[b] tokens of each sequence; q is rotated in
         place at the same positions;
      2. the split count comes from the CU count and the longest possible KV length unless num_splits is given;
      3. split-KV forward over the seqlen_k[b] + n_b keys now in the cache - query i of a sequence sees keys up to
         its own position (bottom-right causal; window_left >= 0 adds a sliding window) - and the LSE combine.
    q/knew/vnew are [B, n, H, D] (n new tokens everywhere) or packed [total_new, H, D] with cu_seqlens_knew and
    max_seqlen_knew.  Nothing is read back from the GPU, so a step only enqueues work on the current stream.
    prefix_lens (with cu_groups, max_group_size, max_prefix_len: see fmha_decode_shared_prefix): the sequences share
    prefixes, and step 3 reads each of them once per group; num_splits is then the split count of the tokens behind them.
    lse (fp32 [B,Hq,n] or [Hq,total_new], optional) receives the log-sum-exp of every row (what fmha_key_weights takes).
    With torch.float8_e4m3fn caches the new rows are quantised on their way in and dequantised by the attention
    kernel, both with the static scales k_descale / v_descale.

    Returns (o, seqlen_k_new): o has q's shape (with Dv); seqlen_k_new = seqlen_k + n_b lives in the workspace and is
    overwritten by the next step; seqlen_k itself is not modified.
    """
    packed = cu_seqlens_knew is not None
    ws = workspace if workspace is not None else DecodeWorkspace()
    B = seqlen_k.numel()
    Hq, D = q.shape[-2], q.shape[-1]
    Hk, Dv = k_cache.shape[2], v_cache.shape[3]
    page = k_cache.shape[1]
    if packed:
        if max_seqlen_knew <= 0:
            raise ValueError("packed new tokens need max_seqlen_knew")
        n = int(max_seqlen_knew)
    else:
        if q.dim() != 4:
            raise ValueError(f"q must be [B, n, Hq, D] without cu_seqlens_knew, got shape {tuple(q.shape)}")
        n = q.shape[1]
    checked = {}
    if prefix_lens is not None and flags.flag("FC_DEBUG_KERNEL_INSTANCE"):
        checked["_read_table"] = _read_entries(block_table, seqlen_k, prefix_lens, cu_groups, max_group_size, page, append=True)
    fmha_fwd_appendkv(q, k_cache, v_cache, knew, vnew, seqlen_k, cu_seqlens_knew=cu_seqlens_knew, max_seqlen_knew=n,
                      rotary_cos=rotary_cos, rotary_sin=rotary_sin, rope_mode=rope_mode, has_mask=True,
                      block_table=block_table, k_descale=k_descale, v_descale=v_descale, **checked)
    kv_fp8 = k_cache.dtype == torch.float8_e4m3fn
    seqlen_new, counts = ws.lengths(B, seqlen_k.device)
    if packed:
        torch.sub(cu_seqlens_knew[1:], cu_seqlens_knew[:-1], out=counts)
        torch.add(seqlen_k, counts, out=seqlen_new)
    else:
        torch.add(seqlen_k, n, out=seqlen_new)
    # a lone new token sees every key: no mask needed unless a sliding window is asked for
    if n == 1 and window_left < 0:
        mask_type, window = MASK_NONE, (-1, -1)
    else:
        mask_type, window = MASK_BOTTOM_RIGHT, (int(window_left), 0)
    if prefix_lens is not None:
        o = fmha_decode_shared_prefix(q, k_cache, v_cache, seqlen_new, block_table, prefix_lens, cu_groups=cu_groups,
                                      max_group_size=max_group_size, max_prefix_len=max_prefix_len, max_seqlen_k=max_seqlen_k,
                                      num_splits=num_splits, cu_seqlens_q=cu_seqlens_knew, max_seqlen_q=n if packed else 0,
                                      scale=scale, mask_type=mask_type, window=window, k_descale=k_descale, v_descale=v_descale,
                                      workspace=ws, out=out, lse=lse)
        return o, seqlen_new
    if num_splits <= 0:
        if max_seqlen_k <= 0:
            max_seqlen_k = block_table.shape[1] * page  # what the block table can address
        num_splits, decode_variant = _auto_num_splits(B, Hq, Hk, n, max_seqlen_k, D, page, q.dtype)
        decode_variant = _usable_variant(decode_variant, Hq, Hk, n, D, Dv, plain=not kv_fp8, page_size=page)
    else:
        decode_variant = 0
    shape_batch, shape_sq = (1, q.shape[0]) if packed else (B, n)
    o_acc, lse_acc = ws.partials(shape_batch, Hq, num_splits, shape_sq, Dv, q.device)
    fmha_fwd_splitkv(q, k_cache, v_cache, num_splits, seqlen_k=seqlen_new, block_table=block_table,
                     cu_seqlens_q=cu_seqlens_knew, max_seqlen_q=n if packed else 0, scale=scale, mask_type=mask_type,
                     window=window, o_acc=o_acc, lse_acc=lse_acc, decode_variant=decode_variant, k_descale=k_descale,
                     v_descale=v_descale, max_seqlen_k=max_seqlen_k)
    extra = {} if lse is None else {"lse": lse}
    o = fmha_fwd_splitkv_combine(lse_acc, o_acc, q.dtype, cu_seqlens_q=cu_seqlens_knew, max_seqlen_q=n if packed else 0,
                                 out=out, **extra)
    return o, seqlen_new


def shared_prefix_splits(batch, num_groups, max_group_size, q_num_heads, kv_num_heads, seqlen_q, head_dim, max_prefix_len,
                         max_own_len, num_cu=0) -> Tuple[int, int]:
    """(prefix splits, own splits) from the CU count, the longest prefix and the most keys behind one.  By default
    fmha_decode_shared_prefix takes these, and more own splits where a sequence without the longest prefix may need them."""
    ns = (ctypes.c_int32(), ctypes.c_int32())
    _call("fck_fmha_shared_prefix_splits", batch, num_groups, max_group_size, q_num_heads, kv_num_heads, seqlen_q, head_dim,
          max_prefix_len, max_own_len, num_cu, ctypes.byref(ns[0]), ctypes.byref(ns[1]))
    return ns[0].value, ns[1].value


def _default_shared_prefix_splits(batch, num_groups, max_group_size, q_num_heads, kv_num_heads, seqlen_q, head_dim, prefix, own, longest):
    """Split counts of a call whose sequences have up to `longest` keys, most of them `own` behind a prefix of `prefix`.

    Nothing says that every sequence has the longest prefix: one without any owns `longest` keys.  So there are at least as many
    own splits as the decode without sharing takes, twice as many where it splits at all, of 2048 keys or more.  32 sequences
    of which one has 33000 keys and no prefix, the others 32768 shared ones: 210 us, without this 741 us, not shared 318 us."""
    ns_prefix, ns_own = shared_prefix_splits(batch, num_groups, max_group_size, q_num_heads, kv_num_heads, seqlen_q, head_dim, prefix, own)
    alone = num_splits_heuristic(batch, q_num_heads, kv_num_heads, seqlen_q, longest, head_dim)
    most = min(2 * alone if alone > 1 else 1, -(-longest // 2048), 64)
    return ns_prefix, max(ns_own, most)


# The split counts are functions of the shapes and the CU count alone: decided once per shape.
_shared_prefix_splits = functools.lru_cache(maxsize=1024)(lambda device, *sizes: _default_shared_prefix_splits(*sizes))
_key_weights_row_splits = functools.lru_cache(maxsize=1024)(
    lambda device, *sizes: int(_lib.load().fck_fmha_key_weights_row_splits(*sizes, 0)))
_evict_workspace_bytes = functools.lru_cache(maxsize=1024)(
    lambda device, *sizes: int(_lib.load().fck_fmha_cache_evict_workspace_bytes(*sizes, 0)))


def _check_same_device(like, **tensors):
    device = like.device
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, the inputs are on {device}")


_HERE = contextlib.nullcontext()


def _on(t):
    """The device of t made current for a launch (the C ABI launches on the current device and its current stream)."""
    return torch.cuda.device(t.device) if t.is_cuda and t.device.index != torch.cuda.current_device() else _HERE


def _at(t):
    """Address of an optional tensor, for arguments declared as pointers."""
    return None if t is None else t.data_ptr()


def _cache_dtype(q, cache):
    """(element type a cache next to q must have, whether it is the quantised one)"""
    kv_fp8 = isinstance(cache, torch.Tensor) and cache.dtype == torch.float8_e4m3fn
    return (torch.float8_e4m3fn if kv_fp8 else q.dtype), kv_fp8


def _check_queries(q, cu_seqlens_q, max_seqlen_q, batch):
    """(group mode, rows of a head, most query tokens of a sequence) of a query tensor"""
    group = cu_seqlens_q is not None
    _check_tensor("q", q, ndim=3 if group else 4)
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"q must be torch.float16 or torch.bfloat16, got {q.dtype}")
    if q.numel() == 0:
        raise ValueError("Input tensor cannot be empty")
    _check_tensor("cu_seqlens_q", cu_seqlens_q, dtype=torch.int32, ndim=1, optional=True)
    if (cu_seqlens_q.numel() - 1 if group else q.shape[0]) != batch:
        raise ValueError("seqlen_k must have one entry per sequence of q")
    if group and max_seqlen_q <= 0:
        raise ValueError("group mode needs max_seqlen_q")
    return group, (q.shape[0] if group else q.shape[1]), (int(max_seqlen_q) if group else q.shape[1])


def fmha_decode_shared_prefix(q, k_cache, v_cache, seqlen_k, block_table, prefix_lens, *, cu_groups=None, max_group_size: int = 0,
                              max_prefix_len: int = 0, max_seqlen_k: int = 0, num_prefix_splits: int = 0, num_splits: int = 0,
                              cu_seqlens_q=None, max_seqlen_q: int = 0, scale: float = 0.0, mask_type: int = MASK_NONE,
                              window=(-1, -1), alibi_slopes=None, logits_soft_cap: float = 0.0, k_descale: float = 1.0,
                              v_descale: float = 1.0, workspace: Optional["DecodeWorkspace"] = None, out=None,
                              lse=None) -> torch.Tensor:
    """Paged decode attention of a batch whose sequences share prefixes: the result of fmha_decode_paged on the same tensors,
    with every shared prefix read once per group instead of once per sequence.

    Group g holds the sequences cu_groups[g] .. cu_groups[g+1] - 1 (int32 [G+1], non-decreasing; None: one group, the whole
    batch) and its sequences have their first prefix_lens[g] tokens (int32 [G], any count) in common.  They are read through
    the block-table row of the group's first sequence; seqlen_k counts them like all other tokens.
    Host-side bounds, all optional: max_group_size (sequences of a group beyond it read their own keys), max_prefix_len and
    max_seqlen_k.  The last two only steer the split counts num_prefix_splits / num_splits (0 = chosen from them and the CU
    count): a split is an equal part of the keys there are, so bounds that are loose or missing cost a few empty partial results
    (32 sequences on 4096 shared keys: 25 us with exact bounds, 32 us with a table for 32768 keys and none).
    q, masks, windows, ALiBi, soft cap and quantised caches as fmha_decode_paged; no elementwise bias.  workspace keeps the
    partial results between steps; lse (fp32 [B,Hq,sq] or [Hq,total_q], optional) receives the log-sum-exp of every row."""
    _check_tensor("seqlen_k", seqlen_k, dtype=torch.int32, ndim=1)
    B = seqlen_k.numel()
    group, sq, sq_max = _check_queries(q, cu_seqlens_q, max_seqlen_q, B)
    cache_dtype, kv_fp8 = _cache_dtype(q, k_cache)
    _check_tensor("k_cache", k_cache, dtype=cache_dtype, ndim=4)
    _check_tensor("v_cache", v_cache, dtype=cache_dtype, ndim=4)
    _check_tensor("block_table", block_table, dtype=torch.int32, ndim=2)
    _check_tensor("prefix_lens", prefix_lens, dtype=torch.int32, ndim=1)
    _check_tensor("cu_groups", cu_groups, dtype=torch.int32, ndim=1, optional=True)
    _check_kv(q, k_cache, v_cache, 4)
    if block_table.shape[0] != B:
        raise ValueError(f"block_table must be [batch, max_pages_per_seq] with batch {B}, got {tuple(block_table.shape)}")
    G = prefix_lens.numel()
    if G < 1 or (G != 1 if cu_groups is None else cu_groups.numel() != G + 1):
        raise ValueError(f"prefix_lens must have one entry per group ({G}), cu_groups one more"
                         f" ({None if cu_groups is None else cu_groups.numel()}; without it there is one group)")
    _check_same_device(q, k_cache=k_cache, v_cache=v_cache, seqlen_k=seqlen_k, block_table=block_table, prefix_lens=prefix_lens,
                       cu_groups=cu_groups, cu_seqlens_q=cu_seqlens_q, alibi_slopes=alibi_slopes)
    Hq, D = q.shape[-2], q.shape[-1]
    page, Hk, Dv = k_cache.shape[1], k_cache.shape[2], v_cache.shape[3]
    capacity = block_table.shape[1] * page
    if capacity == 0:
        raise ValueError("block_table must have at least one page per sequence")
    # sequences of a group: at most (0: any number), and as a rule
    max_group_size = int(max_group_size) if 0 < max_group_size < B else 0
    typical = max_group_size or -(-B // G)
    # the longest prefix, and the keys a sequence that has it has behind it; they steer the splits and nothing else
    longest = min(max_seqlen_k, capacity) if max_seqlen_k > 0 else capacity
    prefix = min(max_prefix_len, longest) if max_prefix_len > 0 else longest
    own = max(longest - prefix, 1)
    if num_prefix_splits <= 0 or num_splits <= 0:
        ns = _shared_prefix_splits(q.device, B, G, typical, Hq, Hk, sq_max, max(D, Dv), prefix, own, longest)
        num_prefix_splits = num_prefix_splits if num_prefix_splits > 0 else ns[0]
        num_splits = num_splits if num_splits > 0 else ns[1]
    if flags.flag("FC_DEBUG_KERNEL_INSTANCE"):
        validate_paged(seqlen_k=seqlen_k, block_table=_read_entries(block_table, seqlen_k, prefix_lens, cu_groups, max_group_size, page),
                       num_total_pages=k_cache.shape[0], page_size=page, check=True)
    o = _out("out", out, (*q.shape[:-1], Dv), q.dtype, q)
    if lse is not None:
        _check_tensor("lse", lse, dtype=torch.float32)
        _check_shape("lse", lse, (Hq, sq) if group else (B, Hq, sq), q)
    shape_batch, total = (1 if group else B), int(num_prefix_splits) + int(num_splits)
    rows = shape_batch * Hq * total * sq
    if workspace is not None:
        o_acc, lse_acc = (x.data_ptr() for x in workspace.partials(shape_batch, Hq, total, sq, Dv, q.device))
    else:  # one buffer: o_acc [Bs,Hq,ns,Sq,Dv] and behind it lse_acc [Bs,Hq,ns,Sq]
        partials = torch.empty(rows * (Dv + 1), dtype=torch.float32, device=q.device)
        o_acc = partials.data_ptr()
        lse_acc = o_acc + rows * Dv * 4
    wl, wr = _window(window)
    at, keep = _attrs(q, None, alibi_slopes, logits_soft_cap, group, B, sq, 1, kv_fp8, k_descale, v_descale)
    with _on(q):
        _call("fck_fmha_decode_shared_prefix", _at(q), _at(k_cache), _at(v_cache), _at(o), _at(lse), lse_acc, o_acc,
              _at(cu_seqlens_q), _at(seqlen_k), _at(block_table), _at(cu_groups), _at(prefix_lens), B, G, max_group_size, sq, Hq,
              Hk, D, Dv, sq_max, int(num_prefix_splits), int(num_splits), prefix, own, block_table.shape[1], page, _scale(scale, D), wl, wr,
              mask_type, _dtype_id(q), at, _stream())
    del keep
    return o


def fmha_key_weights(q, k_cache, lse, seqlen_k, block_table=None, *, weights=None, cu_seqlens_q=None, max_seqlen_q: int = 0,
                     max_seqlen_k: int = 0, scale: float = 0.0, mask_type: int = MASK_NONE, window=(-1, -1), alibi_slopes=None,
                     logits_soft_cap: float = 0.0, k_descale: float = 1.0, num_row_splits: int = 0, out=None) -> torch.Tensor:
    """Attention weight every cached key receives, fp32 [B, Hk, cols]:

        out[b, hk, t] = weights[b, hk, t] + sum over the query heads h of KV head hk and the rows i that see t of
                        exp(score(b, h, i, t) - lse[b, h, i])

    lse (fp32 [B,Hq,sq], packed queries [Hq,total_q]) is what the attention over the same keys returned (lse= of fmha_fwd,
    fmha_batch_prefill, fmha_fwd_pagedkv, fmha_decode_paged, fmha_decode_shared_prefix); rows with -inf add nothing.
    k_cache is a paged cache with block_table, or [B, sk, Hk, D] without one (seqlen_k may then be None).
    weights (optional) are what earlier steps accumulated; out may be the same tensor.  cols is their last dimension, else
    max_seqlen_k, else what the cache can hold.  Entries at and behind a sequence's key count are written as 0, so the tensor
    can go on growing with its cache.  Masks, windows, ALiBi, soft cap and quantised keys as the attention operators.
    num_row_splits: runs a long stretch of queries is cut into (0: chosen from the CU count)."""
    if seqlen_k is None and block_table is not None:
        raise ValueError("a paged cache needs seqlen_k")
    _check_tensor("seqlen_k", seqlen_k, dtype=torch.int32, ndim=1, optional=True)
    if not isinstance(k_cache, torch.Tensor):
        raise TypeError(f"Expected k_cache to be a torch.Tensor, got {type(k_cache)}")
    B = seqlen_k.numel() if seqlen_k is not None else k_cache.shape[0]
    group, sq, sq_max = _check_queries(q, cu_seqlens_q, max_seqlen_q, B)
    cache_dtype, kv_fp8 = _cache_dtype(q, k_cache)
    _check_tensor("k_cache", k_cache, dtype=cache_dtype, ndim=4)
    _check_tensor("block_table", block_table, dtype=torch.int32, ndim=2, optional=True)
    _check_kv(q, k_cache, k_cache, 3 if k_cache.dim() == 3 else 4)
    Hq, D, Hk = q.shape[-2], q.shape[-1], k_cache.shape[2]
    if block_table is not None:
        if block_table.shape[0] != B:
            raise ValueError(f"block_table must be [batch, max_pages_per_seq] with batch {B}, got {tuple(block_table.shape)}")
        stride, page, sk = block_table.shape[1], k_cache.shape[1], 0
        capacity = stride * page
    else:
        if k_cache.shape[0] != B:
            raise ValueError(f"k_cache {tuple(k_cache.shape)} must have one row per sequence ({B}) without a block table")
        stride, page, sk = 0, 0, k_cache.shape[1]
        capacity = sk
    _check_tensor("lse", lse, dtype=torch.float32)
    _check_shape("lse", lse, (Hq, sq) if group else (B, Hq, sq), q)
    _check_tensor("weights", weights, dtype=torch.float32, ndim=3, optional=True)
    _check_tensor("out", out, dtype=torch.float32, ndim=3, optional=True)
    given = weights if weights is not None else out
    cols = given.shape[2] if given is not None else max_seqlen_k if max_seqlen_k > 0 else capacity
    if cols <= 0 or capacity <= 0:
        raise ValueError("the cache and the weights need at least one key per sequence")
    if weights is not None:
        _check_shape("weights", weights, (B, Hk, cols), q)
    _check_same_device(q, k_cache=k_cache, seqlen_k=seqlen_k, block_table=block_table, cu_seqlens_q=cu_seqlens_q,
                       alibi_slopes=alibi_slopes)
    if block_table is not None:
        _debug_validate(seqlen_k=seqlen_k, block_table=block_table, num_total_pages=k_cache.shape[0], page_size=page)
    o = _out("out", out, (B, Hk, cols), torch.float32, q)
    if num_row_splits <= 0:
        num_row_splits = _key_weights_row_splits(q.device, B, Hq, Hk, sq_max, cols, D, mask_type)
    partial = torch.empty(num_row_splits, B, Hk, cols, dtype=torch.float32, device=q.device) if num_row_splits > 1 else None
    wl, wr = _window(window)
    at, keep = _attrs(q, None, alibi_slopes, logits_soft_cap, group, B, sq, 1, kv_fp8, k_descale, 1.0)
    with _on(q):
        _call("fck_fmha_key_weights", _at(q), _at(k_cache), _at(lse), _at(weights), _at(o), _at(partial), _at(cu_seqlens_q), _at(seqlen_k),
              _at(block_table), stride, page, B, sq, sk, cols, Hq, Hk, D, sq_max, num_row_splits, _scale(scale, D), wl, wr, mask_type, _dtype_id(q),
              at, _stream())
    del keep
    return o


def fmha_cache_evict(k_cache, v_cache, weights, seqlen_k, block_table, new_block_table, *, budget: int, recent: int = 0,
                     sinks: int = 0, new_k_cache=None, new_v_cache=None, out_seqlen=None, out_kept=None, out_weights=None):
    """Keep at most `budget` keys of every (sequence, KV head) of a paged cache and move their rows to new pages.

    A sequence of L keys keeps n = min(L, budget): all of them when L <= budget, else its first `sinks`, its last `recent` and,
    of the keys between, those with the largest weights (weights fp32 [B, Hk, cols] as fmha_key_weights accumulates them;
    equal weights: the lower position; NaN counts as -inf).  Slot j of sequence b in the pages of new_block_table (int32
    [B, pages], at least `budget` keys a row) receives, for each head, the row of its j-th kept key in ascending order.
    The rows go to new_k_cache / new_v_cache (default: the same pools); pages that block_table names are never written, as other
    sequences may share them, so new_block_table must name other pages then.  After the call the old pages can be reused.
    Heads keep different positions: masks that go by position do not apply to evicted keys any more, and an append that rotates
    (fmha_decode_step with rotary tables) takes a sequence's new, smaller key count for its position: rotate the new tokens at
    their true positions before, or pass tables whose first row is the number of keys evicted (the same for every sequence).

    Returns (seqlen_k_new int32 [B], kept int32 [B, Hk, budget] with -1 behind the n-th, weights_new fp32 [B, Hk, cols] with
    zeros behind the n-th)."""
    _check_tensor("k_cache", k_cache, ndim=4)
    _dtype_id(k_cache)
    _check_tensor("v_cache", v_cache, dtype=k_cache.dtype, ndim=4)
    _check_tensor("new_k_cache", new_k_cache, dtype=k_cache.dtype, ndim=4, optional=True)
    _check_tensor("new_v_cache", new_v_cache, dtype=k_cache.dtype, ndim=4, optional=True)
    if (new_k_cache is None) != (new_v_cache is None):
        raise ValueError("new_k_cache and new_v_cache must be given together")
    nk, nv = (k_cache, v_cache) if new_k_cache is None else (new_k_cache, new_v_cache)
    if v_cache.shape[:3] != k_cache.shape[:3]:
        raise ValueError(f"v_cache {tuple(v_cache.shape)} does not match k_cache {tuple(k_cache.shape)}")
    if nk.shape[2:] != k_cache.shape[2:] or nv.shape[2:] != v_cache.shape[2:] or nk.shape[:2] != nv.shape[:2]:
        raise ValueError(f"new_k_cache {tuple(nk.shape)} / new_v_cache {tuple(nv.shape)} do not match k_cache {tuple(k_cache.shape)} / "
                         f"v_cache {tuple(v_cache.shape)}")
    _, page, Hk, D = k_cache.shape
    _check_tensor("seqlen_k", seqlen_k, dtype=torch.int32, ndim=1)
    _check_tensor("block_table", block_table, dtype=torch.int32, ndim=2)
    _check_tensor("new_block_table", new_block_table, dtype=torch.int32, ndim=2)
    B = seqlen_k.numel()
    if B == 0 or block_table.shape[0] != B or new_block_table.shape[0] != B or block_table.shape[1] == 0:
        raise ValueError(f"block_table {tuple(block_table.shape)} and new_block_table {tuple(new_block_table.shape)} must have one row per "
                         f"sequence ({B})")
    _check_tensor("weights", weights, dtype=torch.float32, ndim=3)
    cols = weights.shape[2]
    _check_shape("weights", weights, (B, Hk, cols), k_cache)
    budget, recent, sinks = int(budget), int(recent), int(sinks)
    if budget <= 0 or recent < 0 or sinks < 0 or recent + sinks > budget:
        raise ValueError(f"budget {budget} must be positive and hold recent {recent} + sinks {sinks}")
    if new_block_table.shape[1] * nk.shape[1] < budget:
        raise ValueError(f"a row of new_block_table addresses {new_block_table.shape[1] * nk.shape[1]} keys, the budget is {budget}")
    same_pool = nk.data_ptr() == k_cache.data_ptr() or nv.data_ptr() == v_cache.data_ptr()
    if same_pool and new_block_table.data_ptr() == block_table.data_ptr():
        raise ValueError("new_block_table must name other pages than block_table: rows are not moved inside the pages that are read")
    _check_same_device(k_cache, v_cache=v_cache, new_k_cache=nk, new_v_cache=nv, seqlen_k=seqlen_k, block_table=block_table,
                       new_block_table=new_block_table)
    seqlen_new = _out("out_seqlen", out_seqlen, (B,), torch.int32, k_cache)
    kept = _out("out_kept", out_kept, (B, Hk, budget), torch.int32, k_cache)
    weights_new = _out("out_weights", out_weights, (B, Hk, cols), torch.float32, k_cache)
    if weights_new.data_ptr() == weights.data_ptr():
        raise ValueError("out_weights must not be weights")
    if seqlen_new.data_ptr() == seqlen_k.data_ptr():
        raise ValueError("out_seqlen must not be seqlen_k")
    if flags.flag("FC_DEBUG_KERNEL_INSTANCE"):
        validate_paged(seqlen_k=seqlen_k, block_table=block_table, num_total_pages=k_cache.shape[0], page_size=page, check=True)
        _validate_new_pages(seqlen_k, block_table, new_block_table, budget, page, nk, same_pool)
    space = _evict_workspace_bytes(k_cache.device, B, Hk, cols)
    space = torch.empty(space, dtype=torch.uint8, device=k_cache.device) if space else None
    with _on(k_cache):
        _call("fck_fmha_cache_evict", _at(k_cache), _at(v_cache), _at(nk), _at(nv), _at(weights), _at(weights_new), _at(space), _at(seqlen_k),
              _at(seqlen_new), _at(kept), _at(block_table), block_table.shape[1], page, _at(new_block_table), new_block_table.shape[1],
              nk.shape[1], B, Hk, D, v_cache.shape[3], cols, budget, recent, sinks, _dtype_id(k_cache), _stream())
    return seqlen_new, kept, weights_new


def _validate_new_pages(seqlen_k, block_table, new_block_table, budget, page, new_cache, same_pool):
    """The pages an eviction writes: inside the pool, each used once, and none of those it reads (debug aid; synchronises)."""
    new_page = new_cache.shape[1]
    lens, old, new = seqlen_k.tolist(), block_table.tolist(), new_block_table.tolist()
    written = [p for n, row in zip(lens, new) for p in row[:-(-max(min(n, budget), 0) // new_page)]]
    if any(p < 0 or p >= new_cache.shape[0] for p in written):
        raise ValueError(f"new_block_table names a page outside the pool of {new_cache.shape[0]}")
    if len(set(written)) != len(written):
        raise ValueError("new_block_table names a page twice")
    if same_pool and set(written) & {p for n, row in zip(lens, old) for p in row[:-(-max(n, 0) // page)]}:
        raise ValueError("new_block_table names a page that block_table reads")


register_flashck_functions(FlashCKOperationType.FMHA.value, {
    "forward": fmha_fwd,
    "forward_varlen": fmha_fwd_varlen,
    "forward_splitkv": fmha_fwd_splitkv,
    "forward_splitkv_combine": fmha_fwd_splitkv_combine,
    "forward_appendkv": fmha_fwd_appendkv,
    "batch_prefill": fmha_batch_prefill,
    "forward_pagedkv": fmha_fwd_pagedkv,
    "decode_paged": fmha_decode_paged,
    "decode_step": fmha_decode_step,
    "decode_shared_prefix": fmha_decode_shared_prefix,
    "key_weights": fmha_key_weights,
    "cache_evict": fmha_cache_evict,
})
