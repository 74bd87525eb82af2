"""Appending keys and values to the paged pools, with norms and the position rotation on the way.

The write side of the pools that ``paged_attention`` and ``quantized_paged_attention`` read.  The
reference keeps that in its cache managers (mlx_primitives/cache/paged_attention.py:44-105
takes pools that something else has filled); here it is one call (mlxp_paged_append): the new
keys, and the queries beside them, are normed (where weights are given) and rotated in fp32 and
written once, in the pools' type or as 8-bit codes.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _lib

__all__ = ["paged_append"]

# mlxp_paged_append_args: 15 pointers, 14 sizes, 17 strides, eps, stream
_ARGS = _lib.ArgStruct(49, doubles=(47,))


def _overlaps(t: torch.Tensor) -> bool:
    """Whether two elements of a strided tensor may share memory (sufficient for a view of rows)."""
    if t.is_contiguous():
        return False
    span = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride < span:
            return True
        span = stride * (size - 1) + span
    return False


def check_pools(k_pool, v_pool, k_scales, v_scales):
    """Checks that both cache operators make of the pools; returns the cache's dtype code."""
    shape, dtype, strides = k_pool.shape, k_pool.dtype, k_pool.stride()
    if len(shape) != 4 or v_pool.shape != shape:
        raise ValueError("k_pool and v_pool must both be (num_blocks, block_size, heads, head_dim)"
                         f", got {tuple(k_pool.shape)} and {tuple(v_pool.shape)}")
    if v_pool.dtype is not dtype:
        raise ValueError(f"k_pool and v_pool must share a dtype, got {k_pool.dtype} and {v_pool.dtype}")
    if v_pool.stride() != strides or strides[3] != 1:
        raise ValueError("k_pool and v_pool must have the same strides, and unit head_dim stride, "
                         f"got {k_pool.stride()} and {v_pool.stride()}")
    code = _lib.CACHE_DTYPE_CODES.get(dtype)
    if code is None:
        if k_scales is not None or v_scales is not None:
            raise ValueError(f"scales go with float8_e4m3fn or int8 pools, got {k_pool.dtype}")
        return _lib.DTYPE_CODES.get(dtype)
    dev = k_pool.get_device()
    for name, s in (("k_scales", k_scales), ("v_scales", v_scales)):
        if (s is None or s.dtype is not torch.float32 or s.shape != (shape[0], shape[2])
                or s.get_device() != dev):
            raise ValueError(f"{name} must be a float32 tensor (num_blocks, heads) = "
                             f"{(shape[0], shape[2])} beside the pools, got "
                             f"{None if s is None else (s.dtype, tuple(s.shape), s.device)}")
    if k_scales.stride() != v_scales.stride():
        raise ValueError("k_scales and v_scales must have the same strides")
    return code


def refuse_gradients(what, *tensors):
    """Raises where a call without derivatives is given tensors that want one."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"{what} is not differentiable: call it under torch.no_grad()")


def device_ints(t: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    """Tables and lengths as the kernels read them: int32 beside `like`, unit inner stride, rows that
    do not overlap (one table expanded over the batch is copied)."""
    if t.dtype is not torch.int32 or t.get_device() != like.get_device():
        if t.is_floating_point():
            raise ValueError(f"block tables and lengths must be integers, got {t.dtype}")
        t = _lib.int32(t, like.device)
    if t.is_contiguous() or (t.stride(-1) == 1 and (t.ndim < 2 or t.stride(0) >= t.shape[1])):
        return t
    return t.contiguous()


def paged_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    *,
    new_lens: Optional[torch.Tensor] = None,
    q: Optional[torch.Tensor] = None,
    cos_cache: Optional[torch.Tensor] = None,
    sin_cache: Optional[torch.Tensor] = None,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    k_scales: Optional[torch.Tensor] = None,
    v_scales: Optional[torch.Tensor] = None,
) -> Optional[torch.Tensor]:
    """Writes k, v (batch, seq, kv_heads, head_dim) into the pools in place; returns the rotated q
    (batch, seq, heads, head_dim) where one is given.

    Token i < ``new_lens``[b] (default: all) of sequence b has position ``context_lens``[b] + i
    (the tokens cached before) and goes to row position % block_size of pool block
    ``block_tables``[b, position // block_size].  Tokens whose position or block does not exist
    are dropped, as missing blocks are in ``paged_attention``; nothing else is written.  Keys and
    queries are normed with ``k_weight`` / ``q_weight`` and rotated with the tables' rows of their
    positions (each where given; the tables must cover every position of the block tables).
    Rows of q past ``new_lens`` or outside the block table come back as zeros.

    Pools: (num_blocks, block_size, kv_heads, head_dim) of k's dtype, or float8_e4m3fn or int8
    with ``k_scales``, ``v_scales`` (num_blocks, kv_heads) float32: value = code * scale.  A
    block's scale is the least power of two that holds its tokens; it is set when the block
    receives its first row and grows, its earlier codes being rescaled, when a later token needs
    it to.  A block that receives tokens must belong to one sequence (full blocks may be shared):
    the order of two writers of a block is not defined.  Not differentiable, in either mode; the
    pools and scales are marked as changed, as by any operator that writes in place.
    """
    out = _lib.calls().append(k, v, k_pool, v_pool, block_tables, context_lens, new_lens, q, cos_cache,
                              sin_cache, q_weight, k_weight, k_scales, v_scales, eps)
    if out is not None:  # else: not a call that can be made as it is
        if type(out) is int:
            _lib.check(out, "mlxp_paged_append")
        return None if out is True else out
    shape = k.shape
    if len(shape) != 4 or v.shape != shape:
        raise ValueError("k and v must both be (batch, seq, kv_heads, head_dim), got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    B, S, Hk, D = shape
    codes = _lib.DTYPE_CODES
    dtype = k.dtype
    code = codes.get(dtype)
    if code is None or v.dtype is not dtype:
        raise ValueError(f"k and v must share a dtype of float32, bfloat16, float16, got {dtype}, {v.dtype}")
    cache_code = check_pools(k_pool, v_pool, k_scales, v_scales)
    quant = k_scales is not None
    if not quant and k_pool.dtype is not dtype:
        raise ValueError(f"the pools' dtype ({k_pool.dtype}) must be k's ({dtype}) or an 8-bit one")
    num_blocks, block_size, Hp, Dp = k_pool.shape
    if Hp != Hk or Dp != D:
        raise ValueError(f"pools of (heads, head_dim) = {(Hp, Dp)} cannot take k of {(Hk, D)}")
    if D % 2 or D < 2:
        raise ValueError(f"head_dim must be even, got {D}")
    _lib.refuse_tangents("paged_append", k, v, q, k_pool, v_pool, k_scales, v_scales, q_weight, k_weight,
                         cos_cache, sin_cache)
    refuse_gradients("paged_append", k, v, q, k_pool, v_pool, k_scales, v_scales, q_weight, k_weight)
    dev = k.get_device()
    if dev < 0 or k_pool.get_device() != dev or v_pool.get_device() != dev or v.get_device() != dev:
        raise ValueError("k, v and the pools must be on one CUDA device (appending is in place)")
    if _overlaps(k_pool) or (quant and _overlaps(k_scales)):
        raise ValueError("the pools and scales must not overlap themselves (expanded views)")
    bt_shape = block_tables.shape
    if len(bt_shape) != 2 or bt_shape[0] != B:
        raise ValueError(f"block_tables must be (batch, max_blocks), got {tuple(block_tables.shape)}")
    max_blocks = bt_shape[1]
    if context_lens.shape != (B,) or (new_lens is not None and new_lens.shape != (B,)):
        raise ValueError(f"context_lens and new_lens must be (batch,) = ({B},), got "
                         f"{tuple(context_lens.shape)} and {None if new_lens is None else tuple(new_lens.shape)}")
    q_ptr = qo_ptr = Hq = 0
    qs = qo = (0, 0, 0, 1)
    q_out = None
    if q is not None:
        q_shape = q.shape
        if (len(q_shape) != 4 or q_shape[0] != B or q_shape[1] != S or q_shape[3] != D
                or q.dtype is not dtype or q.get_device() != dev):
            raise ValueError(f"q must be ({B}, {S}, heads, {D}) {dtype} beside k, got {tuple(q.shape)} {q.dtype}")
        Hq = q_shape[2]
        qs = q.stride()
        if qs[3] != 1:
            q = q.contiguous()
            qs = q.stride()
        q_out = _lib.rows_like(q)
        q_ptr, qo_ptr, qo = q.data_ptr(), q_out.data_ptr(), q_out.stride()
    elif q_weight is not None:
        raise ValueError("q_weight needs q")
    qw_ptr = kw_ptr = qw_code = kw_code = 0
    if q_weight is not None:
        q_weight = _weight("q_weight", q_weight, D, k)
        qw_ptr, qw_code = q_weight.data_ptr(), codes[q_weight.dtype]
    if k_weight is not None:
        k_weight = _weight("k_weight", k_weight, D, k)
        kw_ptr, kw_code = k_weight.data_ptr(), codes[k_weight.dtype]
    if (cos_cache is None) != (sin_cache is None):
        raise ValueError("cos_cache and sin_cache must be given together")
    n_pos = cos_ptr = sin_ptr = 0
    if cos_cache is not None:
        c_shape = cos_cache.shape
        if len(c_shape) != 2 or c_shape[1] * 2 != D or sin_cache.shape != c_shape:
            raise ValueError("cos/sin caches must both be (max_seq, head_dim // 2)")
        n_pos = c_shape[0]
        if n_pos < max_blocks * block_size:
            raise ValueError(f"cos/sin caches of {n_pos} positions do not cover the block tables' "
                             f"{max_blocks * block_size}")
        if not _lib.plain(cos_cache, dev, torch.float32):
            cos_cache = cos_cache.to(k.device, torch.float32).contiguous()
        if not _lib.plain(sin_cache, dev, torch.float32):
            sin_cache = sin_cache.to(k.device, torch.float32).contiguous()
        cos_ptr, sin_ptr = cos_cache.data_ptr(), sin_cache.data_ptr()
    bt, ctx = device_ints(block_tables, k), device_ints(context_lens, k)
    new_ptr = 0
    if new_lens is not None:
        new_lens = device_ints(new_lens, k)
        new_ptr = new_lens.data_ptr()
    ks, vs = k.stride(), v.stride()
    if ks[3] != 1:
        k = k.contiguous()
        ks = k.stride()
    if vs[3] != 1:
        v = v.contiguous()
        vs = v.stride()
    ps = k_pool.stride()
    ksc_ptr = vsc_ptr = 0
    sc = (0, 0)
    if quant:
        ksc_ptr, vsc_ptr, sc = k_scales.data_ptr(), v_scales.data_ptr(), k_scales.stride()
    with _lib.on_device(dev):
        rc = _lib.lib().mlxp_paged_append(_ARGS.pack(
            k.data_ptr(), v.data_ptr(), q_ptr, qo_ptr, k_pool.data_ptr(), v_pool.data_ptr(),
            ksc_ptr, vsc_ptr, bt.data_ptr(), ctx.data_ptr(), new_ptr, qw_ptr, kw_ptr, cos_ptr,
            sin_ptr, code, cache_code, qw_code, kw_code,
            B, S, Hq, Hk, D, num_blocks, block_size, max_blocks, bt.stride(0), n_pos,
            ks[0], ks[2], ks[1], vs[0], vs[2], vs[1], qs[0], qs[2], qs[1], qo[0], qo[2], qo[1],
            ps[0], ps[1], ps[2], sc[0], sc[1], eps, _lib.raw_stream(dev)))
    if rc:
        _lib.check(rc, "mlxp_paged_append")
    torch.autograd.graph.increment_version((k_pool, v_pool, k_scales, v_scales) if quant else (k_pool, v_pool))
    return q_out


def _weight(name, w, D, k):
    if w.shape != (D,) or w.dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"{name} must be ({D},) of a supported dtype, got {tuple(w.shape)} {w.dtype}")
    return w if _lib.plain(w, k.get_device(), w.dtype) else w.to(k.device).contiguous()
