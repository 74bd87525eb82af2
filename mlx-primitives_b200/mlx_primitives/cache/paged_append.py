"""Appending keys and values to the paged pools, with norms and the position rotation on the way.

The write side of the pools that ``paged_attention`` and ``quantized_paged_attention`` read.  The
reference keeps that in its cache managers (mlx_primitives/cache/paged_attention.py:44-105
takes pools that something else has filled); here it is one launch (mlxp_paged_append): the new
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
    span = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride < span:
            return True
        span = stride * (size - 1) + span
    return False


def check_pools(k_pool, v_pool, k_scales, v_scales):
    """Checks that both cache operators make of the pools; returns the cache's dtype code."""
    if k_pool.ndim != 4 or k_pool.shape != v_pool.shape:
        raise ValueError("k_pool and v_pool must both be (num_blocks, block_size, heads, head_dim)"
                         f", got {tuple(k_pool.shape)} and {tuple(v_pool.shape)}")
    if k_pool.dtype != v_pool.dtype:
        raise ValueError(f"k_pool and v_pool must share a dtype, got {k_pool.dtype} and {v_pool.dtype}")
    if k_pool.stride() != v_pool.stride() or k_pool.stride(3) != 1:
        raise ValueError("k_pool and v_pool must have the same strides, and unit head_dim stride, "
                         f"got {k_pool.stride()} and {v_pool.stride()}")
    code = _lib.CACHE_DTYPE_CODES.get(k_pool.dtype)
    if code is None:
        if k_scales is not None or v_scales is not None:
            raise ValueError(f"scales go with float8_e4m3fn or int8 pools, got {k_pool.dtype}")
        return _lib.DTYPE_CODES.get(k_pool.dtype)
    want = (k_pool.shape[0], k_pool.shape[2])
    for name, s in (("k_scales", k_scales), ("v_scales", v_scales)):
        if s is None or s.dtype != torch.float32 or tuple(s.shape) != want or s.device != k_pool.device:
            raise ValueError(f"{name} must be a float32 tensor (num_blocks, heads) = {want} beside "
                             f"the pools, got {None if s is None else (s.dtype, tuple(s.shape), s.device)}")
    if k_scales.stride() != v_scales.stride():
        raise ValueError("k_scales and v_scales must have the same strides")
    return code


def device_ints(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """Tables and lengths as the kernels read them: int32 on the device, unit inner stride."""
    if t.dtype != torch.int32 or t.device != dev:
        if t.is_floating_point():
            raise ValueError(f"block tables and lengths must be integers, got {t.dtype}")
        t = t.to(dev, torch.int32)
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


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
    Padding rows of q come back as zeros.

    Pools: (num_blocks, block_size, kv_heads, head_dim) of k's dtype, or float8_e4m3fn or int8
    with ``k_scales``, ``v_scales`` (num_blocks, kv_heads) float32: value = code * scale.  A
    block's scale is the least power of two that holds its tokens; it is set when the block
    receives its first row and grows, its earlier codes being rescaled, when a later token needs
    it to.  A block that receives tokens must belong to one sequence (full blocks may be shared):
    the order of two writers of a block is not defined.  Not differentiable.
    """
    if k.ndim != 4 or k.shape != v.shape:
        raise ValueError("k and v must both be (batch, seq, kv_heads, head_dim), got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    B, S, Hk, D = k.shape
    dtype = k.dtype
    code = _lib.DTYPE_CODES.get(dtype)
    if code is None or v.dtype != dtype:
        raise ValueError(f"k and v must share a dtype of float32, bfloat16, float16, got {dtype}, {v.dtype}")
    cache_code = check_pools(k_pool, v_pool, k_scales, v_scales)
    quant = k_pool.dtype in _lib.CACHE_DTYPE_CODES
    if not quant and k_pool.dtype != dtype:
        raise ValueError(f"the pools' dtype ({k_pool.dtype}) must be k's ({dtype}) or an 8-bit one")
    num_blocks, block_size, Hp, Dp = k_pool.shape
    if Hp != Hk or Dp != D:
        raise ValueError(f"pools of (heads, head_dim) = {(Hp, Dp)} cannot take k of {(Hk, D)}")
    if D % 2 or D < 2:
        raise ValueError(f"head_dim must be even, got {D}")
    dev = k.device
    if dev.type != "cuda" or k_pool.device != dev or v_pool.device != dev or v.device != dev:
        raise ValueError("k, v and the pools must be on one CUDA device (appending is in place)")
    if _overlaps(k_pool) or (quant and _overlaps(k_scales)):
        raise ValueError("the pools and scales must not overlap themselves (expanded views)")
    if block_tables.ndim != 2 or block_tables.shape[0] != B:
        raise ValueError(f"block_tables must be (batch, max_blocks), got {tuple(block_tables.shape)}")
    for name, t in (("context_lens", context_lens), ("new_lens", new_lens)):
        if t is not None and tuple(t.shape) != (B,):
            raise ValueError(f"{name} must be (batch,) = ({B},), got {tuple(t.shape)}")
    Hq, q_strides = 0, (0, 0, 0)
    if q is not None:
        if q.ndim != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != D or q.dtype != dtype or q.device != dev:
            raise ValueError(f"q must be ({B}, {S}, heads, {D}) {dtype} beside k, got {tuple(q.shape)} {q.dtype}")
        Hq = q.shape[2]
    elif q_weight is not None:
        raise ValueError("q_weight needs q")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (tuple(w.shape) != (D,) or w.dtype not in _lib.DTYPE_CODES):
            raise ValueError(f"{name} must be ({D},) of a supported dtype, got {tuple(w.shape)} {w.dtype}")
    if (cos_cache is None) != (sin_cache is None):
        raise ValueError("cos_cache and sin_cache must be given together")
    max_blocks = block_tables.shape[1]
    n_pos = 0
    if cos_cache is not None:
        if cos_cache.shape != sin_cache.shape or cos_cache.ndim != 2 or cos_cache.shape[1] != D // 2:
            raise ValueError("cos/sin caches must both be (max_seq, head_dim // 2)")
        n_pos = cos_cache.shape[0]
        if n_pos < max_blocks * block_size:
            raise ValueError(f"cos/sin caches of {n_pos} positions do not cover the block tables' "
                             f"{max_blocks * block_size}")
        cos_cache, sin_cache = (c if c.dtype == torch.float32 and c.device == dev and c.is_contiguous()
                                else c.to(dev, torch.float32).contiguous() for c in (cos_cache, sin_cache))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in
                                       (k, v, q, q_weight, k_weight)):
        raise NotImplementedError("paged_append is not differentiable: call it under torch.no_grad()")
    bt, ctx = device_ints(block_tables, dev), device_ints(context_lens, dev)
    new = None if new_lens is None else device_ints(new_lens, dev)
    k, v = (t if t.stride(3) == 1 else t.contiguous() for t in (k, v))
    q_weight, k_weight = (w if w is None or (w.device == dev and w.is_contiguous())
                          else w.to(dev).contiguous() for w in (q_weight, k_weight))
    q_out, qo_strides = None, (0, 0, 0)
    if q is not None:
        q = q if q.stride(3) == 1 else q.contiguous()
        q_out = torch.empty_like(q)
        q_strides, qo_strides = _lib.seq_strides(q), _lib.seq_strides(q_out)
    a = _lib.address
    codes = _lib.DTYPE_CODES
    with _lib.on_device(dev):
        rc = _lib.lib().mlxp_paged_append(_ARGS.pack(
            k.data_ptr(), v.data_ptr(), a(q), a(q_out), k_pool.data_ptr(), v_pool.data_ptr(),
            a(k_scales), a(v_scales), bt.data_ptr(), ctx.data_ptr(), a(new), a(q_weight),
            a(k_weight), a(cos_cache), a(sin_cache), code, cache_code,
            0 if q_weight is None else codes[q_weight.dtype],
            0 if k_weight is None else codes[k_weight.dtype],
            B, S, Hq, Hk, D, num_blocks, block_size, max_blocks, bt.stride(0), n_pos,
            *_lib.seq_strides(k), *_lib.seq_strides(v), *q_strides, *qo_strides,
            *k_pool.stride()[:3], *(k_scales.stride() if quant else (0, 0)),
            eps, _lib.raw_stream(dev)))
    _lib.check(rc, "mlxp_paged_append")
    return q_out
