"""Paged attention over a cache held in 8 bits, on B200.

``quantized_paged_attention`` is ``paged_attention`` (mlx_primitives/cache/paged_attention.py:44-105)
for pools of float8_e4m3fn or int8 codes with one float32 scale for each block and head, as
``paged_append`` writes them: value = code * scale.  The codes are read in place, once
(mlxp_quant_paged_attn); nothing is expanded in memory.

The queries of a sequence are its last positions (query i of n sits at context_lens[b] - n + i):
one row is a decode step, a few rows are speculated tokens, many a chunk of a prompt whose keys
have been appended before.  (``paged_attention`` counts query positions from 0 for more than one
row, as the reference does.)
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from .paged_append import check_pools, device_ints, refuse_gradients

__all__ = ["quantized_paged_attention"]

# mlxp_quant_paged_attn_args: 10 pointers, 13 sizes, 11 strides, scale, workspace, bytes, stream
_ARGS = _lib.ArgStruct(39, doubles=(35,))
_HEAD_DIMS = (32, 64, 128)


def _rows16(t: torch.Tensor) -> bool:
    es = t.element_size()
    s = t.stride()
    return s[3] == 1 and not (t.data_ptr() | s[0] * es | s[1] * es | s[2] * es) & 15


def quantized_paged_attention(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    scale: Optional[float] = None,
    causal: bool = True,
    window_size: Optional[int] = None,
    query_lens: Optional[torch.Tensor] = None,
    alibi_slopes: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of q (batch, seq_q, heads, head_dim) over 8-bit K/V in a block pool.

    k_pool, v_pool: (num_blocks, block_size, kv_heads, head_dim) float8_e4m3fn or int8, heads a
    multiple of kv_heads, 16-byte aligned with strides that are multiples of 16; k_scales,
    v_scales: (num_blocks, kv_heads) float32, finite, k's of magnitude 2^-100 to 2^100, v's to 2^100
    and within a factor of 2^80 of one another in a sequence and head (below 2^-60, as blocks of
    zeros have it, they count as 2^-60 there and the values may count as 0).  block_tables:
    (batch, max_blocks), ids outside [0, num_blocks) are missing blocks.  context_lens: (batch,)
    cached tokens, the queries' own among them.  ``query_lens`` (batch,): queries of each sequence
    (default seq_q); rows behind them come back as zeros, as do rows that see no key.
    ``window_size`` W keeps keys at most W positions away, as ``sliding_window_attention`` does.
    ALiBi adds slope[h] * (key position - query position).  Returns q's shape and dtype.  Rows and
    blocks behind the contexts or before every query's window may hold anything; a NaN or infinity
    that some query sees may reach all its sequence's rows, also those that do not see it.  Not
    differentiable, in either mode.
    """
    if alibi_slopes is None and (window_size is None or window_size >= 0):
        out = _lib.calls().attend(q, k_pool, v_pool, k_scales, v_scales, block_tables, context_lens,
                                  query_lens, scale, causal,
                                  -1 if window_size is None else window_size)
        if out is not None:  # else: not a call that can be made as it is
            if type(out) is int:
                _lib.check(out, "mlxp_quant_paged_attn")
            return out
    shape = q.shape
    if len(shape) != 4:
        raise ValueError(f"q must be (batch, seq_q, num_heads, head_dim), got {tuple(q.shape)}")
    cache_code = check_pools(k_pool, v_pool, k_scales, v_scales)
    if k_scales is None:
        raise ValueError(f"the pools must be float8_e4m3fn or int8, got {k_pool.dtype}; "
                         "paged_attention reads other types")
    B, Sq, H, D = shape
    num_blocks, block_size, Hk, Dk = k_pool.shape
    if Dk != D:
        raise ValueError(f"pool head_dim ({Dk}) must equal q's head_dim ({D})")
    if D not in _HEAD_DIMS:
        raise ValueError(f"paged attention supports head_dim {_HEAD_DIMS}, got {D}")
    if Hk < 1 or H % Hk or H < 1:
        raise ValueError(f"num_heads ({H}) must be a multiple of the pool's heads ({Hk})")
    code = _lib.DTYPE_CODES.get(q.dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {q.dtype}; expected float32, bfloat16 or float16")
    bt_shape = block_tables.shape
    if len(bt_shape) != 2 or bt_shape[0] != B:
        raise ValueError(f"block_tables must be (batch, max_blocks), got {tuple(block_tables.shape)}")
    if context_lens.shape != (B,):
        raise ValueError(f"context_lens must be (batch,) = ({B},), got {tuple(context_lens.shape)}")
    if query_lens is not None and query_lens.shape != (B,):
        raise ValueError(f"query_lens must be (batch,) = ({B},), got {tuple(query_lens.shape)}")
    if alibi_slopes is not None and alibi_slopes.shape != (H,):
        raise ValueError(f"alibi_slopes must be (num_heads,) = ({H},), got {tuple(alibi_slopes.shape)}")
    if window_size is not None and window_size < 0:
        raise ValueError(f"window_size must be >= 0, got {window_size}")
    _lib.refuse_tangents("quantized_paged_attention", q, k_pool, v_pool, k_scales, v_scales, alibi_slopes)
    refuse_gradients("quantized_paged_attention", q, k_pool, v_pool, k_scales, v_scales, alibi_slopes)
    dev = q.get_device()
    host = dev < 0
    if host:
        if not torch.cuda.is_available():
            raise RuntimeError("attention requires a CUDA device (there is no CPU fallback)")
        dev = torch.cuda.current_device()
        q, k_pool, v_pool, k_scales, v_scales = (
            t.to(dev) for t in (q, k_pool, v_pool, k_scales, v_scales))
    elif k_pool.get_device() != dev or v_pool.get_device() != dev:
        raise ValueError("q, k_pool and v_pool must be on the same device")
    if not _rows16(q):
        q = q.clone(memory_format=torch.contiguous_format)
    bt, ctx = device_ints(block_tables, q), device_ints(context_lens, q)
    lens_ptr = slopes_ptr = 0
    if query_lens is not None:
        query_lens = device_ints(query_lens, q)
        lens_ptr = query_lens.data_ptr()
    if alibi_slopes is not None:
        alibi_slopes = alibi_slopes.to(q.device, torch.float32).contiguous()
        slopes_ptr = alibi_slopes.data_ptr()
    out = torch.empty_like(q)
    qs, os, ps, sc = q.stride(), out.stride(), k_pool.stride(), k_scales.stride()
    L = _lib.lib()
    with _lib.on_device(dev):
        stream = _lib.raw_stream(dev)
        fields = (q.data_ptr(), out.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
                  k_scales.data_ptr(), v_scales.data_ptr(), bt.data_ptr(), ctx.data_ptr(), lens_ptr,
                  slopes_ptr, code, cache_code, B, Sq, H, Hk, D, num_blocks, block_size,
                  bt_shape[1], bt.stride(0), 1 if causal else 0,
                  -1 if window_size is None else int(window_size),
                  qs[0], qs[2], qs[1], os[0], os[2], os[1], ps[0], ps[1], ps[2], sc[0], sc[1],
                  D ** -0.5 if scale is None else scale)
        ws_bytes = L.mlxp_quant_paged_attn_workspace_size(_ARGS.pack(*fields, 0, 0, stream))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
        rc = L.mlxp_quant_paged_attn(_ARGS.pack(*fields, ws.data_ptr(), ws_bytes, stream))
    if rc:
        _lib.check(rc, "mlxp_quant_paged_attn")
    return out.cpu() if host else out
