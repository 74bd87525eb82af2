"""Query/key norms with the position rotation, on B200.

``qk_norm_rope`` takes the projected queries and keys of a layer to what attention reads, in one
launch: each head's row is divided by its root mean square and multiplied by a weight, then
rotated as ``rope_qk`` does (mlx_primitives/kernels/rope.py:499-533; the norm has no counterpart
in the reference).  For x of shape (batch, seq, heads, head_dim), h = head_dim / 2, p the token's
position and r = (mean(x^2) + eps)^(-1/2):
    y = x * r * weight
    out[..., :h] = y[..., :h] * cos[p] - y[..., h:] * sin[p]
    out[..., h:] = y[..., :h] * sin[p] + y[..., h:] * cos[p].
Computed in fp32 and rounded once.  Differentiable in q, k and the weights (mlxp_qk_norm_rope_bwd);
the weights' gradients are summed in fp32 in a fixed order, so every run gives the same bits.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib

__all__ = ["qk_norm_rope"]

# mlxp_qk_norm_rope_args: 13 pointers, 12 sizes, 20 strides, eps, workspace, bytes, stream
_ARGS = _lib.ArgStruct(50, doubles=(46,))
_NO_STRIDES = (0, 0, 0)


def _check(q, k, q_weight, k_weight, cos, sin, positions):
    for name, x in (("Q", q), ("K", k)):
        if x.ndim != 4:
            raise ValueError(f"{name} must be 4D (batch, seq_len, num_heads, head_dim), got {x.ndim}D")
    if q.dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"unsupported dtype {q.dtype}")
    if q.shape[0] != k.shape[0] or q.shape[-1] != k.shape[-1] or q.dtype != k.dtype:
        raise ValueError(f"Q and K must agree in batch, head_dim and dtype, got {tuple(q.shape)} "
                         f"{q.dtype} and {tuple(k.shape)} {k.dtype}")
    D = q.shape[-1]
    if D % 2 or D < 2:
        raise ValueError(f"head_dim must be even, got {D}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight must be given together")
    if q_weight is not None:
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            if tuple(w.shape) != (D,) or w.dtype not in _lib.DTYPE_CODES:
                raise ValueError(f"{name} must be ({D},) of a supported dtype, got {tuple(w.shape)} {w.dtype}")
    if (cos is None) != (sin is None):
        raise ValueError("cos_cache and sin_cache must be given together")
    if cos is not None and (cos.shape != sin.shape or cos.ndim != 2 or cos.shape[1] != D // 2):
        raise ValueError("cos/sin caches must both be (max_seq, head_dim // 2)")
    if positions is not None:
        if q.shape[1] != k.shape[1]:
            raise ValueError("positions need Q and K of one length")
        if tuple(positions.shape) != tuple(q.shape[:2]) or positions.is_floating_point():
            raise ValueError(f"positions must be integers of shape {tuple(q.shape[:2])}, got "
                             f"{positions.dtype} {tuple(positions.shape)}")


def _pack(dev, q, k, q_out, k_out, gq, gk, q_weight, k_weight, dqw, dkw, cos, sin, positions,
          offset, k_offset, eps, ws, ws_bytes) -> bytes:
    B, Sq, Hq, D = q.shape
    _, Sk, Hk, _ = k.shape
    a, strides = _lib.address, _lib.seq_strides
    codes = _lib.DTYPE_CODES
    return _ARGS.pack(
        q.data_ptr(), k.data_ptr(), a(q_out), a(k_out), a(gq), a(gk), a(q_weight), a(k_weight),
        a(dqw), a(dkw), a(cos), a(sin), a(positions), codes[q.dtype],
        0 if q_weight is None else codes[q_weight.dtype],
        0 if k_weight is None else codes[k_weight.dtype],
        B, Sq, Sk, Hq, Hk, D, 0 if cos is None else cos.shape[0], offset, k_offset,
        *((0, 0) if positions is None else positions.stride()),
        *strides(q), *strides(k), *(_NO_STRIDES if q_out is None else strides(q_out)),
        *(_NO_STRIDES if k_out is None else strides(k_out)),
        *(_NO_STRIDES if gq is None else strides(gq)), *(_NO_STRIDES if gk is None else strides(gk)),
        eps, a(ws), ws_bytes, _lib.raw_stream(dev))


def _dense(t):
    return t if t is None or t.stride(-1) == 1 else t.contiguous()


def _forward(q, k, q_weight, k_weight, cos, sin, positions, offset, k_offset, eps):
    dev = q.device
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    with _lib.on_device(dev):
        _lib.check(_lib.lib().mlxp_qk_norm_rope(_pack(
            dev, q, k, q_out, k_out, None, None, q_weight, k_weight, None, None, cos, sin,
            positions, offset, k_offset, eps, None, 0)), "mlxp_qk_norm_rope")
    return q_out, k_out


class _QKNormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, offset, k_offset, eps):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.args = (offset, k_offset, eps)
        return _forward(q, k, q_weight, k_weight, cos, sin, positions, offset, k_offset, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        offset, k_offset, eps = ctx.args
        dev = q.device
        gq, gk = _dense(gq), _dense(gk)
        dq = None if gq is None else torch.empty_like(q)
        dk = None if gk is None else torch.empty_like(k)
        dqw = torch.empty_like(q_weight) if ctx.needs_input_grad[2] else None
        dkw = torch.empty_like(k_weight) if ctx.needs_input_grad[3] else None
        L = _lib.lib()
        ws, ws_bytes = None, 0
        if dqw is not None or dkw is not None:
            ws_bytes = L.mlxp_qk_norm_rope_bwd_workspace_size(q.shape[-1])
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        with _lib.on_device(dev):
            _lib.check(L.mlxp_qk_norm_rope_bwd(_pack(
                dev, q, k, dq, dk, gq, gk, q_weight, k_weight, dqw, dkw, cos, sin, positions,
                offset, k_offset, eps, ws, ws_bytes)), "mlxp_qk_norm_rope_bwd")
        return dq, dk, dqw, dkw, None, None, None, None, None, None


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: Optional[torch.Tensor],
    k_weight: Optional[torch.Tensor],
    cos_cache: Optional[torch.Tensor] = None,
    sin_cache: Optional[torch.Tensor] = None,
    offset: int = 0,
    k_offset: Optional[int] = None,
    positions: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS-normed and rotated q (batch, seq, heads, head_dim) and k (its own length and heads).

    q_weight, k_weight: (head_dim,) of any float type, or both None (no norm).  cos_cache,
    sin_cache: (max_seq, head_dim // 2), or both None (no rotation).  Sequence index s sits at
    position ``offset`` + s (``k_offset`` + s for k, default ``offset``), or at ``positions``
    (batch, seq) where given: a negative position marks padding, whose row becomes zeros and has
    no gradient; one past the tables gives a row of NaN (it is read on the device, where it
    cannot be refused).  head_dim is even and at most 256.
    """
    _check(q, k, q_weight, k_weight, cos_cache, sin_cache, positions)
    host = q.device.type == "cpu"
    if host:
        if not torch.cuda.is_available():
            raise RuntimeError("qk_norm_rope requires a CUDA device (there is no CPU fallback)")
        dev = torch.device("cuda", torch.cuda.current_device())
    else:
        dev = q.device
    if not host and k.device != dev:
        raise ValueError("q and k must be on the same device")
    needs = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (q, k, q_weight, k_weight))
    if host:
        if needs:
            raise NotImplementedError("qk_norm_rope gradients need CUDA tensors")
        q, k = q.to(dev), k.to(dev)
    q, k = _dense(q), _dense(k)
    if q_weight is not None:
        q_weight, k_weight = (w if w.device == dev and w.is_contiguous() else w.to(dev).contiguous()
                              for w in (q_weight, k_weight))
    if cos_cache is not None:
        cos_cache, sin_cache = (c.detach().to(dev, torch.float32).contiguous()
                                for c in (cos_cache, sin_cache))
    if positions is not None and (positions.dtype != torch.int32 or positions.device != dev):
        positions = positions.to(dev, torch.int32)
    offset = int(offset)
    args = (q, k, q_weight, k_weight, cos_cache, sin_cache, positions, offset,
            offset if k_offset is None else int(k_offset), float(eps))
    out = _QKNormRopeFn.apply(*args) if needs else _forward(*args)
    return (out[0].cpu(), out[1].cpu()) if host else out
