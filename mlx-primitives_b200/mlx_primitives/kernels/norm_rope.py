"""Query/key norms with the position rotation, on B200.

``qk_norm_rope`` takes the projected queries and keys of a layer to what attention reads, in one
launch: each head's row is divided by its root mean square and multiplied by a weight, then
rotated as ``rope_qk`` does (mlx_primitives/kernels/rope.py:499-533; the norm has no counterpart
in the reference).  For x of shape (batch, seq, heads, head_dim), h = head_dim / 2, p the token's
position and r = (mean(x^2) + eps)^(-1/2):
    y = x * r * weight
    out[..., :h] = y[..., :h] * cos[p] - y[..., h:] * sin[p]
    out[..., h:] = y[..., :h] * sin[p] + y[..., h:] * cos[p].
Computed in fp32 and rounded once.  Differentiable in q, k and the weights, in reverse mode and
once (mlxp_qk_norm_rope_bwd); the weights' gradients are summed in fp32 in a fixed order, so every
run gives the same bits.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib

__all__ = ["qk_norm_rope"]

# mlxp_qk_norm_rope_args: 13 pointers, 12 sizes, 20 strides, eps, workspace, bytes, stream
_ARGS = _lib.ArgStruct(50, doubles=(46,))
_CODES = _lib.DTYPE_CODES


def _refuse(q, k, q_weight, k_weight, cos, sin, positions):
    """Raises for what qk_norm_rope's quick checks have found wrong."""
    for name, x in (("Q", q), ("K", k)):
        if x.ndim != 4:
            raise ValueError(f"{name} must be 4D (batch, seq_len, num_heads, head_dim), got {x.ndim}D")
    if q.dtype not in _CODES:
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
            if tuple(w.shape) != (D,) or w.dtype not in _CODES:
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
    raise ValueError("invalid arguments")


def _quick_ok(q, k, q_weight, k_weight, cos, sin, positions) -> bool:
    if q.ndim != 4 or k.ndim != 4:
        return False
    (B, Sq, _, D), (Bk, Sk, _, Dk), dtype = q.shape, k.shape, q.dtype
    if B != Bk or D != Dk or k.dtype is not dtype or dtype not in _CODES or D % 2 or D < 2:
        return False
    if q_weight is None or k_weight is None:
        if q_weight is not None or k_weight is not None:
            return False
    elif (q_weight.shape != (D,) or k_weight.shape != (D,) or q_weight.dtype not in _CODES
          or k_weight.dtype not in _CODES):
        return False
    if cos is None or sin is None:
        if cos is not None or sin is not None:
            return False
    else:
        shape = cos.shape
        if len(shape) != 2 or shape[1] * 2 != D or sin.shape != shape:
            return False
    return positions is None or (Sq == Sk and positions.shape == (B, Sq)
                                 and not positions.is_floating_point())


def _pack(dev, q, k, q_out, k_out, gq, gk, q_weight, k_weight, dqw, dkw, cos, sin, positions,
          offset, k_offset, eps, ws, ws_bytes) -> bytes:
    B, Sq, Hq, D = q.shape
    _, Sk, Hk, _ = k.shape
    qs, ks = q.stride(), k.stride()
    # of a tensor that is not there, the strides are not read
    qo = qs if q_out is None else q_out.stride()
    ko = ks if k_out is None else k_out.stride()
    gqs = qs if gq is None else gq.stride()
    gks = ks if gk is None else gk.stride()
    ps0, ps1 = (0, 0) if positions is None else positions.stride()
    qw = kw = wd = kwd = c = s = n_pos = 0
    if q_weight is not None:
        qw, kw, wd, kwd = q_weight.data_ptr(), k_weight.data_ptr(), _CODES[q_weight.dtype], _CODES[k_weight.dtype]
    if cos is not None:
        c, s, n_pos = cos.data_ptr(), sin.data_ptr(), cos.shape[0]
    return _ARGS.pack(
        q.data_ptr(), k.data_ptr(), 0 if q_out is None else q_out.data_ptr(),
        0 if k_out is None else k_out.data_ptr(), 0 if gq is None else gq.data_ptr(),
        0 if gk is None else gk.data_ptr(), qw, kw, 0 if dqw is None else dqw.data_ptr(),
        0 if dkw is None else dkw.data_ptr(), c, s, 0 if positions is None else positions.data_ptr(),
        _CODES[q.dtype], wd, kwd, B, Sq, Sk, Hq, Hk, D, n_pos, offset, k_offset, ps0, ps1,
        qs[0], qs[2], qs[1], ks[0], ks[2], ks[1], qo[0], qo[2], qo[1], ko[0], ko[2], ko[1],
        gqs[0], gqs[2], gqs[1], gks[0], gks[2], gks[1],
        eps, 0 if ws is None else ws.data_ptr(), ws_bytes, _lib.raw_stream(dev))


def _dense(t):
    return t if t is None or t.stride(-1) == 1 else t.contiguous()


def _forward(dev, q, k, q_weight, k_weight, cos, sin, positions, offset, k_offset, eps):
    q_out, k_out = _lib.rows_like(q), _lib.rows_like(k)
    with _lib.on_device(dev):
        rc = _lib.lib().mlxp_qk_norm_rope(_pack(
            dev, q, k, q_out, k_out, None, None, q_weight, k_weight, None, None, cos, sin,
            positions, offset, k_offset, eps, None, 0))
    if rc:
        _lib.check(rc, "mlxp_qk_norm_rope")
    return q_out, k_out


def _as_saved(dev, q, k, q_weight, k_weight, cos, sin, positions, gq, gk) -> bool:
    """Whether the saved tensors are as the forward took them (but for q's and k's strides): hooks on
    saved tensors may give back others, also on the host."""
    return (_quick_ok(q, k, q_weight, k_weight, cos, sin, positions)
            and q.get_device() == dev and k.get_device() == dev
            and all(w is None or _lib.plain(w, dev, w.dtype) for w in (q_weight, k_weight))
            and all(t is None or _lib.plain(t, dev, torch.float32) for t in (cos, sin))
            and (positions is None or (positions.dtype is torch.int32 and positions.get_device() == dev))
            and all(g is None or (g.shape == x.shape and g.dtype is x.dtype) for g, x in ((gq, q), (gk, k))))


class _QKNormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, dev, q, k, q_weight, k_weight, cos, sin, positions, offset, k_offset, eps):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.args = (dev, offset, k_offset, eps)
        return _forward(dev, q, k, q_weight, k_weight, cos, sin, positions, offset, k_offset, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        dev, offset, k_offset, eps = ctx.args
        if not _as_saved(dev, q, k, q_weight, k_weight, cos, sin, positions, gq, gk):
            raise RuntimeError("qk_norm_rope: saved tensors came back changed")
        q, k, gq, gk = _dense(q), _dense(k), _dense(gq), _dense(gk)
        dq = None if gq is None else _lib.rows_like(q)
        dk = None if gk is None else _lib.rows_like(k)
        dqw = torch.empty_like(q_weight) if ctx.needs_input_grad[3] else None
        dkw = torch.empty_like(k_weight) if ctx.needs_input_grad[4] else None
        L = _lib.lib()
        ws, ws_bytes = None, 0
        if dqw is not None or dkw is not None:
            ws_bytes = L.mlxp_qk_norm_rope_bwd_workspace_size(q.shape[-1])
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
        with _lib.on_device(dev):
            _lib.check(L.mlxp_qk_norm_rope_bwd(_pack(
                dev, q, k, dq, dk, gq, gk, q_weight, k_weight, dqw, dkw, cos, sin, positions,
                offset, k_offset, eps, ws, ws_bytes)), "mlxp_qk_norm_rope_bwd")
        return None, dq, dk, dqw, dkw, None, None, None, None, None, None


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
    cannot be refused).  head_dim is even and at most 256.  As for every operator, a training step
    is captured into a CUDA graph while no eager autograd graph of the same leaves is alive: their
    accumulation belongs to the stream of the graph that made it.
    """
    out = _lib.calls().norm_rope(q, k, q_weight, k_weight, cos_cache, sin_cache, positions, offset,
                                 offset if k_offset is None else k_offset, eps)
    if out is not None:  # else: not a call that can be made as it is
        if type(out) is int:
            _lib.check(out, "mlxp_qk_norm_rope")
        return out
    if not _quick_ok(q, k, q_weight, k_weight, cos_cache, sin_cache, positions):
        _refuse(q, k, q_weight, k_weight, cos_cache, sin_cache, positions)
    _lib.refuse_tangents("qk_norm_rope", q, k, q_weight, k_weight, cos_cache, sin_cache)
    needs = torch.is_grad_enabled() and (
        q.requires_grad or k.requires_grad
        or (q_weight is not None and (q_weight.requires_grad or k_weight.requires_grad)))
    dev = q.get_device()
    host = dev < 0
    if host:
        if not torch.cuda.is_available():
            raise RuntimeError("qk_norm_rope requires a CUDA device (there is no CPU fallback)")
        if needs:
            raise NotImplementedError("qk_norm_rope gradients need CUDA tensors")
        dev = torch.cuda.current_device()
        q, k = q.to(dev), k.to(dev)
    elif k.get_device() != dev:
        raise ValueError("q and k must be on the same device")
    q, k = _dense(q), _dense(k)
    if q_weight is not None:
        if not _lib.plain(q_weight, dev, q_weight.dtype):
            q_weight = q_weight.to(q.device).contiguous()
        if not _lib.plain(k_weight, dev, k_weight.dtype):
            k_weight = k_weight.to(q.device).contiguous()
    if cos_cache is not None:
        if not _lib.plain(cos_cache, dev, torch.float32):
            cos_cache = cos_cache.detach().to(q.device, torch.float32).contiguous()
        if not _lib.plain(sin_cache, dev, torch.float32):
            sin_cache = sin_cache.detach().to(q.device, torch.float32).contiguous()
    if positions is not None and (positions.dtype is not torch.int32 or positions.get_device() != dev):
        positions = _lib.int32(positions, q.device)
    offset = int(offset)
    k_offset = offset if k_offset is None else int(k_offset)
    run = _QKNormRopeFn.apply if needs else _forward
    out = run(dev, q, k, q_weight, k_weight, cos_cache, sin_cache, positions, offset, k_offset, float(eps))
    return (out[0].cpu(), out[1].cpu()) if host else out
