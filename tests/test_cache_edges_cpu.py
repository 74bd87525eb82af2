"""CPU checks of the cache operators beside tests/test_cache_ops_cpu.py: conversions and refusals
that are made before any device work."""

import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.int16, torch.uint32, torch.uint8])
def test_integers_are_cut_to_their_nearest(dtype):
    from mlx_primitives import _lib
    top, low = (1 << 31) - 1, -(1 << 31)
    values = {torch.int32: [low, -1, 5, top], torch.int64: [1 << 32, (1 << 32) + 5, -(1 << 32) + 1, -1, 7, 1 << 62],
              torch.int16: [-3, 300], torch.uint32: [1, (1 << 32) - 1, 1 << 31], torch.uint8: [0, 255]}[dtype]
    t = torch.tensor(values, dtype=torch.int64).to(dtype)
    was = t.clone()
    got = _lib.int32(t, torch.device("cpu"))
    assert got.dtype is torch.int32 and got.tolist() == [min(max(v, low), top) for v in values]
    assert torch.equal(t, was)


def test_tables_and_lengths_as_the_kernels_read_them():
    from mlx_primitives.cache.paged_append import device_ints
    like = torch.zeros(1)
    one = torch.arange(5, dtype=torch.int32)[None]
    for t in (one, one.repeat(3, 1), torch.arange(24, dtype=torch.int32).view(3, 8)[:, :5], one.expand(1, 5)):
        assert device_ints(t, like) is t
    for t in (one.expand(3, 5), torch.arange(10, dtype=torch.int32).as_strided((3, 5), (2, 1)),
              torch.arange(15, dtype=torch.int32).view(5, 3).T, one[0, :1].expand(4)):
        got = device_ints(t, like)
        assert got.is_contiguous() and torch.equal(got, t)
    with pytest.raises(ValueError, match="integers"):
        device_ints(one.float(), like)


def test_sizes_that_32_bit_indexes_do_not_hold_are_refused():
    """Up to a thousand below 2^31: the kernels count a few tiles past the last key or row."""
    from mlx_primitives import _lib
    from mlx_primitives.cache.paged_append import _ARGS as APPEND
    from mlx_primitives.cache.quantized_attention import _ARGS as ATTN
    L, top = _lib.lib(), (1 << 31) - 1

    def append(block, mb, v_pool=32):
        return L.mlxp_paged_append(APPEND.pack(
            16, 16, 0, 0, 16, v_pool, 0, 0, 16, 16, 0, 0, 0, 0, 0, 1, 1, 0, 0, 1, 1, 0, 1, 64, 8, block, mb, mb, 0,
            *[64] * 12, *[64] * 3, 1, 1, 1e-6, 0))

    def attn(block, mb, B=1, Sq=1, H=4, scale=0.1):
        return L.mlxp_quant_paged_attn(ATTN.pack(
            16, 16, 16, 16, 16, 16, 16, 16, 0, 0, 1, 3, B, Sq, H, 2, 64, 8, block, mb, mb, 1, -1, 64, 64, 64, 64, 64,
            64, 64, 64, 64, 2, 1, scale, 0, 0, 0))

    for call in (lambda: append(top, 1), lambda: append(1, top - 1022), lambda: append(16, (top >> 4) - 62),
                 lambda: attn(top, 1), lambda: attn(1, top - 1022), lambda: attn(16, (top >> 4) - 62),
                 lambda: attn(16, 4, B=1 << 19, Sq=1 << 10), lambda: attn(16, 4, Sq=(top >> 2) - 254)):
        assert call() == _lib.MLXP_ERR_INVALID
        assert b"too large" in L.mlxp_last_error()
    # the largest that are taken: refused for another reason, which is looked at behind the sizes
    assert append(1, top - 1023, v_pool=16) == _lib.MLXP_ERR_INVALID
    assert b"different" in L.mlxp_last_error()
    assert attn(1, top - 1023, Sq=(top >> 2) - 255, scale=0.0) == _lib.MLXP_ERR_INVALID
    assert b"scale" in L.mlxp_last_error()


def _pool_args(dtype=torch.float32):
    z = lambda *shape: torch.zeros(shape)
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    return z(1, 1, 2, 64), z(3, 16, 2, 64).to(dtype), i(1, 2), i(1), z(3, 2)


def test_calls_without_derivatives_refuse_tensors_that_want_one():
    from mlx_primitives.cache import paged_append, quantized_paged_attention
    k, pool, bt, ctx, sc = _pool_args()
    p8 = pool.to(torch.int8)
    wants = lambda t: t.clone().requires_grad_(True)
    for f in (lambda: paged_append(wants(k), k, pool, pool, bt, ctx), lambda: paged_append(k, wants(k), pool, pool, bt, ctx),
              lambda: paged_append(k, k, wants(pool), pool, bt, ctx), lambda: paged_append(k, k, pool, wants(pool), bt, ctx),
              lambda: paged_append(k, k, pool, pool, bt, ctx, q=wants(k)),
              lambda: paged_append(k, k, pool, pool, bt, ctx, k_weight=wants(torch.ones(64))),
              lambda: paged_append(k, k, p8, p8, bt, ctx, k_scales=wants(sc), v_scales=sc),
              lambda: quantized_paged_attention(k, p8, p8, wants(sc), sc, bt, ctx),
              lambda: quantized_paged_attention(k, p8, p8, sc, wants(sc), bt, ctx),
              lambda: quantized_paged_attention(k, p8, p8, sc, sc, bt, ctx, alibi_slopes=wants(torch.ones(2)))):
        with pytest.raises(NotImplementedError, match="differentiable"):
            f()
        with torch.no_grad():
            try:
                f()
            except (ValueError, RuntimeError) as e:  # not that they want gradients
                assert "CUDA" in str(e)


def test_tangents_are_refused_before_any_device_work():
    import torch.autograd.forward_ad as fwd

    from mlx_primitives.cache import paged_append, quantized_paged_attention
    from mlx_primitives.kernels import qk_norm_rope
    k, pool, bt, ctx, sc = _pool_args()
    p8, w, cs = pool.to(torch.int8), torch.ones(64), torch.zeros(32, 32)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        for f in (lambda: qk_norm_rope(dual(k), k, w, w), lambda: qk_norm_rope(k, k, w, dual(w), cs, cs),
                  lambda: qk_norm_rope(k, k, None, None, cs, dual(cs)),
                  lambda: paged_append(k, dual(k), pool, pool, bt, ctx),
                  lambda: paged_append(k, k, dual(pool), pool, bt, ctx),
                  lambda: paged_append(k, k, pool, pool, bt, ctx, q=dual(k)),
                  lambda: quantized_paged_attention(dual(k), p8, p8, sc, sc, bt, ctx),
                  lambda: quantized_paged_attention(k, p8, p8, sc, dual(sc), bt, ctx)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()
