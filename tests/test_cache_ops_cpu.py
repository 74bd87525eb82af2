"""CPU checks of the norm/rotation, append and 8-bit attention operators: their fp64 oracle
(gradient against differences, code rounding against torch's), the packed argument structs
against the library, and the refusals of the Python entry points and of the C ABI."""

import numpy as np
import pytest
import torch

from oracle import cache_oracle as C


# ---- the oracle ----
@pytest.mark.parametrize("rotate,norm", [(True, True), (False, True), (True, False)])
def test_oracle_gradient_matches_differences(rotate, norm):
    rs = np.random.RandomState(0)
    B, S, H, D, n = 2, 3, 2, 8, 5
    x, w, gy = rs.randn(B, S, H, D), 1 + 0.1 * rs.randn(D), rs.randn(B, S, H, D)
    ang = np.outer(np.arange(n), 10.0 ** -np.arange(D // 2))
    cos, sin = (np.cos(ang), np.sin(ang)) if rotate else (None, None)
    w = w if norm else None
    pos = np.array([[0, 4, 2], [3, -1, 1]])
    f = lambda x, w: (C.norm_rope(x, w, cos, sin, pos) * gy).sum()
    dx, dw, _ = C.norm_rope_grad(gy, x, w, cos, sin, pos)
    d = 1e-6
    for at in [(0, 0, 0, 0), (0, 1, 1, 5), (1, 1, 0, 3), (1, 2, 1, 7)]:
        e = np.zeros_like(x)
        e[at] = d
        # central differences: error O(d^2) of third derivatives, and 1e-16 / d of rounding
        assert abs((f(x + e, w) - f(x - e, w)) / (2 * d) - dx[at]) < 1e-7
    for j in range(D) if norm else ():
        e = np.zeros(D)
        e[j] = d
        assert abs((f(x, w + e) - f(x, w - e)) / (2 * d) - dw[j]) < 1e-7


def test_oracle_e4m3_rounding_is_torchs():
    x = np.concatenate([np.linspace(-448, 448, 20001), np.geomspace(1e-6, 448, 5000),
                        np.arange(-64, 64) / 1024.0])
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    got = C.round_e4m3(x)
    # torch rounds fp64 through fp32, which can move a value within 2^-25 of a tie
    assert np.mean(got != want) < 1e-3
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    every = every[np.isfinite(every)]
    assert np.array_equal(C.round_e4m3(every), every)


def test_oracle_append_grows_a_block_and_rescales():
    new = np.full((1, 1, 1, 4), 900.0)
    pool = np.zeros((2, 4, 1, 4))
    pool[1, :2] = 8.0
    got, scales, written = C.append(new, pool, np.array([[1]]), [2], [1], np.ones((2, 1)), "e4m3")
    assert scales[1, 0] == 4.0 and scales[0, 0] == 1.0  # 900 <= 448 * 4
    assert np.all(got[1, :2] == 2.0) and np.all(got[1, 2] == 224.0) and np.all(got[1, 3] == 0)
    assert written.sum() == 1 and written[1, 2]


# ---- the packed structs ----
@pytest.mark.parametrize("name,module,n", [
    ("mlxp_qk_norm_rope", "kernels.norm_rope", 13), ("mlxp_qk_norm_rope_bwd", "kernels.norm_rope", 13),
    ("mlxp_paged_append", "cache.paged_append", 15), ("mlxp_quant_paged_attn", "cache.quantized_attention", 10)])
def test_argument_structs_have_the_librarys_size(name, module, n):
    import importlib

    from mlx_primitives import _lib
    args = importlib.import_module("mlx_primitives." + module)._ARGS
    fields = args.size // 8 - 1
    fn = getattr(_lib.lib(), name)
    # the right size is read as far as the dtype, which is not one
    assert fn(args.pack(*[0] * n, 77, *[0] * (fields - n - 1))) == _lib.MLXP_ERR_INVALID
    assert b"dtype 77" in _lib.lib().mlxp_last_error()
    other = _lib.ArgStruct(fields + 2)
    assert fn(other.pack(*[0] * (fields + 1))) == _lib.MLXP_ERR_INVALID
    assert b"another size" in _lib.lib().mlxp_last_error()
    assert fn(None) == _lib.MLXP_ERR_INVALID


def test_c_abi_refuses_before_any_launch():
    from mlx_primitives import _lib
    from mlx_primitives.cache.paged_append import _ARGS as APPEND
    from mlx_primitives.cache.quantized_attention import _ARGS as ATTN
    from mlx_primitives.kernels.norm_rope import _ARGS as NORM
    L = _lib.lib()

    def norm(D=8, S=4, n_pos=8, off=0, eps=1e-6, cos=16, sin=16, dtype=1, w=16):
        return L.mlxp_qk_norm_rope(NORM.pack(
            16, 16, 16, 16, 0, 0, w, w, 0, 0, cos, sin, 0, dtype, 0, 0, 1, S, S, 1, 1, D, n_pos,
            off, off, 0, 0, *[0] * 18, eps, 0, 0, 0))

    for kw, why in [(dict(D=7), b"even"), (dict(D=512), b"256"), (dict(S=9), b"exceed"),
                    (dict(off=-1), b"exceed"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"),
                    (dict(sin=0), b"together"), (dict(n_pos=0, S=0), b"empty")]:
        assert norm(**kw) in (_lib.MLXP_ERR_INVALID, _lib.MLXP_ERR_UNSUPPORTED)
        assert why in L.mlxp_last_error(), (kw, L.mlxp_last_error())

    def append(cache=1, B=1, block=16, mb=4, n_pos=64, scales=16, bts=4, k=16, v_pool=32, v_scales=32):
        return L.mlxp_paged_append(APPEND.pack(
            k, 16, 0, 0, 16, v_pool, scales, v_scales, 16, 16, 0, 0, 0, 16, 16, 1, cache, 0, 0, B, 1, 0,
            1, 64, 8, block, mb, bts, n_pos, *[64] * 12, *[64] * 3, 1, 1, 1e-6, 0))

    for kw, why in [(dict(cache=2), b"dtype"), (dict(cache=3, scales=0), b"scales"),
                    (dict(n_pos=63), b"tables"), (dict(block=0), b"invalid shape"),
                    (dict(B=2, bts=3), b"stride"), (dict(k=0), b"non-null"),
                    (dict(v_pool=16), b"different"), (dict(cache=3, v_scales=16), b"different"),
                    (dict(mb=1 << 30, n_pos=1 << 40), b"too large")]:
        assert append(**kw) == _lib.MLXP_ERR_INVALID
        assert why in L.mlxp_last_error(), (kw, L.mlxp_last_error())

    def attn(dtype=1, cache=3, H=4, Hk=2, D=64, ptr=16, ps=64, scale=0.1, window=-1, qs=64):
        return L.mlxp_quant_paged_attn(ATTN.pack(
            ptr, 16, 16, 16, 16, 16, 16, 16, 0, 0, dtype, cache, 1, 1, H, Hk, D, 8, 16, 4, 4, 1,
            window, qs, qs, qs, 64, 64, 64, ps, ps, ps, 2, 1, scale, 0, 0, 0))

    for kw, why in [(dict(cache=1), b"e4m3 or int8"), (dict(H=3), b"divisible"), (dict(D=80), b"head_dim"),
                    (dict(ptr=24), b"aligned"), (dict(ps=24), b"multiples of 16"), (dict(qs=60), b"16 bytes"),
                    (dict(scale=0.0), b"scale"), (dict(scale=float("inf")), b"scale"), (dict(window=-2), b"window")]:
        assert attn(**kw) in (_lib.MLXP_ERR_INVALID, _lib.MLXP_ERR_UNSUPPORTED)
        assert why in L.mlxp_last_error(), (kw, L.mlxp_last_error())


# ---- the Python entry points' refusals (made before any device work) ----
def _t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_qk_norm_rope_refusals():
    from mlx_primitives.kernels import qk_norm_rope as f
    q, w, cs = _t(1, 4, 2, 8), _t(8), _t(4, 4)
    for args, why in [((_t(4, 2, 8), q, w, w, cs, cs), "4D"), ((q, _t(2, 4, 2, 8), w, w, cs, cs), "agree"),
                      ((q, q.half(), w, w, cs, cs), "agree"), ((q.double(), q.double(), w, w, cs, cs), "dtype"),
                      ((_t(1, 4, 2, 7), _t(1, 4, 2, 7), w, w), "even"), ((q, q, w, None, cs, cs), "together"),
                      ((q, q, _t(4), w, cs, cs), "q_weight"), ((q, q, w, w, cs, None), "together"),
                      ((q, q, w, w, _t(4, 3), _t(4, 3)), "caches")]:
        with pytest.raises(ValueError, match=why):
            f(*args)
    with pytest.raises(ValueError, match="one length"):
        f(q, _t(1, 3, 2, 8), w, w, cs, cs, positions=_t(1, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="positions"):
        f(q, q, w, w, cs, cs, positions=_t(1, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="positions"):
        f(q, q, w, w, cs, cs, positions=_t(1, 4))


def test_paged_append_refusals():
    from mlx_primitives.cache import paged_append as f
    k, pool = _t(1, 1, 2, 64), _t(3, 16, 2, 64)
    bt, ctx = _t(1, 2, dtype=torch.int32), _t(1, dtype=torch.int32)
    p8, sc = _t(3, 16, 2, 64).to(torch.float8_e4m3fn), _t(3, 2)
    for args, why in [((_t(1, 2, 64), _t(1, 2, 64), pool, pool, bt, ctx), "batch, seq"),
                      ((k, _t(1, 1, 2, 32), pool, pool, bt, ctx), "batch, seq"),
                      ((k, k.half(), pool, pool, bt, ctx), "dtype"),
                      ((k, k, pool.half(), pool.half(), bt, ctx), "dtype"),
                      ((k, k, pool, _t(2, 16, 2, 64), bt, ctx), "num_blocks"),
                      ((k, k, _t(3, 16, 4, 64), _t(3, 16, 4, 64), bt, ctx), "cannot take"),
                      ((k, k, pool, pool.transpose(1, 2).contiguous().transpose(1, 2), bt, ctx), "strides"),
                      ((k, k, p8, p8, bt, ctx), "k_scales"),
                      ((k, k, pool, pool, bt, ctx), "CUDA")]:
        with pytest.raises(ValueError, match=why):
            f(*args)
    with pytest.raises(ValueError, match="scales go with"):
        f(k, k, pool, pool, bt, ctx, k_scales=sc, v_scales=sc)
    with pytest.raises(ValueError, match="v_scales"):
        f(k, k, p8, p8, bt, ctx, k_scales=sc, v_scales=_t(3, 3))


def test_quantized_paged_attention_refusals():
    from mlx_primitives.cache import quantized_paged_attention as f
    q, pool, sc = _t(2, 1, 4, 64), _t(3, 16, 2, 64, dtype=torch.int8), _t(3, 2)
    bt, ctx = _t(2, 2, dtype=torch.int32), _t(2, dtype=torch.int32)
    for args, why in [((_t(2, 4, 64), pool, pool, sc, sc, bt, ctx), "seq_q"),
                      ((q, _t(3, 16, 2, 64), _t(3, 16, 2, 64), None, None, bt, ctx), "e4m3fn or int8"),
                      ((q, pool, pool, None, sc, bt, ctx), "k_scales"),
                      ((q, pool, pool, sc.double(), sc, bt, ctx), "k_scales"),
                      ((_t(2, 1, 4, 32), pool, pool, sc, sc, bt, ctx), "head_dim"),
                      ((_t(2, 1, 3, 64), pool, pool, sc, sc, bt, ctx), "multiple"),
                      ((q.double(), pool, pool, sc, sc, bt, ctx), "dtype"),
                      ((q, pool, pool, sc, sc, _t(1, 2, dtype=torch.int32), ctx), "block_tables"),
                      ((q, pool, pool, sc, sc, bt, _t(3, dtype=torch.int32)), "context_lens")]:
        with pytest.raises(ValueError, match=why):
            f(*args)
    with pytest.raises(ValueError, match="query_lens"):
        f(q, pool, pool, sc, sc, bt, ctx, query_lens=_t(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="window_size"):
        f(q, pool, pool, sc, sc, bt, ctx, window_size=-1)
    with pytest.raises(ValueError, match="alibi"):
        f(q, pool, pool, sc, sc, bt, ctx, alibi_slopes=_t(3))
    with pytest.raises(NotImplementedError, match="differentiable"):
        f(q.requires_grad_(True), pool, pool, sc, sc, bt, ctx)


def test_short_calls_leave_what_they_do_not_take_to_python():
    """The C++ half of the shim answers None (take the long way) to anything but device tensors
    that can be used as they are, and never raises for them."""
    from mlx_primitives import _lib
    calls = _lib.calls()
    q, w, cs = _t(1, 4, 2, 8), _t(8), _t(4, 4)
    assert calls.norm_rope(q, q, w, w, cs, cs, None, 0, 0, 1e-6) is None           # host tensors
    assert calls.norm_rope(q, 3, w, w, cs, cs, None, 0, 0, 1e-6) is None           # not a tensor
    assert calls.norm_rope(q, q, w, w, cs, cs, None, 0, 0, 1) is None              # eps not a float
    assert calls.norm_rope(q) is None
    pool, i = _t(3, 16, 2, 8), _t(1, dtype=torch.int32)
    assert calls.append(q, q, pool, pool, _t(1, 1, dtype=torch.int32), i, None, None, None, None, None,
                        None, None, None, 1e-6) is None
    assert calls.append(*[None] * 14, 1e-6) is None
    assert calls.attend(q, pool, pool, None, None, _t(1, 1, dtype=torch.int32), i, None, None, True, -1) is None
    assert calls.attend(*[None] * 9, True, -1) is None
