"""Query/key norm + rotation, appending to paged pools and 8-bit paged attention on the GPU,
against their fp64 oracle (oracle/cache_oracle.py) fed the same rounded inputs.

Tolerances.  An output of type T is one rounding of an fp32 result: half a step, eps_T / 2 of the
value, beside the fp32 computation's own error, which is counted against the size of the terms
that were added.  Attention's weights are rounded to fp16 (half a step, 2^-11 of the weight; two
fp16 terms, 2^-22, for fp32 queries) and its scores are fp32 sums, so that error is counted
against the softmax-weighted mean of |v|, which the oracle gives."""

import numpy as np
import pytest
import torch

from oracle import cache_oracle as C

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CACHES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def _n(t):
    return t.detach().to(torch.float64).cpu().numpy()


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _close(got, want, dtype, slack):
    """|got - want| <= half a step of want + slack (an array or number, of the fp32 part)."""
    got = _n(got)
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2  # subnormal half step
    tol = _half(dtype) * np.abs(want) + np.asarray(slack) * (1 + _half(dtype)) + tiny
    # what lies past the largest value by half a step rounds to infinity
    top = torch.finfo(dtype).max * (1 + _half(dtype) / 2)
    inf = np.isinf(got) & (np.sign(got) == np.sign(want)) & (np.abs(want) + np.asarray(slack) >= top)
    got = np.where(inf, want, got)
    off = np.nan_to_num(np.abs(got - want)) - np.nan_to_num(tol)
    assert off.max(initial=-1.0) <= 0, f"worst excess {off.max()}"


def _tables(n, half):
    ang = np.outer(np.arange(n), 10000.0 ** (-np.arange(half) / half))
    return (torch.from_numpy(f(ang)).float().cuda() for f in (np.cos, np.sin))


def _rand(rs, shape, dtype, size=1.0):
    return torch.from_numpy(rs.standard_normal(shape) * size).to(dtype).cuda()


# ------------------------------------------------------------------ norm + rotation
def _amp(y):
    """Row amplitude: what the rotation adds up is at most this, twice."""
    return np.nan_to_num(np.abs(y)).max(-1, keepdims=True)


def _norm_case(B, S, Hq, Hk, D, dtype, seed=0, wdtype=torch.float32, size=1.0):
    rs = np.random.RandomState(seed)
    q, k = _rand(rs, (B, S, Hq, D), dtype, size), _rand(rs, (B, S, Hk, D), dtype, size)
    qw, kw = ((1 + 0.1 * _rand(rs, (D,), torch.float32)).to(wdtype) for _ in range(2))
    return q, k, qw, kw


def _check_norm(q, k, qw, kw, cos, sin, pos, out, eps=1e-6):
    for x, w, y in ((q, qw, out[0]), (k, kw, out[1])):
        c, s = (None, None) if cos is None else (_n(cos), _n(sin))
        want = C.norm_rope(_n(x), None if w is None else _n(w), c, s, pos, eps)
        # norm: ~D/32 + 5 adds and rsqrt, 2^-20 relative; rotation: two terms of at most the amplitude
        _close(y, want, x.dtype, 2.0 ** -20 * 2 * _amp(want))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [2, 6, 32, 64, 80, 96, 128, 250, 256])
def test_norm_rope_forward(dtype, D):
    from mlx_primitives.kernels import qk_norm_rope
    q, k, qw, kw = _norm_case(2, 7, 9, 3, D, TYPES[dtype], seed=D)
    cos, sin = _tables(16, D // 2)
    out = qk_norm_rope(q, k, qw, kw, cos, sin, offset=5)
    assert out[0].dtype == q.dtype and out[0].shape == q.shape
    _check_norm(q, k, qw, kw, cos, sin, np.tile(5 + np.arange(7), (2, 1)), out)


@pytest.mark.parametrize("S", [1, 2, 129])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (32, 8), (33, 5)])
def test_norm_rope_positions_padding_and_past_the_tables(S, Hq, Hk):
    from mlx_primitives.kernels import qk_norm_rope
    q, k, qw, kw = _norm_case(3, S, Hq, Hk, 64, torch.bfloat16, seed=S)
    cos, sin = _tables(40, 32)
    pos = np.random.RandomState(S).randint(-1, 42, (3, S))
    pos[0, 0] = -1
    q[0, 0] = float("nan")  # what padding holds does not matter
    k[0, 0] = float("inf")
    out = qk_norm_rope(q, k, qw, kw, cos, sin, positions=torch.from_numpy(pos).cuda())
    assert torch.all(out[0][0, 0] == 0) and torch.all(out[1][0, 0] == 0)
    _check_norm(q, k, qw, kw, cos, sin, pos, out)


@pytest.mark.parametrize("wdtype", ["bf16", "fp16", "fp32"])
def test_norm_only_and_rotation_only(wdtype):
    from mlx_primitives.kernels import qk_norm_rope, rope_qk
    q, k, qw, kw = _norm_case(2, 5, 4, 2, 128, torch.bfloat16, wdtype=TYPES[wdtype])
    pos = np.tile(np.arange(5), (2, 1))
    _check_norm(q, k, qw, kw, None, None, pos, qk_norm_rope(q, k, qw, kw))
    cos, sin = _tables(8, 64)
    out = qk_norm_rope(q, k, None, None, cos, sin)
    for a, b in zip(out, rope_qk(q, k, cos, sin)):
        assert torch.equal(a, b)  # the same arithmetic as rope's kernel


def test_norm_rope_views_lengths_and_extremes():
    from mlx_primitives.kernels import qk_norm_rope
    rs = np.random.RandomState(3)
    cos, sin = _tables(64, 32)
    w = (1 + 0.1 * _rand(rs, (64,), torch.float32))
    base = _rand(rs, (2, 6, 11, 64), torch.bfloat16)              # BHSD storage
    q = base.transpose(1, 2)
    fused = _rand(rs, (2, 9, 8, 64), torch.bfloat16)              # k as a slice of a projection
    k = fused[:, :, 4:7]
    out = qk_norm_rope(q, k, w, w, cos, sin, offset=3, k_offset=50)
    for x, y, off in ((q, out[0], 3), (k, out[1], 50)):
        want = C.norm_rope(_n(x), _n(w), _n(cos), _n(sin), np.tile(off + np.arange(x.shape[1]), (2, 1)))
        _close(y, want, x.dtype, 2.0 ** -19 * _amp(want))
    odd = _rand(rs, (2 * 5 * 3 * 64 + 1,), torch.bfloat16)[1:].view(2, 5, 3, 64)  # 2-byte aligned
    out = qk_norm_rope(odd, odd, w, w, cos, sin)
    _check_norm(odd, odd, w, w, cos, sin, np.tile(np.arange(5), (2, 1)), out)
    one = _rand(rs, (1, 5, 3, 64), torch.bfloat16).expand(4, 5, 3, 64)
    _check_norm(one, one, w, w, cos, sin, np.tile(np.arange(5), (4, 1)), qk_norm_rope(one, one, w, w, cos, sin))
    # rows of zeros, and of large and small values: r is 1/sqrt(eps), or x's inverse size
    x = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    x[0, 1], x[0, 2], x[0, 3] = 1e18, 1e-4, -3.0
    _check_norm(x, x, w, w, cos, sin, np.arange(4)[None], qk_norm_rope(x, x, w, w, cos, sin))
    # empty batches, lengths and both
    for shape in ((0, 5, 3, 64), (2, 0, 3, 64)):
        e = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        assert qk_norm_rope(e, e, w, w, cos, sin)[0].shape == shape
    h = qk_norm_rope(q.cpu(), k.cpu(), w, w, cos, sin)
    assert h[0].device.type == "cpu" and torch.equal(h[0], qk_norm_rope(q, k, w, w, cos, sin)[0].cpu())


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,S,Hq,Hk,D,padded", [(1, 1, 1, 1, 64, False), (2, 37, 8, 2, 128, True),
                                                (3, 300, 5, 5, 80, False), (2, 65, 4, 1, 256, True),
                                                (1, 50, 3, 2, 6, True)])
def test_norm_rope_gradients(dtype, B, S, Hq, Hk, D, padded):
    from mlx_primitives.kernels import qk_norm_rope
    dt = TYPES[dtype]
    leaves = _norm_case(B, S, Hq, Hk, D, dt, seed=B + S)
    q, k, qw, kw = (t.requires_grad_(True) for t in leaves)
    rs = np.random.RandomState(9)
    gq, gk = _rand(rs, q.shape, dt), _rand(rs, k.shape, dt)
    cos, sin = _tables(S + 4, D // 2)
    pos = np.tile(np.arange(S), (B, 1))
    if padded:
        pos[0, S // 2:] = -1
        with torch.no_grad():
            q[0, S // 2:] = float("nan")
    out = qk_norm_rope(q, k, qw, kw, cos, sin, positions=torch.from_numpy(pos).cuda() if padded else None)
    got = torch.autograd.grad(out, (q, k, qw, kw), (gq, gk))
    again = torch.autograd.grad(qk_norm_rope(q, k, qw, kw, cos, sin, positions=torch.from_numpy(pos).cuda()),
                                (q, k, qw, kw), (gq, gk))
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for x, w, g, dx, dw in ((q, qw, gq, got[0], got[2]), (k, kw, gk, got[1], got[3])):
        want, wsum, wabs = C.norm_rope_grad(_n(g), _n(x), _n(w), _n(cos), _n(sin), pos)
        # terms of dx: r g w and r xhat mean(g w xhat), each at most r |g| |w| sqrt(D)-ish: counted
        # against the row's largest term
        size = np.abs(_n(g)).max(-1, keepdims=True) * 3 / np.sqrt(
            np.where((pos >= 0)[:, :, None, None], (np.nan_to_num(_n(x)) ** 2).mean(-1, keepdims=True), 1) + 1e-6)
        _close(dx, want, dt, 2.0 ** -19 * size)
        # B*S*H terms, added in fp32 in a tree whose longest chain is at most all of them
        chain = B * S * x.shape[2] / 8 + 64
        assert np.all(np.abs(_n(dw) - wsum) <= 2.0 ** -24 * chain * wabs + 2.0 ** -20 * wabs)


def test_norm_rope_gradients_partial_graphs():
    """One output unused, weights frozen, no weights, bf16 weights, expanded output gradients."""
    from mlx_primitives.kernels import qk_norm_rope
    q, k, qw, kw = _norm_case(2, 9, 4, 2, 64, torch.float32)
    cos, sin = _tables(16, 32)
    pos = np.tile(np.arange(9), (2, 1))
    q.requires_grad_(True), k.requires_grad_(True)
    out = qk_norm_rope(q, k, qw, kw, cos, sin)
    out[0].sum().backward()
    want, _, _ = C.norm_rope_grad(np.ones(q.shape), _n(q), _n(qw), _n(cos), _n(sin), pos)
    assert k.grad is None or torch.all(k.grad == 0)
    assert np.abs(_n(q.grad) - want).max() < 1e-4
    kb = kw.bfloat16().requires_grad_(True)
    out = qk_norm_rope(q.detach(), k.detach(), qw.bfloat16(), kb, cos, sin)
    (g,) = torch.autograd.grad(out[1].sum(), (kb,))
    _, wsum, wabs = C.norm_rope_grad(np.ones(k.shape), _n(k), _n(kb), _n(cos), _n(sin), pos)
    assert g.dtype == torch.bfloat16
    assert np.all(np.abs(_n(g) - wsum) <= 2.0 ** -8 * np.abs(wsum) + 2.0 ** -18 * wabs)
    out = qk_norm_rope(q, k, None, None, cos, sin)
    gq, gk = torch.autograd.grad(out[0].sum() + out[1].sum(), (q, k))
    for x, gx in ((q, gq), (k, gk)):
        want, _, _ = C.norm_rope_grad(np.ones(x.shape), _n(x), None, _n(cos), _n(sin), pos)
        assert np.abs(_n(gx) - want).max() < 1e-6
    with pytest.raises(RuntimeError):  # no second derivative: refused, not silently wrong
        x = q.detach().requires_grad_(True)
        (g1,) = torch.autograd.grad(qk_norm_rope(x, k, qw, kw, cos, sin)[0].sum(), (x,), create_graph=True)
        g1.sum().backward()


# ------------------------------------------------------------------ append
def _pool_case(rs, lens, block, Hk, D, dtype, kind, spare=2, mb_extra=1):
    """Tables with shuffled ids, pools of random contents (codes and scales for `kind`)."""
    need = [-(-max(int(n), 0) // block) for n in lens]
    mb = max(need) + mb_extra
    nblk = sum(need) + spare
    ids = rs.permutation(nblk)
    bt = np.full((len(lens), mb), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = ids[at:at + n]
        at += n
    shape = (nblk, block, Hk, D)
    if kind is None:
        return bt, [_rand(rs, shape, dtype) for _ in range(2)], (None, None)
    pools = []
    for _ in range(2):
        x = torch.from_numpy(rs.standard_normal(shape) * 40).float().cuda()
        pools.append(x.to(CACHES[kind]) if kind == "e4m3" else x.round().clamp(-127, 127).to(torch.int8))
    scales = [torch.from_numpy(2.0 ** rs.randint(-8, -3, (nblk, Hk))).float().cuda() for _ in range(2)]
    return bt, pools, scales


def _check_append(k64, v64, rotated, before, pools, scales, bt, ctx, new, kind, dtype):
    """The pools against the oracle's: exact where the values are the inputs', within a rounding
    where they are computed (`rotated`: the keys)."""
    for name, x, was, is_, sc0, sc in (("k", k64, before[0], pools[0], before[2], scales[0]),
                                       ("v", v64, before[1], pools[1], before[3], scales[1])):
        want, wsc, written = C.append(x, was, bt, ctx, new, sc0, kind)
        got = _n(is_)
        exact = not (rotated and name == "k")
        if kind is None:
            if exact:
                assert np.array_equal(got, want), name
            else:
                assert np.array_equal(got[~written], want[~written])
                _close(is_[torch.from_numpy(written).cuda()], want[written], dtype,
                       2.0 ** -19 * _amp(want[written]))
            continue
        assert np.array_equal(_n(sc), wsc), name  # inputs are not within fp32 noise of a border
        if exact:
            assert np.array_equal(got, want, equal_nan=True), name
        else:
            # a code moves one step where fp32 noise (2^-19 of the row) crosses a tie: the steps
            # are at most 32 (e4m3) or 1 (int8) at codes to 448 or 127, so noise hits few
            diff = got != want
            assert diff.mean() < 2e-3
            step = np.maximum(2.0 ** (np.floor(np.log2(np.maximum(np.abs(want), 2.0 ** -6))) - 3), 2.0 ** -9)
            assert np.all(np.abs(got - want)[diff] <= (1.0 if kind == "int8" else step[diff] * 2))


@pytest.mark.parametrize("dtype,D,kind,block", [
    ("bf16", 128, None, 16), ("fp16", 64, None, 24), ("fp32", 96, None, 1), ("bf16", 6, None, 7),
    ("bf16", 128, "e4m3", 16), ("bf16", 128, "int8", 16), ("fp16", 64, "e4m3", 24), ("fp32", 64, "int8", 128),
    ("bf16", 64, "e4m3", 300), ("fp32", 128, "e4m3", 8), ("bf16", 10, "int8", 5), ("bf16", 256, "e4m3", 32),
    ("fp32", 256, "e4m3", 16), ("bf16", 80, "e4m3", 1)])
@pytest.mark.parametrize("S", [1, 5, 70])
def test_append_matches_oracle(dtype, D, kind, block, S):
    from mlx_primitives.cache import paged_append
    rs = np.random.RandomState(D + block + S)
    dt, Hk, Hq = TYPES[dtype], 3, 5
    ctx = np.array([0, 1, 33, block, 4 * block - 1])
    new = np.array([S, max(S - 3, 0), S, S, 1])
    bt, pools, scales = _pool_case(rs, ctx + new, block, Hk, D, dt, kind)
    k, v, q = (_rand(rs, (5, S, h, D), dt, 2.0) for h in (Hk, Hk, Hq))
    cos, sin = _tables(bt.shape[1] * block, D // 2)
    qw, kw = (1 + 0.1 * _rand(rs, (D,), torch.float32) for _ in range(2))
    at = ctx[:, None] + np.arange(S)
    at = np.where(np.arange(S) < new[:, None], at, -1)
    for rotated in (False, True):
        before = [_n(t) if t is not None else None for t in (*pools, *scales)]
        extra = dict(cos_cache=cos, sin_cache=sin, k_weight=kw, q_weight=qw, q=q) if rotated else {}
        qo = paged_append(k, v, *pools, torch.from_numpy(bt).cuda(), torch.from_numpy(ctx).cuda(),
                          new_lens=torch.from_numpy(new).cuda(), k_scales=scales[0], v_scales=scales[1], **extra)
        k64 = C.norm_rope(_n(k), _n(kw), _n(cos), _n(sin), at) if rotated else _n(k)
        _check_append(k64, _n(v), rotated, before, pools, scales, bt, ctx, new, kind, dt)
        if rotated:
            want = C.norm_rope(_n(q), _n(qw), _n(cos), _n(sin), at)
            _close(qo, want, dt, 2.0 ** -19 * _amp(want))
        else:
            assert qo is None


@pytest.mark.parametrize("kind", [None, "e4m3"])
def test_append_drops_what_has_no_place(kind):
    from mlx_primitives.cache import paged_append
    rs = np.random.RandomState(4)
    block, Hk, D, S = 16, 2, 64, 20
    ctx = np.array([-5, 60, 0, 1 << 30, 3])
    new = np.array([20, 20, -1, 20, 99])
    bt, pools, scales = _pool_case(rs, [64] * 5, block, Hk, D, torch.bfloat16, kind, mb_extra=0)
    bt[0, 0] = -1                      # the first block is missing, the token range reaches it
    bt[4, 1] = pools[0].shape[0]       # an id past the pool
    k, v, q = (_rand(rs, (5, S, h, D), torch.bfloat16) for h in (Hk, Hk, 3))
    cos, sin = _tables(64, 32)
    before = [_n(t) if t is not None else None for t in (*pools, *scales)]
    qo = paged_append(k, v, *pools, torch.from_numpy(bt).cuda(), torch.from_numpy(ctx).cuda(), q=q,
                      new_lens=torch.from_numpy(new).cuda(), k_scales=scales[0], v_scales=scales[1],
                      cos_cache=cos, sin_cache=sin)
    at = ctx[:, None] + np.arange(S)
    at = np.where((np.arange(S) < new[:, None]) & (at < 64), at, -1)
    _check_append(C.norm_rope(_n(k), None, _n(cos), _n(sin), at), _n(v), True, before, pools, scales,
                  bt, ctx, new, kind, torch.bfloat16)
    _close(qo, C.norm_rope(_n(q), None, _n(cos), _n(sin), at), torch.bfloat16, 2.0 ** -19 * 6)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_token_by_token_equals_its_definition(kind):
    """A block filled one token at a time: the scale grows with the largest token so far."""
    from mlx_primitives.cache import paged_append
    rs = np.random.RandomState(8)
    block, Hk, D, n = 16, 2, 128, 40
    bt, pools, scales = _pool_case(rs, [n], block, Hk, D, torch.bfloat16, kind)
    want = [_n(pools[1]), _n(scales[1])]
    for t in range(n):
        v = _rand(rs, (1, 1, Hk, D), torch.bfloat16, 2.0 ** rs.randint(-6, 7))
        paged_append(v, v, *pools, torch.from_numpy(bt).cuda(), torch.tensor([t], device="cuda"),
                     k_scales=scales[0], v_scales=scales[1])
        want[0], want[1], _ = C.append(_n(v), want[0], bt, [t], [1], want[1], kind)
        assert np.array_equal(_n(scales[1]), want[1]) and np.array_equal(_n(pools[1]), want[0])
    blocks = torch.from_numpy(bt[0, :3].astype(np.int64)).cuda()
    for a, b in ((pools[0], pools[1]), (scales[0], scales[1])):
        a, b = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (a, b))
        assert torch.equal(a[blocks[0]], b[blocks[0]])


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_zeros_infinities_and_nan(kind):
    from mlx_primitives.cache import paged_append
    rs = np.random.RandomState(5)
    bt, pools, scales = _pool_case(rs, [16, 16, 16], 16, 1, 64, torch.float32, kind)
    v = torch.zeros(3, 16, 1, 64, device="cuda")
    v[1, 3, 0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), 2.0])
    v[2, 0, 0, 0] = 3e38
    paged_append(v, v, *pools, torch.from_numpy(bt).cuda(), torch.zeros(3, dtype=torch.int32, device="cuda"),
                 k_scales=scales[0], v_scales=scales[1])
    blk = bt[:, 0].astype(np.int64)
    sc, codes = _n(scales[1])[blk, 0], _n(pools[1])[blk][:, :, 0]
    qmax = C.QMAX[kind]
    assert sc[0] == 2.0 ** -126 and not codes[0].any()
    assert sc[1] == C.least_scale(2.0, kind)
    row = codes[1, 3, :4]
    assert row[0] == qmax and row[1] == -qmax and row[3] * sc[1] == 2.0
    assert np.isnan(row[2]) if kind == "e4m3" else row[2] == 0
    assert abs(codes[2, 0, 0] * sc[2] / 3e38 - 1) <= 1 / 16 and np.isfinite(sc[2])


@pytest.mark.parametrize("kind", [None, "e4m3"])
def test_append_strides_and_alignment(kind):
    """Pools interleaved in one tensor, heads before tokens, and an unaligned view; k from a fused
    projection."""
    from mlx_primitives.cache import paged_append
    rs = np.random.RandomState(6)
    block, Hk, D, S = 8, 2, 64, 11
    ctx, new = np.array([5, 0]), np.array([S, S])
    dt = torch.bfloat16
    bt, (kp, vp), scales = _pool_case(rs, ctx + new, block, Hk, D, dt, kind)
    qkv = _rand(rs, (2, S, 8, D), dt)
    k, v = qkv[:, :, 4:6], qkv[:, :, 6:]
    raw = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
    es = raw(kp).element_size()

    def interleaved():
        both = torch.stack((raw(kp), raw(vp)), 1)
        return both[:, 0], both[:, 1]

    def heads_first():
        return tuple(raw(t).transpose(1, 2).contiguous().transpose(1, 2) for t in (kp, vp))

    def unaligned():
        out = []
        for t in (kp, vp):
            buf = torch.empty(t.numel() + 1, dtype=raw(t).dtype, device="cuda")
            out.append(buf[1:].view(t.shape))
            out[-1].copy_(raw(t))
            assert out[-1].data_ptr() % 16 == es
        return tuple(out)

    for make in (interleaved, heads_first, unaligned):
        pools = tuple(t.view(kp.dtype) for t in make())
        sc = tuple(None if s is None else s.clone() for s in scales)
        before = [_n(t) if t is not None else None for t in (*pools, *sc)]
        paged_append(k, v, *pools, torch.from_numpy(bt).cuda(), torch.from_numpy(ctx).cuda(),
                     k_scales=sc[0], v_scales=sc[1])
        _check_append(_n(k), _n(v), False, before, pools, sc, bt, ctx, new, kind, dt)
    flat = torch.zeros(1, 8, 2, 64, dtype=dt, device="cuda").expand(4, 8, 2, 64)
    with pytest.raises(ValueError, match="overlap"):
        paged_append(k, v, flat, flat, torch.from_numpy(bt).cuda(), torch.from_numpy(ctx).cuda())
    with pytest.raises(ValueError, match="cover"):
        c, s = _tables(4, 32)
        paged_append(k, v, kp, vp, torch.from_numpy(bt).cuda(), torch.from_numpy(ctx).cuda(), cos_cache=c,
                     sin_cache=s, k_scales=scales[0], v_scales=scales[1])
    with pytest.raises(NotImplementedError, match="no_grad"):
        paged_append(k.detach().requires_grad_(True), v, kp, vp, torch.from_numpy(bt).cuda(),
                     torch.from_numpy(ctx).cuda(), k_scales=scales[0], v_scales=scales[1])


def test_append_past_32_bits():
    """Rows of a pool of more than 2^31 elements."""
    from mlx_primitives.cache import paged_append
    nblk, block, Hk, D = (1 << 31) // (64 * 8 * 128) + 3, 64, 8, 128
    pool = torch.zeros(nblk, block, Hk, D, dtype=torch.int8, device="cuda")
    sc = torch.ones(nblk, Hk, device="cuda")
    rs = np.random.RandomState(1)
    k = _rand(rs, (1, 2, Hk, D), torch.bfloat16)
    bt = torch.tensor([[nblk - 1]], dtype=torch.int32, device="cuda")
    paged_append(k, k, pool, pool.clone(), bt, torch.tensor([5], device="cuda"), k_scales=sc, v_scales=sc.clone())
    want, wsc, _ = C.append(_n(k), np.zeros((1, block, Hk, D)), np.array([[0]]), [5], [2], np.ones((1, Hk)), "int8")
    assert np.array_equal(_n(pool[nblk - 1]), want[0]) and np.array_equal(_n(sc[nblk - 1]), wsc[0])
    assert not pool[:4].any() and not pool[nblk // 2].any()


# ------------------------------------------------------------------ 8-bit attention
def _attn_case(rs, lens, H, Hk, D, block, dtype, kind, Sq=1, qsize=2.0):
    bt, pools, _ = _pool_case(rs, lens, block, Hk, D, dtype, kind, spare=3, mb_extra=2)
    scales = [torch.from_numpy(2.0 ** rs.randint(-7, -4, (pools[0].shape[0], Hk)) *
                               (1 + rs.rand(pools[0].shape[0], Hk))).float().cuda() for _ in range(2)]
    q = _rand(rs, (len(lens), Sq, H, D), dtype, qsize)
    return q, pools, scales, bt, np.asarray(lens, dtype=np.int32)


def _attend(q, pools, scales, bt, ctx, **kw):
    from mlx_primitives.cache import quantized_paged_attention
    kw = {k: torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v for k, v in kw.items()}
    return quantized_paged_attention(q, *pools, *scales, torch.from_numpy(bt).cuda(),
                                     torch.from_numpy(ctx).cuda(), **kw)


def _check_attn(out, q, pools, scales, bt, ctx, **kw):
    kw = {{"window_size": "window", "alibi_slopes": "slopes"}.get(k, k): v for k, v in kw.items()}
    want, size, floor = C.quantized_attention(_n(q), _n(pools[0]), _n(pools[1]), _n(scales[0]),
                                              _n(scales[1]), bt, ctx, **kw)
    assert out.shape == q.shape and out.dtype == q.dtype
    # weights 2^-11 (2^-22 split); scores and sums in fp32, the scores' error (2^-24 times up to
    # a few dozen terms of up to ~2^4 each) turns into the same relative error of the weights
    slack = 2.0 ** -15 if q.dtype == torch.float32 else 2.0 ** -11 + 2.0 ** -14
    # The weights w_t vs_t are held as 2^15 times their ratio to the largest so far.  Below 2^-14
    # (2^-29 of the largest) fp16 is subnormal, its step 2^-24: half of that, 2^-25, is 2^-40 of
    # the largest weight, and each key's code multiplies such an error once.  2^-39: normalised
    # by a sum and a largest weight that carry `slack` themselves.  The many-row kernel (64 query
    # rows a pool head and more, 16-bit) holds them as 2^8 times their ratio to a maximum that the
    # largest may exceed 2^7 times: 2^-25 is then 2^-33 of the largest weight at most, twice that
    # here.
    many = q.dtype != torch.float32 and q.shape[1] * (q.shape[2] // pools[0].shape[2]) >= 64
    _close(out, want, q.dtype, slack * size + 2.0 ** (-32 if many else -39) * floor)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("H,Hk,block", [(8, 2, 16), (4, 4, 24), (12, 1, 64), (6, 3, 8)])
def test_attention_decode(dtype, kind, D, H, Hk, block):
    rs = np.random.RandomState(D + H + block)
    case = _attn_case(rs, [1, 0, 17, 300, 1000, 64, 15, 2048], H, Hk, D, block, TYPES[dtype], kind)
    out = _attend(*case)
    assert torch.all(out[1] == 0)
    _check_attn(out, *case)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("Sq", [2, 3, 9, 40])
@pytest.mark.parametrize("kw", [dict(), dict(causal=False), dict(window_size=0), dict(window_size=37),
                                dict(window_size=20, causal=False)])
def test_attention_rows_masks_and_query_lens(dtype, Sq, kw):
    rs = np.random.RandomState(Sq)
    # a context shorter than the queries: the first rows see nothing
    lens = [Sq, 1, 130, 77, 260, 0]
    case = _attn_case(rs, lens, 8, 2, 64, 16, TYPES[dtype], "e4m3", Sq=Sq)
    _check_attn(_attend(*case, **kw), *case, **kw)
    ql = np.array([Sq, 1, 0, Sq - 1, Sq, 2], dtype=np.int32)
    out = _attend(*case, query_lens=ql, **kw)
    _check_attn(out, *case, query_lens=ql, **kw)
    for b, n in enumerate(ql):
        assert torch.all(out[b, n:] == 0)


@pytest.mark.parametrize("block", [1, 7, 16, 20, 48])
@pytest.mark.parametrize("Sq", [1, 5])
def test_attention_block_sizes_holes_alibi_and_scale(block, Sq):
    from mlx_primitives.cache import get_alibi_slopes
    rs = np.random.RandomState(block)
    q, pools, scales, bt, ctx = _attn_case(rs, [200, 333, 90], 6, 3, 128, block, torch.bfloat16, "int8", Sq=Sq)
    bt[0, 1], bt[1, 0], bt[2, bt.shape[1] // 3] = -1, -7, pools[0].shape[0] + 9  # holes
    slopes = get_alibi_slopes(6).numpy()
    case = (q, pools, scales, bt, ctx)
    _check_attn(_attend(*case), *case)
    _check_attn(_attend(*case, alibi_slopes=slopes, scale=0.3), *case, alibi_slopes=slopes, scale=0.3)
    bt[:] = -1
    assert torch.all(_attend(q, pools, scales, bt, ctx) == 0)


def test_attention_never_reads_stale_bytes():
    """Rows behind the context, unused blocks and their scales may hold anything, NaN codes and
    infinities among it."""
    rs = np.random.RandomState(12)
    for block in (16, 20):
        q, pools, scales, bt, ctx = _attn_case(rs, [37, 80, 5], 8, 2, 64, block, torch.bfloat16, "e4m3", Sq=3)
        used = np.zeros(pools[0].shape[:2], dtype=bool)
        for b, n in enumerate(ctx):
            t = np.arange(n)
            used[bt[b, t // block], t % block] = True
        stale = torch.from_numpy(~used).cuda()
        for p in pools:
            p.view(torch.uint8)[stale] = 0x7F
        free = torch.from_numpy(~used.any(1)).cuda()
        for s in scales:
            s[free] = float("nan")
        clean = [torch.where(stale[..., None, None], torch.zeros_like(p.view(torch.uint8)), p.view(torch.uint8))
                 .view(p.dtype) for p in pools]
        csc = [torch.where(free[:, None], torch.ones_like(s), s) for s in scales]
        out = _attend(q, pools, scales, bt, ctx)
        assert torch.isfinite(out).all()
        _check_attn(out, q, clean, csc, bt, ctx)


def test_attention_scales_of_any_size_and_large_scores():
    rs = np.random.RandomState(13)
    for dtype in (torch.bfloat16, torch.float32):
        q, pools, scales, bt, ctx = _attn_case(rs, [700, 130], 8, 2, 64, 16, dtype, "e4m3")
        # v scales spread over 2^+-40, k scales such that scores differ by hundreds, zero scales
        scales[1] *= torch.from_numpy(2.0 ** rs.randint(-40, 40, scales[1].shape)).float().cuda()
        scales[0] *= torch.from_numpy(2.0 ** rs.randint(-3, 4, scales[0].shape)).float().cuda()
        scales[1][bt[0, 3]] = 0.0
        scales[0][bt[0, 4]] = 0.0
        want, size, floor = C.quantized_attention(_n(q), _n(pools[0]), _n(pools[1]), _n(scales[0]), _n(scales[1]), bt, ctx)
        got = _n(_attend(q, pools, scales, bt, ctx))
        # scores of up to ~2^9, so fp32 sums put 2^-24 * 2^9 * few into the weights' exponents
        slack = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -13
        assert np.all(np.abs(got - want) <= (_half(dtype) + 1e-7) * np.abs(want) + (slack + 2.0 ** -12) * size + 2.0 ** -39 * floor)
        scales[1].zero_()
        assert torch.all(_attend(q, pools, scales, bt, ctx) == 0)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_attention_long_context_split_over_ctas(kind):
    """One sequence split over every SM, beside short ones; a row at each chunk border."""
    rs = np.random.RandomState(14)
    case = _attn_case(rs, [20011, 1, 63, 64, 65, 4096], 8, 2, 64, 32, torch.bfloat16, kind)
    _check_attn(_attend(*case), *case)
    case = _attn_case(rs, [9000], 4, 1, 128, 16, torch.float16, kind, Sq=2)
    _check_attn(_attend(*case), *case)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk,Sq", [(2, 2, 64), (4, 2, 61), (8, 2, 33), (6, 1, 75)])
def test_attention_many_rows(dtype, kind, D, H, Hk, Sq):
    """The many-row kernel: one and two row tiles, partly filled; contexts at its tiles' borders
    and shorter than the queries."""
    rs = np.random.RandomState(D + Sq)
    case = _attn_case(rs, [Sq, 128, 129, 700, 1, 0, 255], H, Hk, D, 16, TYPES[dtype], kind, Sq=Sq)
    out = _attend(*case)
    assert torch.all(out[5] == 0) and torch.all(out[4, :Sq - 1] == 0)
    _check_attn(out, *case)


@pytest.mark.parametrize("kw", [dict(), dict(causal=False), dict(window_size=0), dict(window_size=100),
                                dict(window_size=50, causal=False), dict(scale=0.3)])
def test_attention_many_rows_masks_query_lens_and_holes(kw):
    rs = np.random.RandomState(31)
    q, pools, scales, bt, ctx = _attn_case(rs, [300, 90, 1000, 513], 8, 2, 64, 32, torch.bfloat16, "e4m3", Sq=70)
    bt[0, 2], bt[2, 5], bt[3, 0] = -1, pools[0].shape[0], -1
    ql = np.array([70, 3, 0, 69], dtype=np.int32)
    for lens in (None, ql):
        more = {} if lens is None else dict(query_lens=lens)
        out = _attend(q, pools, scales, bt, ctx, **kw, **more)
        _check_attn(out, q, pools, scales, bt, ctx, **kw, **more)
    for b, n in enumerate(ql):
        assert torch.all(out[b, n:] == 0)
    bt[:] = -1
    assert torch.all(_attend(q, pools, scales, bt, ctx, **kw) == 0)


@pytest.mark.parametrize("Sq", [1, 5, 70])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_windows_wider_than_any_context(Sq, causal):
    case = _attn_case(np.random.RandomState(36), [300, 90], 8, 2, 64, 16, torch.bfloat16, "e4m3", Sq=Sq)
    want = _attend(*case, causal=causal)
    assert want.abs().max() > 0
    for window in (10 ** 6, 2 ** 31, 2 ** 62, 2 ** 63 - 1):
        assert torch.equal(_attend(*case, causal=causal, window_size=window), want)


def test_norm_rope_of_unfolded_views():
    """Queries that overlap themselves, position t + 1 one element behind position t.

    They are not 16-byte aligned, so their sums of 64 squares (and products) run in another order:
    64 half steps, 2^-18 of a term of at most 2^4 (|x|, |g|, |w| < 4), each of four terms: 2^-12."""
    from mlx_primitives.kernels import qk_norm_rope

    tol = 2.0 ** -12
    rs = np.random.RandomState(37)
    D, S = 64, 5
    cos, sin = _tables(16, D // 2)
    base = _rand(rs, (2, 1, D + S), torch.float32)
    w = _rand(rs, (D,), torch.float32)
    views = [base.as_strided((2, S, 1, D), (D + S, 1, D + S, 1)), base.as_strided((2, S, 4, D), (D + S, 0, 1, 1))]
    for x in views:
        for q in (x, x.detach().requires_grad_(True)):
            got = qk_norm_rope(q, q, w, w, cos, sin)
            want = qk_norm_rope(x.contiguous(), x.contiguous(), w, w, cos, sin)
            for i in range(2):
                assert (got[i] - want[i]).abs().max() <= tol
        dense = x.contiguous().requires_grad_(True)
        g = _rand(rs, tuple(x.shape), torch.float32)
        a, = torch.autograd.grad(qk_norm_rope(q, q, w, w, cos, sin)[0], q, g)
        b, = torch.autograd.grad(qk_norm_rope(dense, dense, w, w, cos, sin)[0], dense, g)
        assert (a - b).abs().max() <= tol


def test_norm_rope_graphs_kept_freed_and_modified():
    """A kept graph runs twice, a freed one is refused, as are values changed since; inputs that need
    no gradient get none, and hooks and accumulation see the same gradients."""
    from mlx_primitives.kernels import qk_norm_rope

    rs = np.random.RandomState(38)
    q, k, w = _rand(rs, (2, 7, 4, 64), torch.bfloat16), _rand(rs, (2, 7, 2, 64), torch.bfloat16), _rand(rs, (64,), torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, w, w)]
    out = qk_norm_rope(*leaves)
    g = [torch.ones_like(o) for o in out]
    first = torch.autograd.grad(out, leaves, g, retain_graph=True)
    again = torch.autograd.grad(out, leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, leaves, g)
    only = qk_norm_rope(leaves[0], k, w, leaves[3])
    assert all(o.requires_grad for o in only)
    dq, dkw = torch.autograd.grad(only, (leaves[0], leaves[3]), g)
    assert torch.equal(dq, first[0]) and torch.equal(dkw, first[3])
    seen = []
    leaves[0].register_hook(seen.append)
    for _ in range(2):
        o = qk_norm_rope(leaves[0] * 1.0, *leaves[1:])
        torch.autograd.backward(o, g)
    assert torch.equal(seen[0], first[0]) and torch.equal(leaves[0].grad, first[0] * 2)
    assert torch.equal(leaves[2].grad, first[2] * 2)
    x = q * 1.0
    x.requires_grad_(True)
    y = x * 1.0
    o = qk_norm_rope(y, k, w, w)
    y.mul_(2.0)
    with pytest.raises(RuntimeError):
        o[0].sum().backward()
    o = qk_norm_rope(x, k, w, w)[0]
    o.mul_(2.0)  # the results may be changed
    o.sum().backward()
    assert torch.equal(x.grad, 2.0 * torch.autograd.grad(qk_norm_rope(x, k, w, w)[0].sum(), x)[0])


def test_attention_many_rows_long_split_and_stale():
    """Units split over CTAs, several row tiles a pool head; stale rows of NaN codes; scales of
    many sizes and signs."""
    rs = np.random.RandomState(32)
    case = _attn_case(rs, [6000, 130], 8, 2, 128, 16, torch.bfloat16, "e4m3", Sq=150)
    _check_attn(_attend(*case), *case)
    q, pools, scales, bt, ctx = _attn_case(rs, [333, 700], 4, 1, 64, 48, torch.float16, "e4m3", Sq=80)
    used = np.zeros(pools[0].shape[:2], dtype=bool)
    for b, n in enumerate(ctx):
        t = np.arange(n)
        used[bt[b, t // 48], t % 48] = True
    stale = torch.from_numpy(~used).cuda()
    for p in pools:
        p.view(torch.uint8)[stale] = 0x7F
    free = torch.from_numpy(~used.any(1)).cuda()
    for s in scales:
        s[free] = float("nan")
    scales[1] *= torch.from_numpy(2.0 ** rs.randint(-20, 20, scales[1].shape)).float().cuda()
    scales[1][bt[0, 2]] = 0.0
    scales[0][bt[0, 3]] = 0.0
    scales[0][bt[1, 1]] *= -1.0
    out = _attend(q, pools, scales, bt, ctx)
    clean = [torch.where(stale[..., None, None], torch.zeros_like(p.view(torch.uint8)), p.view(torch.uint8))
             .view(p.dtype) for p in pools]
    csc = [torch.where(free[:, None], torch.ones_like(s), s) for s in scales]
    _check_attn(out, q, clean, csc, bt, ctx)


def test_attention_views_and_host_tensors():
    from mlx_primitives.cache import quantized_paged_attention
    rs = np.random.RandomState(15)
    q, pools, scales, bt, ctx = case = _attn_case(rs, [100, 37], 4, 2, 64, 16, torch.bfloat16, "e4m3", Sq=2)
    want = _attend(*case)
    both = torch.stack([p.view(torch.uint8) for p in pools], 1)  # K and V of a block side by side
    views = [both[:, i].view(torch.float8_e4m3fn) for i in range(2)]
    assert torch.equal(_attend(q, views, scales, bt, ctx), want)
    heads = [p.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(torch.float8_e4m3fn) for p in pools]
    assert torch.equal(_attend(q, heads, scales, bt, ctx), want)
    assert torch.equal(_attend(q.transpose(1, 2).contiguous().transpose(1, 2), pools, scales, bt, ctx), want)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape).copy_(q)
    assert torch.equal(_attend(odd, pools, scales, bt, ctx), want)
    wide = [s.repeat(1, 2)[:, :2] for s in scales]  # strided scales
    assert torch.equal(_attend(q, pools, wide, bt, ctx), want)
    out = quantized_paged_attention(q.cpu(), *(p.cpu() for p in pools), *(s.cpu() for s in scales),
                                    torch.from_numpy(bt).long(), torch.from_numpy(ctx).long())
    assert out.device.type == "cpu" and torch.equal(out, want.cpu())
    e = torch.empty(0, 1, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert _attend(e, pools, scales, bt[:0], ctx[:0]).shape == e.shape
    assert torch.all(_attend(q, pools, scales, bt[:, :0], ctx) == 0)


# ------------------------------------------------------------------ together
def _dequant(pool, scale):
    return _n(pool) * _n(scale)[:, None, :, None]


def test_decode_steps_append_then_attend():
    """Prompt, then tokens one by one: norm + rotate + append, attend; 16-bit and 8-bit caches
    side by side against attention over the oracle's own keys and values."""
    from mlx_primitives.cache import paged_append, paged_attention, quantized_paged_attention
    rs = np.random.RandomState(20)
    B, H, Hk, D, block, steps = 3, 8, 2, 64, 16, 5
    prompt = np.array([30, 7, 16])
    dt = torch.bfloat16
    total = prompt + steps
    bt, (kp, vp), _ = _pool_case(rs, total, block, Hk, D, dt, None)
    k8, v8 = (torch.zeros(kp.shape, device="cuda").to(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.zeros(kp.shape[0], Hk, device="cuda") for _ in range(2))
    cos, sin = _tables(bt.shape[1] * block, D // 2)
    qw, kw = (1 + 0.1 * _rand(rs, (D,), torch.float32) for _ in range(2))
    tbt = torch.from_numpy(bt).cuda()
    hist = np.zeros((B, total.max(), 2, Hk, D))
    ctx = np.zeros(B, dtype=np.int64)
    for step in range(steps + 1):
        n = prompt if step == 0 else np.ones(B, dtype=np.int64)
        S = int(n.max())
        q, k, v = (_rand(rs, (B, S, h, D), dt) for h in (H, Hk, Hk))
        kw_ = dict(new_lens=torch.from_numpy(n).cuda(), q=q, cos_cache=cos, sin_cache=sin, q_weight=qw, k_weight=kw)
        c = torch.from_numpy(ctx).cuda()
        qr = paged_append(k, v, kp, vp, tbt, c, **kw_)
        q8 = paged_append(k, v, k8, v8, tbt, c, k_scales=ks, v_scales=vs, **kw_)
        assert torch.equal(qr, q8)
        at = np.where(np.arange(S) < n[:, None], ctx[:, None] + np.arange(S), -1)
        k64 = C.norm_rope(_n(k), _n(kw), _n(cos), _n(sin), at)
        for b in range(B):
            hist[b, ctx[b]:ctx[b] + n[b], 0] = k64[b, :n[b]]
            hist[b, ctx[b]:ctx[b] + n[b], 1] = _n(v)[b, :n[b]]
        ctx = ctx + n
        c = torch.from_numpy(ctx).cuda()
        o8 = quantized_paged_attention(qr, k8, v8, ks, vs, tbt, c, query_lens=torch.from_numpy(n).cuda())
        # against the cache's own codes: the operator's tolerance
        _check_attn(o8, qr, (k8, v8), (ks, vs), bt, ctx, query_lens=n)
        # the codes against the true keys and values: within half a step of e4m3 (2^-4 relative
        # to 2^-6 of the scale at least)
        for b in range(B):
            t = np.arange(ctx[b])
            for i, (p8, s8) in enumerate(((k8, ks), (v8, vs))):
                got = _dequant(p8, s8)[bt[b, t // block], t % block]
                sc = _n(s8)[bt[b, t // block]][..., None]
                true = hist[b, :ctx[b], i]
                assert np.all(np.abs(got - true) <= 2.0 ** -4 * np.abs(true) * 1.001 + 2.0 ** -10 * sc)
        if step:
            o16 = paged_attention(qr, kp, vp, tbt, c, block_size=block)
            assert (o16.float() - o8.float()).abs().max() < 0.2  # both caches hold the same history


def test_calls_on_streams_and_in_graphs():
    """Work on side streams, captured and replayed with new lengths, two captured graphs and an
    eager call in turn; results equal the plain calls' bits."""
    from mlx_primitives.cache import paged_append, quantized_paged_attention
    rs = np.random.RandomState(21)
    q, pools, scales, bt, ctx = _attn_case(rs, [3000, 500, 64], 8, 2, 128, 16, torch.bfloat16, "e4m3")
    tbt, tctx = torch.from_numpy(bt).cuda(), torch.from_numpy(ctx).cuda()
    short = torch.tensor([1000, 33, 0], dtype=torch.int32, device="cuda")
    f = lambda c: quantized_paged_attention(q, *pools, *scales, tbt, c)
    want, want_short = f(tctx), f(short)
    live = tctx.clone()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs += [f(tctx) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = f(live)
        graphs.append((g, o))
    for c, w in ((tctx, want), (short, want_short), (tctx, want)):
        live.copy_(c)
        for g, _ in graphs:
            g.replay()
        eager = f(c)
        torch.cuda.synchronize()
        assert torch.equal(eager, w) and all(torch.equal(o, w) for _, o in graphs)
    # a captured decode step: append, then attend
    k = _rand(rs, (3, 1, 2, 128), torch.bfloat16)
    start = [p.clone() for p in pools] + [s.clone() for s in scales]
    live.copy_(tctx - 1)

    def step():
        paged_append(k, k, *pools, tbt, live, k_scales=scales[0], v_scales=scales[1])
        return quantized_paged_attention(q, *pools, *scales, tbt, live + 1)
    want = step()
    after = [t.clone() for t in (*pools, *scales)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for t, s in zip((*pools, *scales), start):
        t.copy_(s)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    for t, a in zip((*pools, *scales), after):
        assert torch.equal(t.view(torch.uint8), a.view(torch.uint8))


def test_norm_rope_backward_in_a_graph():
    """A training step captured whole; its leaves have no eager graph alive."""
    from mlx_primitives.kernels import qk_norm_rope
    q, k, qw, kw = _norm_case(2, 33, 4, 2, 64, torch.bfloat16)
    cos, sin = _tables(64, 32)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, qw, kw)]

    def step(a):
        return torch.autograd.grad(qk_norm_rope(*a, cos, sin), a, (gq, gk))
    want = step([t.clone().requires_grad_(True) for t in (q, k, qw, kw)])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(leaves)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        for t in leaves:
            t.mul_(0.5)
    want = step([t.detach().clone().requires_grad_(True) for t in leaves])
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_norm_rope_trains_through_attention():
    """norm + rotation + flash attention, backward through both, against differences of fp64."""
    import mlx_primitives as mp
    from mlx_primitives.kernels import qk_norm_rope
    q, k, qw, kw = (t.requires_grad_(True) for t in _norm_case(1, 40, 4, 4, 64, torch.float32))
    v = _rand(np.random.RandomState(2), k.shape, torch.float32)
    cos, sin = _tables(64, 32)
    gy = torch.randn_like(v)

    def ref(q, k, qw, kw):
        ys = []
        for x, w in ((q, qw), (k, kw)):
            x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
            c, s = (t[:40, None, :].double() for t in (cos, sin))
            a, b = x[..., :32], x[..., 32:]
            ys.append(torch.cat((a * c - b * s, a * s + b * c), -1))
        s = torch.einsum("bshd,bthd->bhst", *ys) / 8
        s = s.masked_fill(torch.ones(40, 40, device="cuda").triu(1).bool(), float("-inf"))
        return torch.einsum("bhst,bthd->bshd", s.softmax(-1), v.double())
    got = torch.autograd.grad(mp.flash_attention(*qk_norm_rope(q, k, qw, kw, cos, sin), v, causal=True),
                              (q, k, qw, kw), gy)
    d = [t.detach().double().requires_grad_(True) for t in (q, k, qw, kw)]
    want = torch.autograd.grad(ref(*d), d, gy.double())
    for a, b in zip(got, want):
        # fp32 throughout: the attention's own fp32 tolerance, 1e-4
        assert (a.double() - b).abs().max() <= 1e-4 * (1 + b.abs().max())
