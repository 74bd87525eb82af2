"""The cache operators where they can go wrong beside tests/test_gpu_cache_ops.py: the limits of
their scales, masks and sizes, autograd's other modes, and the ways a call can take to the kernels.
Tolerances are those of that file, which derives them."""

import ctypes
import math
import subprocess
import threading
import time

import numpy as np
import pytest
import torch

from oracle import cache_oracle as C
from test_gpu_cache_ops import (TYPES, _amp, _attend, _attn_case, _check_append, _check_attn, _check_norm,
                                _close, _n, _norm_case, _pool_case, _rand, _tables)

pytestmark = pytest.mark.gpu


def _check_gradients(leaves, out, pos, cos, sin, eps, seed):
    """Gradients of q, k and both weights against the oracle's, tolerances as in
    test_norm_rope_gradients."""
    q, k, qw, kw = leaves
    rs = np.random.RandomState(seed)
    gq, gk = _rand(rs, q.shape, q.dtype), _rand(rs, k.shape, k.dtype)
    got = torch.autograd.grad(out, leaves, (gq, gk))
    for x, w, g, dx, dw in ((q, qw, gq, got[0], got[2]), (k, kw, gk, got[1], got[3])):
        want, wsum, wabs = C.norm_rope_grad(_n(g), _n(x), _n(w), _n(cos), _n(sin), pos, eps)
        size = np.abs(_n(g)).max(-1, keepdims=True) * 3 / np.sqrt(
            np.where((pos >= 0)[:, :, None, None], (np.nan_to_num(_n(x)) ** 2).mean(-1, keepdims=True), 1) + eps)
        _close(dx, want, x.dtype, 2.0 ** -19 * size)
        chain = x.shape[0] * x.shape[1] * x.shape[2] / 8 + 64
        assert np.all(np.abs(_n(dw) - wsum) <= 2.0 ** -24 * chain * wabs + 2.0 ** -20 * wabs)


@pytest.mark.parametrize("eps", [0.0, 1e-50])  # the second is 0 in fp32
@pytest.mark.parametrize("dtype,Hq,Hk,D", [("bf16", 1, 2, 128), ("bf16", 12, 5, 128), ("fp32", 4, 9, 64),
                                           ("fp16", 8, 3, 80), ("bf16", 3, 1, 6)])
def test_norm_rope_gradients_without_eps(eps, dtype, Hq, Hk, D):
    """Heads that leave part of a warp's rows empty: those must not reach the weights' sums."""
    from mlx_primitives.kernels import qk_norm_rope
    leaves = [t.requires_grad_(True) for t in _norm_case(2, 21, Hq, Hk, D, TYPES[dtype], seed=Hq)]
    cos, sin = _tables(32, D // 2)
    pos = np.tile(np.arange(21), (2, 1))
    pos[1, 13:] = -1
    out = qk_norm_rope(*leaves, cos, sin, positions=torch.from_numpy(pos).int().cuda(), eps=eps)
    _check_norm(*leaves, cos, sin, pos, out, 0.0)
    _check_gradients(leaves, out, pos, cos, sin, 0.0, 5)


@pytest.mark.parametrize("Sq", [1, 5, 70, 300])
@pytest.mark.parametrize("block", [16, 48, 8, 20])
@pytest.mark.parametrize("window,causal", [(0, True), (5, True), (37, True), (150, False)])
def test_attention_never_reads_before_the_window(Sq, block, window, causal):
    """What lies before the first key that any query sees may hold anything: NaN codes in K and V,
    and scales of NaN where a block holds nothing else."""
    rs = np.random.RandomState(Sq + block)
    q, pools, scales, bt, ctx = _attn_case(rs, [1000, 333, Sq + window + 3, 700], 4, 2, 64, block, torch.bfloat16,
                                           "e4m3", Sq=Sq)
    stale = np.zeros(pools[0].shape[:2], dtype=bool)
    for b, n in enumerate(ctx):
        t = np.arange(max(0, n - Sq - window))
        stale[bt[b, t // block], t % block] = True
    stale = torch.from_numpy(stale).cuda()
    clean = [torch.where(stale[..., None, None], torch.zeros_like(p.view(torch.uint8)), p.view(torch.uint8))
             .view(p.dtype) for p in pools]
    csc = [s.clone() for s in scales]
    for p, s in zip(pools, scales):
        p.view(torch.uint8)[stale] = 0x7F
        s[stale.all(1)] = float("nan")
    kw = dict(window_size=window, causal=causal)
    out = _attend(q, pools, scales, bt, ctx, **kw)
    assert torch.isfinite(out).all()
    _check_attn(out, q, clean, csc, bt, ctx, **kw)


@pytest.mark.parametrize("Sq", [1, 3, 70])
@pytest.mark.parametrize("zeros", [2.0 ** -126, 0.0])
def test_attention_blocks_of_zero_values_count(Sq, zeros):
    """Blocks whose values are all zero, as paged_append writes them (scale 2^-126), weigh in the
    softmax like any other, before and behind the others, in one CTA and in many."""
    for blocks, dtype in ((65, torch.bfloat16), (65, torch.float32), (1300, torch.float16)):
        for last in (True, False):
            bt = np.arange(blocks, dtype=np.int32)[None]
            big = blocks - 1 if last else 0
            shape = (blocks, 16, 1, 64)
            k, v = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
            k[..., 0] = -8.0  # scores of 2^-8 in the softmax's base below
            k[big] = 0.0
            v[big] = 1.0
            pools = [t.to(torch.float8_e4m3fn) for t in (k, v)]
            size = 2.0 ** 10 if dtype is torch.float16 else 2.0 ** 20
            scales = [torch.ones(blocks, 1, device="cuda"), torch.full((blocks, 1), zeros, device="cuda")]
            scales[1][big] = size
            q = torch.zeros(1, Sq, 1, 64, dtype=dtype, device="cuda")
            q[..., 0] = 1.0
            out = _attend(q, pools, scales, bt, np.array([16 * blocks], dtype=np.int32), scale=math.log(2.0),
                          causal=False)
            want = np.full(q.shape, size * 16 / (16 + 16 * (blocks - 1) * 2.0 ** -8))
            # two different weights a row and one value: the weights' fp16 rounding, and the sums
            _close(out, want, dtype, (2.0 ** -15 if dtype is torch.float32 else 2.0 ** -11 + 2.0 ** -14) * want)
    scales[1].zero_()
    pools[1].view(torch.uint8).fill_(0x38)
    assert torch.all(_attend(q.bfloat16(), pools, scales, bt, np.array([16 * blocks], dtype=np.int32)) == 0)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("Sq", [1, 5, 70])
def test_attention_value_scales_at_their_limits(dtype, Sq):
    """Scales of values 2^80 apart, block by block and in stretches longer than a CTA's."""
    rs = np.random.RandomState(41)
    case = _attn_case(rs, [2000, 130, 9000], 4, 2, 64, 16, TYPES[dtype], "e4m3", Sq=Sq, qsize=0.5)
    q, pools, scales, bt, ctx = case
    for stretch in (1, 9, 200):
        small = (np.arange(scales[1].shape[0]) // stretch % 2).astype(bool)
        order = np.concatenate([bt[b, :-(-n // 16)] for b, n in enumerate(ctx)])
        for lo, hi in ((2.0 ** -60, 2.0 ** 20), (2.0 ** 20, 2.0 ** 100)):
            vs = np.ones(scales[1].shape[0])
            vs[order] = np.where(small[:order.size], lo, hi)
            scales[1].copy_(torch.from_numpy(vs)[:, None])
            _check_attn(_attend(*case), *case)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("Sq", [1, 3, 70])
def test_attention_queries_near_the_largest_value(dtype, Sq):
    rs = np.random.RandomState(42)
    case = _attn_case(rs, [300, 90], 4, 2, 64, 16, TYPES[dtype], "e4m3", Sq=Sq)
    q, pools, scales, bt, ctx = case
    q.copy_(q.clamp(-4, 4) / 4 * 3e38)
    q[..., 0] = 2.0 ** 127
    scales[0].mul_(2.0 ** -90)  # scores of a few, once multiplied by 2^-36
    _check_attn(_attend(*case, scale=2.0 ** -36), *case, scale=2.0 ** -36)


def test_tangents_are_refused():
    """Forward-mode derivatives are refused by the calls that take the short way, too."""
    import torch.autograd.forward_ad as fwd

    from mlx_primitives.cache import paged_append, quantized_paged_attention
    from mlx_primitives.kernels import qk_norm_rope
    rs = np.random.RandomState(43)
    q, k, qw, kw = _norm_case(2, 7, 4, 2, 64, torch.float32)
    qa, pools, scales, bt, ctx = _attn_case(rs, [100, 37], 4, 2, 64, 16, torch.float32, "e4m3")
    bt, ctx = torch.from_numpy(bt).cuda(), torch.from_numpy(ctx).cuda()
    cos, sin = _tables(16, 32)
    before = [t.view(torch.uint8).clone() for t in pools]
    with fwd.dual_level():
        for grad in (False, True):
            dual = lambda t: fwd.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))
            for args in ((dual(q), k, qw, kw, cos, sin), (q, dual(k), qw, kw, cos, sin), (q, k, dual(qw), kw),
                         (q, k, qw, kw, dual(cos), sin)):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    qk_norm_rope(*args)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                quantized_paged_attention(dual(qa), *pools, *scales, bt, ctx)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                quantized_paged_attention(qa, *pools, dual(scales[0]), scales[1], bt, ctx)
            for which in range(2):
                kv = [k[:, :1], k[:, 1:2]]
                kv[which] = dual(kv[which])
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    paged_append(*kv, *pools, bt, ctx, k_scales=scales[0], v_scales=scales[1])
        assert qk_norm_rope(q, k, qw, kw)[0].shape == q.shape  # without tangents: as ever
    for a, b in zip(pools, before):
        assert torch.equal(a.view(torch.uint8), b)


def test_running_out_of_memory_keeps_its_type():
    """The allocator's own exception, which callers catch to go on with less, by the short way as by
    the long one."""
    from mlx_primitives.cache import paged_append, quantized_paged_attention
    from mlx_primitives.kernels import qk_norm_rope
    w = torch.ones(64, device="cuda")
    wide = torch.ones(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda").expand(1 << 20, 1, 32, 64)  # 4 GB once dense
    pool = torch.zeros(2, 16, 32, 64, dtype=torch.bfloat16, device="cuda")
    p8, sc = pool.to(torch.float8_e4m3fn), torch.ones(2, 32, device="cuda")
    bt = torch.zeros(1 << 20, 1, dtype=torch.int32, device="cuda")
    none = torch.zeros(1 << 20, dtype=torch.int32, device="cuda")
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(0.01)
    try:
        for f in (lambda: qk_norm_rope(wide, wide, w, w),
                  lambda: paged_append(wide, wide, pool, pool.clone(), bt, none, new_lens=none, q=wide),
                  lambda: quantized_paged_attention(wide, p8, p8.clone(), sc, sc, bt, none)):
            with pytest.raises(torch.OutOfMemoryError):
                f()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)


def test_launches_let_other_threads_run(tmp_path):
    """While a call sits in the library (a full launch queue), other Python threads go on.  The
    library's functions are replaced by one that sleeps and returns a status."""
    from mlx_primitives import _lib
    from mlx_primitives.cache import paged_append, quantized_paged_attention
    from mlx_primitives.kernels import qk_norm_rope
    src = tmp_path / "slow.c"
    src.write_text("#include <unistd.h>\nint slow(const void* a) { (void)a; usleep(400000); return 1; }\n")
    so = tmp_path / "slow.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(so), str(src)], check=True)
    address = lambda f: ctypes.cast(f, ctypes.c_void_p).value
    slow, L = address(ctypes.CDLL(str(so)).slow), _lib.lib()
    rs = np.random.RandomState(44)
    q, k, w, _ = _norm_case(2, 1, 4, 2, 64, torch.float32)
    qa, pools, scales, bt, ctx = _attn_case(rs, [100, 37], 4, 2, 64, 16, torch.float32, "e4m3")
    bt, ctx = torch.from_numpy(bt).cuda(), torch.from_numpy(ctx).cuda()
    host = _lib.calls()
    host.bind(slow, address(L.mlxp_qk_norm_rope_bwd), address(L.mlxp_qk_norm_rope_bwd_workspace_size), slow, slow,
              address(L.mlxp_quant_paged_attn_workspace_size))
    try:
        for f in (lambda: qk_norm_rope(q, k, w, w),
                  lambda: paged_append(k, k, *pools, bt, ctx, k_scales=scales[0], v_scales=scales[1]),
                  lambda: quantized_paged_attention(qa, *pools, *scales, bt, ctx)):
            failed = []

            def work():
                try:
                    f()
                except ValueError as e:  # status 1
                    failed.append(e)
            t = threading.Thread(target=work)
            t.start()
            turns = 0
            while t.is_alive():
                time.sleep(0.01)
                turns += 1
            t.join()
            assert failed and turns >= 10, turns
    finally:
        _lib._calls = None
        _lib.calls()
    assert qk_norm_rope(q, k, w, w)[0].shape == q.shape


@pytest.mark.parametrize("ints", [torch.int32, torch.int64])
@pytest.mark.parametrize("kind", [None, "e4m3"])
def test_append_marks_the_pools_as_changed(ints, kind):
    """Autograd sees that the pools (and scales) were written: a gradient that needs their old
    values is refused.  Inference tensors, which have no such mark, are written all the same."""
    from mlx_primitives.cache import paged_append
    rs = np.random.RandomState(45)
    bt, pools, scales = _pool_case(rs, [20, 30], 16, 2, 64, torch.float32, kind)
    k = _rand(rs, (2, 3, 2, 64), torch.float32)
    bt, ctx = torch.from_numpy(bt).cuda().to(ints), torch.tensor([5, 16], device="cuda").to(ints)

    def call(p, s):
        paged_append(k, k, *p, bt, ctx, k_scales=s[0], v_scales=s[1])
    for t in [*pools, *scales][:2 if kind is None else 4]:
        w = torch.ones_like(t, dtype=torch.float32).requires_grad_(True)
        read = t if t.dtype is torch.float32 else t.view(torch.uint8)
        y = (w * read).sum() if t.dtype is torch.float32 else None
        was = t._version
        call(pools, scales)
        assert t._version > was
        if y is not None:
            with pytest.raises(RuntimeError, match="inplace"):
                y.backward()
    with torch.inference_mode():
        frozen = [t.clone() for t in pools]
        fs = [None if s is None else s.clone() for s in scales]
    call(frozen, fs)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(frozen, pools))


def test_gradients_that_would_be_lost_are_refused():
    """Pools, scales and slopes that want gradients: no call drops them without a word."""
    from mlx_primitives.cache import paged_append, quantized_paged_attention
    rs = np.random.RandomState(46)
    q, pools, scales, bt, ctx = _attn_case(rs, [100, 37], 4, 2, 64, 16, torch.float32, "e4m3")
    bt, ctx = torch.from_numpy(bt).cuda(), torch.from_numpy(ctx).cuda()
    wants = lambda t: t.clone().requires_grad_(True)
    for args in ((*pools, wants(scales[0]), scales[1]), (*pools, scales[0], wants(scales[1]))):
        with pytest.raises(NotImplementedError, match="differentiable"):
            quantized_paged_attention(q, *args, bt, ctx)
        with torch.no_grad():
            assert torch.equal(quantized_paged_attention(q, *args, bt, ctx),
                               quantized_paged_attention(q, *pools, *scales, bt, ctx))
    with pytest.raises(NotImplementedError, match="differentiable"):
        quantized_paged_attention(q, *pools, *scales, bt, ctx, alibi_slopes=wants(torch.ones(4, device="cuda")))
    k = _rand(rs, (2, 1, 2, 64), torch.float32)
    pool = torch.zeros(pools[0].shape, device="cuda")
    with pytest.raises(NotImplementedError, match="differentiable"):
        paged_append(k, k, wants(pool), pool.clone(), bt, ctx)
    with pytest.raises(NotImplementedError, match="differentiable"):
        paged_append(k, k, pool, wants(pool), bt, ctx)
    with pytest.raises(NotImplementedError, match="differentiable"):
        paged_append(k, k, *pools, bt, ctx, k_scales=wants(scales[0]), v_scales=scales[1])
    assert not pool.any()


def test_block_tables_shared_by_expansion():
    """One table for all sequences, as a view without a row stride."""
    from mlx_primitives.cache import paged_append, quantized_paged_attention
    rs = np.random.RandomState(47)
    q, pools, scales, bt, ctx = _attn_case(rs, [300], 4, 2, 64, 16, torch.bfloat16, "e4m3")
    one = torch.from_numpy(bt).cuda()
    qs = _rand(rs, (3, 1, 4, 64), torch.bfloat16, 2.0)
    lens = torch.tensor([300, 17, 120], dtype=torch.int32, device="cuda")
    for t in (one, one.long()):
        got = quantized_paged_attention(qs, *pools, *scales, t.expand(3, -1), lens)
        assert torch.equal(got, quantized_paged_attention(qs, *pools, *scales, t.repeat(3, 1), lens))
    k = _rand(rs, (3, 2, 2, 64), torch.bfloat16)
    new = torch.tensor([2, 0, 0], dtype=torch.int32, device="cuda")  # one writer of the shared block
    both = [[t.clone() for t in (*pools, *scales)] for _ in range(2)]
    for t, table in zip(both, (one.expand(3, -1), one.repeat(3, 1))):
        paged_append(k, k, t[0], t[1], table, lens, new_lens=new, k_scales=t[2], v_scales=t[3])
    for a, b in zip(*both):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert not torch.equal(both[0][0].view(torch.uint8), pools[0].view(torch.uint8))


def test_integers_past_32_bits():
    """64-bit lengths, tables and positions are not cut: 2^32 + 1 is no block and no row."""
    from mlx_primitives.cache import paged_append, quantized_paged_attention
    from mlx_primitives.kernels import qk_norm_rope
    rs = np.random.RandomState(48)
    far = 1 << 32
    q, k, qw, kw = _norm_case(1, 4, 4, 2, 64, torch.bfloat16)
    cos, sin = _tables(8, 32)
    pos = np.array([[far + 1, 3, -far, far * 2 - 1]])
    out = qk_norm_rope(q, k, qw, kw, cos, sin, positions=torch.from_numpy(pos).cuda())
    _check_norm(q, k, qw, kw, cos, sin, pos, out)
    qa, pools, scales, bt, ctx = _attn_case(rs, [300, 90], 4, 2, 64, 16, torch.bfloat16, "e4m3")
    holes = bt.copy()
    holes[0, 3], holes[1, 0] = -1, -1
    far_bt = bt.astype(np.int64)
    far_bt[0, 3], far_bt[1, 0] = far + int(bt[0, 3]), -far + int(bt[1, 0])
    want = _attend(qa, pools, scales, holes, ctx)
    assert torch.equal(_attend(qa, pools, scales, far_bt, ctx), want)
    lens = np.array([far + 5, -far + 40])
    assert torch.equal(_attend(qa, pools, scales, bt, lens),
                       _attend(qa, pools, scales, bt, np.array([2 ** 31 - 1, 0], dtype=np.int32)))
    x = _rand(rs, (2, 1, 2, 64), torch.bfloat16)
    before = [t.view(torch.uint8).clone() for t in pools]
    paged_append(x, x, *pools, torch.from_numpy(bt).cuda(), torch.from_numpy(lens).cuda(), k_scales=scales[0],
                 v_scales=scales[1])
    paged_append(x, x, *pools, torch.from_numpy(far_bt).cuda(), torch.tensor([50, 2]).cuda(), k_scales=scales[0],
                 v_scales=scales[1])
    for a, b in zip(pools, before):
        assert torch.equal(a.view(torch.uint8), b)
    paged_append(x, x, *pools, torch.from_numpy(bt).cuda(), torch.tensor([5, 5]).cuda(),
                 new_lens=torch.tensor([far, -far]).cuda(), k_scales=scales[0], v_scales=scales[1])
    same = [torch.equal(p.view(torch.uint8)[bt[b, 0]], w[bt[b, 0]]) for p, w in zip(pools, before) for b in range(2)]
    assert same == [False, True, False, True]


def test_norm_rope_under_compiled_autograd():
    """The graph's node is one that a captured backward takes, as a call of its own."""
    from torch._dynamo import compiled_autograd

    from mlx_primitives.kernels import qk_norm_rope
    q, k, qw, kw = _norm_case(2, 9, 4, 2, 64, torch.float32)
    cos, sin = _tables(16, 32)
    pos = torch.tensor([[0, 1, 2, 3, 4, 5, 6, -1, -1], [3, 4, 5, 6, 7, 8, 9, 10, 11]], dtype=torch.int32, device="cuda")

    def grads(leaves, how, **kw_):
        leaves = [t.clone().requires_grad_(want) for t, want in leaves]
        out = qk_norm_rope(*leaves, **kw_)
        y = out[0].sin().sum() + (out[1] * 2).sum()
        with how():
            y.backward()
        return [t.grad for t in leaves]
    import contextlib
    for wants in ((True,) * 4, (True, False, False, True), (False, False, True, False)):
        for kw_ in (dict(cos_cache=cos, sin_cache=sin), dict(cos_cache=cos, sin_cache=sin, positions=pos),
                    dict(eps=1e-3), dict(cos_cache=cos, sin_cache=sin, offset=2, k_offset=5)):
            leaves = list(zip((q, k, qw, kw), wants))
            want = grads(leaves, contextlib.nullcontext, **kw_)
            got = grads(leaves, lambda: compiled_autograd._enable(lambda gm: gm), **kw_)
            for a, b in zip(got, want):
                assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


class _Spy:
    """The short calls, with a record of whether each was taken."""

    def __init__(self, real):
        self.real, self.taken = real, []

    def __getattr__(self, name):
        def call(*args):
            out = getattr(self.real, name)(*args)
            self.taken.append(out is not None)
            return out
        return call


@pytest.fixture
def spy(monkeypatch):
    from mlx_primitives import _lib
    s = _Spy(_lib.calls())
    monkeypatch.setattr(_lib, "calls", lambda: s)
    return s


@pytest.mark.parametrize("ints", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype,D,kind,block", [("bf16", 128, None, 16), ("fp16", 64, None, 24), ("fp32", 64, "int8", 128),
                                                ("bf16", 128, "e4m3", 16), ("bf16", 10, "int8", 5)])
def test_append_by_either_way(spy, ints, dtype, D, kind, block):
    """Everything that an append takes, by the short way (32-bit integers) and by the long one."""
    from mlx_primitives.cache import paged_append
    rs = np.random.RandomState(D + block)
    dt, Hk, Hq, S = TYPES[dtype], 3, 5, 19
    ctx = np.array([0, 1, 33, block, 4 * block - 1])
    new = np.array([S, S - 3, 0, S, 1])
    bt, pools, scales = _pool_case(rs, ctx + new, block, Hk, D, dt, kind)
    k, v = (_rand(rs, (5, S, Hk, D), dt, 2.0) for _ in range(2))
    fused = _rand(rs, (5, S, Hq + 2, D), dt, 2.0)
    v = v.transpose(1, 2).contiguous().transpose(1, 2)  # strides of their own for each of k, v, q
    q = fused[:, :, 1:Hq + 1]
    cos, sin = _tables(bt.shape[1] * block, D // 2)
    qw, kw = (1 + 0.1 * _rand(rs, (D,), torch.float32)).bfloat16(), 1 + 0.1 * _rand(rs, (D,), torch.float32)
    at = np.where(np.arange(S) < new[:, None], ctx[:, None] + np.arange(S), -1)
    before = [_n(t) if t is not None else None for t in (*pools, *scales)]
    qo = paged_append(k, v, *pools, torch.from_numpy(bt).cuda().to(ints), torch.from_numpy(ctx).cuda().to(ints),
                      new_lens=torch.from_numpy(new).cuda().to(ints), q=q, cos_cache=cos, sin_cache=sin, q_weight=qw,
                      k_weight=kw, eps=1e-3, k_scales=scales[0], v_scales=scales[1])
    assert spy.taken == [ints is torch.int32]
    k64 = C.norm_rope(_n(k), _n(kw), _n(cos), _n(sin), at, 1e-3)
    _check_append(k64, _n(v), True, before, pools, scales, bt, ctx, new, kind, dt)
    want = C.norm_rope(_n(q), _n(qw), _n(cos), _n(sin), at, 1e-3)
    _close(qo, want, dt, 2.0 ** -19 * _amp(want))


@pytest.mark.parametrize("ints", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp32", 64), ("fp16", 6)])
def test_norm_rope_by_either_way(spy, ints, dtype, D):
    """Positions (strided ones) with padding, and the gradients, by the short way and by the long."""
    from mlx_primitives.kernels import qk_norm_rope
    leaves = [t.requires_grad_(True) for t in _norm_case(3, 20, 5, 2, D, TYPES[dtype], seed=D)]
    cos, sin = _tables(40, D // 2)
    pos = np.random.RandomState(D).randint(0, 40, (3, 20))
    pos[0, 11:], pos[2, :4] = -1, -1
    wide = torch.zeros(20, 6, dtype=ints, device="cuda")
    wide[:, ::2] = torch.from_numpy(pos.T).cuda().to(ints)
    out = qk_norm_rope(*leaves, cos, sin, positions=wide[:, ::2].T, eps=1e-3)
    assert spy.taken == [ints is torch.int32]
    _check_norm(*leaves, cos, sin, pos, out, 1e-3)
    _check_gradients(leaves, out, pos, cos, sin, 1e-3, 6)
    out = qk_norm_rope(*[t.detach() for t in leaves], cos, sin, offset=7, k_offset=20)
    assert spy.taken[1]
    for x, w, y, off in ((leaves[0], leaves[2], out[0], 7), (leaves[1], leaves[3], out[1], 20)):
        want = C.norm_rope(_n(x), _n(w), _n(cos), _n(sin), np.tile(off + np.arange(20), (3, 1)))
        _close(y, want, x.dtype, 2.0 ** -20 * 2 * _amp(want))


@pytest.mark.parametrize("ints", [torch.int32, torch.int64])
@pytest.mark.parametrize("Sq", [1, 70])
def test_attention_by_either_way(spy, ints, Sq):
    from mlx_primitives.cache import quantized_paged_attention
    rs = np.random.RandomState(49)
    q, pools, scales, bt, ctx = _attn_case(rs, [Sq + 90, 300, 33], 4, 2, 64, 16, torch.bfloat16, "e4m3", Sq=Sq)
    q = q.transpose(1, 2).contiguous().transpose(1, 2)
    ql = np.array([Sq, 0, min(Sq, 33)], dtype=np.int32)
    t = lambda a: torch.from_numpy(a).cuda().to(ints)
    out = quantized_paged_attention(q, *pools, *scales, t(bt), t(ctx), 0.25, True, 80, t(ql))
    assert spy.taken == [ints is torch.int32]
    _check_attn(out, q, pools, scales, bt, ctx, scale=0.25, window_size=80, query_lens=ql)


def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("dtype,D,Hq,Hk", [("bf16", 64, 19, 9), ("fp32", 64, 19, 2), ("fp16", 10, 3, 1),
                                           ("bf16", 128, 33, 5)])
def test_norm_rope_with_tokens_for_every_warp(spy, dtype, D, Hq, Hk):
    """From 24 tokens an SM a warp takes all heads of a token, some rows at a time."""
    from mlx_primitives.kernels import qk_norm_rope
    B, S = 2, 13 * _sms() + 1
    leaves = [t.requires_grad_(True) for t in _norm_case(B, S, Hq, Hk, D, TYPES[dtype], seed=D)]
    cos, sin = _tables(S, D // 2)
    pos = np.tile(np.arange(S), (B, 1))
    pos[1, S // 2:] = -1
    with torch.no_grad():
        leaves[0][1, S // 2:] = float("nan")
    out = qk_norm_rope(*leaves, cos, sin, positions=torch.from_numpy(pos).int().cuda())
    assert spy.taken == [True]
    _check_norm(*leaves, cos, sin, pos, out)
    _check_gradients(leaves, out, pos, cos, sin, 1e-6, 7)


@pytest.mark.parametrize("kind", [None, "e4m3", "int8"])
def test_append_of_long_prompts(spy, kind):
    """From 64 query rows' units an SM the queries take a launch of their own beside an 8-bit pool;
    ragged prompts, some of them longer than others by orders."""
    from mlx_primitives.cache import paged_append
    rs = np.random.RandomState(50)
    B, S, Hq, Hk, D, block, dt = 3, 22 * _sms(), 19, 2, 64, 16, torch.bfloat16
    ctx, new = np.array([100, 0, 7]), np.array([S, 5, S - 1001])
    bt, pools, scales = _pool_case(rs, ctx + new, block, Hk, D, dt, kind)
    q, k, v = (_rand(rs, (B, S, h, D), dt, 2.0) for h in (Hq, Hk, Hk))
    cos, sin = _tables(bt.shape[1] * block, D // 2)
    qw, kw = (1 + 0.1 * _rand(rs, (D,), torch.float32) for _ in range(2))
    at = np.where(np.arange(S) < new[:, None], ctx[:, None] + np.arange(S), -1)
    before = [_n(t) if t is not None else None for t in (*pools, *scales)]
    ints = lambda a: torch.from_numpy(a).int().cuda()
    qo = paged_append(k, v, *pools, ints(bt), ints(ctx), new_lens=ints(new), q=q, cos_cache=cos, sin_cache=sin,
                      q_weight=qw, k_weight=kw, k_scales=scales[0], v_scales=scales[1])
    assert spy.taken == [True]
    k64 = C.norm_rope(_n(k), _n(kw), _n(cos), _n(sin), at)
    _check_append(k64, _n(v), True, before, pools, scales, bt, ctx, new, kind, dt)
    want = C.norm_rope(_n(q), _n(qw), _n(cos), _n(sin), at)
    _close(qo, want, dt, 2.0 ** -19 * _amp(want))


@pytest.mark.parametrize("block,kw", [(8, dict()), (24, dict()), (16, dict(alibi=True)), (48, dict(alibi=True)),
                                      (20, dict(window_size=60))])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attention_of_chunks_outside_the_many_row_kernel(block, kw, dtype):
    """64 rows a pool head and more with blocks that are not multiples of 16, ALiBi, or in fp32."""
    from mlx_primitives.cache import get_alibi_slopes
    rs = np.random.RandomState(51)
    case = _attn_case(rs, [300, 90, 1000], 8, 2, 64, block, TYPES[dtype], "e4m3", Sq=70)
    kw = {"alibi_slopes": get_alibi_slopes(8).numpy()} if kw.get("alibi") else kw
    _check_attn(_attend(*case, **kw), *case, **kw)


@pytest.mark.parametrize("block", [64, 24])
def test_attention_past_32_bits(block):
    """Blocks behind the first 2^31 elements of a pool, in each kernel."""
    rs = np.random.RandomState(52)
    Hk, D = 8, 128
    nblk = (1 << 31) // (block * Hk * D) + 40
    pools = [torch.zeros(nblk, block, Hk, D, dtype=torch.int8, device="cuda") for _ in range(2)]
    n = np.array([500, 77], dtype=np.int32)
    bt = (nblk - 1 - rs.permutation(2 * 21).reshape(2, 21)).astype(np.int32)
    near = nblk - 42  # the oracle's pools hold the last blocks alone
    scales = [torch.ones(nblk, Hk, device="cuda") for _ in range(2)]
    for p, s in zip(pools, scales):
        p[near:] = torch.randint(-127, 128, (42, block, Hk, D), device="cuda", dtype=torch.int8)
        s[near:] = 2.0 ** -6 * (1 + torch.rand(42, Hk, device="cuda"))
    for Sq in (1, 70):
        q = _rand(rs, (2, Sq, 8, D), torch.bfloat16)
        out = _attend(q, pools, scales, bt, n)
        _check_attn(out, q, [p[near:] for p in pools], [s[near:] for s in scales], bt - near, n)


@pytest.mark.parametrize("ints", [torch.int32, torch.int64])  # the node in C++, the one in Python
def test_norm_rope_with_hooks_on_saved_tensors(ints):
    """Hooks may move what is saved and give it back in another layout; what comes back on the host,
    in another type or shape is refused before the kernel sees its address."""
    from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

    from mlx_primitives.kernels import qk_norm_rope
    leaves = [t.requires_grad_(True) for t in _norm_case(2, 9, 4, 2, 64, torch.float32)]
    cos, sin = _tables(16, 32)
    pos = torch.arange(9, device="cuda").repeat(2, 1).to(ints)
    rs = np.random.RandomState(53)
    g = [_rand(rs, t.shape, torch.float32) for t in leaves[:2]]

    def run(hooks=None):
        if hooks is None:
            out = qk_norm_rope(*leaves, cos, sin, positions=pos)
        else:
            with hooks:
                out = qk_norm_rope(*leaves, cos, sin, positions=pos)
        return torch.autograd.grad(out, leaves, g)
    want = run()
    same = lambda t: t
    turned = lambda t: t.transpose(1, 3).contiguous().transpose(1, 3) if t.dim() == 4 else t
    for hooks in (save_on_cpu(), saved_tensors_hooks(turned, same), saved_tensors_hooks(same, turned)):
        assert all(torch.equal(a, b) for a, b in zip(run(hooks), want))
    for back in (lambda t: t.cpu(), lambda t: t.half(), lambda t: t[:1], lambda t: t.repeat_interleave(2, -1)[..., ::2],
                 lambda t: t if t.dim() == 4 else t.cpu(), lambda t: t if t.dim() != 2 else t.double()):
        with pytest.raises(RuntimeError, match="came back changed"):
            run(saved_tensors_hooks(same, back))
    with saved_tensors_hooks(same, lambda t: t.half()):
        out = qk_norm_rope(leaves[0], leaves[1], None, None, eps=1e-6 if ints is torch.int32 else 1)
    with pytest.raises(RuntimeError, match="came back changed"):
        torch.autograd.grad(out, leaves[:2], g)


@pytest.mark.parametrize("H,Hk,Sq,lens", [(64, 4, 17, 1000), (16, 8, 130, 300), (8, 1, 70, 3000), (8, 8, 129, 140)])
@pytest.mark.parametrize("dtype,kind,D", [("bf16", "e4m3", 64), ("fp16", "int8", 128)])
def test_attention_of_many_rows_whose_last_tile_is_alone(H, Hk, Sq, lens, dtype, kind, D):
    """The last 128 and fewer rows of a pool head leave a CTA's second tile without work; units with
    rows for both follow in the same CTA."""
    rs = np.random.RandomState(Sq)
    B = max(3, 20000 // (Sq * H))
    case = _attn_case(rs, [lens] + rs.randint(1, lens, B - 1).tolist(), H, Hk, D, 16, TYPES[dtype], kind, Sq=Sq)
    _check_attn(_attend(*case), *case)


@pytest.mark.parametrize("Sq", [1, 5])
@pytest.mark.parametrize("kw", [dict(), dict(alibi=True), dict(causal=False, alibi=True), dict(window_size=100)])
def test_attention_of_contexts_longer_than_their_tables(Sq, kw):
    """Tokens past the block table are not there; the queries' positions still count them."""
    from mlx_primitives.cache import get_alibi_slopes
    rs = np.random.RandomState(54)
    q, pools, scales, bt, _ = _attn_case(rs, [300, 90, 200, 31, 400], 8, 2, 64, 16, torch.bfloat16, "e4m3", Sq=Sq)
    cap = bt.shape[1] * 16
    ctx = np.array([300, cap, cap + 3, cap + 10 ** 6, 2 ** 31 - 1], dtype=np.int32)
    kw = dict(kw)
    if kw.pop("alibi", False):
        kw["alibi_slopes"] = get_alibi_slopes(8).numpy()
    case = (q, pools, scales, bt, ctx)
    _check_attn(_attend(*case, **kw), *case, **kw)
