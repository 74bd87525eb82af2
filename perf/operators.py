"""Measured cases of the cache operators: query/key norms with rotation, appending to a paged
cache, and attention over a paged cache held in 8 bits.

``run`` computes an operator's plain form (elementary torch operations in fp32, rounded once), or,
with ``own`` set, makes the calls a user makes of ``mlx_primitives``.  ``exact`` restates each
operator in fp64.

The operators (h = D / 2; cos/sin are rows of the position tables):

* ``norm_rope``: y = x / sqrt(mean(x^2) + eps) * w per head row of q and k, then the half-split
  rotation (y1 cos - y2 sin, y1 sin + y2 cos).  A negative position marks a padding row: zeros and
  no gradient.  With ``backward`` the gradients of q, k and both weights come too.
* ``append``: new token i of sequence b goes to position context_lens[b] + i, that is to row
  pos % block of pool block block_tables[b, pos // block]; keys (and q) are normed where weights
  are given and rotated on the way.  An 8-bit pool keeps one power-of-two scale a (block, head):
  the least 2^k >= 2^-126 with amax <= 448 * 2^k over the block's tokens; a block that already
  holds tokens keeps its scale or grows it, its old codes then rescaled.
* ``attend``: softmax(scale * q k^T) v over codes times scales; the queries of sequence b are its
  last positions.
"""

import functools
import math
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-6
ROPE_BASE = 10000.0
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn
QMAX = {"e4m3": 448.0, "int8": 127.0}


@functools.lru_cache(maxsize=None)
def _package():
    path = os.path.join(os.getcwd(), "mlx-primitives_b200")
    if path not in sys.path:
        sys.path.insert(1, path)
    import mlx_primitives.cache
    import mlx_primitives.kernels

    return mlx_primitives


# ---------------------------------------------------------------------------------- the cases
def _norm_rope(name, B, S, Hq, Hk, D, dtype, backward, padded=False):
    return dict(name=name, op="norm_rope", B=B, S=S, Hq=Hq, Hk=Hk, D=D, dtype=dtype,
                backward=backward, padded=padded)


def _append(name, B, S, Hq, Hk, D, dtype, cache, block, ctx, ragged, norm):
    return dict(name=name, op="append", B=B, S=S, Hq=Hq, Hk=Hk, D=D, dtype=dtype, cache=cache,
                block=block, ctx=ctx, ragged=ragged, norm=norm)


def _attend(name, B, S, Hq, Hk, D, dtype, cache, block, ctx, ragged, window=-1):
    return dict(name=name, op="attend", B=B, S=S, Hq=Hq, Hk=Hk, D=D, dtype=dtype, cache=cache,
                block=block, ctx=ctx, ragged=ragged, window=window)


def listed():
    return [
        # a decode step of 8 sequences: one token's heads each, where only latency counts
        _norm_rope("norm_rope_token", 8, 1, 32, 8, 128, "bf16", False),
        # a training step's forward and backward at the 16K sliding-window configuration's shape
        _norm_rope("norm_rope_train_16k", 2, 16384, 32, 32, 128, "bf16", True),
        # a small fp32 training step, odd length, right-padded batch
        _norm_rope("norm_rope_train_fp32", 2, 1021, 12, 12, 64, "fp32", True, padded=True),
        # decode appends of a large batch to a 16-bit cache
        _append("append_token_bf16", 64, 1, 32, 8, 128, "bf16", "same", 16, 1024, True, False),
        # decode appends of a small batch to an 8-bit cache, with query and key norms
        _append("append_token_e4m3", 8, 1, 32, 8, 128, "bf16", "e4m3", 16, 4096, True, True),
        # prompts of uneven length going into an 8-bit cache behind a cached prefix
        _append("append_prompt_e4m3", 8, 4096, 32, 8, 128, "bf16", "e4m3", 16, 100, True, True),
        # a chunk of prompt tokens into a 16-bit cache, odd sizes
        _append("append_chunk_fp16", 5, 333, 16, 4, 64, "fp16", "same", 24, 700, True, False),
        # decode of one short conversation
        _attend("attend_token_short", 1, 1, 32, 8, 128, "bf16", "e4m3", 16, 777, False),
        # decode of 8 sequences of 4096 cached tokens, a key/value head for each query head
        _attend("attend_token_4k", 8, 1, 32, 32, 128, "bf16", "e4m3", 16, 4096, False),
        # decode of a full batch of uneven conversations over an int8 cache
        _attend("attend_token_ragged", 48, 1, 16, 2, 64, "fp16", "int8", 32, 9000, True),
        # decode of four contexts of 128K tokens, grouped heads
        _attend("attend_token_128k", 4, 1, 32, 8, 128, "bf16", "e4m3", 64, 131072, False),
        # a chunk of prompt tokens against what is cached of its sequences
        _attend("attend_chunk", 4, 512, 32, 8, 128, "bf16", "e4m3", 16, 8192, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "attend"])
    D = rng.choice([64, 128])
    Hk = rng.choice([1, 2, 4, 5, 8, 12])
    Hq = Hk * rng.choice([1, 2, 4, 7, 8])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "norm_rope":
        B, S = _log(rng, 1, 8), _log(rng, 1, 16384)
        while B * S * (Hq + Hk) * D > 60_000_000:
            S = S // 2 + 1
        return _unnamed(_norm_rope("", B, S, Hq, Hk, rng.choice([D, 80, 96]), dtype,
                                   rng.random() < 0.7, rng.random() < 0.4))
    ragged = rng.random() < 0.7
    block = rng.choice([8, 16, 24, 32, 64])
    if op == "append":
        B, S, ctx = _log(rng, 1, 64), rng.choice([1, _log(rng, 1, 2048)]), _log(rng, 1, 4096)
        while B * S * (Hq + 2 * Hk) * D > 30_000_000:
            S = S // 2 + 1
        while B * ctx * Hk * D > 40_000_000:
            ctx = ctx // 2 + 1
        return _unnamed(_append("", B, S, Hq, Hk, D, dtype, rng.choice(["same", "e4m3"]), block,
                                ctx, ragged, rng.random() < 0.5))
    B, ctx = _log(rng, 1, 64), _log(rng, 1, 131072)
    S = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 16, 512)])
    while B * ctx * Hk * D > 120_000_000:
        B, ctx = (B // 2 + 1, ctx) if B > 2 else (B, ctx // 2 + 1)
    while B * ctx * Hq * S > 500_000_000:
        S = S // 2
    S = max(1, min(S, ctx))
    window = rng.choice([-1, -1, -1, _log(rng, 1, max(2, ctx))])
    return _unnamed(_attend("", B, S, Hq, Hk, D, dtype, rng.choice(["e4m3", "int8"]), block, ctx,
                            ragged, window))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def _spread(n, most, ragged, least=1):
    """n lengths in [least, most], a fixed spread (the golden ratio's multiples); the first is
    `most`."""
    if not ragged:
        return [most] * n
    return [most if i == 0 else least + int((most - least) * ((i * 0.6180339887498949) % 1.0))
            for i in range(n)]


def _lengths(case):
    """(cached tokens before, new tokens) of every sequence for append; (cached tokens, queries)
    for attend."""
    B, S, ctx, ragged = case["B"], case["S"], case["ctx"], case["ragged"]
    if case["op"] == "append":
        return _spread(B, ctx, ragged, 0), _spread(B, S, ragged and S > 1)
    return _spread(B, ctx, ragged, min(S, ctx)), [S] * B


def _key_range(case, n, pos):
    """Keys [lo, hi) that the query at position pos of a sequence of n tokens sees."""
    lo = 0 if case["window"] < 0 else max(0, pos - case["window"])
    return lo, min(n, pos + 1)


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    B, S, Hq, Hk, D = (case[k] for k in ("B", "S", "Hq", "Hk", "D"))
    if case["op"] == "norm_rope":
        n = B * S * (Hq + Hk) * D
        tables = S * D * 4
        if not case["backward"]:
            return {"bytes": 2 * n * es + tables, "flops": 8 * n}
        return {"bytes": 4 * n * es + tables, "flops": 26 * n}
    before, new = _lengths(case)
    if case["op"] == "append":
        t = sum(new)
        row = D * es
        kept = D * (1 if case["cache"] == "e4m3" else es)
        return {"bytes": t * (2 * Hq * row + 2 * Hk * row + 2 * Hk * kept + D * 4),
                "flops": t * (Hq + Hk) * D * (8 if case["norm"] else 4)}
    seen = keys = 0
    for n, s in zip(before, new):
        spans = [_key_range(case, n, n - s + i) for i in range(s)]
        seen += sum(hi - lo for lo, hi in spans)
        keys += max(hi for _, hi in spans) - min(lo for lo, _ in spans)
    blocks = sum(-(-n // case["block"]) for n in before)
    return {"bytes": 2 * keys * Hk * D + 2 * blocks * Hk * 4 + blocks * 4 + 2 * B * S * Hq * D * es,
            "flops": 4 * seen * Hq * D}


# ---------------------------------------------------------------------------------- the inputs
def _tables(n, D):
    half = D // 2
    freq = ROPE_BASE ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angle = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _least_scale(amax, qmax):
    """The least power of two s >= 2^-126 with amax <= qmax * s."""
    m, e = torch.frexp(amax)
    mq, eq = math.frexp(qmax)
    e = (e - eq + (m > mq).to(e.dtype)).clamp(min=-126)
    return torch.ldexp(torch.ones_like(amax), e)


def _pools(case, gen, num_blocks):
    """K and V pools of normal values: in the case's type, or as codes and scales."""
    shape = (num_blocks, case["block"], case["Hk"], case["D"])
    out = []
    for _ in range(2):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)
        if case["cache"] == "same":
            out.append((x.to(TYPES[case["dtype"]]), None))
            continue
        # values of different blocks and heads differ in size, as they do in a model
        x *= torch.exp2(2 * torch.rand((num_blocks, 1, case["Hk"], 1), generator=gen,
                                       device="cuda") - 1).half()
        s = _least_scale(x.abs().amax((1, 3)).float(), QMAX[case["cache"]])
        x /= s[:, None, :, None].half()
        codes = x.to(E4M3) if case["cache"] == "e4m3" else x.round_().to(torch.int8)
        out.append((codes, s))
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, S, Hq, Hk, D = (case[k] for k in ("B", "S", "Hq", "Hk", "D"))
    dt = TYPES[case["dtype"]]

    def normal(*shape, size=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * size).to(dt)

    def weight():
        return 1 + 0.1 * torch.randn(D, generator=gen, device="cuda")

    st = {"case": dict(case)}
    if case["op"] == "norm_rope":
        st["q"], st["k"] = normal(B, S, Hq, D), normal(B, S, Hk, D)
        st["q_weight"], st["k_weight"] = weight(), weight()
        st["cos"], st["sin"] = _tables(S, D)
        st["positions"] = None
        if case["padded"]:
            lens = torch.tensor(_spread(B, S, True), device="cuda")
            at = torch.arange(S, device="cuda").expand(B, S)
            st["positions"] = torch.where(at < lens[:, None], at, -1).to(torch.int32)
        if case["backward"]:
            st["gq"], st["gk"] = normal(B, S, Hq, D), normal(B, S, Hk, D)
            for n in ("q", "k", "q_weight", "k_weight"):
                st[n].requires_grad_(True)
        return st
    before, new = _lengths(case)
    total = [a + b for a, b in zip(before, new)] if case["op"] == "append" else before
    need = [-(-n // case["block"]) for n in total]
    mb = max(need)
    ids = np.random.RandomState(seed % (1 << 31)).permutation(sum(need) + 2)  # 3 spare blocks
    bt = np.full((B, mb), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = ids[at:at + n]
        at += n
    st["block_tables"] = torch.from_numpy(bt).cuda()
    st["context_lens"] = torch.tensor(before, dtype=torch.int32, device="cuda")
    (st["k_pool"], st["k_scales"]), (st["v_pool"], st["v_scales"]) = _pools(case, gen, sum(need) + 3)
    st["q"] = normal(B, S, Hq, D, size=2.0)
    if case["op"] == "attend":
        return st
    st["k"], st["v"] = normal(B, S, Hk, D), normal(B, S, Hk, D)
    st["new_lens"] = torch.tensor(new, dtype=torch.int32, device="cuda") if case["ragged"] else None
    st["cos"], st["sin"] = _tables(mb * case["block"], D)
    st["q_weight"], st["k_weight"] = (weight(), weight()) if case["norm"] else (None, None)
    return st


# ---------------------------------------------------------------------------------- one pass
def run(state):
    return {"norm_rope": _run_norm_rope, "append": _run_append, "attend": _run_attend}[
        state["case"]["op"]](state)


def _run_norm_rope(s):
    names = ("q_out", "k_out", "dq", "dk", "dq_weight", "dk_weight")
    if own:
        out = _package().kernels.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"],
                                              s["cos"], s["sin"], positions=s["positions"], eps=EPS)
        if s["case"]["backward"]:
            out = out + torch.autograd.grad(out, (s["q"], s["k"], s["q_weight"], s["k_weight"]),
                                            (s["gq"], s["gk"]))
        return dict(zip(names, out))
    with torch.no_grad():
        q, aq = _plain_norm_rope(s["q"], s["q_weight"], s["cos"], s["sin"], s["positions"])
        k, ak = _plain_norm_rope(s["k"], s["k_weight"], s["cos"], s["sin"], s["positions"])
        out = (q, k)
        if s["case"]["backward"]:
            dq, dqw = _plain_norm_rope_grad(s["gq"], s["q"], s["q_weight"], *aq)
            dk, dkw = _plain_norm_rope_grad(s["gk"], s["k"], s["k_weight"], *ak)
            out = (q, k, dq, dk, dqw, dkw)
        return dict(zip(names, out))


def _run_append(s):
    if own:
        q = _package().cache.paged_append(
            s["k"], s["v"], s["k_pool"], s["v_pool"], s["block_tables"], s["context_lens"],
            new_lens=s["new_lens"], q=s["q"], cos_cache=s["cos"], sin_cache=s["sin"],
            q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS, k_scales=s["k_scales"],
            v_scales=s["v_scales"])
    else:
        q = _plain_append(s)
    # e4m3 pools are floating tensors: their values, beside the scales that multiply them
    return {"q_out": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"], "k_scales": s["k_scales"],
            "v_scales": s["v_scales"]}


def _run_attend(s):
    if own:
        w = s["case"]["window"]
        return _package().cache.quantized_paged_attention(
            s["q"], s["k_pool"], s["v_pool"], s["k_scales"], s["v_scales"], s["block_tables"],
            s["context_lens"], window_size=None if w < 0 else w)
    return _plain_attend(s)


# ---------------------------------------------------------------------------------- plain forms
def _plain_norm_rope(x, w, cos, sin, positions, norm=True):
    """The result in x's type, and what the gradient reuses."""
    x32, half, seen, r = x.float(), x.shape[-1] // 2, None, None
    if positions is None:
        c, s = cos[:x.shape[1], None, :], sin[:x.shape[1], None, :]
    else:
        at = positions.clamp(0, cos.shape[0] - 1).long()
        c, s, seen = cos[at][:, :, None, :], sin[at][:, :, None, :], (positions >= 0)[:, :, None, None]
    if norm:
        r = torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + EPS)
        x32 = x32 * r * w.float()
    y1, y2 = x32[..., :half], x32[..., half:]
    y = torch.cat((y1 * c - y2 * s, y1 * s + y2 * c), -1)
    if seen is not None:
        y = torch.where(seen, y, 0.0)
    return y.to(x.dtype), (r, c, s, seen)


def _plain_norm_rope_grad(gy, x, w, r, c, s, seen):
    g, x32, half = gy.float(), x.float(), x.shape[-1] // 2
    if seen is not None:
        g = torch.where(seen, g, 0.0)
    g1, g2 = g[..., :half], g[..., half:]
    g = torch.cat((g1 * c + g2 * s, g2 * c - g1 * s), -1)
    xhat = x32 * r
    dw = (g * xhat).sum((0, 1, 2))
    g = g * w.float()
    dx = r * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    return dx.to(x.dtype), dw.to(w.dtype)


def _plain_append(s):
    case, ctx = s["case"], s["context_lens"].long()
    B, S, block, bt = case["B"], case["S"], case["block"], s["block_tables"].long()
    pos = ctx[:, None] + torch.arange(S, device="cuda")
    new = s["new_lens"].long() if s["new_lens"] is not None else torch.full_like(ctx, S)
    valid = torch.arange(S, device="cuda") < new[:, None]
    at = torch.where(valid, pos, -1)
    q, _ = _plain_norm_rope(s["q"], s["q_weight"], s["cos"], s["sin"], at, case["norm"])
    spare = s["k_pool"].shape[0] - 1  # a block that no table names: written with what it holds
    if case["cache"] == "same":
        k, _ = _plain_norm_rope(s["k"], s["k_weight"], s["cos"], s["sin"], at, case["norm"])
        slot = pos.clamp(max=bt.shape[1] * block - 1)
        row = torch.where(valid, bt.gather(1, slot // block) * block + slot % block, spare * block)
        for pool, x in ((s["k_pool"], k), (s["v_pool"], s["v"])):
            flat = pool.view(-1, *pool.shape[2:])
            flat[row] = torch.where(valid[..., None, None], x, flat[row])
        return q
    k, _ = _plain_norm_rope(s["k"].float(), s["k_weight"], s["cos"], s["sin"], at, case["norm"])
    # every block that may receive tokens, (B, blocks, block) positions
    first = ctx // block
    nb = (S + block - 2) // block + 1
    slot = first[:, None] + torch.arange(nb, device="cuda")
    p = slot[:, :, None] * block + torch.arange(block, device="cuda")
    is_new = (p >= ctx[:, None, None]) & (p < (ctx + new)[:, None, None])
    is_old = p < ctx[:, None, None]
    touched = is_new.any(-1)
    ids = torch.where(touched, bt.gather(1, slot.clamp(max=bt.shape[1] - 1)), spare)
    src = (p - ctx[:, None, None]).clamp(0, S - 1).view(B, -1)
    for pool, scales, x in ((s["k_pool"], s["k_scales"], k), (s["v_pool"], s["v_scales"], s["v"].float())):
        x = x[torch.arange(B, device="cuda")[:, None], src].view(B, nb, block, *x.shape[2:])
        amax = torch.where(is_new[..., None, None], x.abs(), 0.0).amax((2, 4))
        old_scale = scales[ids]
        least = _least_scale(amax, QMAX["e4m3"])
        scale = torch.where(is_old[:, :, :1], torch.maximum(old_scale, least), least)
        scale = torch.where(touched[:, :, None], scale, old_scale)
        held = pool.view(torch.uint8)[ids]
        old = held.view(E4M3).float() * (old_scale / scale)[:, :, None, :, None]
        fresh = (x / scale[:, :, None, :, None]).clamp(-448.0, 448.0)
        value = torch.where(is_new[..., None, None], fresh, old).to(E4M3).view(torch.uint8)
        value = torch.where((is_new | is_old)[..., None, None] & touched[:, :, None, None, None], value, held)
        pool.view(torch.uint8)[ids] = value
        scales[ids] = scale
    return q


def _plain_attend(s):
    case, ctx = s["case"], s["context_lens"].long()
    B, S, Hq, Hk, D = (case[k] for k in ("B", "S", "Hq", "Hk", "D"))
    ids = s["block_tables"].clamp(min=0).long()

    def values(pool, scales):
        codes = pool.view(torch.uint8)[ids].view(pool.dtype).float()
        codes *= scales[ids][:, :, None, :, None]
        return codes.view(B, -1, Hk, D).transpose(1, 2)  # (B, Hk, T, D)

    k = values(s["k_pool"], s["k_scales"])
    T = k.shape[2]
    q = s["q"].float().view(B, S, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    scores = (q @ k.transpose(-1, -2)).view(B, Hk, Hq // Hk, S, T) * (1.0 / math.sqrt(D))
    del k
    t = torch.arange(T, device="cuda")
    pos = (ctx[:, None] - S + torch.arange(S, device="cuda"))[:, :, None]
    seen = t <= pos
    if case["window"] >= 0:
        seen &= pos - t <= case["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    del scores
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, Hk, -1, T) @ values(s["v_pool"], s["v_scales"])).view(B, Hk, -1, S, D) / total
    return o.permute(0, 3, 1, 2, 4).reshape(B, S, Hq, D).to(s["q"].dtype)


# ---------------------------------------------------------------------------------- fp64
def exact(case, seed):
    return {"norm_rope": _exact_norm_rope, "append": _exact_append, "attend": _exact_attend}[
        case["op"]](prepare(case, seed))


def _exact_rows(x, w, cos, sin, at):
    """Normed (with w) and rotated rows as complex numbers' products; x (..., H, D), at (...)."""
    if w is not None:
        x = x * (x.square().mean(-1, keepdim=True) + EPS).pow(-0.5) * w
    turn = torch.complex(cos.double(), sin.double())[at.clamp(min=0)].unsqueeze(-2)
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * turn
    y = torch.cat((z.real, z.imag), -1)
    return y * (at >= 0)[..., None, None]


def _exact_norm_rope(s):
    B, S = s["case"]["B"], s["case"]["S"]
    at = torch.arange(S, device="cuda").expand(B, S) if s["positions"] is None else s["positions"].long()
    grad = s["case"]["backward"]
    leaf = [s[n].detach().double().requires_grad_(grad) for n in ("q", "k", "q_weight", "k_weight")]
    q = _exact_rows(leaf[0], leaf[2], s["cos"], s["sin"], at)
    k = _exact_rows(leaf[1], leaf[3], s["cos"], s["sin"], at)
    out = {"q_out": q.detach(), "k_out": k.detach()}
    if grad:
        got = torch.autograd.grad((q, k), leaf, (s["gq"].double(), s["gk"].double()))
        out.update(zip(("dq", "dk", "dq_weight", "dk_weight"), got))
    return out


def _round_e4m3(x):
    """Nearest e4m3 value, ties to even, of |x| <= 448 in fp64."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return (x / step).round() * step


def _exact_append(s):
    case = s["case"]
    block, S, Hk, D = case["block"], case["S"], case["Hk"], case["D"]
    before, new = _lengths(case)
    table = s["block_tables"].cpu().numpy()
    at = -np.ones((case["B"], S), dtype=np.int64)
    rows = []  # (sequence, token, pool block, row in the block)
    for b, (c, n) in enumerate(zip(before, new)):
        pos = c + np.arange(n)
        at[b, :n] = pos
        rows.append(np.stack((np.full(n, b), np.arange(n), table[b, pos // block], pos % block)))
    rows = torch.from_numpy(np.concatenate(rows, 1)).cuda()
    at = torch.from_numpy(at).cuda()
    weights = [None if s[n] is None else s[n].double() for n in ("q_weight", "k_weight")]
    out = {"q_out": _exact_rows(s["q"].double(), weights[0], s["cos"], s["sin"], at)}
    k = _exact_rows(s["k"].double(), weights[1], s["cos"], s["sin"], at)
    for name, x in (("k", k), ("v", s["v"].double())):
        x = x[rows[0], rows[1]]
        pool = s[name + "_pool"].double()
        out[name + "_scales"] = None
        if case["cache"] == "e4m3":
            scales = s[name + "_scales"].double()
            nblk = pool.shape[0]
            amax = torch.zeros(nblk, Hk, dtype=torch.float64, device="cuda")
            amax.index_reduce_(0, rows[2], x.abs().amax(-1), "amax")
            least = torch.exp2((amax / 448).log2().ceil().clamp(min=-126))
            opens = torch.zeros(nblk, dtype=torch.bool, device="cuda")
            opens[rows[2][rows[3] == 0]] = True
            hit = torch.zeros(nblk, dtype=torch.bool, device="cuda")
            hit[rows[2]] = True
            grown = torch.where(opens[:, None], least, torch.maximum(scales, least))
            scale = torch.where(hit[:, None], grown, scales)
            # rows of a continued block below its first new token are rescaled
            first = torch.full((nblk,), block, device="cuda", dtype=torch.int64)
            first.index_reduce_(0, rows[2], rows[3], "amin")
            below = torch.arange(block, device="cuda") < torch.where(hit, first, 0)[:, None]
            moved = _round_e4m3(pool * (scales / scale)[:, None, :, None])
            pool = torch.where(below[:, :, None, None], moved, pool)
            x = _round_e4m3((x / scale[rows[2]][..., None]).clamp(-448, 448))
            out[name + "_scales"] = scale
        pool[rows[2], rows[3]] = x
        out[name + "_pool"] = pool
    return out


def _exact_attend(s):
    case = s["case"]
    S, Hq, Hk, D = (case[k] for k in ("S", "Hq", "Hk", "D"))
    o = torch.zeros(case["B"], S, Hq, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)[0]):
        ids = s["block_tables"][b, :-(-n // case["block"])].long()
        seen = torch.zeros(S, n, dtype=torch.bool, device="cuda")
        for i in range(S):
            lo, hi = _key_range(case, n, n - S + i)
            seen[i, lo:hi] = True
        for h in range(Hk):
            k, v = (((s[p + "_pool"].view(torch.uint8)[ids, :, h].view(s[p + "_pool"].dtype).double()
                      * s[p + "_scales"][ids, h].double()[:, None, None]).reshape(-1, D)[:n])
                    for p in ("k", "v"))
            g = slice(h * (Hq // Hk), (h + 1) * (Hq // Hk))
            q = s["q"][b, :, g].double()
            a = torch.einsum("sgd,td->sgt", q, k) / math.sqrt(D)
            a = a.masked_fill(~seen[:, None, :], -math.inf)
            o[b, :, g] = torch.einsum("sgt,td->sgd", torch.softmax(a, -1), v)
    return o
