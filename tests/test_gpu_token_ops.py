"""Token operators on the device against their formulas in 64 bits (tests/token_reference.py).

Tolerances.  A result that is rounded to type t is off by at most half a step of t (``half_step``), plus what fp32
arithmetic leaves: every fp32 operation is off by 2^-24 of its result, and a value that came through a chain of at most CHAIN
operations (products, the levels of a sum over a row, a reciprocal root) by CHAIN 2^-24 of the magnitudes that were added up.
CHAIN = 64: a row sum is 8 + 10 + 16 levels (lane, wave, workgroup), twice for LayerNorm, and there are fewer than 16 other
operations in any chain.  A sum over n rows adds n 2^-24 of its magnitudes (the worst order)."""

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from diffusionnag_amd import arch_functions as AF, ema as ema_lib, losses, run_lib, token_ops as ops, utils
from tests import token_reference as R
from tests.helpers import Cfg
from tests.token_reference import U32, half_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CHAIN = 64 * U32
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def dev(t):
    return None if t is None else t.to(DEV)


def within(got, want, slack, what):
    """|got - want| <= half a step of got's type at want, plus `slack` (absolute, a tensor)."""
    rel, least = half_step(got.dtype)
    got, want = got.detach().cpu().double(), want.double()
    off = (got - want).abs()
    tol = rel * want.abs() * (1 + 1e-12) + least + slack * (1 + rel)
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).max()):.3g} tolerances at {int((off / tol).argmax())}"


# ---------------------------------------------------------------------------------------------------------------
# embedding lookup
# ---------------------------------------------------------------------------------------------------------------
def some_ids(g, rows, V, hot=False):
    ids = torch.randint(0, V, (rows,), generator=g)
    if hot:
        ids[torch.rand(rows, generator=g) < 0.7] = V // 2
    bad = torch.rand(rows, generator=g) < 0.1
    ids[bad] = torch.tensor([-1, -100, V, V + 5, 2 ** 31 - 1])[torch.randint(0, 5, (int(bad.sum()),), generator=g)]
    return ids


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,d", [(1, 1, 1), (3, 7, 64), (5, 2, 7), (64, 100, 8), (65, 33, 65), (257, 1000, 513), (40, 20, 2050), (9, 5, 8192)])
def test_embed_tokens(dtype, rows, V, d):
    g = gen(rows + V + d)
    w, ids = rnd(g, V, d, dtype=dtype), some_ids(g, rows, V)
    scale = d ** 0.5
    want = R.embed(ids, w, scale)
    within(ops.embed_tokens(dev(ids), dev(w), scale=scale), want, 2 * U32 * want.abs(), "int64 ids")
    within(ops.embed_tokens(dev(ids.int()), dev(w), scale=scale), want, 2 * U32 * want.abs(), "int32 ids")
    wide = torch.full((V, d + 3), float("nan"), dtype=dtype)
    wide[:, 1:d + 1] = w                                # rows that start anywhere, NaN around them
    within(ops.embed_tokens(dev(ids).reshape(1, -1), dev(wide)[:, 1:d + 1], scale=scale)[0], want, 2 * U32 * want.abs(), "strided weight")
    within(ops.embed_tokens(dev(ids), dev(w.t().contiguous()).t(), scale=scale), want, 2 * U32 * want.abs(), "transposed weight")


GRAD_SHAPES = [(1, 1, 1), (1, 300, 5), (63, 7, 64), (4097, 7, 64), (300, 16, 65), (5000, 9, 24),            # few tokens
               (33, 17, 8), (100, 1000, 65), (3000, 50, 513), (8192, 300, 9), (8192, 40, 1030),             # sort in LDS
               (8193, 300, 16), (20000, 255, 8), (20000, 256, 8), (9000, 70000, 5), (140001, 65536, 1)]    # radix sort, 1 to 3 digits


@pytest.mark.parametrize("rows,V,d", GRAD_SHAPES)
@pytest.mark.parametrize("hot", [False, True])
def test_embed_tokens_grad(rows, V, d, hot):
    for dtype in DTYPES if rows < 3000 else [DTYPES[(rows + hot) % 3]]:
        g = gen(rows + V + d)
        grad, ids = rnd(g, rows, d, dtype=dtype), some_ids(g, rows, V, hot)
        pad = V // 2 if rows % 2 else None
        want, mag, n = R.embed_grad(ids, grad, V, 1.5, pad)
        got = ops.embed_tokens_grad(dev(grad), dev(ids), V, scale=1.5, padding_idx=pad)
        within(got, want, (n + 2) * U32 * mag, f"{dtype}")
        assert not got[dev((n == 0).squeeze(1))].any()
        again = ops.embed_tokens_grad(dev(grad), dev(ids.int()), V, scale=1.5, padding_idx=pad)
        assert torch.equal(got, again), "the same inputs gave other bits"


def test_embed_grad_strides_empty_and_all_dropped():
    g = gen(1)
    ids = some_ids(g, 60, 30).reshape(4, 15)
    wide = rnd(g, 4, 15, 20)
    want, mag, n = R.embed_grad(ids, wide[..., 3:16], 30, 1.0)
    within(ops.embed_tokens_grad(dev(wide)[..., 3:16], dev(ids), 30), want, (n + 2) * U32 * mag, "strided grad")
    one = rnd(g, 13)
    want, mag, n = R.embed_grad(ids, one.expand(4, 15, 13), 30, 1.0)
    within(ops.embed_tokens_grad(dev(one).expand(4, 15, 13), dev(ids), 30), want, (n + 2) * U32 * mag, "broadcast grad")
    for V in (7, 40, 70000):
        assert not ops.embed_tokens_grad(torch.zeros(0, 9, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV), V).any()
        for rows in (5, 9000):
            nothing = ops.embed_tokens_grad(torch.full((rows, 9), float("nan"), device=DEV), torch.full((rows,), -1, device=DEV), V)
            assert not nothing.any()
    assert ops.embed_tokens(torch.zeros(0, 3, dtype=torch.int64, device=DEV), torch.zeros(4, 5, device=DEV)).shape == (0, 3, 5)


# ---------------------------------------------------------------------------------------------------------------
# norms between blocks
# ---------------------------------------------------------------------------------------------------------------
NAMES = ("x", "y", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias")


def norm_inputs(g, rows, d, groups, xt, yt, wt, kind, has_y=True, pre=True, gate=True):
    t = dict(x=rnd(g, rows, d, dtype=xt, std=2.0), pre_weight=1 + rnd(g, d, std=0.2), pre_bias=rnd(g, d, std=0.2))
    t["pre_weight"], t["pre_bias"] = t["pre_weight"].to(wt), t["pre_bias"].to(wt)
    if has_y:
        t.update(y=rnd(g, rows, d, dtype=yt) + 0.5, post_weight=(1 + rnd(g, d, std=0.2)).to(wt), post_bias=rnd(g, d, std=0.2).to(wt))
        if gate:
            t["gate"] = rnd(g, groups, d, dtype=wt)
    if kind == "rms":
        t["post_bias"] = t["pre_bias"] = None
    if not pre:
        t["pre_weight"] = t["pre_bias"] = None
    return {n: t.get(n) for n in NAMES}


def norm_tolerances(t, kind, eps, rs, pre, cx, ch):
    """The fp32 part of every output's and gradient's tolerance, from magnitudes: M_y, M_x are bounds of what is added up for the
    normalised y and x_new, so a normalised value is off by CHAIN times its row's largest M r."""
    T = {n: None if v is None else v.double() for n, v in t.items()}
    top = lambda v: v.abs().amax(-1, keepdim=True)                                                  # noqa: E731
    avg = lambda v: v.abs().mean(-1, keepdim=True)                                                   # noqa: E731
    one = torch.ones(T["x"].shape[-1]).double()
    pw, qw = (T["post_weight"] if T["post_weight"] is not None else one), (T["pre_weight"] if T["pre_weight"] is not None else one)
    pb, qb = (T["post_bias"] if T["post_bias"] is not None else 0 * one), (T["pre_bias"] if T["pre_bias"] is not None else 0 * one)
    rows, d = T["x"].shape
    A, gate = rs * T["x"].abs(), one.expand(rows, d)
    tol = {}
    yn = ny = ry = None
    if T["y"] is not None:
        if T["gate"] is not None:
            gate = T["gate"].repeat_interleave(rows // T["gate"].shape[0], 0)
        c = T["y"] - T["y"].mean(-1, keepdim=True) if kind == "layer" else T["y"]
        ry = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
        yn = top(T["y"]) * ry + (c * ry).abs()                                                      # what a normalised y is made of
        ny = yn * pw.abs() + pb.abs()
        A = A + gate.abs() * ny
    xn, h = R.block_norms(T, rs, kind, eps, pre)
    tol["x_new"] = CHAIN * A
    gx, gh = cx.double().abs() if cx is not None else 0 * A, None
    if pre:
        c = xn - xn.mean(-1, keepdim=True) if kind == "layer" else xn
        r = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
        xh = top(A) * r + (c * r).abs()
        tol["h"] = CHAIN * (xh * qw.abs() + qb.abs())
        gh = ch.double().abs()
        a = gh * qw.abs()
        gx = gx + r * (a + avg(a) + xh * avg(a * xh))
        tol["pre_weight"] = (CHAIN + rows * U32) * (gh * xh).sum(0)
        tol["pre_bias"] = (CHAIN + rows * U32) * gh.sum(0)
    tol["x"] = 2 * CHAIN * (rs if T["y"] is not None else 1.0) * gx
    if T["y"] is not None:
        G = 1 if T["gate"] is None else T["gate"].shape[0]
        tol["gate"] = (2 * CHAIN + rows // G * U32) * (gx * ny).reshape(G, -1, d).sum(1)
        dn = gx * gate.abs()
        tol["post_weight"] = (2 * CHAIN + rows * U32) * (dn * yn).sum(0)
        tol["post_bias"] = (2 * CHAIN + rows * U32) * dn.sum(0)
        b = dn * pw.abs()
        tol["y"] = 3 * CHAIN * ry * (b + avg(b) + yn * avg(b * yn))
    return tol


def check_norms(t, kind, rs, pre, g, eps=1e-6, grads=True, use=(True, True), views=lambda n, v: dev(v)):
    yt = t["y"].dtype if t["y"] is not None else t["x"].dtype
    T = {n: None if v is None else v.double().requires_grad_(grads) for n, v in t.items()}
    xn, h = R.block_norms(T, rs, kind, eps, pre)
    cx = rnd(g, *t["x"].shape, dtype=t["x"].dtype) if use[0] else None
    ch = rnd(g, *t["x"].shape, dtype=yt) if pre and use[1] else None
    tol = norm_tolerances({n: None if v is None else v.detach() for n, v in T.items()}, kind, eps, rs, pre, cx, ch if ch is not None else 0 * t["x"])
    a = {n: views(n, v) for n, v in t.items()}
    kw = {n: a[n] for n in NAMES[2:]}
    gx_new, gh = ops.block_norms(a["x"], a["y"], residual_scale=rs, norm=kind, eps=eps, pre=pre, **kw)
    if t["y"] is not None:
        within(gx_new, xn.detach(), tol["x_new"], "x_new")
    else:
        assert gx_new is a["x"]
    if pre:
        within(gh, h.detach(), tol["h"], "h")
        assert gh.dtype == yt
    else:
        assert gh is None
    if not grads:
        return
    total = 0.0
    if cx is not None:
        total = total + (xn * cx.double()).sum()
    if ch is not None:
        total = total + (h * ch.double()).sum()
    want = dict(zip([n for n in NAMES if T[n] is not None], torch.autograd.grad(total, [v for v in T.values() if v is not None], allow_unused=True)))
    got = ops.block_norms_grad(dev(cx), dev(ch), a["x"], a["y"], residual_scale=rs, norm=kind, eps=eps, pre=pre, **kw)
    for n in NAMES:
        if t[n] is None:
            assert getattr(got, n) is None
            continue
        w = want[n] if want[n] is not None else torch.zeros_like(T[n])
        assert getattr(got, n).dtype == t[n].dtype and getattr(got, n).shape == a[n].shape
        within(getattr(got, n).reshape(w.shape), w, tol[n], f"gradient of {n}")
    again = ops.block_norms_grad(dev(cx), dev(ch), a["x"], a["y"], residual_scale=rs, norm=kind, eps=eps, pre=pre, **kw)
    assert all(p is None or torch.equal(p, q) for p, q in zip(got, again)), "the same inputs gave other bits"


TYPES = [(torch.float32, torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16, torch.float32),
         (torch.float32, torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows,d,groups", [(1, 1, 1), (7, 5, 7), (40, 64, 5), (96, 63, 1), (64, 65, 32), (12, 250, 3), (10, 512, 1), (6, 513, 2), (9, 1000, 9),
                                           (5, 2050, 1), (4, 4096, 4), (3, 8192, 1), (2, 8200, 1), (2, 16384, 2)])
def test_block_norms(kind, types, rows, d, groups):
    g = gen(rows * d)
    check_norms(norm_inputs(g, rows, d, groups, *types, kind), kind, 0.75, True, g)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,d,groups", [(4096, 64, 512), (3000, 64, 3), (5000, 72, 5000), (2100, 40, 1), (1500, 130, 1), (2048, 300, 16), (4200, 8, 42)])
def test_block_norms_many_rows(kind, rows, d, groups):
    """Rows over many blocks, gates that several blocks share, short runs of rows per gate."""
    g = gen(rows + d)
    check_norms(norm_inputs(g, rows, d, groups, torch.float32, torch.bfloat16, torch.float32, kind), kind, 1.0, True, g)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("d", [64, 257, 4100])
def test_block_norms_forms(kind, d):
    """Entry without y, exit without h, no gate, gradients of one output only, no weights at all."""
    f, b = torch.float32, torch.bfloat16
    g = gen(d)
    for has_y, pre, gate, use in ((False, True, False, (True, True)), (False, True, False, (False, True)), (True, False, True, (True, False)),
                                  (True, True, False, (True, True)), (True, True, True, (False, True)), (True, True, True, (True, False))):
        check_norms(norm_inputs(g, 18, d, 6, f if has_y else b, b, f, kind, has_y, pre, gate), kind, 0.5, pre, g, use=use)
    bare = norm_inputs(g, 18, d, 6, b, b, b, kind)
    check_norms({n: v if n in ("x", "y") else None for n, v in bare.items()}, kind, 0.5, True, g)
    x = rnd(g, 3, 5, d)
    _, h = ops.block_norms(dev(x), pre_weight=torch.ones(d, device=DEV), norm=kind, dtype=b)          # fp32 stream, 16-bit branch
    want = R.norm(x.double(), None, None, kind, 1e-6)
    within(h, want, CHAIN * (want.abs() + x.double().abs().amax(-1, keepdim=True) * 4), "entry in bf16")


def test_block_norms_strides_shapes_and_large_values():
    g = gen(5)
    t = norm_inputs(g, 24, 70, 4, torch.float32, torch.bfloat16, torch.float32, "layer")

    def views(n, v):
        if n in ("x", "y"):                            # rows inside a wider buffer, NaN around them
            wide = torch.full((v.shape[0], v.shape[1] + 5), float("nan"), dtype=v.dtype)
            wide[:, 2:-3] = v
            return dev(wide)[:, 2:-3]
        return dev(v)
    check_norms(t, "layer", 0.9, True, g, views=views)
    # [B, N, d] with a gate [B, 1, d]; a transposed x is copied
    x, y, gate = rnd(g, 4, 6, 70), rnd(g, 4, 6, 70), rnd(g, 4, 1, 70)
    xt = dev(x.transpose(0, 1).contiguous()).transpose(0, 1)
    x_new, h = ops.block_norms(xt, dev(y), gate=dev(gate))
    flat = ops.block_norms(dev(x).reshape(24, 70), dev(y).reshape(24, 70), gate=dev(gate).reshape(4, 70))
    assert x_new.shape == (4, 6, 70) and torch.equal(x_new.reshape(24, 70), flat[0]) and torch.equal(h.reshape(24, 70), flat[1])
    # rows far from zero (LayerNorm's mean first), rows of zeros, values near fp16's end
    for big in (1000.0, -3.0e4):
        t = norm_inputs(g, 8, 96, 1, torch.float16, torch.float16, torch.float16, "layer")
        t["y"] = (rnd(g, 8, 96) * 8 + big).half()
        t["x"][3] = 0
        t["y"][2] = 0
        check_norms(t, "layer", 1.0, True, g, eps=1e-5)
    e = torch.zeros(0, 12, device=DEV)
    x_new, h = ops.block_norms(e, e, pre_weight=torch.ones(12, device=DEV))
    assert x_new.shape == h.shape == (0, 12)
    gr = ops.block_norms_grad(e, e, e, e, pre_weight=torch.ones(12, device=DEV), gate=torch.ones(12, device=DEV))
    assert gr.x.shape == (0, 12) and not gr.pre_weight.any() and not gr.gate.any()


# ---------------------------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------------------------
def distill_inputs(g, rows, V, K, dtype, tdtype=torch.float32):
    logits = rnd(g, rows, V, dtype=dtype, std=2.5)
    ids = torch.randint(0, V, (rows, K), generator=g)
    ids[torch.rand(rows, K, generator=g) < 0.15] = -1
    ids[torch.rand(rows, K, generator=g) < 0.05] = V
    if K > 2:
        ids[:, 2] = ids[:, 0]                          # an index twice
    tl = rnd(g, rows, K, dtype=tdtype, std=2.0)
    tl[torch.rand(rows, K, generator=g) < 0.05] = -float("inf")
    w = torch.rand(rows, generator=g) + 0.2
    if rows > 2:
        ids[1] = -1                                    # no entries
        w[2] = 0.0
        logits[2] = float("nan")                       # and what does not count may hold anything
    return logits, ids, tl, w


def distill_tolerances(logits, ids, tl, tau, w, reduction, grad):
    """fp32 part.  An exponential's argument (s - max) / tau is off by 3 2^-24 of itself (two roundings, log2 e), so its value by as much relative plus
    1 ulp; a sum of n terms in lanes adds CHAIN + n / 64 lanes (V <= 2^18 over at least 8 lanes of 8: the loop of the largest variant adds
    V / 8192 pieces one after the other).  The largest argument that matters is 90 (exp(-90) of the maximum is 0 beside 1)."""
    V = logits.shape[1]
    q = CHAIN + V / 8192 * U32 + 3 * U32 * 90
    weight = torch.ones(len(w)).double() if w is None else w.double().clamp(min=0)
    n = 1.0 if reduction != "mean" else max(float(weight.sum()), 1e-30)
    x = logits.double().nan_to_num(0.0)
    z = x / tau
    span = z.amax(1) - z.amin(1) + 30                  # bound of |log p|, |log q| that enter a row's loss
    row = weight * tau * tau * span * (q + CHAIN)
    if reduction == "none":
        return row, None
    g = (weight * tau)[:, None] * (torch.softmax(z, 1) + torch.zeros_like(z).scatter_add_(1, ids.clamp(0, V - 1), torch.ones_like(tl).double())) * 2 * q / n
    g = g + (weight * tau)[:, None] * 2.0 ** -126 / n  # an exponential below 2^-126 is 0 (v_exp_f32 gives no subnormal numbers)
    return row.sum() / n + len(w) * U32 * float((weight * tau * tau * span).sum()) / n, g


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,K", [(1, 1, 1), (5, 7, 3), (40, 9, 9), (33, 64, 20), (3, 20, 200), (6, 65, 5), (7, 513, 64), (5, 2049, 16), (4, 8200, 30),
                                      (3, 33001, 64), (3, 66001, 7), (3, 131080, 1024)])
def test_distill(dtype, rows, V, K):
    g = gen(V + K)
    tdtype = DTYPES[rows % 3]
    logits, ids, tl, w = distill_inputs(g, rows, V, K, dtype, tdtype)
    for reduction, weight, tau in (("mean", w, 1.0), ("sum", None, 2.5), ("none", w, 0.7)):
        lg = logits.nan_to_num(0.5) if weight is None else logits
        want, grad = R.distill(lg, ids, tl, tau, weight, reduction)
        tol, gtol = distill_tolerances(lg, ids, tl, tau, weight if weight is not None else torch.ones(rows), reduction, grad)
        a = (dev(lg), dev(ids), dev(tl))
        kw = dict(temperature=tau, row_weight=dev(weight), reduction=reduction)
        within(ops.distill_loss(*a, **kw), want, tol, f"loss {reduction}")
        loss, got = ops.distill_loss_and_grad(*a, **kw)
        within(loss, want, tol, f"loss of the step {reduction}")
        leaf = dev(lg).requires_grad_(True)
        auto = ops.distill_loss(leaf, dev(ids.int()), a[2], **kw)
        auto.sum().backward()
        assert torch.equal(auto.detach(), loss)
        if reduction != "none":
            within(got, grad, gtol, f"gradient {reduction}")
            within(leaf.grad, grad, gtol, f"gradient through autograd {reduction}")
        else:
            up = rnd(g, rows)                          # an upstream gradient for each row
            leaf.grad = None
            ops.distill_loss(leaf, a[1], a[2], **kw).backward(dev(up))
            _, gsum = R.distill(lg, ids, tl, tau, weight, "sum")
            _, t2 = distill_tolerances(lg, ids, tl, tau, weight, "sum", gsum)
            within(leaf.grad, gsum * up.double()[:, None], t2 * up.double().abs()[:, None] + U32 * (gsum * up[:, None]).abs(), "per-row upstream")
            within(got, gsum, t2, "gradient none")
        for zero in ((1, 2) if weight is not None and rows > 2 else (1,) if rows > 2 else ()):
            assert not got[zero].any() and not leaf.grad[zero].any()


def test_distill_edges():
    g = gen(9)
    logits, ids, tl, w = distill_inputs(g, 6, 300, 8, torch.float32)
    wide = torch.full((6, 333), float("nan"))
    wide[:, 7:307] = logits.nan_to_num(0.5)
    a = ops.distill_loss_and_grad(dev(wide)[:, 7:307], dev(ids), dev(tl))
    b = ops.distill_loss_and_grad(dev(logits.nan_to_num(0.5)), dev(ids), dev(tl))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # weights that are all zero: a loss of 0, gradients of 0, whatever the logits hold
    loss, grad = ops.distill_loss_and_grad(torch.full((6, 300), float("nan"), device=DEV), dev(ids), dev(tl), row_weight=torch.zeros(6, device=DEV))
    assert float(loss) == 0.0 and not grad.any()
    # masked logits (-inf) that the teacher does not list
    x = rnd(g, 4, 100)
    x[:, 50:] = -float("inf")
    i = torch.randint(0, 50, (4, 5), generator=g)
    t = rnd(g, 4, 5)
    want, wg = R.distill(torch.where(torch.isinf(x), -1e5, x), i, t, 1.0, None, "mean")
    loss, grad = ops.distill_loss_and_grad(dev(x), dev(i), dev(t))
    tol, gt = distill_tolerances(x[:, :50], i, t, 1.0, torch.ones(4), "mean", wg[:, :50])
    within(loss, want, tol, "masked vocabulary")
    within(grad[:, :50], wg[:, :50], gt, "masked vocabulary")
    assert not grad[:, 50:].any()
    # no rows; leading dimensions; the teacher that equals the student
    e = ops.distill_loss_and_grad(torch.zeros(0, 9, device=DEV), torch.zeros(0, 2, dtype=torch.int64, device=DEV), torch.zeros(0, 2, device=DEV))
    assert float(e[0]) == 0.0 and e[1].shape == (0, 9)
    s = rnd(g, 2, 3, 11)
    full = torch.arange(11).expand(2, 3, 11)
    loss, grad = ops.distill_loss_and_grad(dev(s), dev(full), dev(s), reduction="none")
    assert loss.shape == (2, 3) and float(loss.abs().max()) <= 30 * (CHAIN + 3 * U32 * 90) and float(grad.abs().max()) <= 2 * (CHAIN + 3 * U32 * 90)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [7, 300, 5000, 60001, 140000])
def test_distill_masks_of_the_lowest_value(dtype, V):
    """Rows masked with their type's lowest value: in part, at temperatures that take its scaled value out of fp32, and whole (a padded
    row without a weight: every token is as likely).  The exponents of masked tokens are exact (no weight at all, or 0 in the
    whole row), so the tolerances are those of rows with -60 (or 0) in their place."""
    g = gen(V)
    rows, K = 4, 3
    low = torch.finfo(dtype).min
    x = rnd(g, rows, V, dtype=dtype, std=2.0)
    x[0] = low
    x[1, V // 2:] = low
    x[2, 1:] = low
    ids = torch.randint(0, max(1, V // 2), (rows, K), generator=g)
    ids[2] = 0
    x[3] += 30000 if dtype == torch.float16 else 1e7   # far from 0 as a whole, one step apart
    tl = rnd(g, rows, K, dtype=dtype)
    like = torch.where(x == low, -60.0, x.float())
    like[0] = 0
    like[3] -= like[3].max()                           # (exact differences)
    for tau in (0.1, 0.6, 1.0, 1.5, 3.0):
        want, grad = R.distill(x, ids, tl, tau, None, "sum")
        tol, gtol = distill_tolerances(like, ids, tl, tau, torch.ones(rows), "sum", grad)
        loss, got = ops.distill_loss_and_grad(dev(x), dev(ids), dev(tl), temperature=tau, reduction="sum")
        within(loss, want, tol, f"loss, tau {tau}")
        within(got, grad, gtol, f"gradient, tau {tau}")
        leaf = dev(x).requires_grad_(True)
        ops.distill_loss(leaf, dev(ids), dev(tl), temperature=tau, reduction="sum").backward()
        within(leaf.grad, grad, gtol, f"gradient through autograd, tau {tau}")


def test_distill_gradient_against_differences():
    """fp32 on the device: the loss along a direction, both from the kernels.  A loss of about 5 is off by 5 CHAIN; over 2 eps = 0.1 that is
    4e-4, and the third derivative along a unit direction (tau = 1, |v| = 1) is at most 1: eps^2 / 6 = 4e-4."""
    g = gen(11)
    x, ids, tl = rnd(g, 50, 700, std=2.5), torch.randint(0, 700, (50, 9), generator=g), rnd(g, 50, 9)
    _, grad = ops.distill_loss_and_grad(dev(x), dev(ids), dev(tl), reduction="sum")
    v = rnd(g, 50, 700)
    v[:, :9] += 10 * rnd(g, 50, 9)
    v = v / v.norm()
    f = lambda s: float(ops.distill_loss(dev(x + s * v), dev(ids), dev(tl), reduction="none").double().sum())          # noqa: E731
    assert abs((f(0.05) - f(-0.05)) / 0.1 - float((grad.cpu().double() * v.double()).sum())) <= 50 * 5 * CHAIN / 0.1 + 4e-4


# ---------------------------------------------------------------------------------------------------------------
# drawing
# ---------------------------------------------------------------------------------------------------------------
def want_tokens(x, u, temperature, top_k, top_p, min_p):
    at = lambda v, r: float(v[r]) if torch.is_tensor(v) else v                                          # noqa: E731
    return [R.sample_row(x[r].float().numpy(), float(u[r]), at(temperature, r), int(at(top_k, r)), at(top_p, r), at(min_p, r)) for r in range(len(x))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", [(1, 1), (50, 2), (300, 7), (300, 9), (70, 33), (40, 64), (40, 65), (30, 511), (20, 4096), (12, 4097), (6, 20001), (66, 16500), (2, 140000)])
def test_sample_tokens(dtype, rows, V):
    g = gen(rows * V)
    x = rnd(g, rows, V, dtype=dtype, std=2.5)
    if V > 4:
        x[torch.rand(rows, V, generator=g) < 0.1] = -float("inf")
        x[0] = torch.round(x[0] * 2) / 2               # many ties
        x[-1, 1:] = float("nan")                       # one token to draw
        x[-1, 0] = 1.0
    u = torch.rand(rows, generator=g)
    u[0] = 0.0
    rows_of = lambda lo, hi: torch.rand(rows, generator=g) * (hi - lo) + lo                               # noqa: E731
    ks = torch.randint(0, max(2, min(V + 2, 60)), (rows,), generator=g, dtype=torch.int32)
    for settings in (dict(), dict(temperature=0.6, top_k=5), dict(top_p=0.7), dict(top_p=0.999, temperature=1.4), dict(min_p=0.05), dict(top_k=1), dict(temperature=0.0),
                     dict(temperature=rows_of(0.2, 1.5), top_k=ks, top_p=rows_of(0.3, 1.1), min_p=rows_of(0.0, 0.1)),
                     dict(top_k=max(1, V // 2), top_p=0.9, min_p=0.01), dict(top_p=0.0), dict(top_k=V + 1), dict(top_k=max(1, V - 1))):
        full = {**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **settings}
        got = ops.sample_tokens(dev(x), dev(u), **{k: dev(v) if torch.is_tensor(v) else v for k, v in settings.items()})
        assert got.dtype == torch.int64 and got.cpu().tolist() == want_tokens(x, u, **full), f"{settings}"


@pytest.mark.parametrize("V", [7, 64, 100, 4500, 66000])
def test_sample_ties_and_extremes(V):
    g = gen(V)
    u = torch.rand(24, generator=g)
    flat = torch.zeros(24, V)
    flat[8:16] = -0.0
    flat[16:, ::2] = -0.0                              # -0 and +0 are one logit
    cases = [(flat, dict()), (flat, dict(top_k=3)), (flat, dict(top_k=V // 2, top_p=0.5)), (flat, dict(top_p=0.25))]
    two = torch.where(torch.rand(24, V, generator=g) < 0.3, 1.0, 0.0)
    cases += [(two, dict(top_k=2)), (two, dict(top_k=V - 2)), (two, dict(top_p=0.6)), (two, dict(top_k=max(1, 2 * V // 3), top_p=0.9))]
    wide = rnd(g, 24, V, std=1e4)
    cases += [(wide, dict(top_p=0.9)), (wide, dict(top_k=4)), (wide * 1e30, dict(temperature=1e30, top_k=4)), (rnd(g, 24, V) * 1e-30, dict(temperature=1e-30, top_p=0.8))]
    inf = rnd(g, 24, V)
    inf[:, V // 2] = float("inf")
    cases += [(inf, dict()), (inf, dict(top_p=0.5)), (inf, dict(top_k=3))]
    for x, settings in cases:
        full = {**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **settings}
        assert ops.sample_tokens(dev(x), dev(u), **settings).cpu().tolist() == want_tokens(x, u, **full), f"{settings}"
    nothing = torch.full((4, V), -float("inf"))
    nothing[1] = float("nan")
    for settings in (dict(), dict(top_k=2, top_p=0.5), dict(temperature=0.0)):
        assert ops.sample_tokens(dev(nothing), dev(u[:4]), **settings).cpu().tolist() == [-1] * 4
    one = torch.tensor([1.0, 2.0, float("nan"), -1.0])                 # u outside [0, 1): the last or the first kept token
    got = ops.sample_tokens(dev(rnd(g, 4, V)), dev(one), top_k=3).cpu()
    assert ((got >= 0) & (got < V)).all()
    big = ops.sample_tokens(dev(two), dev(u), min_p=torch.full((24,), 2.0, device=DEV)).cpu().tolist()
    assert big == want_tokens(two, u, 1.0, 1, 1.0, 0.0)                # nothing is as likely as twice the largest: the largest stays
    for t in (5e-324, 1e-308, 1e308):                                  # the ends of the temperature's range: the largest logit, or any
        assert ops.sample_tokens(dev(wide), dev(u), temperature=t).cpu().tolist() == want_tokens(wide, u, t if t > 1 else 0.0, 0, 1.0, 0.0)
    strided = torch.full((24, V + 9), float("nan"))
    strided[:, 4:V + 4] = two
    assert torch.equal(ops.sample_tokens(dev(strided)[:, 4:V + 4], dev(u), top_p=0.6), ops.sample_tokens(dev(two), dev(u), top_p=0.6))
    assert ops.sample_tokens(torch.zeros(0, V, device=DEV), torch.zeros(0, device=DEV)).shape == (0,)


@pytest.mark.parametrize("what", ["normal", "near 0", "far", "halves", "few values", "masked low", "one"])
@pytest.mark.parametrize("V", [9001, 65541])
def test_sample_bf16_values(what, V):
    """Rows that the counting of bf16 values meets: spread ones, many within 2^-9 of 0 (more than its list holds, too), beyond 2^9, ties at
    every cut, masked with large negative numbers."""
    g = gen(len(what))
    rows = 6
    x = rnd(g, rows, V, std=2.5)
    if what == "near 0":
        x = x * torch.tensor([1e-4, 1e-3, 4e-3, 0.02, 0.1, 0.3])[:, None]
    elif what == "far":
        x = x * torch.tensor([100.0, 200.0, 1e3, 1e6, 1.0, 1.0])[:, None]
        x[4, 7], x[5, 9] = -3e38, 600.0
    elif what == "halves":
        x = torch.round(x * 2) / 2
    elif what == "few values":
        x = torch.randint(0, 3, (rows, V), generator=g).float() + torch.arange(rows)[:, None] - 3
    elif what == "masked low":
        x[torch.rand(rows, V, generator=g) < 0.9] = -1e9
        x[1] = x[1].clamp(max=-520.0)
        x[2, 1:] = -1e9
    elif what == "one":
        x[:] = -float("inf")
        x[torch.arange(rows), torch.arange(rows) * 1500] = torch.tensor([3.0, 0.0, -0.001, -40.0, 1e-30, 511.0])
    x = x.bfloat16()
    u = torch.rand(rows, generator=g)
    for settings in (dict(), dict(temperature=0.3), dict(top_p=0.9), dict(top_p=0.5, min_p=0.1), dict(min_p=0.02, temperature=2.0), dict(top_k=2000), dict(top_k=V - 3, top_p=0.8),
                     dict(top_k=1500, top_p=0.999, min_p=1e-4), dict(min_p=1.0), dict(temperature=30.0, top_p=0.7)):
        full = {**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **settings}
        assert ops.sample_tokens(dev(x), dev(u), **settings).cpu().tolist() == want_tokens(x, u, **full), f"{settings}"


@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_few_rows_as_many(dtype):
    """Few long rows are shared by many workgroups: the same tokens as among more rows than that, also where a cut by rank meets rows with
    less than k logits, and top-k alone where each group of logits has at most a few of the largest."""
    g = gen(5)
    rows, V = 96, 70001
    x = rnd(g, rows, V, dtype=dtype, std=2.5)
    x[1, 40:] = -float("inf")
    x[2] = torch.round(x[2])
    x[3] = x[3].sort(descending=True).values           # the largest side by side
    x[4] = -float("inf")
    x[5, V - 1] = 40.0
    x, u = dev(x), dev(torch.rand(rows, generator=g))
    many = dict(temperature=torch.rand(rows, generator=g) + 0.2, top_k=torch.randint(0, 40, (rows,), generator=g, dtype=torch.int32) ** 2, top_p=torch.rand(rows, generator=g) + 0.3)
    many = {k: dev(v) for k, v in many.items()}
    many["temperature"][6] = 0.0
    for settings in (dict(), dict(temperature=0.0), dict(min_p=0.05), dict(min_p=3.0), dict(top_k=1), dict(top_k=60), dict(top_k=60, temperature=many["temperature"]), dict(top_k=200, top_p=0.9), dict(top_k=900), dict(top_k=5000, min_p=0.01),
                     dict(top_p=0.9), dict(top_p=0.3, min_p=0.1), dict(temperature=20.0, top_p=0.99), many):
        some = {k: v[:9] if torch.is_tensor(v) else v for k, v in settings.items()}
        assert torch.equal(ops.sample_tokens(x[:9], u[:9], **some), ops.sample_tokens(x, u, **settings)[:9]), f"{settings}"


@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_largest_vocab(dtype):
    g = gen(20)
    x = rnd(g, 2, 1 << 20, dtype=dtype, std=2.5)
    x[1] = 0.0
    x[1, -1] = 0.5
    u = torch.tensor([0.3, 0.9999999])
    for settings in (dict(), dict(top_k=100), dict(top_p=0.9), dict(temperature=0.0), dict(top_k=5000, top_p=0.7, min_p=0.01)):
        full = {**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **settings}
        got = ops.sample_tokens(dev(x), dev(u), **settings)
        assert got.cpu().tolist() == want_tokens(x, u, **full), f"{settings}"
        many = ops.sample_tokens(dev(x).repeat(33, 1), dev(u).repeat(33), **settings)
        assert torch.equal(many.view(33, 2), got.expand(33, 2)), f"{settings}"


def test_sample_more_rows_than_a_launch():
    n = (1 << 21) + 5
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(n, 65, generator=g, device=DEV).half()
    u = torch.rand(n, generator=g, device=DEV)
    rows = dict(temperature=torch.rand(n, generator=g, device=DEV) + 0.5, top_k=torch.randint(0, 9, (n,), generator=g, device=DEV, dtype=torch.int32),
                top_p=torch.rand(n, generator=g, device=DEV) + 0.2, min_p=torch.rand(n, generator=g, device=DEV) * 0.2)
    got = ops.sample_tokens(x, u, **rows)
    for part in (slice(0, 1000), slice(n - 1000, n)):
        assert torch.equal(got[part], ops.sample_tokens(x[part], u[part], **{k: v[part] for k, v in rows.items()}))


def test_sample_frequencies():
    """2^16 draws of one row: each token's count within six standard deviations of its probability."""
    x = torch.tensor([0.3, -1.0, 2.0, 1.9, 0.0, -3.0, 1.0])
    n = 1 << 16
    u = (torch.arange(n, dtype=torch.float32) + 0.5) / n
    for settings, keep in ((dict(), 7), (dict(top_k=3), 3)):
        t = ops.sample_tokens(dev(x.expand(n, 7)), dev(u[torch.randperm(n, generator=gen(1))]), **settings).cpu()
        p = torch.softmax(torch.where(x >= x.sort(descending=True).values[keep - 1], x, -float("inf")).double(), 0)
        c = torch.bincount(t, minlength=7).double()
        assert ((c - n * p).abs() <= 6 * torch.sqrt(n * p * (1 - p)) + 1e-9).all()


def test_drawing_ends_a_sampling_round():
    g = gen(2)
    x = torch.rand(64, 8, 7, generator=g)
    x[:, 0, 0] += 20
    x[:, 7, 1] += 20
    x[:, 1:7, :2] = -float("inf")
    u = torch.rand(64, 8, generator=g)
    one = utils.draw_onehot(dev(x), dev(u), temperature=0.5)
    assert one.shape == x.shape and (one.sum(-1) == 1).all()
    status, code, counts = AF.device_validity(one)
    assert int(counts[0]) == 64 and (status == -1).all()
    want = R.sample_row(x[5, 3].numpy(), float(u[5, 3]), 0.5, 0, 1.0, 0.0)
    assert int(one[5, 3].argmax()) == want


def test_generate_archs_meta_draws():
    """``args.draw_temperature`` ends a round by drawing; without it the sampler's output is thresholded as before."""
    g = gen(3)
    x = torch.rand(32, 8, 7, generator=g)
    x[:, 0, 0] += 20
    x[:, 7, 1] += 20
    x[:, 1:7, :2] = -float("inf")
    sampling_fn = lambda *a, **kw: dev(x)                                                                # noqa: E731
    config, model = SimpleNamespace(device=DEV), torch.nn.Identity()
    run = lambda **kw: run_lib.generate_archs_meta(config, sampling_fn, model, None, model, 32, patient_factor=1,    # noqa: E731
                                                   args=SimpleNamespace(classifier_scale=1.0, scale_step=0.1, **kw))

    def first_seen(sample):
        seen = AF.new_seen_table(DEV)
        AF.device_validity(sample, seen, 0)
        first = seen.cpu()
        codes = (first != AF.UNSEEN).nonzero()[:, 0]
        return [AF.code_to_string(int(c)) for c in codes[first[codes].sort(stable=True).indices]]
    torch.manual_seed(9)
    got = run(draw_temperature=0.7, draw_top_p=0.9, draw_min_p=0.05)
    torch.manual_seed(9)
    u = torch.rand(32, 8, device=DEV)
    assert got == first_seen(utils.draw_onehot(dev(x), u, temperature=0.7, top_p=0.9, min_p=0.05)) and len(got) > 1
    assert run() == run(draw_temperature=0.0) == first_seen(dev(x))


# ---------------------------------------------------------------------------------------------------------------
# together: a token model trained against a teacher's top logits, then drawn from
# ---------------------------------------------------------------------------------------------------------------
def model_loss(p, ids, tids, tl, w, o):
    """Two blocks over tokens; ``o``: the operators (the library's, or plain float64 ones)."""
    d = p["embed"].shape[1]
    x = o.embed(ids, p["embed"], d ** 0.5)
    x, h = o.norms(x, None, None, p["n0"])
    for b in range(2):
        y = torch.tanh(h @ p[f"w{b}"])
        x, h = o.norms(x, y, p[f"g{b}"], p[f"n{b + 1}"])
    logits = h @ p["embed"].t()
    return o.distill(logits, tids, tl, w), logits


class Lib:
    embed = staticmethod(lambda ids, w, s: ops.embed_tokens(ids, w, scale=s))
    norms = staticmethod(lambda x, y, g, w: ops.block_norms(x, y, gate=g, pre_weight=w, residual_scale=0.9))
    distill = staticmethod(lambda l, i, t, w: ops.distill_loss(l, i, t, temperature=1.5, row_weight=w))


class Plain:
    embed = staticmethod(R.embed)

    @staticmethod
    def norms(x, y, g, w):
        flat = dict(x=x.reshape(-1, x.shape[-1]), pre_weight=w)
        if y is not None:
            flat.update(y=y.reshape(-1, x.shape[-1]), gate=g.reshape(1, -1))
        xn, h = R.block_norms(flat, 0.9, "rms", 1e-6, True)
        return xn.reshape(x.shape), h.reshape(x.shape)

    @staticmethod
    def distill(l, i, t, w):
        rows = R.distill_rows(l.reshape(-1, l.shape[-1]), i.reshape(-1, i.shape[-1]), t.reshape(-1, t.shape[-1]), 1.5, w.reshape(-1))
        return rows.sum() / w.double().sum()


def model_inputs(seed, B=6, N=8, V=23, d=40, K=5):
    g = gen(seed)
    p = dict(embed=rnd(g, V, d, std=0.2), w0=rnd(g, d, d, std=0.2), w1=rnd(g, d, d, std=0.2), g0=rnd(g, d), g1=rnd(g, d), n0=1 + rnd(g, d, std=0.1),
             n1=1 + rnd(g, d, std=0.1), n2=1 + rnd(g, d, std=0.1))
    ids = torch.randint(0, V, (B, N), generator=g)
    ids[-1, 5:] = -1
    w = (ids >= 0).float()
    return p, ids, torch.randint(0, V, (B, N, K), generator=g), rnd(g, B, N, K, std=2.0), w


def test_token_model_gradients():
    """Gradients of the whole model against the same model in 64 bits.  Each of the six operators in a row, and the matrix products of
    40 terms between them, passes on a relative error of a few CHAIN: 64 CHAIN of the largest gradient of a tensor covers their product."""
    p, ids, tids, tl, w = model_inputs(1)
    P64 = {n: v.double().requires_grad_(True) for n, v in p.items()}
    want, wl = model_loss(P64, ids, tids, tl, w, Plain)
    wg = torch.autograd.grad(want, list(P64.values()))
    P = {n: dev(v).requires_grad_(True) for n, v in p.items()}
    loss, logits = model_loss(P, dev(ids), dev(tids), dev(tl), dev(w), Lib)
    loss.backward()
    assert abs(float(loss.detach()) - float(want.detach())) <= 64 * CHAIN * abs(float(want.detach()))
    for n, gw in zip(p, wg):
        assert float((P[n].grad.cpu().double() - gw).abs().max()) <= 64 * CHAIN * float(gw.abs().max()), n
    u = torch.rand(ids.shape, generator=gen(3))
    t = ops.sample_tokens(logits, dev(u), temperature=0.8, top_k=8, top_p=0.9)
    assert t.cpu().reshape(-1).tolist() == want_tokens(logits.detach().cpu().reshape(-1, 23), u.reshape(-1), 0.8, 8, 0.9, 0.0)


def test_token_model_trains_with_the_frameworks_optimiser():
    p, ids, tids, tl, w = model_inputs(2)
    P = {n: torch.nn.Parameter(dev(v)) for n, v in p.items()}
    opt = losses.get_optimizer(Cfg(optim=Cfg(optimizer="Adam", lr=1e-2, beta1=0.9, eps=1e-8, weight_decay=0.0)), P.values())
    ema = ema_lib.ExponentialMovingAverage(list(P.values()), decay=0.9)
    before = {n: v.detach().clone() for n, v in P.items()}
    for _ in range(3):
        opt.zero_grad()
        loss, _ = model_loss(P, dev(ids), dev(tids), dev(tl), dev(w), Lib)
        loss.backward()
        opt.step(grad_clip=1.0, ema=ema)
    assert all(torch.isfinite(v).all() and not torch.equal(v, before[n]) for n, v in P.items()) and bool(torch.isfinite(loss))


# ---------------------------------------------------------------------------------------------------------------
# streams and graphs
# ---------------------------------------------------------------------------------------------------------------
def every_call(s):
    """One call of each operator on its inputs."""
    out = [ops.embed_tokens(s["ids"], s["w"], scale=3.0), ops.embed_tokens_grad(s["g"], s["ids"], 500), ops.embed_tokens_grad(s["g"], s["ids"] % 7, 7),
           ops.embed_tokens_grad(s["gl"], s["idl"], 500)]
    out += [t for t in ops.block_norms(s["g"], s["y"], gate=s["y"][:1], pre_weight=s["y"][0], post_weight=s["y"][1])]
    out += [t for t in ops.block_norms_grad(s["y"], s["g"], s["g"], s["y"], gate=s["y"][:2], pre_weight=s["y"][0], post_weight=s["y"][1]) if t is not None]
    out += list(ops.distill_loss_and_grad(s["g"], s["tids"], s["tl"], row_weight=s["rw"])) + [ops.distill_loss(s["g"], s["tids"], s["tl"], reduction="none")]
    out += [ops.sample_tokens(s["w"], s["u"], top_p=0.9, temperature=0.7), ops.sample_tokens(s["w"][:, :40], s["u"], top_k=5), ops.sample_tokens(s["w"], s["u"], top_k=9)]
    return out


def call_inputs(seed):
    g = gen(seed)
    return {k: dev(v) for k, v in dict(ids=some_ids(g, 600, 500), idl=some_ids(g, 9000, 500), w=rnd(g, 500, 96), g=rnd(g, 600, 96), gl=rnd(g, 9000, 96), y=rnd(g, 600, 96),
                                       tids=torch.randint(0, 96, (600, 6), generator=g), tl=rnd(g, 600, 6), rw=torch.rand(600, generator=g),
                                       u=torch.rand(500, generator=g)).items()}


def test_two_streams_at_once():
    a, b = call_inputs(1), call_inputs(2)
    want = every_call(a), every_call(b)
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    got = {}
    for _ in range(5):
        for st, x, k in ((sa, a, 0), (sb, b, 1)):
            with torch.cuda.stream(st):
                got[k] = every_call(x)
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(p, q) for p, q in zip(got[k], want[k]))


def test_captured_and_replayed():
    """Two captured graphs, replayed in turn with other inputs and eager work between, against eager calls."""
    side = torch.cuda.Stream()
    static = [call_inputs(1), call_inputs(2)]
    with torch.cuda.stream(side):
        for s in static:
            every_call(s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(every_call(s))
        graphs.append(gr)
    for seed in (5, 6, 7):
        for k in (0, 1):
            new = call_inputs(seed + 10 * k)
            want = every_call(new)
            for n, v in new.items():
                static[k][n].copy_(v)
            graphs[k].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs[k], want)), f"replay {seed} of graph {k}"


def test_shared_rows_captured_and_on_two_streams():
    """Drawing from few long rows keeps sums in a workspace: two captured graphs replayed in turn on changed logits, and two streams at
    once, against one call at a time."""
    settings = (dict(), dict(top_k=60, top_p=0.9), dict(top_p=0.8), dict(min_p=0.01, temperature=2.0))

    def inputs(seed):
        g = gen(seed)
        return dev(rnd(g, 3, 70001, std=2.5)), dev(torch.rand(3, generator=g))

    def draw(x, u):
        return torch.stack([ops.sample_tokens(x, u, **s) for s in settings])
    static = [inputs(1), inputs(2)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        draw(*static[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(draw(*s))
        graphs.append(gr)
    for seed in (3, 5, 7):
        new = [inputs(seed), inputs(seed + 1)]
        want = [draw(*n) for n in new]
        for k in (0, 1):
            for t, n in zip(static[k], new[k]):
                t.copy_(n)
            graphs[k].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), f"replay {seed}"
        got = []
        for n, stream in zip(new, (side, torch.cuda.Stream())):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got.append([draw(*n) for _ in range(4)])
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for many, w in zip(got, want) for o in many), f"streams {seed}"


def test_captured_training_step_through_autograd():
    """forward and backward captured with fresh leaves; refused where an eager graph of the leaves is alive."""
    g = gen(4)
    w, ids = torch.nn.Parameter(dev(rnd(g, 30, 24))), dev(some_ids(g, 50, 30))
    nw = torch.nn.Parameter(dev(rnd(g, 24)))
    tids, tl = dev(torch.randint(0, 30, (50, 4), generator=g)), dev(rnd(g, 50, 4))

    def step():
        _, h = ops.block_norms(ops.embed_tokens(ids, w), pre_weight=nw)
        loss = ops.distill_loss(h @ w.detach().t(), tids, tl)
        return (loss,) + torch.autograd.grad(loss, (w, nw))
    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = step()
    for _ in range(3):
        for t in got:
            t.detach().fill_(7.0)
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(got, want))
    alive = ops.embed_tokens(ids, w)
    gr2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr2):
        torch.zeros(1, device=DEV)
        with pytest.raises(RuntimeError, match="eager autograd graph"):
            ops.embed_tokens(ids, w)
    del alive


# ---------------------------------------------------------------------------------------------------------------
# workgroups that take several rows, runs or column tiles
# ---------------------------------------------------------------------------------------------------------------
F, B16, H16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("rows,d,groups,types,kind", [
    (700, 4100, 1, (B16, B16, B16), "rms"), (600, 8192, 2, (B16, B16, F), "rms"), (1200, 4104, 600, (H16, H16, H16), "rms"),         # the next row asked for ahead
    (700, 4100, 1, (F, F, F), "layer"), (700, 4100, 7, (F, B16, B16), "rms"), (600, 5000, 2, (B16, B16, B16), "layer"),              # not ahead
    (3000, 640, 3, (B16, B16, F), "rms"), (3000, 640, 3, (F, F, F), "layer"), (1100, 520, 1100, (F, B16, B16), "layer"), (4000, 1100, 2, (B16, B16, B16), "rms"),
    (1300, 2100, 5, (H16, H16, F), "layer"), (600, 8200, 1, (B16, B16, B16), "rms"), (600, 8200, 300, (F, F, F), "layer"), (520, 16384, 1, (F, B16, B16), "rms")])
def test_block_norms_many_rows_of_a_workgroup(rows, d, groups, types, kind):
    """Above 512 columns a team is the workgroup (or one of two halves of it): more rows than workgroups, so that each goes through several rows of
    one gate (700 of 4100: three), or through several gates (1100 gates of 520: two for some)."""
    g = gen(rows + d)
    check_norms(norm_inputs(g, rows, d, groups, *types, kind), kind, 0.9, True, g)


@pytest.mark.parametrize("rows,V,d", [(8200, 300, 2100), (9000, 3000, 520), (8200, 20000, 2100), (60000, 300, 2100), (270000, 20000, 24)])
@pytest.mark.parametrize("hot", [False, True])
def test_embed_grad_wide_rows_and_long_lists(rows, V, d, hot):
    """The sorted list with teams of several widths, several column tiles, zero rows longer than a workgroup clears at once, and chunks of 8 to 64
    entries.  Sums in 64 bits by index_add_."""
    g = gen(rows + V + d + hot)
    dtype = DTYPES[(rows // 1000 + hot) % 3]
    grad, ids = rnd(g, rows, d, dtype=dtype), some_ids(g, rows, V, hot)
    at = torch.where((ids >= 0) & (ids < V), ids, V)
    n = torch.bincount(at, minlength=V + 1)[:V, None].double()
    want = torch.zeros(V + 1, d, dtype=torch.float64).index_add_(0, at, grad.double())[:V] * 1.5
    mag = torch.zeros(V + 1, d, dtype=torch.float64).index_add_(0, at, grad.double().abs())[:V] * 1.5
    got = ops.embed_tokens_grad(dev(grad), dev(ids), V, scale=1.5)
    within(got, want, (n + 2) * U32 * mag, f"{dtype}")
    assert not got[dev((n == 0).squeeze(1))].any()
    assert torch.equal(got, ops.embed_tokens_grad(dev(grad), dev(ids.int()), V, scale=1.5)), "the same inputs gave other bits"


def test_gates_of_positions():
    """A gate for each position of every sequence is expanded to the shape of x; its gradient comes back through the expansion."""
    g = gen(8)
    x, y, gate = rnd(g, 5, 6, 70), rnd(g, 5, 6, 70), rnd(g, 1, 6, 70)
    cx, ch = rnd(g, 5, 6, 70), rnd(g, 5, 6, 70)
    flat = norm_inputs(g, 30, 70, 30, F, F, F, "rms")
    flat.update(x=x.reshape(30, 70), y=y.reshape(30, 70), gate=gate.expand(5, 6, 70).reshape(30, 70))
    tol = norm_tolerances(flat, "rms", 1e-6, 1.0, True, cx.reshape(30, 70), ch.reshape(30, 70))
    T = {n: None if v is None else v.double() for n, v in flat.items()}
    rows_gate = T["gate"].clone().requires_grad_(True)
    xn, h = R.block_norms({**T, "gate": rows_gate}, 1.0, "rms", 1e-6, True)
    (each,) = torch.autograd.grad((xn.reshape(5, 6, 70) * cx).sum() + (h.reshape(5, 6, 70) * ch).sum(), rows_gate)
    each = each.reshape(5, 6, 70)
    leaf = dev(gate).requires_grad_(True)
    x_new, got_h = ops.block_norms(dev(x), dev(y), gate=leaf.expand(5, 6, 70), post_weight=dev(flat["post_weight"]), pre_weight=dev(flat["pre_weight"]))
    within(x_new.reshape(30, 70), xn.detach(), tol["x_new"], "x_new")
    within(got_h.reshape(30, 70), h.detach(), tol["h"], "h")
    (got,) = torch.autograd.grad([x_new, got_h], leaf, [dev(cx), dev(ch)])
    slack = tol["gate"].reshape(5, 6, 70).sum(0) + 6 * U32 * each.abs().sum(0)             # each one rounded to fp32, then five of them added
    within(got[0], each.sum(0), slack, "gradient of the gate")
    for bad in (dev(gate), dev(gate)[0]):
        with pytest.raises(ValueError, match="gate"):
            ops.block_norms(dev(x), dev(y), gate=bad)


@pytest.mark.parametrize("rows", [2047, 2048, 2049, 5000])
@pytest.mark.parametrize("V,d", [(17, 40), (255, 8), (300, 70), (70000, 3)])
def test_embed_grad_on_both_sides_of_the_sorts_border(rows, V, d):
    """Lists of up to 2048 entries are sorted by one workgroup, longer ones by digits; the sums run in the same order, so a list that grows by dropped
    rows over the border gives the same bits."""
    g = gen(rows + V + d)
    grad, ids = rnd(g, rows, d), some_ids(g, rows, V, True)
    want, mag, n = R.embed_grad(ids, grad, V, 1.5, 3)
    got = ops.embed_tokens_grad(dev(grad), dev(ids), V, scale=1.5, padding_idx=3)
    within(got, want, (n + 2) * U32 * mag, "sum")
    assert not got[dev((n == 0).squeeze(1))].any()
    if rows <= 2048:                                   # (as many entries for a team: 8 up to 32768 rows)
        more = ops.embed_tokens_grad(torch.cat([dev(grad), torch.full((3000, d), float("nan"), device=DEV)]), torch.cat([dev(ids), torch.full((3000,), -1, device=DEV)]), V,
                                     scale=1.5, padding_idx=3)
        assert torch.equal(more, got)


def test_compiled_callers():
    """torch.compile breaks its graph around the calls: the same results and gradients as without it."""
    s = call_inputs(3)
    w, g = s["w"].requires_grad_(True), s["y"][0]

    def f(ids, w, y):
        x, h = ops.block_norms(ops.embed_tokens(ids, w, scale=2.0) * 1.5, y + 0.0, pre_weight=g)
        loss = ops.distill_loss(h * 2, s["tids"], s["tl"], row_weight=s["rw"])
        return loss, x, ops.sample_tokens(h.detach() * 3, s["rw"], top_k=5)
    want, got = f(s["ids"], w, s["y"]), torch.compile(f, backend="eager")(s["ids"], w, s["y"])
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    assert torch.equal(*(torch.autograd.grad(o[0], w)[0] for o in (want, got)))
