"""Token operators without a GPU: the oracle against differences, the refusals of the Python face and of the C entries (which
check before they touch the device)."""

import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

from diffusionnag_amd import _lib, token_ops as ops
from tests import token_reference as R


def difference(f, x, v, eps=1e-5):
    """Central difference of f along v, float64."""
    return float((f(x + eps * v) - f(x - eps * v)) / (2 * eps))


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_block_norms_formula_against_differences(kind):
    g = torch.Generator().manual_seed(3)
    t = {n: torch.randn(s, generator=g, dtype=torch.float64) for n, s in
         dict(x=(6, 5), y=(6, 5), gate=(3, 5), post_weight=(5,), pre_weight=(5,)).items()}
    if kind == "layer":
        t["post_bias"], t["pre_bias"] = torch.randn(5, generator=g).double(), torch.randn(5, generator=g).double()
    cx, ch = torch.randn(6, 5, generator=g).double(), torch.randn(6, 5, generator=g).double()

    def f(name, v):
        xn, h = R.block_norms({**t, name: v}, 0.7, kind, 1e-6, True)
        return (xn * cx).sum() + (h * ch).sum()
    for name in t:
        x = t[name].clone().requires_grad_(True)
        (grad,) = torch.autograd.grad(f(name, x), x)
        v = torch.randn(x.shape, generator=g).double()
        want = float((grad * v).sum())
        assert abs(difference(lambda z: f(name, z), t[name], v) - want) <= 1e-7 * max(1.0, abs(want))


def test_distill_formula_against_differences():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(4, 9, generator=g).double()
    ids = torch.tensor([[1, 3, 1], [8, -1, 9], [-1, -1, 12], [0, 2, 4]])
    tl = torch.randn(4, 3, generator=g).double()
    w = torch.tensor([0.5, 2.0, 1.0, 0.0])
    _, grad = R.distill(x, ids, tl, 1.7, w, "mean")
    v = torch.randn(4, 9, generator=g).double()
    want = float((grad * v).sum())
    assert abs(difference(lambda z: R.distill(z, ids, tl, 1.7, w, "mean")[0], x, v) - want) <= 1e-8
    assert not grad[2:].any()


def test_sample_reference_knows_the_easy_cases():
    x = [0.0, 2.0, 2.0, 1.0]
    assert R.sample_row(x, 0.9, 0.0, 0, 1.0, 0.0) == 1                     # greedy, ties to the lowest index
    assert R.sample_row(x, 0.99, 1.0, 1, 1.0, 0.0) == 1
    assert R.sample_row(x, 0.99, 1.0, 2, 1.0, 0.0) == 2
    assert R.sample_row([0.0] * 4, 0.6, 1.0, 0, 0.5, 0.0) == 1             # two of four equal ones hold half
    assert R.sample_row([-np.inf, np.nan], 0.5, 1.0, 0, 1.0, 0.0) == -1
    assert R.sample_row(x, 0.0, 1.0, 0, 1.0, 0.9) == 1 and R.sample_row(x, 0.99, 1.0, 0, 1.0, 0.9) == 2


F32 = torch.float32


def test_cpu_tensors_are_refused():
    ids, w = torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8)
    for call in (lambda: ops.embed_tokens(ids, w), lambda: ops.embed_tokens_grad(torch.zeros(3, 8), ids, 4),
                 lambda: ops.embed_tokens(ids, w.requires_grad_(True)),
                 lambda: ops.block_norms(torch.zeros(2, 8), torch.zeros(2, 8)), lambda: ops.block_norms_grad(None, None, torch.zeros(2, 8)),
                 lambda: ops.distill_loss(torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)),
                 lambda: ops.distill_loss_and_grad(torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)),
                 lambda: ops.sample_tokens(torch.zeros(2, 8), torch.zeros(2))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("call", [
    lambda: ops.embed_tokens(torch.zeros(3), torch.zeros(4, 8)),                                        # ids of no integer type
    lambda: ops.embed_tokens(torch.zeros(3, dtype=torch.int16), torch.zeros(4, 8)),
    lambda: ops.embed_tokens(torch.zeros(3, dtype=torch.int64), torch.zeros(4)),
    lambda: ops.embed_tokens(torch.zeros(3, dtype=torch.int64), torch.zeros(0, 8)),
    lambda: ops.embed_tokens(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8, dtype=torch.float64)),
    lambda: ops.embed_tokens(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8), padding_idx=4),
    lambda: ops.embed_tokens(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8), padding_idx=-1),
    lambda: ops.embed_tokens_grad(torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64), 4),
    lambda: ops.embed_tokens_grad(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), 0),
    lambda: ops.block_norms(torch.zeros(2, 8), torch.zeros(2, 9)),
    lambda: ops.block_norms(torch.zeros(2, 8), torch.zeros(2, 8), norm="batch"),
    lambda: ops.block_norms(torch.zeros(2, 8), torch.zeros(2, 8), eps=-1.0),
    lambda: ops.block_norms(torch.zeros(2, 8), torch.zeros(2, 8), eps=float("nan")),
    lambda: ops.block_norms(torch.zeros(2, 8), torch.zeros(2, 8), pre_bias=torch.zeros(8)),             # RMSNorm has no bias
    lambda: ops.block_norms(torch.zeros(2, 8), gate=torch.zeros(8)),                                     # a gate without y
    lambda: ops.block_norms(torch.zeros(2, 8), pre=False),
    lambda: ops.block_norms(torch.zeros(2, 8), torch.zeros(2, 8), pre=False, pre_weight=torch.zeros(8)),
    lambda: ops.block_norms(torch.zeros(2, 8), torch.zeros(2, 8), post_weight=torch.zeros(7)),
    lambda: ops.block_norms(torch.zeros(2, 8), torch.zeros(2, 8), post_weight=torch.zeros(8).half()),
    lambda: ops.block_norms(torch.zeros(2, 8), torch.zeros(2, 8), gate=torch.zeros(3, 8)),               # 2 rows, 3 gates
    lambda: ops.block_norms(torch.zeros(2, 8).bfloat16(), torch.zeros(2, 8)),                            # 16-bit stream, 32-bit branch
    lambda: ops.block_norms(torch.zeros(2, 8), torch.zeros(2, 8), dtype=torch.bfloat16),
    lambda: ops.block_norms(torch.zeros(1, 16385), torch.zeros(1, 16385)),
    lambda: ops.block_norms(torch.zeros(2, 0), torch.zeros(2, 0)),
    lambda: ops.block_norms(torch.zeros(2, 8), torch.zeros(2, 8), norm="layer", pre_weight=torch.zeros(8), pre_bias=torch.zeros(8).half()),
    lambda: ops.distill_loss(torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 4)),
    lambda: ops.distill_loss(torch.zeros(2, 8), torch.zeros(3, 3, dtype=torch.int64), torch.zeros(3, 3)),
    lambda: ops.distill_loss(torch.zeros(2, 8), torch.zeros(2, 0, dtype=torch.int64), torch.zeros(2, 0)),
    lambda: ops.distill_loss(torch.zeros(2, 8), torch.zeros(2, 1025, dtype=torch.int64), torch.zeros(2, 1025)),
    lambda: ops.distill_loss(torch.zeros(2, 8), torch.zeros(2, 3), torch.zeros(2, 3)),
    lambda: ops.distill_loss(torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3), temperature=0.0),
    lambda: ops.distill_loss(torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3), temperature=float("inf")),
    lambda: ops.distill_loss(torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3), temperature=1e-30),
    lambda: ops.distill_loss(torch.zeros(2, 8).half(), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3), temperature=0.09),
    lambda: ops.distill_loss(torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3), reduction="batchmean"),
    lambda: ops.distill_loss(torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3), row_weight=torch.zeros(3)),
    lambda: ops.distill_loss(torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3), row_weight=torch.zeros(2).half()),
    lambda: ops.distill_loss(torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3, requires_grad=True)),
    lambda: ops.sample_tokens(torch.zeros(2, 8), torch.zeros(3)),
    lambda: ops.sample_tokens(torch.zeros(2, 8), torch.zeros(2).double()),
    lambda: ops.sample_tokens(torch.zeros(2, 0), torch.zeros(2)),
    lambda: ops.sample_tokens(torch.zeros(2, 8).double(), torch.zeros(2)),
    lambda: ops.sample_tokens(torch.zeros(2, 8), torch.zeros(2), temperature=torch.ones(3)),
    lambda: ops.sample_tokens(torch.zeros(2, 8), torch.zeros(2), top_k=torch.ones(2)),
    lambda: ops.sample_tokens(torch.zeros(2, 8), torch.zeros(2), top_p=float("nan")),
    lambda: ops.sample_tokens(torch.zeros(2, 8), torch.zeros(2), temperature=float("inf")),
])
def test_bad_arguments_are_refused(call):
    with pytest.raises(ValueError):
        call()


def refused(rc, words):
    assert rc == -1 or rc == -2, rc
    assert words in _lib.load().dnag_last_error().decode()


def test_c_entries_check_before_they_launch():
    """Addresses that are not NULL stand for device memory; every call below is refused on the host."""
    lib, P = _lib.load(), 4096
    e = lib.dnag_embed_forward
    refused(e(P, 8, 1, P, 8, 4, 8, 7, 1.0, P, None), "dtype")
    refused(e(P, 2, 1, P, 8, 4, 8, 0, 1.0, P, None), "ids of 2 bytes")
    refused(e(P, 8, -1, P, 8, 4, 8, 0, 1.0, P, None), "rows")
    refused(e(P, 8, 1, P, 7, 4, 8, 0, 1.0, P, None), "stride")
    refused(e(P, 8, 1, P, 8, 0, 8, 0, 1.0, P, None), "num_tokens")
    refused(e(P, 8, 1, P, 8, 4, 0, 0, 1.0, P, None), "dim")
    refused(e(None, 8, 1, P, 8, 4, 8, 0, 1.0, P, None), "NULL")
    refused(e(P, 8, 0x7fffffff, P, 4096, 4, 4096, 0, 1.0, P, None), "too many rows")
    assert e(None, 8, 0, None, 8, 4, 8, 0, 1.0, None, None) == 0                      # no rows: nothing to do
    need = lib.dnag_embed_grad_workspace_bytes(1000, 500, 64)
    assert need > 0
    refused(lib.dnag_embed_grad(P, 8, 1000, P, 64, 500, 64, 0, 1.0, -1, P, P, need - 1, None), "workspace")
    refused(lib.dnag_embed_grad(P, 8, 1000, P, 64, 500, 64, 0, 1.0, -1, None, P, need, None), "NULL")
    assert lib.dnag_embed_grad_workspace_bytes(-1, 500, 64) == 0

    def norms(**kw):
        a = _lib.BlockNormsArgsC()
        base = dict(rows=4, dim=8, gate_rows=1, dtype=1, x_dtype=1, pre=1, x=P, y=P, x_stride=8, y_stride=8, x_new=P, h=P, eps=1e-6,
                    grad_x=P, grad_h=P, grad_x_stride=8, grad_h_stride=8, dx=P, dy=P)
        for k, v in {**base, **kw}.items():
            setattr(a, k, v)
        return a
    for kw, words in ((dict(dtype=9), "dtype"), (dict(x_dtype=2), "residual"), (dict(dim=16385), "dim"), (dict(dim=0), "dim"), (dict(gate_rows=3), "gate rows"),
                      (dict(post_bias=P), "no bias"), (dict(y=None, pre=0), "pre must"), (dict(y=None, gate=P), "need y"),
                      (dict(pre=0, pre_weight=P), "without pre"), (dict(x_stride=7), "stride"), (dict(x=None), "NULL"), (dict(h=None), "NULL")):
        refused(lib.dnag_block_norms_forward(C.byref(norms(**kw))), words)
    assert lib.dnag_block_norms_forward(C.byref(norms(rows=0))) == 0
    a = norms(pre_weight=P, d_pre_weight=P, workspace=P)
    need = lib.dnag_block_norms_grad_workspace_bytes(C.byref(a))
    a.workspace_bytes = need - 1
    refused(lib.dnag_block_norms_grad(C.byref(a)), "workspace")
    refused(lib.dnag_block_norms_grad(C.byref(norms(d_gate=P, workspace=P, workspace_bytes=1 << 40))), "not there")
    refused(lib.dnag_block_norms_grad(C.byref(norms(pre=0, workspace=P, workspace_bytes=1 << 40))), "grad_h without pre")
    refused(lib.dnag_block_norms_grad(C.byref(norms(rows=0))), "no rows")
    refused(lib.dnag_block_norms_forward(None), "NULL")

    def distill(**kw):
        a = _lib.DistillArgsC()
        base = dict(rows=4, vocab=8, logits_stride=8, k=3, ids_bytes=8, reduction=2, temperature=1.0, logits=P, teacher_ids=P, teacher_logits=P,
                    loss=P, stats=P, grad_out=P, grad=P, workspace=P, workspace_bytes=1 << 20)
        for k, v in {**base, **kw}.items():
            setattr(a, k, v)
        return a
    for kw, words in ((dict(dtype=3), "dtype"), (dict(teacher_dtype=-1), "dtype"), (dict(ids_bytes=1), "ids of 1"), (dict(vocab=0), "vocab"), (dict(k=0), "k=0"),
                      (dict(k=1025), "k=1025"), (dict(temperature=0.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
                      (dict(logits_stride=7), "stride"), (dict(reduction=3), "reduction"), (dict(loss=None), "NULL"), (dict(workspace_bytes=0), "workspace"),
                      (dict(rows=0), "no rows")):
        refused(lib.dnag_distill_loss(C.byref(distill(**kw))), words)
        refused(lib.dnag_distill_loss_grad(C.byref(distill(**kw))), words)
    refused(lib.dnag_distill_loss_grad(C.byref(distill(grad=None))), "NULL")
    refused(lib.dnag_distill_backward(C.byref(distill(stats=None))), "NULL")
    refused(lib.dnag_distill_backward(C.byref(distill(grad_out=None))), "NULL")

    refused(lib.dnag_distill_loss(C.byref(distill(rows=0x7fffffff, vocab=1000, logits_stride=1000, reduction=0, workspace_bytes=1 << 40))), "too many rows")
    refused(lib.dnag_block_norms_forward(C.byref(norms(rows=0x7fffffff, gate_rows=1, dim=4096, x_stride=4096, y_stride=4096))), "too many rows")

    def sample(**kw):
        a = _lib.SampleArgsC()
        base = dict(rows=4, vocab=8, logits_stride=8, temperature=1.0, top_p=1.0, logits=P, u=P, out=P)
        for k, v in {**base, **kw}.items():
            setattr(a, k, v)
        return a
    for kw, words in ((dict(dtype=3), "dtype"), (dict(rows=-1), "rows"), (dict(vocab=(1 << 20) + 1), "vocab"), (dict(vocab=0), "vocab"),
                      (dict(logits_stride=7), "stride"), (dict(u=None), "NULL"), (dict(out=None), "NULL")):
        refused(lib.dnag_sample_tokens(C.byref(sample(**kw))), words)
    assert lib.dnag_sample_tokens(C.byref(sample(rows=0))) == 0
    few = sample(rows=2, vocab=70000, logits_stride=70000)
    need = lib.dnag_sample_workspace_bytes(C.byref(few))
    assert need >= 2 * 70000 // 128 * 4
    for kw in (dict(workspace=None, workspace_bytes=need), dict(workspace=P, workspace_bytes=need - 1)):
        refused(lib.dnag_sample_tokens(C.byref(sample(rows=2, vocab=70000, logits_stride=70000, **kw))), "workspace")
    for kw in (dict(rows=500), dict(rows=-1), dict(rows=1 << 40), dict(vocab=1 << 21), dict(temperature=0.0), dict(top_k_rows=P), dict(top_k=5000)):
        assert lib.dnag_sample_workspace_bytes(C.byref(sample(**{**dict(rows=2, vocab=70000, logits_stride=70000), **kw}))) == 0


def test_eager_graph_of_the_same_leaf_is_noticed(monkeypatch):
    """_leaf_mark: a leaf whose gradient accumulator lives on from an eager graph is refused under capture, a fresh one is not."""
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    w = torch.zeros(3, requires_grad=True)
    alive = (w * 2).sum()
    ops._leaf_mark(w, None, torch.zeros(3))
    capturing[0] = True
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        ops._leaf_mark(w)
    del alive
    ops._leaf_mark(w)


# calls of every differentiable operator and explicit gradient with one argument given, the others plain
IDS, TIDS = torch.tensor([0, 2, 1]), torch.tensor([[0, 1], [2, -1], [3, 3]])
DIFFERENTIABLE = {
    "embedding weight": ((4, 8), lambda t: ops.embed_tokens(IDS, t)),
    "embedding grad": ((3, 8), lambda t: ops.embed_tokens_grad(t, IDS, 4)),
    "norms x": ((3, 8), lambda t: ops.block_norms(t, torch.ones(3, 8))),
    "norms x alone": ((3, 8), lambda t: ops.block_norms(t)),
    "norms y": ((3, 8), lambda t: ops.block_norms(torch.ones(3, 8), t)),
    "norms gate": ((8,), lambda t: ops.block_norms(torch.ones(3, 8), torch.ones(3, 8), gate=t)),
    "norms weight": ((8,), lambda t: ops.block_norms(torch.ones(3, 8), torch.ones(3, 8), post_weight=t)),
    "norms bias": ((8,), lambda t: ops.block_norms(torch.ones(3, 8), torch.ones(3, 8), norm="layer", pre_bias=t)),
    "norms grad": ((3, 8), lambda t: ops.block_norms_grad(None, t, torch.ones(3, 8))),
    "norms grad's x": ((3, 8), lambda t: ops.block_norms_grad(None, torch.ones(3, 8), t)),
    "distillation": ((3, 8), lambda t: ops.distill_loss(t, TIDS, torch.ones(3, 2))),
    "distillation teacher": ((3, 2), lambda t: ops.distill_loss(torch.ones(3, 8), TIDS, t)),
    "distillation weight": ((3,), lambda t: ops.distill_loss(torch.ones(3, 8), TIDS, torch.ones(3, 2), row_weight=t)),
    "distillation step": ((3, 8), lambda t: ops.distill_loss_and_grad(t, TIDS, torch.ones(3, 2))),
}


@pytest.mark.parametrize("what", DIFFERENTIABLE)
def test_tangents_are_refused(what):
    """A dual tensor has requires_grad False: taken for a plain one, the result would have no tangent, a derivative of zero."""
    from torch.autograd import forward_ad
    shape, call = DIFFERENTIABLE[what]
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(forward_ad.make_dual(torch.ones(shape), torch.ones(shape)))
        with pytest.raises(RuntimeError, match="no CPU fallback"):          # a plain tensor inside the level comes as far as ever
            call(torch.ones(shape))


RECORDED = {**DIFFERENTIABLE, "drawing": ((3, 8), lambda t: ops.sample_tokens(t, torch.zeros(3)))}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("recorder", ["jit", "fx", "fx before dispatch", "fx fake"])
@pytest.mark.parametrize("what", RECORDED)
def test_recording_is_refused(what, recorder, grad, monkeypatch):
    """torch.jit.trace and make_fx see the allocation of the result and not the launch (stubbed here) that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    shape, call = RECORDED[what]
    grad = grad and what not in ("distillation teacher", "distillation weight")         # those must not require one
    monkeypatch.setattr(ops, "_device", lambda *t: 0)
    monkeypatch.setattr(ops, "_launch", lambda *a: None)
    monkeypatch.setattr(ops, "_leaf_mark", lambda *t: None)
    t = torch.ones(shape, requires_grad=grad)
    call(t)                                                                 # not recorded: as ever
    with pytest.raises(RuntimeError, match="cannot be recorded"):
        if recorder == "jit":
            torch.jit.trace(call, t, check_trace=False)
        else:
            make_fx(call, tracing_mode="fake" if recorder == "fx fake" else "real", pre_dispatch=recorder == "fx before dispatch")(t)
    call(t)


@pytest.mark.parametrize("gate,x,fits", [
    ((8,), (6, 4, 8), True), ((1, 8), (6, 4, 8), True), ((1, 1, 8), (6, 4, 8), True), ((6, 1, 8), (6, 4, 8), True), ((6, 4, 8), (6, 4, 8), True),
    ((2, 3, 1, 8), (2, 3, 4, 8), True), ((2, 1, 1, 8), (2, 3, 4, 8), True), ((4, 8), (1, 4, 8), True), ((1, 4, 8), (1, 4, 8), True),
    ((6, 8), (6, 4, 8), True), ((12, 8), (6, 4, 8), True), ((24, 8), (6, 4, 8), True), ((6, 8), (24, 8), True), ((1, 8), (8,), True),   # lists of rows
    ((6, 1, 8), (24, 8), True), ((24, 1, 8), (6, 4, 8), True), ((6, 2, 8), (6, 4, 8), True),
    ((1, 4, 8), (6, 4, 8), False), ((4, 8), (6, 4, 8), False), ((4, 8), (4, 4, 8), False),                    # a row for each position
    ((2, 1, 4, 8), (2, 3, 4, 8), False), ((3, 1, 8), (2, 3, 4, 8), False), ((1, 3, 1, 8), (2, 3, 4, 8), False),
    ((1, 4, 8), (24, 8), False), ((2, 1, 4, 8), (24, 8), False),                                             # neither broadcasts nor is a list
])
def test_gates_mean_runs_of_rows(gate, x, fits, monkeypatch):
    """A gate that is taken means what torch's broadcasting makes of it, or is a list of rows: anything else is refused."""
    monkeypatch.setattr(ops, "_leaf_mark", lambda *t: None)
    a, g = torch.ones(x), torch.randn(gate, generator=torch.Generator().manual_seed(1))
    for call in (lambda: ops.block_norms(a, a, gate=g), lambda: ops.block_norms(a, a, gate=g.clone().requires_grad_(True)), lambda: ops.block_norms_grad(a, a, a, a, gate=g)):
        with pytest.raises(RuntimeError if fits else ValueError, match="no CPU fallback" if fits else "gate"):
            call()
    try:
        broadcast = torch.broadcast_shapes(gate, x) == x
    except RuntimeError:
        broadcast = False
    if fits and broadcast:                                             # the rows that the kernels use
        rows = a.numel() // 8
        used = g.reshape(-1, 8).repeat_interleave(rows // (g.numel() // 8), 0).reshape(x)
        assert torch.equal(used, g.expand(x))


@pytest.mark.parametrize("x,gate", [((0, 4, 8), (0, 1, 8)), ((0, 4, 8), (0, 4, 8)), ((0, 8), (0, 8)), ((0, 4, 8), (8,)), ((0, 4, 8), (3, 1, 8)), ((5, 0, 8), (5, 1, 8))])
def test_empty_batches_with_a_gate(x, gate, monkeypatch):
    """No rows: empty results and gradients of zeros, nothing is launched, whatever number of gate rows goes with them."""
    monkeypatch.setattr(ops, "_device", lambda *t: 0)
    monkeypatch.setattr(ops, "_launch", None)
    a, g = torch.ones(x), torch.ones(gate)
    x_new, h = ops.block_norms(a, a, gate=g, pre_weight=torch.ones(8))
    assert x_new.shape == h.shape == x
    got = ops.block_norms_grad(a, a, a, a, gate=g, pre_weight=torch.ones(8))
    assert got.x.shape == got.y.shape == x and got.gate.shape == gate and not got.gate.any() and got.pre_weight.shape == (8,) and not got.pre_weight.any()


LDS_RACE = r"""
#include "dnag_lds_limit.h"
#include <chrono>
#include <stdio.h>
#include <thread>
// The driver's side: one kernel, one device.  The call with the smaller value takes effect after the one with the larger, if the two overlap.
static std::atomic<size_t> limit{65536};
static std::atomic<int> inside{0}, smaller_done{0}, calls{0};
extern "C" hipError_t hipGetDevice(int *d) { *d = 0; return hipSuccess; }
extern "C" hipError_t hipFuncSetAttribute(const void *, hipFuncAttribute, int bytes) {
    ++calls;
    ++inside;
    for (int i = 0; i < 100 && inside < 2; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(2));     // time for the other one to come
    if (bytes == 80 * 1024) {
        std::this_thread::sleep_for(std::chrono::milliseconds(50));
        limit = bytes;
        smaller_done = 1;
        return hipSuccess;
    }
    limit = bytes;
    for (int i = 0; i < 100 && inside == 2 && !smaller_done; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(2));
    return hipSuccess;
}
int main() {
    static LdsLimit a;
    std::thread small([] { a.allow(nullptr, 80 * 1024); }), large([] { a.allow(nullptr, 120 * 1024); });
    small.join();
    large.join();
    const int before = calls;
    a.allow(nullptr, 120 * 1024);                      // recorded: nothing to set
    a.allow(nullptr, 60 * 1024);
    a.allow(nullptr, 60 * 1024, 8 * 1024);
    printf("%zu %d\n", limit.load(), calls.load() - before);
}
"""


def test_two_first_calls_leave_the_larger_lds_limit(tmp_path):
    """Two threads that ask for different amounts of LDS at once: the larger one has to be set in the end, since it is what is recorded."""
    src, exe = tmp_path / "race.cpp", tmp_path / "race"
    src.write_text(LDS_RACE)
    csrc = os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{csrc}", str(src), "-o", str(exe)], check=True)
    for _ in range(3):
        out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout.split()
        assert out == [str(120 * 1024), "0"], out


def test_every_lds_limit_is_set_under_the_lock():
    csrc = os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc")
    setting = [f for f in sorted(os.listdir(csrc)) if f.endswith((".hip", ".h")) and "hipFuncSetAttribute(" in open(os.path.join(csrc, f)).read()]
    assert setting == ["dnag_lds_limit.h"]


@pytest.mark.parametrize("rows,num_tokens,dim", [(0x7fffffff, 1000, 8), (1 << 30, 17, 1), (1 << 28, 70000, 4096), (600_000_000, 1 << 20, 256)])
def test_embed_grad_refuses_too_many_rows_before_it_launches(rows, num_tokens, dim):
    """Addresses that are not NULL stand for device memory; a launch would end in another error here, without a device."""
    P = 4096
    for dtype in (0, 1, 2):
        refused(_lib.load().dnag_embed_grad(P, 8, rows, P, dim, num_tokens, dim, dtype, 1.0, -1, P, P, 1 << 62, None), "too many rows")


@pytest.mark.parametrize("call", ["dnag_distill_loss", "dnag_distill_loss_grad", "dnag_distill_backward"])
@pytest.mark.parametrize("rows,vocab", [(0x7fffffff, 1000), (1 << 27, 5000), (1 << 25, 100000)])
def test_distill_refuses_too_many_rows_before_it_launches(call, rows, vocab):
    """With row weights and 'mean' the sum of the weights is the first launch; without a device it would end in another error."""
    P = 4096
    for dtype in (0, 1, 2):
        a = _lib.DistillArgsC(rows=rows, vocab=vocab, logits_stride=vocab, k=3, dtype=dtype, ids_bytes=8, reduction=2, temperature=1.0, logits=P, teacher_ids=P,
                              teacher_logits=P, row_weight=P, loss=P, stats=P, grad_out=P, grad=P, workspace=P, workspace_bytes=1 << 60)
        refused(getattr(_lib.load(), call)(C.byref(a)), "too many rows")


@pytest.mark.parametrize("padding_idx", [-1, 4, 10 ** 20])
def test_embed_grad_refuses_the_padding_that_the_lookup_refuses(padding_idx):
    """-1 is torch's name for the last token; taken as none, its row would get a gradient."""
    with pytest.raises(ValueError, match="padding_idx"):
        ops.embed_tokens_grad(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), 4, padding_idx=padding_idx)


def test_other_dispatch_modes_are_no_recording(monkeypatch):
    """Counting or printing modes only look on: the calls work inside them."""
    from torch.utils.flop_counter import FlopCounterMode
    monkeypatch.setattr(ops, "_device", lambda *t: 0)
    monkeypatch.setattr(ops, "_launch", lambda *a: None)
    with FlopCounterMode(display=False):
        assert ops.embed_tokens(IDS, torch.ones(4, 8)).shape == (3, 8) and ops.sample_tokens(torch.ones(3, 8), torch.zeros(3)).shape == (3,)
