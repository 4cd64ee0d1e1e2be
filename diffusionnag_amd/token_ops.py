"""Operators of token models on the HIP library: embedding lookup, the norms between blocks, distillation from a teacher's top
logits, and drawing tokens.

They stand beside the score network's own parts: ``embed_tokens`` is the embedding of nodes whose type is known (the
score network embeds real vectors, ``cate.py``), ``block_norms`` the seam that its encoder layers have inside the fused kernel,
``distill_loss`` a training loss like ``losses.get_sde_loss_fn_nas``, and ``sample_tokens`` the drawing counterpart of the
threshold ``utils.quantize`` (``utils.draw_onehot`` ends a sampling round with it).

Each operator is one call on the current stream.  Tensors live on one HIP device (there is no CPU path); inputs with a
contiguous last dimension are read in place, others are copied first; outputs are new contiguous tensors, workspaces come from torch's
allocator and belong to the call (also under graph capture).  The first three are differentiable through ``torch.autograd``;
``embed_tokens_grad``, ``block_norms_grad`` and ``distill_loss_and_grad`` give the same gradients without it, which is also how to
capture a training step into a graph: a backward pass of ``torch.autograd`` that is captured while an eager graph of the
same leaves is alive ends the process inside torch, so the differentiable calls raise there for leaves that one of them was given in
that graph (a graph that only other operations made is not seen).  There is no forward-mode
derivative: arguments that carry a tangent are refused.  So are torch.jit.trace and make_fx, which would record an empty result;
torch.compile breaks its graph around the calls.
Element types: float32, bfloat16, float16.  All sums and statistics are float32 or wider; results are rounded once.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
from torch._ops import mode_stack_state_for_pre_dispatch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_REDUCE = {"none": _lib.REDUCE_NONE, "sum": _lib.REDUCE_SUM, "mean": _lib.REDUCE_MEAN}
_IDS = {torch.int32: 4, torch.int64: 8}

_MOST = 1.7976931348623157e308

# read by every call, so bound once; [0] of the modes before dispatch is a recording one (or None)
_is_tracing, _dispatch_modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack
_pre_dispatch_modes = vars(mode_stack_state_for_pre_dispatch()).get("_ModeStackStateForPreDispatch__infra_modes", (None,))
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice

Number = Union[int, float]


# ---------------------------------------------------------------------------------------------------------------
# plumbing
# ---------------------------------------------------------------------------------------------------------------
def _dtype(t: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} has dtype {t.dtype}; float32, bfloat16 and float16 are built")
    return code


def _device(*tensors: Optional[torch.Tensor]) -> int:
    """Index of the one HIP device that holds the tensors (the checks and errors of ``_lib.require_device``, at a fifth of its time)."""
    index = -1
    for t in tensors:
        if t is None:
            continue
        k = t.get_device()
        if k < 0 or not t.is_cuda or (index >= 0 and k != index):
            _lib.require_device(*tensors)
        index = k
    return index


def _launch(fn, index: int, what: str, *args) -> None:
    """``fn(*args, stream)`` on the device's current stream, with the device current for the call."""
    stream = _raw_stream(index)
    before = _current_device()
    if before == index:
        rc = fn(*args, stream)
    else:
        torch.cuda.set_device(index)
        try:
            rc = fn(*args, stream)
        finally:
            torch.cuda.set_device(before)
    if rc != 0:
        _lib.check(rc, what)


def _launch_args(fn, index: int, what: str, layout, *fields) -> None:
    """The same for the entries that take one argument struct, whose last field is the stream: ``layout`` packs the fields (None is
    not one of them: 0 stands for NULL)."""
    _launch(lambda *a: fn(layout.pack(*a)), index, what, *fields)


def _rows2d(t: torch.Tensor):
    """([rows, d] view, row stride) of [..., d]: a contiguous last dimension and one row stride; a copy only where the strides ask for it."""
    d = t.shape[-1]
    if t.is_contiguous():
        return (t if t.dim() == 2 else t.view(-1, d) if t.numel() else t.reshape(t.numel() // max(d, 1), d)), d
    if t.dim() != 2:
        t = t.reshape(-1, d)
    if (d > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < d):
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else d


def _p(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _like(t: torch.Tensor) -> torch.Tensor:
    """A new contiguous tensor of the shape and type of ``t`` (empty_like takes half the time of empty: 1.1 and 2.2 us)."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _plain(*tensors: Optional[torch.Tensor]) -> None:
    """Refuses to be recorded or differentiated in ways that would pass the launch over without an error (0.2 us where nothing of the kind goes on).

    torch.jit.trace and make_fx would record the allocation of the result and not the launch that fills it: the recorded program would return
    memory as it is.  Dual tensors of forward-mode differentiation (``tensors``: the differentiable arguments) have requires_grad False; the
    result would have no tangent, which counts as a derivative of zero."""
    if (_is_tracing() or _dispatch_modes() or _pre_dispatch_modes[0] is not None) and (_is_tracing() or get_proxy_mode() is not None):
        raise RuntimeError("the token operators cannot be recorded by torch.jit.trace or make_fx: call them, or capture the calls into a HIP graph")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("the token operators have no forward-mode derivative: an argument carries a tangent (differentiate backward, or "
                                   "take the primal out with torch.autograd.forward_ad.unpack_dual)")


def _leaf_mark(*tensors: Optional[torch.Tensor]) -> None:
    """Refuses to record a backward pass of leaves under graph capture while an eager graph of the same leaves is alive: their
    gradient accumulators belong to the eager graph's stream, and running them inside the capture ends the process."""
    capturing = torch.cuda.is_current_stream_capturing()
    for t in tensors:
        if t is None or not t.requires_grad or not t.is_leaf:
            continue
        node = torch.autograd.graph.get_gradient_edge(t).node
        if not capturing:
            node.metadata["dnag_eager"] = True
        elif node.metadata.get("dnag_eager"):
            raise RuntimeError("an eager autograd graph of the same parameters is alive: free it before capturing, or capture the "
                               "explicit *_grad calls of diffusionnag_amd.token_ops")


# ---------------------------------------------------------------------------------------------------------------
# embedding lookup
# ---------------------------------------------------------------------------------------------------------------
def _check_ids(ids: torch.Tensor) -> torch.Tensor:
    if ids.dtype not in _IDS:
        raise ValueError(f"ids have dtype {ids.dtype}; int32 and int64 are built")
    return ids if ids.is_contiguous() else ids.contiguous()


def _embed(ids: torch.Tensor, weight: torch.Tensor, scale: float) -> torch.Tensor:
    index = _device(ids, weight)
    V, d = weight.shape
    out = weight.new_empty((*ids.shape, d))
    n = ids.numel()
    if n:
        w, stride = _rows2d(weight)
        _launch(_lib.load().dnag_embed_forward, index, "dnag_embed_forward", ids.data_ptr(), _IDS[ids.dtype], n, w.data_ptr(), stride, V, d,
                _DTYPES[weight.dtype], scale, out.data_ptr())
    return out


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.args = weight.shape[0], scale, padding_idx
        return _embed(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        num_tokens, scale, padding_idx = ctx.args
        return None, embed_tokens_grad(grad, ids, num_tokens, scale=scale, padding_idx=padding_idx), None, None


def embed_tokens(ids: torch.Tensor, weight: torch.Tensor, *, scale: Number = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[ids]`` ([*ids.shape, d], the type of ``weight``), rounded once.

    ``ids`` outside ``0 .. len(weight) - 1`` (the -1 or -100 of a padded batch, another shard's tokens) give rows of zeros and
    take no part in the gradient; ``padding_idx`` is looked up but takes no part in the gradient (as in torch)."""
    _plain(weight)
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be [num_tokens, dim], got {tuple(weight.shape)}")
    _dtype(weight, "weight")
    ids = _check_ids(ids)
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"padding_idx={padding_idx} is outside 0 .. {weight.shape[0] - 1}")
    if weight.requires_grad and torch.is_grad_enabled():
        _device(ids, weight)
        _leaf_mark(weight)
        return _EmbedTokens.apply(ids, weight, float(scale), padding_idx)
    return _embed(ids, weight, float(scale))


def embed_tokens_grad(grad: torch.Tensor, ids: torch.Tensor, num_tokens: int, *, scale: Number = 1.0,
                      padding_idx: Optional[int] = None) -> torch.Tensor:
    """Gradient of ``embed_tokens`` with respect to ``weight`` ([num_tokens, d], the type of ``grad``): the rows of ``grad``
    summed by token in float32, in the order of the tokens' positions, the same bits every time."""
    _plain(grad)
    lib = _lib.load()
    ids = _check_ids(ids)
    if grad.dim() < 1 or grad.shape[:-1] != ids.shape:
        raise ValueError(f"grad {tuple(grad.shape)} does not match ids {tuple(ids.shape)}")
    if num_tokens < 1 or grad.shape[-1] < 1:
        raise ValueError(f"num_tokens={num_tokens}, dim={grad.shape[-1]}: both must be positive")
    if padding_idx is not None and not 0 <= padding_idx < num_tokens:
        raise ValueError(f"padding_idx={padding_idx} is outside 0 .. {num_tokens - 1}")
    code = _dtype(grad, "grad")
    index = _device(grad, ids)
    g, stride = _rows2d(grad)
    rows, d = g.shape
    out = grad.new_empty((num_tokens, d))
    nbytes = lib.dnag_embed_grad_workspace_bytes(rows, num_tokens, d)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=grad.device) if nbytes else None
    _launch(lib.dnag_embed_grad, index, "dnag_embed_grad", ids.data_ptr(), _IDS[ids.dtype], rows, g.data_ptr(), stride, num_tokens, d, code, float(scale),
            -1 if padding_idx is None else int(padding_idx), out.data_ptr(), _p(ws), nbytes)
    return out


# ---------------------------------------------------------------------------------------------------------------
# norms between blocks
# ---------------------------------------------------------------------------------------------------------------
class BlockNormsGrad(NamedTuple):
    """Gradients of ``block_norms``, named like its arguments; None where the argument was not given."""
    x: torch.Tensor
    y: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]
    post_weight: Optional[torch.Tensor]
    post_bias: Optional[torch.Tensor]
    pre_weight: Optional[torch.Tensor]
    pre_bias: Optional[torch.Tensor]


def _small(t: Optional[torch.Tensor], name: str, d: int, dtype) -> Optional[torch.Tensor]:
    """A norm's weight or bias: [d], the branch's type or float32."""
    if t is None:
        return None
    if t.shape != (d,):
        raise ValueError(f"{name} must be [{d}], got {tuple(t.shape)}")
    if t.dtype != dtype and t.dtype != torch.float32:
        raise ValueError(f"{name} has dtype {t.dtype}; the branch's ({dtype}) or float32 are built")
    return t if t.is_contiguous() else t.contiguous()


def _check_gate(gate: torch.Tensor, x: torch.Tensor) -> None:
    """The kernels give each row of the gate a run of consecutive rows of ``x``.  Refuses shapes that say something else: a dimension that
    the gate repeats over, in front of one that it does not ([1, N, d] beside [B, N, d], [N, d] beside [B, N, d])."""
    lead, own = x.shape[:-1], gate.shape[:-1]
    over = len(lead) - len(own)
    if over >= 0 and all(g == 1 or g == n for g, n in zip(own, lead[over:])):                # broadcasts
        repeats = [g == 1 and n != 1 for g, n in zip((1,) * over + tuple(own), lead)]
        own = (1,) * over + tuple(own)
    else:                                                                                   # a list of rows
        repeats = [g == 1 for g in own]
    if any(r and any(g != 1 for g in own[k:]) for k, r in enumerate(repeats)):
        raise ValueError(f"gate {tuple(gate.shape)} beside x {tuple(x.shape)} repeats over a dimension in front of its own rows; built is a row for each run of "
                         "consecutive rows ([B, 1, d], [d]) or for each row (expand the gate to the shape of x)")


class _Seam:
    """The checked arguments of one ``block_norms`` call as the library takes them."""
    __slots__ = ("index", "shape", "device", "dtype", "given_x", "given_y", "x", "y", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias", "rows", "d", "pre", "head",
                 "arrays")

    def __init__(self, x, y, gate, residual_scale, post_weight, post_bias, pre_weight, pre_bias, norm, eps, pre, dtype=None):
        layer = norm == "layer"
        if not layer and norm != "rms":
            raise ValueError(f"norm={norm!r}: 'rms' and 'layer' are built")
        if not eps >= 0:
            raise ValueError(f"eps={eps} must not be negative")
        if x.dim() < 1 or x.shape[-1] < 1:
            raise ValueError(f"x must be [..., dim], got {tuple(x.shape)}")
        if y is None:
            if gate is not None or post_weight is not None or post_bias is not None:
                raise ValueError("gate and the norm behind a block need its output y")
            if not pre:
                raise ValueError("without y there is only the norm in front of the next block: pre must be True")
            dtype = dtype or x.dtype
        else:
            if y.shape != x.shape:
                raise ValueError(f"y {tuple(y.shape)} does not match x {tuple(x.shape)}")
            if dtype is not None and dtype != y.dtype:
                raise ValueError("dtype is the type of h at the entry (y=None); with y, h has the type of y")
            dtype = y.dtype
        if not pre and (pre_weight is not None or pre_bias is not None):
            raise ValueError("pre_weight / pre_bias with pre=False")
        if not layer and (post_bias is not None or pre_bias is not None):
            raise ValueError("RMSNorm has no bias")
        code, f32 = _DTYPES.get(dtype), torch.float32
        if code is None:
            raise ValueError(f"dtype {dtype}; float32, bfloat16 and float16 are built")
        if x.dtype != dtype and x.dtype != f32:
            raise ValueError(f"x has dtype {x.dtype}; the branch's ({dtype}) or float32 are built")
        d = x.shape[-1]
        if d > 16384:
            raise ValueError(f"dim={d}: 1 to 16384 are built")
        self.given_x, self.given_y = x, y
        self.x, xs = _rows2d(x)
        rows = self.x.shape[0]
        self.y, ys = (None, 0) if y is None else _rows2d(y)
        small = 0
        self.post_weight, self.post_bias = _small(post_weight, "post_weight", d, dtype), _small(post_bias, "post_bias", d, dtype)
        self.pre_weight, self.pre_bias = _small(pre_weight, "pre_weight", d, dtype), _small(pre_bias, "pre_bias", d, dtype)
        for bit, w, b in ((2, post_weight, post_bias), (4, pre_weight, pre_bias)):
            if w is not None and b is not None and w.dtype != b.dtype:
                raise ValueError(f"a norm's weight and bias have one type, got {w.dtype} and {b.dtype}")
            if (w is not None and w.dtype == f32) or (b is not None and b.dtype == f32):
                small |= bit
        gate_rows = 1
        if gate is not None:
            if gate.shape[-1:] != (d,) or (gate.dtype != dtype and gate.dtype != f32):
                raise ValueError(f"gate must be [..., {d}] of type {dtype} or float32, got {tuple(gate.shape)} {gate.dtype}")
            if gate.dim() > 1 and not gate.dim() == x.dim() == 2:
                _check_gate(gate, x)
            gate_rows = gate.numel() // d
            if rows and (gate_rows < 1 or rows % gate_rows):
                raise ValueError(f"{rows} rows do not divide into {gate_rows} gate rows")
            if gate.dtype == f32:
                small |= 1
            gate = gate if gate.is_contiguous() else gate.contiguous()
        self.gate = gate
        self.index = _device(x, y, gate, post_weight, post_bias, pre_weight, pre_bias)
        self.shape, self.device, self.dtype, self.rows, self.d, self.pre = x.shape, x.device, dtype, rows, d, pre
        self.head = (rows, d, gate_rows, code, _DTYPES[x.dtype], layer, bool(pre), small, float(residual_scale), float(eps))
        self.arrays = (self.x.data_ptr(), _p(self.y), _p(gate), _p(self.post_weight), _p(self.post_bias), _p(self.pre_weight), _p(self.pre_bias), xs, ys)

    def forward(self):
        x_new = _like(self.given_x) if self.y is not None else None
        h = self._branch() if self.pre else None
        if self.rows:
            _launch_args(_lib.load().dnag_block_norms_forward, self.index, "dnag_block_norms_forward", _lib.BLOCK_NORMS_LAYOUT, *self.head, *self.arrays,
                         _p(x_new), _p(h), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
        return x_new, h

    def _branch(self) -> torch.Tensor:
        """A new tensor of the branch's type."""
        if self.given_y is not None:
            return _like(self.given_y)
        return _like(self.given_x) if self.dtype == self.x.dtype else torch.empty(self.shape, dtype=self.dtype, device=self.device)

    def backward(self, grad_x, grad_h, wanted) -> BlockNormsGrad:
        gxs = ghs = 0
        if grad_x is not None:
            if grad_x.shape != self.shape or grad_x.dtype != self.x.dtype:
                raise ValueError(f"grad_x must be {tuple(self.shape)} of type {self.x.dtype}, got {tuple(grad_x.shape)} {grad_x.dtype}")
            grad_x, gxs = _rows2d(grad_x)
        if grad_h is not None:
            if not self.pre:
                raise ValueError("grad_h with pre=False")
            if grad_h.shape != self.shape or grad_h.dtype != self.dtype:
                raise ValueError(f"grad_h must be {tuple(self.shape)} of type {self.dtype}, got {tuple(grad_h.shape)} {grad_h.dtype}")
            grad_h, ghs = _rows2d(grad_h)
        _device(self.x, grad_x, grad_h)
        dev, rows = self.device, self.rows
        new = torch.empty_like if rows else torch.zeros_like                              # (contiguous as they are kept)
        dx = _like(self.given_x)
        dy = self._branch() if self.y is not None else None
        grads = [new(t) if t is not None and n in wanted else None for n, t in
                 zip(_SMALL, (self.gate, self.post_weight, self.post_bias, self.pre_weight, self.pre_bias))]
        if rows:
            lib = _lib.load()
            fields = (*self.head, *self.arrays, 0, 0, _p(grad_x), _p(grad_h), gxs, ghs, dx.data_ptr(), _p(dy), *map(_p, grads))
            nbytes = lib.dnag_block_norms_grad_workspace_bytes(_lib.BLOCK_NORMS_LAYOUT.pack(*fields, 0, 0, 0))
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            _launch_args(lib.dnag_block_norms_grad, self.index, "dnag_block_norms_grad", _lib.BLOCK_NORMS_LAYOUT, *fields, ws.data_ptr(), nbytes)
        return BlockNormsGrad(dx, dy, *grads)


_SMALL = ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias")


class _BlockNorms(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, post_weight, post_bias, pre_weight, pre_bias, residual_scale, norm, eps, pre, dtype):
        seam = _Seam(x, y, gate, residual_scale, post_weight, post_bias, pre_weight, pre_bias, norm, eps, pre, dtype)
        ctx.save_for_backward(x, y, gate, post_weight, post_bias, pre_weight, pre_bias)
        ctx.args = residual_scale, norm, eps, pre, dtype
        ctx.set_materialize_grads(False)
        x_new, h = seam.forward()
        return tuple(t for t in (x_new, h) if t is not None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        x, y, gate, post_weight, post_bias, pre_weight, pre_bias = ctx.saved_tensors
        residual_scale, norm, eps, pre, dtype = ctx.args
        grad_x = grads[0] if y is not None else None
        grad_h = grads[-1] if pre else None
        if grad_x is None and grad_h is None:
            return (None,) * 12
        wanted = {n for n, need in zip(_SMALL, ctx.needs_input_grad[2:7]) if need}
        g = _Seam(x, y, gate, residual_scale, post_weight, post_bias, pre_weight, pre_bias, norm, eps, pre, dtype).backward(grad_x, grad_h, wanted)
        return tuple(g) + (None,) * 5


def block_norms(x: torch.Tensor, y: Optional[torch.Tensor] = None, *, gate: Optional[torch.Tensor] = None, residual_scale: Number = 1.0,
                post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                pre_weight: Optional[torch.Tensor] = None, pre_bias: Optional[torch.Tensor] = None,
                norm: str = "rms", eps: float = 1e-6, pre: bool = True, dtype: Optional[torch.dtype] = None):
    """The seam between two blocks: ``x_new = residual_scale * x + gate * N_post(y)`` and ``h = N_pre(x_new)``; returns
    ``(x_new, h)``.

    ``x`` [..., d] is the residual stream (the branch's type, or float32 beside a 16-bit branch), ``y`` the block's output.
    ``norm``: 'rms' (no bias) or 'layer'.  ``y=None`` is the entry of the first block: ``(x, N_pre(x))``, with ``dtype`` the type of
    ``h`` (default: that of ``x``); ``pre=False`` the exit of the last one: ``(x_new, None)``.  ``h`` is computed from
    the unrounded ``x_new``.  ``gate`` has G rows ([d], [B, 1, d], the shape of ``x``, a list [G, d], ...): every
    G-th part of the rows of ``x``, in order, uses one.  A gate that broadcasting would repeat over a leading dimension ([1, N, d] or [N, d] beside
    [B, N, d]) is refused: expand it to the shape of ``x``.  Weights and gate have the branch's type or float32.  1 <= d <= 16384.  Squares are
    summed in float32: magnitudes up to 1e17."""
    tensors = (x, y, gate, post_weight, post_bias, pre_weight, pre_bias)
    _plain(*tensors)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        _leaf_mark(*tensors)
        out = _BlockNorms.apply(*tensors, residual_scale, norm, eps, pre, dtype)
        if y is None:
            return x, out[0]
        return out if pre else (out[0], None)
    x_new, h = _Seam(x, y, gate, residual_scale, post_weight, post_bias, pre_weight, pre_bias, norm, eps, pre, dtype).forward()
    return (x if y is None else x_new), h


def block_norms_grad(grad_x: Optional[torch.Tensor], grad_h: Optional[torch.Tensor], x: torch.Tensor, y: Optional[torch.Tensor] = None, *,
                     gate: Optional[torch.Tensor] = None, residual_scale: Number = 1.0, post_weight: Optional[torch.Tensor] = None,
                     post_bias: Optional[torch.Tensor] = None, pre_weight: Optional[torch.Tensor] = None,
                     pre_bias: Optional[torch.Tensor] = None, norm: str = "rms", eps: float = 1e-6, pre: bool = True,
                     dtype: Optional[torch.dtype] = None) -> BlockNormsGrad:
    """Gradients of ``block_norms`` (same arguments) for ``grad_x`` and ``grad_h``, the gradients of ``x_new`` and ``h`` (None: zero).
    Nothing of the forward pass but its inputs is needed.  Sums over rows run in one fixed order."""
    _plain(grad_x, grad_h, x, y, gate, post_weight, post_bias, pre_weight, pre_bias)
    seam = _Seam(x, y, gate, residual_scale, post_weight, post_bias, pre_weight, pre_bias, norm, eps, pre, dtype)
    return seam.backward(grad_x, grad_h, _SMALL)


# ---------------------------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------------------------
class _Distill:
    """The checked arguments of one distillation call as the library takes them."""

    def __init__(self, logits, teacher_ids, teacher_logits, temperature, row_weight, reduction):
        if logits.dim() < 1 or logits.shape[-1] < 1:
            raise ValueError(f"logits must be [..., vocab], got {tuple(logits.shape)}")
        if teacher_ids.shape != teacher_logits.shape or teacher_ids.dim() != logits.dim() or teacher_ids.shape[:-1] != logits.shape[:-1]:
            raise ValueError(f"teacher_ids {tuple(teacher_ids.shape)} and teacher_logits {tuple(teacher_logits.shape)} must be "
                             f"[..., k] beside logits {tuple(logits.shape)}")
        if not 1 <= teacher_ids.shape[-1] <= 1024:
            raise ValueError(f"k={teacher_ids.shape[-1]} teacher entries; 1 to 1024 are built")
        if reduction not in _REDUCE:
            raise ValueError(f"reduction={reduction!r}: 'none', 'sum' and 'mean' are built")
        least = 0.1 if logits.dtype == torch.float16 else 1e-6
        if not least <= temperature <= 1e6:
            raise ValueError(f"temperature={temperature} is outside {least} .. 1e6 ({logits.dtype} logits)")
        if teacher_ids.dtype not in _IDS:
            raise ValueError(f"teacher_ids have dtype {teacher_ids.dtype}; int32 and int64 are built")
        self.lead = logits.shape[:-1]
        if row_weight is not None and (row_weight.shape != self.lead or row_weight.dtype != torch.float32):
            raise ValueError(f"row_weight must be {tuple(self.lead)} float32, got {tuple(row_weight.shape)} {row_weight.dtype}")
        code, tcode = _dtype(logits, "logits"), _dtype(teacher_logits, "teacher_logits")
        self.index, self.device, self.reduction = _device(logits, teacher_ids, teacher_logits, row_weight), logits.device, reduction
        self.given = logits
        self.logits, stride = _rows2d(logits)
        self.rows, self.V = self.logits.shape
        self.kept = (teacher_ids.contiguous(), teacher_logits.contiguous(), None if row_weight is None else row_weight.contiguous())
        self.head = (self.rows, self.V, stride, teacher_ids.shape[-1], code, tcode, _IDS[teacher_ids.dtype], _REDUCE[reduction], float(temperature),
                     self.logits.data_ptr(), *map(_p, self.kept))

    def _call(self, fn: str, loss, stats, grad_out, grad) -> None:
        lib = _lib.load()
        fields = (*self.head, _p(loss), _p(stats), _p(grad_out), _p(grad))
        nbytes = lib.dnag_distill_workspace_bytes(_lib.DISTILL_LAYOUT.pack(*fields, 0, 0, 0))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        _launch_args(getattr(lib, fn), self.index, fn, _lib.DISTILL_LAYOUT, *fields, ws.data_ptr(), nbytes)

    def loss(self, stats: bool = False, grad: bool = False):
        none = self.reduction == "none"
        loss = (torch.empty if self.rows else torch.zeros)(self.lead if none else (), dtype=torch.float32, device=self.device)
        st = torch.empty(self.rows, 2, dtype=torch.float32, device=self.device) if stats else None
        g = _like(self.given) if grad else None
        if self.rows:
            self._call("dnag_distill_loss_grad" if grad else "dnag_distill_loss", loss, st, None, g)
        return loss, st, g

    def backward(self, stats, grad_out):
        g = _like(self.given)
        if self.rows:
            self._call("dnag_distill_backward", None, stats, grad_out.to(torch.float32).contiguous(), g)
        return g


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_ids, teacher_logits, temperature, row_weight, reduction):
        loss, stats, _ = _Distill(logits, teacher_ids, teacher_logits, temperature, row_weight, reduction).loss(stats=True)
        ctx.save_for_backward(logits, teacher_ids, teacher_logits, row_weight, stats)
        ctx.args = temperature, reduction
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        logits, teacher_ids, teacher_logits, row_weight, stats = ctx.saved_tensors
        temperature, reduction = ctx.args
        return (_Distill(logits, teacher_ids, teacher_logits, temperature, row_weight, reduction).backward(stats, grad_out),) + (None,) * 5


def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *, temperature: Number = 1.0,
                 row_weight: Optional[torch.Tensor] = None, reduction: str = "mean") -> torch.Tensor:
    """``tau^2 KL(p || q)`` for each row of ``logits`` [..., vocab]: ``q`` the student's distribution at temperature ``tau`` over the
    whole vocabulary, ``p`` the teacher's over its k listed tokens, ``softmax(teacher_logits / tau)``.

    ``teacher_ids`` [..., k] outside ``0 .. vocab - 1`` are no entries (a row shorter than k is filled with -1); repeated ids add up.
    ``row_weight`` [...] float32: rows whose weight is not positive (padding) count nothing and their logits do not
    matter, NaN included.  A row without entries counts 0.  ``reduction``: 'mean' over the positive weights (over all rows
    without weights; 0 where there are none), 'sum', or 'none' (weighted loss of each row).  float32.  ``logits`` masked with -inf
    or their type's lowest value have no probability (a row of nothing but lowest values: one and the same probability).
    ``temperature`` is 1e-6 to 1e6 (float16 logits: from 0.1 on); a row's loss is a difference of float32 logarithms, off by a few
    1e-6 ``temperature``^2 however small it is.  No gradient reaches the
    teacher or the weights: they must not require one."""
    _plain(logits, teacher_logits, row_weight)
    if teacher_logits.requires_grad or (row_weight is not None and row_weight.requires_grad):
        raise ValueError("distill_loss has no gradient for teacher_logits and row_weight: detach them")
    if logits.requires_grad and torch.is_grad_enabled():
        _leaf_mark(logits)
        return _DistillLoss.apply(logits, teacher_ids, teacher_logits, temperature, row_weight, reduction)
    return _Distill(logits, teacher_ids, teacher_logits, temperature, row_weight, reduction).loss()[0]


def distill_loss_and_grad(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *, temperature: Number = 1.0,
                          row_weight: Optional[torch.Tensor] = None, reduction: str = "mean"):
    """``distill_loss`` and its gradient with respect to ``logits`` (for an upstream gradient of 1) in one pass over the logits: two
    thirds of the memory traffic of the loss followed by its backward pass.  Returns ``(loss, grad)``."""
    _plain(logits, teacher_logits, row_weight)
    loss, _, grad = _Distill(logits, teacher_ids, teacher_logits, temperature, row_weight, reduction).loss(grad=True)
    return loss, grad


# ---------------------------------------------------------------------------------------------------------------
# drawing
# ---------------------------------------------------------------------------------------------------------------
def sample_tokens(logits: torch.Tensor, u: torch.Tensor, *, temperature: Union[Number, torch.Tensor] = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: Union[Number, torch.Tensor] = 1.0,
                  min_p: Union[Number, torch.Tensor] = 0.0) -> torch.Tensor:
    """One token per row of ``logits`` [..., vocab] (int64 [...]), drawn with the uniform numbers ``u`` [...] (float32, [0, 1)).

    Order of the filters: ``temperature`` (<= 0: the largest logit), ``top_k`` (<= 0: off), ``top_p`` on what top-k left (>= 1: off,
    at least one token stays), ``min_p`` relative to the largest probability (the largest stays).  Equal logits rank by
    index.  The token is the first one, in index order, whose running sum of kept probability exceeds ``u`` times the total.
    NaN and -inf are never drawn; a row of nothing else gives -1.  Each setting is a number, or a tensor with a value per
    row (float32; int32 for ``top_k``).  The same inputs give the same tokens, whatever else runs.  vocab <= 2^20."""
    _plain()                                           # tokens have no derivative
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [..., vocab], got {tuple(logits.shape)}")
    lead = logits.shape[:-1]
    if u.shape != lead or u.dtype != torch.float32:
        raise ValueError(f"u must be {tuple(lead)} float32, got {tuple(u.shape)} {u.dtype}")
    code = _dtype(logits, "logits")
    numbers, rows = [], []
    for name, value, kind in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                              ("min_p", min_p, torch.float32)):
        if isinstance(value, torch.Tensor):
            if value.shape != lead or value.dtype != kind:
                raise ValueError(f"{name} must be a number or {tuple(lead)} {kind}, got {tuple(value.shape)} {value.dtype}")
            rows.append(value.contiguous())
            numbers.append(0)
        else:
            if not -_MOST <= value <= _MOST:
                raise ValueError(f"{name}={value} must be finite")
            rows.append(None)
            numbers.append(value)
    index = _device(logits, u, *rows)
    lg, stride = _rows2d(logits)
    uc = u.contiguous()
    out = torch.empty_like(uc, dtype=torch.int64)
    n, V = lg.shape
    if n:
        t, k, p, q = numbers
        lib = _lib.load()
        fields = (n, V, stride, code, max(-1, min(int(k), 0x7fffffff)), t, p, q, lg.data_ptr(), uc.data_ptr(), *map(_p, rows), out.data_ptr())
        nbytes = lib.dnag_sample_workspace_bytes(_lib.SAMPLE_LAYOUT.pack(*fields, 0, 0, 0))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=out.device) if nbytes else None
        _launch_args(lib.dnag_sample_tokens, index, "dnag_sample_tokens", _lib.SAMPLE_LAYOUT, *fields, _p(ws), nbytes)
    return out
