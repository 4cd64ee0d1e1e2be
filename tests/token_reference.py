"""The token operators in 64 bits on the CPU, written from their formulas (the oracle of ``diffusionnag_amd.token_ops``)."""

import numpy as np
import torch


def half_step(dtype):
    """Half a rounding step relative to the value, and the half step of the type's smallest numbers."""
    return torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


U32 = 2.0 ** -24


def embed(ids, weight, scale):
    w, ids = weight.double(), ids.long()
    real = (ids >= 0) & (ids < w.shape[0])
    return scale * w[torch.where(real, ids, 0)] * real.unsqueeze(-1)


def embed_grad(ids, grad, num_tokens, scale, padding_idx=None):
    """(gradient, sum of magnitudes, count) by token."""
    ids, g = ids.long().reshape(-1), grad.double().reshape(-1, grad.shape[-1])
    out, mag, n = torch.zeros(num_tokens, g.shape[1]).double(), torch.zeros(num_tokens, g.shape[1]).double(), torch.zeros(num_tokens, 1).double()
    for t, v in enumerate(ids.tolist()):
        if 0 <= v < num_tokens and v != padding_idx:
            out[v] += g[t]
            mag[v] += g[t].abs()
            n[v] += 1
    return out * scale, mag * abs(scale), n


def norm(v, w, b, kind, eps):
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    out = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    if w is not None:
        out = out * w
    return out if b is None else out + b


def block_norms(t, residual_scale, kind, eps, pre):
    """``t``: dict of float64 tensors x [rows, d], y, gate [G, d], post_weight, ... (None where absent) -> (x_new, h)."""
    x = t["x"]
    if t.get("y") is not None:
        n = norm(t["y"], t.get("post_weight"), t.get("post_bias"), kind, eps)
        if t.get("gate") is not None:
            g = t["gate"]
            n = (n.reshape(g.shape[0], -1, g.shape[1]) * g[:, None, :]).reshape(x.shape)
        x = residual_scale * x + n
    return x, norm(x, t.get("pre_weight"), t.get("pre_bias"), kind, eps) if pre else None


def distill_rows(logits, ids, tlogits, tau, weight):
    """Weighted loss of each row, differentiable in ``logits`` (float64)."""
    out = []
    for r in range(logits.shape[0]):
        real = [(int(i), k) for k, i in enumerate(ids[r].tolist()) if 0 <= int(i) < logits.shape[1] and float(tlogits[r, k]) > -np.inf]
        w = 1.0 if weight is None else float(weight[r])
        if not real or not w > 0:
            out.append(logits[r].new_zeros(()))
            continue
        logp = torch.log_softmax(torch.tensor([float(tlogits[r, k]) / tau for _, k in real], dtype=torch.float64), 0)
        logq = torch.log_softmax(logits[r] / tau, 0)
        out.append(w * tau * tau * sum(p.exp() * (p - logq[i]) for p, (i, _) in zip(logp, real)))
    return torch.stack(out)


def distill(logits, ids, tlogits, tau, weight, reduction):
    """(loss, gradient) in float64."""
    x = logits.double().clone()
    if weight is not None:
        x[~(weight > 0)] = 0.0                     # rows that do not count may hold anything
    x.requires_grad_(True)
    rows = distill_rows(x, ids, tlogits, tau, weight)
    total = rows.sum()
    if reduction == "mean":
        n = float(x.shape[0]) if weight is None else float(weight.double().clamp(min=0).sum())
        total = total / n if n > 0 else total * 0
    (g,) = torch.autograd.grad(total, x)
    return (rows if reduction == "none" else total).detach(), g


def sample_row(logits, u, temperature, top_k, top_p, min_p):
    """One row by sorting, float64."""
    x = np.asarray(logits, np.float64) + 0.0
    x[np.isnan(x)] = -np.inf
    m = x.max() if len(x) else -np.inf
    if m == -np.inf:
        return -1
    order = np.lexsort((np.arange(len(x)), -x))     # falling logits, rising index
    if not temperature > 0:
        return int(order[0])
    live = order[x[order] > -np.inf]
    if top_k > 0:
        live = live[:top_k]
    with np.errstate(invalid="ignore"):
        e = np.where(x[live] == m, 1.0, np.exp((x[live] - m) / temperature))
    if top_p < 1:
        before = np.cumsum(e) - e
        n = max(1, int((before < top_p * e.sum()).sum()))
        live, e = live[:n], e[:n]
    keep = e >= min_p
    keep[0] = True
    live, e = live[keep], e[keep]
    by_index = np.argsort(live)
    live, e = live[by_index], e[by_index]
    sums = np.cumsum(e)
    return int(live[min(int((sums <= u * sums[-1]).sum()), len(live) - 1)])
