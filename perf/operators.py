"""What is measured of the token operators (``diffusionnag_amd.token_ops``), with their plain forms.

The four operators stand around the blocks of a network over tokens -- architecture nodes here, any vocabulary in
general: the embedding lookup with its gradient, the norms after and before a block with the block's gate and the
residual scale, the distillation loss against a teacher's top logits, and drawing tokens from logits.

``own = False``: ``run`` computes an operator in elementary torch operations; ``own = True``: it calls the framework.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the tokens of one serving step: 64 requests look up one token each; latency counts
        dict(name="embed_decode", op="embed", grad=False, rows=64, vocab=32000, dim=2048, dtype="bf16", zipf=True, pad=0.0),
        # a prompt batch, padded at its end
        dict(name="embed_prompt", op="embed", grad=False, rows=16384, vocab=64000, dim=4096, dtype="bf16", zipf=True, pad=0.05),
        # 4096 graphs of 8 nodes over 7 node types, the widths of the NAS-Bench-201 score network: every type is hot
        dict(name="embed_grad_nodes", op="embed", grad=True, rows=32768, vocab=7, dim=64, dtype="f32", zipf=False, pad=0.0),
        # a training batch over a large vocabulary with a natural (Zipf) distribution and padded sequences
        dict(name="embed_grad_train", op="embed", grad=True, rows=32768, vocab=64000, dim=2048, dtype="bf16", zipf=True, pad=0.05),
        # a serving step of 16 requests: one block's exit and the next block's entry
        dict(name="block_decode", op="block", grad=False, rows=16, dim=4096, groups=1, xtype="bf16", dtype="bf16", norm="rms", pre=True),
        # a long prompt batch of the same block
        dict(name="block_prompt", op="block", grad=False, rows=16384, dim=4096, groups=1, xtype="bf16", dtype="bf16", norm="rms", pre=True),
        # 4096 graphs of 8 nodes at the score network's width, LayerNorm, a gate per graph (from its time condition)
        dict(name="block_grad_nodes", op="block", grad=True, rows=32768, dim=64, groups=4096, xtype="f32", dtype="f32", norm="layer", pre=True),
        # a training batch: residual stream in 32 bits beside a 16-bit branch, 16 sequences with a gate each
        dict(name="block_grad_train", op="block", grad=True, rows=16384, dim=2048, groups=16, xtype="f32", dtype="bf16", norm="rms", pre=True),
        # evaluation of a student over an odd vocabulary, loss for each token
        dict(name="distill_eval", op="distill", grad=False, rows=1000, vocab=50001, k=20, dtype="f16", tau=1.0, masked=0.1),
        # a training batch: loss and gradient of the student's logits
        dict(name="distill_train", op="distill", grad=True, rows=8192, vocab=32000, k=64, dtype="bf16", tau=2.0, masked=0.1),
        # one request over a large vocabulary: the latency of a serving step
        dict(name="sample_one", op="sample", rows=1, vocab=128000, dtype="bf16", per_row=False, temperature=0.8, top_k=50, top_p=0.95, min_p=0.0, masked=0.0),
        # 256 requests with settings of their own, no top-k: the nucleus comes from the whole vocabulary
        dict(name="sample_batch", op="sample", rows=256, vocab=128000, dtype="bf16", per_row=True, temperature=0.9, top_k=0, top_p=0.9, min_p=0.02, masked=0.05),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    d = _log_int(rng, lo, hi)
    return max(lo, d // 64 * 64) if rng.random() < 0.5 and d >= 64 else d


def draw(rng):
    op = rng.choice(["embed", "block", "distill", "sample"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "embed":
        while True:
            rows, vocab, dim = _log_int(rng, 1, 65536), _log_int(rng, 7, 262144), _width(rng, 32, 8192)
            if (rows + vocab) * dim * (2 if dtype == "f32" else 1) <= 190_000_000:
                return dict(op=op, grad=rng.random() < 0.6, rows=rows, vocab=vocab, dim=dim, dtype=dtype, zipf=rng.random() < 0.7,
                            pad=rng.choice([0.0, 0.05, 0.3]))
    if op == "block":
        while True:
            groups, each, dim = _log_int(rng, 1, 4096), _log_int(rng, 1, 65536), _width(rng, 32, 16384)
            rows = groups * each
            if rows <= 65536 and rows * dim * (2 if dtype == "f32" else 1) <= 33_000_000:
                return dict(op=op, grad=rng.random() < 0.5, rows=rows, dim=dim, groups=groups, xtype=rng.choice([dtype, "f32"]), dtype=dtype,
                            norm=rng.choice(["rms", "layer"]), pre=rng.random() < 0.8)
    if op == "distill":
        while True:
            rows, vocab = _log_int(rng, 1, 65536), _log_int(rng, 7, 200000)
            if rows * vocab * (2 if dtype == "f32" else 1) <= 260_000_000:
                return dict(op=op, grad=rng.random() < 0.6, rows=rows, vocab=vocab, k=_log_int(rng, 1, min(vocab, 128)), dtype=dtype,
                            tau=round(rng.uniform(0.7, 4.0), 2), masked=rng.choice([0.0, 0.1, 0.5]))
    while True:
        rows, vocab = _log_int(rng, 1, 65536), _log_int(rng, 2, 200000)
        if rows * vocab <= 32_000_000:
            return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, per_row=rng.random() < 0.5, temperature=round(rng.uniform(0.3, 1.5), 2),
                        top_k=rng.choice([0, 0, 1, _log_int(rng, 2, 1000)]), top_p=rng.choice([1.0, round(rng.uniform(0.1, 0.99), 2)]),
                        min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.2), 3)]), masked=rng.choice([0.0, 0.05, 0.9]))


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    s = dict(case)
    if case["op"] == "embed":
        T, V, d = case["rows"], case["vocab"], case["dim"]
        u = uniform(T)
        ids = (torch.exp(u * math.log(V + 1)) - 1).long() if case["zipf"] else (u * V).long()
        ids = ids.clamp_(0, V - 1)
        npad = int(T * case["pad"])
        if npad:
            ids[T - npad:] = -1                        # the end of a padded batch
        s["ids"], s["scale"] = ids, math.sqrt(d)       # the score network scales its embedding by sqrt(d) too
        if case["grad"]:
            s["dout"] = normal(T, d)
        else:
            s["weight"] = normal(V, d, std=0.02)
    elif case["op"] == "block":
        T, d, G = case["rows"], case["dim"], case["groups"]
        xt = DTYPES[case["xtype"]]
        s["x"], s["y"] = normal(T, d, std=2.0, dtype=xt), normal(T, d)
        s["gate"] = normal(G, d, std=0.5) + 0.5
        s["post_weight"], s["pre_weight"] = 1 + normal(d, std=0.1), 1 + normal(d, std=0.1)
        s["post_bias"] = s["pre_bias"] = None
        if case["norm"] == "layer":
            s["post_bias"], s["pre_bias"] = normal(d, std=0.1), normal(d, std=0.1)
        if not case["pre"]:
            s["pre_weight"] = s["pre_bias"] = None
        s["residual_scale"], s["eps"] = 0.875, 1e-6
        if case["grad"]:
            s["grad_x"] = normal(T, d, dtype=xt)
            s["grad_h"] = normal(T, d) if case["pre"] else None
    elif case["op"] == "distill":
        T, V, K = case["rows"], case["vocab"], case["k"]
        s["logits"] = normal(T, V, std=2.5)
        # a teacher's top entries: distinct tokens, falling logits, rows with fewer entries than K filled with -1
        first, step = (uniform(T, 1) * V).long(), max(1, V // K)
        s["teacher_ids"] = (first + torch.arange(K, device=DEV) * step) % V
        s["teacher_logits"] = torch.sort(normal(T, K, std=2.5, dtype=torch.float32) + 4, dim=1, descending=True).values
        short = uniform(T) < 0.2
        s["teacher_ids"][short, (K + 1) // 2:] = -1
        s["row_weight"] = (uniform(T) >= case["masked"]).float()
    else:
        T, V = case["rows"], case["vocab"]
        x = torch.randn(T, V, generator=g, device=DEV) * 2.5
        if case["masked"]:
            x = torch.where(uniform(T, V) < case["masked"], float("-inf"), x)
            x[:, 0] = 0.0
        s["logits"], s["u"] = x.to(dt), uniform(T)
        if case["per_row"]:
            s["temperature"] = case["temperature"] * (0.75 + 0.5 * uniform(T))
            s["top_k"] = (case["top_k"] * (0.5 + uniform(T))).int() if case["top_k"] else torch.zeros(T, dtype=torch.int32, device=DEV)
            s["top_p"] = (case["top_p"] * (0.9 + 0.2 * uniform(T))).clamp(max=1.0)
            s["min_p"] = case["min_p"] * uniform(T)
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        if s["op"] == "embed":
            return _plain_embed_grad(s) if s["grad"] else _plain_embed(s)
        if s["op"] == "block":
            return _plain_block_grad(s) if s["grad"] else _plain_block(s)
        if s["op"] == "distill":
            return _plain_distill(s)
        return _plain_sample(s)


def _own(s):
    from diffusionnag_amd import token_ops as ops
    if s["op"] == "embed":
        if s["grad"]:
            return ops.embed_tokens_grad(s["dout"], s["ids"], s["vocab"], scale=s["scale"])
        return ops.embed_tokens(s["ids"], s["weight"], scale=s["scale"])
    if s["op"] == "block":
        kw = dict(gate=s["gate"], residual_scale=s["residual_scale"], post_weight=s["post_weight"], post_bias=s["post_bias"],
                  pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], norm=s["norm"], eps=s["eps"], pre=s["pre"])
        if s["grad"]:
            g = ops.block_norms_grad(s["grad_x"], s["grad_h"], s["x"], s["y"], **kw)
            return {k: v for k, v in g._asdict().items() if v is not None}
        x_new, h = ops.block_norms(s["x"], s["y"], **kw)
        return {"x_new": x_new, "h": h} if s["pre"] else {"x_new": x_new}
    if s["op"] == "distill":
        args = (s["logits"], s["teacher_ids"], s["teacher_logits"])
        if s["grad"]:
            loss, grad = ops.distill_loss_and_grad(*args, temperature=s["tau"], row_weight=s["row_weight"], reduction="mean")
            return {"loss": loss, "grad": grad}
        return ops.distill_loss(*args, temperature=s["tau"], row_weight=s["row_weight"], reduction="none")
    return ops.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


def _plain_embed(s):
    ids, w = s["ids"], s["weight"]
    real = (ids >= 0) & (ids < w.shape[0])
    rows = w[torch.where(real, ids, 0)].float() * s["scale"]
    return torch.where(real[:, None], rows, 0.0).to(w.dtype)


def _plain_embed_grad(s):
    ids, dout, V = s["ids"], s["dout"], s["vocab"]
    real = (ids >= 0) & (ids < V)
    out = torch.zeros(V + 1, dout.shape[1], device=dout.device)
    out.index_add_(0, torch.where(real, ids, V), dout.float())
    return (out[:V] * s["scale"]).to(dout.dtype)


def _norm_parts(v, norm, eps):
    mean = v.mean(1, keepdim=True) if norm == "layer" else 0.0
    c = v - mean
    r = torch.rsqrt((c * c).mean(1, keepdim=True) + eps)
    return c * r, r


def _per_row(gate, rows):
    return gate.float().repeat_interleave(rows // gate.shape[0], 0) if gate.shape[0] > 1 else gate.float()


def _affine(v, w, b):
    v = v * w.float()
    return v if b is None else v + b.float()


def _plain_block(s):
    x, y = s["x"], s["y"]
    yhat, _ = _norm_parts(y.float(), s["norm"], s["eps"])
    new = x.float() * s["residual_scale"] + _per_row(s["gate"], x.shape[0]) * _affine(yhat, s["post_weight"], s["post_bias"])
    out = {"x_new": new.to(x.dtype)}
    if s["pre"]:
        xhat, _ = _norm_parts(new, s["norm"], s["eps"])
        out["h"] = _affine(xhat, s["pre_weight"], s["pre_bias"]).to(y.dtype)
    return out


def _norm_back(dhat, hat, r, norm):
    d = dhat - hat * (dhat * hat).mean(1, keepdim=True)
    if norm == "layer":
        d = d - dhat.mean(1, keepdim=True)
    return d * r


def _plain_block_grad(s):
    x, y, rows = s["x"], s["y"], s["x"].shape[0]
    gate = _per_row(s["gate"], rows)
    yhat, ry = _norm_parts(y.float(), s["norm"], s["eps"])
    n = _affine(yhat, s["post_weight"], s["post_bias"])
    dnew = s["grad_x"].float()
    out = {}
    if s["pre"]:
        xhat, rx = _norm_parts(x.float() * s["residual_scale"] + gate * n, s["norm"], s["eps"])
        dh = s["grad_h"].float()
        dnew = dnew + _norm_back(dh * s["pre_weight"].float(), xhat, rx, s["norm"])
        out["pre_weight"] = (dh * xhat).sum(0).to(s["pre_weight"].dtype)
        if s["pre_bias"] is not None:
            out["pre_bias"] = dh.sum(0).to(s["pre_bias"].dtype)
    out["x"] = (dnew * s["residual_scale"]).to(x.dtype)
    G = s["gate"].shape[0]
    out["gate"] = (dnew * n).view(G, rows // G, -1).sum(1).to(s["gate"].dtype)
    dn = dnew * gate
    out["post_weight"] = (dn * yhat).sum(0).to(s["post_weight"].dtype)
    if s["post_bias"] is not None:
        out["post_bias"] = dn.sum(0).to(s["post_bias"].dtype)
    out["y"] = _norm_back(dn * s["post_weight"].float(), yhat, ry, s["norm"]).to(y.dtype)
    return out


def _plain_distill(s):
    tau, w, ids = s["tau"], s["row_weight"], s["teacher_ids"]
    z = s["logits"].float() / tau
    top = z.max(1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    real = (ids >= 0) & (ids < z.shape[1])
    t = torch.where(real, s["teacher_logits"].float() / tau, float("-inf"))
    tmax = t.max(1, keepdim=True).values
    some = torch.isfinite(tmax)
    te = torch.where(real, torch.exp(t - torch.where(some, tmax, 0.0)), 0.0)
    p = te / te.sum(1, keepdim=True).clamp(min=1e-30)
    at = torch.where(real, ids, 0)
    logq = z.gather(1, at) - top - torch.log(total)
    terms = torch.where(p > 0, p * (torch.log(p) - logq), 0.0)
    loss = torch.where(w > 0, tau * tau * w * terms.sum(1), 0.0)
    if not s["grad"]:
        return loss
    denominator = w.sum().clamp(min=1e-30)
    c = torch.where(some[:, 0], w, 0.0) * tau / denominator
    grad = e.div_(total).mul_(c[:, None])
    grad.scatter_add_(1, at, -p * c[:, None])
    return {"loss": loss.sum() / denominator, "grad": grad.to(s["logits"].dtype)}


def _plain_sample(s):
    # in 64 bits: the token changes where a sum passes a border
    V = s["logits"].shape[1]

    def column(v):
        return v.double()[:, None] if torch.is_tensor(v) else torch.full((1, 1), float(v), device=DEV, dtype=torch.float64)

    x = s["logits"].double()
    top = x.max(1, keepdim=True).values
    order = torch.sort(x, dim=1, descending=True, stable=True)
    e = torch.exp((order.values - top) / column(s["temperature"]))
    k = column(s["top_k"])
    place = torch.arange(V, device=DEV)[None]
    kept = (place < k) | (k <= 0)
    e = torch.where(kept, e, 0.0)
    before = torch.cumsum(e, 1) - e
    p = column(s["top_p"])
    kept = kept & ((before < p * e.sum(1, keepdim=True)) | (p >= 1) | (place == 0)) & ((e >= column(s["min_p"])) | (place == 0))
    e = torch.zeros_like(e).scatter_(1, order.indices, torch.where(kept, e, 0.0))
    sums = torch.cumsum(e, 1)
    return (sums <= s["u"].double()[:, None] * sums[:, -1:]).sum(1)


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        ids, V = s["ids"], case["vocab"]
        at = torch.nonzero((ids >= 0) & (ids < V))[:, 0]
        if case["grad"]:
            out = torch.zeros(V, case["dim"], dtype=torch.float64, device=DEV)
            return out.index_put_((ids[at],), s["dout"].double()[at] * s["scale"], accumulate=True)
        out = torch.zeros(case["rows"], case["dim"], dtype=torch.float64, device=DEV)
        out[at] = s["weight"].double()[ids[at]] * s["scale"]
        return out
    if case["op"] == "block":
        return _exact_block(case, s)
    if case["op"] == "distill":
        return _exact_distill(case, s)
    return None                                        # tokens: whole numbers


def _exact_block(case, s):
    names = ("x", "y", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias")
    v = {n: s[n].double().requires_grad_(case["grad"]) for n in names if s[n] is not None}

    def normed(a, which):
        centred = a - a.sum(1, keepdim=True) / a.shape[1] if case["norm"] == "layer" else a
        size = torch.sqrt(centred.pow(2).sum(1, keepdim=True) / a.shape[1] + s["eps"])
        out = centred / size * v[which + "_weight"]
        return out + v[which + "_bias"] if which + "_bias" in v else out

    branch = normed(v["y"], "post").reshape(case["groups"], -1, case["dim"]) * v["gate"][:, None, :]
    new = s["residual_scale"] * v["x"] + branch.reshape(case["rows"], case["dim"])
    outs = {"x_new": new}
    if case["pre"]:
        outs["h"] = normed(new, "pre")
    if not case["grad"]:
        return outs
    back = [s["grad_x"].double()] + ([s["grad_h"].double()] if case["pre"] else [])
    grads = torch.autograd.grad(list(outs.values()), list(v.values()), back)
    return dict(zip(v, grads))


def _exact_distill(case, s):
    V, tau = case["vocab"], case["tau"]
    loss = torch.zeros(case["rows"], dtype=torch.float64, device=DEV)
    grad = torch.zeros(case["rows"], V, dtype=torch.float64, device=DEV) if case["grad"] else None
    total = float(s["row_weight"].double().sum())
    step = max(1, 40_000_000 // V)
    for a in range(0, case["rows"], step):
        z = s["logits"][a:a + step].double() / tau
        logq = torch.log_softmax(z, 1)
        w, ids = s["row_weight"][a:a + step].double(), s["teacher_ids"][a:a + step]
        inside = (ids >= 0) & (ids < V)
        logp = torch.log_softmax((s["teacher_logits"][a:a + step].double() / tau).masked_fill(~inside, -1e300), 1)
        p = logp.exp() * inside
        spread = torch.zeros_like(z).scatter_add_(1, ids.clamp(0, V - 1), p)
        loss[a:a + step] = w * tau ** 2 * ((p * logp.clamp(min=-1e5)).sum(1) - (spread * logq).sum(1)) * inside.any(1)
        if case["grad"]:
            grad[a:a + step] = (w * inside.any(1))[:, None] * tau * (logq.exp() - spread) / max(total, 1e-300)
    if case["grad"]:
        return {"loss": loss.sum() / max(total, 1e-300), "grad": grad}
    return loss


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "embed":
        T, V, d = case["rows"], case["vocab"], case["dim"]
        if case["grad"]:
            return {"bytes": 8 * T + e * d * (T + V), "flops": 2 * T * d}
        return {"bytes": 8 * T + e * d * (T + min(T, V)), "flops": T * d}
    if case["op"] == "block":
        n, ex = case["rows"] * case["dim"], 4 if case["xtype"] == "f32" else 2
        h = 1 if case["pre"] else 0
        small = e * case["dim"] * (case["groups"] + 4)
        if case["grad"]:
            return {"bytes": n * (3 * ex + (2 + h) * e) + 2 * small, "flops": 40 * n}
        return {"bytes": n * (2 * ex + (1 + h) * e) + small, "flops": 12 * n}
    n = case["rows"] * case["vocab"]
    if case["op"] == "distill":
        rest = case["rows"] * (12 * case["k"] + 8)
        return {"bytes": n * e * (2 if case["grad"] else 1) + rest, "flops": n * (7 if case["grad"] else 4)}
    return {"bytes": n * e + 28 * case["rows"], "flops": 6 * n}


