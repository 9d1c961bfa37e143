"""Measured cases of the class-target operators: softmax cross entropy of a linear head with
its gradients, and the global gradient norm with clipping.

A case is a dict of plain values.  op "xent": logits z = x w^T + bias over n rows, d features and
c classes; mode "loss" returns the rows' losses, "step" the losses with the gradients of w and bias
(the features are data), "train" also the gradient of x, through autograd.  op "clip": the 2-norm
over a list of gradient tensors and the gradients scaled to a largest norm; mode "norm" stops at
the norm.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------ cases ----
def listed():
    return [
        # the README's 1,000 x 50 table with a binary target: one step of a fit, latency
        dict(name="step 1000x50 c2", op="xent", mode="step", n=1000, d=50, c=2, type="fp32",
             columns=True, left_out=0.0),
        # the 1e6 x 256 table, binary target, features resident column by column
        dict(name="step 1e6x256 c2", op="xent", mode="step", n=1_000_000, d=256, c=2, type="fp32",
             columns=True, left_out=0.0),
        # the 4e6 x 128 table with its three classes; a tenth of the rows held out
        dict(name="step 4e6x128 c3", op="xent", mode="step", n=4_000_000, d=128, c=3, type="fp32",
             columns=True, left_out=0.1),
        # scoring a wide table (2048 features, rows in numpy's order) against a fitted head
        dict(name="loss 300001x2048 c5", op="xent", mode="loss", n=300_001, d=2048, c=5, type="fp32",
             columns=False, left_out=0.0),
        # a regression target cut into 255 bins
        dict(name="step 120000x100 c255", op="xent", mode="step", n=120_000, d=100, c=255, type="fp32",
             columns=True, left_out=0.0),
        # a categorical column of cardinality 1000 as the target, features from a layer below
        dict(name="train 200000x256 c1000", op="xent", mode="train", n=200_000, d=256, c=1000,
             type="fp32", columns=False, left_out=0.05),
        # a large vocabulary in 16 bits: one training step's token batch, a fifth of it padding
        dict(name="train 8192x1024 c32768 bf16", op="xent", mode="train", n=8192, d=1024, c=32768,
             type="bf16", columns=False, left_out=0.2),
        # one row against a large vocabulary
        dict(name="loss 1x1000 c50000 bf16", op="xent", mode="loss", n=1, d=1000, c=50_000, type="bf16",
             columns=False, left_out=0.0),
        # nothing aligned: odd rows, features and classes
        dict(name="train 4097x333 c10007 fp16", op="xent", mode="train", n=4097, d=333, c=10_007,
             type="fp16", columns=False, left_out=0.3),
        # the two tensors of a small head: latency
        dict(name="clip 2 tensors", op="clip", mode="clip", tensors=2, total=1028, type="fp32"),
        # a model of many ragged tensors, in 16 and 32 bits
        dict(name="clip 401 tensors mixed", op="clip", mode="clip", tensors=401, total=200_000_000,
             type="mixed"),
        # the norm alone, over one large embedding gradient and its neighbours
        dict(name="norm 9 tensors fp32", op="clip", mode="norm", tensors=9, total=500_000_000, type="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["table", "table", "classes", "classes", "clip"])
    if kind == "clip":
        return dict(op="clip", mode=rng.choice(["clip", "clip", "norm"]), tensors=_log(rng, 1, 600),
                    total=_log(rng, 1000, 200_000_000), type=rng.choice(["fp32", "bf16", "fp16", "mixed"]))
    left_out = rng.choice([0.0, 0.0, 0.1, 0.5])
    mode = rng.choice(["loss", "step", "train"])
    if kind == "table":
        d, c = _log(rng, 1, 2048), rng.randint(2, 16)
        n = min(_log(rng, 50, 2_000_000), 500_000_000 // d)
        return dict(op="xent", mode=mode, n=n, d=d, c=c, type=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                    columns=rng.random() < 0.5, left_out=left_out)
    d, c = _log(rng, 8, 2048), _log(rng, 17, 50_000)
    n = max(1, min(_log(rng, 1, 200_000), 250_000_000 // c, 250_000_000 // d, int(2.5e11 / (d * c))))
    return dict(op="xent", mode=mode, n=n, d=d, c=c, type=rng.choice(["fp32", "bf16", "fp16"]),
                columns=rng.random() < 0.25, left_out=left_out)


def work(case):
    if case["op"] == "clip":
        sizes = _tensor_sizes(case)
        size = sum(m * SIZE[t] for m, t in zip(sizes, _tensor_types(case)))
        return {"bytes": size * (2 if case["mode"] == "clip" else 1), "flops": 2 * sum(sizes)}
    n, d, c, s = case["n"], case["d"], case["c"], SIZE[case["type"]]
    products = {"loss": 1, "step": 2, "train": 3}[case["mode"]]
    size = n * d * s + c * d * s + c * 4 + n * 8 + n * 4
    if case["mode"] != "loss":
        size += c * d * s + c * 4 + n * 4
    if case["mode"] == "train":
        size += n * d * s
    return {"bytes": size, "flops": 2 * products * n * d * c}


# ----------------------------------------------------------------- inputs ----
def _tensor_sizes(case):
    """Ragged sizes over a factor of about a thousand, summing to `total`."""
    r = np.random.RandomState(case["tensors"])
    share = np.exp(r.uniform(-7.0, 0.0, case["tensors"]))
    sizes = np.maximum(1, (share / share.sum() * case["total"]).astype(np.int64))
    return [int(m) for m in sizes]


def _tensor_types(case):
    if case["type"] != "mixed":
        return [case["type"]] * case["tensors"]
    return [("bf16", "fp32", "fp16")[i % 3] for i in range(case["tensors"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "clip":
        sizes, types = _tensor_sizes(case), _tensor_types(case)
        # layers differ in the size of their gradients
        spread = [0.01 * 2.0 ** (i % 7) for i in range(len(sizes))]
        grads = [(torch.randn(m, generator=g, device="cuda") * a).to(TYPES[t])
                 for m, a, t in zip(sizes, spread, types)]
        state = dict(case=case, grads=grads)
        if case["mode"] == "clip":
            # the clipped gradients go to flat buffers, one a type, so that a pass finds the
            # gradients as the one before did; every tensor starts on a multiple of 16 bytes
            state["flat"], state["out"] = {}, [None] * len(grads)
            for t in sorted(set(types)):
                at, places = 0, []
                for i, m in enumerate(sizes):
                    if types[i] == t:
                        places.append((i, at))
                        at += (m + 7) // 8 * 8
                state["flat"][t] = torch.zeros(at, dtype=TYPES[t], device="cuda")
                for i, a in places:
                    state["out"][i] = state["flat"][t][a:a + sizes[i]]
            # about a third of the norm that these gradients have
            state["max_norm"] = 0.37 * math.sqrt(sum(m * a * a for m, a in zip(sizes, spread)))
        return state
    n, d, c, t = case["n"], case["d"], case["c"], TYPES[case["type"]]
    shape = (d, n) if case["columns"] else (n, d)
    x = torch.randn(shape, generator=g, device="cuda")
    x = (x.t() if case["columns"] else x)
    # half of the features heavy-tailed, as in the mixed tables
    x[:, : d // 2] = torch.exp(0.5 * x[:, : d // 2])
    x = x.to(t)
    w = (torch.randn((c, d), generator=g, device="cuda") * (1.5 / math.sqrt(d))).to(t)
    bias = torch.randn(c, generator=g, device="cuda") * 0.5
    # classes of unequal frequency
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    labels = (u * u * c).long().clamp_(max=c - 1)
    out = torch.rand(n, generator=g, device="cuda") < case["left_out"]
    labels = torch.where(out, torch.full_like(labels, -1), labels)
    row_weight = torch.rand(n, generator=g, device="cuda") + 0.5
    # the mean over the rows; in fp16 times a loss scale, as its training needs
    row_weight *= (1024.0 if case["type"] == "fp16" else 1.0) / n
    state = dict(case=case, x=x, w=w, bias=bias, labels=labels, row_weight=row_weight)
    if case["mode"] == "train":
        for k in ("x", "w", "bias"):
            state[k].requires_grad_(True)
    return state


# ------------------------------------------------------------------- pass ----
def run(state):
    case = state["case"]
    if own:
        from gafime_b200 import ops
        if case["op"] == "clip":
            if case["mode"] == "norm":
                return {"norm": ops.grad_norm(state["grads"])}
            norm = ops.clip_grad_norm(state["grads"], state["max_norm"], out=state["out"])
            return {"norm": norm, "grads": state["flat"]}
        x, w, bias, labels = state["x"], state["w"], state["bias"], state["labels"]
        if case["mode"] == "loss":
            return {"loss": ops.softmax_xent(x, w, labels, bias)}
        if case["mode"] == "step":
            r = ops.softmax_xent_grad(x, w, labels, bias, row_weight=state["row_weight"], need_dx=False)
            return {"loss": r.loss, "dw": r.dw, "dbias": r.dbias}
        loss = ops.softmax_xent(x, w, labels, bias)
        dx, dw, dbias = torch.autograd.grad(loss, (x, w, bias), grad_outputs=state["row_weight"])
        return {"loss": loss.detach(), "dx": dx, "dw": dw, "dbias": dbias}
    if case["op"] == "clip":
        return _plain_clip(state)
    with torch.no_grad():
        return _plain_xent(state)


def _plain_clip(state):
    case = state["case"]
    squares = [t.double().square().sum() for t in state["grads"]]
    norm = torch.stack(squares).sum().sqrt()
    if case["mode"] == "norm":
        return {"norm": norm.float()}
    factor = torch.clamp(state["max_norm"] / norm, max=1.0).float()
    for t, o in zip(state["grads"], state["out"]):
        o.copy_(t.float() * factor)
    return {"norm": norm.float(), "grads": state["flat"]}


def _plain_xent(state):
    case = state["case"]
    x, w, bias, labels = state["x"], state["w"], state["bias"], state["labels"]
    kept = labels >= 0
    xf = torch.where(kept[:, None], x.float(), 0.0)
    wf = w.float()
    z = xf @ wf.t() + bias
    top = z.max(dim=1, keepdim=True).values
    p = torch.exp(z - top)
    total = p.sum(dim=1, keepdim=True)
    at = labels.clamp(min=0)[:, None]
    loss = (total.log() + top - z.gather(1, at))[:, 0]
    loss = torch.where(kept, loss, 0.0)
    if case["mode"] == "loss":
        return {"loss": loss}
    p = p / total
    p.scatter_add_(1, at, torch.full_like(total, -1.0))
    p *= torch.where(kept, state["row_weight"], 0.0)[:, None]
    grads = {"loss": loss, "dw": (p.t() @ xf).to(w.dtype), "dbias": p.double().sum(0).float()}
    if case["mode"] == "train":
        grads["dx"] = (p @ wf).to(x.dtype)
    return grads


# ------------------------------------------------------------- definition ----
def exact(case, seed):
    """The definition in 64 bits, block of rows by block of rows."""
    s = prepare(case, seed)
    if case["op"] == "clip":
        total = sum(float(torch.dot(t.double(), t.double())) for t in s["grads"])
        norm = math.sqrt(total)
        if case["mode"] == "norm":
            return {"norm": torch.tensor(norm, dtype=torch.float64)}
        k = s["max_norm"] / norm if norm > s["max_norm"] else 1.0
        flat = {}
        for t, dtype in TYPES.items():
            blocks = [torch.nn.functional.pad(v.double() * k, (0, -len(v) % 8)) for v in s["grads"] if v.dtype == dtype]
            if blocks:
                flat[t] = torch.cat(blocks)
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": flat}
    n, d, c = case["n"], case["d"], case["c"]
    x, w, bias = (s[k].detach() for k in ("x", "w", "bias"))
    w64, b64 = w.double(), bias.double()
    losses = torch.zeros(n, dtype=torch.float64, device="cuda")
    step, train = case["mode"] != "loss", case["mode"] == "train"
    dw = torch.zeros((c, d), dtype=torch.float64, device="cuda")
    db = torch.zeros(c, dtype=torch.float64, device="cuda")
    dx = torch.zeros((n, d), dtype=torch.float64, device="cuda") if train else None
    rows = max(1, min(n, 200_000_000 // max(c, d)))
    for r0 in range(0, n, rows):
        r1 = min(n, r0 + rows)
        idx = torch.nonzero(s["labels"][r0:r1] >= 0)[:, 0]
        y = s["labels"][r0:r1][idx]
        xb = x[r0:r1][idx].double()
        logp = torch.log_softmax(torch.addmm(b64, xb, w64.t()), dim=1)
        losses[r0 + idx] = -logp[torch.arange(len(idx), device="cuda"), y]
        if step:
            g = logp.exp_()
            g[torch.arange(len(idx), device="cuda"), y] -= 1.0
            g *= s["row_weight"][r0:r1][idx].double()[:, None]
            dw += g.t() @ xb
            db += g.sum(0)
            if train:
                dx[r0 + idx] = g @ w64
    out = {"loss": losses}
    if step:
        out.update(dw=dw, dbias=db)
    if train:
        out["dx"] = dx
    return out
