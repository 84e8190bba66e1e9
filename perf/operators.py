"""Workloads of the token operators: the gated recurrence, the distillation loss and the sampler.

Three operators that stand next to the routed layers in a token model:

* ``recurrence``: h_t = a_t h_{t-1} + (1 - a_t) x_t with a = sigmoid(gate), over whole sequences
  (training with its backward, prefill) and for one token (decode);
* ``distill``: the loss of a student's logits against a teacher's top logits, mixed with the label
  cross-entropy, with its gradient;
* ``sample``: temperature, top-k, top-p and min-p sampling from given uniform numbers.

``own`` selects this package's kernels; otherwise ``run`` is the plain form in 32-bit torch
operations. Sampling weighs a token by the whole number round(2^31 exp((x - max) / T)), so that its
sums do not depend on their order and a token is exact.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------ cases


def listed():
    return [
        # One decoded token of a small serving batch: the smallest call, where latency counts.
        {"name": "rec_step_8x1024_bf16", "op": "recurrence", "kind": "step", "dtype": "bf16", "batch": 8, "steps": 1,
         "dim": 1024, "fused": True, "reset": False},
        # A training step's mixer over ordinary sequences: gate and value are the halves of one projection.
        {"name": "rec_train_8x2048x1024_bf16", "op": "recurrence", "kind": "train", "dtype": "bf16", "batch": 8,
         "steps": 2048, "dim": 1024, "fused": True, "reset": False},
        # Packed documents of odd sizes in f32: resets where a document starts, nothing a multiple of a tile.
        {"name": "rec_train_3x1531x777_f32_packed", "op": "recurrence", "kind": "train", "dtype": "f32", "batch": 3,
         "steps": 1531, "dim": 777, "fused": False, "reset": True},
        # Prefill of one long context: few channels, so the sequence itself has to be split.
        {"name": "rec_prefill_1x65536x256_f16", "op": "recurrence", "kind": "prefill", "dtype": "f16", "batch": 1,
         "steps": 65536, "dim": 256, "fused": True, "reset": False},
        # The classifier step's rows and classes (512 rows, 47 classes), distilled: launch latency.
        {"name": "distill_train_512x47_f32", "op": "distill", "kind": "loss", "dtype": "f32", "rows": 512, "vocab": 47,
         "top": 8, "temperature": 2.0, "label_weight": 0.5, "ragged": False},
        # A training step's loss over an ordinary vocabulary through autograd, labels mixed in.
        {"name": "distill_train_4096x32000_bf16", "op": "distill", "kind": "loss", "dtype": "bf16", "rows": 4096,
         "vocab": 32000, "top": 64, "temperature": 2.0, "label_weight": 0.25, "ragged": False},
        # Ragged teachers (fewer than K entries, rows with none, ignored labels) over an odd vocabulary.
        {"name": "distill_fused_1000x50001_f16_ragged", "op": "distill", "kind": "fused", "dtype": "f16", "rows": 1000,
         "vocab": 50001, "top": 20, "temperature": 1.5, "label_weight": 0.3, "ragged": True},
        # Loss and gradient in one call for a large vocabulary, teacher only: the largest case.
        {"name": "distill_fused_8192x131072_bf16", "op": "distill", "kind": "fused", "dtype": "bf16", "rows": 8192,
         "vocab": 131072, "top": 64, "temperature": 1.0, "label_weight": 0.0, "ragged": False},
        # One interactive request: f32 logits, the usual top-k with top-p.
        {"name": "sample_1x32000_f32_k50_p90", "op": "sample", "kind": "fixed", "dtype": "f32", "rows": 1,
         "vocab": 32000, "temperature": 0.8, "top_k": 50, "top_p": 0.9, "min_p": 0.0},
        # A serving batch over a large vocabulary with a nucleus alone.
        {"name": "sample_64x131072_bf16_p95", "op": "sample", "kind": "fixed", "dtype": "bf16", "rows": 64,
         "vocab": 131072, "temperature": 1.0, "top_k": 0, "top_p": 0.95, "min_p": 0.0},
        # Requests with settings of their own, greedy ones among them, over an odd vocabulary.
        {"name": "sample_200x50001_f16_mixed", "op": "sample", "kind": "mixed", "dtype": "f16", "rows": 200,
         "vocab": 50001, "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0},
        # Rollouts for training: many rows, temperature and a min-p floor.
        {"name": "sample_512x131072_bf16_min05", "op": "sample", "kind": "fixed", "dtype": "bf16", "rows": 512,
         "vocab": 131072, "temperature": 0.9, "top_k": 0, "top_p": 1.0, "min_p": 0.05},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["recurrence", "distill", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "recurrence":
        kind = rng.choice(["step", "train", "train", "prefill"])
        if kind == "step":
            return {"op": op, "kind": kind, "dtype": dtype, "batch": _log(rng, 1, 512), "steps": 1,
                    "dim": _log(rng, 64, 4096), "fused": rng.random() < 0.5, "reset": rng.random() < 0.5}
        batch = _log(rng, 1, 8) if kind == "train" else _log(rng, 1, 2)
        dim = _log(rng, 16, 2048)
        steps = _log(rng, 1, min(16384 if kind == "train" else 65536, max(1, (1 << 24) // (batch * dim))))
        return {"op": op, "kind": kind, "dtype": dtype, "batch": batch, "steps": steps, "dim": dim,
                "fused": rng.random() < 0.5, "reset": rng.random() < 0.5}
    if op == "distill":
        vocab = _log(rng, 10, 131072)
        rows = _log(rng, 1, min(8192, (1 << 29) // vocab))
        return {"op": op, "kind": rng.choice(["loss", "fused"]), "dtype": dtype, "rows": rows, "vocab": vocab,
                "top": _log(rng, 1, min(128, vocab)), "temperature": rng.choice([1.0, 1.5, 2.0, 4.0]),
                "label_weight": rng.choice([0.0, 0.25, 0.5, 1.0]), "ragged": rng.random() < 0.5}
    return {"op": op, "kind": rng.choice(["fixed", "fixed", "mixed"]), "dtype": dtype, "rows": _log(rng, 1, 512),
            "vocab": _log(rng, 100, 131072), "temperature": rng.choice([0.5, 0.7, 1.0, 1.3]),
            "top_k": rng.choice([0, 0, 1, 40, 500]), "top_p": rng.choice([1.0, 0.5, 0.9, 0.99]),
            "min_p": rng.choice([0.0, 0.0, 0.02, 0.1])}


def work(case):
    b = _BYTES[case["dtype"]]
    if case["op"] == "recurrence":
        n, state = case["batch"] * case["steps"] * case["dim"], 4 * case["batch"] * case["dim"]
        mask = case["batch"] * case["steps"] if case["reset"] else 0
        if case["kind"] == "train":  # reads gate, value, grad; writes h, grad gate, grad value; 4 state-sized f32
            return {"bytes": 6 * n * b + 4 * state + mask, "flops": 30 * n}
        return {"bytes": 3 * n * b + 2 * state + mask, "flops": 10 * n}
    n = case["rows"] * case["vocab"]
    if case["op"] == "distill":  # reads the logits, the teacher and the labels; writes the gradient and the losses
        side = case["rows"] * (case["top"] * (b + 8) + 8 + 4)
        return {"bytes": 2 * n * b + side, "flops": 12 * n}
    return {"bytes": n * b + case["rows"] * 12, "flops": 6 * n}


# ----------------------------------------------------------------------------------------- inputs


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    make = {"recurrence": _prepare_recurrence, "distill": _prepare_distill, "sample": _prepare_sample}[case["op"]]
    state = make(case, gen, _DTYPES[case["dtype"]])
    state["case"] = case
    return state


def _prepare_recurrence(case, gen, dtype):
    B, S, D = case["batch"], case["steps"], case["dim"]
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    # Gates around sigmoid(2): memories of a few to some hundred tokens, another for each channel.
    bias = 2.0 + 1.5 * randn(D)
    gate, value = randn(B, S, D) + bias, randn(B, S, D)
    if case["fused"]:  # the halves of one projection's output
        both = torch.cat([gate, value], dim=2).to(dtype)
        gate, value = both[..., :D], both[..., D:]
    else:
        gate, value = gate.to(dtype), value.to(dtype)
    h0 = 0.5 * randn(B, D)
    reset = torch.rand(B, S, generator=gen, device="cuda") < 1.0 / 200 if case["reset"] else None
    if case["kind"] == "step":
        return {"gate": gate[:, 0], "value": value[:, 0], "h0": h0, "reset": None if reset is None else reset[:, 0]}
    state = {"gate": gate, "value": value, "h0": h0, "reset": reset}
    if case["kind"] == "train":
        for name in ("gate", "value", "h0"):
            state[name] = state[name].detach().requires_grad_()
        state["grad"] = randn(B, S, D).to(dtype)
        state["grad_last"] = randn(B, D)
    return state


def _prepare_distill(case, gen, dtype):
    N, V, K = case["rows"], case["vocab"], case["top"]
    rand = lambda *shape: torch.rand(*shape, generator=gen, device="cuda")  # noqa: E731
    logits = torch.randn(N, V, generator=gen, device="cuda", dtype=torch.float32).mul_(2.0)
    # K distinct tokens a row, at an odd pace through the vocabulary.
    first = (rand(N, 1) * V).long().clamp_(max=V - 1)
    pace = 1 + (rand(N, 1) * (V // K)).long().clamp_(max=max(0, V // K - 1))
    at = (first + pace * torch.arange(K, device="cuda")) % V
    teacher = (torch.randn(N, K, generator=gen, device="cuda") * 2.5 + 6.0).sort(dim=1, descending=True).values
    # A student that has learnt part of it.
    logits.scatter_add_(1, at, 0.7 * teacher)
    labels = torch.where(rand(N) < 0.7, at[:, 0], (rand(N) * V).long().clamp_(max=V - 1))
    if case["ragged"]:
        count = (rand(N) * (K + 1)).long()  # 0 to K entries of the teacher
        at = torch.where(torch.arange(K, device="cuda") < count[:, None], at, torch.full_like(at, -1))
        labels = torch.where(rand(N) < 0.2, torch.full_like(labels, -100), labels)
    state = {"logits": logits.to(dtype), "teacher": teacher.to(dtype), "at": at, "labels": labels,
             "row_scale": (0.5 + rand(N)) / N}
    if case["kind"] == "loss":
        state["logits"].requires_grad_()
    return state


def _prepare_sample(case, gen, dtype):
    N, V = case["rows"], case["vocab"]
    rand = lambda *shape: torch.rand(*shape, generator=gen, device="cuda")  # noqa: E731
    # Rows from flat to peaked, with a few likely tokens each.
    logits = torch.randn(N, V, generator=gen, device="cuda").mul_(1.0 + 2.0 * rand(N, 1))
    likely = (rand(N, 8) * V).long().clamp_(max=V - 1)
    logits.scatter_add_(1, likely, 9.0 * rand(N, 8))
    state = {"logits": logits.to(dtype), "u": rand(N)}
    for name in ("temperature", "top_k", "top_p", "min_p"):
        state[name] = case[name]
    if case["kind"] == "mixed":  # each request with settings of its own
        pick = lambda values, t: torch.tensor(values, device="cuda", dtype=t)[  # noqa: E731
            (rand(N) * len(values)).long().clamp_(max=len(values) - 1)]
        state["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.2], torch.float32)
        state["top_k"] = pick([0, 0, 1, 20, 100, 1000], torch.int32)
        state["top_p"] = pick([1.0, 0.8, 0.95, 0.99], torch.float32)
        state["min_p"] = pick([0.0, 0.0, 0.01, 0.1], torch.float32)
    return state


# -------------------------------------------------------------------------------------------- run


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    return {"recurrence": _plain_recurrence, "distill": _plain_distill, "sample": _plain_sample}[case["op"]](case, state)


def _run_own(case, s):
    import tropnn_b200

    if case["op"] == "recurrence":
        if case["kind"] == "step":
            h = tropnn_b200.gated_recurrence_step_b200(s["gate"], s["value"], s["h0"], reset=s["reset"])
            return {"h": h, "h_last": s["h0"]}
        h, h_last = tropnn_b200.gated_recurrence_b200(s["gate"], s["value"], s["h0"], reset=s["reset"])
        if case["kind"] == "prefill":
            return {"h": h, "h_last": h_last}
        dgate, dvalue, dh0 = torch.autograd.grad([h, h_last], [s["gate"], s["value"], s["h0"]], [s["grad"], s["grad_last"]])
        return {"h": h.detach(), "h_last": h_last.detach(), "grad_gate": dgate, "grad_value": dvalue, "grad_h0": dh0}
    if case["op"] == "distill":
        args = dict(temperature=case["temperature"], label_weight=case["label_weight"])
        if case["kind"] == "fused":
            losses, grad = tropnn_b200.distill_loss_grad_b200(
                s["logits"], s["teacher"], s["at"], s["labels"], row_scale=s["row_scale"], **args)
            return {"loss": losses, "grad": grad}
        loss = tropnn_b200.distill_loss_b200(s["logits"], s["teacher"], s["at"], s["labels"], **args)
        (grad,) = torch.autograd.grad(loss, s["logits"])
        return {"loss": loss.detach(), "grad": grad}
    return {"token": tropnn_b200.sample_tokens_b200(
        s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])}


def _scan(a, b):
    """y_t = a_t y_{t-1} + b_t over dim 1 (y before the first is 0), by doubling."""
    d = 1
    while d < b.shape[1]:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], dim=1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], dim=1)
        d *= 2
    return b


@torch.no_grad()
def _plain_recurrence(case, s):
    dtype = s["gate"].dtype
    gate, x, h0 = s["gate"].float(), s["value"].float(), s["h0"]
    if case["kind"] == "step":
        keep = torch.sigmoid(gate) if s["reset"] is None else torch.sigmoid(gate) * (~s["reset"])[:, None]
        h = keep * h0 + torch.sigmoid(-gate) * x
        h0.copy_(h)  # decoding updates the state in place
        return {"h": h.to(dtype), "h_last": h0}
    a, c = torch.sigmoid(gate), torch.sigmoid(-gate)
    on = torch.ones_like(a[:, :, :1]) if s["reset"] is None else (~s["reset"])[:, :, None].float()
    keep = a * on  # what is kept of the state before
    drive = c * x
    drive = torch.cat([drive[:, :1] + keep[:, :1] * h0[:, None], drive[:, 1:]], dim=1)
    h = _scan(keep, drive)
    out = {"h": h.to(dtype), "h_last": h[:, -1].clone()}
    if case["kind"] == "prefill":
        return out
    g = s["grad"].float()
    g = torch.cat([g[:, :-1], g[:, -1:] + s["grad_last"][:, None]], dim=1)
    after = torch.cat([keep[:, 1:], torch.zeros_like(keep[:, :1])], dim=1)
    ds = _scan(after.flip(1), g.flip(1)).flip(1)  # the whole gradient of each h_t
    before = on * torch.cat([h0[:, None], h[:, :-1]], dim=1)
    return {**out, "grad_gate": (ds * (before - x) * a * c).to(dtype), "grad_value": (ds * c).to(dtype),
            "grad_h0": keep[:, 0] * ds[:, 0]}


@torch.no_grad()
def _plain_distill(case, s):
    T, w = case["temperature"], case["label_weight"]
    N, V = s["logits"].shape
    x = s["logits"].float()
    there = (s["at"] >= 0) & (s["at"] < V)
    at = s["at"].clamp(0, V - 1)
    teacher = torch.where(there, s["teacher"].float() / T, torch.full_like(at, -math.inf, dtype=torch.float32))
    has = there.any(dim=1)
    top = torch.where(has, teacher.amax(dim=1), torch.zeros_like(x[:, 0]))
    q = torch.exp(teacher - top[:, None])
    total = q.sum(dim=1)
    q = torch.where(there, q / total[:, None], torch.zeros_like(q))
    log_q = torch.where(there, teacher - (top + torch.log(total))[:, None], torch.zeros_like(q))
    big = x.amax(dim=1, keepdim=True)
    e = torch.exp((x - big) / T)
    lse = torch.log(e.sum(dim=1, keepdim=True)) + big / T
    log_p = x.gather(1, at) / T - lse
    kl = T * T * torch.where(there, q * (log_q - log_p), torch.zeros_like(q)).sum(dim=1)
    labelled = (s["labels"] >= 0) & (s["labels"] < V)
    label = s["labels"].clamp(0, V - 1)
    e1 = torch.exp(x - big)
    lse1 = torch.log(e1.sum(dim=1)) + big[:, 0]
    ce = torch.where(labelled, lse1 - x.gather(1, label[:, None])[:, 0], torch.zeros_like(kl))
    losses = (1 - w) * torch.where(has, kl, torch.zeros_like(kl)) + w * ce
    valid = (has & (w < 1)) | (labelled & (w > 0))
    scale = s["row_scale"] if case["kind"] == "fused" else (valid / valid.sum().clamp(min=1)).float()
    grad = e / e.sum(dim=1, keepdim=True)
    grad.scatter_add_(1, at, -q)
    grad *= ((1 - w) * T * has * scale)[:, None]
    if w > 0:
        e1 /= e1.sum(dim=1, keepdim=True)
        e1.scatter_add_(1, label[:, None], -torch.ones_like(e1[:, :1]))
        grad += (w * labelled * scale)[:, None] * e1
    loss = losses if case["kind"] == "fused" else losses.sum() / valid.sum().clamp(min=1)
    return {"loss": loss, "grad": grad.to(s["logits"].dtype)}


@torch.no_grad()
def _plain_sample(case, s):
    x = s["logits"].float()
    N, V = x.shape
    row = lambda v, t: v.to(t) if isinstance(v, torch.Tensor) else torch.full((N,), v, device=x.device, dtype=t)  # noqa: E731
    T, k = row(s["temperature"], torch.float32), row(s["top_k"], torch.int64)
    p, min_p = row(s["top_p"], torch.float32), row(s["min_p"], torch.float32)
    ordered, order = torch.sort(x, dim=1, descending=True, stable=True)
    best = ordered[:, :1]
    inverse = torch.where(T > 0, 1.0 / T, torch.zeros_like(T))[:, None]
    z = (ordered - best) * inverse
    e = torch.exp(torch.where(ordered == best, torch.zeros_like(z), z))
    weight = torch.round(e * 2.0**31).to(torch.int64)
    rank = torch.arange(V, device=x.device)
    keep = (rank < torch.where(k > 0, k, torch.full_like(k, V))[:, None])
    kept = weight * keep
    before = torch.cumsum(kept, dim=1) - kept
    keep &= before.double() < (p.double() * kept.sum(dim=1).double())[:, None]
    keep &= e >= min_p[:, None]
    keep |= rank == 0  # the likeliest token always stays
    kept = torch.zeros_like(weight).scatter_(1, order, weight * keep)  # back in the vocabulary's order
    upto = torch.cumsum(kept, dim=1)
    total = upto[:, -1]
    target = torch.minimum((s["u"].double() * total.double()).floor().long(), total - 1)
    token = (upto <= target[:, None]).sum(dim=1)
    return {"token": torch.where(T > 0, token, order[:, 0])}


# ---------------------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    if case["op"] == "sample":  # whole numbers: nothing to be off by
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        return (_exact_recurrence if case["op"] == "recurrence" else _exact_distill)(case, s)


def _exact_recurrence(case, s):
    gate, x, h = s["gate"].detach().double(), s["value"].detach().double(), s["h0"].detach().double()
    if case["kind"] == "step":
        gate, x = gate[:, None], x[:, None]
    reset = s["reset"] if case["kind"] != "step" or s["reset"] is None else s["reset"][:, None]
    a = 1 / (1 + torch.exp(-gate))
    S = gate.shape[1]
    befores, hs = torch.empty_like(x), torch.empty_like(x)
    for t in range(S):  # the definition, one step after the other
        if reset is not None:
            h = torch.where(reset[:, t, None], torch.zeros_like(h), h)
        befores[:, t] = h
        h = a[:, t] * h + (1 - a[:, t]) * x[:, t]
        hs[:, t] = h
    if case["kind"] == "step":
        return {"h": hs[:, 0], "h_last": h}
    out = {"h": hs, "h_last": h}
    if case["kind"] == "prefill":
        return out
    g, d = s["grad"].double(), s["grad_last"].double()
    ds = torch.empty_like(x)
    for t in reversed(range(S)):
        d = d + g[:, t]
        ds[:, t] = d
        d = d * a[:, t]
        if reset is not None:
            d = torch.where(reset[:, t, None], torch.zeros_like(d), d)
    return {**out, "grad_gate": ds * (befores - x) * a * (1 - a), "grad_value": ds * (1 - a), "grad_h0": d}


def _exact_distill(case, s):
    T, w = case["temperature"], case["label_weight"]
    x = s["logits"].detach().double()
    N, V = x.shape
    K = s["at"].shape[1]
    spot = torch.where(s["at"] >= 0, s["at"], V)  # a column of its own for the entries that are not there
    teacher = torch.full((N, V + 1), -math.inf, dtype=torch.float64, device=x.device)
    teacher.scatter_(1, spot, s["teacher"].double())
    teacher = teacher[:, :V]
    has = (s["at"] >= 0).any(dim=1)
    q = torch.where(has[:, None], torch.softmax(teacher / T, dim=1), torch.zeros_like(teacher))
    del teacher
    log_p = torch.log_softmax(x / T, dim=1)
    kl = T * T * (torch.special.xlogy(q, q) - q * log_p).sum(dim=1)
    labelled = s["labels"] >= 0
    valid = (has & (w < 1)) | (labelled & (w > 0))
    scale = s["row_scale"].double() if case["kind"] == "fused" else valid.double() / max(1, int(valid.sum()))
    grad = log_p.exp_().sub_(q).mul_(((1 - w) * T * has * scale)[:, None])
    losses = (1 - w) * kl * has
    del q
    if w > 0:
        log_p1 = torch.log_softmax(x, dim=1)
        label = s["labels"].clamp(min=0)[:, None]
        losses = losses - w * labelled * log_p1.gather(1, label)[:, 0]
        p1 = log_p1.exp_()
        p1.scatter_(1, label, p1.gather(1, label) - 1)
        grad += p1.mul_((w * labelled * scale)[:, None])
    return {"loss": losses if case["kind"] == "fused" else losses.sum() / max(1, int(valid.sum())), "grad": grad}
