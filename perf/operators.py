"""What is measured of the operators on class scores: log probabilities with entropy and top alternatives, and
distillation from a teacher's top log probabilities, each with its gradient.

Every case is one call of a public entry point of ``vitm_amd`` (``own``) or the same operator in elementary torch
operations in 32 bits, rounded once at the end.  ``exact`` holds the definitions in 64 bits."""
import math
import os
import sys

import torch

own = False

MAX_ELEMENTS = 4096 * 131072        # logits of the largest case; a drawn case stays below
IGNORE = -100


# ---- cases ------------------------------------------------------------------------------------------------------
def _lp(name, rows, classes, dtype, top_k, targets, entropy, temperature=1.0, masked=False, grad=False):
    return dict(name=name, op="log_probs", rows=rows, classes=classes, dtype=dtype, top_k=top_k, targets=targets,
                entropy=entropy, temperature=temperature, masked=masked, grad=grad)


def _ds(name, rows, classes, dtype, top_k, temperature, label_weight, tail, mode):
    return dict(name=name, op="distill", rows=rows, classes=classes, dtype=dtype, top_k=top_k, temperature=temperature,
                label_weight=label_weight, tail=tail, mode=mode)


def listed():
    return [
        # one token of a served model: its log probability, the entropy and 20 alternatives; latency counts
        _lp("lp_token", 1, 131072, "bf16", 20, 1, True),
        # the classifier's answer for one batch of 256 images, 1000 classes: five best classes and the label's log probability
        _lp("lp_classify", 256, 1000, "bf16", 5, 1, False),
        # scoring a prompt: the given tokens' log probabilities and entropies, a vocabulary of odd size (rows start anywhere)
        _lp("lp_prompt", 4096, 65537, "bf16", 0, 1, True),
        # a batch of sampled tokens with many alternatives, part of the vocabulary masked by a grammar
        _lp("lp_top64", 1024, 131072, "bf16", 64, 1, True, temperature=0.7, masked=True),
        # the same answer in fp32 over a middle-sized class list
        _lp("lp_fp32", 2048, 21001, "fp32", 10, 2, True),
        # a policy step: gradient of log probabilities and entropies with respect to the logits
        _lp("lp_train", 2048, 32001, "bf16", 0, 1, True, grad=True),
        # the loss of a small image batch in a training step (32 images, 10 classes): loss and gradient in one call
        _ds("ds_cifar", 32, 10, "fp32", 5, 2.0, 0.5, False, "fused"),
        # the same at 256 images and 1000 classes
        _ds("ds_classes", 256, 1000, "fp32", 20, 3.0, 0.5, False, "fused"),
        # a student language model with a large vocabulary, teacher's 64 best stored beforehand, tail kept: one training step's loss
        _ds("ds_vocab", 4096, 131072, "bf16", 64, 1.0, 0.0, True, "fused"),
        # the same through loss.backward(), labels mixed in, a temperature, fp32 logits of odd length
        _ds("ds_fp32", 1024, 50001, "fp32", 32, 2.0, 0.3, False, "autograd"),
        # few rows of a large vocabulary (one short document), loss and gradient
        _ds("ds_rows", 24, 131072, "bf16", 32, 2.0, 0.1, True, "autograd"),
        # the losses of the rows alone (validation)
        _ds("ds_eval", 2048, 32001, "bf16", 50, 1.0, 0.2, True, "loss"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    classes = _log_int(rng, 2, 150000)
    rows = _log_int(rng, 1, 4096)
    while rows * classes > MAX_ELEMENTS:
        rows = max(1, rows // 2)
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if dtype == "fp32":
        while rows * classes * 2 > MAX_ELEMENTS:
            rows = max(1, rows // 2)
    if rng.random() < 0.5:
        grad = rng.random() < 0.4
        top_k = min(classes, rng.choice([0, 0, 1, 5, rng.randint(2, 100)]))
        case = _lp("", rows, classes, dtype, top_k, rng.choice([1, 1, 2, 5]), rng.random() < 0.7,
                   rng.choice([1.0, 1.0, 0.7, 2.0]), classes >= 64 and 4 * top_k <= classes and rng.random() < 0.3, grad)
    else:
        case = _ds("", rows, classes, dtype, min(classes, rng.randint(1, 100)), rng.choice([1.0, 2.0, 4.0]),
                   rng.choice([0.0, 0.3, 0.5, 1.0]), rng.random() < 0.5, rng.choice(["fused", "autograd", "loss"]))
        if case["tail"] and 2 * case["top_k"] > classes:      # a tail needs classes outside the list
            case["tail"] = False
    del case["name"]
    return case


# ---- inputs -----------------------------------------------------------------------------------------------------
def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    R, V, K = case["rows"], case["classes"], case["top_k"]
    z = torch.randn(R, V, generator=g, device=dev).mul_(2.5)
    labels = torch.randint(0, V, (R,), generator=g, device=dev)
    dropped = torch.rand(R, generator=g, device=dev) < 0.05
    s = {"case": case}
    if case["op"] == "log_probs":
        if case["masked"]:
            z.masked_fill_(torch.rand(R, V, generator=g, device=dev) < 0.4, float("-inf"))
        G = case["targets"]
        t = torch.randint(0, V, (R, G), generator=g, device=dev)
        likely = torch.randn(R, 1, generator=g, device=dev) * 2 + 4        # given tokens are likely and allowed ones
        z.scatter_(1, t, likely.expand(R, G))
        t[:, 0] = torch.where(dropped, torch.full_like(labels, IGNORE), t[:, 0])
        s["targets"] = t[:, 0].contiguous() if G == 1 else t
        s["logits"] = z.to(_dtype(case))
        if case["grad"]:
            s["g_logprobs"] = torch.randn(s["targets"].shape, generator=g, device=dev)
            s["g_entropy"] = torch.randn(R, generator=g, device=dev) * 0.1
            s["g_top"] = torch.randn(R, K, generator=g, device=dev) if K else None
        return s
    # distinct classes of every row in mixed order, and the teacher's log probabilities of them with some mass left over
    gaps = torch.randint(1, V // K + 1, (R, K), generator=g, device=dev)
    idx = gaps.cumsum(1) - 1
    idx = idx.gather(1, torch.rand(R, K, generator=g, device=dev).argsort(1))
    t = torch.cat([torch.randn(R, K, generator=g, device=dev) * 2, torch.rand(R, 1, generator=g, device=dev) * 3 - 1], 1)
    s["teacher"] = torch.log_softmax(t, 1)[:, :K].contiguous()
    z.scatter_add_(1, idx, torch.full((R, K), 3.0, device=dev))
    if K > 2:                                                   # stored lists are ragged: some rows hold fewer entries
        short = torch.rand(R, generator=g, device=dev) < 0.1
        idx[:, -1] = torch.where(short, torch.full_like(labels, -1), idx[:, -1])
    s["indices"] = idx
    s["logits"] = z.to(_dtype(case))
    s["labels"] = torch.where(dropped, torch.full_like(labels, IGNORE), labels)
    return s


# ---- the framework's calls --------------------------------------------------------------------------------------
def _package():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vision-transformer_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import vitm_amd
    from vitm_amd import training
    return vitm_amd, training


def _run_own(s):
    vitm, training = _package()
    c = s["case"]
    if c["op"] == "log_probs":
        z = s["logits"]
        if c["grad"]:
            z = z.detach().requires_grad_(True)
        r = vitm.log_probs(z, s["targets"], top_k=c["top_k"], entropy=c["entropy"], temperature=c["temperature"])
        out = {"logprobs": r.logprobs, "lse": r.lse}
        if c["entropy"]:
            out["entropy"] = r.entropy
        if c["top_k"]:
            out["top_logprobs"], out["top_indices"] = r.top_logprobs, r.top_indices
        if c["grad"]:
            heads, ups = [r.logprobs], [s["g_logprobs"]]
            if c["entropy"]:
                heads, ups = heads + [r.entropy], ups + [s["g_entropy"]]
            if c["top_k"]:
                heads, ups = heads + [r.top_logprobs], ups + [s["g_top"]]
            (out["dlogits"],) = torch.autograd.grad(heads, z, ups)
            out = {k: v.detach() for k, v in out.items()}
        return out
    loss_fn = training.DistillationLoss(temperature=c["temperature"], label_weight=c["label_weight"], tail=c["tail"],
                                        reduction="none" if c["mode"] == "loss" else "mean")
    args = (s["teacher"], s["indices"], s["labels"])
    if c["mode"] == "fused":
        loss, dz = loss_fn.loss_and_grad(s["logits"], *args)
        return {"loss": loss, "dlogits": dz}
    if c["mode"] == "loss":
        return {"loss": loss_fn(s["logits"], *args)}
    z = s["logits"].detach().requires_grad_(True)
    loss = loss_fn(z, *args)
    (dz,) = torch.autograd.grad(loss, z)
    return {"loss": loss.detach(), "dlogits": dz}


# ---- plain forms ------------------------------------------------------------------------------------------------
def _softmax_parts(x):
    """(x - max, exp of it, its sum) along the rows."""
    d = x - x.amax(1, keepdim=True)
    e = torch.exp(d)
    return d, e, e.sum(1, keepdim=True)


def _top(x, k):
    """Indices of the k largest of every row, equal values in the order of their index: one integer key per element."""
    bits = x.view(torch.int32).to(torch.int64)
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    low = (1 << 20) - 1
    key = (key << 20) + (low - torch.arange(x.shape[1], device=x.device))
    return low - (torch.topk(key, k, dim=1).values & low)


def _plain_log_probs(s):
    c = s["case"]
    invt = 1.0 / c["temperature"]
    x = s["logits"].float() * invt
    d, e, tot = _softmax_parts(x)
    lnsum = torch.log(tot)
    t = s["targets"] if s["targets"].dim() == 2 else s["targets"][:, None]
    seen = t != IGNORE
    ti = torch.where(seen, t, torch.zeros_like(t))
    lp = torch.where(seen, d.gather(1, ti) - lnsum, torch.zeros((), device=x.device))
    out = {"logprobs": lp.reshape(s["targets"].shape), "lse": (x.amax(1, keepdim=True) + lnsum)[:, 0]}
    logp = d - lnsum
    p = e / tot
    finite = torch.where(p > 0, logp, torch.zeros((), device=x.device))
    if c["entropy"]:
        out["entropy"] = -(p * finite).sum(1)
    if c["top_k"]:
        out["top_indices"] = _top(s["logits"].float(), c["top_k"])
        out["top_logprobs"] = logp.gather(1, out["top_indices"])
    if c["grad"]:
        gl = torch.where(seen, s["g_logprobs"].reshape(t.shape), torch.zeros((), device=x.device))
        coef = -gl.sum(1, keepdim=True)
        if c["top_k"]:
            coef = coef - s["g_top"].sum(1, keepdim=True)
        if c["entropy"]:
            coef = coef - s["g_entropy"][:, None] * (finite + out["entropy"][:, None])
        dz = p * coef
        dz.scatter_add_(1, ti, gl)
        if c["top_k"]:
            dz.scatter_add_(1, out["top_indices"], s["g_top"])
        out["dlogits"] = (dz * invt).to(s["logits"].dtype)
    return out


def _plain_distill(s):
    c = s["case"]
    T, a = c["temperature"], c["label_weight"]
    z = s["logits"].float()
    zero = torch.zeros((), device=z.device)
    ninf = torch.full((), float("-inf"), device=z.device)
    there = s["indices"] >= 0
    idx = torch.where(there, s["indices"], torch.zeros_like(s["indices"]))
    tl = torch.where(there, s["teacher"], ninf)
    if not c["tail"]:
        tl = tl - torch.logsumexp(tl, 1, keepdim=True)
    q = torch.exp(tl)
    d, e, tot = _softmax_parts(z / T)
    p = e / tot
    logp = d.gather(1, idx) - torch.log(tot)
    kl = torch.where(there, q * (torch.where(there, tl, zero) - logp), zero).sum(1)
    Q = q.sum(1, keepdim=True)
    inlist = torch.zeros(z.shape, device=z.device).scatter_add_(1, idx, there.float()) > 0
    if c["tail"]:
        rest = torch.where(inlist, zero, e)
        srest = rest.sum(1, keepdim=True)
        qr = torch.clamp(1.0 - Q, min=0.0)
        lnr = (torch.log(srest) - torch.log(tot))[:, 0]
        kl = kl + torch.where(qr[:, 0] > 0, qr[:, 0] * (torch.log(qr[:, 0]) - lnr), zero)
        Q = Q + qr
    keep = s["labels"] != IGNORE
    y = torch.where(keep, s["labels"], torch.zeros_like(s["labels"]))[:, None]
    d1, e1, tot1 = (d, e, tot) if T == 1.0 else _softmax_parts(z)
    ce = torch.log(tot1)[:, 0] - d1.gather(1, y)[:, 0]
    rows = torch.where(keep, (1 - a) * T * T * kl + a * ce, zero)
    if c["mode"] == "loss":
        return {"loss": rows}
    n = keep.sum().clamp(min=1).float()
    out = {"loss": rows.sum() / n}
    dz = p * Q
    if c["tail"]:
        dz = dz - rest * (qr / srest)
    dz.scatter_add_(1, idx, torch.where(there, -q, zero))
    dz = dz * ((1 - a) * T)
    if a:
        dz = dz + (e1 / tot1) * a
        dz.scatter_add_(1, y, torch.full(y.shape, -a, device=z.device))
    out["dlogits"] = (dz * (keep.float() / n)[:, None]).to(s["logits"].dtype)
    return out


def run(state):
    if own:
        return _run_own(state)
    return _plain_log_probs(state) if state["case"]["op"] == "log_probs" else _plain_distill(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------
def work(case):
    R, V, K = case["rows"], case["classes"], case["top_k"]
    es = 2 if case["dtype"] == "bf16" else 4
    n = R * V
    if case["op"] == "log_probs":
        b = n * es + R * (case["targets"] * 12 + 4 + (4 if case["entropy"] else 0) + K * 12)
        f = n * (4 + (2 if case["entropy"] else 0))
        if case["grad"]:
            b, f = b + n * es + R * case["targets"] * 4, f + n * 5
        return {"bytes": b, "flops": f}
    two = 2 if case["temperature"] != 1.0 and case["label_weight"] else 1
    b, f = n * es + R * (K * 12 + 12), n * 4 * two
    if case["mode"] != "loss":
        b, f = b + n * es, f + n * 4 * two
    return {"bytes": b, "flops": f}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------
def _chunks(R, V):
    step = max(1, (1 << 25) // V)
    return [(r, min(R, r + step)) for r in range(0, R, step)]


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_log_probs(s) if case["op"] == "log_probs" else _exact_distill(s)


def _exact_log_probs(s):
    c = s["case"]
    parts = []
    for a, b in _chunks(c["rows"], c["classes"]):
        z = s["logits"][a:b].double().clamp(min=-1e6).requires_grad_(c["grad"])     # a masked class: probability 0 in 64 bits
        lse = torch.logsumexp(z / c["temperature"], 1)
        logp = z / c["temperature"] - lse[:, None]
        t = s["targets"][a:b].reshape(b - a, -1)
        lp = torch.where(t == IGNORE, torch.zeros((), dtype=z.dtype, device=z.device), logp.gather(1, t.clamp(min=0)))
        o = {"logprobs": lp.reshape(s["targets"][a:b].shape), "lse": lse}
        if c["entropy"]:
            o["entropy"] = -(logp.exp() * logp).sum(1)
        if c["top_k"]:
            order = torch.sort(s["logits"][a:b].double(), dim=1, descending=True, stable=True).indices
            o["top_indices"] = order[:, :c["top_k"]]
            o["top_logprobs"] = logp.gather(1, o["top_indices"])
        if c["grad"]:
            total = (lp * s["g_logprobs"][a:b].reshape(lp.shape).double()).sum()
            if c["entropy"]:
                total = total + (o["entropy"] * s["g_entropy"][a:b].double()).sum()
            if c["top_k"]:
                total = total + (o["top_logprobs"] * s["g_top"][a:b].double()).sum()
            (o["dlogits"],) = torch.autograd.grad(total, z)
        parts.append({k: v.detach() for k, v in o.items()})
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _exact_distill(s):
    c = s["case"]
    T, a = c["temperature"], c["label_weight"]
    n = max(1, int((s["labels"] != IGNORE).sum()))
    losses, grads = [], []
    for lo, hi in _chunks(c["rows"], c["classes"]):
        z = s["logits"][lo:hi].double().requires_grad_(c["mode"] != "loss")
        idx, y = s["indices"][lo:hi], s["labels"][lo:hi]
        logp = torch.log_softmax(z / T, 1)
        # the teacher as a dense distribution over the classes and one more place for the absent entries
        teacher = s["teacher"][lo:hi].double()
        weight = torch.where(idx >= 0, teacher.exp(), torch.zeros((), dtype=z.dtype, device=z.device))
        if not c["tail"]:
            weight = weight / weight.sum(1, keepdim=True)
        V = c["classes"]
        dense = torch.zeros(hi - lo, V + 1, dtype=z.dtype, device=z.device)
        dense.scatter_(1, torch.where(idx >= 0, idx, torch.full_like(idx, V)), weight)
        dense = dense[:, :V]
        kl = (torch.xlogy(dense, dense) - dense * logp).sum(1)
        if c["tail"]:
            left = (1 - weight.sum(1)).clamp(min=0)
            outside = torch.logsumexp(logp.masked_fill(dense > 0, float("-inf")), 1)
            kl = kl + torch.xlogy(left, left) - left * outside
        ce = torch.nn.functional.cross_entropy(z, y, ignore_index=IGNORE, reduction="none")
        rows = torch.where(y != IGNORE, (1 - a) * T * T * kl + a * ce, torch.zeros((), dtype=z.dtype, device=z.device))
        if c["mode"] == "loss":
            losses.append(rows)
            continue
        total = rows.sum() / n
        grads.append(torch.autograd.grad(total, z)[0])
        losses.append(total.detach())
    if c["mode"] == "loss":
        return {"loss": torch.cat(losses)}
    return {"loss": torch.stack(losses).sum(), "dlogits": torch.cat(grads)}
