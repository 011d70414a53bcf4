"""Cases of the vocabulary-head operators beside the cross-entropy loss: what they cost and what they answer.

Three operators, as a distillation loop uses them one after the other:

* ``linear_distillation`` -- the loss of a student head against a teacher's top logits, with both gradients;
* ``top_logits``          -- the teacher's side: the largest logits of each row with the row's log-sum-exp;
* ``sample_logits``       -- the head's answers: temperature, top-k, top-p and min-p from given random numbers.

``run`` computes each in its plain form (elementary torch operations) or, with ``own`` set, through the package.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a step on a handful of tokens (the end of an on-policy rollout): nothing but latency
        dict(name="distill_16_rows", op="distill", N=16, H=256, V=4096, K=8, type="bf16", T=1.0, tail=False, pads=False),
        # sizes that are multiples of nothing, half precision, teacher lists of different lengths, softened targets
        dict(name="distill_ragged_fp16", op="distill", N=1000, H=1000, V=50257, K=17, type="fp16", T=2.0, tail=False, pads=True),
        # one chunk of an ordinary training step; the teacher's log-sum-exp says how much mass its list leaves out
        dict(name="distill_4096_rows", op="distill", N=4096, H=2048, V=32768, K=32, type="bf16", T=1.0, tail=True, pads=False),
        # the head of the default benchmark point, two chunks
        dict(name="distill_large_vocab", op="distill", N=8192, H=2048, V=131072, K=64, type="bf16", T=1.0, tail=False, pads=True),
        # alternatives shown for one generated token
        dict(name="top_1_row", op="top", N=1, V=131072, k=64, type="fp32", T=1.0),
        # a vocabulary that is a multiple of nothing: rows start at odd addresses
        dict(name="top_ragged_fp16", op="top", N=333, V=50257, k=100, type="fp16", T=2.0),
        # a teacher's logits for one chunk of tokens
        dict(name="top_teacher", op="top", N=4096, V=131072, k=64, type="bf16", T=1.0),
        # long lists from few, long rows
        dict(name="top_long_lists", op="top", N=48, V=262144, k=512, type="fp32", T=1.0),
        # one chat: one row, the usual settings
        dict(name="sample_1_row", op="sample", B=1, V=50257, type="bf16", T=0.8, top_k=50, top_p=0.9, min_p=0.0,
             rows="alike", masked=0.0),
        # nucleus sampling without a cap on the number of tokens
        dict(name="sample_nucleus", op="sample", B=64, V=131072, type="fp32", T=1.0, top_k=0, top_p=0.95, min_p=0.0,
             rows="alike", masked=0.0),
        # a served batch: every request has its own settings, some answer greedily, some under a grammar's mask
        dict(name="sample_mixed", op="sample", B=256, V=131072, type="bf16", T=1.0, top_k=40, top_p=0.9, min_p=0.05,
             rows="mixed", masked=0.5),
        # many rollouts of one policy, nearly unfiltered
        dict(name="sample_rollouts", op="sample", B=1024, V=32768, type="fp16", T=1.0, top_k=0, top_p=1.0, min_p=0.001,
             rows="alike", masked=0.0),
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["distill", "top", "sample"])
    if op == "distill":
        while True:
            c = dict(op=op, N=_between(rng, 1, 8192), H=_between(rng, 64, 2048), V=_between(rng, 500, 131072),
                     K=_between(rng, 1, 128), type=rng.choice(["bf16", "fp16"]), T=round(rng.uniform(0.7, 4.0), 2),
                     tail=rng.random() < 0.4, pads=rng.random() < 0.5)
            if c["N"] * c["H"] * c["V"] <= 8192 * 2048 * 131072 / 8:
                return c
    if op == "top":
        c = dict(op=op, N=_between(rng, 1, 4096), V=_between(rng, 1000, 262144), type=rng.choice(["fp32", "bf16", "fp16"]),
                 T=round(rng.uniform(0.5, 3.0), 2))
        c["N"] = max(1, min(c["N"], 4096 * 65536 // c["V"]))
        c["k"] = _between(rng, 1, 512)
        return c
    c = dict(op=op, B=_between(rng, 1, 1024), V=_between(rng, 1000, 262144), type=rng.choice(["fp32", "bf16", "fp16"]),
             T=round(rng.uniform(0.3, 1.6), 2), top_k=rng.choice([0, 0, _between(rng, 1, 2000)]),
             top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.999), 3)]), min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 3)]),
             rows=rng.choice(["alike", "mixed"]), masked=rng.choice([0.0, 0.0, 0.5, 0.95]))
    c["B"] = max(1, min(c["B"], 256 * 131072 // c["V"]))
    return c


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g = _generator(seed)
    dt = _TYPES[case["type"]]
    if case["op"] == "distill":
        N, H, V, K, T = case["N"], case["H"], case["V"], case["K"], case["T"]
        x = torch.randn(N, H, generator=g, device="cuda").to(dt)
        At = torch.empty(H, V, dtype=dt, device="cuda")
        for h0 in range(0, H, 256):  # normal clipped at two sigma, as language-model heads start
            blk = torch.randn(min(256, H - h0), V, generator=g, device="cuda").clamp_(-2.0, 2.0)
            At[h0:h0 + 256] = (blk * H ** -0.5).to(dt)
        # K different tokens of each row, the first ones the likeliest
        gaps = torch.randint(1, max(2, V // K + 1), (N, K), generator=g, device="cuda")
        idx = (torch.randint(0, V, (N, 1), generator=g, device="cuda") + gaps.cumsum(1)) % V
        idx = idx.gather(1, torch.rand(N, K, generator=g, device="cuda").argsort(1))
        t = (2.5 * torch.randn(N, K, generator=g, device="cuda") + 8.0).sort(1, descending=True).values.to(dt)
        if case["pads"]:  # lists of different lengths; some rows (prompt tokens) have none
            length = torch.randint(1, K + 1, (N, 1), generator=g, device="cuda")
            length[torch.rand(N, 1, generator=g, device="cuda") < 0.02] = 0
            if N <= 4:
                length.clamp_(min=1)
            pad = torch.arange(K, device="cuda") >= length
            idx = idx.masked_fill(pad, -1)
            t = t.masked_fill(pad, float("-inf"))
        lse = None
        if case["tail"]:
            lse = torch.logsumexp(t.float() / T, 1) + 0.3 * torch.rand(N, generator=g, device="cuda")
            lse = torch.where(torch.isfinite(lse), lse, torch.zeros_like(lse))
        return dict(case=case, x=x, At=At, t=t, idx=idx, lse=lse)
    rows = case["N"] if case["op"] == "top" else case["B"]
    V = case["V"]
    logits = torch.empty(rows, V, dtype=dt, device="cuda")
    step = max(1, (1 << 26) // V)
    for r in range(0, rows, step):
        logits[r:r + step] = (3.0 * torch.randn(min(step, rows - r), V, generator=g, device="cuda")).to(dt)
    if case["op"] == "top":
        return dict(case=case, logits=logits)
    if case["masked"]:  # half of the rows follow a grammar that allows a share of the tokens
        for r in range(0, rows, 2):
            drop = torch.rand(V, generator=g, device="cuda") < case["masked"]
            drop[r % V] = False
            logits[r].masked_fill_(drop, float("-inf"))
    u = torch.rand(rows, generator=g, device="cuda")
    T, top_k, top_p, min_p = case["T"], case["top_k"], case["top_p"], case["min_p"]
    if case["rows"] == "mixed":
        r = torch.rand(4, rows, generator=g, device="cuda")
        T = torch.where(r[0] < 0.125, torch.zeros_like(r[0]), T * (0.5 + r[0]))
        if top_k:
            top_k = torch.where(r[1] < 0.25, torch.zeros_like(r[1]), 1 + r[1] * 2 * top_k).to(torch.int32)
        top_p = torch.where(r[2] < 0.25, torch.ones_like(r[2]), top_p * r[2])
        min_p = torch.where(r[3] < 0.5, torch.zeros_like(r[3]), min_p * r[3])
    return dict(case=case, logits=logits, u=u, T=T, top_k=top_k, top_p=top_p, min_p=min_p)


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_distill(s):
    T = s["case"]["T"]
    x, At, idx = s["x"].float(), s["At"].float(), s["idx"]
    N, V = x.shape[0], At.shape[1]
    there = (idx >= 0) & (idx < V)
    at = idx.clamp(0, V - 1)
    t = torch.where(there, s["t"].float() / T, torch.full_like(at, float("-inf"), dtype=torch.float32))
    if s["lse"] is None:
        top = t.amax(1, keepdim=True)
        e = torch.where(there, torch.exp(t - torch.where(torch.isfinite(top), top, torch.zeros_like(top))), torch.zeros_like(t))
        total = e.sum(1, keepdim=True)
        q = torch.where(total > 0, e / total, torch.zeros_like(e))
    else:
        q = torch.where(there, torch.exp(t - s["lse"][:, None]), torch.zeros_like(t))
    mass = q.sum(1)
    n = (mass > 0).sum().float()
    logq = torch.log(torch.where(q > 0, q, torch.ones_like(q)))
    dx = torch.empty_like(x)
    dAt = torch.zeros_like(At)
    loss = torch.zeros((), dtype=torch.float64, device=x.device)
    for r in range(0, N, 2048):
        xr, qr, ar, mr = x[r:r + 2048], q[r:r + 2048], at[r:r + 2048], mass[r:r + 2048]
        z = (xr @ At) / T
        top = z.amax(1, keepdim=True)
        p = torch.exp(z - top)
        total = p.sum(1, keepdim=True)
        lse = (top + torch.log(total)).squeeze(1)
        loss += (qr * (logq[r:r + 2048] - z.gather(1, ar) + lse[:, None])).sum(dtype=torch.float64)
        p *= mr[:, None] / total
        p.scatter_add_(1, ar, -qr)
        dx[r:r + 2048] = (p @ At.T) * (T / n)
        dAt += xr.T @ p
    return (loss * (T * T) / n).float(), dx.to(s["x"].dtype), (dAt * (T / n)).to(s["At"].dtype)


def _plain_top(s):
    T, k = s["case"]["T"], s["case"]["k"]
    logits = s["logits"]
    rows, V = logits.shape
    values, indices, lse = [], [], []
    step = max(1, (1 << 28) // V)
    for r in range(0, rows, step):
        v, i = torch.sort(logits[r:r + step], dim=1, descending=True, stable=True)  # equal values by index
        values.append(v[:, :k])
        indices.append(i[:, :k])
        z = logits[r:r + step].float() / T
        top = z.amax(1, keepdim=True)
        lse.append((top + torch.log(torch.exp(z - top).sum(1, keepdim=True))).squeeze(1))
    return torch.cat(values), torch.cat(indices), torch.cat(lse)


def _column(v, rows):
    v = v.double() if isinstance(v, torch.Tensor) else torch.full((rows,), float(v), dtype=torch.float64, device="cuda")
    return v[:, None]


def _plain_sample(s):
    """In 64 bits throughout: a token is right or wrong, and the borders between tokens lie close together."""
    rows, V = s["logits"].shape
    tokens, logprobs = [], []
    step = max(1, (1 << 25) // V)
    T_all, k_all, p_all, m_all = (_column(s[n], rows) for n in ("T", "top_k", "top_p", "min_p"))
    for r in range(0, rows, step):
        T, top_k, top_p, min_p = (v[r:r + step] for v in (T_all, k_all, p_all, m_all))
        logits, order = torch.sort(s["logits"][r:r + step], dim=1, descending=True, stable=True)
        rank = torch.arange(V, device="cuda")[None, :]
        d = (logits - logits[:, :1].double()) / torch.where(T > 0, T, torch.ones_like(T))
        keep = ((rank < top_k) | (top_k <= 0)) & ((T > 0) | (rank < 1))
        w = torch.exp(d) * keep
        before = w.cumsum(1) - w
        keep &= (before < top_p * w.sum(1, keepdim=True)) | (rank == 0) | (top_p >= 1)
        keep &= (torch.exp(d) >= min_p)
        w *= keep
        by_index = torch.zeros_like(w).scatter_(1, order, w)
        total = w.sum(1, keepdim=True)
        token = (by_index.cumsum(1) > s["u"][r:r + step].double()[:, None] * total).to(torch.int8).argmax(1, keepdim=True)
        tokens.append(token.squeeze(1))
        logprobs.append(torch.log(by_index.gather(1, token) / total).squeeze(1))
    return torch.cat(tokens), torch.cat(logprobs).float()


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if op == "distill":
        if own:
            from linear_cross_entropy_loss_b200 import linear_distillation

            x, At = state["x"].detach().requires_grad_(), state["At"].detach().requires_grad_()
            loss = linear_distillation(x, state["t"], state["idx"], At, teacher_lse=state["lse"], temperature=state["case"]["T"])
            dx, dAt = torch.autograd.grad(loss, (x, At))
            loss = loss.detach()
        else:
            loss, dx, dAt = _plain_distill(state)
        return {"loss": loss, "dx": dx, "dAt": dAt}
    if op == "top":
        if own:
            from linear_cross_entropy_loss_b200 import top_logits

            values, indices, lse = top_logits(state["logits"], state["case"]["k"], temperature=state["case"]["T"])
        else:
            values, indices, lse = _plain_top(state)
        return {"values": values, "indices": indices, "lse": lse}
    if own:
        from linear_cross_entropy_loss_b200 import sample_logits

        tokens, logprobs = sample_logits(state["logits"], state["u"], temperature=state["T"], top_k=state["top_k"],
                                         top_p=state["top_p"], min_p=state["min_p"])
    else:
        tokens, logprobs = _plain_sample(state)
    return {"tokens": tokens, "logprobs": logprobs}


def work(case):
    es = 4 if case["type"] == "fp32" else 2
    if case["op"] == "distill":
        N, H, V, K = case["N"], case["H"], case["V"], case["K"]
        return {"bytes": 2 * es * (N * H + H * V) + N * K * (8 + es) + (4 * N if case["tail"] else 0) + 4, "flops": 6 * N * H * V}
    if case["op"] == "top":
        return {"bytes": case["N"] * (case["V"] * es + case["k"] * (8 + es) + 4), "flops": 4 * case["N"] * case["V"]}
    return {"bytes": case["B"] * (case["V"] * es + 4 + 12 + (16 if case["rows"] == "mixed" else 0)), "flops": 4 * case["B"] * case["V"]}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "distill":
        return _exact_distill(s)
    if case["op"] == "top":
        k, T = case["k"], case["T"]
        values, lse = [], []
        for row in s["logits"].split(max(1, (1 << 27) // case["V"])):
            values.append(torch.topk(row.double(), k, dim=1).values)
            lse.append(torch.logsumexp(row.double() / T, 1))
        return {"values": torch.cat(values), "indices": None, "lse": torch.cat(lse)}
    return _exact_sample(s)


def _exact_distill(s):
    """Through the definition's derivative by automatic differentiation, a block of rows at a time."""
    T = s["case"]["T"]
    x, At, idx = s["x"].double(), s["At"].double(), s["idx"]
    V = At.shape[1]
    q = torch.zeros(idx.shape, dtype=torch.float64, device=x.device)
    for col in range(idx.shape[1]):
        q[:, col] = torch.where(idx[:, col] >= 0, torch.exp(s["t"][:, col].double() / T), torch.zeros_like(q[:, col]))
    q = q / q.sum(1, keepdim=True).clamp(min=1e-300) if s["lse"] is None else q * torch.exp(-s["lse"].double())[:, None]
    n = int((q.sum(1) > 0).sum())
    At.requires_grad_()
    loss, dx, dAt = 0.0, [], torch.zeros_like(At)
    for r in range(0, x.shape[0], 1024):
        xr = x[r:r + 1024].detach().requires_grad_()
        logp = torch.log_softmax((xr @ At) / T, dim=1).gather(1, idx[r:r + 1024].clamp(min=0))
        part = (torch.special.xlogy(q[r:r + 1024], q[r:r + 1024]) - q[r:r + 1024] * logp).sum() * (T * T / n)
        gx, gA = torch.autograd.grad(part, (xr, At))
        loss = loss + part.detach()
        dx.append(gx)
        dAt += gA
    return {"loss": loss, "dx": torch.cat(dx), "dAt": dAt}


def _exact_sample(s):
    """Row by row on the host, from the definition: rank, cut, draw."""
    logits, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    if logits.size > 1 << 26:
        return None

    def of_row(v, r):
        return float(v[r]) if isinstance(v, torch.Tensor) else float(v)

    logprobs = np.empty(len(logits))
    for r, row in enumerate(logits):
        T, top_k, top_p, min_p = (of_row(s[n], r) for n in ("T", "top_k", "top_p", "min_p"))
        if T <= 0:
            logprobs[r] = 0.0
            continue
        finite = np.flatnonzero(row > -np.inf)
        ranked = finite[np.lexsort((finite, -row[finite]))]
        if top_k > 0:
            ranked = ranked[:int(top_k)]
        w = np.exp((row[ranked] - row[ranked[0]]) / T)
        if top_p < 1:
            mass = np.cumsum(w)
            ranked = ranked[:max(1, 1 + int(np.searchsorted(mass, top_p * mass[-1], side="left")))]
        w = w[:len(ranked)]
        ranked, w = ranked[w >= min_p], w[w >= min_p]
        by_index = np.argsort(ranked)
        ranked, w = ranked[by_index], w[by_index]
        mass = np.cumsum(w)
        at = min(int(np.searchsorted(mass, u[r] * mass[-1], side="right")), len(w) - 1)
        logprobs[r] = math.log(w[at] / mass[-1])
    return {"tokens": None, "logprobs": logprobs}
