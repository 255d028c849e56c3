"""What the operators of a tuning step cost: the scaled embedding, the shared projection with the low-rank adapters of many
requests, and the distillation loss from a teacher's top logits, each beside its plain form in elementary torch operations.

`own` selects the side: False computes the plain forms (32-bit arithmetic, one rounding at the end), True calls the
framework.  `listed()` are the cases, `draw(rng)` makes more of the same ranges, `prepare` the inputs on the GPU, `run` one
pass, `work` what a pass cannot do without and `exact` the results in 64 bits."""
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}


# ------------------------------------------------------------------------------------------------ cases
def _emb(name, T, V, D, dtype, idx, ids, pad, bwd, scale):
    return dict(name=name, op="embedding", T=T, V=V, D=D, dtype=dtype, idx=idx, ids=ids, pad=pad, bwd=bwd, scale=scale)


def _ada(name, T, K, N, r, G, dtype, ids, pad, bias, bwd):
    return dict(name=name, op="adapter", T=T, K=K, N=N, r=r, G=G, dtype=dtype, ids=ids, pad=pad, bias=bias, bwd=bwd)


def _dis(name, N, V, K, dtype, tdtype, idx, temp, weights, pad, reduction, bwd):
    return dict(name=name, op="distill", N=N, V=V, K=K, dtype=dtype, tdtype=tdtype, idx=idx, temp=temp, weights=weights, pad=pad,
                reduction=reduction, bwd=bwd)


def listed():
    return [
        # conditioning vectors of one batch of cases: a lookup of a few rows, where only latency counts
        _emb("embed_batch64_f32", 64, 1024, 128, "f32", "i64", "uniform", 0.0, False, 1.0),
        # a training step's token table: hot and rare ids, a dense gradient
        _emb("embed_train_bf16", 16384, 32768, 1024, "bf16", "i64", "skewed", 0.0, True, 32.0),
        # a padded batch, a row length that no vector divides, 32-bit ids
        _emb("embed_train_odd_f32", 5003, 9973, 331, "f32", "i32", "skewed", 0.1, True, math.sqrt(331.0)),
        # the latent MLPs' hidden layer and batch, one adapter per machine, tuned
        _ada("adapter_latent_f32", 256, 256, 256, 8, 16, "f32", "random", 0.0, True, True),
        # one request, one token
        _ada("adapter_one_token_bf16", 1, 2048, 2048, 8, 4, "bf16", "random", 0.0, True, False),
        # a serving step: a single token of each of 64 requests, nearly as many adapters, some requests without one
        _ada("adapter_tokens64_bf16", 64, 4096, 4096, 16, 64, "bf16", "random", 0.1, False, False),
        # the prompts of eight requests and one without an adapter
        _ada("adapter_prompts_bf16", 8192, 4096, 4096, 16, 8, "bf16", "segments", 0.1, True, False),
        # tuning four adapters at once beside the frozen projection
        _ada("adapter_train_bf16", 4096, 2048, 4096, 32, 4, "bf16", "segments", 0.0, True, True),
        # the same with sizes that no tile or vector divides, adapters in mixed order
        _ada("adapter_train_odd_bf16", 1027, 517, 1001, 5, 7, "bf16", "random", 0.1, True, True),
        # a discretised posterior over parameter bins, the batch of the latent trainers
        _dis("distill_bins_f32", 256, 1024, 16, "f32", "f32", "i64", 2.0, False, 0.0, "mean", True),
        # a large vocabulary
        _dis("distill_large_bf16", 2048, 131072, 64, "bf16", "f32", "i32", 1.0, True, 0.0, "mean", True),
        # rows that start off a vector's boundary, padded teacher lists, a loss per row
        _dis("distill_rows_odd_bf16", 1021, 49999, 33, "bf16", "bf16", "i64", 4.0, True, 0.2, "none", True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / (5e14 if case["dtype"] == "bf16" else 5e13)


def draw(rng):
    op = rng.choice(["embedding", "adapter", "distill"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        dtype = rng.choice(["f32", "bf16"])
        if op == "embedding":
            c = _emb("", _log_int(rng, 1, 65536), _log_int(rng, 50, 131072), _log_int(rng, 8, 2048), dtype, rng.choice(["i32", "i64"]),
                     rng.choice(["uniform", "skewed"]), rng.choice([0.0, 0.1, 0.6]), rng.random() < 0.7, rng.choice([1.0, 0.5, 32.0, 18.2]))
        elif op == "adapter":
            c = _ada("", _log_int(rng, 1, 8192), _log_int(rng, 16, 4096), _log_int(rng, 16, 4096), _log_int(rng, 1, 64), _log_int(rng, 1, 128),
                     dtype, rng.choice(["random", "segments"]), rng.choice([0.0, 0.1, 0.5]), rng.random() < 0.5, rng.random() < 0.5)
            if rng.random() < 0.5:                      # half of them with the round widths that layers mostly have
                c["K"], c["N"] = max(16, c["K"] // 64 * 64), max(16, c["N"] // 64 * 64)
                c["r"] = max(4, c["r"] // 4 * 4)
        else:
            V = _log_int(rng, 17, 131072)
            c = _dis("", _log_int(rng, 1, 8192), V, min(V, _log_int(rng, 1, 128)), dtype, rng.choice(["f32", "bf16"]), rng.choice(["i32", "i64"]),
                     rng.choice([1.0, 1.5, 2.0, 4.0]), rng.random() < 0.5, rng.choice([0.0, 0.2]), rng.choice(["mean", "sum", "none"]),
                     rng.random() < 0.8)
        if _cost(c) <= most:
            del c["name"]
            return c


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)


def prepare(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    it = torch.int32 if case.get("idx") == "i32" else torch.int64
    s = dict(case=case)
    if case["op"] == "embedding":
        T, V, D = case["T"], case["V"], case["D"]
        u = _rand(g, T)
        ids = torch.exp(u * math.log(V)).long() - 1 if case["ids"] == "skewed" else (u * V).long()
        ids = ids.clamp_(0, V - 1)
        ids = torch.where(_rand(g, T) < case["pad"], torch.full_like(ids, -1), ids)
        s["ids"] = ids.to(it)
        s["table"] = (_randn(g, V, D) * 0.05).to(dt).requires_grad_(case["bwd"])
        s["dout"] = _randn(g, T, D).to(dt) if case["bwd"] else None
    elif case["op"] == "adapter":
        T, K, N, r, G = (case[k] for k in ("T", "K", "N", "r", "G"))
        if case["ids"] == "random":
            ids = (_rand(g, T) * G).long().clamp_(0, G - 1)
            ids = torch.where(_rand(g, T) < case["pad"], torch.full_like(ids, -1), ids)
        else:                                           # the tokens of a request lie together, its length is its own
            parts = G + (1 if case["pad"] > 0 else 0)
            cuts = (_rand(g, parts) + 0.2).cumsum(0)
            cuts = (cuts / cuts[-1] * T).long()
            ids = torch.searchsorted(cuts, torch.arange(T, device="cuda"), right=True).clamp_(0, parts - 1)
            ids = torch.where(ids >= G, torch.full_like(ids, -1), ids)
        s["ids"] = ids
        s["x"] = _randn(g, T, K).to(dt).requires_grad_(case["bwd"])
        s["w"] = (_randn(g, N, K) / math.sqrt(K)).to(dt)
        s["bias"] = _randn(g, N).to(dt) if case["bias"] else None
        s["A"] = (_randn(g, G, r, K) / math.sqrt(K)).to(dt).requires_grad_(case["bwd"])
        s["B"] = (_randn(g, G, N, r) / math.sqrt(r)).to(dt).requires_grad_(case["bwd"])
        s["scales"] = 0.25 + _rand(g, G)
        s["dy"] = _randn(g, T, N).to(dt) if case["bwd"] else None
    else:
        N, V, K = case["N"], case["V"], case["K"]
        z = torch.empty(N, V, device="cuda", dtype=dt)
        step = max(1, (1 << 27) // V)
        for a in range(0, N, step):
            z[a:a + step] = (_randn(g, min(step, N - a), V) * 2.0).to(dt)
        top = torch.sort(_randn(g, N, K) * 1.5 + 8.0, dim=1, descending=True).values
        part = torch.randperm(K, generator=g, device="cuda").float()        # one entry from each K-th of the vocabulary: no two alike
        lo, hi = torch.floor(part * V / K).long(), torch.floor((part + 1) * V / K).long()
        idx = lo + torch.minimum((_rand(g, N, K) * (hi - lo)).long(), hi - lo - 1)
        z.scatter_(1, idx, (top + _randn(g, N, K)).to(dt))          # the student is near the teacher there
        short = _rand(g, N, K) < case["pad"]
        idx = torch.where(short, torch.full_like(idx, -1), idx)
        s["logits"] = z.requires_grad_(case["bwd"])
        s["top"], s["idx"] = top.to(_DT[case["tdtype"]]), idx.to(it)
        s["weights"] = (_rand(g, N) < 0.8).float() if case["weights"] else None
        s["dloss"] = _randn(g, N) if case["reduction"] == "none" else None
    return s


# ------------------------------------------------------------------------------------------------ one pass
def _run_own(s):
    c = s["case"]
    if c["op"] == "embedding":
        from unet_amd.embedding import scaled_embedding
        out = scaled_embedding(s["ids"], s["table"], scale=c["scale"])
        if not c["bwd"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, (s["table"],), s["dout"]))
    if c["op"] == "adapter":
        from unet_amd.adapters import adapter_linear
        y = adapter_linear(s["x"], s["w"], s["bias"], s["A"], s["B"], s["ids"], scales=s["scales"])
        if not c["bwd"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["A"], s["B"]), s["dy"]))
    from unet_amd.losses import distillation_loss
    loss = distillation_loss(s["logits"], s["top"], s["idx"], temperature=c["temp"], weights=s["weights"], reduction=c["reduction"])
    if not c["bwd"]:
        return loss
    return (loss.detach(), *torch.autograd.grad(loss, (s["logits"],), s["dloss"]))


def _run_plain(s):
    c = s["case"]
    f = torch.float32
    if c["op"] == "embedding":
        table = s["table"].detach()
        ids = s["ids"].long()
        ok = ((ids >= 0) & (ids < c["V"])).unsqueeze(1)
        safe = ids.clamp(0, c["V"] - 1)
        out = torch.where(ok, table[safe].to(f) * c["scale"], torch.zeros((), device=table.device)).to(table.dtype)
        if not c["bwd"]:
            return out
        d = torch.where(ok, s["dout"].to(f) * c["scale"], torch.zeros((), device=table.device))
        grad = torch.zeros(c["V"], c["D"], dtype=f, device=table.device).index_add_(0, safe, d)
        return out, grad.to(table.dtype)
    if c["op"] == "adapter":
        T, K, N, r, G = (c[k] for k in ("T", "K", "N", "r", "G"))
        dt = s["x"].dtype
        x, w, A, B = s["x"].detach().to(f), s["w"].to(f), s["A"].detach().to(f), s["B"].detach().to(f)
        # the scaled one-hot row of each token's adapter; a token without one has none
        pick = (s["ids"].unsqueeze(1) == torch.arange(G, device=x.device)).to(f) * s["scales"]
        pick = pick.unsqueeze(2).expand(T, G, r).reshape(T, G * r)
        Acat = A.reshape(G * r, K)
        Bcat = B.permute(0, 2, 1).reshape(G * r, N)
        h = (x @ Acat.t()) * pick
        y = x @ w.t() + h @ Bcat
        if s["bias"] is not None:
            y = y + s["bias"].to(f)
        if not c["bwd"]:
            return y.to(dt)
        dy = s["dy"].to(f)
        dh = (dy @ Bcat.t()) * pick
        dx = dy @ w + dh @ Acat
        dA = (dh.t() @ x).reshape(G, r, K)
        dB = (h.t() @ dy).reshape(G, r, N).permute(0, 2, 1)
        return y.to(dt), dx.to(dt), dA.to(dt), dB.contiguous().to(dt)
    tau, V = c["temp"], c["V"]
    logits = s["logits"].detach()
    z = logits.to(f) / tau
    zmax = z.max(dim=1, keepdim=True).values
    ex = torch.exp(z - zmax)
    tot = ex.sum(dim=1, keepdim=True)
    idx = s["idx"].long()
    ok = (idx >= 0) & (idx < V)
    safe = idx.clamp(0, V - 1)
    t = torch.where(ok, s["top"].to(f) / tau, torch.full((), -math.inf, device=z.device))
    tmax = t.max(dim=1, keepdim=True).values
    tmax = torch.where(torch.isfinite(tmax), tmax, torch.zeros_like(tmax))
    te = torch.exp(t - tmax)
    tt = te.sum(dim=1, keepdim=True)
    some = tt > 0
    tt = torch.where(some, tt, torch.ones_like(tt))
    p = te / tt
    logq = torch.gather(z, 1, safe) - zmax - torch.log(tot)
    logp = t - tmax - torch.log(tt)
    row = (torch.where(p > 0, p * (logp - logq), torch.zeros_like(p))).sum(dim=1) * (tau * tau)
    wt = s["weights"] if s["weights"] is not None else torch.ones(c["N"], device=z.device)
    row = torch.where(wt != 0, row * wt, torch.zeros_like(row))
    den = wt.sum().clamp_min(1e-8) if c["reduction"] == "mean" else 1.0
    loss = row if c["reduction"] == "none" else row.sum() / den
    if not c["bwd"]:
        return loss
    k = torch.where(wt != 0, wt, torch.zeros_like(wt)) * (tau / den)
    if s["dloss"] is not None:
        k = k * s["dloss"]
    k = torch.where(some, k.unsqueeze(1), torch.zeros((), device=z.device))
    grad = (ex / tot).scatter_add_(1, safe, torch.where(ok, -p, torch.zeros_like(p))) * k
    return loss, grad.to(logits.dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "embedding":
        T, V, D = case["T"], case["V"], case["D"]
        ib = 4 if case["idx"] == "i32" else 8
        b = T * ib + min(T, V) * D * e + T * D * e
        fl = T * D
        if case["bwd"]:
            b += T * D * e + V * D * e
            fl += 2 * T * D
        return {"bytes": b, "flops": fl}
    if case["op"] == "adapter":
        T, K, N, r, G = (case[k] for k in ("T", "K", "N", "r", "G"))
        used = min(T, G)
        b = e * (T * K + N * K + used * r * (K + N) + T * N + (N if case["bias"] else 0)) + 8 * T + 4 * G
        fl = 2 * T * N * K + 2 * T * r * (N + K)
        if case["bwd"]:
            b += e * (T * N + T * K + G * r * (K + N))
            fl += 2 * T * N * K + 4 * T * r * (N + K)
        return {"bytes": b, "flops": fl}
    N, V, K = case["N"], case["V"], case["K"]
    b = N * V * e + N * K * (_SIZE[case["tdtype"]] + (4 if case["idx"] == "i32" else 8)) + 4 * N
    fl = 4 * N * V
    if case["bwd"]:
        b += N * V * e
        fl += 2 * N * V
    return {"bytes": b, "flops": fl}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64
    if case["op"] == "embedding":
        ids = s["ids"].cpu().numpy().astype(np.int64)
        table = s["table"].detach().cpu().to(d).numpy()
        out = np.zeros((case["T"], case["D"]))
        live = np.flatnonzero((ids >= 0) & (ids < case["V"]))
        out[live] = table[ids[live]] * case["scale"]
        if not case["bwd"]:
            return torch.from_numpy(out)
        dout = s["dout"].cpu().to(d).numpy()
        grad = np.zeros_like(table)
        order = live[np.argsort(ids[live], kind="stable")]
        if order.size:
            first = np.flatnonzero(np.r_[True, np.diff(ids[order]) != 0])
            grad[ids[order][first]] = np.add.reduceat(dout[order], first, axis=0) * case["scale"]
        return torch.from_numpy(out), torch.from_numpy(grad)
    if case["op"] == "adapter":
        x, w = s["x"].detach().to(d), s["w"].to(d)
        ids, sc = s["ids"].cpu().tolist(), s["scales"].to(d)
        y = torch.addmm(s["bias"].to(d), x, w.t()) if s["bias"] is not None else torch.mm(x, w.t())
        rows = {}
        for t, a in enumerate(ids):
            if a >= 0:
                rows.setdefault(a, []).append(t)
        bwd = case["bwd"]
        if bwd:
            dy = s["dy"].to(d)
            dx = torch.mm(dy, w)
            dA, dB = torch.zeros_like(s["A"], dtype=d), torch.zeros_like(s["B"], dtype=d)
        for a, tt in rows.items():
            tt = torch.tensor(tt, device=x.device)
            Aa, Ba = s["A"][a].detach().to(d), s["B"][a].detach().to(d)
            h = torch.mm(x[tt], Aa.t().contiguous()) * sc[a]
            y[tt] += torch.mm(h, Ba.t().contiguous())
            if bwd:
                dh = torch.mm(dy[tt], Ba) * sc[a]
                dx[tt] += torch.mm(dh, Aa)
                dA[a] = torch.mm(dh.t().contiguous(), x[tt])
                dB[a] = torch.mm(dy[tt].t().contiguous(), h)
        return (y, dx, dA, dB) if bwd else y
    N, V, tau = case["N"], case["V"], case["temp"]
    idx, top = s["idx"].long(), s["top"].to(d) / tau
    wt = (s["weights"] if s["weights"] is not None else torch.ones(N, device="cuda")).to(d)
    den = wt.sum().clamp_min(1e-8) if case["reduction"] == "mean" else torch.ones((), dtype=d, device="cuda")
    rows = torch.zeros(N, dtype=d, device="cuda")
    grad = torch.zeros(N, V, dtype=d, device="cuda") if case["bwd"] else None
    step = max(1, (1 << 26) // V)
    for a in range(0, N, step):
        b = min(N, a + step)
        logq = torch.log_softmax(s["logits"][a:b].detach().to(d) / tau, dim=1)
        ok = (idx[a:b] >= 0) & (idx[a:b] < V)
        some = ok.any(dim=1)
        logp = torch.log_softmax(torch.where(ok, top[a:b], torch.full_like(top[a:b], -1e300)), dim=1)
        p = torch.where(ok, torch.exp(logp), torch.zeros_like(logp))
        at = idx[a:b].clamp(0, V - 1)
        kl = torch.where(p > 0, p * (logp - torch.gather(logq, 1, at)), torch.zeros_like(p)).sum(dim=1)
        rows[a:b] = torch.where(some, kl * tau * tau * wt[a:b], torch.zeros_like(kl))
        if grad is not None:
            gr = torch.exp(logq)
            gr.scatter_add_(1, at, -p)
            k = torch.where(some, wt[a:b] * tau / den, torch.zeros_like(kl))
            if s["dloss"] is not None:
                k = k * s["dloss"][a:b].to(d)
            grad[a:b] = gr * k.unsqueeze(1)
    loss = rows if case["reduction"] == "none" else rows.sum() / den
    return (loss, grad) if grad is not None else loss
