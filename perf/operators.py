"""Workloads of the operators that stand around the quantized products of a mixture-of-experts or adapted model: routing to
experts in groups, low-rank adapters of many requests beside a shared projection, and the same beside an expert stack.

`own` chooses what `run` computes them with: False, elementary torch operations in 32 bits (64 where a selection hangs on the last
bits); True, the package's operators as a user calls them. Sizes: the hidden and feed-forward widths of the package's benchmark and
tests, 128 experts of width 768 on 2048, ranks from 4 to 64."""
import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _route(T, E, groups, top_groups, k, scoring, bias, norm, dtype, group_top, grad=False):
    return dict(op="route", T=T, E=E, groups=groups, top_groups=top_groups, k=k, scoring=scoring, bias=bias, norm=norm,
                dtype=dtype, group_top=group_top, grad=grad)


def _lora(T, K, N, r, G, dtype, params, grad=False):
    return dict(op="lora", T=T, K=K, N=N, r=r, G=G, dtype=dtype, params=params, grad=grad)


def _experts(T, k, E, K, N, r, G, dtype, params, shared, grad=False):
    return dict(op="experts", T=T, k=k, E=E, K=K, N=N, r=r, G=G, dtype=dtype, params=params, shared=shared, grad=grad)


def listed():
    named = {
        # one token of a decode step: 256 experts in 8 groups, sigmoid scores with a bias for balance
        "route_token": _route(1, 256, 8, 4, 8, "sigmoid", True, True, "bf16", 2),
        # a batch of decoded tokens of a model that keeps the groups with the best expert, weights not renormalised
        "route_batch": _route(61, 160, 8, 3, 6, "softmax", False, False, "f16", 1),
        # a long prompt, router computed in float32
        "route_prompt": _route(16384, 256, 8, 4, 8, "sigmoid", True, True, "f32", 2),
        # a training step's routing and its gradient, 128 experts without groups
        "route_train": _route(8192, 128, 1, 1, 8, "softmax", False, True, "bf16", 1, grad=True),
        # one request's token on the attention projection of the benchmark's decode shape
        "lora_token": _lora(1, 4096, 4096, 16, 8, "bf16", "bf16"),
        # a batch of requests with adapters of their own on an up projection, some without one
        "lora_batch": _lora(61, 4096, 14336, 32, 32, "f16", "f16"),
        # prompts of several requests side by side
        "lora_prompt": _lora(8192, 4096, 4096, 64, 8, "bf16", "bf16"),
        # a training step of one adapter held in float32 beside a frozen up projection
        "lora_train": _lora(4096, 4096, 14336, 16, 1, "bf16", "f32", grad=True),
        # a few decoded tokens: gate | up of 128 experts, each request's adapter has a pair of matrices for every expert
        "experts_batch": _experts(8, 8, 128, 2048, 1536, 8, 4, "bf16", "bf16", True),
        # the down product of a prompt, a row of its own for every slot
        "experts_prompt": _experts(4096, 8, 128, 768, 2048, 16, 2, "f16", "f16", False),
        # a training step of adapters on gate | up
        "experts_train": _experts(509, 8, 128, 2048, 1536, 16, 1, "bf16", "f32", True, grad=True),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("route", "lora", "experts"))
    grad = rng.random() < 0.4
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        size = _log(rng, 8, 256 // groups)
        E = groups * size
        top_groups = rng.randint(1, groups)
        k = rng.randint(1, min(12, top_groups * size))
        scoring = rng.choice(("sigmoid", "softmax"))
        T = min(_log(rng, 1, 16384), 16384 * 128 // E if grad else 16384)
        return _route(T, E, groups, top_groups, k, scoring, rng.random() < 0.5, rng.random() < 0.7,
                      rng.choice(("f32", "f16", "bf16")), rng.choice((1, 2)), grad)
    dtype = rng.choice(("bf16", "f16"))
    params = rng.choice((dtype, "f32")) if grad else dtype
    width = lambda: rng.choice((256, 768, 1024, 1536, 2048, 4096, 8 * rng.randint(32, 512)))  # noqa: E731
    r = rng.choice((4, 8, 12, 16, 24, 32, 48, 64))
    if op == "lora":
        return _lora(_log(rng, 1, 4096 if grad else 8192), width(), width() + rng.choice((0, 0, 0, 1, 20)), r,
                     rng.choice((1, 2, 3)) if grad else _log(rng, 1, 48), dtype, params, grad)
    K = rng.choice((256, 768, 1024, 2048))
    return _experts(_log(rng, 1, 509 if grad else 2048), rng.randint(1, 8), rng.choice((8, 32, 60, 128)), K, rng.choice((512, 768, 1536)),
                    min(r, 16), 1 if grad else rng.randint(1, 4), dtype, params, rng.random() < 0.5, grad)


# ------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    T = case["T"]
    if case["op"] == "route":
        s = dict(case=case, logits=(randn(T, case["E"]) * 1.5).to(dt), bias=randn(case["E"]) * 0.1 if case["bias"] else None)
        if case["grad"]:
            s["logits"].requires_grad_()
            s["dw"] = randn(T, case["k"])
        return s
    K, N, r, G = case["K"], case["N"], case["r"], case["G"]
    pt = _DT[case["params"]]
    if case["op"] == "lora":
        x, y = randn(T, K).to(dt), randn(T, N).to(dt)
        a, b = (randn(G, r, K) * K ** -0.5).to(pt), (randn(G, N, r) * 0.05).to(pt)
    else:
        k, E = case["k"], case["E"]
        x = randn(T, K) if case["shared"] else randn(T, k, K)
        x, y = x.to(dt), randn(T, k, N).to(dt)
        a, b = (randn(G, E, r, K) * K ** -0.5).to(pt), (randn(G, E, N, r) * 0.05).to(pt)
    s = dict(case=case, x=x, y=y, a=a, b=b, scaling=1.0 + torch.rand(G, device="cuda", generator=g))
    # a batch of up to 64 tokens has a request for each; beyond that the rows of a request lie side by side, runs with one adapter, as
    # prompts of different lengths have them; one request in sixteen has none
    rng = np.random.RandomState(seed % (1 << 31))
    runs = T if T <= 64 else 3 * G + 5
    cuts = np.sort(rng.choice(np.arange(1, T), size=min(runs, T) - 1, replace=False)) if T > 1 else np.zeros(0, np.int64)
    of_run = rng.randint(0, G, size=len(cuts) + 1)
    of_run = np.where(rng.randint(0, 16, size=len(cuts) + 1) == 0, -1, of_run) if not case["grad"] and T > 1 else of_run
    ids = of_run[np.searchsorted(cuts, np.arange(T), side="right")].astype(np.int32)
    s["adapter_ids"] = torch.from_numpy(ids).cuda() if G > 1 else None
    if case["op"] == "experts":
        # every token takes k different experts
        s["indices"] = torch.argsort(torch.rand(T, case["E"], device="cuda", generator=g), dim=1)[:, :case["k"]].to(torch.int32).contiguous()
    if case["grad"]:
        for t in (s["x"], s["a"], s["b"]):
            t.requires_grad_()
        s["dy"] = randn(*y.shape).to(dt)
    return s


# -------------------------------------------------------------------------------------------------------- plain forms
def _scores(x, scoring):
    if scoring == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    e = torch.exp(x - x.amax(dim=1, keepdim=True))
    return e / e.sum(dim=1, keepdim=True)


def _plain_route(s):
    c = s["case"]
    T, E, G = c["T"], c["E"], c["groups"]
    logits = s["logits"].detach()
    # what is ranked stands in 64 bits: neighbours may differ in the last ones
    key = _scores(logits.double(), c["scoring"])
    if s["bias"] is not None:
        key = key + s["bias"].double()
    if G > 1:
        best = torch.sort(key.view(T, G, E // G), dim=2, descending=True).values[:, :, :c["group_top"]].sum(dim=2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        mask = (kept[:, :, None] == torch.arange(G, device=kept.device)).any(dim=1)
        mask = mask[:, :, None].expand(T, G, E // G).reshape(T, E)
    if s["bias"] is None:
        key = logits.double()  # the scores rise with the logits
    if G > 1:
        key = torch.where(mask, key, -torch.inf)
    idx = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :c["k"]]
    score = _scores(logits.float(), c["scoring"])
    picked = torch.gather(score, 1, idx)
    total = picked.sum(dim=1, keepdim=True) + 1e-20 if c["norm"] else 1.0
    out = {"indices": idx.to(torch.int32), "weights": picked / total * 2.5}
    if not c["grad"]:
        return out
    dw = s["dw"] * 2.5
    if c["norm"]:
        dw = (dw - (dw * (picked / total)).sum(dim=1, keepdim=True)) / total
    ds = torch.zeros_like(score).scatter_(1, idx, dw)
    if c["scoring"] == "sigmoid":
        dl = ds * score * (1.0 - score)
    else:
        dl = score * (ds - (ds * score).sum(dim=1, keepdim=True))
    return dict(out, dlogits=dl.to(logits.dtype))


def _plain_lora(s):
    """All adapters' products side by side, the others' columns times zero."""
    c = s["case"]
    x, y, a, b = s["x"].detach(), s["y"], s["a"].detach(), s["b"].detach()
    T, K, N, r, G = c["T"], c["K"], c["N"], c["r"], c["G"]
    slots = c.get("k", 1)
    ids = torch.zeros(T, dtype=torch.int64, device=x.device) if s["adapter_ids"] is None else s["adapter_ids"].long()
    own_rows = c["op"] == "experts" and not c["shared"]
    group, n = ids, G
    factor = torch.where(ids >= 0, s["scaling"][ids.clamp(min=0)], 0.0)
    if c["op"] == "experts":
        n = G * c["E"]
        group = (ids[:, None] * c["E"] + s["indices"].long()).reshape(-1)
        factor = factor.repeat_interleave(slots)
    mask = (group[:, None] == torch.arange(n, device=x.device)).float() * factor[:, None]
    A, B = a.float().reshape(n * r, K), b.float().reshape(n, N, r).transpose(1, 2).reshape(n * r, N)
    x32 = x.float().reshape(-1, K)
    u = x32 @ A.T
    if not own_rows and slots > 1:
        u = u.repeat_interleave(slots, dim=0)
    u = (u.view(-1, n, r) * mask[:, :, None]).view(-1, n * r)
    out = (y.float().reshape(-1, N) + u @ B).to(y.dtype).view(y.shape)
    if not c["grad"]:
        return {"y": out}
    dy = s["dy"].float().reshape(-1, N)
    v = ((dy @ B.T).view(-1, n, r) * mask[:, :, None]).view(-1, n * r)
    db = (u.T @ dy).view(n, r, N).transpose(1, 2).reshape(b.shape)
    if not own_rows and slots > 1:
        v = v.view(T, slots, n * r).sum(dim=1)
    return {"y": out, "dx": (v @ A).to(x.dtype).view(x.shape), "da": (v.T @ x32).view(a.shape).to(a.dtype), "db": db.to(b.dtype)}


# ------------------------------------------------------------------------------------------------------- own operators
def _own(s):
    c = s["case"]
    if c["op"] == "route":
        from mlx_kquant_b200.moe import moe_router_grouped

        idx, w = moe_router_grouped(s["logits"], c["k"], c["groups"], c["top_groups"], scoring=c["scoring"], bias=s["bias"],
                                    group_top=c["group_top"], norm_topk_prob=c["norm"], scale=2.5)
        out = {"indices": idx, "weights": w}
        if c["grad"]:
            out["dlogits"] = torch.autograd.grad(w, s["logits"], s["dw"])[0]
        return out
    if c["op"] == "lora":
        from mlx_kquant_b200 import lora_update

        y = lora_update(s["y"], s["x"], s["a"], s["b"], s["adapter_ids"], s["scaling"])
    else:
        from mlx_kquant_b200.moe import gather_lora_update

        y = gather_lora_update(s["y"], s["x"], s["a"], s["b"], s["indices"], s["adapter_ids"], s["scaling"])
    if not c["grad"]:
        return {"y": y}
    dx, da, db = torch.autograd.grad(y, (s["x"], s["a"], s["b"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "da": da, "db": db}


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return _plain_route(s) if s["case"]["op"] == "route" else _plain_lora(s)


def work(case):
    """Each input read once, each output written once; of the adapters those that some row uses."""
    T, e = case["T"], _SIZE[case["dtype"]]
    if case["op"] == "route":
        E, k = case["E"], case["k"]
        nbytes, flops = T * E * e + T * k * 8, T * E * 8
        if case["grad"]:
            nbytes, flops = nbytes + T * E * e + T * k * 4, flops + T * E * 4
        return {"bytes": nbytes, "flops": flops}
    K, N, r, p = case["K"], case["N"], case["r"], _SIZE[case["params"]]
    rows, groups = T * case.get("k", 1), case["G"] * case.get("E", 1)
    used = groups if case["grad"] else groups * (1.0 - (1.0 - 1.0 / groups) ** rows)
    x_rows = T if case.get("shared", True) else rows
    nbytes = x_rows * K * e + 2 * rows * N * e + used * r * (K + N) * p + 4 * rows
    flops = 2 * rows * r * (K + N)
    if case["grad"]:
        nbytes += rows * N * e + x_rows * K * e + groups * r * (K + N) * p
        flops *= 3
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_route(s):
    c = s["case"]
    x = s["logits"].detach().double().cpu().numpy()
    T, E, G = c["T"], c["E"], c["groups"]
    if c["scoring"] == "sigmoid":
        p = np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))
    else:
        p = np.exp(x - x.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    bias = None if s["bias"] is None else s["bias"].double().cpu().numpy()
    rank = p if bias is None else p + bias
    alive = np.ones((T, E), bool)
    if G > 1:
        top = -np.sort(-rank.reshape(T, G, E // G), axis=2)[:, :, :c["group_top"]]
        order = np.argsort(-top.sum(2), axis=1, kind="stable")[:, :c["top_groups"]]
        alive = np.zeros((T, G), bool)
        np.put_along_axis(alive, order, True, axis=1)
        alive = np.repeat(alive, E // G, axis=1)
    rank = np.where(alive, x if bias is None else rank, -np.inf)
    idx = np.argsort(-rank, axis=1, kind="stable")[:, :c["k"]]
    q = np.take_along_axis(p, idx, axis=1)
    S = q.sum(1, keepdims=True) + 1e-20 if c["norm"] else np.ones((T, 1))
    out = {"indices": torch.from_numpy(idx.astype(np.int32)), "weights": torch.from_numpy(2.5 * q / S)}
    if c["grad"]:
        dw = 2.5 * s["dw"].double().cpu().numpy()
        if c["norm"]:
            dw = (dw - (dw * q / S).sum(1, keepdims=True)) / S
        dl = np.zeros((T, E))
        if c["scoring"] == "sigmoid":
            np.put_along_axis(dl, idx, dw * q * (1 - q), axis=1)
        else:
            np.put_along_axis(dl, idx, dw * q, axis=1)
            dl -= p * (dw * q).sum(1, keepdims=True)
        out["dlogits"] = torch.from_numpy(dl)
    return out


def _exact_lora(s):
    """Adapter after adapter, the rows of each picked out."""
    c = s["case"]
    T, K, N, r, G = c["T"], c["K"], c["N"], c["r"], c["G"]
    slots, E = c.get("k", 1), c.get("E", 1)
    x, a, b = s["x"].detach().double(), s["a"].detach().double().reshape(-1, r, K), s["b"].detach().double().reshape(-1, N, r)
    per_slot = c["op"] == "experts" and not c["shared"]
    xr = x.reshape(-1, K)
    y = s["y"].double().reshape(-1, N).clone()
    dy = s["dy"].double().reshape(-1, N) if c["grad"] else None
    dx, da, db = torch.zeros_like(xr), torch.zeros_like(a), torch.zeros_like(b)
    ids = np.zeros(T, np.int64) if s["adapter_ids"] is None else s["adapter_ids"].cpu().numpy().astype(np.int64)
    owner = np.repeat(ids, slots)
    which = s["indices"].cpu().numpy().reshape(-1) if c["op"] == "experts" else np.zeros(T, np.int64)
    group = np.where(owner >= 0, owner * E + which, -1)
    for g in np.unique(group[group >= 0]):
        rows = torch.from_numpy(np.nonzero(group == g)[0]).to(x.device)
        src = rows if per_slot else rows // slots
        f = s["scaling"][int(g) // E].double()
        u = xr[src] @ a[g].T
        y[rows] += f * (u @ b[g].T)
        if c["grad"]:
            v = f * (dy[rows] @ b[g])
            dx.index_add_(0, src, v @ a[g])
            da[g] = v.T @ xr[src]
            db[g] = f * (dy[rows].T @ u)
    out = {"y": y.view(s["y"].shape)}
    if c["grad"]:
        out.update(dx=dx.view(x.shape), da=da.view(s["a"].shape), db=db.view(s["b"].shape))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_route(s) if case["op"] == "route" else _exact_lora(s)
