"""Cases that time and check the routing and adapter operators of libhymoe.

Four operators: `route` (scores, groups, top-k and weights of every token), `route_backward`
(its gradient to the logits), `adapt` (low-rank adapters of many requests beside a projection
they share) and `adapt_backward` (gradients of the inputs and of the adapters).  `run` computes
them in elementary torch operations, or, with `own` set, through the library's public calls.
"""
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
BIG = torch.finfo(torch.float32).max


def _route(name, op, tokens, experts, topk, score, dtype, **more):
    case = {"name": name, "op": op, "tokens": tokens, "experts": experts, "topk": topk, "score": score,
            "type": dtype, "bias": False, "groups": 0, "kept": 0, "group_score": "max", "norm": True,
            "scale": 1.0, "scores": False, "closed": 0.0}
    case.update(more)
    return case


def _adapt(name, op, tokens, n_in, n_out, rank, adapters, ids, x, w, y):
    return {"name": name, "op": op, "tokens": tokens, "in": n_in, "out": n_out, "rank": rank,
            "adapters": adapters, "ids": ids, "x": x, "w": w, "y": y}


def listed():
    return [
        # one decoding step of eight sequences, the block's own router: latency
        _route("route decode", "route", 8, 64, 8, "softmax", "f32"),
        # an image's tokens through the block's router, selection corrected by a balance bias;
        # the scores go on to a balance loss
        _route("route block", "route", 4096, 64, 8, "softmax", "f32", bias=True, scores=True),
        # a long odd batch over many experts in groups, bf16 logits from a mixed-precision router
        _route("route groups", "route", 8323, 256, 8, "sigmoid", "bf16", bias=True, groups=8, kept=4,
               group_score="top2", scale=2.5),
        # the tokens of a training step at once; some experts closed to some tokens
        _route("route large", "route", 131072, 128, 6, "sigmoid", "bf16", bias=True, closed=0.05),
        # the gradient of a step of the block's router, with a balance loss on its scores
        _route("route grad block", "route_backward", 4096, 64, 8, "softmax", "f32", scores=True, norm=False),
        # the gradient over a training step's tokens
        _route("route grad large", "route_backward", 65536, 256, 8, "sigmoid", "bf16", scale=2.5),
        # one token of one request: latency
        _adapt("adapt token", "adapt", 1, 4096, 4096, 16, 4, "requests", "f16", "f16", "f16"),
        # a decoding step of 64 requests, each with an adapter of its own choice
        _adapt("adapt decode", "adapt", 64, 4096, 6144, 32, 32, "mixed", "bf16", "bf16", "bf16"),
        # one image's sequence in a few requests, fp32 result beside the block's fp32 rows
        _adapt("adapt image", "adapt", 4160, 4096, 4096, 16, 3, "requests", "f16", "f16", "f32"),
        # the largest batch of the block, tokens of sixteen adapters in any order
        _adapt("adapt large", "adapt", 8192, 4096, 6144, 64, 16, "mixed", "bf16", "bf16", "bf16"),
        # fine-tuning on short captions: a small batch of one adapter
        _adapt("adapt grad small", "adapt_backward", 77, 4096, 4096, 16, 1, "requests", "bf16", "bf16", "bf16"),
        # several adapters trained together on one large batch
        _adapt("adapt grad large", "adapt_backward", 8192, 4096, 6144, 64, 8, "requests", "bf16", "bf16", "bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number of lo..hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["route", "route", "route_backward", "adapt", "adapt", "adapt_backward"])
    if op.startswith("route"):
        while True:
            experts = rng.choice([8, 16, 60, 64, 72, 96, 128, 160, 255, 256, 384, 512])
            topk = rng.randint(1, min(16, experts))
            groups = rng.choice([0, 0, 2, 4, 8])
            if groups and experts % groups:
                groups = 0
            kept = rng.randint(1, groups) if groups else 0
            tokens = _log(rng, 1, 131072)
            if tokens * experts <= 131072 * 128:
                break
        score = rng.choice(["softmax", "sigmoid"])
        return {**_route("", op, tokens, experts, topk, score, rng.choice(["f32", "f16", "bf16"]),
                         bias=rng.random() < 0.5, groups=groups, kept=kept,
                         group_score=rng.choice(["max", "top2"]), norm=rng.random() < 0.6,
                         scale=rng.choice([1.0, 2.5, 16.0]), scores=rng.random() < 0.4,
                         closed=rng.choice([0.0, 0.0, 0.1, 0.9])), "name": "drawn"}
    while True:
        n_in, n_out = _log(rng, 64, 8192), _log(rng, 64, 8192)
        if rng.random() < 0.8:  # rows of whole 16-byte pieces, as real projections have them
            n_in, n_out = max(64, n_in // 8 * 8), max(64, n_out // 8 * 8)
        rank = rng.choice([4, 8, 8, 16, 16, 32, 32, 64, 64, 128, rng.randint(1, 128)])
        adapters, tokens = _log(rng, 1, 64), _log(rng, 1, 8192)
        # the plain form multiplies every token with every adapter
        if (tokens * adapters * rank * (n_in + n_out) <= 8192 * 8 * 64 * 10240
                and tokens * (n_in + n_out) <= 8192 * 10240 and tokens * adapters * rank <= 8192 * 1024):
            break
    w = rng.choice(["f16", "bf16"])
    return {**_adapt("", op, tokens, n_in, n_out, rank, adapters, rng.choice(["requests", "mixed"]),
                     rng.choice([w, w, "f32"]), w, rng.choice([w, w, "f32"])), "name": "drawn"}


# ---------------------------------------------------------------- inputs


def _normal(g, shape, std, dtype):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    T = case["tokens"]
    if case["op"].startswith("route"):
        E, K = case["experts"], case["topk"]
        # every expert has its own mean logit: routers do not spread evenly
        z = torch.randn((T, E), generator=g, device="cuda") * 1.5 + torch.randn((1, E), generator=g, device="cuda")
        if case["closed"]:
            z = z.masked_fill(torch.rand((T, E), generator=g, device="cuda") < case["closed"], float("-inf"))
            if T > 1:
                z[T // 2] = float("-inf")  # a padded token: nothing is open
        s = {"case": case, "logits": z.to(TYPES[case["type"]]), "bias": None}
        if case["bias"]:
            s["bias"] = torch.randn((E,), generator=g, device="cuda") * (0.1 if case["score"] == "sigmoid" else 0.02)
        if case["op"] == "route_backward":
            s["idx"] = _route_plain(s["logits"], s["bias"], case)["idx"]
            s["d_weights"] = torch.randn((T, K), generator=g, device="cuda")
            s["d_scores"] = torch.randn((T, E), generator=g, device="cuda") * 0.1 if case["scores"] else None
        return s
    n, r, n_in, n_out = case["adapters"], case["rank"], case["in"], case["out"]
    if case["ids"] == "mixed":  # any order; a few tokens have no adapter
        ids = torch.randint(0, n, (T,), generator=g, device="cuda")
        ids = ids.masked_fill(torch.rand((T,), generator=g, device="cuda") < 0.05, -1)
    else:  # requests one after another, each with an adapter
        cuts = torch.sort(torch.randint(0, T, (max(1, 2 * n),), generator=g, device="cuda")).values
        ids = torch.randint(0, n, (max(1, 2 * n) + 1,), generator=g, device="cuda")[
            torch.bucketize(torch.arange(T, device="cuda"), cuts, right=True)]
    w = TYPES[case["w"]]
    s = {"case": case, "ids": ids.to(torch.int32),
         "a": _normal(g, (n, r, n_in), n_in ** -0.5, w), "b": _normal(g, (n, n_out, r), 0.02, w),
         "scale": torch.rand((n,), generator=g, device="cuda") + 0.5,
         "x": _normal(g, (T, n_in), 1.0, TYPES[case["x"]])}
    if case["op"] == "adapt":
        s["base"] = _normal(g, (T, n_out), 0.3, TYPES[case["y"]])
    else:
        s["dy"] = _normal(g, (T, n_out), 1.0, TYPES[case["y"]])
        s["base"] = _normal(g, (T, n_in), 0.3, TYPES[case["x"]])
    return s


# ---------------------------------------------------------------- the plain forms


def _scores_plain(logits, case):
    """Scores in 64 bits: the order of two experts can hang on their last bits."""
    z = logits.double()
    z = torch.where(torch.isnan(z), torch.full_like(z, float("-inf")), z).clamp(max=BIG)
    is_open = z > float("-inf")
    if case["score"] == "sigmoid":
        return torch.where(is_open, 1.0 / (1.0 + torch.exp(-z)), torch.zeros_like(z)), z, is_open
    m = z.max(dim=1, keepdim=True).values
    e = torch.where(is_open, torch.exp(z - m), torch.zeros_like(z))
    return e / e.sum(dim=1, keepdim=True).clamp(min=1.0), z, is_open


def _route_plain(logits, bias, case):
    s, z, is_open = _scores_plain(logits, case)
    T, E = s.shape
    K, G = case["topk"], case["groups"]
    closed = torch.full_like(s, float("-inf"))
    c = torch.where(is_open, s if bias is None else s + bias.double(), closed)
    if G:
        best = torch.sort(c.view(T, G, E // G), dim=2, descending=True).values
        value = best[:, :, 0]
        if case["group_score"] == "top2" and E // G > 1:
            value = value + torch.where(best[:, :, 1] > float("-inf"), best[:, :, 1], torch.zeros_like(value))
        order = torch.sort(value, dim=1, descending=True, stable=True).indices[:, :case["kept"]]
        kept = torch.zeros((T, G), dtype=torch.bool, device=s.device).scatter_(1, order, True)
        c = torch.where(kept.repeat_interleave(E // G, dim=1), c, closed)
    top = torch.sort(c, dim=1, descending=True, stable=True)
    picked = top.values[:, :K] > float("-inf")
    idx = top.indices[:, :K]
    w = torch.where(picked, s.gather(1, idx), torch.zeros((), dtype=s.dtype, device=s.device))
    if case["norm"]:
        w = w / w.sum(dim=1, keepdim=True).clamp(min=1e-300)
    out = {"idx": torch.where(picked, idx, torch.full_like(idx, -1)).to(torch.int32),
           "weights": (w * case["scale"]).float()}
    out["counts"] = torch.zeros((E,), dtype=torch.int32, device=s.device).scatter_add_(
        0, idx.reshape(-1), picked.reshape(-1).to(torch.int32))
    if case["scores"]:
        out["scores"] = s.float()
    return out


def _route_backward_plain(s):
    case = s["case"]
    p, z, is_open = _scores_plain(s["logits"], case)
    picked = s["idx"] >= 0
    idx = s["idx"].clamp(min=0).long()
    dw = torch.where(picked, s["d_weights"].double(), torch.zeros((), dtype=p.dtype, device=p.device)) * case["scale"]
    sel = torch.where(picked, p.gather(1, idx), torch.zeros_like(dw))
    if case["norm"]:
        total = sel.sum(dim=1, keepdim=True).clamp(min=1e-300)
        dw = (dw - (dw * sel).sum(dim=1, keepdim=True) / total) / total
    ds = torch.zeros_like(p).scatter_add_(1, idx, torch.where(picked, dw, torch.zeros_like(dw)))
    if s["d_scores"] is not None:
        ds = ds + s["d_scores"].double()
    if case["score"] == "sigmoid":
        d = ds * p * (1.0 - p)
    else:
        d = p * (ds - (ds * p).sum(dim=1, keepdim=True))
    return torch.where(is_open, d, torch.zeros_like(d)).to(s["logits"].dtype)


def _low_plain(x, weight, ids, scale):
    """[T, n * r]: every token's product with its own adapter's rows, zero at the others'."""
    n = weight.shape[0]
    v = x.float() @ weight.float().reshape(n * weight.shape[1], -1).t()
    hot = (ids[:, None] == torch.arange(n, device=ids.device)[None, :]) * scale[None, :]
    return (v.view(x.shape[0], n, -1) * hot[:, :, None]).view(x.shape[0], -1)


def _adapt_plain(s):
    v = _low_plain(s["x"], s["a"], s["ids"], s["scale"])
    wide = s["b"].float().permute(0, 2, 1).reshape(v.shape[1], -1)
    return (s["base"].float() + v @ wide).to(s["base"].dtype)


def _adapt_backward_plain(s):
    n, r, n_in = s["a"].shape
    v = _low_plain(s["x"], s["a"], s["ids"], s["scale"])
    u = _low_plain(s["dy"], s["b"].permute(0, 2, 1), s["ids"], s["scale"])
    dx = (s["base"].float() + u @ s["a"].float().reshape(n * r, n_in)).to(s["base"].dtype)
    da = (u.t() @ s["x"].float()).view(n, r, n_in)
    db = (v.t() @ s["dy"].float()).view(n, r, -1).permute(0, 2, 1).contiguous()
    return {"dx": dx, "da": da, "db": db}


# ---------------------------------------------------------------- the library's calls


def _handle(s):
    """The plan or adapter set that a user's program makes once and keeps."""
    if "handle" not in s:
        package = os.path.join(ROOT, "hunyuan-image-3-80b.cpp_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        import hymoe
        c = s["case"]
        if c["op"].startswith("route"):
            s["handle"] = hymoe.Gate(c["experts"], c["topk"], score=c["score"],
                                     group=(c["groups"], c["kept"]) if c["groups"] else None,
                                     group_score=c["group_score"], norm_topk_prob=c["norm"], scale=c["scale"])
        else:
            s["handle"] = hymoe.Adapters(s["a"], s["b"], s["scale"])
    return s["handle"]


def _run_own(s):
    c, h = s["case"], _handle(s)
    if c["op"] == "route":
        return h.route(s["logits"], bias=s["bias"], scores=c["scores"], counts=True)
    if c["op"] == "route_backward":
        return h.backward(s["logits"], s["idx"], s["d_weights"], d_scores=s["d_scores"])
    if c["op"] == "adapt":
        return h.apply(s["x"], s["ids"], base=s["base"])
    return h.backward(s["x"], s["dy"], s["ids"], base=s["base"])


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "route":
        return _route_plain(state["logits"], state["bias"], state["case"])
    if op == "route_backward":
        return _route_backward_plain(state)
    return _adapt_plain(state) if op == "adapt" else _adapt_backward_plain(state)


def work(case):
    T = case["tokens"]
    if case["op"].startswith("route"):
        E, K, b = case["experts"], case["topk"], BYTES[case["type"]]
        size = T * E * b + T * K * 8 + (T * E * 4 if case["scores"] else 0)
        if case["op"] == "route":
            # a score and K comparisons for each expert
            return {"bytes": size + E * 4 * (2 if case["bias"] else 1), "flops": T * E * (8 + K)}
        return {"bytes": size + T * E * b, "flops": T * E * 12}
    n, r, i, o = case["adapters"], case["rank"], case["in"], case["out"]
    used = min(n, T)
    weights = used * r * (i + o) * BYTES[case["w"]] + n * 4 + T * 4
    if case["op"] == "adapt":
        return {"bytes": T * i * BYTES[case["x"]] + 2 * T * o * BYTES[case["y"]] + weights, "flops": 2 * T * r * (i + o)}
    return {"bytes": 3 * T * i * BYTES[case["x"]] + T * o * BYTES[case["y"]] + weights + n * r * (i + o) * 4,
            "flops": 2 * T * r * (3 * i + 2 * o)}


# ---------------------------------------------------------------- 64 bits, from the definitions


def _exact_route(s):
    """Selected experts and their weights through logarithms of the scores."""
    c = s["case"]
    z = s["logits"].double()
    z = z.masked_fill(z.isnan(), float("-inf")).clamp(max=BIG)
    T, E = z.shape
    shut = z.isinf()
    log_s = (torch.nn.functional.logsigmoid(z) if c["score"] == "sigmoid" else
             z - torch.logsumexp(z.masked_fill(shut.all(1, keepdim=True), 0.0), 1, keepdim=True))
    score = log_s.exp().masked_fill(shut, 0.0)
    choice = (score + s["bias"].double() if s["bias"] is not None else score).masked_fill(shut, float("-inf"))
    if c["groups"]:
        G = c["groups"]
        two = choice.view(T, G, E // G).topk(min(2, E // G), dim=2).values
        value = two[:, :, 0] if c["group_score"] == "max" else two[:, :, :1].sum(2) + two[:, :, 1:].clamp(min=-1e300).sum(2).masked_fill((two[:, :, 1:] < -1e200).any(2), 0.0)
        rank = (value[:, None, :] > value[:, :, None]).sum(2) + ((value[:, None, :] == value[:, :, None]) & (
            torch.arange(G, device=z.device)[None, None, :] < torch.arange(G, device=z.device)[None, :, None])).sum(2)
        choice = choice.masked_fill((rank >= c["kept"])[:, :, None].expand(T, G, E // G).reshape(T, E), float("-inf"))
    value, idx = choice.sort(dim=1, descending=True, stable=True)
    value, idx = value[:, :c["topk"]], idx[:, :c["topk"]]
    none = value == float("-inf")
    log_w = log_s.gather(1, idx).masked_fill(none, float("-inf"))
    if c["norm"]:
        log_w = log_w - torch.logsumexp(log_w.masked_fill(none.all(1, keepdim=True), 0.0), 1, keepdim=True)
    w = log_w.exp().masked_fill(none, 0.0) * c["scale"]
    out = {"idx": None, "weights": w, "counts": None}
    if c["scores"]:
        out["scores"] = score
    return out


def _exact_route_backward(s):
    """The weights' definition written once more in 64 bits and differentiated by torch."""
    c = s["case"]
    z = s["logits"].double()
    z = z.masked_fill(z.isnan(), float("-inf")).clamp(max=BIG)
    shut = z.isinf()
    with torch.enable_grad():
        leaf = z.masked_fill(shut, -1e4).requires_grad_()
        s_all = (leaf.sigmoid() if c["score"] == "sigmoid" else leaf.softmax(1)).masked_fill(shut, 0.0)
        sel = s_all.gather(1, s["idx"].clamp(min=0).long()).masked_fill(s["idx"] < 0, 0.0)
        w = sel / sel.sum(1, keepdim=True).clamp(min=1e-300) if c["norm"] else sel
        loss = (w * s["d_weights"].double()).sum() * c["scale"]
        if s["d_scores"] is not None:
            loss = loss + (s_all * s["d_scores"].double()).sum()
        return torch.autograd.grad(loss, leaf)[0].masked_fill(shut, 0.0)


def _exact_adapt(s):
    """One adapter after another over the tokens that ask for it."""
    back = s["case"]["op"] == "adapt_backward"
    out = s["base"].double().clone()
    da, db = torch.zeros(s["a"].shape, dtype=torch.double, device="cuda"), torch.zeros(s["b"].shape, dtype=torch.double, device="cuda")
    for k in range(s["a"].shape[0]):
        rows = (s["ids"] == k).nonzero().flatten()
        x, f = s["x"][rows].double(), s["scale"][k].double()
        v = x @ s["a"][k].double().t()
        if not back:
            out[rows] += f * (v @ s["b"][k].double().t())
            continue
        dy = s["dy"][rows].double()
        u = f * (dy @ s["b"][k].double())
        out[rows] += u @ s["a"][k].double()
        da[k], db[k] = u.t() @ x, f * (dy.t() @ v)
    return {"dx": out, "da": da, "db": db} if back else out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(s)
    return _exact_route_backward(s) if case["op"] == "route_backward" else _exact_adapt(s)
