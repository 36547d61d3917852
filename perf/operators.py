"""What the operators around one expert layer cost: routing, the block's norms
with its gate and residual, and per-request low-rank adapters.

``listed()`` and ``draw()`` give the cases, ``prepare()`` a case's inputs,
``run()`` one pass (in elementary torch operations, or with ``own`` through
the framework) and ``exact()`` the same outputs in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6

MOST_ROUTE = 8192 * 256        # logits of the largest routing case
MOST_NORM = 8192 * 2048        # values per tensor of the largest norm case
MOST_ADAPT = 4096 * (2048 + 2048)


def _route(name, n, n_expert, k, score="softmax", bias=False, n_group=1, topk_group=1, group_top=1,
           renorm=True, scale=1.0, dtype="f32", masked=0):
    return {"name": name, "op": "route", "n": n, "n_expert": n_expert, "k": k, "score": score, "bias": bias,
            "n_group": n_group, "topk_group": topk_group, "group_top": group_top, "renorm": renorm,
            "scale": scale, "dtype": dtype, "masked": masked}


def _norm(name, n, n_embd, source="rows", k=0, post=True, gate="none", act="none", scale=1.0, pre=True,
          offset=0.0, resid="f32", dtype="f32"):
    return {"name": name, "op": "norm", "n": n, "n_embd": n_embd, "source": source, "k": k, "post": post,
            "gate": gate, "act": act, "scale": scale, "pre": pre, "offset": offset, "resid": resid,
            "dtype": dtype}


def _adapt(name, n, n_in, n_out, n_adapters, rank, order="requests", dtype="f32", weights="bf16", out="f32",
           ragged=False):
    return {"name": name, "op": "adapters", "n": n, "n_in": n_in, "n_out": n_out, "n_adapters": n_adapters,
            "rank": rank, "order": order, "dtype": dtype, "weights": weights, "out": out, "ragged": ragged}


def listed():
    return [
        # one decoded token of the 128-expert stack
        _route("route one token", 1, 128, 8),
        # a batched decode or a prefill chunk with balance bias and expert groups
        _route("route 512 grouped", 512, 256, 8, score="sigmoid", bias=True, n_group=4, topk_group=2,
               group_top=2, scale=1.5),
        # an odd batch over an odd number of experts, some of them switched off
        _route("route 1031 odd", 1031, 157, 6, bias=True, renorm=False, dtype="bf16", masked=9),
        # a long prompt in one call
        _route("route 8192 grouped", 8192, 256, 8, score="sigmoid", bias=True, n_group=4, topk_group=2,
               group_top=2, scale=1.5, dtype="bf16"),
        # the end of the layer for one decoded token: combine, norms, residual
        _norm("norm one token, combined", 1, 2048, source="combine", k=8),
        # the same for a 512-token prefill chunk, with a gate per token
        _norm("norm 512 combined", 512, 2048, source="combine", k=9, gate="token", act="sigmoid", scale=0.5),
        # rows of an odd width that no vector load fits
        _norm("norm 777 odd", 777, 1537, gate="channel", scale=0.25, offset=1.0),
        # a long prompt, bf16 block output beside an fp32 residual
        _norm("norm 8192", 8192, 2048, gate="full", act="sigmoid", dtype="bf16"),
        # the router's adapters of one decoded token
        _adapt("adapters one token, router", 1, 2048, 128, 4, 8),
        # batched decode: every request with an adapter of its own choice
        _adapt("adapters 32 requests", 32, 2048, 2048, 16, 16, order="mixed"),
        # an odd mixed batch, adapters of several ranks, some rows without one
        _adapt("adapters 777 odd", 777, 2048, 1001, 6, 24, dtype="bf16", ragged=True),
        # prefill chunks of several requests
        _adapt("adapters 4096 prompts", 4096, 2048, 2048, 8, 64, dtype="bf16", out="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["route", "norm", "adapters"])
    if op == "route":
        n_group = rng.choice([1, 1, 2, 4, 8])
        n_expert = n_group * _log_int(rng, max(2, 16 // n_group), 512 // n_group)
        topk_group = rng.randint(1, n_group)
        k = min(rng.randint(1, 16), n_expert // n_group * topk_group)
        n = _log_int(rng, 1, min(8192, MOST_ROUTE // n_expert))
        c = _route("", n, n_expert, k, score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.6,
                   n_group=n_group, topk_group=topk_group, group_top=rng.choice([1, 2]),
                   renorm=rng.random() < 0.7, scale=rng.choice([1.0, 1.5]),
                   dtype=rng.choice(["f32", "f32", "bf16", "f16"]), masked=rng.choice([0, 0, 3]))
    elif op == "norm":
        n_embd = _log_int(rng, 64, 8192)
        if rng.random() < 0.7:
            n_embd = (n_embd + 63) // 64 * 64
        source = rng.choice(["rows", "rows", "combine"])
        k = rng.randint(1, 9) if source == "combine" else 0
        n = _log_int(rng, 1, max(1, MOST_NORM // n_embd // (1 + k)))
        resid, dtype = ("f32", "f32") if k else rng.choice(
            [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
        gate = rng.choice(["none", "token", "channel", "full"])
        c = _norm("", n, n_embd, source=source, k=k, post=rng.random() < 0.7, gate=gate,
                  act=rng.choice(["none", "sigmoid"]) if gate != "none" else "none",
                  scale=rng.choice([1.0, 0.5, 0.22]), pre=rng.random() < 0.8, offset=rng.choice([0.0, 1.0]),
                  resid=resid, dtype=dtype)
    else:
        n_in = _log_int(rng, 256, 4096)
        if rng.random() < 0.8:
            n_in = (n_in + 63) // 64 * 64
        n_out = _log_int(rng, 64, 4096)
        n = _log_int(rng, 1, min(4096, MOST_ADAPT // (n_in + n_out)))
        dtype, weights, out = rng.choice([("f32", "bf16", "f32"), ("f32", "f16", "f32"), ("bf16", "bf16", "bf16"),
                                          ("bf16", "bf16", "f32"), ("f16", "f16", "f16"), ("f16", "f16", "f32")])
        n_adapters = _log_int(rng, 1, 16)
        c = _adapt("", n, n_in, n_out, n_adapters, _log_int(rng, 4, min(64, 512 // n_adapters)),
                   order=rng.choice(["requests", "requests", "mixed"]), dtype=dtype, weights=weights, out=out,
                   ragged=rng.random() < 0.5)
    del c["name"]
    return c


# ---- inputs -----------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    s = {"case": case}
    n = case["n"]
    if case["op"] == "route":
        e = case["n_expert"]
        s["logits"] = (1.5 * randn(n, e)).to(DTYPES[case["dtype"]])
        if case["masked"]:    # experts that a request may not use
            off = torch.randint(0, e, (n, case["masked"]), generator=g, device="cuda")
            s["logits"].scatter_(1, off, -math.inf)
        s["bias"] = 0.05 * randn(e) if case["bias"] else None
        if own:
            from moe_prefetch_b200 import Routing
            s["op"] = Routing(e, case["k"], score=case["score"], bias=s["bias"], n_group=case["n_group"],
                              topk_group=case["topk_group"], group_top=case["group_top"],
                              renorm=case["renorm"], scale=case["scale"])
    elif case["op"] == "norm":
        h, t = case["n_embd"], DTYPES[case["dtype"]]
        s["r"] = (3.0 * randn(n, h)).to(DTYPES[case["resid"]])
        if case["source"] == "combine":
            k = case["k"]
            s["y_rows"] = randn(n * k, h)
            s["pos"] = torch.randperm(n * k, generator=g, device="cuda").to(torch.int32).view(n, k)
            s["w"] = torch.softmax(randn(n, k), dim=-1)
        else:
            s["y"] = randn(n, h, dtype=t)
        s["post"] = (1.0 - case["offset"] + 0.2 * randn(h)) if case["post"] else None
        s["pre"] = (1.0 - case["offset"] + 0.2 * randn(h)) if case["pre"] else None
        shape = {"none": None, "token": (n, 1), "channel": (h,), "full": (n, h)}[case["gate"]]
        s["gate"] = None if shape is None else randn(*shape, dtype=torch.float32 if case["gate"] == "channel" else t)
        if own:
            from moe_prefetch_b200 import BlockNorm
            s["op"] = BlockNorm(h, post=s["post"], pre=s["pre"], gate_act=case["act"], scale=case["scale"],
                                eps=EPS, weight_offset=case["offset"])
    else:
        n_in, n_out, na, r = case["n_in"], case["n_out"], case["n_adapters"], case["rank"]
        wt = DTYPES[case["weights"]]
        s["x"] = randn(n, n_in, dtype=DTYPES[case["dtype"]])
        s["y"] = randn(n, n_out, dtype=DTYPES[case["out"]])
        s["a"] = (randn(na, r, n_in) / math.sqrt(n_in)).to(wt)
        s["b"] = (randn(na, n_out, r) / math.sqrt(r)).to(wt)
        s["scale"] = 0.5 + torch.rand(na, generator=g, device="cuda")
        s["rank"] = (torch.randint(1, r + 1, (na,), generator=g, device="cuda").to(torch.int32)
                     if case["ragged"] else None)
        lo = -1 if case["ragged"] else 0     # -1: a row without an adapter
        if case["order"] == "mixed":
            ids = torch.randint(lo, na, (n,), generator=g, device="cuda")
        else:                                # the tokens of a request follow one another
            m = min(n, 2 * na)
            ends = torch.sort(torch.rand(m, generator=g, device="cuda"))[0]
            at = torch.searchsorted(ends, (torch.arange(n, device="cuda") + 0.5) / n)
            ids = torch.randint(lo, na, (m + 1,), generator=g, device="cuda")[at]
        s["ids"] = ids.to(torch.int32)
        if own:
            from moe_prefetch_b200 import AdapterSet
            s["op"] = AdapterSet(s["a"], s["b"], scale=s["scale"], rank=s["rank"])
    return s


# ---- the operators ------------------------------------------------------------

def _best_k(choice, k):
    """Indices of the k largest of each row, in order, ties to the lowest index."""
    return torch.sort(choice, dim=-1, descending=True, stable=True)[1][..., :k]


def _plain_route(case, logits, bias):
    l64 = logits.double()      # 64 bits: which of two close scores is larger
    if case["score"] == "softmax":
        m = l64.amax(-1, keepdim=True)
        e = torch.where(m == -math.inf, 0.0, torch.exp(l64 - m))
        total = e.sum(-1, keepdim=True)
        score = torch.where(total == 0, 0.0, e / total)
    else:
        score = 1.0 / (1.0 + torch.exp(-l64))
    by_logit = bias is None and (case["n_group"] == 1 or case["group_top"] == 1)
    choice = l64 if by_logit else score if bias is None else score + bias.double()
    choice = torch.where(torch.isnan(choice), -math.inf, choice)
    if case["n_group"] > 1:
        n, per = logits.shape[0], case["n_expert"] // case["n_group"]
        in_groups = choice.view(n, case["n_group"], per)
        best = torch.sort(in_groups, dim=-1, descending=True)[0][..., :min(case["group_top"], per)].sum(-1)
        best = torch.where(torch.isnan(best), -math.inf, best)
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, _best_k(best, case["topk_group"]), True)
        # an expert of a group left out comes after every other
        choice = torch.where(kept[..., None], in_groups.clamp(min=-torch.finfo(torch.float64).max),
                             -math.inf).view(n, -1)
    ids = _best_k(choice, case["k"])
    w = score.float().gather(1, ids)
    if case["renorm"]:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total == 0, 0.0, w / total)
    return ids.to(torch.int32), w * case["scale"]


def _plain_norm(case, s):
    def rms(v, w):
        return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * (w + case["offset"])

    if case["source"] == "combine":
        y = (s["w"][..., None] * s["y_rows"][s["pos"].long()]).sum(1)
    else:
        y = s["y"].float()
    if s["post"] is not None:
        y = rms(y, s["post"])
    if s["gate"] is not None:
        gate = s["gate"].float()
        y = y * (1.0 / (1.0 + torch.exp(-gate)) if case["act"] == "sigmoid" else gate)
    r = s["r"].float() + case["scale"] * y
    x = None if s["pre"] is None else rms(r, s["pre"]).to(DTYPES[case["dtype"]])
    return [r.to(DTYPES[case["resid"]])] + ([] if x is None else [x])


def _plain_adapters(s):
    na, r, n_in = s["a"].shape
    a, b = s["a"].float(), s["b"].float()
    # every adapter's low-rank products of every token, those of its own kept
    low = (s["x"].float() @ a.view(na * r, n_in).t()).view(-1, na, r)
    keep = s["ids"][:, None] == torch.arange(na, device="cuda")
    keep = keep[..., None].expand(-1, -1, r)
    if s["rank"] is not None:
        keep = keep & (torch.arange(r, device="cuda") < s["rank"][:, None])
    low = torch.where(keep, low * s["scale"][:, None], 0.0)
    delta = low.reshape(-1, na * r) @ b.permute(0, 2, 1).reshape(na * r, -1)
    return (s["y"].float() + delta).to(s["y"].dtype)


def run(state):
    case = state["case"]
    if case["op"] == "route":
        if own:
            return list(state["op"](state["logits"]))
        return list(_plain_route(case, state["logits"], state["bias"]))
    if case["op"] == "norm":
        if own:
            if case["source"] == "combine":
                out = state["op"].combine(state["r"], state["y_rows"], state["pos"], state["w"], gate=state["gate"])
            else:
                out = state["op"](state["r"], state["y"], gate=state["gate"])
            return [t for t in out if t is not None]
        return _plain_norm(case, state)
    if own:
        return [state["op"](state["x"], state["ids"], state["y"])]
    return [_plain_adapters(state)]


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    n = case["n"]
    if case["op"] == "route":
        e = case["n_expert"]
        return {"bytes": n * e * size[case["dtype"]] + (4 * e if case["bias"] else 0) + 8 * n * case["k"],
                "flops": 4 * n * e}
    if case["op"] == "norm":
        h, t = case["n_embd"], size[case["dtype"]]
        gate = {"none": 0, "token": n * t, "channel": 4 * h, "full": n * h * t}[case["gate"]]
        y = n * case["k"] * (4 * h + 8) if case["source"] == "combine" else n * h * t
        return {"bytes": y + gate + 2 * n * h * size[case["resid"]] + (n * h * t if case["pre"] else 0) +
                4 * h * (int(case["post"]) + int(case["pre"])),
                "flops": n * h * (8 + 2 * case["k"])}
    n_in, n_out, r = case["n_in"], case["n_out"], case["rank"]
    used = min(case["n_adapters"], n)
    return {"bytes": n * n_in * size[case["dtype"]] + 2 * n * n_out * size[case["out"]] + 4 * n +
            used * r * (n_in + n_out) * size[case["weights"]],
            "flops": 2 * n * r * (n_in + n_out)}


# ---- the same from the definitions, in 64 bits ---------------------------------

def _exact_route(case, s):
    logits = s["logits"].double().cpu()
    bias = None if s["bias"] is None else s["bias"].double().cpu()
    n, e, k = case["n"], case["n_expert"], case["k"]
    score = torch.sigmoid(logits) if case["score"] == "sigmoid" else torch.nan_to_num(torch.softmax(logits, -1), nan=0.0)
    choice = score if bias is None else score + bias
    by_logit = bias is None and (case["n_group"] == 1 or case["group_top"] == 1)
    rank_by = logits if by_logit else choice
    allowed = torch.ones(n, e, dtype=torch.bool)
    if case["n_group"] > 1:
        per = e // case["n_group"]
        parts = [rank_by[:, i * per:(i + 1) * per].topk(min(case["group_top"], per))[0].sum(-1)
                 for i in range(case["n_group"])]
        strength = torch.stack(parts, 1).tolist()
        for t in range(n):
            order = sorted(range(case["n_group"]), key=lambda i: (-strength[t][i], i))
            for i in order[case["topk_group"]:]:
                allowed[t, i * per:(i + 1) * per] = False
    values, may = rank_by.tolist(), allowed.tolist()
    ids = torch.tensor([sorted((i for i in range(e) if may[t][i]), key=lambda i: (-values[t][i], i))[:k]
                        for t in range(n)])
    w = torch.gather(score, 1, ids)
    if case["renorm"]:
        w = torch.nan_to_num(w / w.sum(-1, keepdim=True), nan=0.0)
    return [ids.to(torch.int32), w * case["scale"]]


def _exact_norm(case, s):
    h = case["n_embd"]
    if case["source"] == "combine":
        y = torch.zeros(case["n"], h, dtype=torch.float64, device="cuda")
        for j in range(case["k"]):
            y += s["w"][:, j, None].double() * s["y_rows"].index_select(0, s["pos"][:, j].long()).double()
    else:
        y = s["y"].double()
    if s["post"] is not None:
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / h + EPS) * (s["post"].double() + case["offset"])
    if s["gate"] is not None:
        gate = s["gate"].double()
        y = y * (torch.sigmoid(gate) if case["act"] == "sigmoid" else gate)
    r = s["r"].double() + case["scale"] * y
    out = [r]
    if s["pre"] is not None:
        out.append(r / torch.sqrt(r.pow(2).sum(-1, keepdim=True) / h + EPS) * (s["pre"].double() + case["offset"]))
    return out


def _exact_adapters(s):
    y = s["y"].double()
    ids = s["ids"].tolist()
    for i in range(s["a"].shape[0]):
        rows = torch.tensor([t for t, a in enumerate(ids) if a == i], dtype=torch.long, device="cuda")
        if len(rows):
            r = s["a"].shape[1] if s["rank"] is None else int(s["rank"][i])
            low = s["x"][rows].double() @ s["a"][i, :r].double().t()
            y[rows] += float(s["scale"][i]) * (low @ s["b"][i, :, :r].double().t())
    return [y]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(case, s)
    if case["op"] == "norm":
        return _exact_norm(case, s)
    return _exact_adapters(s)
