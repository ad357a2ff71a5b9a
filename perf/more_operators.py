"""The products of ragged rows around the attention of a language model, as measurable cases.

- `route`: Context.expert_route, the experts of each row from its logits, their weights, and the rows grouped by expert.
- `expert`: Context.expert_product, each group's rows times its own expert's matrix; `up` gathers the rows of the layer's
  input and closes with the gated activation, `down` takes those results and leaves them by row and choice.
- `join`: Context.expert_join, a row's results times their weights, summed onto the layer's input.
- `adapter`: Context.adapter_product, a projection that all rows share plus the low-rank adapter of each row's request.

Where `own` is false `run` computes the same in elementary torch operations in 32 bits.  Matrices are [outputs][inputs].
Inputs come from the seed alone; which experts and adapters the rows take from the case (`plan`).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one token of one conversation
        {"name": "route_token", "kind": "route", "rows": 1, "experts": 64, "top": 8, "type": "f32", "score": "softmax",
         "renorm": True, "plan": 1},
        # prompts of 16,384 tokens together, logits as the router's product leaves them in 16 bits (with ties)
        {"name": "route_prompt", "kind": "route", "rows": 16384, "experts": 128, "top": 8, "type": "bf16", "score": "softmax",
         "renorm": True, "plan": 2},
        # one token's gated products: the call that a decoding step makes in every layer, bound by the experts' bytes
        {"name": "expert_token", "kind": "expert", "way": "up", "rows": 1, "experts": 64, "top": 8, "in": 2048, "out": 1024,
         "gate": "silu", "type": "bf16", "plan": 3},
        # a decoding step of 64 conversations, the second product
        {"name": "expert_batch", "kind": "expert", "way": "down", "rows": 64, "experts": 64, "top": 8, "in": 1024, "out": 2048,
         "gate": "none", "type": "bf16", "plan": 4},
        # a piece of a prompt over few large experts, sizes that no tile divides
        {"name": "expert_chunk", "kind": "expert", "way": "up", "rows": 777, "experts": 8, "top": 2, "in": 1048, "out": 2500,
         "gate": "gelu", "type": "f16", "plan": 5},
        # prompts of 8,192 tokens: both products, bound by the matrix cores
        {"name": "expert_prompt_up", "kind": "expert", "way": "up", "rows": 8192, "experts": 64, "top": 8, "in": 2048,
         "out": 1024, "gate": "silu", "type": "bf16", "plan": 6},
        {"name": "expert_prompt_down", "kind": "expert", "way": "down", "rows": 8192, "experts": 64, "top": 8, "in": 1024,
         "out": 2048, "gate": "none", "type": "bf16", "plan": 6},
        # a decoding step's results, and those of the prompts
        {"name": "join_batch", "kind": "join", "rows": 64, "experts": 64, "top": 8, "out": 2048, "type": "bf16", "plan": 4},
        {"name": "join_prompt", "kind": "join", "rows": 8192, "experts": 64, "top": 8, "out": 2048, "type": "bf16", "plan": 6},
        # one token of one voice's conversation: latency, and the matrix's bytes
        {"name": "adapter_token", "kind": "adapter", "n": 1, "new_lo": 1, "new_hi": 1, "adapters": 8, "rank": 16, "in": 4096,
         "out": 4096, "type": "bf16", "result": "bf16", "bias": False, "plan": 7},
        # a decoding step of 96 conversations in 40 voices: queries, keys and values in one projection
        {"name": "adapter_batch", "kind": "adapter", "n": 96, "new_lo": 1, "new_hi": 1, "adapters": 40, "rank": 32, "in": 4096,
         "out": 6144, "type": "bf16", "result": "bf16", "bias": True, "plan": 8},
        # twelve prompts of 200 to 1,500 tokens, each in its voice
        {"name": "adapter_prompt", "kind": "adapter", "n": 12, "new_lo": 200, "new_hi": 1500, "adapters": 10, "rank": 64,
         "in": 4096, "out": 4096, "type": "bf16", "result": "bf16", "bias": False, "plan": 9},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "expert", "expert", "expert", "join", "adapter", "adapter", "adapter"])
    case = {"kind": kind, "plan": rng.randrange(10, 1 << 20), "type": rng.choice(["bf16", "bf16", "f16"])}
    if kind == "adapter":
        case["in"] = rng.choice([512, 768, 1024, 2048, 4096, 8 * rng.randrange(20, 500)])
        case["out"] = rng.choice([178, 768, 1024, 2048, 4096, 6144, rng.randrange(100, 5000)])
        case["adapters"], case["rank"] = _log_int(rng, 1, 64), rng.choice([8, 16, 16, 24, 32, 64])
        most = min(9000, int(2.4e11 / (2 * case["in"] * case["out"])))
        rows = _log_int(rng, 1, most)
        case["n"] = rng.choice([min(rows, 256), _log_int(rng, 1, min(rows, 32))])  # many short requests, or few
        case["new_hi"] = max(1, rows // case["n"])
        case["new_lo"] = max(1, int(case["new_hi"] * rng.uniform(0.2, 1.0)))
        case["result"], case["bias"] = rng.choice([case["type"], case["type"], "f32"]), rng.random() < 0.4
        return case
    case["experts"], case["top"] = rng.choice([(8, 2), (16, 2), (16, 4), (32, 4), (64, 6), (64, 8), (100, 5), (128, 8), (8, 1)])
    if kind == "route":
        case["rows"], case["type"] = _log_int(rng, 1, 16384), rng.choice(["bf16", "f16", "f32", "f32"])
        case["score"], case["renorm"] = rng.choice(["softmax", "softmax", "sigmoid"]), rng.random() < 0.7
        return case
    case["rows"] = _log_int(rng, 1, 8192)
    if kind == "join":
        case["out"] = rng.choice([512, 768, 1024, 2048, rng.randrange(200, 2048)])
        return case
    case["way"] = rng.choice(["up", "down"])
    case["gate"] = rng.choice(["silu", "silu", "gelu", "none"]) if case["way"] == "up" else "none"
    case["in"] = rng.choice([512, 768, 1024, 2048, 8 * rng.randrange(20, 300)])
    case["out"] = rng.choice([512, 768, 1024, 2048, rng.randrange(100, 2500)])
    while case["experts"] * case["in"] * case["out"] * (1 + (case["gate"] != "none")) > 270000000:
        case["out"] = max(64, case["out"] // 2)
    cost = 2.0 * case["top"] * case["in"] * case["out"] * (1 + (case["gate"] != "none"))
    case["rows"] = max(1, min(case["rows"], int(5.4e11 / cost)))
    return case


def _experts(case):
    """Each row's experts, the best first: some are wanted more than others, and every thirtieth row is padding without any."""
    rng = np.random.default_rng(case["plan"])
    want = rng.gumbel(size=(case["rows"], case["experts"])) + 0.5 * rng.standard_normal(case["experts"])
    chosen = np.argsort(-want, axis=1, kind="stable")[:, :case["top"]]
    chosen[np.arange(case["rows"]) % 30 == 29] = -1
    return chosen.astype(np.int64)


def _grouped(case):
    """The choices in the order of their experts, by row and choice within an expert, and where each expert's begin."""
    flat = _experts(case).reshape(-1)
    count = np.bincount(flat[flat >= 0], minlength=case["experts"])
    place = np.argsort(flat, kind="stable")[int((flat < 0).sum()):]
    return place, np.concatenate([[0], np.cumsum(count)])


def _adapters(case):
    """Each row's adapter: a request's rows share one, and some requests have none."""
    rng = np.random.default_rng(case["plan"])
    new = rng.integers(case["new_lo"], case["new_hi"] + 1, case["n"])
    ids = rng.integers(0, case["adapters"], case["n"])
    ids[rng.random(case["n"]) < 0.1 * (case["n"] > 1)] = -1
    return np.repeat(ids, new)


def work(case):
    e, top = (4 if case["type"] == "f32" else 2), case.get("top", 0)
    if case["kind"] == "route":
        return {"bytes": case["rows"] * (case["experts"] * e + 12 * top) + 4 * case["experts"],
                "flops": 6.0 * case["rows"] * case["experts"]}
    if case["kind"] == "adapter":
        ids = _adapters(case)
        rows, used, with_one = len(ids), len(set(ids[ids >= 0].tolist())), int((ids >= 0).sum())
        r, k, n = case["rank"], case["in"], case["out"]
        return {"bytes": 2 * (rows * k + n * k + used * r * (n + k)) + rows * n * (4 if case["result"] == "f32" else 2),
                "flops": 2.0 * rows * k * n + 2.0 * with_one * r * (k + n)}
    place, start = _grouped(case)
    entries, rows = len(place), len(set((place // top).tolist()))
    if case["kind"] == "join":
        return {"bytes": 2 * case["out"] * (entries + 2 * case["rows"]) + 8 * case["rows"] * top,
                "flops": 2.0 * entries * case["out"]}
    wide = case["out"] * (1 + (case["gate"] != "none"))
    read = rows if case["way"] == "up" else entries
    return {"bytes": 2 * (int((np.diff(start) > 0).sum()) * wide * case["in"] + read * case["in"] + entries * case["out"]) + 4 * entries,
            "flops": 2.0 * entries * wide * case["in"]}


# ------------------------------------------------------------------ inputs


def _dev(x, dtype=torch.int32):
    return torch.tensor(np.asarray(x), dtype=dtype, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]

    def randn(*shape, size=1.0, kept=dtype):
        return (torch.randn(shape, generator=gen, device="cuda") * size).to(kept)

    s = {"case": case}
    if case["kind"] == "route":
        rows, n = case["rows"], case["experts"]
        logits = torch.randn(rows, n, generator=gen, device="cuda") * 1.5 + 0.7 * torch.randn(n, generator=gen, device="cuda")
        logits[29::30] = -math.inf  # padding
        s["logits"], s["scale"] = logits.to(dtype), 1.0 if case["renorm"] else 2.5
        return s
    if case["kind"] == "adapter":
        ids, k, n, r = _adapters(case), case["in"], case["out"], case["rank"]
        s["x"], s["w"] = randn(len(ids), k), randn(n, k, size=k ** -0.5)
        s["a"], s["b"] = randn(case["adapters"], r, k, size=k ** -0.5), randn(case["adapters"], n, r, size=0.3 * r ** -0.5)
        s["scale"] = 0.5 + 1.5 * torch.rand(case["adapters"], generator=gen, device="cuda")
        s["bias"] = randn(n, size=0.2, kept=torch.float32) if case["bias"] else None
        s["adapter"] = _dev(ids)
        s["rows"] = {i: _dev(np.flatnonzero(ids == i), torch.int64) for i in sorted(set(ids[ids >= 0].tolist()))}
        return s
    top, rows = case["top"], case["rows"]
    place, start = _grouped(case)
    if case["kind"] == "join":
        s["y"], s["base"] = randn(rows * top, case["out"]), randn(rows, case["out"])
        s["expert"] = _dev(_experts(case))
        weight = torch.rand(rows, top, generator=gen, device="cuda") + 0.05
        s["weight"] = torch.where(s["expert"] >= 0, weight / weight.sum(1, keepdim=True), 0.0).contiguous()
        return s
    wide = case["out"] * (1 + (case["gate"] != "none"))
    s["place"] = torch.full((rows * top,), -1, dtype=torch.int32, device="cuda")
    s["place"][:len(place)] = _dev(place)
    s["start"], s["counts"] = _dev(start), np.diff(start).tolist()
    s["x"] = randn(rows if case["way"] == "up" else rows * top, case["in"])
    s["w"] = torch.empty(case["experts"], wide, case["in"], dtype=dtype, device="cuda")
    for e in range(case["experts"]):
        s["w"][e] = randn(wide, case["in"], size=case["in"] ** -0.5)
    return s


def run(s):
    if own:
        return _kernels(s)
    return {"route": _plain_route, "expert": _plain_expert, "join": _plain_join, "adapter": _plain_adapter}[s["case"]["kind"]](s)


# ------------------------------------------------------------------ the framework's operators

_ctx = None


def _api():
    root = os.path.join(os.getcwd(), "kokoro-rust_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from kokoro_hip import api
    return api


def _space(h, args, size):
    """A workspace of the size that the operator asks for."""
    h["space"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
    args.workspace, args.workspace_bytes = h["space"].data_ptr(), h["space"].numel()


def _handle(s):
    """What a program keeps for calls on these buffers: their descriptors, outputs and workspace."""
    global _ctx
    api, case = _api(), s["case"]
    if _ctx is None:
        _ctx = api.Context(0)
    codes = {"bf16": api.BF16, "f16": api.F16, "f32": api.F32}
    code, dtype = codes[case["type"]], TYPES[case["type"]]
    h = {"ctx": _ctx}
    if case["kind"] == "route":
        rows, n, top = case["rows"], case["experts"], case["top"]
        h["out"] = {"expert": torch.empty(rows, top, dtype=torch.int32, device="cuda"),
                    "weight": torch.empty(rows, top, device="cuda"),
                    "start": torch.empty(n + 1, dtype=torch.int32, device="cuda"),
                    "place": torch.empty(rows * top, dtype=torch.int32, device="cuda")}
        h["args"] = api.ExpertRoute(
            type=code, rows=rows, experts=n, top=top, logits=s["logits"].data_ptr(), logits_row=n,
            score=api.SCORE_SOFTMAX if case["score"] == "softmax" else api.SCORE_SIGMOID, renorm=int(case["renorm"]),
            scale=s["scale"], **{k: v.data_ptr() for k, v in h["out"].items()})
        _space(h, h["args"], _ctx.expert_route_workspace(h["args"]))
        h["call"] = _ctx.expert_route
    elif case["kind"] == "adapter":
        rows, k, n, r = s["x"].shape[0], case["in"], case["out"], case["rank"]
        h["out"] = torch.empty(rows, n, dtype=TYPES[case["result"]], device="cuda")
        h["args"] = api.AdapterProduct(
            type=code, out_type=codes[case["result"]], rows=rows, inputs=k, outputs=n, x=s["x"].data_ptr(), x_row=k,
            w=s["w"].data_ptr(), w_row=k, bias=None if s["bias"] is None else s["bias"].data_ptr(), y=h["out"].data_ptr(), y_row=n,
            adapters=case["adapters"], rank=r, a=s["a"].data_ptr(), b=s["b"].data_ptr(), scale=s["scale"].data_ptr(),
            adapter=s["adapter"].data_ptr())
        _space(h, h["args"], _ctx.adapter_product_workspace(h["args"]))
        h["call"] = _ctx.adapter_product
    elif case["kind"] == "join":
        rows, n, top = case["rows"], case["out"], case["top"]
        h["out"] = torch.empty(rows, n, dtype=dtype, device="cuda")
        h["args"] = api.ExpertJoin(
            type=code, rows=rows, top=top, values=n, y=s["y"].data_ptr(), y_row=n, expert=s["expert"].data_ptr(),
            weight=s["weight"].data_ptr(), base=s["base"].data_ptr(), base_row=n, out=h["out"].data_ptr(), out_row=n)
        h["call"] = _ctx.expert_join
    else:
        k, n, top = case["in"], case["out"], case["top"]
        entries, wide = case["rows"] * top, s["w"].shape[1]
        h["out"] = torch.zeros(entries, n, dtype=dtype, device="cuda")
        h["args"] = api.ExpertProduct(
            type=code, groups=case["experts"], entries=entries, inputs=k, outputs=n, start=s["start"].data_ptr(),
            x=s["x"].data_ptr(), x_rows=s["x"].shape[0], x_row=k, w=s["w"].data_ptr(), w_row=k, w_group=wide * k,
            gate={"none": api.GATE_NONE, "silu": api.GATE_SILU, "gelu": api.GATE_GELU}[case["gate"]], y=h["out"].data_ptr(),
            y_rows=entries, y_row=n)
        if case["way"] == "up":
            h["args"].x_place, h["args"].x_div = s["place"].data_ptr(), top
        else:
            h["args"].y_place = s["place"].data_ptr()
        h["call"] = _ctx.expert_product
    return h


def _kernels(s):
    h = s.get("handle")
    if h is None:
        h = s["handle"] = _handle(s)
    h["call"](h["args"], torch.cuda.current_stream().cuda_stream)
    return h["out"]


# ------------------------------------------------------------------ their plain form


def _plain_route(s):
    case, x = s["case"], s["logits"].float()
    rows, n, top = case["rows"], case["experts"], case["top"]
    order = torch.sort(x, dim=1, descending=True, stable=True)
    kept, expert = order.values[:, :top], order.indices[:, :top].int()
    if case["score"] == "softmax":
        most = x.amax(1, keepdim=True).clamp(min=-3e38)
        weight = torch.exp(kept - most) / torch.exp(x - most).sum(1, keepdim=True)
    else:
        weight = 1.0 / (1.0 + torch.exp(-kept))
    none = kept == -math.inf
    expert, weight = torch.where(none, -1, expert), torch.where(none, 0.0, weight)
    if case["renorm"]:
        total = weight.sum(1, keepdim=True)
        weight = weight / torch.where(total > 0, total, 1.0)
    flat = expert.view(-1)
    key = torch.where(flat < 0, n, flat)
    place = torch.sort(key, stable=True).indices.int()
    start = (key[:, None] < torch.arange(n + 1, device="cuda")).sum(0).int()
    place = torch.where(torch.arange(rows * top, device="cuda") < start[n], place, -1)
    return {"expert": expert, "weight": weight * s["scale"], "start": start, "place": place}


def _gated(g, kind):
    if kind == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))


def _plain_expert(s):
    case = s["case"]
    n, top, at = case["out"], case["top"], 0
    out = torch.zeros(case["rows"] * top, n, dtype=s["x"].dtype, device="cuda")
    for e, count in enumerate(s["counts"]):
        if not count:
            continue
        place = s["place"][at:at + count].long()
        x = s["x"][place // top] if case["way"] == "up" else s["x"][at:at + count]
        y = x.float() @ s["w"][e].float().T
        if case["gate"] != "none":
            y = _gated(y[:, :n], case["gate"]) * y[:, n:]
        if case["way"] == "up":
            out[at:at + count] = y.to(out.dtype)
        else:
            out[place] = y.to(out.dtype)
        at += count
    return out


def _plain_join(s):
    case = s["case"]
    y = s["y"].view(case["rows"], case["top"], -1).float()
    live = (s["expert"] >= 0)[:, :, None]
    return (s["base"].float() + torch.where(live, y * s["weight"][:, :, None], 0.0).sum(1)).to(s["y"].dtype)


def _plain_adapter(s):
    x = s["x"].float()
    y = x @ s["w"].float().T
    if s["bias"] is not None:
        y = y + s["bias"]
    for i, rows in s["rows"].items():
        h = x[rows] @ s["a"][i].float().T
        y[rows] += (h @ s["b"][i].float().T) * s["scale"][i]
    return y.to(TYPES[s["case"]["result"]])


# ------------------------------------------------------------------ the definition in 64 bits


def _exact_route(case, s):
    x = s["logits"].double().cpu().numpy()
    rows, n, top = case["rows"], case["experts"], case["top"]
    expert = np.argsort(-x, axis=1, kind="stable")[:, :top]
    kept = np.take_along_axis(x, expert, 1)
    live = kept > -math.inf
    with np.errstate(all="ignore"):
        score = np.exp(x) if case["score"] == "softmax" else 1.0 / (1.0 + np.exp(-x))
        weight = np.where(live, np.take_along_axis(score, expert, 1), 0.0)
        if case["score"] == "softmax":
            weight = np.where(live, weight / score.sum(1, keepdims=True), 0.0)
        if case["renorm"]:
            weight = np.where(live, weight / weight.sum(1, keepdims=True), 0.0)
    expert = np.where(live, expert, -1)
    lists = [np.flatnonzero(expert.reshape(-1) == e) for e in range(n)]
    place = np.full(rows * top, -1)
    start = np.concatenate([[0], np.cumsum([len(p) for p in lists])])
    place[:start[-1]] = np.concatenate(lists)
    return {"expert": _dev(expert), "weight": _dev(weight * s["scale"], torch.float64), "start": _dev(start), "place": _dev(place)}


def _exact_expert(case, s):
    top, n = case["top"], case["out"]
    chosen = torch.tensor(_experts(case).reshape(-1), device="cuda")
    to = torch.empty_like(chosen)  # each choice's place in the order of the experts
    order = torch.tensor(_grouped(case)[0], device="cuda")
    to[order] = torch.arange(len(order), device="cuda")
    out = torch.zeros(case["rows"] * top, n, dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        i = (chosen == e).nonzero()[:, 0]
        x = s["x"][i.div(top, rounding_mode="floor") if case["way"] == "up" else to[i]].double()
        w = s["w"][e].double()
        y = x @ w[:n].t()
        if case["gate"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["gate"] == "gelu":
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        if case["gate"] != "none":
            y = y * (x @ w[n:].t())
        out[to[i] if case["way"] == "up" else i] = y
    return out


def _exact_join(case, s):
    y = s["y"].double().view(case["rows"], case["top"], -1)
    out = s["base"].double()
    for j in range(case["top"]):
        out = out + y[:, j] * s["weight"][:, j, None].double()
    return out


def _exact_adapter(case, s):
    x = s["x"].double()
    out = x @ s["w"].double().t()
    for i in range(case["adapters"]):
        rows = (s["adapter"] == i).nonzero()[:, 0]
        out[rows] += s["scale"][i].double() * (x[rows] @ s["a"][i].double().t() @ s["b"][i].double().t())
    return out if s["bias"] is None else out + s["bias"].double()


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "expert": _exact_expert, "join": _exact_join, "adapter": _exact_adapter}[case["kind"]](case, s)
