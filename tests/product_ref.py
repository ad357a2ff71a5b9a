"""The products of ragged rows in 64 bits, with a bound of what the kernels' arithmetic may be off by, and their calls from tensors.

Products of two 16-bit values are exact in f32, and a matrix instruction adds 16 (32) of them to a running f32 sum, so with K inputs a
value passes at most K / 16 + 32 additions (32: those within an instruction, and the joining of parts), each off by 2^-23 of a
partial sum, which the sum of sizes bounds."""
import torch

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def code(kind):
    from kokoro_hip import api
    return {"bf16": api.BF16, "f16": api.F16, "f32": api.F32}[kind]


def kind_of(t):
    return {v: k for k, v in TYPES.items()}[t.dtype]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):  # half the type's smallest number
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def product(x, w):
    """x w^T of rows x, and its bound."""
    x, w = x.double(), w.double()
    return x @ w.t(), (x.shape[1] / 16 + 32) * 2.0 ** -23 * (x.abs() @ w.abs().t())


def gate(kind, g, dg, z, dz):
    """f(g) z and its bound: |f'| < 1.2 for both gates; exp2 is off by the size of its argument times 2^-23, and a few steps more."""
    if kind == "silu":
        f = g * torch.sigmoid(g)
        u = g.abs()
    else:
        inner = (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3)
        f = 0.5 * g * (1 + torch.tanh(inner))
        u = 2 * inner.abs()
    # sigmoid'(u) u <= 1/4 u exp(-u) ...: the argument's error counts through f = g sigmoid(u), at most |g| u exp(-u) 2^-22
    df = 1.2 * dg + 2.0 ** -20 * f.abs() + 2.0 ** -22 * g.abs() * torch.clamp(u * torch.exp(-u), min=2.0 ** -126)
    return f * z, df * (z.abs() + dz) + f.abs() * dz + 2.0 ** -22 * (f * z).abs()


def close(got, want, bound):
    """got, rounded once from a value within the bound of `want`."""
    tol = bound + half_step(got.dtype) * (want.abs() + bound) + least(got.dtype)
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), f"off by {(off / tol).max().item():.3f} of the tolerance"


def ptr(t):
    return None if t is None else t.data_ptr()


def space(n):
    """A workspace of n bytes, filled with NaN: it need not be cleared."""
    return torch.full((max(n, 16) // 4 + 4,), float("nan"), device="cuda")


def route(ctx, logits, top, score="softmax", renorm=True, scale=1.0, stream=0):
    from kokoro_hip import api
    rows, n = logits.shape
    out = {"expert": torch.full((rows, top), -7, dtype=torch.int32, device="cuda"), "weight": torch.full((rows, top), -7.0, device="cuda"),
           "start": torch.full((n + 1,), -7, dtype=torch.int32, device="cuda"),
           "place": torch.full((rows * top,), -7, dtype=torch.int32, device="cuda")}
    a = api.ExpertRoute(type=code(kind_of(logits)), rows=rows, experts=n, top=top, logits=ptr(logits), logits_row=logits.stride(0),
                        score=api.SCORE_SOFTMAX if score == "softmax" else api.SCORE_SIGMOID, renorm=int(renorm), scale=scale,
                        **{k: ptr(v) for k, v in out.items()})
    ws = space(ctx.expert_route_workspace(a))
    a.workspace, a.workspace_bytes = ptr(ws), ws.numel() * 4
    ctx.expert_route(a, stream)
    out["kept"] = (a, ws, logits)
    return out


def route_ref(logits, top, score, renorm, scale):
    """expert, weight, start and place, from the definition."""
    x = logits.double().cpu()
    x = torch.where(x.isnan(), -torch.inf, x).clamp(max=torch.finfo(torch.float32).max)
    order = torch.sort(x, dim=1, descending=True, stable=True)
    value, expert = order.values[:, :top], order.indices[:, :top]
    live = value > -torch.inf
    if score == "softmax":
        top1 = torch.where(live[:, :1], value[:, :1], 0.0)
        e, den = torch.exp(value - top1), torch.exp(x - top1).sum(1, keepdim=True)
    else:
        e, den = torch.sigmoid(value), torch.ones(len(x), 1, dtype=torch.float64)
    e = torch.where(live, e, 0.0)
    if renorm:
        den = e.sum(1, keepdim=True)
    weight = torch.where(den > 0, e / torch.where(den > 0, den, 1.0), 0.0) * scale
    expert = torch.where(live, expert, -1)
    flat = expert.reshape(-1)
    n = logits.shape[1]
    lists = [(flat == i).nonzero()[:, 0] for i in range(n)]
    place = torch.full_like(flat, -1)
    got = torch.cat(lists)
    place[:len(got)] = got
    start = torch.tensor([0] + [len(p) for p in lists]).cumsum(0)
    return {"expert": expert, "weight": weight, "start": start, "place": place}


def expert_args(x, w, start, y, entries=None, gate_kind="none", bias=None, x_place=None, x_div=1, y_place=None, fault=None):
    from kokoro_hip import api
    gates = {"none": api.GATE_NONE, "silu": api.GATE_SILU, "gelu": api.GATE_GELU}
    groups, wide, k = w.shape
    if entries is None:
        entries = len(x_place if x_place is not None else y_place if y_place is not None else x)
    return api.ExpertProduct(
        type=code(kind_of(x)), groups=groups, entries=entries, inputs=k, outputs=wide // (1 if gate_kind == "none" else 2),
        start=ptr(start), x=ptr(x), x_rows=x.shape[0], x_row=x.stride(0), x_place=ptr(x_place), x_div=x_div, w=ptr(w), w_row=w.stride(1),
        w_group=w.stride(0), bias=ptr(bias), gate=gates[gate_kind], y=ptr(y), y_rows=y.shape[0], y_row=y.stride(0), y_place=ptr(y_place),
        fault=ptr(fault))


def expert_ref(x, w, start, y, gate_kind="none", bias=None, x_place=None, x_div=1, y_place=None):
    """y as it is afterwards, in 64 bits, the bound, and which rows were written."""
    want, bound = y.double().clone(), torch.zeros_like(y, dtype=torch.float64)
    written = torch.zeros(len(y), dtype=torch.bool, device=y.device)
    start = start.tolist()
    for g in range(len(w)):
        i = torch.arange(start[g], start[g + 1], device=y.device)
        if len(i) == 0:
            continue
        rows = x[i if x_place is None else x_place[i].long() // x_div]
        z, dz = product(rows, w[g])
        if bias is not None:
            z = z + bias[g].double()
            dz = dz + 2.0 ** -23 * z.abs()
        if gate_kind != "none":
            n = z.shape[1] // 2
            z, dz = gate(gate_kind, z[:, :n], dz[:, :n], z[:, n:], dz[:, n:])
        to = i if y_place is None else y_place[i].long()
        want[to], bound[to], written[to] = z, dz, True
    return want, bound, written


def join_args(y, expert, weight, out, base=None):
    from kokoro_hip import api
    rows, top = expert.shape
    return api.ExpertJoin(type=code(kind_of(y)), rows=rows, top=top, values=out.shape[1], y=ptr(y), y_row=y.stride(0),
                          expert=ptr(expert), weight=ptr(weight), base=ptr(base), base_row=0 if base is None else base.stride(0),
                          out=ptr(out), out_row=out.stride(0))


def join_ref(y, expert, weight, base=None):
    """The sums, and their bound: top + 1 additions."""
    rows, top = expert.shape
    live = (expert >= 0)[:, :, None]
    part = torch.where(live, y[:rows * top].double().view(rows, top, -1) * weight.double()[:, :, None], 0.0)
    parts = part if base is None else torch.cat([base.double()[:, None], part], 1)
    return parts.sum(1), (top + 2) * 2.0 ** -24 * parts.abs().sum(1)


def adapter_args(x, w, y, bias=None, a=None, b=None, scale=None, adapter=None, fault=None):
    from kokoro_hip import api
    r = api.AdapterProduct(type=code(kind_of(x)), out_type=code(kind_of(y)), rows=x.shape[0], inputs=w.shape[1], outputs=w.shape[0],
                           x=ptr(x), x_row=x.stride(0), w=ptr(w), w_row=w.stride(0), bias=ptr(bias), y=ptr(y), y_row=y.stride(0),
                           fault=ptr(fault))
    if a is not None:
        r.adapters, r.rank, r.a, r.b = a.shape[0], a.shape[1], ptr(a), ptr(b)
        r.scale, r.adapter = ptr(scale), ptr(adapter)
    return r


def adapter_run(ctx, args, stream=0):
    ws = space(ctx.adapter_product_workspace(args))
    args.workspace, args.workspace_bytes = ptr(ws), ws.numel() * 4
    ctx.adapter_product(args, stream)
    return ws


def adapter_ref(x, w, bias=None, a=None, b=None, scale=None, adapter=None):
    """The results and their bound: a_i x is kept to 2^-17 of a value (f16: of the row's largest) or better."""
    y, dy = product(x, w)
    for i in range(0 if a is None else len(a)):
        rows = ((adapter == i).nonzero()[:, 0]) if adapter is not None else []
        if len(rows) == 0:
            continue
        h, dh = product(x[rows], a[i])
        dh = dh + 2.0 ** -17 * h.abs().amax(1, keepdim=True)
        s = scale[i].double()
        more = (h @ b[i].double().t()) * s
        size = (h.abs() @ b[i].double().abs().t()) * s.abs()
        # the adapters' share enters the same running sum: its additions, and those behind it, count its size too
        dmore = (dh @ b[i].double().abs().t()) * s.abs() + ((x.shape[1] + 2 * a.shape[1]) / 16 + 64) * 2.0 ** -23 * size
        y[rows] += more
        dy[rows] += dmore
    if bias is not None:
        y = y + bias.double()
        dy = dy + 2.0 ** -23 * (y.abs() + bias.double().abs())
    return y, dy
