"""The operators over a cache held in 8 bits, as measurable cases.

- `rope`: Context.qk_norm_rope, the RMS norms of queries and keys for each head and the position
  rotation in one pass, from the packed q | k | v rows of a projection.
- `write`: Context.kv_write of new tokens into a paged 8-bit cache, then Context.kv_read of the pages
  it touched (what is stored, as the values it stands for).
- `read`: Context.kv_read of whole sequences, as a program does that moves or re-encodes them.
- `attend`: Context.kv_attention of new rows (single tokens, drafts, prompts) over the cache.

Where `own` is false `run` computes the same in elementary torch operations in 32 bits.  A cache is
pages of 64 tokens: K [pages][heads][64][dim] and V [pages][heads][dim][64] bytes (int8, or e4m3), and
for each (page, head) one f32 scale of K and one of V.  Inputs come from the seed alone.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 64
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TOP = {"int8": 127.0, "e4m3": 448.0}  # largest stored value
LEAST = 2.0 ** -90                    # smallest scale of a page that holds anything but zeros


def listed():
    return [
        # one token of one conversation: the call that a decoding step makes in every layer
        {"name": "rope_token", "kind": "rope", "rows": 1, "hq": 32, "hk": 8, "dim": 128, "rot": 128, "inter": False,
         "type": "bf16", "far": 8192, "theta": 10000.0},
        # a decoding step of 96 conversations, half of each head rotated in interleaved pairs
        {"name": "rope_batch", "kind": "rope", "rows": 96, "hq": 16, "hk": 4, "dim": 96, "rot": 48, "inter": True,
         "type": "f16", "far": 1000000, "theta": 1000000.0},
        # the text encoder's heads over a batch of utterances, in its f32
        {"name": "rope_text", "kind": "rope", "rows": 4801, "hq": 12, "hk": 12, "dim": 64, "rot": 64, "inter": False,
         "type": "f32", "far": 512, "theta": 10000.0},
        # prompts of 16,384 tokens together
        {"name": "rope_prompt", "kind": "rope", "rows": 16384, "hq": 32, "hk": 8, "dim": 128, "rot": 128, "inter": False,
         "type": "bf16", "far": 16384, "theta": 500000.0},
        # the tokens of a decoding step of 64 conversations, each into a page that is partly full
        {"name": "write_step", "kind": "write", "n": 64, "new_lo": 1, "new_hi": 1, "ctx_lo": 100, "ctx_hi": 4000,
         "lengths": 1, "hq": 32, "hk": 8, "dim": 128, "cache": "e4m3", "type": "bf16"},
        # eight prompts as they are read in
        {"name": "write_prompt", "kind": "write", "n": 8, "new_lo": 300, "new_hi": 4096, "ctx_lo": 0, "ctx_hi": 0,
         "lengths": 2, "hq": 32, "hk": 8, "dim": 128, "cache": "int8", "type": "bf16"},
        # one long conversation taken out of the cache
        {"name": "read_long", "kind": "read", "n": 1, "ctx_lo": 32001, "ctx_hi": 32001, "lengths": 3, "hq": 32, "hk": 8,
         "dim": 128, "cache": "int8", "type": "bf16"},
        # one token of one short conversation: latency
        {"name": "attend_token", "kind": "attend", "n": 1, "new_lo": 1, "new_hi": 1, "ctx_lo": 500, "ctx_hi": 500,
         "lengths": 4, "hq": 32, "hk": 8, "dim": 128, "cache": "int8", "type": "bf16", "causal": True, "window": 0},
        # a decoding step of 64 conversations of 200 to 8191 tokens
        {"name": "attend_serving", "kind": "attend", "n": 64, "new_lo": 1, "new_hi": 1, "ctx_lo": 200, "ctx_hi": 8191,
         "lengths": 5, "hq": 32, "hk": 8, "dim": 128, "cache": "int8", "type": "bf16", "causal": True, "window": 0},
        # five drafted tokens checked at the end of a very long text
        {"name": "attend_drafts", "kind": "attend", "n": 1, "new_lo": 5, "new_hi": 5, "ctx_lo": 131000, "ctx_hi": 131000,
         "lengths": 6, "hq": 32, "hk": 8, "dim": 128, "cache": "e4m3", "type": "f16", "causal": True, "window": 0},
        # pieces of prompts behind what is cached already, with a sliding window
        {"name": "attend_chunk", "kind": "attend", "n": 3, "new_lo": 200, "new_hi": 700, "ctx_lo": 1000, "ctx_hi": 9000,
         "lengths": 7, "hq": 16, "hk": 4, "dim": 96, "cache": "e4m3", "type": "f16", "causal": True, "window": 1000},
        # four whole prompts of up to 4096 tokens
        {"name": "attend_prompt", "kind": "attend", "n": 4, "new_lo": 1000, "new_hi": 4096, "ctx_lo": 0, "ctx_hi": 0,
         "lengths": 8, "hq": 32, "hk": 8, "dim": 128, "cache": "int8", "type": "bf16", "causal": True, "window": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(32, 8, 128), (32, 8, 128), (16, 2, 128), (12, 12, 64), (16, 2, 64), (16, 4, 96), (8, 1, 256), (16, 4, 256),
         (8, 2, 192), (9, 3, 64), (28, 4, 128)]


def draw(rng):
    kind = rng.choice(["rope", "rope", "write", "write", "read", "attend", "attend", "attend", "attend"])
    hq, hk, dim = rng.choice(HEADS)
    if kind == "rope":
        if rng.random() < 0.3:
            hq, hk, dim = rng.choice([(16, 4, 80), (5, 1, 72), (8, 8, 40), (3, 0, 128)])
        rot, kept = rng.choice([dim, dim, dim, dim // 2]), rng.choice(["bf16", "bf16", "f16", "f32"])
        most = (40000000 if kept == "f32" else 80000000) // ((hq + hk) * dim)
        return {"kind": kind, "rows": _log_int(rng, 1, min(16384, most)), "hq": hq, "hk": hk, "dim": dim, "rot": rot,
                "inter": rng.random() < 0.3, "type": kept, "far": _log_int(rng, 600, 4000000),
                "theta": rng.choice([10000.0, 500000.0, 1000000.0])}
    case = {"kind": kind, "lengths": rng.randrange(1, 1 << 20), "hq": hq, "hk": hk, "dim": dim,
            "cache": rng.choice(["int8", "e4m3"]), "type": rng.choice(["bf16", "bf16", "f16"])}
    if kind == "attend":
        case["causal"], case["window"] = rng.random() < 0.85, 0
        if case["causal"] and rng.random() < 0.25:
            case["window"] = _log_int(rng, 1, 4000)
        if rng.random() < 0.6:  # decoding
            n, new = _log_int(rng, 1, 96), rng.choice([1, 1, 1, 1, 2, 3, 5, 8])
            top = min(131000, 200000000 // (n * hk * dim))
            ctx = _log_int(rng, 1, max(1, top))
        else:
            n, new = _log_int(rng, 1, 8), _log_int(rng, 9, 2500)
            top = int(4.5e10 / (hq * dim * n * new)) - new
            while top < 0:
                new, top = new // 2, int(4.5e10 / (hq * dim * n * (new // 2))) - new // 2
            ctx = rng.choice([0, _log_int(rng, 1, max(1, min(30000, top)))])
    elif kind == "write":
        n = _log_int(rng, 1, 64)
        new, ctx = _log_int(rng, 1, max(1, min(8000, 16000000 // (n * hk * dim)))), _log_int(rng, 1, 4000)
    else:
        n, new = _log_int(rng, 1, 16), 0
        ctx = _log_int(rng, 1, max(1, min(32000, 32000000 // (n * hk * dim))))
    case["n"], case["ctx_hi"], case["ctx_lo"] = n, ctx, max(int(kind == "read"), int(ctx * rng.uniform(0.1, 1.0)))
    if kind != "read":
        case["new_hi"], case["new_lo"] = new, max(1, int(new * rng.uniform(0.2, 1.0)))
    return case


def _lengths(case):
    """Each sequence's new rows and its tokens in the cache with them."""
    rng = np.random.default_rng(case["lengths"])
    ctx = rng.integers(case["ctx_lo"], case["ctx_hi"] + 1, case["n"])
    new = ctx if case["kind"] == "read" else rng.integers(case["new_lo"], case["new_hi"] + 1, case["n"])
    return new.astype(np.int64), (ctx if case["kind"] == "read" else ctx + new).astype(np.int64)


def _pairs(case, new, lens):
    """How many (row, token) pairs of one head attend."""
    total = 0
    for m, n in zip(new.tolist(), lens.tolist()):
        if not case["causal"]:
            total += m * n
            continue
        seen = np.arange(n - m + 1, n + 1)
        total += int((np.minimum(seen, case["window"]) if case["window"] else seen).sum())
    return total


def work(case):
    e = 4 if case["type"] == "f32" else 2
    if case["kind"] == "rope":
        vals = case["rows"] * (case["hq"] + case["hk"]) * case["dim"]
        return {"bytes": 2 * vals * e + 4 * case["rows"] + 8 * case["dim"], "flops": 8 * vals}
    new, lens = _lengths(case)
    hk, dim = case["hk"], case["dim"]
    if case["kind"] == "attend":
        first = np.zeros_like(lens)
        if case["window"]:
            first = np.maximum(0, lens - new + 1 - case["window"])
        toks, pages = int((lens - first).sum()), int((-(-lens // PAGE) - first // PAGE).sum())
        return {"bytes": 2 * toks * hk * dim + 12 * pages * hk + 2 * int(new.sum()) * case["hq"] * dim * e,
                "flops": 4.0 * dim * case["hq"] * _pairs(case, new, lens)}
    back = int((lens - (lens - new) // PAGE * PAGE).sum())
    vals = 2 * hk * dim * (int(new.sum()) * (e + 1) * (case["kind"] == "write") + back * (1 + 2))
    return {"bytes": vals, "flops": 3.0 * vals}


# ------------------------------------------------------------------ inputs


def _ragged(new, lens, table):
    """A batch over the cache: row_start, len and table on the device, and the host's bounds."""
    start = np.concatenate([[0], np.cumsum(new)])
    return {"n": len(lens), "rows": int(start[-1]), "max_new": int(new.max()), "max_len": int(lens.max()),
            "row_start": torch.tensor(start, dtype=torch.int32, device="cuda"),
            "len": torch.tensor(lens, dtype=torch.int32, device="cuda"), "table": table}


def _filled(case, lens, gen):
    """A cache whose pages all hold tokens, in an order of their own, and its page table."""
    need = -(-lens // PAGE)
    pages, hk, dim = int(need.sum()) + 3, case["hk"], case["dim"]
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), int(need.max()) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, p in enumerate(need.tolist()):
        table[b, :p] = order[at:at + p]
        at += p
    made = {}
    for part in ("k", "v"):
        kind = torch.int8 if case["cache"] == "int8" else torch.uint8
        shape = (pages, hk, PAGE, dim) if part == "k" else (pages, hk, dim, PAGE)
        data, scale = torch.empty(shape, dtype=kind, device="cuda"), torch.empty(pages, hk, device="cuda")
        step = max(1, (1 << 27) // (hk * PAGE * dim))
        for p in range(0, pages, step):
            x = torch.randn((min(step, pages - p),) + shape[1:], generator=gen, device="cuda")
            s = torch.exp(0.3 * torch.randn(x.shape[:2], generator=gen, device="cuda"))
            top = x.abs().amax((2, 3), keepdim=True)
            y = x * (TOP[case["cache"]] / top)
            data[p:p + step] = y.round().to(torch.int8) if kind == torch.int8 else y.to(torch.float8_e4m3fn).view(torch.uint8)
            scale[p:p + step] = top[:, :, 0, 0] * s / TOP[case["cache"]]
        made[part], made[part + "_scale"] = data, scale
    return {"type": case["cache"], "heads": hk, "dim": dim, "pages": pages, **made}, table


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]
    if case["kind"] == "rope":
        rows, hq, hk, dim = (case[k] for k in ("rows", "hq", "hk", "dim"))
        qkv = (torch.randn(rows, (hq + 2 * hk) * dim, generator=gen, device="cuda") * 2).to(dtype)
        return {"case": case, "qkv": qkv, "eps": 1e-6,
                "pos": torch.randint(0, case["far"], (rows,), generator=gen, device="cuda", dtype=torch.int32),
                "wq": 1 + 0.2 * torch.randn(dim, generator=gen, device="cuda"),
                "wk": 1 + 0.2 * torch.randn(dim, generator=gen, device="cuda")}
    new, lens = _lengths(case)
    cache, table = _filled(case, lens, gen)
    s = {"case": case, "cache": cache, "batch": _ragged(new, lens, table)}
    rows, hq, hk, dim = s["batch"]["rows"], case["hq"], case["hk"], case["dim"]
    if case["kind"] == "write":
        s["qkv"] = torch.randn(rows, (hq + 2 * hk) * dim, generator=gen, device="cuda").to(dtype)
        back = lens - (lens - new) // PAGE * PAGE  # from the start of the first page that is written
        s["back"] = _ragged(back, lens, table)
    elif case["kind"] == "attend":
        s["q"] = torch.randn(rows, hq, dim, generator=gen, device="cuda").to(dtype)
        s["scale"] = 1.5 / math.sqrt(dim)
    return s


def run(s):
    if own:
        return _kernels(s)
    kind = s["case"]["kind"]
    if kind == "rope":
        return _plain_rope(s)
    if kind == "attend":
        return _plain_attend(s)
    if kind == "write":
        _plain_write(s)
    return _plain_read(s, s["back"] if kind == "write" else s["batch"])


# ------------------------------------------------------------------ the framework's operators

_ctx = None


def _api():
    root = os.path.join(os.getcwd(), "kokoro-rust_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from kokoro_hip import api
    return api


def _handle(s):
    """What a program keeps for calls on these buffers: their descriptors, outputs and workspace."""
    global _ctx
    api, case = _api(), s["case"]
    if _ctx is None:
        _ctx = api.Context(0)
    code = {"bf16": api.BF16, "f16": api.F16, "f32": api.F32}[case["type"]]
    hq, hk, dim = case["hq"], case["hk"], case["dim"]
    dtype, e = TYPES[case["type"]], 4 if case["type"] == "f32" else 2
    h = {"ctx": _ctx}
    if case["kind"] == "rope":
        wide, rows = (hq + 2 * hk) * dim, case["rows"]
        h["out"] = {"q": torch.empty(rows, hq, dim, dtype=dtype, device="cuda"),
                    "k": torch.empty(rows, hk, dim, dtype=dtype, device="cuda")}
        h["args"] = api.NormRope(
            type=code, dim=dim, rows=rows, q_heads=hq, k_heads=hk, q=s["qkv"].data_ptr(), q_row=wide, q_head=dim,
            k=s["qkv"].data_ptr() + hq * dim * e, k_row=wide, k_head=dim, q_out=h["out"]["q"].data_ptr(),
            q_out_row=hq * dim, q_out_head=dim, k_out=h["out"]["k"].data_ptr(), k_out_row=hk * dim, k_out_head=dim,
            norm=1, eps=s["eps"], q_weight=s["wq"].data_ptr(), k_weight=s["wk"].data_ptr(), pos=s["pos"].data_ptr(),
            rot=case["rot"], interleaved=int(case["inter"]), theta=case["theta"])
        return h
    c = s["cache"]
    h["cache"] = api.KvCache(type=api.KV_INT8 if c["type"] == "int8" else api.KV_E4M3, heads=hk, dim=dim,
                             pages=c["pages"], k=c["k"].data_ptr(), v=c["v"].data_ptr(),
                             k_scale=c["k_scale"].data_ptr(), v_scale=c["v_scale"].data_ptr())

    def batch(b):
        return api.KvBatch(n=b["n"], rows=b["rows"], max_new=b["max_new"], max_len=b["max_len"],
                           row_start=b["row_start"].data_ptr(), len=b["len"].data_ptr(), table=b["table"].data_ptr(),
                           table_width=b["table"].shape[1], table_stride=b["table"].stride(0))

    h["batch"] = batch(s["batch"])
    if case["kind"] == "attend":
        h["out"] = torch.empty(s["q"].shape, dtype=dtype, device="cuda")
        h["args"] = api.KvAttention(type=code, heads=hq, q=s["q"].data_ptr(), q_row=hq * dim, q_head=dim,
                                    out=h["out"].data_ptr(), out_row=hq * dim, out_head=dim, scale=s["scale"],
                                    causal=int(case["causal"]), window=case["window"])
        h["space"] = torch.empty(max(1, _ctx.kv_attention_workspace(h["cache"], h["batch"], h["args"])),
                                 dtype=torch.uint8, device="cuda")
        h["args"].workspace, h["args"].workspace_bytes = h["space"].data_ptr(), h["space"].numel()
        return h
    back = s["back"] if case["kind"] == "write" else s["batch"]
    h["back"] = batch(back)
    h["out"] = {x: torch.empty(back["rows"], hk, dim, dtype=dtype, device="cuda") for x in ("k", "v")}
    h["into"] = api.KvRows(type=code, k=h["out"]["k"].data_ptr(), k_row=hk * dim, k_head=dim,
                           v=h["out"]["v"].data_ptr(), v_row=hk * dim, v_head=dim)
    if case["kind"] == "write":
        wide, at = (hq + 2 * hk) * dim, s["qkv"].data_ptr() + hq * dim * e
        h["rows"] = api.KvRows(type=code, k=at, k_row=wide, k_head=dim, v=at + hk * dim * e, v_row=wide, v_head=dim)
        h["out"] |= {"k_scale": c["k_scale"], "v_scale": c["v_scale"]}
    return h


def _kernels(s):
    h = s.get("handle")
    if h is None:
        h = s["handle"] = _handle(s)
    ctx, kind, stream = h["ctx"], s["case"]["kind"], torch.cuda.current_stream().cuda_stream
    if kind == "rope":
        ctx.qk_norm_rope(h["args"], stream)
    elif kind == "attend":
        ctx.kv_attention(h["cache"], h["batch"], h["args"], stream)
    else:
        if kind == "write":
            ctx.kv_write(h["cache"], h["batch"], h["rows"], stream)
        ctx.kv_read(h["cache"], h["back"], h["into"], stream)
    return h["out"]


# ------------------------------------------------------------------ their plain form


def _plain_rope(s):
    case = s["case"]
    rows, hq, hk, dim, rot = (case[k] for k in ("rows", "hq", "hk", "dim", "rot"))
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    angle = s["pos"].double()[:, None, None] * torch.exp(i * (-2.0 / rot * math.log(case["theta"])))
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def one(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * w
        y = x.clone()
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if case["inter"] else (slice(0, rot // 2), slice(rot // 2, rot))
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., b] * cos + x[..., a] * sin
        return y.to(TYPES[case["type"]])

    q, k = s["qkv"][:, :hq * dim].view(rows, hq, dim), s["qkv"][:, hq * dim:(hq + hk) * dim].view(rows, hk, dim)
    return {"q": one(q, s["wq"]), "k": one(k, s["wk"])}


def _values(data):
    """The numbers that stored bytes stand for, without their scale."""
    return data.float() if data.dtype == torch.int8 else data.view(torch.float8_e4m3fn).float()


def _stored(x, data):
    """The bytes for numbers in units of their scale, in the type of `data`."""
    if data.dtype == torch.int8:
        return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127).to(torch.int8)
    x = torch.nan_to_num(x, nan=0.0, posinf=448.0, neginf=-448.0).clamp(-448, 448)
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _places(b):
    """Each row's sequence, its place among the sequence's rows, and its page and slot in the cache."""
    row = torch.arange(b["rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(b["row_start"][1:], row, right=True)
    new = b["row_start"][1:] - b["row_start"][:-1]
    i = row - b["row_start"][seq]
    pos = (b["len"][seq] - new[seq] + i).long()
    return seq, i.long(), b["table"][seq, pos // PAGE].long(), pos % PAGE


def _plain_write(s):
    case, c = s["case"], s["cache"]
    hq, hk, dim, top = case["hq"], case["hk"], case["dim"], TOP[case["cache"]]
    _, _, page, slot = _places(s["batch"])
    first = torch.full((c["pages"],), PAGE, device="cuda").scatter_reduce(0, page, slot, "amin")
    touched, fresh = (first < PAGE)[:, None], (first == 0)[:, None]
    some = touched[:, 0].nonzero()[:, 0]
    for j, part in enumerate(("k", "v")):
        at = (hq + j * hk) * dim
        x = s["qkv"][:, at:at + hk * dim].view(-1, hk, dim).float()
        size = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
        most = torch.zeros(c["pages"], hk, device="cuda").index_reduce(0, page, size, "amax")
        want = torch.where(most > 0, (most * np.float32(1 / top).item()).clamp(min=LEAST), 0.0)
        data, scale = c[part], c[part + "_scale"]
        old = torch.where(fresh, 0.0, scale)
        now = torch.where(touched, torch.maximum(old, want), scale)
        grown = touched & ~fresh & (now > old)
        ratio = torch.where(grown, old / now, 1.0)
        view = data if part == "k" else data.transpose(2, 3)
        before = view[some]
        again = _stored(_values(before.contiguous()) * ratio[some][:, :, None, None], data)
        kept = torch.arange(PAGE, device="cuda") < first[some][:, None]
        change = kept[:, None, :, None] & grown[some][:, :, None, None]
        view[some] = torch.where(change, again, before)
        inv = torch.where(now > 0, 1.0 / now, 0.0)
        view[page, :, slot] = _stored(x * inv[page][:, :, None], data)
        scale.copy_(now)


def _plain_read(s, b):
    c = s["cache"]
    _, _, page, slot = _places(b)
    out = {}
    for part in ("k", "v"):
        view = c[part] if part == "k" else c[part].transpose(2, 3)
        out[part] = (_values(view[page, :, slot].contiguous()) * c[part + "_scale"][page][:, :, None]).to(TYPES[s["case"]["type"]])
    if s["case"]["kind"] == "write":
        out |= {"k_scale": c["k_scale"], "v_scale": c["v_scale"]}
    return out


def _plain_attend(s):
    case, c, b = s["case"], s["cache"], s["batch"]
    hq, hk, dim, n, most = case["hq"], case["hk"], case["dim"], b["n"], b["max_new"]
    width = -(-b["max_len"] // PAGE)
    table = b["table"][:, :width].clamp(min=0).long()
    k = (_values(c["k"][table]) * c["k_scale"][table][..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, hk, width * PAGE, dim)
    v = (_values(c["v"][table]) * c["v_scale"][table][..., None, None]).permute(0, 2, 1, 4, 3).reshape(n, hk, width * PAGE, dim)
    seq, i, _, _ = _places(b)
    q = torch.zeros(n, most, hq, dim, device="cuda")
    q[seq, i] = s["q"].float()
    q = q.view(n, most, hk, hq // hk, dim).permute(0, 2, 1, 3, 4).reshape(n, hk, -1, dim)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    new = (b["row_start"][1:] - b["row_start"][:-1])[:, None, None]
    pos = b["len"][:, None, None] - new + torch.arange(most, device="cuda")[:, None]
    token = torch.arange(width * PAGE, device="cuda")
    seen = (token < b["len"][:, None, None]).expand(n, most, -1)
    if case["causal"]:
        seen = seen & (token <= pos)
    if case["window"]:
        seen = seen & (token > pos - case["window"])
    seen = seen[:, None, :, None].expand(n, hk, most, hq // hk, -1).reshape(n, hk, -1, width * PAGE)
    score = torch.where(seen, score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    out = out.view(n, hk, most, hq // hk, dim).permute(0, 2, 1, 3, 4).reshape(n, most, hq, dim)
    return out[seq, i].to(TYPES[case["type"]])


# ------------------------------------------------------------------ the definition in 64 bits


def _exact_rope(case, s):
    hq, hk, dim, rot = (case[k] for k in ("hq", "hk", "dim", "rot"))
    freq = torch.tensor([case["theta"] ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones(1, 1, dtype=torch.float64, device="cuda"), s["pos"].double()[:, None] * freq)[:, None]
    heads = s["qkv"][:, :(hq + hk) * dim].view(-1, hq + hk, dim).double()
    done = []
    for x, w in ((heads[:, :hq], s["wq"]), (heads[:, hq:], s["wk"])):
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * w.double()
        pair = x[..., :rot].reshape(*x.shape[:2], rot // 2, 2) if case["inter"] else x[..., :rot].reshape(*x.shape[:2], 2, rot // 2).transpose(2, 3)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z if case["inter"] else z.transpose(2, 3)
        done.append(torch.cat([z.reshape(*x.shape[:2], rot), x[..., rot:]], -1))
    return {"q": done[0], "k": done[1]}


def _exact_values(data):
    if data.dtype == torch.int8:
        return data.double()
    bits = data.to(torch.int64)
    e, m = (bits >> 3) & 15, (bits & 7).double()
    v = torch.where(e > 0, (8 + m) * torch.exp2((e - 10).double()), m * 2.0 ** -9)
    return torch.where(bits >= 128, -v, v)


def _exact_round(x, cache):
    if cache == "int8":
        return x.round().clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_cache(case, s):
    """What is written and read back, page by page."""
    c, b = s["cache"], s["batch"]
    hq, hk, dim, top = case["hq"], case["hk"], case["dim"], TOP[case["cache"]]
    new, lens = _lengths(case)
    table = b["table"].cpu().numpy()
    out = {"k": [], "v": []}
    scales = {p: c[p + "_scale"].double() for p in out}
    for part in out:
        if case["kind"] == "write":
            at = (hq + (part == "v") * hk) * dim
            x = s["qkv"][:, at:at + hk * dim].view(-1, hk, dim).double().transpose(0, 1)
        row = 0
        for j, (n, m) in enumerate(zip(lens.tolist(), new.tolist())):
            seq, pos = [], n - m
            for p in range(pos // PAGE, -(-n // PAGE)):
                page = int(table[j, p])
                stored = _exact_values(c[part][page])
                stored = stored if part == "k" else stored.transpose(1, 2)
                lo, hi = max(pos, p * PAGE) - p * PAGE, min(n, (p + 1) * PAGE) - p * PAGE
                scale = scales[part][page]
                if case["kind"] == "write":
                    t = x[:, row:row + hi - lo]
                    want = t.abs().amax((1, 2)) / top
                    now = want if lo == 0 else torch.maximum(scale, want)
                    stored = _exact_round(stored[:, :lo] * (scale / now)[:, None, None], case["cache"]) if lo else stored[:, :0]
                    stored = torch.cat([stored, _exact_round(t / now[:, None, None], case["cache"])], 1)
                    scales[part][page] = scale = now
                    lo, row = 0, row + t.shape[1]
                seq.append(stored[:, lo:hi] * scale[:, None, None])
            out[part].append(torch.cat(seq, 1).transpose(0, 1) if seq else torch.zeros(0, hk, dim, device="cuda"))
    out = {p: torch.cat(v) for p, v in out.items()}
    if case["kind"] == "write":
        out |= {"k_scale": scales["k"], "v_scale": scales["v"]}
    return out


def _exact_attend(case, s):
    c, b = s["cache"], s["batch"]
    hq, hk = case["hq"], case["hk"]
    new, lens = _lengths(case)
    group, row, out = hq // hk, 0, []
    for j, (n, m) in enumerate(zip(lens.tolist(), new.tolist())):
        pages = b["table"][j, :-(-n // PAGE)].long()
        pos = torch.arange(n - m, n, device="cuda")[:, None, None]
        token = torch.arange(n, device="cuda")
        hidden = token > pos if case["causal"] else token < 0
        if case["window"]:
            hidden = hidden | (token <= pos - case["window"])
        heads = []
        for h in range(hk):
            k = (_exact_values(c["k"][pages, h]) * c["k_scale"][pages, h].double()[:, None, None]).reshape(-1, case["dim"])[:n]
            v = (_exact_values(c["v"][pages, h]) * c["v_scale"][pages, h].double()[:, None, None]).transpose(1, 2).reshape(-1, case["dim"])[:n]
            q = s["q"][row:row + m, h * group:(h + 1) * group].double()
            a = torch.softmax((q.reshape(m * group, -1) @ k.T * s["scale"]).view(m, group, n).masked_fill(hidden, -math.inf), -1)
            heads.append((a.view(m * group, n) @ v).view(m, group, -1))
        out.append(torch.cat(heads, 1))
        row += m
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "write": _exact_cache, "read": _exact_cache, "attend": _exact_attend}[case["kind"]](case, s)
