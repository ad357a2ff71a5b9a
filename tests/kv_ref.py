"""The cache operators' definitions for their tests, in numpy and torch on the CPU: what is stored, bit for bit (the
documented f32 steps), attention and rotation in 64 bits; and the buffers that a caller of the library holds."""
import ctypes as C

import numpy as np
import torch

PAGE = 64
TOP = {"int8": 127.0, "e4m3": 448.0}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}     # of a value, the largest rounding error
LEAST_STEP = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25, "f32": 2.0 ** -150}  # half a step of the subnormals


def values(data):
    """Stored bytes as numbers (f64)."""
    return data.to(torch.float64) if data.dtype == torch.int8 else data.view(torch.float8_e4m3fn).to(torch.float64)


def store(x, kind):
    """f32 numbers in units of their scale to stored bytes."""
    top = TOP[kind]
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=top, neginf=-top).clamp(-top, top)
    return x.round().to(torch.int8) if kind == "int8" else x.to(torch.float8_e4m3fn).view(torch.uint8)


class Cache:
    """A cache on the device and what the definition says it holds, on the host."""

    def __init__(self, kind, heads, dim, pages, fill=0x7f):
        from kokoro_hip import api
        self.kind, self.heads, self.dim, self.pages = kind, heads, dim, pages
        d = torch.int8 if kind == "int8" else torch.uint8
        # every byte that has not been written is the NaN code of e4m3, every scale NaN
        self.ref = {"k": torch.full((pages, heads, PAGE, dim), fill, dtype=d), "v": torch.full((pages, heads, dim, PAGE), fill, dtype=d),
                    "k_scale": torch.full((pages, heads), float("nan")), "v_scale": torch.full((pages, heads), float("nan"))}
        self.dev = {k: v.cuda() for k, v in self.ref.items()}
        self.fault = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.args = api.KvCache(type=api.KV_INT8 if kind == "int8" else api.KV_E4M3, heads=heads, dim=dim, pages=pages,
                                fault=self.fault.data_ptr(), **{k: v.data_ptr() for k, v in self.dev.items()})

    def write(self, page, lo, x, part):
        """x: [tokens, heads, dim] f32 into slots lo.. of a page, as documented for kk_kv_write."""
        top, data, scale = TOP[self.kind], self.ref[part], self.ref[part + "_scale"]
        tokens = data[page] if part == "k" else data[page].transpose(1, 2)  # [heads][64][dim]
        size = torch.where(torch.isfinite(x), x.abs(), torch.zeros(())).amax((0, 2))
        want = torch.where(size > 0, (size * torch.tensor(np.float32(1 / top))).clamp(min=2.0 ** -90), torch.zeros(()))
        was = scale[page].clone() if lo else torch.zeros(self.heads)
        now = torch.maximum(was, want)
        for h in range(self.heads):
            if lo and now[h] > was[h]:
                tokens[h, :lo] = store(values(tokens[h, :lo].contiguous()).float() * (was[h] / now[h]), self.kind)
            inv = 1 / now[h] if now[h] > 0 else torch.zeros(())
            tokens[h, lo:lo + len(x)] = store(x[:, h] * inv, self.kind)
        scale[page] = now

    def tokens(self, pages, n, part):
        """The first n tokens of a sequence in those pages: [n, heads, dim] in f64."""
        t = values(self.ref[part][pages].contiguous()) * self.ref[part + "_scale"][pages].double()[:, :, None, None]
        t = t if part == "k" else t.transpose(2, 3)
        return t.transpose(1, 2).reshape(-1, self.heads, self.dim)[:n]

    def scales(self, pages, n):
        """V's scale of each of those tokens: [n, heads]."""
        return self.ref["v_scale"][pages].double().repeat_interleave(PAGE, 0)[:n]

    def same(self):
        for k, v in self.ref.items():
            got = self.dev[k].cpu()
            assert torch.equal(got.view(torch.int32) if got.dtype == torch.float32 else got,
                               v.view(torch.int32) if v.dtype == torch.float32 else v), k
        return True


class Batch:
    """kk_kv_batch: sequences of `new` rows and `lens` tokens with their page numbers."""

    def __init__(self, new, lens, tables, max_new=None, max_len=None, rows=None, first=0, width=None):
        from kokoro_hip import api
        self.new, self.lens, self.tables = list(new), list(lens), [list(t) for t in tables]
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) + first
        self.rows = int(self.start[-1]) if rows is None else rows
        width = max([len(t) for t in self.tables] + [1]) if width is None else width
        table = np.full((max(1, len(self.tables)), width + 2), -1, np.int32)
        for b, t in enumerate(self.tables):
            table[b, :len(t)] = t
        self.dev = [torch.from_numpy(a).cuda() for a in (self.start, np.asarray(self.lens or [0], np.int32), table)]
        self.args = api.KvBatch(n=len(self.lens), rows=self.rows, max_new=max(self.new + [0]) if max_new is None else max_new,
                                max_len=max(self.lens + [0]) if max_len is None else max_len, row_start=self.dev[0].data_ptr(),
                                len=self.dev[1].data_ptr(), table=self.dev[2].data_ptr(), table_width=width,
                                table_stride=width + 2)

    def of(self, b):
        return range(self.start[b], self.start[b + 1])


def deal(lens, pages, rng):
    """Page numbers for sequences of those lengths, none shared."""
    order = rng.permutation(pages)
    out, at = [], 0
    for n in lens:
        need = -(-n // PAGE)
        out.append(order[at:at + need].tolist())
        at += need
    assert at <= pages
    return out


def rows_of(type_, k, v):
    """kk_kv_rows over device tensors [rows, heads, dim] of any strides."""
    from kokoro_hip import api
    assert k.stride(2) == 1 and v.stride(2) == 1
    return api.KvRows(type=type_, k=k.data_ptr(), k_row=k.stride(0), k_head=k.stride(1), v=v.data_ptr(), v_row=v.stride(0),
                      v_head=v.stride(1))


def write(ctx, cache, batch, k, v, type_, stream=0):
    """kk_kv_write of device tensors k, v, and the same on the reference side."""
    ctx.kv_write(cache.args, batch.args, rows_of(type_, k, v), stream)
    for part, x in (("k", k.float().cpu()), ("v", v.float().cpu())):
        for b, n in enumerate(batch.lens):
            rows, pos = list(batch.of(b)), n - batch.new[b]
            while rows:
                lo = pos % PAGE
                take = min(len(rows), PAGE - lo)
                cache.write(batch.tables[b][pos // PAGE], lo, x[rows[:take]], part)
                rows, pos = rows[take:], pos + take


def attend(q, k, v, b, scale, causal, window):
    """Rows q [m, heads, dim] at the end of tokens k, v [n, cache heads, dim] whose V has scales b [n, cache heads], in f64: the
    result, and what rounding errors are in proportion to: sum p |v|, the largest sum |q k| scale of a row, and each (row, head)'s
    largest p b."""
    m, n, group = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    if n == 0:
        return torch.zeros_like(q), torch.zeros_like(q), 0.0, torch.zeros(m, q.shape[1], 1)
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("mhd,nhd->hmn", q, k) * scale
    size = float((torch.einsum("mhd,nhd->hmn", q.abs(), k.abs()) * scale).max()) if m else 0.0
    pos = torch.arange(n - m, n)[:, None]
    t = torch.arange(n)
    seen = torch.ones(m, n, dtype=torch.bool)
    if causal:
        seen = t <= pos
    if window:
        seen = seen & (t > pos - window)
    s = s.masked_fill(~seen, -torch.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    most = (p * b.repeat_interleave(group, 1).T[:, None]).amax(-1).T[:, :, None]
    return torch.einsum("hmn,nhd->mhd", p, v), torch.einsum("hmn,nhd->mhd", p, v.abs()), size, most


def attention_args(ctx, cache, batch, q, out, type_, scale, causal=True, window=0):
    """kk_kv_attention_args and the workspace that they need (with a guard behind it)."""
    from kokoro_hip import api
    a = api.KvAttention(type=type_, heads=q.shape[1], q=q.data_ptr(), q_row=q.stride(0), q_head=q.stride(1), out=out.data_ptr(),
                        out_row=out.stride(0), out_head=out.stride(1), scale=scale, causal=int(causal), window=window)
    n = ctx.kv_attention_workspace(cache.args, batch.args, a)
    space = torch.full((n + 256,), 0xA5, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = space.data_ptr(), n
    return a, space


def check_attention(out, q, cache, batch, scale, causal, window, kind, only=None):
    """out against f64 over what the cache holds.  Error bound per value:
    - the result's own rounding, half a step;
    - P held in f16: 2^-11 of each p |v|; and below f16's normal numbers half its smallest step, 2^-25, where the row's largest P
      is at least 2^11 (the lift): 2^-36 of the largest p b for every token, times its stored number, at most `top`;
    - scores in f32, off by at most (dim + 8) 2^-24 of sum |q k| scale (dim products summed, the scale and the exponent's
      arithmetic), which changes each p, and the sum that they are divided by, by that much."""
    q = q.cpu().double()
    for b, n in enumerate(batch.lens):
        if only is not None and b not in only:
            continue
        r = slice(int(batch.start[b]), int(batch.start[b + 1]))
        k, v = [cache.tokens(batch.tables[b], n, p) for p in "kv"]
        want, size, score, most = attend(q[r], k, v, cache.scales(batch.tables[b], n), scale, causal, window)
        tol = HALF_STEP[kind] * want.abs() + LEAST_STEP[kind] + n * 2.0 ** -36 * TOP[cache.kind] * most
        tol = tol + (2.0 ** -11 + 2 * (q.shape[2] + 8) * 2.0 ** -24 * score) * size
        off = (out[r].cpu().double() - want).abs()
        assert bool((off <= tol).all()), (b, n, float((off / tol).nan_to_num(nan=1e9).max()))
