"""The operators over an 8-bit cache on the GPU, through the library's entry points, against their definitions in 64 bits
(tests/kv_ref.py): writing and reading back bit for bit, attention within a bound derived there, a decoding loop of all of them,
graphs, streams, and batches whose arrays are wrong."""
import numpy as np
import pytest
import torch

import kv_ref as R

pytestmark = pytest.mark.gpu
PAGE = R.PAGE


@pytest.fixture(scope="module")
def ctx():
    from kokoro_hip import api
    torch.cuda.init()
    c = api.Context(0)
    yield c
    c.close()


def _code(kind):
    from kokoro_hip import api
    return {"bf16": api.BF16, "f16": api.F16, "f32": api.F32}[kind]


def _kv(rows, heads, dim, kind, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, rows, heads, dim, generator=g) * scale * torch.exp(0.7 * torch.randn(2, rows, 1, 1, generator=g))
    return [t.to(R.TYPES[kind]).cuda() for t in x]


# ------------------------------------------------------------------ writing and reading back


@pytest.mark.parametrize("cache_kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dim, heads, kind", [(64, 1, "f32"), (96, 3, "f16"), (128, 2, "bf16"), (192, 1, "bf16"), (256, 2, "f16")])
def test_write_and_read(ctx, cache_kind, dim, heads, kind):
    """Prompts, then pieces and single tokens behind them (pages that grow), bit for bit; the reading back of all tokens, rounded
    once; and the error of each stored token within half a step for its page's scale and for each time the scale grew."""
    rng = np.random.default_rng(dim)
    lens = [1, 63, 64, 65, 0, 200, 127]
    add = [[1, 1, 1, 1, 0, 1, 1], [70, 5, 64, 0, 130, 17, 1], [0, 1, 1, 2, 1, 0, 63]]
    total = [n + sum(a[b] for a in add) for b, n in enumerate(lens)]
    cache = R.Cache(cache_kind, heads, dim, sum(-(-n // PAGE) for n in total) + 3)
    tables = R.deal(total, cache.pages, rng)
    have, truth, grown = [0] * len(lens), [[[], []] for _ in lens], [np.zeros((2, n, heads)) for n in total]
    for step, new in enumerate([lens] + add):
        scale = {p: cache.ref[p + "_scale"].clone() for p in "kv"}
        start = have[:]
        have = [h + n for h, n in zip(have, new)]
        batch = R.Batch(new, have, tables, max_len=max(have) + 5)
        k, v = _kv(batch.rows, heads, dim, kind, 10 * dim + step, 1.0 + 2.0 * step)
        R.write(ctx, cache, batch, k, v, _code(kind))
        cache.same()
        for b in range(len(lens)):
            for j, x in enumerate((k, v)):
                truth[b][j].append(x[list(batch.of(b))].double().cpu())
            p = start[b] // PAGE  # the page that was partly full
            if start[b] % PAGE and new[b]:
                for j, part in enumerate("kv"):
                    more = (cache.ref[part + "_scale"][tables[b][p]] > scale[part][tables[b][p]]).numpy()
                    grown[b][j, p * PAGE:start[b]] += more
    batch = R.Batch(have, have, tables)
    out = [torch.full((batch.rows + 2, heads, dim), 7.0, dtype=R.TYPES[kind], device="cuda") for _ in range(2)]
    ctx.kv_read(cache.args, batch.args, R.rows_of(_code(kind), *out))
    top = R.TOP[cache_kind]
    for j, part in enumerate("kv"):
        got = out[j].cpu()
        assert (got[batch.rows:] == 7.0).all()
        for b, n in enumerate(have):
            # stored number times scale in f32 is one rounding, to the type a second (of f32 to f32: none)
            want = cache.tokens(tables[b], n, part)
            assert torch.equal(got[list(batch.of(b))], want.float().to(R.TYPES[kind]))
            x = torch.cat(truth[b][j])
            scale = cache.ref[part + "_scale"][tables[b]].double().repeat_interleave(PAGE, 0)[:n][:, :, None]
            # half a step (e4m3: of the number, at least of its subnormals), once and once for each growth, and what
            # the reciprocal and the products round
            step = scale * 0.5 if cache_kind == "int8" else torch.maximum(2.0 ** -4 * x.abs(), scale * 2.0 ** -10)
            if cache_kind == "e4m3":  # a later step is a half step of a number that is off by the earlier ones
                step = step * (1 + 2.0 ** -4) ** torch.from_numpy(grown[b][j])[:, :, None]
            tol = step * (1 + torch.from_numpy(grown[b][j])[:, :, None]) + 2.0 ** -20 * (x.abs() + top * scale * 2.0 ** -10)
            assert ((want - x).abs() <= tol).all()
    assert int(cache.fault) == 0


@pytest.mark.parametrize("cache_kind", ["int8", "e4m3"])
def test_write_special_values(ctx, cache_kind):
    """Zeros, infinities, NaN, the smallest and largest values: scales and bytes as documented."""
    cache = R.Cache(cache_kind, 4, 64, 4)
    x = torch.randn(5, 4, 64, generator=torch.Generator().manual_seed(3))
    x[:, 0] = 0.0
    x[1, 1, 3], x[2, 1, 4], x[3, 1, 5] = np.inf, -np.inf, np.nan
    x[:, 2] *= 1e-39
    x[:, 3] *= 3e37
    one = R.Batch([5], [5], [[2]])
    R.write(ctx, cache, one, x.cuda(), -x.cuda(), _code("f32"))
    cache.same()
    only = torch.full((1, 4, 64), np.nan)
    only[0, 1] = np.inf
    R.write(ctx, cache, R.Batch([1], [6], [[2]]), only.cuda(), only.cuda(), _code("f32"))  # no finite value: the scales stay
    cache.same()
    R.write(ctx, cache, R.Batch([1], [7], [[2]]), x[:1].cuda() + 1e30, x[:1].cuda(), _code("f32"))  # zeros grow to a scale
    cache.same()
    out = [torch.empty(7, 4, 64, device="cuda") for _ in range(2)]
    ctx.kv_read(cache.args, R.Batch([7], [7], [[2]]).args, R.rows_of(_code("f32"), *out))
    for part, o in zip("kv", out):
        assert torch.equal(o.cpu(), cache.tokens([2], 7, part).float())


@pytest.mark.parametrize("cache_kind", ["int8", "e4m3"])
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_write_beside_infinities(ctx, cache_kind, kind):
    """Infinities and NaN in some heads of a page that is written in two calls, none in the others; values that round to the
    largest number of their type; ties of the 8-bit rounding."""
    cache = R.Cache(cache_kind, 3, 96, 3)
    g = torch.Generator().manual_seed(7)
    x = torch.randn(80, 3, 96, generator=g)
    x[:, 2] = torch.randint(-254, 255, (80, 96), generator=g) / 2.0  # halves in units of a scale of 1
    x[0, 2, 0] = x[70, 2, 1] = 127.0
    x[3, 0, 5], x[4, 0, 6], x[70, 0, 7], x[50, 1, 9] = np.inf, -np.inf, np.nan, torch.finfo(R.TYPES[kind]).max
    x = x.to(R.TYPES[kind]).cuda()
    for start, n in ((0, 30), (30, 40), (70, 10)):
        batch = R.Batch([n], [start + n], [[2, 0]], max_len=100, width=2)
        R.write(ctx, cache, batch, x[start:start + n], -x[start:start + n], _code(kind))
        cache.same()


@pytest.mark.parametrize("n, most", [(90, 1), (40, 9), (3, 2000)])
def test_write_many_sequences(ctx, n, most):
    """Batches on both ways of finding a block's page (each sequence's pages, and a search), ragged, some without rows; packed
    q | k | v rows as input, unaligned rows as well, and rows outside the sequences."""
    rng = np.random.default_rng(n)
    new = rng.integers(0, most + 1, n)
    new[0] = most
    if most == 2000:
        new[1:] = [0, 3]
    lens = new + rng.integers(0, 90, n)
    cache = R.Cache("int8", 2, 128, int(sum(-(-lens // PAGE))) + 2)
    tables = R.deal(lens, cache.pages, rng)
    before = R.Batch(lens - new, lens - new, tables)
    k, v = _kv(max(1, before.rows), 2, 128, "bf16", 1)
    R.write(ctx, cache, before, k, v, _code("bf16"))
    batch = R.Batch(new, lens, tables, rows=int(new.sum()) + 9, first=4)
    for shift in (0, 1):  # the second time the same tokens from rows that are not 16-byte aligned
        packed = torch.full((batch.rows, 6 * 128 + shift), float("nan"), dtype=torch.bfloat16, device="cuda")
        a = [packed[:, (2 + 2 * j) * 128 + shift:(4 + 2 * j) * 128 + shift].unflatten(1, (2, 128)) for j in range(2)]
        k, v = _kv(batch.rows, 2, 128, "bf16", 2)
        a[0][4:-5], a[1][4:-5] = k[4:-5], v[4:-5]
        R.write(ctx, cache, batch, a[0], a[1], _code("bf16"))
        cache.same()
    out = [torch.zeros(batch.rows, 5, 129, dtype=torch.bfloat16, device="cuda")[:, 1:3, 1:] for _ in range(2)]
    ctx.kv_read(cache.args, batch.args, R.rows_of(_code("bf16"), *out))
    for part, o in zip("kv", out):
        for b in range(n):
            want = cache.tokens(tables[b], int(lens[b]), part)[int(lens[b] - new[b]):]
            assert torch.equal(o[list(batch.of(b))].cpu(), want.float().bfloat16())
        assert not o[:4].any() and not o[batch.start[-1]:].any()
    assert int(cache.fault) == 0


# ------------------------------------------------------------------ attention


def _filled(ctx, cache_kind, heads, dim, lens, seed, spread=0.5, spare=2):
    """A cache that holds those sequences (written by the library, checked), and its tables."""
    rng = np.random.default_rng(seed)
    cache = R.Cache(cache_kind, heads, dim, sum(-(-n // PAGE) for n in lens) + spare)
    tables = R.deal(lens, cache.pages, rng)
    batch = R.Batch(lens, lens, tables)
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(max(1, batch.rows), heads, dim, generator=g) * torch.exp(spread * torch.randn(max(1, batch.rows), 1, 1, generator=g))
            for _ in range(2))
    R.write(ctx, cache, batch, k.cuda(), v.cuda(), _code("f32"))
    cache.same()
    return cache, tables


CASES = [
    # cache, type, heads, group, dim, new rows, tokens, causal, window, bound on the tokens (0: the longest)
    ("int8", "bf16", 2, 1, 64, [1], [1], True, 0, 0),
    ("int8", "bf16", 2, 4, 128, [1, 1, 1, 0, 1], [1, 63, 64, 70, 65], True, 0, 0),
    ("e4m3", "f16", 1, 16, 96, [1, 1, 1], [500, 1, 129], True, 0, 0),
    ("e4m3", "bf16", 2, 5, 192, [3, 2, 3], [3, 64, 700], True, 0, 0),             # 15 rows
    ("int8", "f16", 1, 8, 256, [4, 1, 3], [1100, 600, 3], True, 0, 0),            # 32 rows, the axis in parts
    ("int8", "bf16", 3, 3, 64, [1, 1], [3000, 17], True, 0, 0),                   # parts, one sequence with one
    ("e4m3", "f16", 2, 4, 128, [5, 5], [1500, 1024], True, 0, 20000),             # parts by a bound far above
    ("int8", "bf16", 1, 4, 128, [8, 3], [900, 1000], True, 100, 0),               # a window of few rows
    ("int8", "bf16", 2, 4, 128, [9], [9], True, 0, 0),                            # 36 rows: the kernel for prompts
    ("e4m3", "bf16", 1, 2, 64, [64, 65, 1, 0, 200], [64, 65, 300, 5, 263], True, 0, 0),
    ("int8", "f16", 2, 3, 96, [130, 43], [130, 1000], True, 0, 0),                # groups that do not divide a block
    ("int8", "bf16", 1, 8, 128, [100], [2500], True, 0, 0),                       # prompts, the axis in parts
    ("e4m3", "f16", 1, 4, 128, [140, 70], [900, 70], True, 33, 0),                # window smaller than a page
    ("int8", "bf16", 1, 1, 192, [150], [400], True, 128, 0),
    ("e4m3", "bf16", 1, 2, 256, [90, 40], [90, 333], True, 0, 0),
    ("int8", "bf16", 2, 2, 64, [20, 70, 3], [100, 30, 0], False, 0, 0),           # without causal: more rows than tokens, none
    ("e4m3", "f16", 1, 2, 128, [3, 2], [200, 0], False, 0, 0),
    ("int8", "f16", 1, 2, 64, [70, 40], [50, 40], True, 0, 0),                    # rows before the first token see nothing
    ("int8", "bf16", 1, 2, 128, [7, 2], [4, 2], True, 3, 0),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(ctx, case):
    cache_kind, kind, heads, group, dim, new, lens, causal, window, bound = CASES[case]
    cache, tables = _filled(ctx, cache_kind, heads, dim, lens, case)
    batch = R.Batch(new, lens, tables, first=2, rows=sum(new) + 5, max_len=bound, width=-(-bound // PAGE)) if bound else \
        R.Batch(new, lens, tables, first=2, rows=sum(new) + 5)
    g = torch.Generator().manual_seed(case)
    q = (torch.randn(batch.rows, heads * group, dim, generator=g) * 2).to(R.TYPES[kind]).cuda()
    out = torch.full((batch.rows, heads * group, dim), 9.0, dtype=R.TYPES[kind], device="cuda")
    args, space = R.attention_args(ctx, cache, batch, q, out, _code(kind), 1.3 / dim ** 0.5, causal, window)
    ctx.kv_attention(cache.args, batch.args, args)
    R.check_attention(out, q, cache, batch, 1.3 / dim ** 0.5, causal, window, kind)
    assert (out[:2] == 9.0).all() and (out[batch.start[-1]:] == 9.0).all()
    assert (space[args.workspace_bytes:] == 0xA5).all()
    assert int(cache.fault) == 0
    again = out.clone()
    ctx.kv_attention(cache.args, batch.args, args)
    assert torch.equal(out, again)


def test_attention_of_many_sequences(ctx):
    """700 sequences, most of them short, some without rows or tokens, a few long ones: parts that only some sequences have."""
    rng = np.random.default_rng(11)
    lens = rng.integers(0, 90, 700)
    lens[[3, 300, 301, 699]] = [1500, 9000, 64, 4321]
    new = (rng.random(700) < 0.8).astype(int) * (lens > 0)
    new[[3, 300, 699, 0]] = [3, 1, 2, 1]
    lens[0] = 0  # a row that sees nothing
    cache, tables = _filled(ctx, "int8", 1, 64, lens.tolist(), 12)
    batch = R.Batch(new.tolist(), lens.tolist(), tables)
    q = torch.randn(batch.rows, 4, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    out = torch.full_like(q, 9.0)
    args, space = R.attention_args(ctx, cache, batch, q, out, _code("bf16"), 0.2)
    assert args.workspace_bytes > 0
    ctx.kv_attention(cache.args, batch.args, args)
    R.check_attention(out, q, cache, batch, 0.2, True, 0, "bf16")
    assert (space[args.workspace_bytes:] == 0xA5).all() and int(cache.fault) == 0


@pytest.mark.parametrize("cache_kind, kind, group, dim, causal, window", [
    ("int8", "bf16", 1, 128, True, 0), ("e4m3", "f16", 3, 64, True, 0), ("e4m3", "bf16", 2, 128, True, 700),
    ("int8", "f16", 4, 96, False, 0), ("int8", "bf16", 1, 192, True, 0)])
@pytest.mark.parametrize("n", [62, 130])
def test_attention_of_many_rows(ctx, n, cache_kind, kind, group, dim, causal, window):
    """Prompts over up to 150 pages, from sequences of one page up, with rows that see nothing and blocks that are mostly empty:
    130 sequences' blocks of 256 rows (128 for heads of 192 values) fill the device and are not split, 62 are fewer."""
    rng = np.random.default_rng(dim + group)
    new, lens = rng.integers(1, 60, n), rng.integers(0, 700, n)
    new[[0, 1, 2, 3, 4, 5]], lens[[0, 1, 2, 3, 4, 5]] = [300, 40, 50, 0, 129, 1], [9500, 4200, 5, 80, 129, 64]
    if causal:
        lens[6:] += new[6:]
    cache, tables = _filled(ctx, cache_kind, 4, dim, lens.tolist(), 12)
    batch = R.Batch(new.tolist(), lens.tolist(), tables, first=1)
    g = torch.Generator().manual_seed(dim)
    q = (2 * torch.randn(batch.rows, 4 * group, dim, generator=g)).to(R.TYPES[kind]).cuda()
    out = torch.full_like(q, 9.0)
    args, _ = R.attention_args(ctx, cache, batch, q, out, _code(kind), 1.2 / dim ** 0.5, causal, window)
    assert n == 62 or args.workspace_bytes == 0
    ctx.kv_attention(cache.args, batch.args, args)
    R.check_attention(out, q, cache, batch, 1.2 / dim ** 0.5, causal, window, kind)
    again = torch.full_like(q, 9.0)
    args.out = again.data_ptr()
    ctx.kv_attention(cache.args, batch.args, args)
    assert torch.equal(out, again) and int(cache.fault) == 0


@pytest.mark.parametrize("new", [1, 40])
def test_attention_rows_and_strides(ctx, new):
    """Queries and outputs in wider rows, aligned to 16 bytes and not; the same values as from packed ones."""
    cache, tables = _filled(ctx, "int8", 2, 128, [300], 5)
    batch = R.Batch([new], [300], tables)
    q = torch.randn(new, 6, 128, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    outs = []
    for wide, at in ((768, 0), (1024, 8), (1001, 3)):
        buf = torch.full((new, wide), 5.0, dtype=torch.bfloat16, device="cuda")
        res = torch.full((new, wide), 5.0, dtype=torch.bfloat16, device="cuda")
        view, out = (x[:, at:at + 768].unflatten(1, (6, 128)) for x in (buf, res))
        view.copy_(q)
        args, _ = R.attention_args(ctx, cache, batch, view, out, _code("bf16"), 0.09)
        ctx.kv_attention(cache.args, batch.args, args)
        outs.append(out.clone())
        assert (res[:, :at] == 5.0).all() and (res[:, at + 768:] == 5.0).all()
    R.check_attention(outs[0], q, cache, batch, 0.09, True, 0, "bf16")
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("cache_kind", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [2, 50])
@pytest.mark.parametrize("unit", [1.0, 2.0 ** -70, 2.0 ** 60])
def test_attention_page_scales(ctx, cache_kind, new, unit):
    """Pages of zeros, pages 2^40 times larger that no row attends to, and 2^10 times smaller ones that all do; all of V in several
    units (a page of zeros has none and must not set one)."""
    lens = [320]
    cache = R.Cache(cache_kind, 1, 64, 7)
    tables = R.deal(lens, 7, np.random.default_rng(2))
    g = torch.Generator().manual_seed(8)
    k, v = torch.randn(320, 1, 64, generator=g), torch.randn(320, 1, 64, generator=g)
    k[:64], v[:64] = 0.0, 0.0              # zeros: scores of 0 and nothing to add, but weight in the sum
    v[64:128] *= 2.0 ** 40                 # large and far below every row's best score
    k[64:128] = -k[64:128].abs() * 4
    v[192:256] *= 2.0 ** -10
    v[256:] = 0.0
    R.write(ctx, cache, R.Batch(lens, lens, tables), k.cuda(), (v * unit).cuda(), _code("f32"))
    batch = R.Batch([new], lens, tables)
    q = (2 + torch.rand(new, 2, 64, generator=g)).bfloat16().cuda()
    out = torch.empty(new, 2, 64, dtype=torch.bfloat16, device="cuda")
    args, _ = R.attention_args(ctx, cache, batch, q, out, _code("bf16"), 0.25)
    ctx.kv_attention(cache.args, batch.args, args)
    R.check_attention(out, q, cache, batch, 0.25, True, 0, "bf16")


@pytest.mark.parametrize("new", [1, 40])
def test_attention_small_weights_add_up(ctx, new):
    """One token far above 19,000 others whose weights are below 2^-24 of its own and still add up to part of the result."""
    n = 19000
    cache = R.Cache("int8", 1, 64, 300)
    tables = R.deal([n], 300, np.random.default_rng(3))
    k = torch.full((n, 1, 64), -1.0)
    v = torch.ones(n, 1, 64) * torch.linspace(0.5, 1.0, 64)
    k[77], v[77] = 1.0, -1.0
    whole = R.Batch([n], [n], tables)
    R.write(ctx, cache, whole, k.cuda(), v.cuda(), _code("f32"))
    batch = R.Batch([new], [n], tables)
    q = torch.ones(new, 1, 64).half().cuda()
    out = torch.empty(new, 1, 64, dtype=torch.float16, device="cuda")
    for bits in (12.5, 20.0, 27.0):  # each weighs 2^-bits: together 2.7 times the one, 2^-6 and 2^-13 of it
        scale = bits * 0.6931 / 128  # q . k is 64 and -64
        args, _ = R.attention_args(ctx, cache, batch, q, out, _code("f16"), scale)
        ctx.kv_attention(cache.args, batch.args, args)
        R.check_attention(out, q, cache, batch, scale, True, 0, "f16")


@pytest.mark.parametrize("new", [3, 40])
def test_attention_bad_values_stay_in_their_row(ctx, new):
    """NaN and infinity in one query row make that row NaN and no other; a large query keeps its softmax."""
    cache, tables = _filled(ctx, "int8", 1, 128, [200], 6)
    batch = R.Batch([new], [200], tables)
    q = torch.randn(new, 2, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    q[1, 0, 5], q[2, 1, 7] = float("nan"), float("inf")
    q[0, 1] *= 1e4
    q = q.cuda()
    out = torch.empty_like(q)
    args, _ = R.attention_args(ctx, cache, batch, q, out, _code("bf16"), 0.1)
    ctx.kv_attention(cache.args, batch.args, args)
    bad = torch.zeros(new, 2, dtype=torch.bool)
    bad[1, 0] = bad[2, 1] = True
    assert torch.equal(out.isnan().all(-1).cpu(), bad) and torch.equal(out.isnan().any(-1).cpu(), bad)
    q[1, 0, 5], q[2, 1, 7] = 0.0, 0.0
    clean = torch.empty_like(q)
    args.out = clean.data_ptr()
    ctx.kv_attention(cache.args, batch.args, args)
    out, clean = out.cpu(), clean.cpu()
    assert torch.equal(out[~bad], clean[~bad])
    R.check_attention(clean, q, cache, batch, 0.1, True, 0, "bf16")


# ------------------------------------------------------------------ batches whose device arrays are wrong


def test_bad_pages(ctx):
    """Page numbers outside the cache: nothing of them is written, what is read there is NaN, the others are as they should be."""
    from kokoro_hip import api
    cache, tables = _filled(ctx, "e4m3", 2, 64, [130, 70], 9)
    bad = [[tables[0][0], cache.pages, tables[0][2]], [-5, tables[1][1]]]
    batch = R.Batch([3, 1], [130, 70], bad)
    k, v = _kv(4, 2, 64, "bf16", 1)
    cache.write(tables[0][2], 0, k[1:3].float().cpu(), "k")  # rows 0 (page `pages`) and 3 (page -5's second page is fine)
    cache.write(tables[0][2], 0, v[1:3].float().cpu(), "v")
    cache.write(tables[1][1], 5, k[3:].float().cpu(), "k")
    cache.write(tables[1][1], 5, v[3:].float().cpu(), "v")
    ctx.kv_write(cache.args, batch.args, R.rows_of(_code("bf16"), k, v))
    cache.same()
    assert int(cache.fault) == api.KV_BAD_PAGE
    cache.fault.zero_()
    out = [torch.zeros(200, 2, 64, device="cuda") for _ in range(2)]
    whole = R.Batch([130, 70], [130, 70], bad)
    ctx.kv_read(cache.args, whole.args, R.rows_of(_code("f32"), *out))
    for o, part in zip(out, "kv"):
        o = o.cpu()
        assert o[64:128].isnan().all() and o[130:194].isnan().all()
        assert torch.equal(o[:64], cache.tokens(tables[0], 64, part).float())
        assert torch.equal(o[194:], cache.tokens(tables[1], 70, part)[64:].float())
    assert int(cache.fault) == api.KV_BAD_PAGE
    for new in ([1, 1], [40, 40]):
        cache.fault.zero_()
        batch = R.Batch(new, [130, 70], bad)
        q = torch.randn(sum(new), 2, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
        o = torch.zeros_like(q)
        args, _ = R.attention_args(ctx, cache, batch, q, o, _code("bf16"), 0.1)
        ctx.kv_attention(cache.args, batch.args, args)
        assert o.isnan().all() and int(cache.fault) == api.KV_BAD_PAGE
        args.window = 2  # the last rows see good pages only
        args, _ = R.attention_args(ctx, cache, batch, q, o, _code("bf16"), 0.1, True, 2)
        ctx.kv_attention(cache.args, batch.args, args)
        assert not o[new[0] - 1].isnan().any() and not o[-1].isnan().any()


@pytest.mark.parametrize("new", [1, 2, 40])
@pytest.mark.parametrize("wrong", ["long", "rows", "fall", "negative"])
@pytest.mark.parametrize("bound", [150, 5000])
def test_bad_sequences(ctx, new, wrong, bound):
    """A sequence whose length or rows leave the bounds is left out and reported; its neighbours are computed."""
    from kokoro_hip import api
    lens = [100, 150, 80]
    cache, tables = _filled(ctx, "int8", 1, 64, lens, 4)
    batch = R.Batch([new] * 3, lens, tables, first=3, rows=3 * new + 3, max_len=bound, width=-(-bound // PAGE))
    start, length = batch.dev[0], batch.dev[1]
    if wrong == "long":
        length[1] = bound + 1
    elif wrong == "negative":
        length[1] = -1
    elif wrong == "rows":
        start[3] = batch.rows + 1  # the last one's rows
    else:
        start[0] = 1 << 30         # the first one's
    out = {"long": 1, "negative": 1, "rows": 2, "fall": 0}[wrong]
    q = torch.randn(batch.rows, 2, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    o = torch.full_like(q, 4.0)
    args, _ = R.attention_args(ctx, cache, batch, q, o, _code("f16"), 0.1)
    ctx.kv_attention(cache.args, batch.args, args)
    assert int(cache.fault) == api.KV_BAD_BATCH
    k, v = _kv(batch.rows, 1, 64, "f16", 1)
    cache.fault.zero_()
    ctx.kv_write(cache.args, batch.args, R.rows_of(_code("f16"), k, v))
    assert int(cache.fault) == api.KV_BAD_BATCH
    for b in range(3):
        rows = list(batch.of(b))
        if b == out:
            assert (o[rows] == 4.0).all()
            continue
        R.check_attention(o, q, cache, batch, 0.1, True, 0, "f16", only=[b])
        pos = lens[b] - new
        for part, x in (("k", k), ("v", v)):
            x, p = x[rows].float().cpu(), pos
            while len(x):
                take = min(len(x), PAGE - p % PAGE)
                cache.write(tables[b][p // PAGE], p % PAGE, x[:take], part)
                x, p = x[take:], p + take
    cache.same()  # the good ones' tokens are there, the other's as they were


def test_rows_without_their_tokens(ctx):
    """Rows that exceed their sequence's tokens cannot be written or read back; attention lets the first ones see nothing."""
    from kokoro_hip import api
    cache, tables = _filled(ctx, "int8", 1, 64, [10], 4)
    batch = R.Batch([12], [10], tables)
    k, v = _kv(12, 1, 64, "f16", 1)
    ctx.kv_write(cache.args, batch.args, R.rows_of(_code("f16"), k, v))
    assert int(cache.fault) == api.KV_BAD_BATCH and cache.same()
    cache.fault.zero_()
    before = k.clone()
    ctx.kv_read(cache.args, batch.args, R.rows_of(_code("f16"), k, v))
    assert int(cache.fault) == api.KV_BAD_BATCH and torch.equal(k, before)


def test_workspace_refusals(ctx):
    from kokoro_hip import api
    cache, tables = _filled(ctx, "int8", 1, 64, [2000], 4)
    batch = R.Batch([1], [2000], tables)
    q = torch.zeros(1, 2, 64, dtype=torch.float16, device="cuda")
    args, space = R.attention_args(ctx, cache, batch, q, torch.empty_like(q), _code("f16"), 0.1)
    assert args.workspace_bytes > 0
    for change in (dict(workspace_bytes=args.workspace_bytes - 1), dict(workspace=0), dict(workspace=space.data_ptr() + 4)):
        was = {k: getattr(args, k) for k in change}
        for k, x in change.items():
            setattr(args, k, x)
        with pytest.raises(api.KKError, match="workspace") as e:
            ctx.kv_attention(cache.args, batch.args, args)
        assert e.value.code == api.KK_ERR_INVALID
        for k, x in was.items():
            setattr(args, k, x)
    ctx.kv_attention(cache.args, batch.args, args)


# ------------------------------------------------------------------ together, as they are used


def _step(ctx, api, cache, batch, qkv, qr, kr, out, pos, w, heads, group, dim, attn, stream=0):
    hq = heads * group
    wide = qkv.stride(0)
    e = qkv.element_size()
    ctx.qk_norm_rope(api.NormRope(type=api.BF16, dim=dim, rows=qkv.shape[0], q_heads=hq, k_heads=heads, q=qkv.data_ptr(), q_row=wide,
                                  q_head=dim, k=qkv.data_ptr() + hq * dim * e, k_row=wide, k_head=dim, q_out=qr.data_ptr(),
                                  q_out_row=hq * dim, q_out_head=dim, k_out=kr.data_ptr(), k_out_row=heads * dim, k_out_head=dim,
                                  norm=1, eps=1e-6, q_weight=w[0].data_ptr(), k_weight=w[1].data_ptr(), pos=pos.data_ptr(),
                                  rot=dim, theta=1e4), stream)
    ctx.kv_write(cache.args, batch.args, api.KvRows(type=api.BF16, k=kr.data_ptr(), k_row=heads * dim, k_head=dim,
                                                    v=qkv.data_ptr() + (hq + heads) * dim * e, v_row=wide, v_head=dim), stream)
    ctx.kv_attention(cache.args, batch.args, attn, stream)


@pytest.mark.parametrize("cache_kind", ["int8", "e4m3"])
def test_decoding_loop(ctx, cache_kind):
    """Two prompts of different lengths, then tokens one by one over page borders: norms and rotation, the cache, attention.
    Attention is checked against f64 over what the cache holds, and the cache against the rotated keys."""
    from kokoro_hip import api
    heads, group, dim = 2, 4, 64
    hq = heads * group
    cache = R.Cache(cache_kind, heads, dim, 8)
    tables = R.deal([140, 140], 8, np.random.default_rng(1))
    g = torch.Generator().manual_seed(5)
    w = [(1 + 0.3 * torch.randn(dim, generator=g)).cuda() for _ in range(2)]
    have, new = [0, 0], [120, 61]
    for step in range(12):
        have = [h + n for h, n in zip(have, new)]
        batch = R.Batch(new, have, tables, max_len=140)
        qkv = torch.randn(batch.rows, (hq + 2 * heads) * dim, generator=g).bfloat16().cuda()
        pos = torch.cat([torch.arange(h - n, h) for h, n in zip(have, new)]).int().cuda()
        qr, kr = (torch.empty(batch.rows, h, dim, dtype=torch.bfloat16, device="cuda") for h in (hq, heads))
        out = torch.empty_like(qr)
        attn, space = R.attention_args(ctx, cache, batch, qr, out, api.BF16, 0.3)
        _step(ctx, api, cache, batch, qkv, qr, kr, out, pos, w, heads, group, dim, attn)
        v = qkv[:, (hq + heads) * dim:].unflatten(1, (heads, dim))
        for part, x in (("k", kr.float().cpu()), ("v", v.float().cpu())):
            for b in range(2):
                x_b, p = x[list(batch.of(b))], have[b] - new[b]
                while len(x_b):
                    take = min(len(x_b), PAGE - p % PAGE)
                    cache.write(tables[b][p // PAGE], p % PAGE, x_b[:take], part)
                    x_b, p = x_b[take:], p + take
        cache.same()
        R.check_attention(out, qr, cache, batch, 0.3, True, 0, "bf16")
        new = [1, 1]


@pytest.mark.parametrize("parts", [False, True])
def test_graph_of_a_decoding_step(ctx, parts):
    """A step captured into a graph and replayed with new rows, lengths and tables in the same buffers, with eager work and
    synchronizations between; each replay against the same calls made eagerly on a copy of the cache."""
    from kokoro_hip import api
    heads, group, dim, n = 2, 4, 64, 3
    hq = heads * group
    top = 2000 if parts else 400
    cache, tables = _filled(ctx, "int8", heads, dim, [top] * n, 2)
    twin, _ = _filled(ctx, "int8", heads, dim, [top] * n, 2)
    assert all(torch.equal(cache.dev[k], twin.dev[k]) for k in ("k", "v"))
    batch = R.Batch([1] * n, [1] * n, tables, max_len=top)
    g = torch.Generator().manual_seed(5)
    w = [(1 + 0.3 * torch.randn(dim, generator=g)).cuda() for _ in range(2)]
    qkv = torch.zeros(n, (hq + 2 * heads) * dim, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(n, dtype=torch.int32, device="cuda")
    qr, kr = (torch.empty(n, h, dim, dtype=torch.bfloat16, device="cuda") for h in (hq, heads))
    out = torch.empty_like(qr)
    attn, space = R.attention_args(ctx, cache, batch, qr, out, api.BF16, 0.3)
    assert bool(attn.workspace_bytes) == parts
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(ctx, api, cache, batch, qkv, qr, kr, out, pos, w, heads, group, dim, attn, torch.cuda.current_stream().cuda_stream)
    out2 = torch.empty_like(out)
    attn2, space2 = R.attention_args(ctx, twin, batch, qr, out2, api.BF16, 0.3)
    for replay in range(5):
        lens = [1 + (replay * 97 + 131 * b) % top for b in range(n)]
        batch.dev[1].copy_(torch.tensor(lens, dtype=torch.int32))
        pos.copy_(torch.tensor(lens, dtype=torch.int32) - 1)
        qkv.copy_(torch.randn(qkv.shape, generator=g).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        _step(ctx, api, twin, batch, qkv, qr, kr, out2, pos, w, heads, group, dim, attn2)
        torch.cuda.synchronize()
        assert torch.equal(got, out2)
        assert all(torch.equal(cache.dev[k].view(torch.uint8), twin.dev[k].view(torch.uint8)) for k in cache.dev)


def test_streams(ctx):
    """Work on a side stream that waits for its inputs, and calls that overlap on two streams with a workspace each."""
    from kokoro_hip import api
    cache, tables = _filled(ctx, "int8", 2, 128, [3000, 2500], 3)
    batch = R.Batch([1, 1], [3000, 2500], tables)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(1)).half().cuda()
    outs = [torch.empty_like(q) for _ in range(2)]
    calls = [R.attention_args(ctx, cache, batch, q, o, _code("f16"), 0.1) for o in outs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for s, (args, _) in zip(streams, calls):
            ctx.kv_attention(cache.args, batch.args, args, s.cuda_stream)
    torch.cuda.synchronize()
    R.check_attention(outs[0], q, cache, batch, 0.1, True, 0, "f16")
    assert torch.equal(outs[0], outs[1])
    assert api.lib() is not None


def test_nothing_to_do(ctx):
    cache, tables = _filled(ctx, "int8", 1, 64, [10], 4)
    q = torch.zeros(1, 1, 64, dtype=torch.float16, device="cuda")
    for batch in (R.Batch([], [], []), R.Batch([0], [10], tables), R.Batch([0, 0], [10, 0], tables * 2, rows=1, max_new=1)):
        ctx.kv_write(cache.args, batch.args, R.rows_of(_code("f16"), q, q))
        ctx.kv_read(cache.args, batch.args, R.rows_of(_code("f16"), q, q))
        args, _ = R.attention_args(ctx, cache, batch, q, torch.zeros_like(q), _code("f16"), 0.1)
        ctx.kv_attention(cache.args, batch.args, args)
    cache.same()
    assert not q.any() and int(cache.fault) == 0


@pytest.mark.parametrize("new", [1, 40])
def test_no_tokens_and_no_table(ctx, new):
    """max_len 0 needs no page table, whatever its width says: rows that see nothing give zeros."""
    cache, _ = _filled(ctx, "int8", 1, 64, [10], 4)
    batch = R.Batch([new], [0], [[]], max_len=0, width=4)
    batch.args.table = None
    q = torch.ones(new, 1, 64, dtype=torch.float16, device="cuda")
    out = torch.ones_like(q)
    args, _ = R.attention_args(ctx, cache, batch, q, out, _code("f16"), 0.1)
    ctx.kv_attention(cache.args, batch.args, args)
    assert not out.any() and int(cache.fault) == 0


@pytest.mark.parametrize("cache_kind, group", [("int8", 1), ("e4m3", 12)])
def test_far_addresses(ctx, cache_kind, group):
    """Pages and rows that lie more than 2^32 bytes and 2^31 values into their arrays give, bit for bit, what near ones give."""
    from kokoro_hip import api
    heads, dim, n, far_pages = 4, 256, 130, (1 << 16) + 9
    g = torch.Generator().manual_seed(group)
    k, v = (torch.randn(n, heads, dim, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    q = torch.randn(3, heads * group, dim, generator=g).to(torch.bfloat16).cuda()
    row = (1 << 30) + 8  # rows 1 and 2 are 2^30 and 2^31 values behind row 0
    width = (heads * group + 2 * heads) * dim

    def run(pages, numbers, row):
        rows = torch.empty(2 * row + 2 * width, dtype=torch.bfloat16, device="cuda")
        kind = torch.int8 if cache_kind == "int8" else torch.uint8
        dev = {"k": torch.empty(pages, heads, PAGE, dim, dtype=kind, device="cuda"), "v": torch.empty(pages, heads, dim, PAGE, dtype=kind, device="cuda"),
               "k_scale": torch.empty(pages, heads, device="cuda"), "v_scale": torch.empty(pages, heads, device="cuda")}
        for part in ("k", "v"):
            dev[part][numbers] = 0
        fault = torch.zeros(1, dtype=torch.int32, device="cuda")
        cache = api.KvCache(type=api.KV_INT8 if cache_kind == "int8" else api.KV_E4M3, heads=heads, dim=dim, pages=pages,
                            fault=fault.data_ptr(), **{x: y.data_ptr() for x, y in dev.items()})
        view = lambda at, h: rows[at:].as_strided((3, h, dim), (row, dim, 1))  # noqa: E731
        qr, kr, vr, out = view(0, heads * group), view(heads * group * dim, heads), view((heads * group + heads) * dim, heads), view(width, heads * group)
        qr.copy_(q), kr.copy_(k[-3:]), vr.copy_(v[-3:])
        first, last, whole = R.Batch([n - 3], [n - 3], [numbers]), R.Batch([3], [n], [numbers]), R.Batch([n], [n], [numbers])
        ctx.kv_write(cache, first.args, R.rows_of(_code("bf16"), k, v))
        ctx.kv_write(cache, last.args, R.rows_of(_code("bf16"), kr, vr))
        back = torch.empty(2, n, heads, dim, dtype=torch.bfloat16, device="cuda")
        ctx.kv_read(cache, whole.args, R.rows_of(_code("bf16"), back[0], back[1]))
        holder = type("", (), {"args": cache})
        args, space = R.attention_args(ctx, holder, last, qr, out, _code("bf16"), 0.07)
        ctx.kv_attention(cache, last.args, args)
        kr.zero_(), vr.zero_()
        ctx.kv_read(cache, last.args, R.rows_of(_code("bf16"), kr, vr))
        turned = out.clone()
        pos = torch.arange(3, dtype=torch.int32, device="cuda")
        rope = api.NormRope(type=_code("bf16"), dim=dim, rows=3, q_heads=heads * group, k_heads=0, q=qr.data_ptr(), q_row=row, q_head=dim,
                            q_out=out.data_ptr(), q_out_row=row, q_out_head=dim, norm=1, eps=1e-6, pos=pos.data_ptr(), rot=dim, theta=1e4)
        ctx.qk_norm_rope(rope)
        got = [back.cpu(), turned.cpu(), out.clone().cpu(), kr.clone().cpu(), vr.clone().cpu()] + [dev[x][numbers].cpu() for x in dev]
        assert int(fault) == 0
        return got

    near = run(5, [3, 0, 4], 2 * width)
    far = run(far_pages, [far_pages - 1, 1, far_pages - 2], row)
    for a, b in zip(near, far):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert near[1].isfinite().all() and near[1].float().abs().amax() > 0
