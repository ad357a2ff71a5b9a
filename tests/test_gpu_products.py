"""The products of ragged rows on the GPU, through the library's entry points, against their definitions in 64 bits
(tests/product_ref.py): routing bit for bit but for the weights, products within a derived bound, adapters in any order of rows,
bad device arrays, graphs, streams, and a whole layer of the operators together."""
import numpy as np
import pytest
import torch

import kv_ref as K
import product_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from kokoro_hip import api
    torch.cuda.init()
    c = api.Context(0)
    yield c
    c.close()


def _randn(shape, seed, kind="bf16", size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * size).to(R.TYPES[kind])


# ------------------------------------------------------------------ routing


def _same_route(got, want):
    for k in ("expert", "start", "place"):
        assert torch.equal(got[k].cpu().long(), want[k].long()), k
    w = want["weight"]
    # exp: the argument's rounding (2^-24 of a difference below 2^8) and the function's, a sum of at most 1,024, a division, a product
    assert ((got["weight"].cpu().double() - w).abs() <= 2.0 ** -14 * w.abs() + 2.0 ** -140).all()


@pytest.mark.parametrize("rows, experts, top", [
    (1, 1, 1), (1, 64, 8), (3, 8, 2), (7, 16, 16), (64, 17, 5), (65, 100, 6), (130, 128, 8), (16, 1024, 32), (17, 1000, 9), (40, 257, 20),
    (300, 512, 32), (5000, 60, 4), (20000, 8, 1)])
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_route(ctx, rows, experts, top, kind):
    """Random logits (in 16 bits with ties), every thirtieth row padding, some experts masked in some rows."""
    x = _randn((rows, experts), rows + experts, "f32", 2.0)
    x[::7, :: max(2, experts // 3)] = -torch.inf
    x[29::30] = -torch.inf
    x = x.to(R.TYPES[kind])
    for score, renorm, scale in (("softmax", True, 1.0), ("softmax", False, 2.5), ("sigmoid", True, 0.5), ("sigmoid", False, 1.0)):
        got = R.route(ctx, x, top, score, renorm, scale)
        _same_route(got, R.route_ref(x, top, score, renorm, scale))


@pytest.mark.parametrize("experts", [8, 100, 300])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_special_logits(ctx, experts, score):
    """Rows that are all equal, all masked, NaN, infinite, of the type's lowest value, zeros of both signs; fewer experts than `top`;
    rows that lie apart at odd distances."""
    wide = torch.full((40, experts + 3), float("nan"), device="cuda")
    x = wide[:, 1:experts + 1]
    x[:] = _randn((40, experts), 5, "f32")
    low, high = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max
    x[0], x[1], x[2] = 0.0, -torch.inf, torch.nan
    x[3, 2:5] = torch.inf
    x[4] = low
    x[5, 1:] = low
    x[6, ::2], x[6, 1::2] = 0.0, -0.0
    x[7, 3:] = -torch.inf
    x[8, 1], x[8, 4], x[8, 6] = high, torch.inf, torch.nan
    x[9] *= 1e-42
    x[10] = torch.inf
    for renorm in (True, False):
        got = R.route(ctx, x, 6, score, renorm)
        _same_route(got, R.route_ref(x, 6, score, renorm, 1.0))
    assert (got["expert"][1:3] == -1).all() and (got["expert"][7, 3:] == -1).all()


def test_route_nothing(ctx):
    got = R.route(ctx, torch.empty(0, 8, device="cuda"), 2)
    assert not got["start"].any()


# ------------------------------------------------------------------ products by expert


def _groups(sizes):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32, device="cuda")


SIZES = {
    "few": [0, 1, 16, 3, 0, 17, 15, 40, 0],
    "one": [1],
    "some": [64, 0, 65, 1, 130, 31],
    "many": [128, 300, 0, 127, 129],
    "most": [700, 513, 1],
    "largest": [1200, 0, 900, 3],
    "empty": [0, 0, 0],
}


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("k, n", [(8, 1), (24, 33), (64, 64), (136, 100), (1032, 130), (2048, 256)])
def test_expert_product(ctx, kind, sizes, k, n):
    """Every kernel, with groups and sizes that no tile divides; gates and biases; gathered rows in, scattered rows out."""
    start = _groups(SIZES[sizes])
    total = int(start[-1])
    entries = total + 5  # some behind the last group
    groups = len(start) - 1
    perm = torch.randperm(entries * 3, generator=torch.Generator().manual_seed(k)).int().cuda()
    for i, gate in enumerate(("none", "silu", "gelu")):
        wide = n * (1 if gate == "none" else 2)
        w = _randn((groups, wide, k), i + n, kind, k ** -0.5 * 1.5)
        bias = _randn((groups, wide), i, "f32", 0.3) if i != 1 else None
        # gathered: three places a row
        x = _randn((entries, k), i + 3, kind)
        y = torch.full((entries, n), 7.0, dtype=R.TYPES[kind], device="cuda")
        want, bound, written = R.expert_ref(x, w, start, y, gate, bias, x_place=perm[:entries], x_div=3)
        ctx.expert_product(R.expert_args(x, w, start, y, entries, gate, bias, x_place=perm[:entries], x_div=3))
        R.close(y[written], want[written], bound[written])
        assert (y[~written] == 7.0).all() and int(written.sum()) == total
        # scattered, to rows of an odd stride
        room = torch.full((entries * 3, n + 3), 7.0, dtype=R.TYPES[kind], device="cuda")
        y = room[:, 1:n + 1]
        want, bound, written = R.expert_ref(x, w, start, y, gate, bias, y_place=perm[:entries])
        ctx.expert_product(R.expert_args(x, w, start, y, entries, gate, bias, y_place=perm[:entries]))
        R.close(y[written], want[written], bound[written])
        assert (y[~written] == 7.0).all() and (room[:, 0] == 7.0).all() and (room[:, n + 1:] == 7.0).all()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("sizes, k, n", [("many", 72, 4500), ("many", 136, 4613), ("most", 64, 3333), ("largest", 104, 5301), ("largest", 1032, 5312), ("largest", 72, 10611)])
def test_expert_product_larger_tiles(ctx, kind, sizes, k, n):
    """The same where there are enough outputs for tiles of 128 and 256 rows."""
    test_expert_product(ctx, kind, sizes, k, n)


@pytest.mark.parametrize("sizes, k, n", [([30, 0, 1, 64, 65] * 20, 72, 1500), ([300, 128, 0, 129] * 5, 200, 5000), ([1900, 0, 700], 64, 16400)])
def test_expert_product_tile_after_tile(ctx, sizes, k, n):
    """More tiles than the device holds at once, so that blocks go on to others, with places in and out."""
    start = _groups(sizes)
    total = int(start[-1])
    groups = len(sizes)
    w = _randn((groups, n, k), 1, "bf16", k ** -0.5)
    x = _randn((total // 2 + 1, k), 2)
    g = torch.Generator().manual_seed(k)
    x_place, y_place = torch.randint(0, 2 * len(x), (total,), generator=g).int().cuda(), torch.randperm(total, generator=g).int().cuda()
    y = torch.full((total, n), 7.0, dtype=torch.bfloat16, device="cuda")
    want, bound, written = R.expert_ref(x, w, start, y, x_place=x_place, x_div=2, y_place=y_place)
    ctx.expert_product(R.expert_args(x, w, start, y, x_place=x_place, x_div=2, y_place=y_place))
    assert written.all()
    R.close(y, want, bound)


def test_expert_product_many_groups(ctx):
    """1,024 groups, most of them empty, the first and the last not."""
    g = torch.Generator().manual_seed(4)
    sizes = (torch.randint(0, 5, (1024,), generator=g) * (torch.rand(1024, generator=g) < 0.2)).tolist()
    sizes[0], sizes[1023], sizes[500] = 3, 2, 300
    start = _groups(sizes)
    x, w = _randn((int(start[-1]), 64), 1), _randn((1024, 24, 64), 2)
    y = torch.zeros(len(x), 24, dtype=torch.bfloat16, device="cuda")
    want, bound, written = R.expert_ref(x, w, start, y)
    ctx.expert_product(R.expert_args(x, w, start, y))
    assert written.all()
    R.close(y, want, bound)


def test_expert_product_strides(ctx):
    """Rows and matrices that lie apart; infinities behind each row's end are not read into it."""
    k, n, start = 72, 40, _groups([20, 200, 3])
    xs = torch.full((223, k + 24), torch.inf, dtype=torch.bfloat16, device="cuda")
    ws = torch.full((3, n + 2, k + 8), torch.nan, dtype=torch.bfloat16, device="cuda")
    x, w = xs[:, 8:8 + k], ws[:, :n, :k]
    x[:], w[:] = _randn((223, k), 1), _randn((3, n, k), 2)
    y = torch.zeros(223, n, dtype=torch.bfloat16, device="cuda")
    want, bound, _ = R.expert_ref(x, w, start, y)
    ctx.expert_product(R.expert_args(x, w, start, y))
    R.close(y, want, bound)


@pytest.mark.parametrize("n", [6, 600])
def test_expert_product_bad_arrays(ctx, n):
    """A group that leaves the entries or ends before it begins is left out, an entry with a bad place too; the others are whole."""
    from kokoro_hip import api
    x, w = _randn((4 * n, 64), 1), _randn((4, 48, 64), 2)
    for start, bad in (([0, n, n - 5, 2 * n, 3 * n], [1]), ([-1, n, 2 * n, 3 * n, 4 * n], [0]), ([0, n, 2 * n, 3 * n, 4 * n + 1], [3]),
                       ([0, n, 2 * n, 3 * n, 2 ** 31 - 1], [3]), ([0, n, -(2 ** 31), 3 * n, 4 * n], [1, 2])):
        y = torch.full((4 * n, 48), 7.0, dtype=torch.bfloat16, device="cuda")
        fault = torch.zeros(1, dtype=torch.int32, device="cuda")
        args = R.expert_args(x, w, torch.tensor(start, dtype=torch.int32, device="cuda"), y, fault=fault)
        ctx.expert_product(args)
        assert int(fault) == api.KK_PRODUCT_BAD_START
        for g in range(4):
            if g in bad or (start[g + 1] < start[g]):
                continue
            one = slice(start[g], start[g + 1])
            if start == [0, n, n - 5, 2 * n, 3 * n] and g in (0, 2):
                one = slice(start[g], n - 5) if g == 0 else slice(n, start[g + 1])  # they overlap
            want, bound = R.product(x[one], w[g])
            R.close(y[one], want, bound)
    # groups that overlap, more rows of them than entries: nothing outside y is written
    room = torch.full((4 * n + 2, 48), 7.0, dtype=torch.bfloat16, device="cuda")
    wild = torch.tensor([0, 4 * n] * 300, dtype=torch.int32, device="cuda")
    fault = torch.zeros(1, dtype=torch.int32, device="cuda")
    ctx.expert_product(R.expert_args(x, _randn((599, 48, 64), 2), wild, room[1:-1], fault=fault))
    assert int(fault) == api.KK_PRODUCT_BAD_START and (room[0] == 7.0).all() and (room[-1] == 7.0).all()
    start = _groups([n, n, n, n])
    place = torch.arange(4 * n, dtype=torch.int32, device="cuda")
    bad = torch.zeros(4 * n, dtype=torch.bool, device="cuda")
    for i, v in ((0, -1), (n + 1, 4 * n), (2 * n, 2 ** 31 - 1), (4 * n - 1, -(2 ** 31))):
        place[i], bad[i] = v, True
    want, bound, _ = R.expert_ref(x, w, start, torch.zeros(4 * n, 48, device="cuda"))
    for way in ("x_place", "y_place"):
        y = torch.full((4 * n, 48), 7.0, dtype=torch.bfloat16, device="cuda")
        fault = torch.zeros(1, dtype=torch.int32, device="cuda")
        ctx.expert_product(R.expert_args(x, w, start, y, fault=fault, **{way: place}))
        assert int(fault) == api.KK_PRODUCT_BAD_PLACE
        R.close(y[~bad], want[~bad], bound[~bad])
        assert (y[bad] == 7.0).all()


# ------------------------------------------------------------------ the join


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows, top, n", [(1, 1, 1), (3, 8, 64), (33, 2, 100), (5, 32, 2048), (700, 9, 72), (2, 3, 1001)])
def test_join(ctx, kind, rows, top, n):
    y = _randn((rows * top, n), 1, kind)
    base = _randn((rows, n), 2, kind)
    g = torch.Generator(device="cuda").manual_seed(3)
    expert = torch.randint(-1, 3, (rows, top), generator=g, device="cuda", dtype=torch.int32)
    weight = torch.rand(rows, top, generator=g, device="cuda")
    y[(expert < 0).view(-1)] = torch.nan  # not read
    room = torch.zeros(rows, n + 1, dtype=y.dtype, device="cuda")
    for out, b in ((torch.empty_like(base), base), (torch.empty_like(base), None), (room[:, 1:], base), (base.clone(), "in place")):
        b = out if isinstance(b, str) else b
        want, bound = R.join_ref(torch.nan_to_num(y), expert, weight, None if b is None else b.clone())
        ctx.expert_join(R.join_args(y, expert, weight, out, b))
        R.close(out, want, bound)


# ------------------------------------------------------------------ adapters


def _adapters(n, rank, k, outs, kind):
    g = torch.Generator(device="cuda").manual_seed(rank)
    a, b = _randn((n, rank, k), 4, kind, k ** -0.5), _randn((n, outs, rank), 5, kind, rank ** -0.5)
    return a, b, torch.rand(n, generator=g, device="cuda") * 3 - 1


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 5, 17, 64, 129, 600])
@pytest.mark.parametrize("k, n, rank", [(64, 40, 8), (264, 130, 24), (1032, 178, 64), (512, 4, 128), (80, 1027, 256)])
def test_adapter_product(ctx, kind, rows, k, n, rank):
    """Rows of requests one after the other, each row with another adapter, some without, all without; both output types."""
    x, w = _randn((rows, k), 1, kind), _randn((n, k), 2, kind, k ** -0.5)
    many = 7
    a, b, scale = _adapters(many, rank, k, n, kind)
    bias = _randn((n,), 3, "f32")
    g = torch.Generator(device="cuda").manual_seed(rows)
    mixed = torch.randint(-1, many, (rows,), generator=g, device="cuda", dtype=torch.int32)
    for ids, out, use in ((torch.sort(mixed).values, kind, None), (mixed, "f32", bias), (torch.full_like(mixed, -3), kind, bias),
                          (torch.full_like(mixed, many - 1), kind, None)):
        y = torch.full((rows, n), 7.0, dtype=R.TYPES[out], device="cuda")
        want, bound = R.adapter_ref(x, w, use, a, b, scale, ids)
        R.adapter_run(ctx, R.adapter_args(x, w, y, use, a, b, scale, ids))
        R.close(y, want, bound)
    room = torch.full((rows, n + 3), 7.0, dtype=R.TYPES[kind], device="cuda")
    R.adapter_run(ctx, R.adapter_args(x, w, room[:, 1:n + 1], bias))
    want, bound = R.adapter_ref(x, w, bias)
    R.close(room[:, 1:n + 1], want, bound)
    assert (room[:, 0] == 7.0).all() and (room[:, n + 1:] == 7.0).all()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows, n, k, rank", [(6000, 2000, 200, 40), (3000, 4100, 64, 64), (4200, 4096, 136, 8), (8300, 2111, 128, 256)])
def test_adapter_product_many_rows(ctx, kind, rows, n, k, rank):
    """Enough tiles for the adapters to go through the main product, in every way that a tile's rows can share them; rows behind the
    last whole round of large tiles; a bias; both output types."""
    many = 11
    x, w = _randn((rows, k), 1, kind), _randn((n, k), 2, kind, k ** -0.5)
    a, b, scale = _adapters(many, rank, k, n, kind)
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.sort(torch.randint(-1, many, (rows,), generator=g, device="cuda", dtype=torch.int32)).values
    ids[1000:1500] = torch.randint(-1, many, (500,), generator=g, device="cuda", dtype=torch.int32)
    ids[1500:2100] = -1
    for out, bias in ((kind, None), ("f32", _randn((n,), 3, "f32"))):
        y = torch.empty(rows, n, dtype=R.TYPES[out], device="cuda")
        want, bound = R.adapter_ref(x, w, bias, a, b, scale, ids)
        R.adapter_run(ctx, R.adapter_args(x, w, y, bias, a, b, scale, ids))
        R.close(y, want, bound)
    y = torch.empty(rows, n, dtype=R.TYPES[kind], device="cuda")
    want, bound = R.adapter_ref(x, w)
    R.adapter_run(ctx, R.adapter_args(x, w, y))
    R.close(y, want, bound)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows, n", [(40, 100), (300, 700), (6000, 2000)])
def test_adapter_product_keeps_requests_apart(ctx, kind, rows, n):
    """An adapter of infinities and NaN reaches its own rows and no others, wherever they lie."""
    k, rank, many = 72, 16, 5
    x, w = _randn((rows, k), 1, kind), _randn((n, k), 2, kind, k ** -0.5)
    a, b, scale = _adapters(many, rank, k, n, kind)
    g = torch.Generator(device="cuda").manual_seed(rows)
    ids = torch.randint(-1, many, (rows,), generator=g, device="cuda", dtype=torch.int32)
    ids[rows // 2:] = torch.sort(ids[rows // 2:]).values
    want, bound = R.adapter_ref(x, w, None, a, b, scale, ids)
    good = (ids != 2) & (ids != 3)
    b[2, ::3], b[2, 1::3], a[3, 1] = torch.nan, torch.inf, -torch.inf
    y = torch.empty(rows, n, dtype=R.TYPES[kind], device="cuda")
    R.adapter_run(ctx, R.adapter_args(x, w, y, None, a, b, scale, ids))
    R.close(y[good], want[good], bound[good])
    assert not torch.isfinite(y[ids == 2][:, :2]).any() and not torch.isfinite(y[ids == 3]).any()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows, n, rank", [(40, 100, 24), (6000, 2000, 24), (8300, 2111, 8), (4200, 4096, 40)])
def test_adapter_product_keeps_f32(ctx, kind, rows, n, rank):
    """Where y is f32 nothing of a x is lost: whole numbers below 2^24, whose sums in any order are exact, come out as they are."""
    k, many = 64, 7
    g = torch.Generator(device="cuda").manual_seed(rank)

    def whole(shape, most):
        return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(R.TYPES[kind])
    x, w = whole((rows, k), 127), whole((n, k), 1)
    a, b, scale = whole((many, rank, k), 63), whole((many, n, rank), 1), torch.tensor([1.0, -1.0, 0.5, 2.0, 1.0, 0.0, -0.25], device="cuda")
    ids = torch.sort(torch.randint(-1, many, (rows,), generator=g, device="cuda", dtype=torch.int32)).values
    want, _ = R.adapter_ref(x, w, None, a, b, scale, ids)
    size = max((x.float() @ a[i].float().t()).abs().sum(1).max().item() for i in range(many))
    assert 2 * size + 127 * k < 2 ** 22  # in quarters
    y = torch.empty(rows, n, device="cuda")
    R.adapter_run(ctx, R.adapter_args(x, w, y, None, a, b, scale, ids))
    assert torch.equal(y.double(), want)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows, n", [(40, 100), (6000, 2000)])
def test_adapter_product_infinite_rows(ctx, kind, rows, n):
    """An infinity in a row of x stays one where every term has its sign, whether the adapter's share goes through 16-bit parts or not,
    and is NaN where they differ; the other rows are as without it."""
    k, rank = 72, 16
    x, w = _randn((rows, k), 1, kind), _randn((n, k), 2, kind).abs() + 0.5
    a, b, scale = _randn((2, rank, k), 3, kind).abs() + 0.5, _randn((2, n, rank), 4, kind).abs() + 0.5, torch.ones(2, device="cuda")
    ids = (torch.arange(rows, device="cuda") % 3 - 1).int()
    ids[rows // 2:] = 1
    want, bound = R.adapter_ref(x, w, None, a, b, scale, ids)
    up, down, both = [torch.tensor(i, device="cuda") for i in ((1, rows - 3), (5, rows - 4), (7, rows - 5))]
    x[up, 3], x[down, 70], x[both, 5], x[both, 6] = torch.inf, -torch.inf, torch.inf, -torch.inf
    good = torch.ones(rows, dtype=torch.bool, device="cuda")
    good[torch.cat([up, down, both])] = False
    for out in (kind, "f32"):
        y = torch.empty(rows, n, dtype=R.TYPES[out], device="cuda")
        R.adapter_run(ctx, R.adapter_args(x, w, y, None, a, b, scale, ids))
        R.close(y[good], want[good], bound[good])
        assert (y[up] == torch.inf).all() and (y[down] == -torch.inf).all() and torch.isnan(y[both]).all()


@pytest.mark.parametrize("rows", [3, 300, 6000])
def test_adapter_product_sizes_out_of_f16(ctx, rows):
    """a x beyond f16's range, with b small: neither overflows on the way."""
    k, n, rank = 512, 1000, 16
    x, w = _randn((rows, k), 1, "f16", 8.0), _randn((n, k), 2, "f16", 0.01)
    a, b = _randn((2, rank, k), 4, "f16", 400.0), _randn((2, n, rank), 5, "f16", 1e-5)
    scale = torch.tensor([1.0, 30.0], device="cuda")
    ids = (torch.arange(rows, device="cuda") % 3 - 1).int()
    y = torch.empty(rows, n, dtype=torch.float16, device="cuda")
    want, bound = R.adapter_ref(x, w, None, a, b, scale, ids)
    R.adapter_run(ctx, R.adapter_args(x, w, y, None, a, b, scale, ids))
    R.close(y, want, bound)


@pytest.mark.parametrize("rows", [5, 300, 6000])
def test_adapter_product_bad_adapters(ctx, rows):
    from kokoro_hip import api
    k, n, rank = 64, 1000, 8
    x, w = _randn((rows, k), 1), _randn((n, k), 2)
    a, b, scale = _adapters(3, rank, k, n, "bf16")
    ids = (torch.arange(rows, device="cuda") % 3).int()
    ids[1], ids[rows - 1] = 3, 2 ** 31 - 1
    y = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    fault = torch.zeros(1, dtype=torch.int32, device="cuda")
    want, bound = R.adapter_ref(x, w, None, a, b, scale, ids)
    R.adapter_run(ctx, R.adapter_args(x, w, y, None, a, b, scale, ids, fault))
    assert int(fault) == api.KK_PRODUCT_BAD_ADAPTER
    R.close(y, want, bound)


# ------------------------------------------------------------------ together


class Layer:
    """A layer of a language model with the operators, cache and all, as a program runs it: projections with an adapter for each
    request, norms and rotation, attention over the cache, experts; buffers and descriptors made once."""

    def __init__(self, ctx, new, cap=200, seed=0):
        from kokoro_hip import api
        self.ctx, self.api, self.new = ctx, api, new
        self.d, self.hq, self.hk, self.dim, self.e, self.top, self.f, self.rank = 256, 4, 2, 64, 12, 3, 136, 16
        rows = self.rows = sum(new)
        d, qkv = self.d, (self.hq + 2 * self.hk) * self.dim

        def mat(*shape):
            nonlocal seed
            seed += 1
            return _randn(shape, 1000 + seed, "bf16", shape[-1] ** -0.5)

        self.w_qkv, self.w_out, self.w_route = mat(qkv, d), mat(d, self.hq * self.dim), mat(self.e, d)
        self.a1, self.b1, self.a2, self.b2 = mat(3, self.rank, d), mat(3, qkv, self.rank), mat(3, self.rank, d), mat(3, d, self.rank)
        self.scale = torch.tensor([0.5, 1.0, 2.0], device="cuda")
        self.w1, self.w2 = mat(self.e, 2 * self.f, d), mat(self.e, d, self.f)
        self.adapter = torch.tensor([b % 4 - 1 for b, n in enumerate(new) for _ in range(n)], dtype=torch.int32, device="cuda")
        self.pos = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.x = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
        like = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
        self.qkv, self.q, self.k = like(rows, qkv), like(rows, self.hq, self.dim), like(rows, self.hk, self.dim)
        self.att, self.mid, self.logits = like(rows, self.hq * self.dim), like(rows, d), like(rows, self.e, t=torch.float32)
        self.h, self.y, self.out = like(rows * self.top, self.f), like(rows * self.top, d), like(rows, d)
        self.route = {"expert": like(rows, self.top, t=torch.int32), "weight": like(rows, self.top, t=torch.float32),
                      "start": like(self.e + 1, t=torch.int32), "place": like(rows * self.top, t=torch.int32)}
        pages = -(-cap // K.PAGE)
        self.cache = K.Cache("int8", self.hk, self.dim, pages * len(new) + 1)
        self.tables = [list(range(b * pages, (b + 1) * pages)) for b in range(len(new))]
        self.len = torch.zeros(len(new), dtype=torch.int32, device="cuda")
        self.table = torch.tensor(self.tables, dtype=torch.int32, device="cuda")
        self.row_start = _groups(new)
        self.batch = api.KvBatch(n=len(new), rows=rows, max_new=max(new), max_len=cap, row_start=R.ptr(self.row_start), len=R.ptr(self.len),
                                 table=R.ptr(self.table), table_width=pages, table_stride=pages)
        self.keep = []

        def adapted(x, w, y, a=None, b=None):
            r = R.adapter_args(x, w, y, None, a, b, self.scale, self.adapter)
            ws = R.space(ctx.adapter_product_workspace(r))
            r.workspace, r.workspace_bytes = R.ptr(ws), ws.numel() * 4
            self.keep.append(ws)
            return r

        self.p_qkv, self.p_out = adapted(self.x, self.w_qkv, self.qkv, self.a1, self.b1), adapted(self.att, self.w_out, self.mid, self.a2, self.b2)
        self.p_route = adapted(self.mid, self.w_route, self.logits)
        e, hq, hk, dim = 2, self.hq, self.hk, self.dim
        self.rope = api.NormRope(type=api.BF16, dim=dim, rows=rows, q_heads=hq, k_heads=hk, q=R.ptr(self.qkv), q_row=qkv, q_head=dim,
                                 k=R.ptr(self.qkv) + hq * dim * e, k_row=qkv, k_head=dim, q_out=R.ptr(self.q), q_out_row=hq * dim, q_out_head=dim,
                                 k_out=R.ptr(self.k), k_out_row=hk * dim, k_out_head=dim, norm=1, eps=1e-6, pos=R.ptr(self.pos), rot=dim, theta=1e4)
        self.kv = api.KvRows(type=api.BF16, k=R.ptr(self.k), k_row=hk * dim, k_head=dim, v=R.ptr(self.qkv) + (hq + hk) * dim * e, v_row=qkv, v_head=dim)
        self.attn = api.KvAttention(type=api.BF16, heads=hq, q=R.ptr(self.q), q_row=hq * dim, q_head=dim, out=R.ptr(self.att), out_row=hq * dim,
                                    out_head=dim, scale=dim ** -0.5, causal=1)
        ws = R.space(ctx.kv_attention_workspace(self.cache.args, self.batch, self.attn))
        self.attn.workspace, self.attn.workspace_bytes = R.ptr(ws), ws.numel() * 4
        self.router = api.ExpertRoute(type=api.F32, rows=rows, experts=self.e, top=self.top, logits=R.ptr(self.logits), logits_row=self.e, renorm=1,
                                      scale=1.0, **{k: R.ptr(v) for k, v in self.route.items()})
        ws2 = R.space(ctx.expert_route_workspace(self.router))
        self.router.workspace, self.router.workspace_bytes = R.ptr(ws2), ws2.numel() * 4
        self.keep += [ws, ws2]
        self.up = R.expert_args(self.mid, self.w1, self.route["start"], self.h, rows * self.top, "silu", x_place=self.route["place"], x_div=self.top)
        self.down = R.expert_args(self.h, self.w2, self.route["start"], self.y, rows * self.top, y_place=self.route["place"])
        self.join = R.join_args(self.y, self.route["expert"], self.route["weight"], self.out, self.mid)

    def step(self, stream):
        c = self.ctx
        c.adapter_product(self.p_qkv, stream)
        c.qk_norm_rope(self.rope, stream)
        c.kv_write(self.cache.args, self.batch, self.kv, stream)
        c.kv_attention(self.cache.args, self.batch, self.attn, stream)
        c.adapter_product(self.p_out, stream)
        c.adapter_product(self.p_route, stream)
        c.expert_route(self.router, stream)
        c.expert_product(self.up, stream)
        c.expert_product(self.down, stream)
        c.expert_join(self.join, stream)

    def set(self, x, have):
        """The next rows, behind `have` tokens of each sequence."""
        self.x.copy_(x)
        self.len.copy_(torch.tensor([h + n for h, n in zip(have, self.new)], dtype=torch.int32))
        self.pos.copy_(torch.cat([torch.arange(h, h + n, dtype=torch.int32) for h, n in zip(have, self.new)]))

    def check(self):
        """Every product of the step against what it was made from."""
        want, bound = R.adapter_ref(self.x, self.w_qkv, None, self.a1, self.b1, self.scale, self.adapter)
        R.close(self.qkv, want, bound)
        want, bound = R.adapter_ref(self.att, self.w_out, None, self.a2, self.b2, self.scale, self.adapter)
        R.close(self.mid, want, bound)
        want, bound = R.adapter_ref(self.mid, self.w_route)
        R.close(self.logits, want, bound)
        _same_route(self.route, R.route_ref(self.logits, self.top, "softmax", True, 1.0))
        want, bound, _ = R.expert_ref(self.mid, self.w1, self.route["start"], self.h, "silu", x_place=self.route["place"], x_div=self.top)
        R.close(self.h, want, bound)
        want, bound, _ = R.expert_ref(self.h, self.w2, self.route["start"], self.y, y_place=self.route["place"])
        R.close(self.y, want, bound)
        want, bound = R.join_ref(self.y, self.route["expert"], self.route["weight"], self.mid)
        R.close(self.out, want, bound)


@pytest.mark.parametrize("new", [[70, 1, 33, 5, 0, 120], [1] * 9])
def test_layer(ctx, new):
    """Prompts, and then single tokens behind them, through all of the operators."""
    layer = Layer(ctx, new)
    have = [0] * len(new)
    for step in range(3 if max(new) == 1 else 1):
        layer.set(_randn((layer.rows, layer.d), step), have)
        layer.step(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        layer.check()
        have = [h + n for h, n in zip(have, new)]


def test_layer_in_graphs(ctx):
    """Two layers' steps captured, each with its workspaces, replayed beside each other on two streams and in turn with eager work; every
    replay is the eager result on its inputs."""
    layers = [Layer(ctx, [1] * 7, seed=100 * i) for i in range(2)]
    eager = [Layer(ctx, [1] * 7, seed=100 * i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in layers]
    graphs = []
    for layer, s in zip(layers, streams):
        layer.set(_randn((7, layer.d), 1), [0] * 7)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            layer.step(s.cuda_stream)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            layer.step(s.cuda_stream)
        graphs.append(graph)
    for step in range(4):
        for i in range(2):
            for of in (layers[i], eager[i]):
                of.set(_randn((7, of.d), 10 * i + step), [step] * 7)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            eager[i].step(torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            for name in ("qkv", "mid", "logits", "out"):
                assert torch.equal(getattr(layers[i], name), getattr(eager[i], name)), (step, i, name)
            for k, v in layers[i].route.items():
                assert torch.equal(v, eager[i].route[k])


def test_results_repeat(ctx):
    """The same call twice gives the same bits, and a row's result does not depend on how many times it is asked for."""
    k, n, start = 520, 300, _groups([100, 3, 700, 0, 41])
    total = int(start[-1])
    x, w = _randn((total, k), 1), _randn((5, n, k), 2)
    ys = [torch.zeros(total, n, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for y in ys:
        ctx.expert_product(R.expert_args(x, w, start, y))
    assert torch.equal(*ys)
    a, b, scale = _adapters(4, 32, k, n, "bf16")
    ids = (torch.arange(total, device="cuda") // 50 % 5 - 1).int()
    for y in ys:
        R.adapter_run(ctx, R.adapter_args(x, w[0], y, None, a, b, scale, ids))
    assert torch.equal(*ys)


def test_workspaces_too_small(ctx):
    from kokoro_hip import api
    x, w = _randn((100, 64), 1), _randn((40, 64), 2)
    y = torch.zeros(100, 40, dtype=torch.bfloat16, device="cuda")
    a, b, scale = _adapters(2, 8, 64, 40, "bf16")
    args = R.adapter_args(x, w, y, None, a, b, scale, torch.zeros(100, dtype=torch.int32, device="cuda"))
    need = ctx.adapter_product_workspace(args)
    ws = R.space(need + 16)
    for at, size in ((0, need), (R.ptr(ws), need - 1), (R.ptr(ws) + 4, need)):
        args.workspace, args.workspace_bytes = at, size
        with pytest.raises(api.KKError) as e:
            ctx.adapter_product(args)
        assert "workspace" in str(e.value)
    assert need > 0 and not y.any()
    logits = _randn((5000, 8), 1, "f32")
    got = R.route(ctx, logits, 2)
    args, ws, _ = got["kept"]
    args.workspace_bytes = ctx.expert_route_workspace(args) - 1
    with pytest.raises(api.KKError) as e:
        ctx.expert_route(args)
    assert "workspace" in str(e.value)
