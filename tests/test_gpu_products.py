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
@pytest.mark.parametrize("rows, n", [(6000, 2000), (3000, 4100)])
def test_adapter_product_many_rows(ctx, kind, rows, n):
    """Enough tiles for the adapters to go through the main product's own steps, in every way that a tile's rows can share them."""
    k, rank, many = 200, 40, 11
    x, w = _randn((rows, k), 1, kind), _randn((n, k), 2, kind, k ** -0.5)
    a, b, scale = _adapters(many, rank, k, n, kind)
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.sort(torch.randint(-1, many, (rows,), generator=g, device="cuda", dtype=torch.int32)).values
    ids[1000:1500] = torch.randint(-1, many, (500,), generator=g, device="cuda", dtype=torch.int32)
    ids[1500:2100] = -1
    y = torch.empty(rows, n, dtype=R.TYPES[kind], device="cuda")
    want, bound = R.adapter_ref(x, w, None, a, b, scale, ids)
    R.adapter_run(ctx, R.adapter_args(x, w, y, None, a, b, scale, ids))
    R.close(y, want, bound)


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
