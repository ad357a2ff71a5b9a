"""The products of ragged rows on the GPU where offsets pass 2^31 values and 2^32 bytes: rows, matrices, adapters and workspaces of that size, against
their formulas in 64 bits (tests/product_ref.py)."""
import pytest
import torch

import product_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture
def ctx():
    from kokoro_hip import api
    torch.cuda.init()
    c = api.Context(0)
    yield c
    c.close()
    torch.cuda.empty_cache()


def _randn(shape, seed, kind="bf16", size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * size).to(R.TYPES[kind])


def _apart(values, *strides):
    """The values in rows that lie so far apart, the last row ending the memory."""
    size = sum((n - 1) * s for n, s in zip(values.shape, strides)) + values.shape[-1]
    assert size > 2 ** 31
    out = torch.empty(size, dtype=values.dtype, device="cuda").as_strided(values.shape, (*strides, 1))
    out.copy_(values)
    return out


def test_expert_product_far_apart(ctx):
    k, n = 72, 40
    start = torch.tensor([0, 20, 65, 70], dtype=torch.int32, device="cuda")
    x, w = _apart(_randn((70, k), 1), 2 ** 25 + 8), _apart(_randn((3, n, k), 2), 3 * 2 ** 29, 2 ** 25 + 8)
    y = _apart(torch.full((70, n), 7.0, dtype=torch.bfloat16, device="cuda"), 2 ** 26 + 16)
    perm = torch.randperm(70, generator=torch.Generator().manual_seed(1)).int().cuda()
    want, bound, written = R.expert_ref(x, w, start, y, x_place=perm.flip(0), y_place=perm)
    ctx.expert_product(R.expert_args(x, w, start, y, x_place=perm.flip(0).contiguous(), y_place=perm))
    assert written.all()
    R.close(y, want, bound)


def test_route_far_apart(ctx):
    x = _apart(_randn((40, 100), 1, "f16"), 2 ** 26 + 8)
    got, want = R.route(ctx, x, 6), R.route_ref(x, 6, "softmax", True, 1.0)
    for name in ("expert", "start", "place"):
        assert torch.equal(got[name].cpu().long(), want[name].long()), name
    # as for rows next to each other: rounded arguments of exponentials, a sum, a division, a product
    assert ((got["weight"].cpu().double() - want["weight"]).abs() <= 2.0 ** -14 * want["weight"]).all()


@pytest.mark.parametrize("n", [520, 37])
def test_join_far_apart(ctx, n):
    rows, top = 14, 5
    y, base = _apart(_randn((rows * top, n), 1), 2 ** 25 + 8), _apart(_randn((rows, n), 2), 2 ** 28 + 8)
    out = _apart(torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda"), 2 ** 28 + 8)
    g = torch.Generator(device="cuda").manual_seed(3)
    expert = torch.randint(-1, 3, (rows, top), generator=g, device="cuda", dtype=torch.int32)
    weight = torch.rand(rows, top, generator=g, device="cuda")
    want, bound = R.join_ref(y.contiguous(), expert, weight, base)
    ctx.expert_join(R.join_args(y, expert, weight, out, base))
    R.close(out, want, bound)


@pytest.mark.parametrize("n", [130, 33000])
def test_adapter_product_far_apart(ctx, n):
    """Rows of x, w and y, with the parts summed up by a kernel of their own and with the adapters as more inputs."""
    rows, k, rank = 70, 72, 16
    x, w = _apart(_randn((rows, k), 1), 2 ** 25 + 8), _apart(_randn((n, k), 2, "bf16", k ** -0.5), (2 ** 32 // n) // 8 * 8)
    a, b, scale = _randn((3, rank, k), 3, "bf16", k ** -0.5), _randn((3, n, rank), 4, "bf16", rank ** -0.5), torch.tensor([1.0, -1.0, 2.0], device="cuda")
    ids = (torch.arange(rows, device="cuda") // 10 % 4 - 1).int()
    y = _apart(torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda"), 2 ** 26 + 16)
    want, bound = R.adapter_ref(x, w, None, a, b, scale, ids)
    R.adapter_run(ctx, R.adapter_args(x, w, y, None, a, b, scale, ids))
    R.close(y, want, bound)


@pytest.mark.parametrize("rows, many, n, k", [(3, 5, 8, 2 ** 21), (3, 300, 32000, 64), (3, 5, 2 ** 21 + 8, 64), (600, 5, 256, 2 ** 21)])
def test_adapter_product_large_adapters(ctx, rows, many, n, k):
    """Adapters whose a or b together have more than 2^31 values, of which the first and the last are used."""
    rank = 256
    x, w = _randn((rows, k), 1), _randn((n, k), 2, "bf16", k ** -0.5)
    a = torch.empty(many, rank, k, dtype=torch.bfloat16, device="cuda")
    b = torch.empty(many, n, rank, dtype=torch.bfloat16, device="cuda")
    assert max(a.numel(), b.numel()) > 2 ** 31
    for i in (0, many - 1):
        a[i], b[i] = _randn((rank, k), 3 + i, "bf16", k ** -0.5), _randn((n, rank), 4 + i, "bf16", rank ** -0.5)
    ids = torch.tensor([-1, 0, many - 1], dtype=torch.int32, device="cuda")[torch.arange(rows, device="cuda") * 3 // rows].contiguous()
    scale = torch.full((many,), 0.5, device="cuda")
    y = torch.empty(rows, n, device="cuda")
    R.adapter_run(ctx, R.adapter_args(x, w, y, None, a, b, scale, ids))
    for r in (0, rows // 2, rows - 1):  # a row at a time: 64-bit copies are large
        i = int(ids[r])
        more = (None, None, None, None) if i < 0 else (a[i:i + 1], b[i:i + 1], scale[:1], torch.zeros(1, dtype=torch.int32, device="cuda"))
        want, bound = R.adapter_ref(x[r:r + 1], w, None, *more)
        R.close(y[r:r + 1], want, bound)


def test_adapter_product_large_workspace(ctx):
    """Nine million rows: a x and its parts of 16 bits have more than 2^31 values each."""
    rows, n, k, rank = 9_000_000, 8, 64, 256
    x, w = _randn((rows, k), 1), _randn((n, k), 2, "bf16", k ** -0.5)
    a, b, scale = _randn((3, rank, k), 3, "bf16", k ** -0.5), _randn((3, n, rank), 4, "bf16", rank ** -0.5), torch.tensor([1.0, -1.0, 2.0], device="cuda")
    ids = (torch.arange(rows, device="cuda") // 1_000_000 % 4 - 1).int()
    y = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    ws = R.adapter_run(ctx, R.adapter_args(x, w, y, None, a, b, scale, ids))
    assert rows * rank > 2 ** 31 and ws.numel() > 2 ** 31
    some = torch.cat([torch.arange(1000), torch.randint(0, rows, (5000,)), torch.arange(rows - 1000, rows)]).cuda()
    want, bound = R.adapter_ref(x[some], w, None, a, b, scale, ids[some])
    R.close(y[some], want, bound)
