"""Projections with adapters on the GPU with infinities and NaN in an adapter's second matrix, against what the formula gives."""
import pytest
import torch

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


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows, n, k, rank", [(40, 100, 72, 16), (700, 200, 72, 40), (3000, 1000, 72, 24), (6000, 2000, 1544, 16), (4200, 4096, 1032, 64)])
@pytest.mark.parametrize("order", ["one", "sorted", "mixed"])
def test_adapter_product_infinite_b(ctx, kind, rows, n, k, rank, order):
    """An infinity or NaN in a row of an adapter's b makes that output what the formula says (infinite with the sign of its a x, NaN where two
    differ) in the rows of that adapter, however many rows the call has; every other output is as without it."""
    x, w = _randn((rows, k), 1, kind).abs() + 0.5, _randn((n, k), 2, kind, k ** -0.5)
    a, b = _randn((4, rank, k), 3, kind, k ** -1).abs() + 0.5 / k, _randn((4, n, rank), 4, kind, rank ** -0.5)
    scale = torch.tensor([1.0, 0.5, -2.0, 1.0], device="cuda")  # every a x is positive, so the sign is the scale's
    if order == "one":
        ids = torch.full((rows,), 2, dtype=torch.int32, device="cuda")
    else:
        ids = torch.randint(-1, 4, (rows,), generator=torch.Generator(device="cuda").manual_seed(5), device="cuda", dtype=torch.int32)
        ids = torch.sort(ids).values if order == "sorted" else ids
    wild = torch.zeros(4, n, rank, device="cuda")
    for i in (1, 2):
        wild[i, i::7, 3], wild[i, i + 1::7, rank - 1], wild[i, i + 2::7, 0] = torch.inf, -torch.inf, torch.nan
        wild[i, i + 3::7, 1], wild[i, i + 3::7, 5] = torch.inf, -torch.inf
    bad = ~torch.isfinite(wild).all(2)
    b = torch.where(wild == 0, b.float(), 0.0).to(b.dtype)  # finite: the same without the wild ones
    full = torch.where(wild == 0, b.float(), wild).to(b.dtype)
    pattern = wild.sum(2) * scale[:, None]  # of an output with wild ones
    for out, bias in ((kind, None), ("f32", _randn((n,), 6, "f32"))):
        want, bound = R.adapter_ref(x, w, bias, a, b, scale, ids)
        y = torch.empty(rows, n, dtype=R.TYPES[out], device="cuda")
        R.adapter_run(ctx, R.adapter_args(x, w, y, bias, a, full, scale, ids))
        at = (ids >= 0)[:, None] & bad[ids.clamp(min=0).long()]
        R.close(y[~at], want[~at], bound[~at])
        says = pattern[ids.clamp(min=0).long()][at]
        got = y[at].float()
        assert torch.equal(torch.isnan(got), torch.isnan(says))
        assert torch.equal(got[~torch.isnan(says)], says[~torch.isnan(says)])


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows, n", [(40, 100), (3000, 1000), (4200, 4096)])
def test_adapter_product_rows_of_nan(ctx, kind, rows, n):
    """Rows of NaN (a padded batch's) beside infinities in one adapter's b: those rows are NaN, every other one is what the formula says."""
    k, rank = 72, 24
    x, w = _randn((rows, k), 1, kind).abs() + 0.5, _randn((n, k), 2, kind, k ** -0.5)
    a, b = _randn((3, rank, k), 3, kind, k ** -1).abs() + 0.5 / k, _randn((3, n, rank), 4, kind, rank ** -0.5)
    scale, ids = torch.ones(3, device="cuda"), (torch.arange(rows, device="cuda") // 5 % 4 - 1).int()
    want, bound = R.adapter_ref(x, w, None, a, b, scale, ids)
    none = torch.arange(rows, device="cuda") % 13 == 7
    x[none], x[none, 3:] = torch.nan, 1.0
    b[1, ::9, 7] = torch.inf
    y = torch.empty(rows, n, dtype=R.TYPES[kind], device="cuda")
    R.adapter_run(ctx, R.adapter_args(x, w, y, None, a, b, scale, ids))
    far = torch.zeros(rows, n, dtype=torch.bool, device="cuda")
    far[:, ::9] = (ids == 1)[:, None]
    assert torch.isnan(y[none]).all() and (y[far & ~none[:, None]] == torch.inf).all()
    good = ~far & ~none[:, None]
    R.close(y[good], want[good], bound[good])
