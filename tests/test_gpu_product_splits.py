"""Projections with adapters on the GPU where the inputs are taken in several parts, and products of as many groups as there can be, against their
formulas in 64 bits (tests/product_ref.py).  tests/test_product_splits.py shows that these sizes are launched that way."""
import pytest
import torch

import product_ref as R
import product_shapes as S

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


def _ids(rows, many, seed=1):
    """Each row's adapter: half of the rows by request, half in no order; some have none."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(-1, many, (rows,), generator=g, device="cuda", dtype=torch.int32)
    ids[:rows // 2] = torch.sort(ids[:rows // 2]).values
    ids[rows - 1] = many - 1
    return ids


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows, n, k, many, rank", S.JOINED + S.MANY)
def test_adapter_product_parts(ctx, kind, rows, n, k, many, rank):
    x, w = _randn((rows, k), 1, kind), _randn((n, k), 2, kind, k ** -0.5)
    a, b = _randn((many, rank, k), 4, kind, k ** -0.5), _randn((many, n, rank), 5, kind, 3 * rank ** -0.5)
    scale = torch.linspace(-1.0, 2.0, many, device="cuda")
    ids = _ids(rows, many)
    for out, bias in ((kind, None), ("f32", _randn((n,), 3, "f32"))):
        want, bound = R.adapter_ref(x, w, bias, a, b, scale, ids)
        y = torch.empty(rows, n, dtype=R.TYPES[out], device="cuda")
        R.adapter_run(ctx, R.adapter_args(x, w, y, bias, a, b, scale, ids))
        R.close(y, want, bound)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows, n, k, many, rank", S.JOINED + S.MANY)
def test_adapter_product_parts_whole_numbers(ctx, kind, rows, n, k, many, rank):
    """Whole numbers, whose f32 sums are exact in any order and in any parts, come out as they are."""
    g = torch.Generator(device="cuda").manual_seed(rank)

    def whole(shape, most):
        return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(R.TYPES[kind])
    x, w, a, b = whole((rows, k), 7), whole((n, k), 3), whole((many, rank, k), 3), whole((many, n, rank), 1)
    scale = torch.tensor([1.0, -1.0, 0.5, 2.0, 0.0], device="cuda")[torch.arange(many, device="cuda") % 5].contiguous()
    ids = _ids(rows, many, 2)
    want, _ = R.adapter_ref(x, w, None, a, b, scale, ids)
    most = max((x.float() @ a[i].float().t()).abs().sum(1).max().item() for i in range(many))
    assert 2 * most + 21 * k < 2 ** 23  # in halves
    y = torch.empty(rows, n, device="cuda")
    R.adapter_run(ctx, R.adapter_args(x, w, y, None, a, b, scale, ids))
    assert torch.equal(y.double(), want)


@pytest.mark.parametrize("groups, entries, n, k, m", S.GROUPS)
def test_expert_product_most_groups(ctx, groups, entries, n, k, m):
    """1,024 groups of any size at each kind of tile: the largest tables in LDS beside them."""
    g = torch.Generator().manual_seed(m)
    share = torch.rand(groups, generator=g, dtype=torch.float64) ** 3
    share[::5] = 0
    sizes = (share / share.sum() * (entries - groups)).long()
    sizes[groups - 1] += 3
    start = torch.cat([torch.zeros(1, dtype=torch.long), sizes.cumsum(0)]).int().cuda()
    total = int(start[-1])
    x, w = _randn((entries, k), 1), _randn((groups, n, k), 2, "bf16", k ** -0.5)
    y = torch.full((entries, n), 7.0, dtype=torch.bfloat16, device="cuda")
    want, bound, written = R.expert_ref(x, w, start, y)
    assert int(written.sum()) == total <= entries
    ctx.expert_product(R.expert_args(x, w, start, y))
    R.close(y[written], want[written], bound[written])
    assert (y[~written] == 7.0).all()
