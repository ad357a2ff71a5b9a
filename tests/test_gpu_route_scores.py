"""The weights of routing on the GPU where scores leave f32's range, against the definition in 64 bits."""
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


def _same_weights(got, want):
    for k in ("expert", "start", "place"):
        assert torch.equal(got[k].cpu().long(), want[k].long()), k
    w = want["weight"]
    # a score: two exponentials of arguments below 2^10, rounded by 2^-24 of them, and a few steps; a sum, a division, a product
    assert ((got["weight"].cpu().double() - w).abs() <= 2.0 ** -12 * w.abs() + 2.0 ** -140).all()


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("experts", [8, 100, 300])
def test_route_sigmoid_far_below_zero(ctx, kind, experts):
    """Sigmoids divided by their sum: rows whose logits are all far below 0 (their exponentials leave f32) have weights that add up to the
    scale all the same, as the definition's do; without the division a score below f32's range is 0."""
    x = _randn((40, experts), 7, "f32")
    for row, least in enumerate((-1.0, -80.0, -88.0, -90.0, -95.0, -103.0, -110.0, -150.0, -300.0, -600.0)):
        x[row] += least
        x[10 + row, 1:] += least - 5.0
        x[20 + row] = x[20 + row] * abs(least) / 4 + least
    x[30, 3:], x[31, ::2], x[32, 1:] = -torch.inf, -torch.inf, -torch.inf
    x[30:33] -= 100.0
    x[33] = torch.finfo(R.TYPES[kind]).min
    x = x.clamp(min=torch.finfo(R.TYPES[kind]).min).to(R.TYPES[kind])
    x[30, 3:], x[31, ::2], x[32, 1:] = -torch.inf, -torch.inf, -torch.inf
    for renorm, scale in ((True, 1.0), (True, 2.5), (False, 1.0)):
        got = R.route(ctx, x, 6, "sigmoid", renorm, scale)
        _same_weights(got, R.route_ref(x, 6, "sigmoid", renorm, scale))
        if renorm:
            some = (got["expert"][:33] >= 0).any(1)
            assert ((got["weight"][:33].sum(1) - scale).abs() <= 2.0 ** -18 * scale)[some].all() and some.all()
            assert not got["weight"][33].any()
