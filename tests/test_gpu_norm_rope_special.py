"""kk_qk_norm_rope of heads that hold an infinity, at every place of heads of every kind of layout: the norm divides by an infinite
mean, so finite values become zeros, the infinity NaN, and nothing else of the head."""
import math

import pytest
import torch

from kv_ref import TYPES
from test_gpu_norm_rope import _define, _run, _tables, ctx  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dim, rot", [(64, 64), (96, 96), (80, 80), (96, 48), (72, 72), (40, 20), (510, 254), (192, 0), (6, 2)])
def test_an_infinity_leaves_the_rest_of_its_head(ctx, dim, rot, inter, kind):  # noqa: F811
    x = torch.randn(dim, 3, dim, generator=torch.Generator().manual_seed(dim)).to(TYPES[kind])
    x[torch.arange(dim), 1, torch.arange(dim)] = math.inf  # row r: value r of head 1
    x = x.cuda()
    out = torch.empty_like(x)
    pos = torch.arange(1, dim + 1, dtype=torch.int32, device="cuda")
    _run(ctx, kind, x[:, :2], x[:, 2:], out[:, :2], out[:, 2:], pos, rot, inter)
    want = _define(x.cpu(), None, pos.cpu(), rot, inter, _tables(rot, 1e4), 1, 1e-6)[0]
    out = out.cpu().double()
    assert torch.equal(out.isnan(), want.isnan())
    assert not out[:, 1].nan_to_num(0.0).any() and out[:, [0, 2]].isfinite().all()
