"""The join of experts' results on the GPU at the sizes that one launch just holds."""
import pytest
import torch

import product_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind, rows, n", [("bf16", (1 << 23) + 5, 512), ("f32", (1 << 23) + 3, 516)])
def test_join_of_many_rows(kind, rows, n):
    """Millions of rows of 16-byte pieces: a wave takes 512 (256) values, and the rows that hold 2^32 threads of one value each are taken."""
    from kokoro_hip import api
    torch.cuda.init()
    ctx = api.Context(0)
    g = torch.Generator(device="cuda").manual_seed(1)
    y, base = torch.randn(1, n, generator=g, device="cuda").to(R.TYPES[kind]), torch.randn(1, n, generator=g, device="cuda").to(R.TYPES[kind])
    expert = torch.randint(-1, 2, (rows, 1), generator=g, device="cuda", dtype=torch.int32)
    weight = torch.rand(rows, 1, generator=g, device="cuda")
    out = torch.empty(rows, n, dtype=R.TYPES[kind], device="cuda")
    args = R.join_args(y, expert, weight, out, base)
    args.y_row = args.base_row = 0  # one row for all
    ctx.expert_join(args)
    some = torch.cat([torch.arange(1000), torch.randint(0, rows, (5000,)), torch.arange(rows - 1000, rows)]).cuda()
    want, bound = R.join_ref(y.expand(len(some), n), expert[some], weight[some], base.expand(len(some), n))
    R.close(out[some], want, bound)
    # one value a lane: 2^32 threads and more are refused, with nothing written
    out[:, 0] = 7.0
    args.out, args.values = R.ptr(out) + out.element_size(), n - 1
    with pytest.raises(api.KKError) as e:
        ctx.expert_join(args)
    assert "too large" in str(e.value) and (out[:, 0] == 7.0).all()
    ctx.close()
