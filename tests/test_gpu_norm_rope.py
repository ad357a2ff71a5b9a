"""kk_qk_norm_rope against its definition in 64 bits, through the library's entry point."""
import math

import numpy as np
import pytest
import torch

from kv_ref import HALF_STEP, LEAST_STEP, TYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from kokoro_hip import api
    torch.cuda.init()
    c = api.Context(0)
    yield c
    c.close()


def _define(x, w, pos, rot, inter, freq, norm, eps):
    """(y, bound): f64 values, and for each pair |a| + |b| of the values that it turns (else |a|)."""
    x = x.double()
    if norm:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
        x = x * w.double() if w is not None else x
    t = pos.double()[:, None, None] * freq
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    y, size = x.clone(), x.abs()
    y[..., a] = x[..., a] * torch.cos(t) - x[..., b] * torch.sin(t)
    y[..., b] = x[..., b] * torch.cos(t) + x[..., a] * torch.sin(t)
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs())
    return y, size


def _tables(rot, theta):
    return torch.tensor([theta ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64)


def _run(ctx, kind, q, k, qo, ko, pos, rot, inter=False, theta=1e4, wq=None, wk=None, norm=1, eps=1e-6, freq=None):
    from kokoro_hip import api
    p = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    s = lambda t, i: t.stride(i) if t is not None else 0   # noqa: E731
    args = api.NormRope(
        type={"bf16": api.BF16, "f16": api.F16, "f32": api.F32}[kind], dim=(q if q is not None else k).shape[2], rows=len(pos),
        q_heads=q.shape[1] if q is not None else 0, k_heads=k.shape[1] if k is not None else 0, q=p(q), q_row=s(q, 0),
        q_head=s(q, 1), k=p(k), k_row=s(k, 0), k_head=s(k, 1), q_out=p(qo), q_out_row=s(qo, 0), q_out_head=s(qo, 1), k_out=p(ko),
        k_out_row=s(ko, 0), k_out_head=s(ko, 1), norm=norm, eps=eps, q_weight=p(wq), k_weight=p(wk), pos=p(pos), rot=rot,
        interleaved=int(inter), theta=theta, freq=p(freq))
    ctx.qk_norm_rope(args)


def _check(got, x, w, pos, rot, inter, freq, norm, eps, kind):
    """The bound: half a step of the result's type, and the f32 steps: the norm's sum of dim squares in at most 16 + 6
    additions a lane and its root (half of the sum's error), a product with the weight, the turn's fraction (2^-25 of a turn:
    2^-22.3 rad), sine and cosine (2 steps each) and two products and a sum -- below 64 steps of 2^-24 of |a| + |b|.  Scalar heads
    add up 8 squares a lane and are covered too."""
    want, size = _define(x.cpu(), w.cpu() if w is not None else None, pos.cpu(), rot, inter, freq, norm, eps)
    off = (got.cpu().double() - want).abs()
    tol = HALF_STEP[kind] * want.abs() + LEAST_STEP[kind] + 64 * 2.0 ** -24 * size
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("rows, hq, hk, dim, rot", [
    (1, 1, 0, 2, 2), (1, 32, 8, 128, 128), (5, 3, 1, 64, 64), (7, 12, 12, 64, 32), (33, 5, 1, 72, 72), (3, 8, 8, 40, 20),
    (9, 16, 4, 80, 80), (2, 2, 2, 96, 48), (4, 0, 3, 256, 256), (6, 3, 2, 512, 512), (5, 2, 1, 510, 254), (300, 9, 3, 128, 64),
    (2, 2, 2, 64, 0), (4100, 2, 1, 16, 16)])
def test_norm_and_rotation(ctx, kind, inter, rows, hq, hk, dim, rot):
    g = torch.Generator().manual_seed(dim + rows)
    wide = (hq + 2 * hk + 1) * dim
    buf = (torch.randn(rows, wide, generator=g) * 3).to(TYPES[kind]).cuda()
    pos = torch.randint(-3, 5000, (rows,), generator=g, dtype=torch.int32).cuda()
    wq, wk = ((1 + 0.4 * torch.randn(dim, generator=g)).cuda() for _ in range(2))
    q = buf[:, :hq * dim].unflatten(1, (hq, dim)) if hq else None
    k = buf[:, hq * dim:(hq + hk) * dim].unflatten(1, (hk, dim)) if hk else None
    qo, ko = (torch.empty(x.shape, dtype=x.dtype, device="cuda") if x is not None else None for x in (q, k))
    kept = buf.clone()
    _run(ctx, kind, q, k, qo, ko, pos, rot, inter, 1e4, wq, wk)
    freq = _tables(rot, 1e4)
    for x, o, w in ((q, qo, wq), (k, ko, wk)):
        if x is not None:
            _check(o, x, w, pos, rot, inter, freq, 1, 1e-6, kind)
    assert torch.equal(buf, kept)
    # in place, and nothing else of the rows touched
    _run(ctx, kind, q, k, q, k, pos, rot, inter, 1e4, wq, wk)
    for x, o in ((q, qo), (k, ko)):
        assert x is None or torch.equal(x, o)
    assert torch.equal(buf[:, (hq + hk) * dim:], kept[:, (hq + hk) * dim:])


@pytest.mark.parametrize("theta", [1e4, 5e5, 1.0])
def test_far_positions(ctx, theta):
    """Positions over the whole range of int32: the angle's error stays what 64 bits and one turn's fraction give."""
    pos = torch.tensor([0, 1, -1, 131071, 10 ** 6, 2 ** 24 + 1, -2 ** 30 - 1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32).cuda()
    x = torch.randn(len(pos), 3, 128, generator=torch.Generator().manual_seed(1)).cuda()
    out = torch.empty_like(x)
    _run(ctx, "f32", x, None, out, None, pos, 128, theta=theta)
    want, size = _define(x.cpu(), None, pos.cpu(), 128, False, _tables(128, theta), 1, 1e-6)
    # and f_i itself in 64 bits on both sides: some 2^-49 of an angle of up to 2^31
    angle = pos.cpu().double().abs()[:, None, None] * _tables(128, theta).repeat(2)
    assert ((out.cpu().double() - want).abs() <= (66 * 2.0 ** -24 + angle * 2.0 ** -48) * size).all()


@pytest.mark.parametrize("shift", [0, 1])
def test_no_norm_table_and_unaligned(ctx, shift):
    """Rotation alone by a table of frequencies, without weights; rows that are not 16-byte aligned."""
    g = torch.Generator().manual_seed(2)
    buf = torch.randn(11, 6 * 64 + 7, generator=g).bfloat16().cuda()
    res = torch.full_like(buf, 8.0)
    view, out = (b[:, shift:shift + 6 * 64].unflatten(1, (6, 64)) for b in (buf, res))
    pos = torch.randint(0, 9000, (11,), generator=g, dtype=torch.int32).cuda()
    freq = torch.rand(32, generator=g, dtype=torch.float64).cuda()
    for norm in (0, 1):
        _run(ctx, "bf16", view[:, :4], view[:, 4:], out[:, :4], out[:, 4:], pos, 64, norm=norm, freq=freq, theta=-1.0)
        _check(out, view, None, pos, 64, False, freq.cpu(), norm, 1e-6, "bf16")
        assert (res[:, :shift] == 8.0).all() and (res[:, shift + 6 * 64:] == 8.0).all()


def test_special_values(ctx):
    """Zeros stay zeros; NaN and infinity stay in their head; values whose squares overflow or vanish in f32 follow f32."""
    x = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(3))
    x[0, 0] = 0.0
    x[1, 1, 5], x[2, 2, 6] = math.nan, math.inf
    x[0, 3] *= 1e-25
    x = x.cuda()
    out = torch.empty_like(x)
    pos = torch.tensor([0, 7, 99], dtype=torch.int32).cuda()
    _run(ctx, "f32", x, None, out, None, pos, 32)
    out = out.cpu()
    assert not out[0, 0].any()
    assert out[1, 1].isnan().all() and out[2, 2].isnan().any()
    bad = torch.zeros(3, 4, dtype=torch.bool)
    bad[1, 1] = bad[2, 2] = True
    assert out[~bad].isfinite().all()
    want, size = _define(x.cpu(), None, pos.cpu(), 32, False, _tables(32, 1e4), 1, 1e-6)
    assert ((out.double() - want).abs()[~bad] <= 65 * 2.0 ** -24 * size[~bad] + 2.0 ** -126).all()


def test_rows_do_not_depend_on_each_other(ctx):
    """A row alone gives the same bits as among 2,000 others (other ways of sharing the work between waves)."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2000, 10, 128, generator=g).half().cuda()
    pos = torch.randint(0, 4000, (2000,), generator=g, dtype=torch.int32).cuda()
    w = (1 + 0.1 * torch.randn(128, generator=g)).cuda()
    out = torch.empty_like(x)
    _run(ctx, "f16", x[:, :8], x[:, 8:], out[:, :8], out[:, 8:], pos, 128, wq=w, wk=w)
    for r in (0, 1, 777, 1999):
        one = torch.empty_like(x[r:r + 1])
        _run(ctx, "f16", x[r:r + 1, :8], x[r:r + 1, 8:], one[:, :8], one[:, 8:], pos[r:r + 1], 128, wq=w, wk=w)
        assert torch.equal(one, out[r:r + 1])
    assert np.isfinite(out.float().cpu().numpy()).all()
