"""kk_kv_attention where pages that a row attends to have scales of V far apart: a token's weight in the softmax does not depend
on its value's size, so pages of small values count in full in the sum that the result is divided by."""
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


# (new rows, tokens, cache heads, group, values a head, sequences in the batch, whether the axis is split).  Up to 32 rows of a
# (sequence, cache head) and more; one part and several; 130 sequences, the others of one token, fill the device with blocks of 256 rows.
PLANS = {
    "few": (2, 320, 1, 2, 64, 1, False), "few, two tiles": (5, 320, 1, 5, 128, 1, False), "few, parts": (2, 2000, 1, 2, 96, 1, True),
    "many": (50, 320, 1, 2, 64, 1, False), "many, 192 values": (50, 320, 1, 1, 192, 1, False),
    "many, parts": (50, 1700, 1, 2, 128, 1, True), "many, 256 rows": (50, 1700, 4, 2, 128, 130, False),
}


def _bound(want, size, score, most, n, dim, kind, top):
    """- the result's own rounding, half a step;
    - P in f16: 2^-11 of each p |v|; and below f16's normal numbers off by 2^-25 where the row's largest is 2^11 or more, 2^-36 of the
      largest p b a token, times a stored number;
    - scores in f32: (dim + 8) 2^-24 of sum |q k| scale, which changes each p, and their sum, by that much;
    - the sum, in f32: 32 additions of a page's tokens, then 3 steps for each page, 2^-24 each of the result, which is at most `size`."""
    rel = 2.0 ** -11 + (2 * (dim + 8) * score + 40 + 3 * n / PAGE) * 2.0 ** -24
    return R.HALF_STEP[kind] * want.abs() + R.LEAST_STEP[kind] + n * 2.0 ** -36 * top * most + rel * size


@pytest.mark.parametrize("cache_kind, kind", [("int8", "bf16"), ("e4m3", "f16")])
@pytest.mark.parametrize("bits", [28, 40, 80, 97])
@pytest.mark.parametrize("order", ["large first", "large last", "large in the middle", "small ahead"])
@pytest.mark.parametrize("plan", PLANS)
def test_small_values_keep_their_weight(ctx, plan, order, bits, cache_kind, kind):
    """One page's values are 2^bits times larger than the others' (97: from near the smallest scale there is, 2^-90).  Scores are
    level over all pages, or some 8 bits higher on two pages of small values."""
    new, n, heads, group, dim, seqs, parts = PLANS[plan]
    pages = -(-n // PAGE)
    cache = R.Cache(cache_kind, heads, dim, pages + 2)
    tables = R.deal([n], pages + 1, np.random.default_rng(bits))
    g = torch.Generator().manual_seed(bits + dim)
    k, v = (torch.randn(n, heads, dim, generator=g) for _ in range(2))
    at = {"large first": 0, "small ahead": 0, "large last": (n - new - 1) // PAGE, "large in the middle": 1}[order]
    far = torch.ones(n, dtype=torch.bool)
    far[at * PAGE:(at + 1) * PAGE] = False
    v *= 2.0 ** 12 if bits > 80 else 1.0
    v[far] *= 2.0 ** -bits
    q = 1 + 0.3 * torch.randn(new + seqs - 1, heads * group, dim, generator=g)
    scale = 1.0 / dim ** 0.5
    if order == "small ahead":
        k[PAGE:3 * PAGE] += 8 * 0.6931 / dim ** 0.5
    R.write(ctx, cache, R.Batch([n], [n], tables), k.cuda(), v.cuda(), 3)
    assert cache.same()
    other = next(p for p in range(cache.pages) if p not in tables[0])  # the other sequences' one token
    if seqs > 1:
        one = torch.randn(2, 1, heads, dim, generator=g).cuda()
        R.write(ctx, cache, R.Batch([1], [1], [[other]]), one[0], one[1], 3)
    batch = R.Batch([new] + [1] * (seqs - 1), [n] + [1] * (seqs - 1), tables + [[other]] * (seqs - 1))
    q = q.to(R.TYPES[kind]).cuda()
    out = torch.full_like(q, 9.0)
    args, _ = R.attention_args(ctx, cache, batch, q, out, {"bf16": 1, "f16": 2}[kind], scale)
    assert bool(args.workspace_bytes) == parts
    ctx.kv_attention(cache.args, batch.args, args)
    for b, length in list(enumerate(batch.lens))[:2]:
        r = slice(int(batch.start[b]), int(batch.start[b + 1]))
        kt, vt = [cache.tokens(batch.tables[b], length, p) for p in "kv"]
        want, size, score, most = R.attend(q[r].cpu().double(), kt, vt, cache.scales(batch.tables[b], length), scale, True, 0)
        tol = _bound(want, size, score, most, length, dim, kind, R.TOP[cache_kind])
        off = (out[r].cpu().double() - want).abs()
        assert bool((off <= tol).all()), (b, float((off / tol).nan_to_num(nan=1e9).max()))
