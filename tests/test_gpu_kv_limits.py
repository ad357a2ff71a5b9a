"""kk_kv_attention of as many sequences as a batch may have, whose bound would split the axis into more blocks than a launch holds."""
import numpy as np
import pytest
import torch

import kv_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from kokoro_hip import api
    torch.cuda.init()
    c = api.Context(0)
    yield c
    c.close()


def test_a_million_sequences(ctx):
    """2^20 sequences that share a page table, 20,000 tokens, of which the first and the last have a row: 4.2 million blocks a part."""
    from kokoro_hip import api
    n, tokens, heads, dim = 1 << 20, 20000, 4, 64
    cache = R.Cache("int8", heads, dim, 320)
    tables = R.deal([tokens], 320, np.random.default_rng(1))
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(tokens, heads, dim, generator=g).cuda() for _ in range(2))
    R.write(ctx, cache, R.Batch([tokens], [tokens], tables), k, v, api.F32)
    start = torch.ones(n + 1, dtype=torch.int32, device="cuda")
    start[0], start[n] = 0, 2
    lens = torch.full((n,), tokens, dtype=torch.int32, device="cuda")
    table = torch.tensor(tables[0], dtype=torch.int32, device="cuda")
    batch = api.KvBatch(n=n, rows=2, max_new=1, max_len=tokens, row_start=start.data_ptr(), len=lens.data_ptr(),
                        table=table.data_ptr(), table_width=len(table), table_stride=0)
    q = torch.randn(2, 2 * heads, dim, generator=g).bfloat16().cuda()
    out = torch.zeros_like(q)
    args, space = R.attention_args(ctx, cache, type("", (), {"args": batch}), q, out, api.BF16, 0.2)
    assert 1 << 10 < args.workspace_bytes < 1 << 16  # some parts
    ctx.kv_attention(cache.args, batch, args)
    R.check_attention(out, q, cache, R.Batch([1, 1], [tokens] * 2, tables * 2), 0.2, True, 0, "bf16")
    assert (space[args.workspace_bytes:] == 0xA5).all() and int(cache.fault) == 0


def test_large_bounds(ctx):
    """Workspaces of serving steps with generous bounds exist, and grow no more than the bounds."""
    from kokoro_hip import api
    p = 1 << 20  # passes as a pointer: the arguments are checked, nothing is launched
    cache = api.KvCache(type=api.KV_INT8, heads=8, dim=128, pages=9, k=p, v=p, k_scale=p, v_scale=p)
    args = api.KvAttention(type=api.BF16, heads=32, q=p, q_row=4096, q_head=128, out=2 * p, out_row=4096, out_head=128, scale=0.1, causal=1)
    for n, bound in ((5000, 1000000), (300000, 5000), (1 << 20, 1 << 30)):
        batch = api.KvBatch(n=n, rows=n, max_new=1, max_len=bound, row_start=p, len=p, table=p, table_width=-(-bound // 64), table_stride=0)
        parts = ctx.kv_attention_workspace(cache, batch, args) / (n * 32 * (128 + 2) * 4)
        assert parts == int(parts) <= min(256, -(-bound // 64)) and parts * n * 8 * 256 < 1 << 32


@pytest.mark.parametrize("said", [1 << 40, (1 << 63) + 5, (1 << 64) - 1])
def test_a_workspace_of_any_stated_size(ctx, said):
    """A workspace that is as large as needed and said to be larger, up to the largest number that its size can be."""
    from kokoro_hip import api
    cache = R.Cache("int8", 1, 64, 40)
    tables = R.deal([2000], 40, np.random.default_rng(1))
    k, v = torch.randn(2, 2000, 1, 64, generator=torch.Generator().manual_seed(2)).cuda()
    R.write(ctx, cache, R.Batch([2000], [2000], tables), k, v, api.F32)
    batch = R.Batch([1], [2000], tables)
    q = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    out = torch.zeros_like(q)
    args, space = R.attention_args(ctx, cache, batch, q, out, api.BF16, 0.2)
    need, args.workspace_bytes = args.workspace_bytes, said
    assert need > 0
    ctx.kv_attention(cache.args, batch.args, args)
    R.check_attention(out, q, cache, batch, 0.2, True, 0, "bf16")
    assert (space[need:] == 0xA5).all()
