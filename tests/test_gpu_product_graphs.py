"""The products of ragged rows of prompts' sizes captured into graphs that are replayed beside each other, and at the largest numbers of rows."""
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
    torch.cuda.empty_cache()


def _randn(shape, seed, kind="bf16", size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * size).to(R.TYPES[kind])


class Prompts:
    """Many rows through an adapted projection in three kernels and more, routing in two, products of large tiles, the join."""

    def __init__(self, ctx, rows=2300, d=1032, n=4096, experts=8, top=2, seed=0):
        from kokoro_hip import api
        self.ctx, self.rows, self.d, self.many = ctx, rows, d, 6
        like = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
        self.x, self.y, self.ids = like(rows, d), like(rows, n), like(rows, t=torch.int32)
        self.logits = like(rows, experts, t=torch.float32)
        w, a, b = _randn((n, d), seed + 1, size=d ** -0.5), _randn((self.many, 24, d), seed + 2, size=d ** -0.5), _randn((self.many, n, 24), seed + 3, size=0.2)
        scale = torch.linspace(0.5, 2.0, self.many, device="cuda")
        self.adapted = R.adapter_args(self.x, w, self.y, None, a, b, scale, self.ids)
        ws = R.space(ctx.adapter_product_workspace(self.adapted))
        self.adapted.workspace, self.adapted.workspace_bytes = R.ptr(ws), ws.numel() * 4
        self.route = {"expert": like(rows, top, t=torch.int32), "weight": like(rows, top, t=torch.float32),
                      "start": like(experts + 1, t=torch.int32), "place": like(rows * top, t=torch.int32)}
        self.router = api.ExpertRoute(type=api.F32, rows=rows, experts=experts, top=top, logits=R.ptr(self.logits), logits_row=experts, renorm=1,
                                      scale=1.0, score=api.SCORE_SIGMOID, **{k: R.ptr(v) for k, v in self.route.items()})
        ws2 = R.space(ctx.expert_route_workspace(self.router))
        self.router.workspace, self.router.workspace_bytes = R.ptr(ws2), ws2.numel() * 4
        w1, w2 = _randn((experts, 2 * 520, n), seed + 4, size=n ** -0.5), _randn((experts, n, 520), seed + 5, size=0.05)
        self.h, self.z, self.out = like(rows * top, 520), like(rows * top, n), like(rows, n)
        self.up = R.expert_args(self.y, w1, self.route["start"], self.h, rows * top, "silu", x_place=self.route["place"], x_div=top)
        self.down = R.expert_args(self.h, w2, self.route["start"], self.z, rows * top, y_place=self.route["place"])
        self.join = R.join_args(self.z, self.route["expert"], self.route["weight"], self.out, self.y)
        self.kept = (w, a, b, scale, ws, ws2, w1, w2)

    def set(self, seed):
        self.x.copy_(_randn((self.rows, self.d), seed))
        self.logits.copy_(_randn(self.logits.shape, seed + 1, "f32", 2.0))
        self.logits[seed % 7::30] = -torch.inf
        self.ids.copy_(torch.sort(torch.randint(-1, self.many, (self.rows,), generator=torch.Generator().manual_seed(seed))).values)

    def step(self, stream):
        c = self.ctx
        c.adapter_product(self.adapted, stream)
        c.expert_route(self.router, stream)
        c.expert_product(self.up, stream)
        c.expert_product(self.down, stream)
        c.expert_join(self.join, stream)


def test_prompts_in_graphs(ctx):
    """Two graphs with a workspace each, replayed at the same time on two streams; every replay is the eager result on its inputs."""
    steps, eager = [Prompts(ctx, seed=100 * i) for i in range(2)], [Prompts(ctx, seed=100 * i) for i in range(2)]
    streams, graphs = [torch.cuda.Stream() for _ in steps], []
    for one, s in zip(steps, streams):
        one.set(1)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            one.step(s.cuda_stream)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            one.step(s.cuda_stream)
        graphs.append(graph)
    for n in range(4):
        for i in range(2):
            steps[i].set(10 * n + i), eager[i].set(10 * n + i)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            eager[i].step(torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            assert torch.isfinite(eager[i].out).all()
            for k, v in steps[i].route.items():
                assert torch.equal(v, eager[i].route[k]), (n, i, k)
            # rows that no entry goes to are left as the step before left them
            entries, live = int(eager[i].route["start"][-1]), (eager[i].route["expert"] >= 0).view(-1)
            assert 0 < entries < len(live) and entries == int(live.sum())
            for name, rows in (("y", slice(None)), ("h", slice(entries)), ("z", live), ("out", slice(None))):
                assert torch.equal(getattr(steps[i], name)[rows], getattr(eager[i], name)[rows]), (n, i, name)


def test_route_most_rows(ctx):
    """2^28 rows of two experts."""
    rows = 1 << 28
    x = torch.randint(-2, 3, (rows, 2), device="cuda", dtype=torch.int8).to(torch.bfloat16)
    x[12345::1 << 20] = -torch.inf
    got = R.route(ctx, x, 1)
    expert = torch.where(x[:, 0] == -torch.inf, -1, (x[:, 1] > x[:, 0]).int())
    assert torch.equal(got["expert"][:, 0], expert)
    assert torch.equal(got["weight"][:, 0], (expert >= 0).float())
    at = 0
    for e in range(2):
        assert int(got["start"][e]) == at
        places = (expert == e).nonzero()[:, 0]
        assert torch.equal(got["place"][at:at + len(places)].long(), places)
        at += len(places)
    assert int(got["start"][2]) == at < rows and (got["place"][at:] == -1).all()


def test_expert_product_most_entries(ctx):
    """2^28 entries, of which two groups have nearly all."""
    entries = 1 << 28
    start = torch.tensor([0, 100_000_001, 100_000_001, entries - 3], dtype=torch.int32, device="cuda")
    x, w = torch.randint(-3, 4, (entries, 8), device="cuda", dtype=torch.int8).to(torch.bfloat16), _randn((3, 1, 8), 2)
    y = torch.full((entries, 1), 7.0, dtype=torch.bfloat16, device="cuda")
    ctx.expert_product(R.expert_args(x, w, start, y))
    assert (y[-3:] == 7.0).all()
    some = torch.cat([torch.arange(500), torch.arange(99_999_500, 100_000_500), torch.randint(0, entries - 3, (5000,)), torch.arange(entries - 500, entries - 3)]).cuda()
    for g, rows in ((0, some[some < 100_000_001]), (2, some[some >= 100_000_001])):
        want, bound = R.product(x[rows], w[g])
        R.close(y[rows], want, bound)
