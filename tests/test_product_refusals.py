"""What the products of ragged rows refuse, on the CPU: every argument check runs before the context and the device are looked at, so
a call without a context shows its message (and one whose arguments are fine shows that there is no context)."""
import ctypes as C

import pytest

P = 1 << 20  # a number that passes as a device pointer: nothing is read from it


def _call(name, args):
    from kokoro_hip import api
    err = C.create_string_buffer(512)
    tail = () if name.endswith("workspace") else (None,)
    rc = getattr(api.lib(), name)(None, C.byref(args) if args is not None else None, *tail, err, 512)
    return rc, err.value.decode()


def _route(**kw):
    from kokoro_hip import api
    base = dict(type=api.F32, rows=10, experts=64, top=8, logits=P, logits_row=64, score=0, renorm=1, scale=1.0, expert=2 * P,
                weight=3 * P, start=4 * P, place=5 * P, workspace=6 * P, workspace_bytes=1 << 40)
    return api.ExpertRoute(**{**base, **kw})


def _expert(**kw):
    from kokoro_hip import api
    base = dict(type=api.BF16, groups=8, entries=20, inputs=64, outputs=33, start=P, x=2 * P, x_rows=20, x_row=64, x_div=0, w=3 * P,
                w_row=64, w_group=64 * 33, gate=0, y=4 * P, y_rows=20, y_row=33)
    return api.ExpertProduct(**{**base, **kw})


def _join(**kw):
    from kokoro_hip import api
    base = dict(type=api.F16, rows=10, top=4, values=100, y=P, y_row=100, expert=2 * P, weight=3 * P, base=4 * P, base_row=100, out=5 * P,
                out_row=100)
    return api.ExpertJoin(**{**base, **kw})


def _adapter(**kw):
    from kokoro_hip import api
    base = dict(type=api.BF16, out_type=api.BF16, rows=10, inputs=64, outputs=33, x=P, x_row=64, w=2 * P, w_row=64, y=3 * P, y_row=33,
                adapters=3, rank=16, a=4 * P, b=5 * P, scale=6 * P, adapter=7 * P, workspace=8 * P, workspace_bytes=1 << 40)
    return api.AdapterProduct(**{**base, **kw})


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("kw, word", [
    (dict(type=0), "type"), (dict(type=4), "type"), (dict(experts=0), "expert count"), (dict(experts=1025), "expert count"),
    (dict(top=0), "top"), (dict(top=33), "top"), (dict(top=9, experts=8), "top"), (dict(rows=-1), "rows"), (dict(rows=1 << 26), "rows"),
    (dict(score=2), "score"), (dict(renorm=2), "renorm"), (dict(scale=NAN), "scale"), (dict(scale=INF), "scale"),
    (dict(logits=None), "null"), (dict(place=None), "null"), (dict(rows=0, start=None), "null"), (dict(logits=P + 2), "aligned"),
    (dict(weight=P + 2), "aligned"), (dict(start=P + 1), "aligned")])
def test_route_refusals(kw, word):
    from kokoro_hip import api
    for name in ("kk_expert_route", "kk_expert_route_workspace"):
        rc, msg = _call(name, _route(**kw))
        assert rc == api.KK_ERR_INVALID and word in msg, msg


@pytest.mark.parametrize("kw, word", [
    (dict(type=3), "type"), (dict(type=0), "type"), (dict(groups=0), "group count"), (dict(groups=1025), "group count"),
    (dict(entries=-1), "entries"), (dict(entries=(1 << 28) + 1), "entries"), (dict(inputs=0), "inputs"), (dict(inputs=60), "inputs"),
    (dict(inputs=-8), "inputs"), (dict(outputs=0), "outputs"), (dict(gate=3), "gate"), (dict(gate=-1), "gate"), (dict(start=None), "null"),
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"), (dict(x=P + 8), "16-byte"), (dict(w=P + 4), "16-byte"),
    (dict(x_row=65), "16-byte"), (dict(w_row=68), "16-byte"), (dict(w_group=4), "16-byte"), (dict(y=P + 1), "aligned"),
    (dict(start=P + 2), "aligned"), (dict(bias=P + 2), "aligned"), (dict(fault=P + 1), "aligned"), (dict(x_place=P + 2), "aligned"),
    (dict(x_place=P, x_div=0), "x_div"), (dict(x_rows=19), "x has fewer"), (dict(x_place=P, x_div=2, x_rows=0), "x has fewer"),
    (dict(y_rows=19), "y has fewer"), (dict(y_place=P, y_rows=0), "y has fewer"), (dict(y=2 * P), "output is an input")])
def test_expert_refusals(kw, word):
    from kokoro_hip import api
    rc, msg = _call("kk_expert_product", _expert(**kw))
    assert rc == api.KK_ERR_INVALID and word in msg, msg


@pytest.mark.parametrize("kw, word", [
    (dict(type=7), "type"), (dict(top=0), "top"), (dict(top=33), "top"), (dict(rows=-1), "rows"), (dict(rows=1 << 27), "rows"),
    (dict(values=0), "values"), (dict(y=None), "null"), (dict(expert=None), "null"), (dict(weight=None), "null"), (dict(out=None), "null"),
    (dict(y=P + 1), "aligned"), (dict(base=P + 1), "aligned"), (dict(expert=P + 2), "aligned"), (dict(out=P), "output is an input"),
    (dict(out=4 * P, out_row=104), "strides")])
def test_join_refusals(kw, word):
    from kokoro_hip import api
    rc, msg = _call("kk_expert_join", _join(**kw))
    assert rc == api.KK_ERR_INVALID and word in msg, msg


@pytest.mark.parametrize("kw, word", [
    (dict(type=3, out_type=3), "type"), (dict(out_type=2), "type"), (dict(rows=-1), "rows"), (dict(rows=(1 << 24) + 1), "rows"),
    (dict(inputs=4), "inputs"), (dict(outputs=0), "outputs"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"),
    (dict(x=P + 2), "16-byte"), (dict(w_row=66), "16-byte"), (dict(y=P + 1), "aligned"), (dict(out_type=3, y=P + 2), "aligned"),
    (dict(bias=P + 2), "aligned"), (dict(fault=P + 2), "aligned"), (dict(adapters=-1), "adapters"), (dict(rank=0), "rank"),
    (dict(rank=12), "rank"), (dict(rank=264), "rank"), (dict(a=None), "null"), (dict(b=None), "null"), (dict(scale=None), "null"),
    (dict(adapter=None), "null"), (dict(a=P + 8), "16-byte"), (dict(b=P + 8), "16-byte"), (dict(adapter=P + 1), "aligned"),
    (dict(y=P), "output is an input"), (dict(y=2 * P), "output is an input")])
def test_adapter_refusals(kw, word):
    from kokoro_hip import api
    for name in ("kk_adapter_product", "kk_adapter_product_workspace"):
        rc, msg = _call(name, _adapter(**kw))
        assert rc == api.KK_ERR_INVALID and word in msg, msg


@pytest.mark.parametrize("name, args", [
    ("kk_expert_route", {}), ("kk_expert_route", dict(rows=0, logits=None, expert=None, weight=None, place=None)),
    ("kk_expert_product", {}), ("kk_expert_product", dict(entries=0, x=None, y=None, start=None)),
    ("kk_expert_product", dict(x_place=P, x_div=4, x_rows=1, y_place=P, y_rows=1, bias=P + 4)),
    ("kk_expert_join", {}), ("kk_expert_join", dict(rows=0, y=None, out=None)), ("kk_expert_join", dict(base=None, out=4 * P)),
    ("kk_expert_join", dict(out=4 * P)), ("kk_adapter_product", {}), ("kk_adapter_product", dict(rows=0, x=None, y=None, adapter=None)),
    ("kk_adapter_product", dict(adapters=0, rank=0, a=None, b=None, scale=None, adapter=None)), ("kk_adapter_product", dict(out_type=3))])
def test_accepted(name, args):
    from kokoro_hip import api
    make = {"kk_expert_route": _route, "kk_expert_product": _expert, "kk_expert_join": _join, "kk_adapter_product": _adapter}[name]
    assert _call(name, make(**args)) == (api.KK_ERR_INVALID, "null context")


def test_null_arguments():
    from kokoro_hip import api
    for name in ("kk_expert_route", "kk_expert_route_workspace", "kk_expert_product", "kk_expert_join", "kk_adapter_product",
                 "kk_adapter_product_workspace"):
        assert _call(name, None) == (api.KK_ERR_INVALID, "null arguments")
    assert api.lib().kk_expert_join(None, None, None, None, 0) == api.KK_ERR_INVALID  # a message needs no buffer
