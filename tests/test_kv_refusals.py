"""What the cache operators refuse, on the CPU: every argument check runs before the context and the device are looked at, so a
call without a context shows its message (and one whose arguments are fine shows that there is no context)."""
import ctypes as C

import pytest

P = 1 << 20  # a number that passes as a device pointer: nothing is read from it


def _call(name, *args):
    from kokoro_hip import api
    err = C.create_string_buffer(512)
    tail = () if name.endswith("workspace") else (None,)
    rc = getattr(api.lib(), name)(None, *(C.byref(a) if a is not None else None for a in args), *tail, err, 512)
    return rc, err.value.decode()


def _rope(**kw):
    from kokoro_hip import api
    base = dict(type=api.BF16, dim=128, rows=4, q_heads=8, k_heads=2, q=P, q_row=1280, q_head=128, k=2 * P, k_row=1280,
                k_head=128, q_out=3 * P, q_out_row=1024, q_out_head=128, k_out=4 * P, k_out_row=256, k_out_head=128, norm=1,
                eps=1e-6, pos=5 * P, rot=128, theta=1e4)
    return api.NormRope(**{**base, **kw})


def _cache(**kw):
    from kokoro_hip import api
    return api.KvCache(**{**dict(type=api.KV_INT8, heads=2, dim=128, pages=9, k=P, v=2 * P, k_scale=3 * P, v_scale=4 * P), **kw})


def _batch(**kw):
    from kokoro_hip import api
    base = dict(n=2, rows=10, max_new=5, max_len=300, row_start=5 * P, len=6 * P, table=7 * P, table_width=5, table_stride=5)
    return api.KvBatch(**{**base, **kw})


def _rows(**kw):
    from kokoro_hip import api
    return api.KvRows(**{**dict(type=api.BF16, k=8 * P, k_row=256, k_head=128, v=9 * P, v_row=256, v_head=128), **kw})


def _attn(**kw):
    from kokoro_hip import api
    base = dict(type=api.F16, heads=8, q=8 * P, q_row=1024, q_head=128, out=9 * P, out_row=1024, out_head=128, scale=0.1,
                causal=1, window=0, workspace=10 * P, workspace_bytes=1 << 40)
    return api.KvAttention(**{**base, **kw})


@pytest.mark.parametrize("kw, word", [
    (dict(type=0), "type"), (dict(type=4), "type"), (dict(dim=0), "dimension"), (dict(dim=127), "dimension"),
    (dict(dim=514), "dimension"), (dict(rows=-1), "rows"), (dict(rows=(1 << 28) + 1), "rows"), (dict(q_heads=-1), "head count"),
    (dict(k_heads=5000), "head count"), (dict(rot=130), "rot"), (dict(rot=63), "rot"), (dict(rot=-2), "rot"),
    (dict(norm=2), "norm"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(interleaved=3), "interleaved"),
    (dict(theta=0.0), "theta"), (dict(theta=float("inf")), "theta"), (dict(q=None), "null"), (dict(k_out=None), "null"),
    (dict(pos=None), "null"), (dict(q=P + 1), "aligned"), (dict(q_weight=P + 2), "aligned"), (dict(freq=P + 4), "aligned"),
    (dict(q_out=P), "strides"), (dict(k_out=2 * P), "strides"),
])
def test_norm_rope_refusals(kw, word):
    from kokoro_hip import api
    rc, msg = _call("kk_qk_norm_rope", _rope(**kw))
    assert rc == api.KK_ERR_INVALID and word in msg, msg


@pytest.mark.parametrize("kw", [{}, dict(rows=0, q=None, k=None, pos=None), dict(q_heads=0, q=None, q_out=None),
                                dict(theta=-1.0, freq=P), dict(theta=-1.0, rot=0), dict(norm=0, eps=-1.0),
                                dict(q_out=P, q_out_row=1280), dict(q_weight=P + 4, k_weight=P + 8)])
def test_norm_rope_accepts(kw):
    assert _call("kk_qk_norm_rope", _rope(**kw))[1] == "null context"


CACHE = [(dict(type=0), "cache type"), (dict(type=3), "cache type"), (dict(dim=80), "dimension"), (dict(dim=512), "dimension"),
         (dict(heads=0), "head count"), (dict(heads=5000), "head count"), (dict(pages=0), "pages"), (dict(k=None), "null"),
         (dict(v_scale=None), "null"), (dict(k=P + 8), "16-byte"), (dict(v=P + 4), "16-byte"), (dict(k_scale=P + 2), "aligned"),
         (dict(fault=P + 1), "aligned")]
BATCH = [(dict(n=-1), "sequence count"), (dict(n=(1 << 20) + 1), "sequence count"), (dict(rows=-1), "rows"),
         (dict(max_new=-1), "rows"), (dict(max_len=-1), "max_len"), (dict(max_len=321), "width"),
         (dict(table_width=-1), "width"), (dict(max_len=(1 << 30) + 64, table_width=1 << 25), "max_len"),
         (dict(row_start=None), "null"), (dict(len=None), "null"), (dict(table=None), "null"), (dict(len=P + 2), "aligned")]


@pytest.mark.parametrize("cache, batch, word", [(c, {}, w) for c, w in CACHE] + [({}, b, w) for b, w in BATCH])
def test_cache_and_batch_refusals(cache, batch, word):
    from kokoro_hip import api
    c, b = _cache(**cache), _batch(**batch)
    for name, last in (("kk_kv_write", _rows()), ("kk_kv_read", _rows()), ("kk_kv_attention", _attn()),
                       ("kk_kv_attention_workspace", _attn())):
        rc, msg = _call(name, c, b, last)
        assert rc == api.KK_ERR_INVALID and word in msg, (name, msg)


@pytest.mark.parametrize("kw, word", [(dict(type=9), "type"), (dict(k=None), "null"), (dict(v=None), "null"),
                                      (dict(k=P + 1), "aligned"), (dict(type=3, v=P + 2), "aligned")])
def test_rows_refusals(kw, word):
    from kokoro_hip import api
    for name in ("kk_kv_write", "kk_kv_read"):
        rc, msg = _call(name, _cache(), _batch(), _rows(**kw))
        assert rc == api.KK_ERR_INVALID and word in msg, msg


@pytest.mark.parametrize("kw, word", [
    (dict(type=3), "type"), (dict(heads=0), "multiple"), (dict(heads=7), "multiple"), (dict(heads=8192), "multiple"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(causal=2), "causal"),
    (dict(window=-1), "window"), (dict(window=(1 << 30) + 1), "window"), (dict(window=5, causal=0), "causal"),
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(q=P + 1), "aligned"), (dict(out=8 * P), "queries")])
def test_attention_refusals(kw, word):
    from kokoro_hip import api
    for name in ("kk_kv_attention", "kk_kv_attention_workspace"):
        rc, msg = _call(name, _cache(), _batch(), _attn(**kw))
        assert rc == api.KK_ERR_INVALID and word in msg, msg


def test_null_arguments():
    from kokoro_hip import api
    assert _call("kk_qk_norm_rope", None) == (api.KK_ERR_INVALID, "null arguments")
    for name, last in (("kk_kv_write", _rows()), ("kk_kv_read", _rows()), ("kk_kv_attention", _attn()),
                       ("kk_kv_attention_workspace", _attn())):
        for args in ((None, _batch(), last), (_cache(), None, last), (_cache(), _batch(), None)):
            assert _call(name, *args) == (api.KK_ERR_INVALID, "null arguments")
        assert _call(name, _cache(), _batch(), last) == (api.KK_ERR_INVALID, "null context")
        # nothing to do is no reason to refuse null arrays
        empty = _batch(rows=0, row_start=None, len=None, table=None)
        assert _call(name, _cache(), empty, last) == (api.KK_ERR_INVALID, "null context")
    # a message needs no buffer
    assert api.lib().kk_kv_write(None, None, None, None, None, None, 0) == api.KK_ERR_INVALID
