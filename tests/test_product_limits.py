"""The sizes that include/kokoro_hip.h names for the products of ragged rows are those that the library takes, on the CPU: the largest of each
gets as far as the missing context, one more is refused."""
import os
import re

import pytest

import test_product_refusals as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _most(struct, field):
    """What the comment beside the field of the struct says: at most 2^n."""
    with open(os.path.join(ROOT, "include", "kokoro_hip.h")) as f:
        text = f.read()
    body = text[:text.index("} " + struct + ";")].rsplit("typedef struct {", 1)[1]
    comment = re.search(r"int32_t " + field + r";\s*/\*(.*?)\*/", body, re.S).group(1)
    return 1 << int(re.search(r"at most 2\^(\d+)", comment).group(1))


@pytest.mark.parametrize("name, struct, make, field, by, more", [
    ("kk_expert_route", "kk_expert_route_args", P._route, "rows", 8, {}),
    ("kk_expert_route", "kk_expert_route_args", P._route, "rows", 1, {"top": 1}),
    ("kk_expert_product", "kk_expert_product_args", P._expert, "entries", 1, {"x_rows": 1 << 30, "y_rows": 1 << 30}),
    ("kk_expert_product", "kk_expert_product_args", P._expert, "inputs", 1, {}),
    ("kk_expert_product", "kk_expert_product_args", P._expert, "outputs", 1, {}),
    ("kk_expert_join", "kk_expert_join_args", P._join, "rows", 4, {}),
    ("kk_expert_join", "kk_expert_join_args", P._join, "values", 1, {}),
    ("kk_adapter_product", "kk_adapter_product_args", P._adapter, "rows", 1, {}),
    ("kk_adapter_product", "kk_adapter_product_args", P._adapter, "inputs", 1, {}),
    ("kk_adapter_product", "kk_adapter_product_args", P._adapter, "outputs", 1, {})])
def test_sizes_of_the_header(name, struct, make, field, by, more):
    from kokoro_hip import api
    most = _most(struct, field) // by
    step = 8 if field == "inputs" else 1
    assert P._call(name, make(**{**more, field: most})) == (api.KK_ERR_INVALID, "null context")
    rc, msg = P._call(name, make(**{**more, field: most + step}))
    assert rc == api.KK_ERR_INVALID and field in msg, msg
