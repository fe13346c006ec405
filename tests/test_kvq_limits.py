"""Sizes at and past the limits of the operators over quantised caches: refused on the host."""
import pytest
from test_kvq_capi import gqa, lib, paged  # noqa: F401 (lib: a fixture)


@pytest.mark.parametrize("kw", [
    dict(B=1 << 32, S=1 << 32), dict(B=1 << 62, S=4), dict(B=1, S=1 << 62), dict(cap=1 << 40),
    dict(cap=(1 << 31) - 4097), dict(B=1 << 31, S=1), dict(B=1 << 20, S=1 << 9),
])
def test_slabs(lib, kw):  # noqa: F811
    rc, msg = gqa(lib, **kw)
    assert rc == 1 and "too many rows" in msg, msg


@pytest.mark.parametrize("kw,word", [
    (dict(ctx=1 << 40, blk=1 << 20, maxb=1 << 11), "too many keys"),
    (dict(ctx=(1 << 31) - 4096, blk=1 << 16, maxb=1 << 15), "too many keys"),
    (dict(T=1 << 30), "too many rows"), (dict(batch=1 << 31), "batch shape"),
])
def test_pages(lib, kw, word):  # noqa: F811
    rc, msg = paged(lib, **kw)
    assert rc == 1 and word in msg, msg


def test_workspace_sizes_of_anything(lib):  # noqa: F811
    """No size ends the process; those that a call refuses need nothing."""
    big = (0, -1, 1, 2, 1 << 31, 1 << 32, 1 << 62)
    for f in (lib.ortmi_group_query_attention_quantized_workspace_size,
              lib.ortmi_paged_attention_quantized_workspace_size):
        for x in big:
            for i in range(6):
                args = [3, 2, 4, 2, 64, 4096]
                args[i] = x
                assert f(*args) >= 0
                if x < 0 and i < 5 or x > 1 << 31 and i < 4:
                    assert f(*args) == 0
