"""Argument checks of the paged operators that need no GPU: C ABI refusals and the Python form's on CPU tensors."""
import ctypes as C

import pytest
import torch


def _p(buf):
    return C.cast(buf, C.c_void_p)


def test_paged_descriptor_layout_matches_header():
    from cachalot_b200 import _lib

    assert C.sizeof(_lib.PagedKV) == 4 * 8 + 6 * 8 + 5 * 4 + 4


def test_plan_pages_refusals():
    from cachalot_b200 import _lib

    lib, p = _lib.lib, _p((C.c_int32 * 64)())
    call = lambda r=2, stride=4, width=4, n_free=4, page=16, tokens=4, ctx=p, free=p, out=p: lib.cachalot_plan_pages(  # noqa: E731
        ctx, p, r, p, stride, width, free, n_free, p, page, tokens, out, p, p, p, p, p, None, None)
    for kw, word in ((dict(r=-1), "negative"), (dict(tokens=-1), "negative"), (dict(page=0), "page_size"), (dict(ctx=None), "null"),
                     (dict(free=None), "null"), (dict(out=None), "null"), (dict(stride=3), "overlap")):
        assert call(**kw) == _lib.EINVAL and word in _lib.last_error(), kw
    assert call(r=8193) == _lib.EUNSUPPORTED


def test_cpu_tensors_are_refused():
    import cachalot_b200 as cb

    t = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensors"):
        cb.plan_pages(t, t, t.reshape(2, 1), t, t[:1], page_size=16, tokens=2)
