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


def test_rope_frequencies():
    import cachalot_b200 as cb

    f, m = cb.rope_frequencies(64, device="cpu")
    assert m == 1.0 and f.dtype == torch.float64 and f.tolist() == [10000.0 ** (-2 * i / 64) for i in range(32)]
    assert torch.allclose(cb.rope_frequencies(64, scaling="linear", factor=4.0, device="cpu")[0], f / 4, rtol=1e-15)
    g, _ = cb.rope_frequencies(64, scaling="ntk", factor=4.0, device="cpu")
    assert g[0] == 1.0 and abs(float(g[-1] / f[-1]) - 0.25) < 1e-12
    y, m = cb.rope_frequencies(64, scaling="yarn", factor=32.0, trained_len=4096, device="cpu")
    assert abs(m - (0.1 * 3.4657359027997265 + 1)) < 1e-12
    turns = f * 4096 / (2 * 3.141592653589793)
    assert torch.equal(y[turns > 33], f[turns > 33]) and torch.allclose(y[turns < 0.75], f[turns < 0.75] / 32, rtol=1e-12)
    assert (y <= f).all() and (y >= f / 32 * (1 - 1e-12)).all()
    for kw in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, scaling="yarn", factor=2.0)):
        with pytest.raises(ValueError):
            cb.rope_frequencies(**kw, device="cpu")


def test_qk_norm_rope_refusals():
    from cachalot_b200 import _lib

    buf = (C.c_int32 * 4096)()
    base = C.addressof(buf) + (-C.addressof(buf)) % 16
    lib, p = _lib.lib, C.c_void_p(base)

    def cache(**kw):
        d = _lib.PagedKV()
        d.k = d.v = base
        d.k_page_stride = d.v_page_stride = 256
        d.k_head_stride, d.v_head_stride = 128, 128
        d.k_token_stride, d.v_token_stride = 64, 64
        d.n_pages, d.page_size, d.kv_heads, d.head_dim, d.dtype = 2, 2, 2, 64, _lib.BF16
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    def call(q=p, qs=128, dtype=_lib.BF16, tokens=1, heads=2, kv=2, dim=64, w=None, wdt=_lib.BF16, pos=p, rot=64, out=p, ko=None, d=None, slots=p, none=False):
        d = None if none else C.byref(d or cache())
        return lib.cachalot_qk_norm_rope(q, qs, 64, p, 128, 64, p, 128, 64, dtype, tokens, heads, kv, dim, w, w, wdt, 1e-6, pos, p, rot, 0, 1.0, out, ko, d, slots,
                                         None, None)

    odd = C.c_void_p(base + 8)
    for kw, rc, word in ((dict(tokens=-1), _lib.EINVAL, "shape"), (dict(dtype=_lib.F32), _lib.EINVAL, "float16"), (dict(dim=264), _lib.EUNSUPPORTED, "264"),
                         (dict(rot=3), _lib.EINVAL, "rotary"), (dict(rot=66), _lib.EINVAL, "rotary"), (dict(w=p, wdt=_lib.F16), _lib.EINVAL, "weights"),
                         (dict(none=True), _lib.EINVAL, "nowhere"), (dict(pos=None), _lib.EINVAL, "null"), (dict(q=odd), _lib.EALIGN, "16-byte"),
                         (dict(qs=12), _lib.EALIGN, "16-byte"), (dict(out=odd), _lib.EALIGN, "16-byte"), (dict(slots=None), _lib.EINVAL, "slots"),
                         (dict(d=cache(k=None)), _lib.EINVAL, "null"), (dict(d=cache(dtype=_lib.F32)), _lib.EINVAL, "cache"),
                         (dict(d=cache(dtype=_lib.F16)), _lib.EINVAL, "differ"), (dict(d=cache(kv_heads=1)), _lib.EINVAL, "holds"),
                         (dict(d=cache(k_token_stride=63)), _lib.EALIGN, "strides"), (dict(d=cache(v_page_stride=-64)), _lib.EALIGN, "strides"),
                         (dict(d=cache(n_pages=2 ** 30)), _lib.EUNSUPPORTED, "slots"), (dict(d=cache(n_pages=0)), _lib.EINVAL, "empty")):
        assert call(**kw) == rc and word in _lib.last_error(), (kw, _lib.last_error())


def test_paged_attention_refusals():
    from cachalot_b200 import _lib

    buf = (C.c_int32 * 4096)()
    base = C.addressof(buf) + (-C.addressof(buf)) % 256
    lib, p = _lib.lib, C.c_void_p(base)

    def call(qs=256, dtype=_lib.BF16, requests=1, heads=4, kv=2, dim=64, cdt=_lib.BF16, table=p, stride=4, width=4, lens=p, window=0, cap=0.0, ws=p, room=1 << 40,
             odt=_lib.BF16, q=p, far=0):
        d = _lib.PagedKV()
        d.k = d.v = base
        d.k_page_stride = d.v_page_stride = 16 * kv * dim
        d.k_head_stride = d.v_head_stride = 16 * dim
        d.k_token_stride = d.v_token_stride = dim
        d.v_page_stride += far
        d.n_pages, d.page_size, d.kv_heads, d.head_dim, d.dtype = 2, 16, kv, dim, cdt
        return lib.cachalot_paged_attention(q, qs, dim, dtype, requests, heads, C.byref(d), table, stride, width, lens, 0.125, window, cap, ws, room, p, odt, None,
                                            None, None)

    for kw, rc, word in ((dict(requests=-1), _lib.EINVAL, "shape"), (dict(dtype=_lib.F32), _lib.EINVAL, "queries"), (dict(odt=_lib.E4M3), _lib.EINVAL, "output"),
                         (dict(heads=5), _lib.EINVAL, "heads"), (dict(cdt=_lib.F16), _lib.EINVAL, "differ"), (dict(window=-1), _lib.EINVAL, "window"),
                         (dict(cap=-1.0), _lib.EINVAL, "softcap"), (dict(cap=float("nan")), _lib.EINVAL, "softcap"), (dict(dim=80), _lib.EUNSUPPORTED, "80"),
                         (dict(far=2 ** 31), _lib.EUNSUPPORTED, "apart"), (dict(table=None), _lib.EINVAL, "null"), (dict(lens=None), _lib.EINVAL, "null"), (dict(ws=None), _lib.EINVAL, "null"),
                         (dict(q=C.c_void_p(base + 2)), _lib.EALIGN, "4-byte"), (dict(qs=255), _lib.EALIGN, "4-byte"),
                         (dict(requests=2, stride=3), _lib.EINVAL, "overlap"), (dict(ws=C.c_void_p(base + 16)), _lib.EALIGN, "256"),
                         (dict(room=1000), _lib.ESCRATCH, "workspace")):
        assert call(**kw) == rc and word in _lib.last_error(), (kw, _lib.last_error())
    assert call(requests=0, lens=None) == _lib.OK
    size = lib.cachalot_paged_attention_workspace_bytes
    assert size(64, 8, 128, _lib.BF16) > 0 and size(64, 8, 80, _lib.BF16) == 0 and size(64, 7, 128, _lib.BF16) == 0 and size(64, 0, 128, _lib.E4M3) == 0


def test_token_logprobs_refusals():
    from cachalot_b200 import _lib

    lib, p = _lib.lib, _p((C.c_int32 * 64)())
    call = lambda x=p, dt=_lib.F32, rows=1, vocab=8, ids=p, top=2, tops=p: lib.cachalot_token_logprobs(x, dt, vocab, rows, vocab, ids, top, p, p, tops, tops, None, None)  # noqa: E731
    for kw, rc, word in ((dict(rows=-1), _lib.EINVAL, "shape"), (dict(vocab=0), _lib.EINVAL, "shape"), (dict(dt=_lib.E4M3), _lib.EINVAL, "float32"),
                         (dict(top=9), _lib.EINVAL, "9 alternatives"), (dict(top=-1), _lib.EINVAL, "alternatives"), (dict(vocab=50, top=33), _lib.EUNSUPPORTED, "33"),
                         (dict(x=None), _lib.EINVAL, "null"), (dict(ids=None), _lib.EINVAL, "null"), (dict(tops=None), _lib.EINVAL, "null"),
                         (dict(x=C.c_void_p(p.value + 2)), _lib.EALIGN, "aligned")):
        assert call(**kw) == rc and word in _lib.last_error(), (kw, _lib.last_error())
    assert call(rows=0, x=None) == _lib.OK


def test_paged_attention_refuses_an_infinite_softcap():
    from cachalot_b200 import _lib

    buf = (C.c_int32 * 4096)()
    base = C.addressof(buf) + (-C.addressof(buf)) % 256
    p, d = C.c_void_p(base), _lib.PagedKV()
    d.k = d.v = base
    d.k_page_stride = d.v_page_stride = 16 * 64
    d.k_head_stride = d.v_head_stride = 16 * 64
    d.k_token_stride = d.v_token_stride = 64
    d.n_pages, d.page_size, d.kv_heads, d.head_dim, d.dtype = 2, 16, 1, 64, _lib.BF16
    # room for no workspace: the call ends before its launch whatever it thinks of the cap
    call = lambda cap: _lib.lib.cachalot_paged_attention(p, 64, 64, _lib.BF16, 1, 1, C.byref(d), p, 2, 2, p, 0.125, 0, cap, p, 0, p, _lib.BF16, None, None, None)  # noqa: E731
    assert call(float("inf")) == _lib.EINVAL and "softcap" in _lib.last_error()
    assert call(1e39) == _lib.EINVAL and call(3e38) == _lib.ESCRATCH and call(0.0) == _lib.ESCRATCH


def test_int64_values_beyond_int32_are_not_wrapped():
    from cachalot_b200 import paged

    wide = torch.tensor([2 ** 32 + 5, -2 ** 40, 7, 2 ** 31 - 1, -2 ** 31, 2 ** 31, 2 ** 63 - 1], dtype=torch.int64)
    got = paged._ints(wide, "lens", (7,))
    assert got.dtype == torch.int32 and got.tolist() == [2 ** 31 - 1, -2 ** 31, 7, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1]
    same = torch.tensor([1, 2], dtype=torch.int32)
    assert paged._ints(same, "lens", (2,)) is same
