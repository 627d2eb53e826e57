"""GPU parity: norm, rotation and cache write of queries and keys against float64.

Tolerance per element: half a step of the output type relative to the value (2^-8 bf16, 2^-11 float16, 2^-4 E4M3; for
float16 and E4M3 also half of the smallest subnormal, 2^-25 and 2^-10), and 2^-17 of the rotated pair's length for the
fp32 arithmetic in front of it: mean of squares over up to 256 elements by at most 13 dependent additions (13 * 2^-24, half of
it after the root), rsqrt and division (4 * 2^-24), two products (2 * 2^-24), sine and cosine (2 * 2^-24 and 2 pi * 2^-24
of a turn's rounding), products and sum of the rotation (3 * 2^-24): under 32 * 2^-24 = 2^-19, doubled twice for the
pair's two terms and for scales."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from oracle import paged  # noqa: E402

HALF = {torch.bfloat16: (2.0 ** -8, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.float8_e4m3fn: (2.0 ** -4, 2.0 ** -10)}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _near(got, want, length, dtype):
    got = got.double().cpu().numpy()
    rel, absolute = HALF[dtype]
    bad = ~(np.abs(got - want) <= rel * np.abs(want) * (1 + 2.0 ** -10) + absolute + 2.0 ** -17 * length)
    assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])


def _case(tokens, heads, kv_heads, dim, rotary, dtype, *, interleaved=False, cache=None, norm=True, w_dtype=None, page=16, pages=None, seed=0, far=1000,
          magnitude=1.0, order="heads", eps=1e-6, scales=True):
    import cachalot_b200 as cb

    g = _gen(seed)
    x = (torch.randn((tokens, (heads + 2 * kv_heads) * dim), device="cuda", generator=g) * 1.5).to(dtype).view(tokens, heads + 2 * kv_heads, dim)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    qw, kw = ((torch.rand(dim, device="cuda", generator=g) + 0.5).to(w_dtype or dtype) if norm else None for _ in "qk")
    freq = cb.rope_frequencies(rotary)[0] if rotary else torch.zeros(0, dtype=torch.float64, device="cuda")
    pos = torch.randint(0, far, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    kw_args = dict(q_weight=qw, k_weight=kw, eps=eps, interleaved=interleaved, magnitude=magnitude)

    def want(t, w):
        y = t.double().cpu().numpy()
        y = paged.rms_norm(y, None if w is None else w.double().cpu().numpy(), eps) if norm else y
        f = freq.cpu().numpy()
        r = paged.rotate(y, pos.cpu().numpy(), f, interleaved, magnitude)
        # length of each element's pair
        half = len(f)
        length = np.abs(y)
        a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
        length[..., a] = length[..., b] = magnitude * np.hypot(y[..., a], y[..., b])
        return r, length

    wq, wk = want(q, qw), want(k, kw)
    if cache is None:
        y, ko = cb.qk_norm_rope(q, k, pos, freq, **kw_args)
        _near(y, *wq, dtype), _near(ko, *wk, dtype)
        return
    pages = pages or tokens // page + 3
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens].to(torch.int32)
    slots[::5] = -1
    shape = (pages, kv_heads, page, dim) if order == "heads" else (pages, page, kv_heads, dim)
    caches = [torch.randint(0, 100, shape, device="cuda", generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn) if cache == torch.float8_e4m3fn
              else torch.randn(shape, device="cuda", generator=g).to(cache) for _ in "kv"]
    if order != "heads":
        caches = [t.transpose(1, 2) for t in caches]
    ks = vs = None
    if cache == torch.float8_e4m3fn and scales:
        ks, vs = (torch.rand(kv_heads, device="cuda", generator=g) * 0.02 + 0.004 for _ in "kv")  # some values saturate
    raw = torch.uint8 if cache == torch.float8_e4m3fn else torch.int16
    before = [t.contiguous().view(raw).cpu() for t in caches]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y, ko = cb.qk_norm_rope(q, k, pos, freq, v=v, k_cache=caches[0], v_cache=caches[1], slots=slots, k_scale=ks, v_scale=vs, status=status, **kw_args)
    assert ko is None and int(status.item()) == 0
    _near(y, *wq, dtype)
    live = (slots >= 0).cpu().numpy()
    s = slots.cpu().numpy()[live]
    vv = v.double().cpu().numpy()
    for t, old, (w, length), scale in ((caches[0], before[0], wk, ks), (caches[1], before[1], (vv, np.zeros_like(vv)), vs)):
        sc = np.ones(kv_heads) if scale is None else scale.double().cpu().numpy()
        w, length = w[live] / sc[:, None], length[live] / sc[:, None]
        if cache == torch.float8_e4m3fn:
            w = np.clip(w, -448, 448)
        _near(t[torch.from_numpy(s // page).cuda().long(), :, torch.from_numpy(s % page).cuda().long()] if cache != torch.float8_e4m3fn else
              t.view(torch.uint8)[torch.from_numpy(s // page).cuda().long(), :, torch.from_numpy(s % page).cuda().long()].view(cache), w, length, cache)
        now = t.contiguous().view(raw).cpu()
        untouched = torch.ones((pages, page), dtype=torch.bool)
        untouched[s // page, s % page] = False
        m = untouched[:, None, :, None].expand(now.shape)
        assert torch.equal(now[m], old[m])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(8, 8), (24, 24), (64, 64), (80, 20), (96, 96), (96, 2), (128, 64), (128, 128), (192, 64), (200, 130), (256, 256), (64, 0)])
def test_shapes(dim, rotary, interleaved, dtype):
    _case(5, 3, 2, dim, rotary, dtype, interleaved=interleaved, seed=dim + rotary)


@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (1, 64, 16), (2, 17, 1), (67, 9, 3), (700, 4, 2)])
@pytest.mark.parametrize("cache", [None, torch.bfloat16, torch.float8_e4m3fn])
def test_tokens_and_heads(tokens, heads, kv_heads, cache):
    _case(tokens, heads, kv_heads, 128, 64, torch.bfloat16, cache=cache, page=24, seed=tokens)


@pytest.mark.parametrize("order", ["heads", "tokens"])
@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.float8_e4m3fn),
                                         (torch.float16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("dim,page", [(64, 1), (96, 16), (256, 7)])
def test_caches(dim, page, dtype, cache, order):
    _case(19, 6, 2, dim, dim // 2, dtype, cache=cache, page=page, order=order, interleaved=dim == 96, seed=page)


@pytest.mark.parametrize("cache", [None, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("dim,heads,kv_heads,rotary,interleaved", [(64, 3, 1, 64, False), (128, 6, 2, 44, False), (128, 6, 2, 44, True), (192, 7, 1, 114, False),
                                                                  (256, 1, 1, 256, False), (80, 17, 3, 6, True), (128, 20, 4, 128, False)])
def test_many_tokens_of_few_heads(dim, heads, kv_heads, rotary, interleaved, cache):
    """Several tokens share a CTA; their number is no multiple of what a CTA takes."""
    _case(9607, heads, kv_heads, dim, rotary, torch.bfloat16, interleaved=interleaved, cache=cache, page=16, seed=dim)


def test_options():
    _case(9, 4, 2, 128, 128, torch.bfloat16, norm=False)
    _case(9, 4, 2, 128, 128, torch.bfloat16, w_dtype=torch.float32)
    _case(9, 4, 2, 128, 128, torch.float16, magnitude=1.3466, cache=torch.float16)
    _case(9, 4, 2, 128, 128, torch.bfloat16, cache=torch.float8_e4m3fn, scales=False)
    _case(9, 4, 2, 128, 128, torch.bfloat16, eps=1.0)


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(interleaved):
    """A turn is reduced in 64 bits: positions up to 2^31 keep their angle."""
    _case(33, 2, 1, 128, 128, torch.float16, far=2 ** 31 - 1, interleaved=interleaved)


def test_slots_outside_the_cache_are_flagged_and_left_out():
    import cachalot_b200 as cb

    q = torch.randn((3, 2, 64), device="cuda").to(torch.bfloat16)
    cache = [torch.zeros((2, 2, 4, 64), dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    pos, freq = torch.arange(3, dtype=torch.int32, device="cuda"), cb.rope_frequencies(64)[0]
    cb.qk_norm_rope(q, q, pos, freq, v=q, k_cache=cache[0], v_cache=cache[1], slots=torch.tensor([8, -5, 2 ** 31 - 1], dtype=torch.int32, device="cuda"), status=status)
    assert int(status.item()) == 1 and not cache[0].any() and not cache[1].any()


def test_no_tokens_and_zero_heads():
    import cachalot_b200 as cb

    freq = cb.rope_frequencies(64)[0]
    e = torch.empty((0, 4, 64), dtype=torch.bfloat16, device="cuda")
    y, k = cb.qk_norm_rope(e, e[:, :2], torch.empty(0, dtype=torch.int32, device="cuda"), freq)
    assert y.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    z = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")  # a head of zeros: eps keeps it zero
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    y, k = cb.qk_norm_rope(z, z, torch.arange(2, dtype=torch.int32, device="cuda"), freq, q_weight=w, k_weight=w)
    assert not y.any() and not k.any()


@pytest.mark.parametrize("rotary,interleaved", [(16, False), (20, False), (22, False), (20, True), (32, True)])
def test_nan_and_inf_stay_in_their_pair_without_a_norm(rotary, interleaved):
    import cachalot_b200 as cb

    q = torch.randn((2, 3, 64), device="cuda").to(torch.bfloat16)
    pos, freq = torch.arange(1, 3, dtype=torch.int32, device="cuda"), cb.rope_frequencies(rotary)[0]
    clean = cb.qk_norm_rope(q, q, pos, freq, interleaved=interleaved)[0]
    for at, value in ((1, float("nan")), (rotary - 1, float("inf")), (rotary, float("nan")), (rotary + 1, float("inf")), (63, float("nan"))):
        bad = q.clone()
        bad[1, 2, at] = value
        y = cb.qk_norm_rope(bad, bad, pos, freq, interleaved=interleaved)[0]
        mate = at if at >= rotary else at ^ 1 if interleaved else (at + rotary // 2) % rotary
        same = torch.ones(64, dtype=torch.bool, device="cuda")
        same[[at, mate]] = False
        assert torch.equal(y[1, 2, same], clean[1, 2, same]) and torch.equal(y[0], clean[0]) and not torch.isfinite(y[1, 2, [at, mate]]).any()
        if at >= rotary:
            assert torch.equal(y[1, 2, at].isnan(), torch.tensor(value != value, device="cuda"))


def test_nan_and_inf_stay_in_their_head():
    import cachalot_b200 as cb

    q = torch.randn((2, 3, 64), device="cuda").to(torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    pos, freq = torch.arange(2, dtype=torch.int32, device="cuda"), cb.rope_frequencies(64)[0]
    clean = cb.qk_norm_rope(q, q, pos, freq, q_weight=w, k_weight=w)[0]
    bad = q.clone()
    bad[0, 1, 5], bad[1, 2, 7] = float("nan"), float("inf")
    y = cb.qk_norm_rope(bad, bad, pos, freq, q_weight=w, k_weight=w)[0]
    hit = torch.zeros((2, 3), dtype=torch.bool, device="cuda")
    hit[0, 1] = hit[1, 2] = True
    assert torch.equal(y[~hit], clean[~hit]) and y[0, 1].isnan().all() and not y[1, 2].isfinite().all()


def test_layouts_of_the_inputs():
    """Rows that are not 16-byte aligned, int64 positions and strided weights go through the general form: the same bits."""
    import cachalot_b200 as cb

    g = _gen(3)
    wide = torch.randn((7, 5 * 64 + 3), device="cuda", generator=g).to(torch.float16)
    odd = wide[:, 1:1 + 5 * 64].unflatten(1, (5, 64))
    w = torch.rand((64, 2), device="cuda", generator=g).to(torch.float16)[:, 1]
    pos, freq = torch.arange(7, dtype=torch.int32, device="cuda"), cb.rope_frequencies(32)[0]
    a = cb.qk_norm_rope(odd[:, :3], odd[:, 3:], pos.long(), freq, q_weight=w, k_weight=w)
    c = odd.contiguous()
    b = cb.qk_norm_rope(c[:, :3], c[:, 3:], pos, freq, q_weight=w.contiguous(), k_weight=w.contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    t = cb.qk_norm_rope(c.transpose(0, 1).contiguous().transpose(0, 1)[:, :3], c[:, 3:], pos, freq, q_weight=w.contiguous(), k_weight=w.contiguous())
    assert torch.equal(t[0], b[0])


def test_graph_and_stream():
    import cachalot_b200 as cb

    x = torch.randn((4, 6, 128), device="cuda").to(torch.bfloat16)
    pos, freq = torch.arange(4, dtype=torch.int32, device="cuda"), cb.rope_frequencies(128)[0]
    cache = [torch.zeros((2, 2, 4, 128), dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    slots = torch.tensor([0, 5, 2, 7], dtype=torch.int32, device="cuda")
    call = lambda: cb.qk_norm_rope(x[:, :2], x[:, 2:4], pos, freq, v=x[:, 4:], k_cache=cache[0], v_cache=cache[1], slots=slots)[0]  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(call(), want)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    x.mul_(-1), slots.copy_(slots.flip(0))
    graph.replay()
    assert torch.equal(y, call())
    assert torch.equal(cache[1][slots.long() // 4, :, slots.long() % 4], x[:, 4:])


def test_refusals():
    import cachalot_b200 as cb

    freq = cb.rope_frequencies(64)[0]
    x = torch.zeros((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    pos = torch.arange(3, dtype=torch.int32, device="cuda")
    c = torch.zeros((2, 2, 4, 64), dtype=torch.bfloat16, device="cuda")
    s = torch.ones(2, device="cuda")
    full = dict(v=x, k_cache=c, v_cache=c.clone(), slots=pos)
    bad = [((x.float(), x.float(), pos, freq), {}), ((x, x.half(), pos, freq), {}), ((x, x[:2], pos, freq), {}), ((x, x, pos[:2], freq), {}),
           ((x, x, pos, freq.float()), {}), ((x, x, pos, cb.rope_frequencies(66)[0]), {}), ((x, x, pos, freq), dict(q_weight=x[0, 0, :32])),
           ((x, x, pos, freq), dict(q_weight=x[0, 0].half())), ((x, x, pos, freq), dict(q_weight=x[0, 0], k_weight=x[0, 0].float())),
           ((x, x, pos, freq), dict(v=x)), ((x, x, pos, freq), {**full, "slots": None}), ((x, x, pos, freq), {**full, "v_cache": None}),
           ((x, x, pos, freq), {**full, "v": x[:, :1]}), ((x, x, pos, freq), {**full, "k_scale": s}), ((x, x, pos, freq), {**full, "k_cache": c[:1]}),
           ((x, x, pos, freq), {**full, "k_cache": c.half(), "v_cache": c.half()}), ((x[:, :1], x[:, :1], pos, freq), {**full, "v": x[:, :1]}),
           ((x, x, pos, freq), {**full, "k_cache": c.to(torch.float8_e4m3fn), "v_cache": c.to(torch.float8_e4m3fn), "k_scale": s[:1]}),
           ((x.cpu(), x, pos, freq), {}), ((x, x, pos.cpu(), freq), {})]
    for args, kw in bad:
        with pytest.raises(ValueError):
            cb.qk_norm_rope(*args, **kw)
    wide = torch.zeros((1, 1, 264), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(NotImplementedError, match="264"):
        cb.qk_norm_rope(wide, wide, pos[:1], freq)
    with pytest.raises(NotImplementedError, match="20"):
        cb.qk_norm_rope(x[..., :20].contiguous(), x[..., :20].contiguous(), pos, cb.rope_frequencies(20)[0])


def test_int64_slots_beyond_int32():
    import cachalot_b200 as cb

    x = torch.randn((3, 2, 64), device="cuda").to(torch.bfloat16)
    cache = [torch.zeros((2, 2, 4, 64), dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cb.qk_norm_rope(x, x, torch.arange(3, device="cuda"), cb.rope_frequencies(64)[0], v=x, k_cache=cache[0], v_cache=cache[1],
                    slots=torch.tensor([2 ** 32 + 1, -2 ** 32 + 2, 2 ** 31], device="cuda"), status=status)
    assert int(status.item()) == 1 and not cache[0].any() and not cache[1].any()


def test_interleaved_that_has_no_truth_value():
    import cachalot_b200 as cb

    x, pos, freq = torch.zeros((3, 2, 64), dtype=torch.bfloat16, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda"), cb.rope_frequencies(64)[0]
    with pytest.raises((RuntimeError, ValueError)):  # int() of two elements; not an error of the interpreter itself
        cb.qk_norm_rope(x, x, pos, freq, interleaved=torch.ones(2))
    assert not cb.qk_norm_rope(x, x, pos, freq)[0].any()
