"""GPU parity: decode attention over a paged cache against float64.

Tolerance per output element, with spread = sum p |v| / sum p of the element's head:
  * a score carries at most dim * 2^-22 of its sum of magnitudes (fp32 accumulation of exact products, in the tensor core's
    order, and the scaling; `reach` bounds it) and, under a soft cap, cap * 2^-18 of the approximate exp and reciprocal;
    a bf16 query over an E4M3 cache is held in f16 relative to its largest element (2^-24 of it per element, under dim
    times reach * 2^-24): e^d - 1 <= 2 d of every weight, in the sum above and below: 4 d * spread;
  * a weight is rounded to the matrix type: over a 16-bit cache twice, the second time what the first left (half a step of half
    a step: 2^-16 bf16, 2^-22 f16, of spread), over an E4M3 cache once to f16 (2^-11); in f16 also 2^-25 absolute on weights
    that are shifted by 2^7 over the running maximum: 2^-32 of floor = sum |v| / sum p;
  * exp2 and the fp32 sums: 2^-16 of spread;
  * the result is rounded: half a step of the output type (none for float32).
lse: the scores' d, 2^-16 for the sum of weights, 2^-22 of the value."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from oracle import paged  # noqa: E402

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Case:
    def __init__(self, lens, heads, kv_heads, dim, page, dtype=BF16, cache=None, *, seed=0, order="heads", width=None, hidden="nan", q_scale=2.0, scales=True):
        g = _gen(seed)
        self.page, self.dim, self.heads, self.kv_heads = page, dim, heads, kv_heads
        used = [-(-n // page) for n in lens]
        width = max(max(used), 1) if width is None else width
        pages = sum(used) + 3
        perm = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        self.table = torch.full((len(lens), width), 2 ** 30, dtype=torch.int32, device="cuda")  # entries that no visible token needs
        at = 0
        for r, n in enumerate(used):
            self.table[r, :n] = perm[at:at + n]
            at += n
        self.lens = _int(list(lens))
        cache = cache or dtype
        shape = (pages, kv_heads, page, dim) if order == "heads" else (pages, page, kv_heads, dim)
        self.scales = [None, None]
        self.caches = []
        for i in range(2):
            x = torch.randn(shape, device="cuda", generator=g)
            if cache == E4M3:
                x = x * 40
                if scales:
                    self.scales[i] = (torch.rand(kv_heads, device="cuda", generator=g) + 0.5) / 40
            x = x.to(cache)
            self.caches.append(x if order == "heads" else x.transpose(1, 2))
        self.q = (torch.randn((len(lens), heads, dim), device="cuda", generator=g) * q_scale).to(dtype)
        if hidden == "nan":  # everything that is not a visible token
            seen = torch.zeros((pages, page), dtype=torch.bool, device="cuda")
            for r, n in enumerate(lens):
                j = torch.arange(n, device="cuda")
                seen[self.table[r, (j // page).long()].long(), (j % page).long()] = True
            for x in self.caches:
                if cache == E4M3:
                    x.view(torch.uint8)[(~seen)[:, None, :, None].expand(x.shape)] = 0x7F
                else:
                    x[(~seen)[:, None, :, None].expand(x.shape)] = float("nan")

    def run(self, **kw):
        import cachalot_b200 as cb

        return cb.paged_attention(self.q, *self.caches, self.table, self.lens, k_scale=self.scales[0], v_scale=self.scales[1], **kw)

    def want(self, scale=None, window=0, softcap=0.0):
        kv = []
        for x, s in zip(self.caches, self.scales):
            x = x.double() if x.dtype != E4M3 else x.float().double()
            kv.append((x if s is None else x * s.double()[:, None, None]).cpu().numpy())
        return paged.paged_attention(self.q.double().cpu().numpy(), *kv, self.table.cpu().numpy(), self.lens.tolist(), self.page,
                                     self.dim ** -0.5 if scale is None else scale, window, softcap)

    def check(self, status=0, out_dtype=None, **kw):
        word = _int([0])
        out, lse = self.run(want_lse=True, status=word, out_dtype=out_dtype, **kw)
        assert int(word.item()) == status
        assert out.dtype == (out_dtype or self.q.dtype) and lse.dtype == F32
        self.compare(out, lse, self.want(**kw), kw.get("softcap", 0.0))
        return out, lse

    def compare(self, out, lse, want, softcap=0.0):
        wout, wlse, spread, reach, floor = want
        f16 = self.caches[0].dtype != BF16
        d = (self.dim * 2.0 ** -22 * reach + softcap * 2.0 ** -18 + (self.dim * 2.0 ** -24 * reach if self.caches[0].dtype == E4M3 else 0))
        weight = {BF16: 2.0 ** -16, F16: 2.0 ** -22, E4M3: 2.0 ** -11}[self.caches[0].dtype]
        tol = (4 * d[..., None] + 2.0 ** -16 + weight) * spread + (2.0 ** -32 * floor if f16 else 0)
        tol = tol + HALF[out.dtype] * (np.abs(wout) + tol) + (2.0 ** -25 if out.dtype == F16 else 0)
        got = out.double().cpu().numpy()
        bad = ~(np.abs(got - wout) <= tol)
        assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], wout[bad][:4], tol[bad][:4])
        got = lse.double().cpu().numpy()
        empty = wlse == -np.inf
        assert np.array_equal(got == -np.inf, empty)
        err = np.abs(got[~empty] - wlse[~empty])
        assert (err <= d[~empty] + 2.0 ** -16 + 2.0 ** -22 * np.abs(wlse[~empty])).all(), err.max()


EDGES = [1, 2, 7, 8, 9, 15, 16, 17, 63, 64, 65, 129, 0, 300]


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 7])
def test_types_and_head_sizes(dim, dtype, cache, page):
    Case(EDGES, 6, 2, dim, page, dtype, cache, seed=dim).check()


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 5, 8, 9, 16, 17, 24, 33, 40, 64, 65, 130])
def test_groups(group, dim, cache):
    Case([1, 40, 200, 0], 2 * group, 2, dim, 8, BF16, cache, seed=group).check()


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("dim", [96, 192])
@pytest.mark.parametrize("group", [9, 16, 17, 24, 48, 56, 70])
def test_groups_of_other_head_sizes(group, dim, cache):
    Case([1, 40, 200, 0], 2 * group, 2, dim, 16, BF16, cache, seed=group).check()


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)])
@pytest.mark.parametrize("dim,group", [(64, 8), (96, 3), (128, 1), (128, 13), (192, 9), (256, 16)])
def test_many_short_requests(dim, group, dtype, cache):
    lens = (EDGES * 6)[:80]
    Case(lens, 8 * group, 8, dim, 16, dtype, cache, seed=dim).check()
    Case(lens, 8 * group, 8, dim, 24, dtype, cache, seed=dim).check(window=33, softcap=20.0)


def test_more_requests_than_a_warp_adds_up_at_once():
    lens = [(i * 37) % 23 for i in range(700)]
    Case(lens, 8, 2, 64, 8, BF16, BF16, seed=3).check()
    Case([0] * 600 + [5] + [0] * 99 + [300], 8, 2, 64, 8, BF16, E4M3, seed=3).check()
    Case([0, 1, 2] * 800, 2, 2, 64, 8, F16, F16, seed=3).check()


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 40, 64, 100, 256])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_pages(page, order):
    Case(EDGES, 8, 2, 128, page, order=order, seed=page).check()


@pytest.mark.parametrize("window", [1, 2, 8, 15, 16, 17, 64, 100, 1000])
@pytest.mark.parametrize("page", [5, 8, 64])
def test_windows(window, page):
    Case(EDGES, 8, 2, 64, page, F16, seed=window).check(window=window)


def test_pages_before_the_window_are_not_looked_at():
    c = Case([200, 130], 4, 2, 64, 16, seed=1)
    c.table[0, :11] = -1                                   # the window of 16 begins at token 184, on page 11
    c.table[1, :7] = 2 ** 30                               # ... at token 114, on page 7
    out, lse = c.check(window=16)
    assert torch.isfinite(lse).all()


@pytest.mark.parametrize("softcap", [0.5, 30.0])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_softcap_and_scale(softcap, cache):
    Case(EDGES, 6, 2, 128, 16, BF16, cache, q_scale=4.0).check(softcap=softcap)
    Case(EDGES, 6, 2, 128, 16, BF16, cache).check(scale=0.3)
    Case(EDGES, 6, 2, 128, 16, BF16, cache).check(scale=-0.05)


def test_out_types_and_no_scales():
    for dt in (BF16, F16, F32):
        Case([5, 100], 8, 2, 128, 16, BF16).check(out_dtype=dt)
        Case([5, 100], 8, 2, 128, 16, F16, E4M3, scales=False).check(out_dtype=dt, scale=2.0 ** -11)


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("lens", [[30000], [20000, 1, 0, 900, 64], [1000] * 9, [3] * 700])
def test_work_that_crosses_ctas(lens, cache):
    Case(lens, 8, 2, 64 if len(lens) > 100 else 128, 16, BF16, cache, seed=len(lens)).check()


def test_large_groups_of_a_long_request():
    Case([5000, 77], 40, 1, 128, 16).check()
    Case([5000, 77], 24, 1, 256, 16).check()


def test_scores_that_grow_and_shrink():
    """The running maximum moves rarely, often, and by more than its slack: keys along the query with a ramp."""
    for sign in (1, -1):
        for dtype, cache in ((BF16, BF16), (F16, F16), (BF16, E4M3)):
            c = Case([2000], 2, 2, 64, 16, dtype, cache, hidden="", scales=False)
            ramp = torch.linspace(-1, 1, 2000, device="cuda") * sign
            j = torch.arange(2000, device="cuda")
            q = torch.ones((1, 2, 64), device="cuda", dtype=dtype)
            keys = (ramp[:, None, None] * torch.ones((2000, 2, 64), device="cuda")).to(cache)
            c.caches[0].view(torch.uint8 if cache == E4M3 else cache)[c.table[0, (j // 16).long()].long(), :, (j % 16).long()] = keys.view(torch.uint8) if cache == E4M3 else keys
            c.q.copy_(q)
            c.check(scale=2.0)


def test_small_weights_of_many_tokens_count():
    """One token far above 60000 others that together weigh as much: weights of 2^-16 in f16 keep their precision."""
    n = 60000
    for dtype, cache in ((F16, F16), (BF16, E4M3), (BF16, BF16)):
        c = Case([n], 1, 1, 64, 64, dtype, cache, hidden="", scales=False)
        keys = torch.zeros((n, 1, 64), device="cuda")
        keys[7] = 1.375
        j = torch.arange(n, device="cuda")
        kc = keys.to(cache)
        c.caches[0].view(torch.uint8 if cache == E4M3 else cache)[c.table[0, (j // 64).long()].long(), :, (j % 64).long()] = kc.view(torch.uint8) if cache == E4M3 else kc
        c.q.fill_(1.0)
        c.check(scale=0.125)


def test_rows_without_keys_and_hidden_pages():
    c = Case([0, 40, 0], 4, 2, 128, 16)
    out, lse = c.check()
    assert not out[0].any() and not out[2].any() and (lse[0] == -float("inf")).all()
    c = Case([64, 64, 20], 4, 2, 128, 16)
    c.table[0, 1], c.table[1, :], c.table[2, 0] = -1, 10 ** 6, -5
    out, lse = c.check(status=1)
    assert not out[1].any() and (lse[1] == -float("inf")).all()
    c = Case([64, 20], 4, 2, 128, 5)                        # pages that are no multiple of 8
    c.table[0, 1] = -1
    c.check(status=1)


def test_lengths_past_the_table_and_negative():
    c = Case([64, 30], 4, 2, 64, 16)
    c.lens.copy_(_int([1000, -3]))
    out, _ = c.check(status=32)
    assert not out[1].any()


def test_scores_of_minus_infinity():
    c = Case([20, 20], 2, 2, 64, 16, hidden="")
    c.q.fill_(1.0)
    pages = c.table[0, :2].long()
    c.caches[0][pages] = -float("inf")
    out, lse = c.run(want_lse=True)
    assert not out[0].any() and (lse[0] == -float("inf")).all() and torch.isfinite(out[1].float()).all()
    c.caches[0][pages[0], :, 3] = 0.5                        # one that counts: its value alone
    out, lse = c.run(want_lse=True)
    assert torch.equal(out[0], c.caches[1][pages[0], :, 3]) and torch.allclose(lse[0], torch.full_like(lse[0], 4.0))


def test_nan_of_a_visible_token_reaches_its_heads_only():
    c = Case([50, 50], 4, 2, 64, 16)
    clean = c.run()
    c.caches[1][c.table[0, 0].long(), 1, 3, 5] = float("nan")
    out = c.run()
    assert out[0, 2:, 5].isnan().all()
    out[0, 2:, 5] = clean[0, 2:, 5]
    assert torch.equal(out, clean)


def test_offsets_beyond_32_bits():
    """Pages at the far end of caches of 5 GB each, by both operators that address them."""
    import cachalot_b200 as cb

    pages, heads, page, dim = 40000, 8, 64, 256
    k, v = (torch.empty((pages, heads, page, dim), dtype=torch.uint8, device="cuda").view(E4M3) for _ in "kv")
    table = _int([[pages - 1, 3, pages - 2]])
    x = torch.randn((150, 3 * heads, dim), device="cuda").to(BF16)
    j = torch.arange(150, device="cuda")
    slots = (table[0, j // page] * page + j % page).to(torch.int32)
    cb.qk_norm_rope(x[:, :heads], x[:, heads:2 * heads], j.to(torch.int32), cb.rope_frequencies(64)[0], v=x[:, 2 * heads:], k_cache=k, v_cache=v, slots=slots)
    q = torch.randn((1, heads, dim), device="cuda").to(BF16)
    got = cb.paged_attention(q, k, v, table, _int([150]))
    near = [t.view(torch.uint8)[table[0].long()].clone().view(E4M3) for t in (k, v)]
    assert torch.equal(got, cb.paged_attention(q, *near, _int([[0, 1, 2]]), _int([150])))
    assert (near[1].float()[0, :, :5] - x[:5, 2 * heads:].transpose(0, 1).float()).abs().max() < 0.5 and got.abs().max() > 0


def test_strided_inputs_and_general_form():
    c = Case([33, 70], 8, 2, 128, 16)
    want = c.run()
    wide = torch.zeros((2, 8, 2, 128), dtype=BF16, device="cuda")
    wide[:, :, 1] = c.q
    c.q = wide[:, :, 1]
    assert torch.equal(c.run(), want)
    store = torch.full((2, c.table.shape[1] + 5), 9, dtype=torch.int32, device="cuda")
    store[:, :c.table.shape[1]] = c.table
    c.table = store[:, :c.table.shape[1]]
    assert torch.equal(c.run(), want)
    odd = torch.zeros(2 * 8 * 128 + 1, dtype=BF16, device="cuda")
    odd[1:] = c.q.reshape(-1)
    c.q, c.lens = odd[1:].view(2, 8, 128), c.lens.long()
    assert torch.equal(c.run(), want)


def test_same_bits_every_time():
    c = Case([9000, 1, 500, 64], 16, 2, 128, 16, hidden="")
    want = c.run(want_lse=True)
    for _ in range(20):
        got = c.run(want_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_many_requests_replayed_with_other_lengths():
    """The form of the call is chosen by what the table holds; the lengths may become anything up to that."""
    c = Case([160] * 90, 32, 8, 64, 16, seed=9)
    c.run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = c.run(want_lse=True)
    for lens in ([160] * 90, [0] * 90, [(7 * i) % 161 for i in range(90)], [0] * 89 + [160]):
        c.lens.copy_(_int(lens))
        g.replay()
        torch.cuda.synchronize()
        c.compare(out, lse, c.want())


def test_graphs_and_streams():
    """Two captured calls replayed at the same time on two streams, with lengths that changed after the capture."""
    a, b = Case([3000, 100], 16, 2, 128, 16, seed=1), Case([10, 4000], 16, 2, 128, 16, BF16, E4M3, seed=2)
    a.run(), b.run()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.run(want_lse=True))
        graphs.append(g)
    a.lens.copy_(_int([2001, 64])), b.lens.copy_(_int([0, 3999]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c, o in zip((a, b), outs):
        c.compare(*o, c.want())


def test_no_requests():
    c = Case([5], 4, 2, 64, 16)
    import cachalot_b200 as cb

    out, lse = cb.paged_attention(c.q[:0], *c.caches, c.table[:0], c.lens[:0], want_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_refusals():
    import cachalot_b200 as cb

    c = Case([5, 9], 4, 2, 64, 16)
    k, v = c.caches
    one = torch.ones(2, device="cuda")
    bad = [((c.q.float(), k, v, c.table, c.lens), {}), ((c.q.half(), k, v, c.table, c.lens), {}), ((c.q[:, :3], k, v, c.table, c.lens), {}),
           ((c.q[..., :32], k, v, c.table, c.lens), {}), ((c.q, k, v[:1], c.table, c.lens), {}), ((c.q, k, v.half(), c.table, c.lens), {}),
           ((c.q, k, v, c.table[:1], c.lens), {}), ((c.q, k, v, c.table.long(), c.lens), {}), ((c.q, k, v, c.table, c.lens[:1]), {}),
           ((c.q, k, v, c.table, c.lens.float()), {}), ((c.q[0], k, v, c.table, c.lens), {}), ((c.q, k, v, c.table, c.lens), dict(window=-1)),
           ((c.q, k, v, c.table, c.lens), dict(softcap=-1.0)), ((c.q, k, v, c.table, c.lens), dict(softcap=float("nan"))),
           ((c.q, k, v, c.table, c.lens), dict(k_scale=one)), ((c.q, k, v, c.table, c.lens), dict(out_dtype=torch.float64)),
           ((c.q, k.transpose(2, 3), v.transpose(2, 3), c.table, c.lens), {}), ((c.q.cpu(), k, v, c.table, c.lens), {}),
           ((c.q, k, v, c.table.cpu(), c.lens), {}), ((c.q, k, v, c.table, c.lens), dict(window=2 ** 32))]
    for args, kw in bad:
        with pytest.raises(ValueError):
            cb.paged_attention(*args, **kw)
    n = torch.zeros((2, 2, 16, 48), dtype=BF16, device="cuda")
    with pytest.raises(NotImplementedError, match="head size 48"):
        cb.paged_attention(torch.zeros((2, 4, 48), dtype=BF16, device="cuda"), n, n.clone(), c.table, c.lens)


NAN_CACHES = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)]


def _set_keys(c, request, tokens, head, value):
    """Element 5 of these keys of one key-value head."""
    at = c.table[request].long()
    raw = c.caches[0].view(torch.uint8) if c.caches[0].dtype == E4M3 else c.caches[0]
    raw[at[tokens // c.page], head, tokens % c.page, 5] = (0x7F if c.caches[0].dtype == E4M3 else value)


def _nan_where(c, hit, **kw):
    """NaN for these (request, head) pairs, in every element and in the log sum exp; returns what the call gave."""
    out, lse = c.run(want_lse=True, **kw)
    assert out[hit].isnan().all() and lse[hit].isnan().all()
    return out, lse


# a unit of a CTA, of several, of CTAs of one warp; a last tile of one token
NAN_LENS = {"whole": [40, 1, 65, 0], "joined": [20001, 33], "one warp": [i % 50 for i in range(90)]}


@pytest.mark.parametrize("lens", NAN_LENS)
@pytest.mark.parametrize("dtype,cache", NAN_CACHES)
def test_nan_in_a_query_makes_its_head_nan(dtype, cache, lens):
    c = Case(NAN_LENS[lens], 16, 8, 64, 16, dtype, cache, hidden="")
    for kw in ({}, dict(softcap=5.0)):
        clean, want, keep = c.run(want_lse=True, **kw), c.want(**kw), c.q.clone()
        c.q[0, 3, 7] = c.q[1, 9, 63] = float("nan")
        hit = torch.zeros(c.q.shape[:2], dtype=torch.bool, device="cuda")
        hit[0, 3], hit[1, 9] = c.lens[0] > 0, c.lens[1] > 0
        got = _nan_where(c, hit, **kw)
        c.q = keep
        for a, b in zip(got, clean):  # the others are right, though not the clean call's bits: heads of a unit move their maxima together
            a[hit] = b[hit]
        c.compare(*got, want, kw.get("softcap", 0.0))


@pytest.mark.parametrize("which", ["first", "last", "many", "whole tiles", "all"])
@pytest.mark.parametrize("lens", NAN_LENS)
@pytest.mark.parametrize("dtype,cache", NAN_CACHES)
def test_nan_in_keys_reaches_the_log_sum_exp(dtype, cache, lens, which):
    c = Case(NAN_LENS[lens], 16, 8, 64, 16, dtype, cache, hidden="")
    clean = c.run(want_lse=True)
    hit = torch.zeros(c.q.shape[:2], dtype=torch.bool, device="cuda")
    for r, n in enumerate(NAN_LENS[lens]):
        if r % 3 == 2 and lens == "one warp" or n == 0:
            continue
        tokens = torch.arange(*{"first": (0, 1), "last": (n - 1, n), "many": (n // 2, n), "whole tiles": (n // 2 // 128 * 128, n), "all": (0, n)}[which], device="cuda")
        _set_keys(c, r, tokens, 2, float("nan"))
        hit[r, 4:6] = True
    got = _nan_where(c, hit)
    assert all(torch.equal(a[~hit], b[~hit]) for a, b in zip(got, clean))


def test_an_infinite_softcap_is_refused():
    import cachalot_b200 as cb

    c = Case([5, 9], 4, 2, 64, 16)
    for lens in (c.lens, c.lens.long()):  # the native call path and the general form
        for cap in (float("inf"), 1e39):
            with pytest.raises(ValueError, match="softcap"):
                cb.paged_attention(c.q, *c.caches, c.table, lens, softcap=cap)


@pytest.mark.parametrize("softcap", [1e-3, 0.5, 8.0, 50.0, 1e3, 1e4, 1e5, 1e30, 3e38])
@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (F16, E4M3)])
def test_softcap_is_as_accurate_as_the_scores(dtype, cache, softcap):
    """The error that the cap adds is relative to the capped score, whatever the cap.  Up to 0.4 of the cap a series of five
    terms: what is left out is 0.009 z^10 < 2^-19.9, its roundings (in terms of z^2 / 3 and less) below 2^-22.  Above, with x = |z|, 1 - 2 / (1 +
    e^2x): the exponential's 2^-22 times the slope, at most 1/2; its argument, 2^-23 times x / cosh^2 x < 0.45; the sum's 2^-24 and the
    reciprocal's 2^-23 of at most 1; the last rounding 2^-25: 2^-21.3 of the cap, which is less than 2^-19 of a score that is capped to
    0.37 of it or more.  A capped score is below `reach`, and the derivative of the cap at most 1: reach * 2^-18 on top of what an
    uncapped score carries."""
    for q_scale in (2.0, 0.02):
        c = Case([1, 2, 40, 300, 0], 6, 2, 64, 16, dtype, cache, q_scale=q_scale, seed=5)
        for scale in (None, -0.2):
            out, lse = c.run(want_lse=True, softcap=softcap, out_dtype=F32, scale=scale)
            want = c.want(softcap=softcap, scale=scale)
            c.compare(out, lse, want, want[3])


def test_softcap_keeps_the_order_of_scores_around_the_border():
    """Where the two forms meet, z = 0.4: one key each, so the log sum exp is the capped score itself."""
    c = Case([1] * 64, 1, 1, 64, 16, F16)
    c.q.zero_()
    c.q[:, 0, 0] = torch.linspace(0.3, 0.5, 64, device="cuda").to(F16)
    for sign in (1.0, -1.0):
        c.caches[0].zero_()
        c.caches[0][..., 0] = sign
        _, lse = c.run(want_lse=True, softcap=1.0, scale=1.0)
        want = torch.tanh(c.q[:, 0, 0].double() * sign)
        assert ((lse[:, 0].double() - want).abs() <= 2.0 ** -18 * want.abs() + 2.0 ** -22).all()
        assert (lse[1:, 0] * sign >= lse[:-1, 0] * sign).all()


def test_int64_lengths_beyond_int32():
    import cachalot_b200 as cb

    c = Case([64, 30], 4, 2, 64, 16)
    word = _int([0])
    out = cb.paged_attention(c.q, *c.caches, c.table, torch.tensor([2 ** 32 + 5, -2 ** 32 - 3], device="cuda"), status=word)
    want = cb.paged_attention(c.q, *c.caches, c.table, _int([64, 0]))
    assert torch.equal(out, want) and int(word.item()) == 32


def test_want_lse_that_has_no_truth_value():
    c = Case([5], 4, 2, 64, 16)
    with pytest.raises(RuntimeError, match="ambiguous"):
        c.run(want_lse=torch.ones(2))
    assert torch.isfinite(c.run().float()).all()


@pytest.mark.parametrize("dim,group,page", [(64, 3, 16), (128, 9, 16), (128, 20, 8), (96, 1, 7), (192, 24, 16), (256, 5, 24)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_float32_results_over_an_e4m3_cache(dtype, dim, group, page):
    """Two f16 terms of every weight, as over an f16 cache: 2^-22 of spread instead of 2^-11.  Small scores and few tokens, so that
    what the scores carry does not cover the difference."""
    for lens in ([2, 3, 5, 6, 40, 0, 1], [i % 7 for i in range(90)], [20000]):
        heads = 2 if len(lens) == 7 else 8 if len(lens) > 7 else 1
        if len(lens) == 1 and dim != 64:
            continue
        c = Case(lens, group * heads, heads, dim, page, dtype, E4M3, q_scale=0.02, seed=dim + group)
        out, lse = c.run(want_lse=True, out_dtype=F32)
        wout, wlse, spread, reach, floor = c.want()
        d = dim * (2.0 ** -22 + 2.0 ** -24) * reach
        tol = (4 * d[..., None] + 2.0 ** -16 + 2.0 ** -22) * spread + 2.0 ** -32 * floor
        tol = tol + HALF[F32] * (np.abs(wout) + tol)
        assert (np.abs(out.double().cpu().numpy() - wout) <= tol).all(), (np.abs(out.double().cpu().numpy() - wout) / np.maximum(tol, 1e-30)).max()
        live = wlse > -np.inf
        assert (np.abs(lse.double().cpu().numpy()[live] - wlse[live]) <= d[live] + 2.0 ** -16 + 2.0 ** -22 * np.abs(wlse[live])).all()


@pytest.mark.parametrize("dim,group", [(64, 3), (128, 9), (192, 24)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_float16_results_over_an_e4m3_cache(dtype, dim, group):
    """As float32 ones (test_float32_results_over_an_e4m3_cache), then rounded: the weights' part is far below that rounding."""
    for lens in ([2, 3, 5, 6, 40, 0, 1], [i % 7 for i in range(90)]):
        heads = 2 if len(lens) == 7 else 8
        c = Case(lens, group * heads, heads, dim, 16, dtype, E4M3, q_scale=0.02, seed=dim + group)
        out = c.run(out_dtype=F16).double().cpu().numpy()
        wout, _, spread, reach, floor = c.want()
        d = dim * (2.0 ** -22 + 2.0 ** -24) * reach
        tol = (4 * d[..., None] + 2.0 ** -16 + 2.0 ** -22) * spread + 2.0 ** -32 * floor
        tol = tol + HALF[F16] * (np.abs(wout) + tol) + 2.0 ** -25
        assert (np.abs(out - wout) <= tol).all(), (np.abs(out - wout) / tol).max()
