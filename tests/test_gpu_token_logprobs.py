"""GPU parity: log probabilities, entropy and alternatives against float64.

Tolerance: the sum of weights is off by at most one part in 2^24 per dependent addition (a thread adds vocab / 256 terms, then 64
covers the joins, the approximate exp2 and its argument's rounding for terms that matter); that goes into ln S as it is,
and into U / S times U / S + 1 <= entropy + ln S + 1.  On top, the log probability itself is rounded (2^-23 of it).  (256: at
least 128 threads with two sums each.  The 64 threads that a row gets where there are more than 1184 add vocab / 128.)"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from oracle import paged  # noqa: E402

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _check(x, tokens, top, status=0, sums=256):
    import cachalot_b200 as cb

    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    r = cb.token_logprobs(x, torch.tensor(tokens, dtype=torch.int32, device="cuda"), top=top, status=word)
    assert int(word.item()) == status
    h = x.double().cpu().numpy()
    lp, ent, ids, best = paged.token_logprobs(h, tokens, top)
    rows, vocab = h.shape
    assert r.logprobs.shape == r.entropy.shape == (rows,) and r.top_ids.shape == r.top_logprobs.shape == (rows, top)
    assert np.array_equal(r.top_ids.cpu().numpy(), ids)
    step = (vocab / sums + 64) * 2.0 ** -24
    for got, want in ((r.logprobs, lp), (r.top_logprobs, best)):
        got = got.double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got == -np.inf, want == -np.inf)
        fin = np.isfinite(want)
        assert (np.abs(got[fin] - want[fin]) <= step + 2.0 ** -23 * np.abs(want[fin])).all(), np.abs(got[fin] - want[fin]).max()
    got = r.entropy.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(ent))
    fin = np.isfinite(ent)
    assert (np.abs(got[fin] - ent[fin]) <= step * (1 + ent[fin] + np.log(vocab)) + 2.0 ** -23 * ent[fin]).all()
    return r


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 9, 31, 33, 127, 1000, 4099, 32768, 50257])
@pytest.mark.parametrize("top", [0, 1, 20])
def test_vocabularies(vocab, dtype, top):
    g = _gen(vocab)
    x = (torch.randn((5, vocab), device="cuda", generator=g) * 3).to(dtype)
    _check(x, torch.randint(0, vocab, (5,), generator=torch.Generator().manual_seed(1)).tolist(), min(top, vocab))


@pytest.mark.parametrize("rows", [1, 2, 40, 150, 700])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_a_head(rows, dtype):
    x = (torch.randn((rows, 12928), device="cuda", generator=_gen(rows)) * 2.5).to(dtype)
    _check(x, [(i * 977) % 12928 for i in range(rows)], 32)


def test_whole_head():
    x = torch.randn((2, 129280), device="cuda", generator=_gen(1)) * 2.5
    _check(x, [0, 129279], 32)
    _check(x.to(BF16), [5, 129278], 7)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("order", ["up", "down", "equal", "two", "late"])
def test_orders_and_ties(order, dtype):
    """Ascending logits replace the list all the time; equal ones never do; ties go to the lower index."""
    v = 20000
    i = torch.arange(v, device="cuda", dtype=torch.float32)
    x = {"up": i / 1000, "down": -i / 1000, "equal": torch.zeros_like(i), "two": (i.to(torch.int32) % 97 == 96).float(), "late": (i >= v - 5).float() * 3}[order]
    _check(x.to(dtype)[None].repeat(2, 1), [3, v - 1], 32)


@pytest.mark.parametrize("rows", [600, 1200])
@pytest.mark.parametrize("vocab,dtype", [(1, F32), (37, BF16), (1001, F16), (1023, F32), (2049, BF16), (4100, F16), (9001, F32), (30001, BF16)])
def test_many_rows(rows, vocab, dtype):
    """Each of the orders above and rows of random logits, masked ones among them."""
    g, i = _gen(vocab), torch.arange(vocab, device="cuda", dtype=torch.float32)
    x = torch.randn((rows, vocab), device="cuda", generator=g) * 3
    x[0::7], x[1::7], x[2::7], x[3::7] = i / 100, -i / 100, 0.0, (i.to(torch.int32) % 97 == 96).float()
    x[4::7, vocab // 3:] = -float("inf")
    x[5::7, vocab // 2:] = torch.finfo(dtype).min
    _check(x.to(dtype), [(k * 977) % vocab for k in range(rows)], min(vocab, 32), sums=256 if rows == 600 else 128)


@pytest.mark.parametrize("offset", range(1, 9))
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_that_are_not_aligned(offset, dtype):
    wide = torch.randn((3, 2100), device="cuda", generator=_gen(offset)).to(dtype)
    _check(wide[:, offset:offset + 2000 + offset], [0, offset, 1999], 8)


def test_masks():
    g = _gen(2)
    x = torch.randn((6, 5000), device="cuda", generator=g) * 2
    x[0] = -float("inf")                                    # nothing left
    x[1, 1:] = -float("inf")                                # one left
    x[2, torch.arange(5000, device="cuda") % 7 != 3] = -float("inf")
    x[3, 10:] = torch.finfo(F32).min                        # masked by the lowest value
    x[4] = torch.finfo(F32).min                             # ... all of it: uniform
    r = _check(x, [4, 0, 3, 5, 6, 7], 12)
    assert r.logprobs[0] == -float("inf") and r.entropy[0] == 0 and r.top_ids[0].tolist() == list(range(12))
    assert r.logprobs[1] == 0 and r.entropy[1] == 0 and abs(float(r.logprobs[4]) + np.log(5000)) < 1e-4
    for dtype in (BF16, F16):
        y = x.to(dtype)
        y[3, 10:] = y[4] = torch.finfo(dtype).min
        _check(y, [4, 0, 3, 5, 6, 7], 12)


def test_zeros_of_either_sign_tie():
    x = torch.full((2, 3000), -1.0, device="cuda")
    x[:, 100:2000:3], x[:, 101:2000:3] = -0.0, 0.0
    _check(x, [100, 101], 32), _check(x.to(F16), [100, 101], 32)


def test_too_few_alternatives_that_are_numbers():
    x = torch.full((2, 40000), float("nan"), device="cuda")
    x[0, 5::10000], x[1, ::2] = 1.0, -float("inf")
    _check(x, [5, 6], 32)


def test_padding_and_tokens_outside():
    x = torch.randn((4, 300), device="cuda", generator=_gen(3))
    _check(x, [-1, 5, -100, 299], 3)
    _check(x, [-1, 300, 2 ** 31 - 1, 1], 3, status=2)


def test_nan_and_infinity():
    x = torch.randn((4, 3000), device="cuda", generator=_gen(4))
    x[0, 17], x[2, 2999] = float("nan"), float("nan")
    _check(x, [1, 2, 3, 4], 5)
    y = x[3:].clone()
    y[0, 100] = float("inf")
    import cachalot_b200 as cb

    r = cb.token_logprobs(y, torch.tensor([1], dtype=torch.int32, device="cuda"), top=2)
    assert r.logprobs.isnan().all() and r.entropy.isnan().all() and int(r.top_ids[0, 0]) == 100


def test_extreme_logits():
    x = torch.randn((3, 4000), device="cuda", generator=_gen(5)) * 1e4
    x[1] += 1e6
    x[2, 7] = 3e38
    r = _check(x, [1, 2, 7], 4)
    assert (r.entropy >= 0).all()


def test_general_form_graph_and_stream():
    import cachalot_b200 as cb

    x = torch.randn((3, 2000), device="cuda", generator=_gen(6))
    t = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    want = cb.token_logprobs(x, t, top=4)
    got = cb.token_logprobs(x.t().contiguous().t(), t.long(), top=4)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cb.token_logprobs(x, t, top=4)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = cb.token_logprobs(x, t, top=4)
    x.mul_(-2), t.add_(5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(r, cb.token_logprobs(x, t, top=4)))


def test_refusals():
    import cachalot_b200 as cb

    x, t = torch.zeros((3, 50), device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for args, kw in (((x.double(), t), {}), ((x[0], t), {}), ((x, t[:2]), {}), ((x, t.float()), {}), ((x, t), dict(top=51)), ((x, t), dict(top=-1)), ((x, t), dict(top=2 ** 32 + 1)),
                     ((x[:, :0], t), {}), ((x.cpu(), t), {}), ((x, t.cpu()), {}), ((x, t), dict(status=t.long()))):
        with pytest.raises(ValueError):
            cb.token_logprobs(*args, **kw)
    with pytest.raises(NotImplementedError, match="33 alternatives"):
        cb.token_logprobs(x, t, top=33)
    assert cb.token_logprobs(x[:0], t[:0], top=2).top_ids.shape == (0, 2)


def test_int64_tokens_beyond_int32():
    import cachalot_b200 as cb

    x, word = torch.randn((3, 300), device="cuda", generator=_gen(8)), torch.zeros(1, dtype=torch.int32, device="cuda")
    r = cb.token_logprobs(x, torch.tensor([2 ** 32 + 5, -2 ** 33 + 5, 5], device="cuda"), status=word)
    assert r.logprobs[:2].tolist() == [0.0, 0.0] and int(word.item()) == 2 and float(r.logprobs[2]) < 0


def test_outputs_of_one_call_do_not_overlap():
    """They may be pieces of one allocation: writing into one leaves the others as they are."""
    import cachalot_b200 as cb

    r = cb.token_logprobs(torch.randn((3, 300), device="cuda"), torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda"), top=7)
    for i, t in enumerate(r):
        before = [u.clone() for u in r]
        t.fill_(-77)
        assert all(torch.equal(a, b) for j, (a, b) in enumerate(zip(before, r)) if j != i) and (t == -77).all()
