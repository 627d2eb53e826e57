"""GPU parity: the page plan against its definition in Python integers."""
import pathlib
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from oracle import paged  # noqa: E402


def _cuda(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _check(context, new, page, tokens, width, n_free, count=None, table=None, seed=0, stride=None):
    import cachalot_b200 as cb

    rng = np.random.default_rng(seed)
    r = len(context)
    free = rng.permutation(100000)[:n_free]
    count = n_free if count is None else count
    if table is None:
        table = rng.integers(0, 50000, (r, width))
    store = torch.full((r, stride or width), -7, dtype=torch.int32, device="cuda")
    store[:, :width] = _cuda(np.asarray(table).reshape(r, width).tolist()).reshape(r, width)
    dev, status, cnt = store[:, :width], _cuda([0]), _cuda([count])
    got = cb.plan_pages(_cuda(context), _cuda(new), dev, _cuda(free.tolist()), cnt, page_size=page, tokens=tokens, status=status)
    want = paged.plan_pages(context, new, table, free, count, page, tokens)
    for name, w in zip(("starts", "requests", "positions", "slots", "lens"), want):
        assert getattr(got, name).tolist() == list(w), name
    assert got.free_count.tolist() == [want[5]]
    assert dev.tolist() == want[6].tolist()
    assert store[:, width:].eq(-7).all() and cnt.tolist() == [count]
    assert int(status.item()) == want[7]
    return got


@pytest.mark.parametrize("page", [1, 3, 16, 64])
@pytest.mark.parametrize("requests", [1, 2, 31, 64, 255, 256, 257, 700])
def test_decode_step(requests, page):
    rng = np.random.default_rng(requests * 100 + page)
    ctx = rng.integers(0, 5 * page, requests)
    _check(ctx.tolist(), rng.integers(0, 2, requests).tolist(), page, requests + 5, 8, requests + 3, stride=11)


@pytest.mark.parametrize("page", [1, 16, 24])
@pytest.mark.parametrize("tokens", [1, 255, 256, 257, 3000])
def test_prompt_chunks(tokens, page):
    rng = np.random.default_rng(tokens + page)
    new = rng.multinomial(tokens * 9 // 10, [0.4, 0.0, 0.3, 0.2, 0.1])
    _check(rng.integers(0, 200, 5).tolist(), new.tolist(), page, tokens, (200 + tokens) // page + 1, tokens // page + 10)


def test_no_new_tokens_and_no_requests():
    _check([5, 0, 17], [0, 0, 0], 16, 4, 3, 2)
    _check([5], [3], 16, 0, 3, 2)
    _check([], [], 16, 3, 1, 2, table=np.zeros((0, 1)))


def test_pages_run_out_and_lengths_are_cut():
    _check([0, 10, 3], [40, 30, 20], 8, 90, 12, 5)            # five pages for ten
    _check([0, 10, 3], [40, 30, 20], 8, 50, 12, 50)           # more tokens than the step holds
    _check([0, 90, 3], [40, 30, 20], 8, 100, 12, 50)          # past the table
    _check([200, 1], [4, 4], 8, 8, 12, 50)                    # the context alone is past the table
    _check([-3, 4, 4], [2, -2, 2], 8, 8, 2, 5)                # negative lengths count as none
    _check([0, 0], [9, 9], 8, 18, 3, 3, count=0)
    _check([0, 0], [9, 9], 8, 18, 3, 3, count=9)              # more than the list holds: cut to it
    _check([4, 8], [2, 2], 8, 4, 2, 3, table=[[-1, 5], [6, 7]])  # a page that is missing already


def test_slots_beyond_32_bits_are_left_out():
    import cachalot_b200 as cb

    status = _cuda([0])
    p = cb.plan_pages(_cuda([0]), _cuda([2]), _cuda([[0]]), _cuda([2 ** 30]), _cuda([1]), page_size=16, tokens=2, status=status)
    assert p.slots.tolist() == [-1, -1] and int(status.item()) == 1


def test_many_requests():
    rng = np.random.default_rng(3)
    _check(rng.integers(0, 40, 8192).tolist(), rng.integers(0, 3, 8192).tolist(), 16, 9000, 4, 8192)


def test_general_form_streams_and_graphs():
    """int64 lengths take the general form; a captured step replays on new lengths; a stream of its own works."""
    import cachalot_b200 as cb

    ctx, new, free, count = _cuda([3, 20]), _cuda([1, 14]), _cuda(list(range(100, 110))), _cuda([10])
    table = _cuda([[1, -1, -1], [2, 3, -1]])
    a = cb.plan_pages(ctx, new, table.clone(), free, count, page_size=16, tokens=16)
    b = cb.plan_pages(ctx.long(), new.long(), table.clone(), free.long(), count.long(), page_size=16, tokens=16)
    assert all(torch.equal(getattr(a, k), getattr(b, k)) for k in ("starts", "requests", "positions", "slots", "lens", "free_count"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    live = table.clone()
    with torch.cuda.stream(side):
        cb.plan_pages(ctx, new, live, free, count, page_size=16, tokens=16)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = cb.plan_pages(ctx, new, live, free, count, page_size=16, tokens=16)
    ctx.copy_(_cuda([15, 31])), new.copy_(_cuda([2, 2])), live.copy_(_cuda([[1, -1, -1], [2, 3, -1]]))
    graph.replay()
    want = paged.plan_pages([15, 31], [2, 2], [[1, -1, -1], [2, 3, -1]], list(range(100, 110)), 10, 16, 16)
    assert p.slots.tolist() == want[3] and live.tolist() == want[6].tolist() and p.free_count.tolist() == [want[5]]


def test_refusals():
    import cachalot_b200 as cb

    ok = dict(page_size=16, tokens=4)
    ctx, new, table, free, count = _cuda([3, 20]), _cuda([1, 1]), _cuda([[1, -1], [2, 3]]), _cuda([4, 5]), _cuda([2])
    for bad in ((ctx, new[:1], table, free, count), (ctx, new, table[:1], free, count), (ctx, new, table.long(), free, count),
                (ctx.float(), new, table, free, count), (ctx, new, table.t(), free, count), (ctx, new, table, free, free),
                (ctx.cpu(), new, table, free, count), (ctx, new, table.cpu(), free, count)):
        with pytest.raises(ValueError):
            cb.plan_pages(*bad, **ok)
    for kw in (dict(page_size=0, tokens=4), dict(page_size=16, tokens=-1), dict(page_size=16, tokens=2 ** 31), dict(page_size=2 ** 32 + 16, tokens=4)):
        with pytest.raises(ValueError):
            cb.plan_pages(ctx, new, table, free, count, **kw)
    with pytest.raises(NotImplementedError, match="8193 requests"):
        many = torch.zeros(8193, dtype=torch.int32, device="cuda")
        cb.plan_pages(many, many, torch.zeros((8193, 1), dtype=torch.int32, device="cuda"), free, count, **ok)


def test_requests_around_the_default_shared_memory_limit():
    """Each in a process of its own: a larger call before it would have raised the kernel's limit for good."""
    root = pathlib.Path(__file__).resolve().parents[1]
    code = "import sys; sys.path[:0] = ['.', 'tests']; import test_gpu_plan_pages as t; n = int(sys.argv[1]); t._check([i % 40 for i in range(n)], [i % 3 for i in range(n)], 16, n + 9, 4, n)"
    for n in (6135, 6136, 6143, 6144):
        run = subprocess.run([sys.executable, "-c", code, str(n)], cwd=root, capture_output=True, text=True, timeout=300)
        assert run.returncode == 0, (n, run.stderr[-2000:])


def test_outputs_of_one_call_do_not_overlap():
    """They may be pieces of one allocation: writing into one leaves the others as they are."""
    import cachalot_b200 as cb

    p = cb.plan_pages(_cuda([3, 20]), _cuda([1, 14]), _cuda([[1, -1, -1], [2, 3, -1]]), _cuda(list(range(100, 110))), _cuda([10]), page_size=16, tokens=16)
    for i, t in enumerate(p):
        before = [u.clone() for u in p]
        t.fill_(-77)
        assert all(torch.equal(a, b) for j, (a, b) in enumerate(zip(before, p)) if j != i) and (t == -77).all()
