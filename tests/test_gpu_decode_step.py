"""The operators around the experts run together as a program uses them: several decode steps of a batch through one layer
(page plan, FP8 projection, query/key preparation into the cache, attention, output projection, experts, head, log
probabilities), against the same steps in float64 over dense tensors.  Every stage of the check starts from what the GPU gave
the stage before, so the bounds are those of a single operator."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from oracle import paged  # noqa: E402

HEADS, KV, DIM, PAGE, HIDDEN, VOCAB = 8, 2, 64, 16, 512, 1000


class Layer:
    def __init__(self, cache_dtype, seed=0):
        import cachalot_b200 as cb

        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.pages = 40
        self.kc, self.vc = (torch.full((self.pages, KV, PAGE, DIM), float("nan"), device="cuda").to(cache_dtype) for _ in "kv")
        scaled = cache_dtype == torch.float8_e4m3fn
        self.ks, self.vs = ((torch.rand(KV, device="cuda", generator=self.g) + 0.5) / 32 if scaled else None for _ in "kv")
        self.qw, self.kw = ((torch.rand(DIM, device="cuda", generator=self.g) + 0.5).to(torch.bfloat16) for _ in "qk")
        self.freq, self.magnitude = cb.rope_frequencies(DIM, scaling="yarn", factor=4.0, trained_len=256)
        self.qkv_w, self.qkv_s = self.fp8((HEADS + 2 * KV) * DIM, HIDDEN)
        self.out_w, self.out_s = self.fp8(HIDDEN, HEADS * DIM)
        self.bank = cb.SlabBank(cb.FP4_FORMAT, HIDDEN, 384, 8)
        self.bank.fill_random(self.g)
        self.head = (torch.randn((VOCAB, HIDDEN), device="cuda", generator=self.g) / 16).to(torch.bfloat16)
        self.table = torch.full((4, 10), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(self.pages, device="cuda", generator=self.g).to(torch.int32)
        self.free_count = torch.tensor([self.pages], dtype=torch.int32, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def fp8(self, n, k):
        w = (torch.randn((n, k), device="cuda", generator=self.g) * 64).to(torch.float8_e4m3fn).view(torch.uint8)
        return w, torch.full((n // 128, k // 128), 1 / (64 * k ** 0.5), device="cuda")

    def step(self, x, ctx, new, tokens, sampled):
        """x bf16 [tokens, HIDDEN], one new token per request with new = 1 -> everything the stages gave."""
        import cachalot_b200 as cb

        plan = cb.plan_pages(ctx, new, self.table, self.free, self.free_count, page_size=PAGE, tokens=tokens, status=self.status)
        rows = cb.fp8_linear(x, self.qkv_w, self.qkv_s).view(tokens, HEADS + 2 * KV, DIM)
        q, k, v = rows[:, :HEADS], rows[:, HEADS:HEADS + KV], rows[:, HEADS + KV:]
        y, _ = cb.qk_norm_rope(q, k, plan.positions, self.freq, q_weight=self.qw, k_weight=self.kw, magnitude=self.magnitude, v=v, k_cache=self.kc, v_cache=self.vc,
                               slots=plan.slots, k_scale=self.ks, v_scale=self.vs, status=self.status)
        att = cb.paged_attention(y, self.kc, self.vc, self.table, plan.lens, k_scale=self.ks, v_scale=self.vs, status=self.status)
        h = cb.fp8_linear(att.view(tokens, HEADS * DIM), self.out_w, self.out_s)
        slots = torch.arange(tokens * 2, device="cuda", dtype=torch.int32).view(tokens, 2) % 8
        e = cb.moe_forward(h, slots, torch.full((tokens, 2), 0.5, device="cuda"), self.bank)
        logits = cb.bf16_gemv_f32(e / e.abs().amax(), self.head)
        return plan, rows, y, att, logits, cb.token_logprobs(logits, sampled, top=5, status=self.status)


@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("captured", [False, True])
def test_decode_steps(cache, captured):
    import cachalot_b200 as cb

    layer = Layer(cache)
    n = 4
    ctx = torch.zeros(n, dtype=torch.int32, device="cuda")
    new = torch.ones(n, dtype=torch.int32, device="cuda")
    x = torch.zeros((n, HIDDEN), dtype=torch.bfloat16, device="cuda")
    sampled = torch.tensor([1, 2, -1, 999], dtype=torch.int32, device="cuda")
    graph = None
    if captured:
        keep = layer.table.clone()
        layer.step(x, ctx, new, n, sampled)  # allocations and kernel attributes first
        layer.table.copy_(keep)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = layer.step(x, ctx, new, n, sampled)
        layer.table.copy_(keep)
    context = [0] * n
    history = [[] for _ in range(n)]  # normalised and rotated keys, values, in float64
    table, free, count = np.full((n, 10), -1), layer.free.tolist(), layer.pages
    for step in range(20):
        x.copy_(torch.randn((n, HIDDEN), device="cuda", generator=layer.g))
        ctx.copy_(torch.tensor(context, dtype=torch.int32))
        layer.free_count.fill_(count)
        if captured:
            graph.replay()
        else:
            got = layer.step(x, ctx, new, n, sampled)
        plan, rows, y, att, logits, lp = got
        want = paged.plan_pages(context, [1] * n, table, free, count, PAGE, n)
        assert plan.slots.tolist() == want[3] and plan.positions.tolist() == want[2] and plan.lens.tolist() == want[4]
        table, count = want[6], want[5]
        assert layer.table.tolist() == table.tolist() and plan.free_count.tolist() == [count]
        r = rows.double().cpu().numpy()
        f = layer.freq.cpu().numpy()
        q, k = (paged.rotate(paged.rms_norm(part, w.double().cpu().numpy(), 1e-6), want[2], f, magnitude=layer.magnitude)
                for part, w in ((r[:, :HEADS], layer.qw), (r[:, HEADS:HEADS + KV], layer.kw)))
        assert np.abs(y.double().cpu().numpy() - q).max() <= (2.0 ** -8 + 2.0 ** -15) * np.abs(q).max()
        at = torch.tensor(want[3], device="cuda")
        for buf, scale, ref in ((layer.kc, layer.ks, k), (layer.vc, layer.vs, r[:, HEADS + KV:])):
            stored = buf.view(torch.uint8)[at // PAGE, :, at % PAGE].view(cache).double()
            stored = (stored if scale is None else stored * scale.double()[:, None]).cpu().numpy()
            half = 2.0 ** -8 if scale is None else 2.0 ** -4
            low = 0.0 if scale is None else 2.0 ** -10 * float(scale.max())  # half of the smallest E4M3 step
            assert (np.abs(stored - ref) <= (half + 2.0 ** -15) * np.abs(ref) + low + 2.0 ** -15 * np.abs(ref).max()).all()
            for i in range(n):
                history[i].append(stored[i])
        for i in range(n):
            keys, values = np.array(history[i][0::2]), np.array(history[i][1::2])
            for h in range(HEADS):
                g = h // (HEADS // KV)
                o = paged.attend(y[i, h].double().cpu().numpy(), keys[:, g], values[:, g], DIM ** -0.5)
                assert (np.abs(att[i, h].double().cpu().numpy() - o[0]) <= 2.0 ** -8 * np.abs(o[0]) + (2.0 ** -10 + 4 * DIM * 2.0 ** -22 * o[3]) * o[2]).all()
        a, b, ids, top = paged.token_logprobs(logits.cpu().numpy(), sampled.tolist(), 5)
        assert lp.top_ids.tolist() == ids.tolist()
        for have, ref in ((lp.logprobs, a), (lp.entropy, b), (lp.top_logprobs, top)):
            assert np.abs(have.double().cpu().numpy() - ref).max() <= 2.0 ** -16 * 20
        context = [c + 1 for c in context]
    assert int(layer.status.item()) == 0


def test_prompt_chunk_then_decode():
    """A ragged chunk goes into the cache in one call; a token after it sees all of it."""
    import cachalot_b200 as cb

    layer = Layer(torch.bfloat16, 3)
    lens = [37, 0, 5, 16]
    ctx, new = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda")
    plan = cb.plan_pages(ctx, new, layer.table, layer.free, layer.free_count, page_size=PAGE, tokens=64, status=layer.status)
    rows = torch.randn((64, HEADS + 2 * KV, DIM), device="cuda").to(torch.bfloat16)
    y, _ = cb.qk_norm_rope(rows[:, :HEADS], rows[:, HEADS:HEADS + KV], plan.positions, layer.freq, v=rows[:, HEADS + KV:], k_cache=layer.kc, v_cache=layer.vc,
                           slots=plan.slots)
    _, ko = cb.qk_norm_rope(rows[:, :HEADS], rows[:, HEADS:HEADS + KV], plan.positions, layer.freq)
    q = torch.randn((4, HEADS, DIM), device="cuda").to(torch.bfloat16)
    out = cb.paged_attention(q, layer.kc, layer.vc, layer.table, plan.lens, out_dtype=torch.float32).double().cpu().numpy()
    starts = plan.starts.tolist()
    for i in range(4):
        keys, values = (t[starts[i]:starts[i + 1]].double().cpu().numpy() for t in (ko, rows[:, HEADS + KV:]))
        for h in range(HEADS):
            o = paged.attend(q[i, h].double().cpu().numpy(), keys[:, h // 4], values[:, h // 4], DIM ** -0.5)
            assert (np.abs(out[i, h] - o[0]) <= (2.0 ** -14 + 4 * DIM * 2.0 ** -22 * o[3]) * o[2]).all()
    assert int(layer.status.item()) == 0 and plan.free_count.tolist() == [layer.pages - 3 - 1 - 1]


@pytest.mark.parametrize("last", ["kernel", "copy", "operator"])
def test_captured_forks_that_meet_in_front_of_the_operators(last):
    """Two captured streams join right before each operator (which is launched early): it has to wait for both."""
    import cachalot_b200 as cb

    page, dim = 16, 64
    base = {k: torch.zeros(n, dtype=torch.int32, device="cuda") for k, n in dict(ctx=2, new=2, count=1).items()}
    ctx, new, count = base["ctx"], base["new"], base["count"]
    table, free = torch.full((2, 8), -1, dtype=torch.int32, device="cuda"), torch.arange(16, dtype=torch.int32, device="cuda")
    x = torch.zeros((8, 4, dim), dtype=torch.bfloat16, device="cuda")
    src = {k: torch.zeros_like(v) for k, v in dict(ctx=ctx, new=new, x=x).items()}
    kc, vc = (torch.zeros((16, 1, page, dim), dtype=torch.bfloat16, device="cuda") for _ in "kv")
    freq = cb.rope_frequencies(dim)[0]
    filler = torch.zeros(1 << 22, device="cuda")
    logits, ids = torch.zeros((2, 4000), device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    noise = torch.randn((2, 4000), device="cuda")

    def slow(dst, source):  # a write that comes late
        filler.add_(1.0), filler.mul_(0.5)
        if last == "copy":
            dst.copy_(source)
        elif last == "kernel":
            torch.add(source, 0, out=dst)
        else:
            dst.copy_(source)
            cb.token_logprobs(noise, ids)

    def forked(side, pairs):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            slow(*pairs[0])
        slow(*pairs[1])
        here.wait_stream(side)

    def step(side):
        forked(side, [(ctx, src["ctx"]), (new, src["new"])])
        plan = cb.plan_pages(ctx, new, table, free, count, page_size=page, tokens=8)
        forked(side, [(x[:4], src["x"][:4]), (x[4:], src["x"][4:])])
        y, _ = cb.qk_norm_rope(x[:, :2], x[:, 2:3], plan.positions, freq, v=x[:, 3:], k_cache=kc, v_cache=vc, slots=plan.slots)
        q = torch.zeros((2, 2, dim), dtype=torch.bfloat16, device="cuda")
        forked(side, [(q[:1], y[:1]), (q[1:], y[4:5])])
        att = cb.paged_attention(q, kc, vc, table, plan.lens)
        forked(side, [(logits[:1], noise[:1] * 2), (logits[1:], noise[1:] * 3)])
        return (*plan, y, att, *cb.token_logprobs(logits, ids, top=4))

    side = torch.cuda.Stream()

    def fresh(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        src["ctx"].zero_(), src["new"].copy_(torch.tensor([4, 4], device="cuda"))
        src["x"].copy_(torch.randn(x.shape, device="cuda", generator=g)), noise.copy_(torch.randn(noise.shape, device="cuda", generator=g))
        for t in (ctx, new, x, kc, vc, logits):
            t.zero_()
        table.fill_(-1), count.fill_(16)

    fresh(1), step(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(side)
    for seed in (2, 3, 4):
        fresh(seed)
        want = [t.clone() for t in step(side)]
        torch.cuda.synchronize()
        fresh(seed), graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert want[3].tolist()[:8] == [240 + i for i in range(4)] + [224 + i for i in range(4)] and want[7].float().abs().max() > 0
