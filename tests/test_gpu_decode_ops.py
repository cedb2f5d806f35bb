"""GPU: the decoder operators together, as a decoder uses them: a ragged prompt pass and single-token steps of append -> attention -> logits -> sampling,
eager and as a replayed graph, and sampling of the rows that the engine's own rules produce.  The model around them is torch's elementwise work; every attention
result is held to the 64-bit formula over the rows appended so far, every drawn id to the 64-bit sampler on the logits it was drawn from."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from speaksense_amd import ops  # noqa: E402
from test_gpu_kv_ops import DT, quantise, values  # noqa: E402
from test_gpu_sample_ops import check, plain  # noqa: E402

pytestmark = pytest.mark.gpu

LAYERS, HEADS, GROUPS, DIM, VOCAB, PAGE, STEPS = 2, 2, 3, 64, 500, 16, 5
PROMPTS = [37, 1, 16]


class Decoder:
    """Embedding -> layers of attention with elementwise projections -> logits, over one cache a layer."""

    def __init__(self, kind, dt, seed=0):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
        self.kind, self.dt, n = kind, DT[dt], len(PROMPTS)
        self.emb = r(VOCAB, HEADS * GROUPS, DIM).to(self.dt).cuda()
        self.scale_q, self.scale_k, self.scale_v = ((0.5 + torch.rand((LAYERS, 1, h, DIM), generator=g)).to(self.dt).cuda() for h in (HEADS * GROUPS, HEADS, HEADS))
        self.head = (r(VOCAB, HEADS * GROUPS * DIM) * 0.15).cuda()
        most = -(-(max(PROMPTS) + STEPS + 1) // PAGE)
        self.pages = torch.randperm(n * most + 2, generator=g)[:n * most].reshape(n, most).int().cuda()
        self.caches = [ops.KvCache.empty(n * most + 2, HEADS, PAGE, DIM, kind=kind, dtype=self.dt) for _ in range(LAYERS)]
        self.lens = torch.tensor(PROMPTS, dtype=torch.int32).cuda()
        starts = [0] + list(np.cumsum(PROMPTS))
        self.prompt = ops.KvBatch(self.pages, torch.tensor(starts, dtype=torch.int32).cuda(), self.lens, n_tokens=starts[-1], max_new=max(PROMPTS), min_new=min(PROMPTS))
        self.single = ops.KvBatch(self.pages, torch.arange(n + 1, dtype=torch.int32).cuda(), self.lens, n_tokens=n, max_new=1, min_new=1, max_len=max(PROMPTS) + STEPS + 1)
        self.last = torch.tensor(starts[1:]).cuda() - 1
        self.first = torch.randint(0, VOCAB, (starts[-1],), generator=g).cuda()
        self.uniform = torch.rand((STEPS + 1, n), generator=g, dtype=torch.float64).cuda()
        self.settings = dict(temperature=torch.tensor([0.7, 0.0, 1.3]).cuda(), top_k=torch.tensor([40, 0, 0], dtype=torch.int32).cuda(),
                             top_p=torch.tensor([0.95, 1.0, 0.9]).cuda(), min_p=torch.tensor([0.0, 0.0, 0.01]).cuda())

    def forward(self, ids, batch, rows, u):
        x = self.emb.index_select(0, ids.long())
        seen = []
        for i, cache in enumerate(self.caches):
            q, k, v = x * self.scale_q[i], x[:, ::GROUPS] * self.scale_k[i], x[:, 1::GROUPS] * self.scale_v[i]
            ops.kv_append(cache, batch, k, v)
            o = ops.kv_attention(cache, batch, q)
            seen.append((q, k, v, o))
            x = (x + o) * 0.7
        x = x if rows is None else x.index_select(0, rows)
        logits = (x.reshape(x.shape[0], 1, -1).float() * self.head).sum(-1)
        return seen, logits, ops.sample_rows(logits, u, **self.settings)


def held(rows, kind):
    """CPU: what a cache gives back for appended rows."""
    rows = rows.cpu()
    return values(*quantise(rows, kind), kind).double() if kind != "same" else rows.double()


def check_steps(m, steps, kind):
    """Every step's attention against 64 bits, over all rows appended before it; every draw against the plain sampler."""
    n, half_out = len(PROMPTS), torch.finfo(m.dt).eps / 2
    half_p = torch.finfo(torch.bfloat16 if kind == "same" and m.dt == torch.bfloat16 else torch.float16).eps / 2
    past = [[([], []) for _ in range(LAYERS)] for _ in range(n)]
    for at, (seen, logits, got, u) in enumerate(steps):
        starts = [0] + list(np.cumsum(PROMPTS)) if at == 0 else list(range(n + 1))
        for i, (q, k, v, o) in enumerate(seen):
            hk, hv, q, o = held(k, kind), held(v, kind), q.cpu().double(), o.cpu().double()
            for s in range(n):
                a, b = starts[s], starts[s + 1]
                keys, vals = past[s][i]
                keys += list(hk[a:b])
                vals += list(hv[a:b])
                kk, vv = torch.stack(keys), torch.stack(vals)                 # [len, heads, dim]
                for t in range(a, b):
                    end = len(keys) - (b - 1 - t)
                    for h in range(HEADS * GROUPS):
                        p = torch.softmax(kk[:end, h // GROUPS] @ q[t, h] * DIM ** -0.5, 0)
                        w = vv[:end, h // GROUPS]
                        want = p @ w
                        tol = half_out * want.abs() + (half_p + 2.0 ** -15) * (p @ w.abs()) + end * 2.0 ** -24 * w.abs().max() + 2.0 ** -24
                        assert ((o[t, h] - want).abs() <= tol).all(), (at, i, s, t, h)
        x = logits.cpu()
        f = {k: v.cpu() for k, v in m.settings.items()}
        for s in range(n):
            want = plain(x[s], float(u[s]), float(f["temperature"][s]), int(f["top_k"][s]), float(f["top_p"][s]), float(f["min_p"][s]))
            assert (int(got.id[s]), int(got.n_kept[s])) == (want[0], want[3]), (at, s)
            assert abs(float(got.p[s]) - want[1]) <= 2.0 ** -20 * want[1] and abs(float(got.logprob[s]) - want[2]) <= 2.0 ** -20 * max(1.0, abs(want[2]))


def keep(seen, logits, got, u):
    return [tuple(t.clone() for t in row) for row in seen], logits.clone(), ops.Sampled(*(t.clone() for t in got)), u.tolist()


def run(m, graph):
    """The prompt pass, then STEPS single tokens; the steps eager, or one captured graph replayed with eager work in between."""
    m.lens.copy_(torch.tensor(PROMPTS, dtype=torch.int32))
    steps = [keep(*m.forward(m.first, m.prompt, m.last, m.uniform[0]), m.uniform[0])]
    ids, u = steps[0][2].id.clone(), m.uniform[1].clone()

    def step():
        m.lens.add_(1)
        seen, logits, got = m.forward(ids, m.single, None, u)
        ids.copy_(got.id)
        return seen, logits, got

    if graph:
        g = torch.cuda.CUDAGraph()                       # (the eager run before has done the first calls' setup)
        with torch.cuda.graph(g):
            out = step()
    for i in range(1, STEPS + 1):
        u.copy_(m.uniform[i])
        if graph:
            g.replay()
            torch.randn(1000, device="cuda").sum().item()
        else:
            out = step()
        steps.append(keep(*out, m.uniform[i]))
    torch.cuda.synchronize()
    return steps


@pytest.mark.parametrize("kind,dt", [("same", "bf16"), ("e4m3", "f16"), ("int8", "f16")])
def test_a_decoder(kind, dt):
    m = Decoder(kind, dt)
    eager = run(m, False)
    check_steps(m, eager, kind)
    for a, b in zip(eager, run(m, True)):
        assert all(torch.equal(x, y) for ra, rb in zip(a[0], b[0]) for x, y in zip(ra, rb)) and torch.equal(a[1], b[1])
        assert all(torch.equal(x, y) for x, y in zip(a[2], b[2]))


def test_prompt_in_chunks_is_the_prompt():
    """A prompt appended and attended in two chunks gives what it gives in one pass: the keys are the same, so every row is within two roundings."""
    g = torch.Generator().manual_seed(4)
    n, cut = 45, 19
    q, k, v = (torch.randn((n, h, DIM), generator=g).half().cuda() for h in (HEADS * GROUPS, HEADS, HEADS))
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32).cuda()
    t32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    outs = []
    for spans in ([(0, n)], [(0, cut), (cut, n)]):
        cache = ops.KvCache.empty(4, HEADS, PAGE, DIM)
        rows = []
        for a, b in spans:
            batch = ops.KvBatch(table, t32(0, b - a), t32(b), n_tokens=b - a, max_new=b - a)
            ops.kv_append(cache, batch, k[a:b], v[a:b])
            rows.append(ops.kv_attention(cache, batch, q[a:b]))
        whole = ops.KvBatch(table, t32(0, n), t32(n), n_tokens=n, max_new=n)
        rk, rv = ops.kv_read(cache, whole)
        assert torch.equal(rk, k) and torch.equal(rv, v)
        outs.append(torch.cat(rows).double())
    # each result is within half_out |o| + (half_p + 2^-15) A + n 2^-24 vmax of the formula; |o| <= A <= vmax
    vmax = float(v.abs().max())
    assert float((outs[0] - outs[1]).abs().max()) <= 2 * (2 * 2.0 ** -11 + 2.0 ** -15 + n * 2.0 ** -24) * vmax


def test_rows_of_the_engine_rules(toy_ml_path):
    """The engine's processed rows (log-probabilities, -inf where a rule masks the id) are logits as they are: greedy takes the id that the engine takes, with its
    log-probability, and no draw takes a masked id."""
    from speaksense_amd import binding
    e = binding.Engine(toy_ml_path, dtype=binding.DTYPE_F16, max_batch=2)
    rng = np.random.default_rng(11)
    rows, want = [], []
    for hist, has_ts in (([], False), ([e.beg + 3, 700], True), ([e.beg, 900, e.beg + 10, e.beg + 10], True)):
        for _ in range(3):
            r = e.process_logits(rng.standard_normal(e.n_vocab).astype(np.float32) * 3, hist, has_ts, 0, binding.default_params(), want_row=True)
            rows.append(torch.from_numpy(r["logprobs"]))
            want.append(r)
    e.close()
    x = torch.stack(rows)
    assert torch.isneginf(x).any(1).all()
    n = len(want)
    u = torch.from_numpy(rng.random(n)).cuda()
    r = ops.sample_rows(x.cuda(), u, temperature=torch.zeros(n, device="cuda"))
    assert r.id.tolist() == [w["id"] for w in want]
    assert max(abs(a - w["plog"]) for a, w in zip(r.logprob.tolist(), want)) < 2e-5     # the rows' own float32 normalisation
    check(x, u.tolist(), t=[0.2 * (i + 1) for i in range(n)], k=[0, 50, 0] * 3, p=[1.0, 0.95, 0.8] * 3)
    for _ in range(4):
        got = ops.sample_rows(x.cuda(), torch.from_numpy(rng.random(n)).cuda()).id.cpu().long()
        assert math.isfinite(float(x.gather(1, got[:, None]).min()))


def test_inputs_that_ask_for_a_gradient_are_refused():
    cache = ops.KvCache.empty(1, 1, 16, 64)
    t32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    b = ops.KvBatch(t32(0)[None], t32(0, 1), t32(1), n_tokens=1, max_new=1)
    x = torch.ones((1, 1, 64), dtype=torch.float16, device="cuda")
    g = x.clone().requires_grad_()
    rows = torch.zeros((1, 9), device="cuda", requires_grad=True)
    u = torch.zeros(1, dtype=torch.float64, device="cuda")
    for call in (lambda: ops.kv_append(cache, b, g, x), lambda: ops.kv_append(cache, b, x, g), lambda: ops.kv_attention(cache, b, g), lambda: ops.sample_rows(rows, u)):
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()
    assert torch.equal(ops.kv_attention(cache, b, g.detach()), x)


def test_every_tensor_that_asks_for_a_gradient_is_refused():
    """Settings of the sampler and tensors of the cache too, in reverse and in forward mode."""
    from torch.autograd import forward_ad
    t32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    b = ops.KvBatch(t32(0)[None], t32(0, 1), t32(1), n_tokens=1, max_new=1)
    x = torch.ones((1, 1, 64), dtype=torch.float16, device="cuda")
    h = lambda *s, dtype=torch.float16: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    logits, u, one = h(1, 9, dtype=torch.float32), h(1, dtype=torch.float64), h(1, dtype=torch.float32) + 0.5

    def calls(mark):
        """(call, its tensors of which `mark` changes one)"""
        for at in range(2):
            kv = [h(1, 1, 16, 64), h(1, 1, 16, 64)]
            kv[at] = mark(kv[at])
            c = ops.KvCache(*kv)
            sc = [h(1, 1, 16, dtype=torch.float32), h(1, 1, 16, dtype=torch.float32)]
            sc[at] = mark(sc[at])
            c8 = ops.KvCache(h(1, 1, 16, 64, dtype=torch.int8), h(1, 1, 16, 64, dtype=torch.int8), *sc, kind="int8", dtype=torch.float16)
            for cache in (c, c8):
                yield from (lambda cache=cache: ops.kv_append(cache, b, x, x), lambda cache=cache: ops.kv_read(cache, b), lambda cache=cache: ops.kv_attention(cache, b, x))
        plain = ops.KvCache(h(1, 1, 16, 64), h(1, 1, 16, 64))
        m = mark(x.clone())
        yield from (lambda: ops.kv_append(plain, b, m, x), lambda: ops.kv_append(plain, b, x, m), lambda: ops.kv_attention(plain, b, m), lambda: ops.kv_attention(plain, b, x, out=mark(x.clone())))
        yield from (lambda: ops.sample_rows(mark(logits.clone()), u), lambda: ops.sample_rows(logits, mark(u.clone())))
        for name in ("temperature", "top_p", "min_p"):
            yield lambda name=name: ops.sample_rows(logits, u, **{name: mark(one.clone())})

    n = 0
    for call in calls(lambda t: t.requires_grad_()):
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()
        n += 1
    with forward_ad.dual_level():
        for call in calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t))):
            with pytest.raises(ValueError, match="gradient"):
                call()
            n -= 1
        ops.sample_rows(logits, u, temperature=one)        # nothing that carries one
    assert n == 0
    with torch.no_grad():
        ops.sample_rows(logits.requires_grad_(), u)
