"""GPU: filtered sampling (speaksense_amd.ops.sample_rows) against a plain implementation in 64 bits on the CPU.  Ids and counts have to be equal: the seeds
are fixed and the reference asserts that no uniform number lies within 1e-9 of a boundary.  p and logprob: float32 results of sums good to 2^-20."""
import math

import pytest

torch = pytest.importorskip("torch")
from speaksense_amd import ops  # noqa: E402

pytestmark = pytest.mark.gpu


def plain(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """One row, 64 bits: (id, p, logprob, n_kept)."""
    x = x.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    n = x.numel()
    top = x.max()
    if top == -math.inf:
        return -1, 0.0, -math.inf, 0
    if top == math.inf:
        x = torch.where(x == math.inf, 0.0, -math.inf).double()
        top = torch.zeros((), dtype=torch.float64)
    if not t > 0:
        return int((x == top).nonzero()[0]), 1.0, -float(torch.logsumexp(x - top, 0)), 1
    w = torch.where(x > -math.inf, torch.exp((x - top) / t), 0.0)
    w[x == top] = 1.0
    order = torch.sort(x, descending=True, stable=True)[1]
    order = order[x[order] > -math.inf]
    if 0 < k < n:
        order = order[:k]
    if p < 1:
        before = w[order].cumsum(0) - w[order]
        cut = max(p, 0.0) * w[order].sum()
        assert p <= 0 or float((before[1:] - cut).abs().min() if len(order) > 1 else 1) > 1e-9 or float(w[order].std()) == 0, "a seed on the border"
        order = order[(before < cut) | (torch.arange(len(order)) == 0)]
    if m > 0:
        order = order[w[order] >= min(m, 1.0)]
    kept = torch.zeros(n, dtype=torch.float64)
    kept[order] = w[order]
    run = kept.cumsum(0)
    target = min(max(u, 0.0), 1.0) * run[-1] if u == u else 0.0
    at = ((run > target) & (kept > 0)).nonzero()
    i = int(at[0]) if len(at) else int((kept > 0).nonzero()[-1])
    if 0 < u < 1 and len(at):
        assert min(abs(float(run[i] - target)), abs(float(run[i] - kept[i] - target))) > 1e-9 or float(w[order].std()) == 0, "a seed on the border"
    return i, float(kept[i] / run[-1]), float((x[i] - top) / t - torch.log(w.sum())), len(order)


def check(x, u, t=None, k=None, p=None, m=None):
    n = x.shape[0]
    dev = lambda v, dt: None if v is None else torch.tensor(v, dtype=dt).cuda()  # noqa: E731
    r = ops.sample_rows(x.cuda(), torch.tensor(u, dtype=torch.float64).cuda(), temperature=dev(t, torch.float32), top_k=dev(k, torch.int32), top_p=dev(p, torch.float32), min_p=dev(m, torch.float32))
    ids, ps, lps, ns = (v.cpu() for v in r)
    f32 = lambda v, i, off: off if v is None else float(torch.tensor(v[i], dtype=torch.float32))  # noqa: E731
    for i in range(n):
        w = plain(x[i], u[i], f32(t, i, 1.0), 0 if k is None else k[i], f32(p, i, 1.0), f32(m, i, 0.0))
        got = (int(ids[i]), float(ps[i]), float(lps[i]), int(ns[i]))
        assert (got[0], got[3]) == (w[0], w[3]), (i, got, w)
        assert abs(got[1] - w[1]) <= 2.0 ** -20 * w[1]
        assert got[2] == w[2] or abs(got[2] - w[2]) <= 2.0 ** -20 * max(1.0, abs(w[2])), (i, got, w)
    return r


def rows(g, n, v, dt, spread=2.5):
    x = torch.randn((n, v), generator=g) * spread
    x.scatter_add_(1, torch.randint(0, v, (n, 6), generator=g), torch.rand((n, 6), generator=g) * 9)
    x[torch.rand((n, v), generator=g) < 0.05] = -math.inf
    return x.to(dt)


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 2, 63, 64, 65, 255, 1023, 2049, 51866, 70001])
def test_plain_temperature(dt, v):
    g = torch.Generator().manual_seed(v)
    n = 9
    x = rows(g, n, v, dt)
    x[:, v // 2] = 1.0                                    # never all masked
    u = torch.rand(n, generator=g, dtype=torch.float64).tolist()
    check(x, u)
    check(x, u, t=[0.0, -1.0, math.nan, 0.2, 0.4, 0.6, 0.8, 1.0, 3.0])


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("v", [40, 1000, 51866])
@pytest.mark.parametrize("seed", [0, 1])
def test_filters(dt, v, seed):
    g = torch.Generator().manual_seed(seed * 1000 + v)
    n = 24
    x = rows(g, n, v, dt)
    x[:, 0] = 0.0
    u = torch.rand(n, generator=g, dtype=torch.float64).tolist()
    t = (torch.rand(n, generator=g) * 1.5 + 0.1).tolist()
    k = [0, 1, 2, 5, 50, 200, 1500, v, v + 5, -3, v - 1, 7] * 2
    p = [1.0, 0.9, 0.5, 0.99, 0.05, 1.5, 0.95, 0.999, 0.7, 0.3, 0.6, math.nan, 0.8] * 2
    m = [0.0, 0.1, 0.0, 0.5, 0.01, 0.0, 1.0, 0.001, -1.0, math.nan, 0.0] * 3
    check(x, u, t, k=k)
    check(x, u, t, p=p[:n])
    check(x, u, t, m=m[:n])
    check(x, u, t, k, p[:n], m[:n])


def test_equal_logits():
    """Rows of one value, of two, of a few thousand equal ids in front or behind: ties go to the lowest ids and sums of equal weights are exact."""
    v = 9000
    x = torch.zeros(8, v)
    x[1, 5000:] = -1
    x[2, :3000] = -2
    x[3, ::3] = 4
    x[4, 1:] = -0.0                                       # equal to 0.0
    x[5, :4000] = -math.inf
    x[6, 17] = 30
    x[7] = -5.5
    # row 3 has period 3: a tenth of its weight ends exactly between two ids, where 64 bits cannot tell (0.1 was refused by the reference's own assertion)
    u = [0.5, 0.25, 0.75, 0.1003, 0.9, 0.3, 0.999, 0.0]
    check(x, u)
    check(x, u, k=[1, 4500, 6500, 2999, 1025, 1024, 2000, 8999])
    check(x, u, p=[0.5] * 8)
    check(x, u, k=[4096] * 8, p=[0.25] * 8, m=[0.5] * 8)
    check(x, u, p=[0.0, -1.0, 0.0, 1e-9, 0.0, 0.0, 0.0, 0.0])


def test_crowded_logits():
    """Thousands of different logits within a few float steps of each other, and logits over the whole range of floats: the histogram's steps hold too many."""
    g = torch.Generator().manual_seed(5)
    v = 20000
    x = torch.empty(5, v)
    x[0] = 1.0 + torch.randint(0, 4000, (v,), generator=g) * 2.0 ** -23
    x[1] = torch.cat([torch.tensor([80.0]), -1.0 + torch.randint(0, 9000, (v - 1,), generator=g) * 2.0 ** -23])
    x[2] = torch.randn(v, generator=g) * 1e-30
    x[3] = torch.randn(v, generator=g)
    x[3, 0], x[3, 1] = 3e38, -3e38
    x[4] = torch.exp(torch.rand(v, generator=g) * 80)
    u = torch.rand(5, generator=g, dtype=torch.float64).tolist()
    check(x, u, t=[1.0, 100.0, 1e-30, 1e36, 1e30], k=[5000, 12345, 3000, 7000, 1500])
    check(x, u, t=[1.0, 100.0, 1e-30, 1e36, 1e30], p=[0.3, 0.6, 0.7, 0.8, 0.9])


def test_special_rows():
    """All masked, NaN, infinities, one unmasked id, uniform numbers at and outside the ends."""
    x = torch.randn((12, 300), generator=torch.Generator().manual_seed(1))
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 7:] = math.nan
    x[3, 40] = x[3, 50] = x[3, 290] = math.inf
    x[4] = -math.inf
    x[4, 299] = -1e30
    x[5] = math.inf
    x[6, :] = -math.inf
    x[6, [3, 200]] = torch.tensor([1.0, 1.0])
    u = [0.5, 0.5, 0.9, 0.5, 0.7, 0.999, 0.5, 0.0, 1.0, 2.0, -1.0, math.nan]
    r = check(x, u)
    assert r.id[:2].tolist() == [-1, -1] and r.id[3] == 50 and r.id[4] == 299 and r.id[6] == 200
    check(x, u, k=[2] * 12, p=[0.6] * 12, m=[0.1] * 12)
    check(x, u, t=[0.0] * 12)
    t = [1e-38, 1e-45, 1e-10, 1e38, math.inf, 1.0, math.inf, math.inf, 1e-44, 1e-38, 1e10, 1e-20]
    check(x, u, t)
    check(x, u, t, k=[250] * 12, m=[0.01] * 12)


def test_strided_and_misaligned_rows():
    g = torch.Generator().manual_seed(2)
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        big = rows(g, 6, 5003, dt).cuda()
        u = torch.rand(6, generator=g, dtype=torch.float64).cuda()
        for view in (big[:, 1:4000], big[:, 3:5003], big[::2, :777], big[1:2, 5:9]):
            n = view.shape[0]
            k = torch.full((n,), 30, dtype=torch.int32, device="cuda")
            a, b = ops.sample_rows(view, u[:n].contiguous(), top_k=k), ops.sample_rows(view.contiguous(), u[:n].contiguous(), top_k=k)
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_large_vocabulary_and_many_rows():
    g = torch.Generator().manual_seed(3)
    for v, n, dt in ((1 << 20, 2, torch.float32), ((1 << 20) - 1, 3, torch.bfloat16), (400, 700, torch.float16)):
        x = rows(g, n, v, dt)
        u = torch.rand(n, generator=g, dtype=torch.float64).tolist()
        check(x, u)
        check(x, u, k=[100] * n, p=[0.9] * n)


def test_results_repeat():
    g = torch.Generator().manual_seed(4)
    x = rows(g, 64, 51866, torch.float32).cuda()
    u = torch.rand(64, generator=g, dtype=torch.float64).cuda()
    kw = dict(top_p=torch.full((64,), 0.97, device="cuda"), temperature=torch.full((64,), 1.3, device="cuda"))
    a = ops.sample_rows(x, u, **kw)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(a, ops.sample_rows(x, u, **kw)))


def test_frequencies():
    """20 000 uniform numbers in equal steps over one row: every kept id comes as often as its share says, to one step at either end."""
    n = 20000
    x = torch.tensor([2.0, -math.inf, 1.0, 3.0, 0.0, 2.5, -1.0]).repeat(n, 1).cuda()
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).cuda()
    r = ops.sample_rows(x, u, temperature=torch.full((n,), 0.8, device="cuda"), top_k=torch.full((n,), 4, dtype=torch.int32, device="cuda"))
    w = torch.exp(torch.tensor([2.0, 0.0, 1.0, 3.0, 0.0, 2.5, 0.0], dtype=torch.float64) / 0.8)
    w[[1, 4, 6]] = 0
    share = w / w.sum()
    assert ((torch.bincount(r.id.cpu().long(), minlength=7) - share * n).abs() <= 1.0).all()


def test_refusals_and_empty():
    x, u = torch.zeros((3, 10), device="cuda"), torch.zeros(3, dtype=torch.float64, device="cuda")
    for call in (lambda: ops.sample_rows(x.double(), u), lambda: ops.sample_rows(x, u.float()), lambda: ops.sample_rows(x, u[:2]), lambda: ops.sample_rows(x.t(), u), lambda: ops.sample_rows(x[0], u),
                 lambda: ops.sample_rows(x, u, top_k=torch.zeros(3, device="cuda")), lambda: ops.sample_rows(x, u, top_p=torch.zeros(2, device="cuda")),
                 lambda: ops.sample_rows(x, u, temperature=torch.zeros(3)), lambda: ops.sample_rows(x, u.cpu())):
        with pytest.raises(ValueError):
            call()
    from speaksense_amd.binding import SpeakSenseError
    with pytest.raises(SpeakSenseError):
        ops.sample_rows(torch.zeros((1, 0), device="cuda"), u[:1])
    with pytest.raises(SpeakSenseError):
        ops.sample_rows(torch.zeros((1, (1 << 20) + 1), device="cuda"), u[:1])
    with pytest.raises(SpeakSenseError):
        ops.sample_rows(x[:1].expand(3, -1), u)           # rows on top of each other: stride 0
    assert ops.sample_rows(x[:0], u[:0]).id.shape == (0,)


def test_captured_sampling():
    g = torch.Generator().manual_seed(6)
    x, u = torch.zeros((5, 3001), device="cuda"), torch.zeros(5, dtype=torch.float64, device="cuda")
    p, k = torch.full((5,), 0.9, device="cuda"), torch.full((5,), 60, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.sample_rows(x, u, top_k=k, top_p=p)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = ops.sample_rows(x, u, top_k=k, top_p=p)
    for i in range(5):
        x.copy_(rows(g, 5, 3001, torch.float32))
        u.copy_(torch.rand(5, generator=g, dtype=torch.float64))
        p.fill_(0.5 + 0.1 * i)
        k.fill_(20 + 700 * i)
        want = ops.sample_rows(x, u, top_k=k, top_p=p)
        torch.cuda.synchronize()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(r, want)), i


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("share", [0.02, 0.995])
def test_masks_of_the_lowest_number(dt, share):
    """Ids that a mask holds at the type's lowest number are ordinary logits that weigh nothing; they must not blunt the histograms of the others."""
    g = torch.Generator().manual_seed(12)
    n, v = 8, 5000
    x = (torch.randn((n, v), generator=g) * 3).to(dt)
    x.masked_fill_(torch.rand((n, v), generator=g) < share, torch.finfo(dt).min)
    x[-1].fill_(torch.finfo(dt).min)
    u = torch.rand((n,), generator=g, dtype=torch.float64).tolist()
    check(x, u, t=[0.7] * n, k=[0, 40, 900, 0, 7, 0, 1, 3], p=[1.0, 1.0, 1.0, 0.9, 0.8, 0.6, 1.0, 1.0], m=[0.0] * 4 + [0.02] * 4)


def test_long_lists_and_wide_nuclei():
    """top-k on both sides of the bound of 512, with more ids than the list of 1024 above the bound or in the nucleus, and logits of a wide span."""
    g = torch.Generator().manual_seed(13)
    for scale in (2.5, 40.0):
        x = torch.randn((8, 30000), generator=g) * scale
        x[6, 100:2000] = x[6].max()                                     # more best ids than the list holds
        u = torch.rand((8,), generator=g, dtype=torch.float64).tolist()
        check(x, u, t=[1.0, 1.0, 3.0, 2.0, 1.0, 4.0, 1.0, 2.0], k=[511, 512, 513, 1500, 20000, 0, 700, 0], p=[1.0, 0.9, 1.0, 0.99, 1.0, 0.97, 0.5, 0.9])


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_rows_whose_first_ids_are_masked(dt):
    """As under a rule that leaves only the last ids of the vocabulary: nothing of what comes first says how the logits are spread."""
    g = torch.Generator().manual_seed(14)
    x = (torch.randn((8, 20000), generator=g) * 2.5).to(dt)
    x[:, :18500] = -math.inf
    u = torch.rand((8,), generator=g, dtype=torch.float64).tolist()
    check(x, u, t=[1.0] * 8, k=[0, 40, 0, 600, 1, 1499, 0, 5], p=[1.0, 1.0, 0.9, 1.0, 1.0, 0.95, 0.5, 0.7], m=[0.0] * 6 + [0.05] * 2)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_rows_of_infinities_wherever_the_drawn_one_lies(dt):
    """The drawn infinity in every lane and element of a wave's load, in the first, a middle and the last group, alone and among others."""
    v = 3000
    at = torch.cat([torch.arange(0, 520), torch.arange(1400, 1500), torch.arange(v - 300, v)])
    x = torch.zeros((len(at), v), dtype=dt)
    x[torch.arange(len(at)), at] = math.inf
    u = torch.rand(len(at), generator=torch.Generator().manual_seed(21), dtype=torch.float64).tolist()
    r = check(x, u)
    assert torch.equal(r.id.cpu().long(), at)
    x[:, [7, 900, 2999]] = math.inf
    check(x, u)
    check(x, u, k=[2] * len(at))
    check(x, u, t=[0.0] * len(at))


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("v", [900, 40000])
def test_min_p_below_the_weights_steps(dt, v):
    """min_p from 1e-14 to float32's smallest: ids too light to be drawn are still counted or left out as the rule says."""
    g = torch.Generator().manual_seed(22)
    m = [1e-14, 1e-16, 1e-18, 1e-20, 1e-25, 1e-38, 1e-44, 1e-30, 1e-22]
    n = len(m)
    x = torch.randn((n, v), generator=g) * 12
    x[:, 11] = 40.0
    x[-1, 5:200] = torch.finfo(dt).min
    x = x.to(dt)
    u = torch.rand(n, generator=g, dtype=torch.float64).tolist()
    check(x, u, m=m)
    check(x, u, t=[0.5] * n, m=m)
    check(x, u, t=[0.7] * n, k=[50, 0, 700, 0, 880, 0, 3, 0, 0], p=[1.0, 0.9] * 4 + [1.0], m=m)
