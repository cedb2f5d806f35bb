"""GPU: paged-cache operators where the inputs' sizes lie far apart, and where lengths on the device and numbers of the host disagree.

Attention is held to the formula in 64 bits with a bound that looks only at the keys a row sees:
    |o - o64| <= h_out |o| + (h_p + 2^-15) A + n 2^-21 max_j(p_j amax_j) / l + half a subnormal step of the result's type
h_out, h_p, A, l as in test_gpu_kv_ops.py.  The third term is f16's subnormal terms: each is off by at most 2^-25, the row's largest term p_j s_j (s_j a value row's
scale) is held at 2^-3 or above, a code weighs at most amax_j / s_j <= 448, and amax_j > 224 s_j: 2^-25 2^3 2 = 2^-21 of max_j(p_j amax_j) a key."""
import math

import pytest

torch = pytest.importorskip("torch")
from speaksense_amd import ops  # noqa: E402
from test_gpu_kv_ops import DT, Step, quantise  # noqa: E402

pytestmark = pytest.mark.gpu

KINDS8 = ["e4m3", "int8"]


def attend_seen(st, q, scale, causal):
    """CPU, 64 bits: result and its bound of the rows that a sequence owns."""
    groups = q.shape[1] // st.heads
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros_like(out)
    half_out = torch.finfo(st.dt).eps / 2
    half_p = torch.finfo(torch.bfloat16 if st.kind == "same" and st.dt == torch.bfloat16 else torch.float16).eps / 2
    step = torch.finfo(st.dt).tiny * half_out
    for s in range(len(st.lens)):
        a, b = st.starts[s], st.starts[s + 1]
        k, v = st.dense(s, "k").double(), st.dense(s, "v").double()
        pos = torch.arange(st.lens[s] - (b - a), st.lens[s])
        seen = torch.arange(st.lens[s])[None] <= pos[:, None] if causal else torch.ones(b - a, st.lens[s], dtype=torch.bool)
        for h in range(q.shape[1]):
            x = torch.where(seen, (q[a:b, h].double() @ k[:, h // groups].t()) * scale, -math.inf)
            p = torch.exp(x - x.amax(-1, keepdim=True))
            l, w = p.sum(-1, keepdim=True), v[:, h // groups]
            out[a:b, h] = p @ w / l
            most = (p * w.abs().amax(-1)).amax(-1, keepdim=True)
            tol[a:b, h] = half_out * out[a:b, h].abs() + (half_p + 2.0 ** -15) * (p @ w.abs() / l) + seen.sum(-1, keepdim=True) * 2.0 ** -21 * most / l + step
    return out, tol


def refill(st, k, v):
    """New contents of a Step's cache: float32 rows [n_pages, heads, page, dim]."""
    k, v = k.to(st.dt), v.to(st.dt)
    if st.kind == "same":
        st.k, st.v = k, v
    else:
        (st.k, st.ks), (st.v, st.vs) = quantise(k, st.kind), quantise(v, st.kind)


def scored_step(lens, new, dim, kind, dt, seed=0):
    """Keys that score 0.3 randn, and a way to give a position a score and its value row a size."""
    st = Step(lens, [new] * len(lens), 1, dim, 16, kind, dt, seed=seed)
    k = torch.randn(st.k.shape, generator=st.g) * 0.3
    k[..., 0] = 0
    v = torch.randn(st.k.shape, generator=st.g)
    q = (torch.randn((st.n, 3, dim), generator=st.g) * 0.3).to(st.dt)
    q[..., 0] = 4.0

    def put(s, pos, log2_score, log2_size):
        pg, r = int(st.table[s, pos // 16]), pos % 16
        k[pg, 0, r, 0] = log2_score * math.log(2.0) * dim ** 0.5 / 4.0
        v[pg, 0, r] *= 2.0 ** log2_size

    return st, k, v, q, put


def hold(st, q, causal=True):
    st.cuda()
    want, tol = attend_seen(st, q, st.dim ** -0.5, causal)
    got = ops.kv_attention(st.cache, st.batch, q.cuda(), causal=causal).cpu().double()
    over = (got - want).abs() - tol
    assert not torch.isnan(got).any() and float(over.max()) <= 0, (float(over.max()), int((over > 0).sum()), over.numel())


# new tokens a sequence and its lengths: the few-row kernel, the tile kernel, either with its keys cut
SHAPES = [(1, [180, 333]), (40, [180, 333]), (1, [3000, 65]), (40, [2500])]


@pytest.mark.parametrize("kind", KINDS8)
@pytest.mark.parametrize("dt,gap,base", [("bf16", 24, 0), ("bf16", 60, -30), ("f16", 20, -8)])
@pytest.mark.parametrize("new,lens", SHAPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_values_far_below_the_largest(kind, dt, gap, base, new, lens, dim):
    """Value rows 2^gap times the others: one that only the last token sees; one that all see and that weighs little or as much as the rest; one small row of nearly
    all weight among them."""
    for low in (0, 30):
        st, k, v, q, put = scored_step(lens, new, dim, kind, dt)
        v *= 2.0 ** base
        for s, n in enumerate(lens):
            put(s, n - 1, 0, gap)                          # the last position
        refill(st, k, v)
        hold(st, q)
        for s, n in enumerate(lens):
            put(s, n // 3, -gap - low, gap)
        refill(st, k, v)
        hold(st, q)
        hold(st, q, causal=False)
    st, k, v, q, put = scored_step(lens, new, dim, kind, dt)
    v *= 2.0 ** (base + gap)
    for s, n in enumerate(lens):
        put(s, 1, 20, -gap)
    refill(st, k, v)
    hold(st, q)


@pytest.mark.parametrize("kind", KINDS8)
@pytest.mark.parametrize("new,lens", SHAPES)
def test_values_of_subnormal_scales(kind, new, lens):
    """bfloat16 values near the smallest normal number: an int8 row's scale then is subnormal, an e4m3 row's the smallest there is."""
    st, k, v, q, put = scored_step(lens, new, 64, kind, "bf16")
    refill(st, k, v * 2.0 ** -122)
    hold(st, q)


@pytest.mark.parametrize("kind", KINDS8)
@pytest.mark.parametrize("new", [1, 40])
def test_values_that_rise_and_fall_along_the_keys(kind, new):
    """Sizes that grow by 2^2 every few keys, against falling scores, and the other way round: the running scale moves in most tiles, and each row's largest term with it."""
    for up in (1, -1):
        st, k, v, q, put = scored_step([300, 140], new, 64, kind, "bf16")
        for s, n in enumerate(st.lens):
            for p in range(n):
                put(s, p, -up * (p // 5) * 2 if p % 7 else 0, up * (p // 5) * 2 - (0 if up > 0 else -60))
        refill(st, k, v)
        hold(st, q)


# ---------------------------------------------------------------------------------------------------------------------------------
# spans longer than the host's max_new (q_start lies on the device and may change under a captured graph)
# ---------------------------------------------------------------------------------------------------------------------------------
def raw_attention(st, q, max_new, max_len, causal=True):
    """The C call with results filled with 7 and a workspace of NaN."""
    b = ops.KvBatch(st.batch.page_table, st.batch.q_start, st.batch.kv_len, n_tokens=st.n, max_new=max_new, max_len=max_len)
    heads, L = q.shape[1], ops._lib()
    out, lse = torch.full(q.shape, 7.0, dtype=st.dt, device="cuda"), torch.full(q.shape[:2], 7.0, device="cuda")
    need = L.ss_kv_attention_workspace(st.cache._c, b._c, heads)
    work = torch.full((need // 4 + 4,), math.nan, device="cuda")
    rows = lambda t: ops._rows(t, "t", st.cache, b, heads)  # noqa: E731
    assert L.ss_kv_attention(st.cache._c, b._c, rows(q), heads, st.dim ** -0.5, 1 if causal else 0, rows(out), lse.data_ptr(), work.data_ptr(), need, 0, ops._stream(0)) == 0
    return out.cpu(), lse.cpu(), need


@pytest.mark.parametrize("kind,dt,dim", [("same", "bf16", 64), ("int8", "f16", 128)])
@pytest.mark.parametrize("max_new,groups", [(1, 1), (1, 2), (3, 5), (2, 20), (33, 2)])      # the last two: the tile kernel
@pytest.mark.parametrize("lens,news", [([60, 90], [3, 40]), ([3000, 700, 50], [3, 40, 1])])
@pytest.mark.parametrize("causal", [True, False])
def test_spans_longer_than_max_new(kind, dt, dim, max_new, groups, lens, news, causal):
    """Their first max_new tokens are computed, at their positions; results of the rest are left as they were, with and without a cut over the keys."""
    st = Step(lens, news, 1, dim, 16, kind, dt, extra_rows=2)
    st.cuda()
    q = torch.randn((st.n, groups, dim), generator=st.g).to(st.dt)
    want, tol, wlse = st.attend(q, dim ** -0.5, causal)
    out, lse, need = raw_attention(st, q.cuda(), max_new, max(lens), causal)
    assert (need > 0) == (max(lens) > 512)
    done = torch.zeros(st.n, dtype=torch.bool)
    for s, n in enumerate(news):
        done[st.starts[s]:st.starts[s] + min(n, max_new)] = True
    assert ((out.double() - want).abs() <= tol)[done].all() and ((lse.double() - wlse).abs() <= 2.0 ** -12)[done].all()
    assert (out[~done] == 7.0).all() and (lse[~done] == 7.0).all()


# ---------------------------------------------------------------------------------------------------------------------------------
# append of infinities
# ---------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["same", "e4m3", "int8"])
@pytest.mark.parametrize("dim", [64, 128])
def test_append_of_infinities(kind, dt, dim):
    """They read back with their signs, at either end of a row and beside the largest finite numbers; a NaN stays one; rows beside them are what they are without."""
    st = Step([32], [32], 2, dim, 16, kind, dt)
    cache, batch = st.cuda()
    x = st.rows((32, 2, dim))
    plain = x.clone()
    inf, nan, big = math.inf, math.nan, torch.finfo(st.dt).max
    marks = {0: {0: inf}, 3: {dim - 1: -inf}, 4: {0: -inf, 1: inf, 17: -inf, 40: inf}, 9: {5: inf, 6: big, 7: -big}, 10: {8: nan}, 16: {2: nan, 3: inf}, 17: dict.fromkeys(range(dim), -inf)}
    for t, m in marks.items():
        for i, v in m.items():
            x[t, 1, i] = v
    want = []
    for y in (plain, x):
        ops.kv_append(cache, batch, y.cuda(), (-y).cuda())
        want.append([t.cpu() for t in ops.kv_read(cache, batch)])
    for sign, without, got in ((1, want[0][0], want[1][0]), (-1, want[0][1], want[1][1])):
        rest = [t for t in range(32) if t not in marks]
        assert torch.equal(got[rest], without[rest]) and torch.equal(got[:, 0], without[:, 0])
        for t, m in marks.items():
            mixed = nan in m.values() and kind != "same"
            for i, v in m.items():
                g = float(got[t, 1, i])
                assert math.isnan(g) if math.isnan(v) or (mixed and math.isinf(v)) else g == sign * v if math.isinf(v) else True, (t, i, v, g)
        if kind == "same":
            assert torch.equal(torch.nan_to_num(got, 7.0), torch.nan_to_num(sign * x, 7.0))


@pytest.mark.parametrize("kind", ["same", "e4m3", "int8"])
def test_a_cache_of_one_head_seen_the_other_way_round(kind):
    """[page, row, head] tensors of one head are [page, head, row] ones: the stride over a single head says nothing."""
    st = Step([40, 33], [40, 33], 1, 64, 16, kind, "f16")
    plain, batch = st.cuda()
    turn = lambda t: torch.empty_strided(t.shape, (t.stride(0), t.stride(2)) + t.stride()[2:], dtype=t.dtype, device="cuda").copy_(t)  # noqa: E731
    turned = [None if t is None else turn(t) for t in (plain.k, plain.v, plain.k_scale, plain.v_scale)]
    assert turned[0].stride(1) == 64 and (kind == "same" or turned[2].stride(1) == 1)
    cache = ops.KvCache(*turned, kind=kind, dtype=st.dt)
    x = [st.rows((st.n, 1, 64)).cuda() for _ in "kvq"]
    for c in (plain, cache):
        ops.kv_append(c, batch, x[0], x[1])
    assert all(torch.equal(a, b) for a, b in zip(ops.kv_read(plain, batch), ops.kv_read(cache, batch)))
    assert torch.equal(ops.kv_attention(plain, batch, x[2]), ops.kv_attention(cache, batch, x[2]))
    with pytest.raises(ValueError, match="contiguous"):
        ops.KvCache(torch.zeros((4, 16, 2, 64), dtype=torch.float16, device="cuda").transpose(1, 2), torch.zeros((4, 2, 16, 64), dtype=torch.float16, device="cuda"))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["same", "e4m3", "int8"])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("n,log2,cut", [(60000, 20, True), (4000, 20, False), (300, 18, False)])
def test_a_long_tail_below_one_key(dt, kind, new, n, log2, cut):
    """One key takes nearly all weight and holds a value of zero: what comes out is the sum of the tail, whose probabilities all are alike, so that a rounding of
    theirs would show in full (cut False: one workgroup takes all keys, as in a call of many sequences).  Bound: as above, with the tail's own terms normal f16 numbers (2^7 2^-20 > 2^-14; 8-bit caches: lifted to the row's largest)."""
    st = Step([n], [new], 1, 64, 256, kind, dt)
    k = torch.zeros(st.k.shape)
    v = torch.ones(st.k.shape)
    pg, r = int(st.table[0, 3 // 256]), 3
    k[pg, 0, r, 0] = (log2 - math.log2(1.03)) * math.log(2.0) * 8 / 4
    v[pg, 0, r] = 0
    refill(st, k, v)
    q = torch.zeros((st.n, 3, 64), dtype=st.dt)
    q[..., 0] = 4.0
    st.cuda()
    x = float(st.dense(0, "k")[3, 0, 0]) * 4 / 8          # the cached key's score
    one = float(st.dense(0, "v")[0, 0, 0])
    seen = torch.arange(n - new, n, dtype=torch.float64) if new > 1 else torch.tensor([n - 1.0], dtype=torch.float64)
    p = math.exp(-x)
    want = (seen * p * one / (1 + seen * p))[:, None, None]
    half_out, half_p = torch.finfo(st.dt).eps / 2, torch.finfo(torch.bfloat16 if kind == "same" and dt == "bf16" else torch.float16).eps / 2
    batch = ops.KvBatch(st.batch.page_table, st.batch.q_start, st.batch.kv_len, n_tokens=st.n, max_new=new, max_len=n if cut else 1)
    assert (ops._lib().ss_kv_attention_workspace(st.cache._c, batch._c, 3) > 0) == cut
    got = ops.kv_attention(st.cache, batch, q.cuda()).cpu().double()
    assert ((got - want).abs() <= (half_out + half_p + 2.0 ** -15 + 2.0 ** -20) * want).all(), float(((got - want) / want).abs().max())


@pytest.mark.parametrize("kind", ["same", "e4m3", "int8"])
@pytest.mark.parametrize("new,groups", [(1, 8), (40, 2)])
def test_queries_of_nan_and_infinity_keep_to_themselves(kind, new, groups):
    """Rows of the same tile, wave and workgroup stay within their bounds beside rows that can only be NaN."""
    st = Step([700, 90, 64], [new] * 3, 1, 64, 16, kind, "bf16")
    q = (torch.randn((st.n, groups, 64), generator=st.g) * 1.5).to(st.dt)
    st.cuda()
    want, tol = attend_seen(st, q, 0.125, True)
    bad = torch.zeros(q.shape[:2], dtype=torch.bool)
    for t, h, v in ((0, 1, math.nan), (new - 1, 0, math.inf), (st.n - 1, 1, -math.inf)):
        q[t, h, 5] = v
        bad[t, h] = True
    for max_len in (1, 700):
        b = ops.KvBatch(st.batch.page_table, st.batch.q_start, st.batch.kv_len, n_tokens=st.n, max_new=new, max_len=max_len)
        got = ops.kv_attention(st.cache, b, q.cuda()).cpu().double()
        assert ((got - want).abs() <= tol)[~bad].all() and torch.isnan(got[bad]).all()


@pytest.mark.parametrize("kind", ["same", "e4m3", "int8"])
@pytest.mark.parametrize("new,lens", SHAPES)
def test_scores_beyond_2_to_the_12(kind, new, lens):
    """Scores of thousands in log2 units that differ by halves, of exact products, over value rows of very different sizes; in each sequence they rise once from some
    hundreds to thousands, so that the difference is formed first from there on."""
    st = Step(lens, [new] * len(lens), 1, 64, 16, kind, "bf16")
    top = {"same": 127.0, "e4m3": 448.0, "int8": 127.0}[kind]          # scale 1: the cache holds these keys exactly
    k = torch.zeros(st.k.shape)
    k[..., 2] = top
    k[..., 1] = torch.randint(0, 11, k.shape[:3], generator=st.g).float()
    v = torch.randn(k.shape, generator=st.g) * torch.exp2(torch.randint(-20, 21, k.shape[:3] + (1,), generator=st.g).float())
    for s, n in enumerate(lens):
        for p in range(n):
            k[int(st.table[s, p // 16]), 0, p % 16, 0] = 8.0 if p < n // 2 else 120.0
    refill(st, k, v)
    q = torch.zeros((st.n, 3, 64), dtype=st.dt)
    q[..., 0], q[..., 1] = 80.0, 1.0                      # 80 x 120 / 2 = 4800 in log2 units
    q[:, 1] = -q[:, 1]
    q[:, 2, 0] = 1.0
    st.cuda()
    scale = 0.5 * math.log(2.0)
    for causal in (True, False):
        want, tol = attend_seen(st, q, scale, causal)
        got = ops.kv_attention(st.cache, st.batch, q.cuda(), scale=scale, causal=causal).cpu().double()
        assert not torch.isnan(got).any() and ((got - want).abs() <= tol).all(), float(((got - want).abs() - tol).max())
