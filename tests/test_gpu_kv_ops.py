"""GPU: paged cache append / read / attention (speaksense_amd.ops) against plain implementations.

Append and read are held exactly: the codes, scales and 16-bit values have one right answer (a power of two, an IEEE division, one rounding each), which torch
gives on the CPU.  Attention is held to the formula in 64 bits with a bound of its own roundings, per element:
    |o - o64| <= h_out |o| + (h_p + 2^-15) A + n 2^-24 vmax / l
h_out, h_p: half a step of the result's type and of the type the probabilities are rounded to (bf16 2^-8, f16 2^-11); A = sum_j p_j |v_j| / sum_j p_j, what a
relative error of every probability can move; 2^-15: float32 scores up to 2^7 in log2 units (2^-24 2^7 2^1 for the score's product and sum) and exp2; the
last term: n probabilities that f16 holds as subnormals (half a step 2^-25, value scales taken off within a factor 2), l = sum_j exp(x_j - max) >= 1."""
import math

import pytest

torch = pytest.importorskip("torch")
from speaksense_amd import ops  # noqa: E402

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def _exponent(amax):
    bits = amax.view(torch.int32)
    return (((bits >> 23) & 255) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(1, 253)


def _pow2(e):
    return (e.int() << 23).view(torch.float32)


def quantise(x, kind):
    """CPU: codes, scales of rows [..., D]."""
    x = x.float()
    amax = x.abs().amax(-1)
    if kind == "e4m3":
        e = _exponent(amax)
        return (x * _pow2(254 - e)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), e.to(torch.uint8)
    s = amax / 127.0
    return torch.round(x / torch.where(s > 0, s, torch.ones_like(s))[..., None]).clamp(-127, 127).to(torch.int8), s


def values(codes, scale, kind):
    """CPU: float32 values (exact for e4m3; one product for int8)."""
    if kind == "same":
        return codes.float()
    return codes.view(torch.float8_e4m3fn).float() * _pow2(scale)[..., None] if kind == "e4m3" else codes.float() * scale[..., None]


class Step:
    """A cache filled with random rows on the CPU, its copy on the GPU, and the sequences of a step."""

    def __init__(self, lens, news, heads, dim, page, kind, dt, seed=0, spare=2, extra_rows=0, extra_pages=0):
        self.g = torch.Generator().manual_seed(seed)
        self.kind, self.dt, self.heads, self.dim, self.page = kind, DT[dt], heads, dim, page
        self.lens, self.news = lens, news
        need = [-(-n // page) for n in lens]
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, generator=self.g).tolist()
        self.table = torch.full((len(lens), max(need + [1]) + extra_pages), -1, dtype=torch.int32)
        for i, n in enumerate(need):
            self.table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.starts = [0]
        for n in news:
            self.starts.append(self.starts[-1] + n)
        self.n = self.starts[-1] + extra_rows
        x = [self.rows((self.n_pages, heads, page, dim)) for _ in "kv"]
        if kind == "same":
            self.k, self.v, self.ks, self.vs = x[0], x[1], None, None
        else:
            (self.k, self.ks), (self.v, self.vs) = quantise(x[0], kind), quantise(x[1], kind)

    def rows(self, shape):
        x = torch.randn(shape, generator=self.g)
        x[..., 3] *= 5
        return x.to(self.dt)

    def cuda(self):
        c = lambda t: None if t is None else t.cuda()  # noqa: E731
        self.cache = ops.KvCache(c(self.k), c(self.v), c(self.ks), c(self.vs), kind=self.kind, dtype=self.dt)
        self.batch = ops.KvBatch(self.table.cuda(), torch.tensor(self.starts, dtype=torch.int32).cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda(), n_tokens=self.n,
                                 max_new=max(self.news + [0]), min_new=min(self.news + [0]), max_len=max(self.lens + [0]))
        return self.cache, self.batch

    def dense(self, s, name):
        """CPU: values [len, heads, dim] of sequence s, NaN where there is no page."""
        n = self.lens[s]
        out = torch.full((n, self.heads, self.dim), math.nan)
        for p in range(n):
            pg = int(self.table[s, p // self.page])
            if 0 <= pg < self.n_pages:
                r = p % self.page
                scale = getattr(self, name + "s")
                out[p] = values(getattr(self, name)[pg, :, r], None if scale is None else scale[pg, :, r], self.kind)
        return out

    def attend(self, q, scale, causal):
        """CPU, 64 bits: result, its bound, lse; rows without a sequence stay NaN."""
        groups = q.shape[1] // self.heads
        out = torch.full(q.shape, math.nan, dtype=torch.float64)
        tol, lse = torch.zeros_like(out), torch.full(q.shape[:2], math.nan, dtype=torch.float64)
        half_out = torch.finfo(self.dt).eps / 2
        half_p = torch.finfo(torch.bfloat16 if self.kind == "same" and self.dt == torch.bfloat16 else torch.float16).eps / 2
        for s in range(len(self.lens)):
            a, b = self.starts[s], self.starts[s + 1]
            if a == b:
                continue
            k, v = self.dense(s, "k").double(), self.dense(s, "v").double()
            held = ~torch.isnan(k[:, 0, 0])
            pos = torch.arange(self.lens[s] - (b - a), self.lens[s])
            seen = held[None] & ((torch.arange(self.lens[s])[None] <= pos[:, None]) if causal else torch.ones(b - a, self.lens[s], dtype=torch.bool))
            v = torch.where(held[:, None, None], v, 0.0)
            for h in range(q.shape[1]):
                x = (q[a:b, h].double() @ torch.where(held[:, None], k[:, h // groups], 0.0).t()) * scale
                x = torch.where(seen, x, -math.inf)
                m = x.amax(-1, keepdim=True) if x.shape[1] else torch.full((b - a, 1), -math.inf, dtype=torch.float64)
                p = torch.exp(x - torch.where(m > -math.inf, m, 0.0))
                l = p.sum(-1, keepdim=True)
                d = torch.where(l > 0, l, 1.0)
                w = v[:, h // groups]
                out[a:b, h] = p @ w / d
                vmax = float(w.abs().max()) if w.numel() else 0.0
                tol[a:b, h] = half_out * out[a:b, h].abs() + (half_p + 2.0 ** -15) * (p @ w.abs() / d) + self.lens[s] * 2.0 ** -24 * vmax / d + 2.0 ** -24
                lse[a:b, h] = torch.where(l > 0, torch.log(d) + m, torch.full_like(m, -math.inf))[:, 0]
        return out, tol, lse


def check_attention(st, heads_q, causal, scale=None, q=None, lse=True):
    st.cuda()
    q = torch.randn((st.n, heads_q, st.dim), generator=st.g).mul(1.5).to(st.dt) if q is None else q
    scale = st.dim ** -0.5 if scale is None else scale
    want, tol, wlse = st.attend(q, scale, causal)
    out = torch.full(q.shape, 7.0, dtype=st.dt, device="cuda")
    got, glse = ops.kv_attention(st.cache, st.batch, q.cuda(), scale=scale, causal=causal, out=out, return_lse=True)
    assert got.data_ptr() == out.data_ptr()
    got, glse = got.cpu().double(), glse.cpu().double()
    owned = st.starts[-1]
    assert (got[owned:] == 7.0).all(), "rows behind the last sequence were written"
    bad = (got[:owned] - want[:owned]).abs() - tol[:owned]
    assert not torch.isnan(got[:owned]).any() and float(bad.max() if bad.numel() else -1) <= 0, (float(bad.max()), int((bad > 0).sum()))
    empty = wlse[:owned] == -math.inf
    assert (glse[:owned][empty] == -math.inf).all() and (got[:owned][empty] == 0).all()
    err = (glse[:owned] - wlse[:owned])[~empty].abs()
    assert err.numel() == 0 or float(err.max()) <= 2.0 ** -15 + 2.0 ** -23 * float(wlse[:owned][~empty].abs().max())
    return got


KINDS = ["same", "e4m3", "int8"]


# ---------------------------------------------------------------------------------------------------------------------------------
# append / read
# ---------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,page,heads", [(64, 16, 3), (64, 256, 20), (128, 32, 1), (128, 64, 5)])
def test_append_then_read(dt, kind, dim, page, heads):
    lens, news = [1, 40, 17, 0, 300, 16, 33], [1, 7, 17, 0, 130, 0, 2]
    st = Step(lens, news, heads, dim, page, kind, dt, extra_rows=3)
    cache, batch = st.cuda()
    k, v = st.rows((st.n, heads, dim)), st.rows((st.n, heads, dim))
    k[2] = 0                                             # a row of zeros
    k[3] *= 2.0 ** -8
    v[4, 0, 1:] = 0
    want = [t if t is None else t.clone() for t in (st.k, st.v, st.ks, st.vs)]
    for s in range(len(lens)):
        for i in range(news[s]):
            p, t = lens[s] - news[s] + i, st.starts[s] + i
            pg, r = int(st.table[s, p // page]), p % page
            for j, x in enumerate((k[t], v[t])):
                if kind == "same":
                    want[j][pg, :, r] = x
                else:
                    want[j][pg, :, r], want[2 + j][pg, :, r] = quantise(x, kind)
    ops.kv_append(cache, batch, k.cuda(), v.cuda())
    for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        assert w is None or torch.equal(got.cpu(), w)    # every code of every page: nothing else was touched
    # whole contexts back, more rows than the sequences own
    st2 = Step.__new__(Step)
    st2.__dict__.update(st.__dict__)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    b2 = ops.KvBatch(batch.page_table, torch.tensor(starts, dtype=torch.int32).cuda(), batch.kv_len, n_tokens=starts[-1] + 2, max_new=max(lens))
    out = [torch.full((starts[-1] + 2, heads, dim), 7.0, dtype=st.dt, device="cuda") for _ in "kv"]
    ops.kv_read(cache, b2, out=out)
    st.k, st.v, st.ks, st.vs = want
    for name, o in zip("kv", out):
        assert torch.equal(o[:-2].cpu(), torch.cat([st.dense(s, name) for s in range(len(lens))]).to(st.dt))
        assert (o[-2:] == 7.0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_append_ignores_what_does_not_exist(kind):
    """Pages outside the cache, spans that leave the rows, positions before the start or behind the table: dropped; the rest is written."""
    st = Step([20, 20, 5, 64, 20], [2, 2, 8, 3, 2], 2, 64, 16, kind, "f16", extra_pages=0)
    st.cuda()
    st.table[0, 1] = st.n_pages                          # one past the end
    st.table[1, 1] = -7
    lens = torch.tensor([20, 20, 5, 1 << 30, 20], dtype=torch.int32)     # sequence 3: far behind the table
    starts = torch.tensor([0, 2, 4, 12, 15, 17], dtype=torch.int32)      # sequence 2: 8 new tokens of 5 positions
    k, v = st.rows((17, 2, 64)), st.rows((17, 2, 64))
    want = [t if t is None else t.clone() for t in (st.k, st.v, st.ks, st.vs)]
    for s, first, at in ((2, 4, range(-3, 5)), (4, 15, range(18, 20))):
        for i, p in enumerate(at):
            if p < 0:
                continue
            pg, r = int(st.table[s, p // 16]), p % 16
            for j, x in enumerate((k[first + i], v[first + i])):
                if kind == "same":
                    want[j][pg, :, r] = x
                else:
                    want[j][pg, :, r], want[2 + j][pg, :, r] = quantise(x, kind)
    b = ops.KvBatch(st.table.cuda(), starts.cuda(), lens.cuda(), n_tokens=17, max_new=8)
    ops.kv_append(st.cache, b, k.cuda(), v.cuda())
    for got, w in zip((st.cache.k, st.cache.v, st.cache.k_scale, st.cache.v_scale), want):
        assert w is None or torch.equal(got.cpu(), w)
    for bad in ([0, 2, 4, 12, 15, 18], [0, 2, 1, 0, -3, 2], [5, 4, 3, 2, 1, 0], [-9, -8, -7, -6, -5, -4], [1 << 30, 1 << 30, 1 << 30, 1 << 30, 1 << 30, 1 << 30]):
        b = ops.KvBatch(st.table.cuda(), torch.tensor(bad, dtype=torch.int32).cuda(), torch.tensor([20, 20, 5, 64, 20], dtype=torch.int32).cuda(), n_tokens=17, max_new=8)
        ops.kv_append(st.cache, b, k.cuda(), v.cuda())   # every write lands in the cache or nowhere
        r = ops.kv_read(st.cache, b, out=[torch.full((17, 2, 64), 7.0, dtype=torch.float16, device="cuda") for _ in "kv"])
        o = ops.kv_attention(st.cache, b, st.rows((17, 2, 64)).cuda())
        torch.cuda.synchronize()
        assert o.shape == (17, 2, 64) and len(r) == 2
    r = ops.kv_read(st.cache, ops.KvBatch(st.table.cuda(), starts.cuda(), lens.cuda(), n_tokens=17, max_new=8))
    assert (r[0][:4] == 0).all() and (r[0][4:7] == 0).all() and (r[0][12:15] == 0).all() and not (r[0][15:] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_append_special_values(kind):
    """Largest and smallest magnitudes, borders of the exponent rule, ties of the rounding; a NaN stays one."""
    st = Step([16], [16], 1, 64, 16, kind, "bf16")
    cache, batch = st.cuda()
    x = torch.zeros(16, 1, 64)
    x[0, 0, 0] = 3e38
    x[1, 0, :2] = torch.tensor([1e-38, -1e-38])
    x[2, 0, :4] = torch.tensor([448.0, 1.0, -0.5, 17.0])
    x[3, 0, :4] = torch.tensor([450.0, 1.0, 0.0, 26.0])
    x[4, 0] = torch.arange(64) * 0.25
    x[5, 0] = -torch.arange(64).float() - 64
    x[6, 0, :3] = torch.tensor([127.0, 0.5, 1.5])
    x[7, 0, :4] = torch.tensor([127.0, 2.5, -3.5, -126.5])
    x[8, 0, 63] = 1.0
    x[9, 0] = 2.0 ** -100
    k = x.to(torch.bfloat16)
    ops.kv_append(cache, batch, k.cuda(), k.cuda())
    if kind == "same":
        want, scale = k, None
    else:
        want, scale = quantise(k, kind)
        assert torch.equal(cache.k_scale[int(st.table[0, 0]), 0].cpu(), scale[:, 0])
    assert torch.equal(cache.k[int(st.table[0, 0]), 0].cpu().view(torch.uint8), want[:, 0].contiguous().view(torch.uint8))
    k[3, 0, 9] = math.nan
    ops.kv_append(cache, batch, k.cuda(), k.cuda())
    r = ops.kv_read(cache, batch)[0].cpu()
    assert torch.isnan(r[3, 0, 9]) and not torch.isnan(r[[0, 1, 2, 4, 5, 6, 7]]).any()


# ---------------------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("heads,groups", [(3, 1), (1, 8), (2, 5)])
def test_attention_single_tokens(dt, kind, dim, page, heads, groups):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 0, 500]
    check_attention(Step(lens, [1] * len(lens), heads, dim, page, kind, dt, extra_rows=2, extra_pages=3), heads * groups, True)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 32), (128, 16)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_chunks(dt, kind, dim, page, causal):
    """Spans from none to several tiles, short sequences (few rows) among long ones, more new tokens than positions never."""
    lens, news = [70, 1, 200, 64, 0, 129, 300, 5], [70, 1, 3, 64, 0, 65, 140, 5]
    check_attention(Step(lens, news, 2, dim, page, kind, dt, extra_rows=3), 4, causal)


@pytest.mark.parametrize("groups,news", [(17, [1, 1]), (16, [1, 1]), (3, [5, 6]), (4, [4, 5]), (1, [16, 17]), (32, [2, 3])])
def test_attention_around_sixteen_rows(groups, news):
    for causal in (True, False):
        check_attention(Step([90, 41], news, 2, 64, 16, "same", "f16"), 2 * groups, causal)
        check_attention(Step([90, 41], news, 1, 128, 16, "int8", "bf16"), groups, causal)


@pytest.mark.parametrize("kind,dt,dim", [("same", "f16", 64), ("same", "bf16", 128), ("e4m3", "bf16", 64), ("int8", "f16", 128)])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_cut_over_keys(kind, dt, dim, new):
    """Long contexts beside short ones: several key ranges per row, most of them empty for the short ones."""
    st = Step([3000, 1, 257, 700][: 4 if new == 1 else 1] + ([] if new == 1 else [41]), [new] * (4 if new == 1 else 2), 1, dim, 64, kind, dt)
    st.cuda()
    assert ops._lib().ss_kv_attention_workspace(st.cache._c, st.batch._c, 2) > 0
    check_attention(st, 2, True)
    check_attention(st, 2, False)


def test_attention_of_more_new_tokens_than_positions():
    """kv_len below the span: the first tokens sit before position 0 and see nothing (causal); without a mask all see all."""
    for causal in (True, False):
        st = Step([8, 70], [8, 70], 2, 64, 16, "same", "f16")
        st.cuda()
        q = torch.randn((78, 4, 64), generator=st.g).half()
        lens = torch.tensor([5, 33], dtype=torch.int32)
        b = ops.KvBatch(st.batch.page_table, st.batch.q_start, lens.cuda(), n_tokens=78, max_new=70)
        got, lse = ops.kv_attention(st.cache, b, q.cuda(), causal=causal, return_lse=True)
        if causal:
            assert (got[:3] == 0).all() and (got[8:45] == 0).all() and (lse[:3] == -math.inf).all() and (lse[3:8] > -math.inf).all()
            sub = Step.__new__(Step)
            sub.__dict__.update(st.__dict__)
            sub.lens, sub.news, sub.starts = [5, 33], [5, 33], [0, 5, 38]
            want, tol, _ = sub.attend(torch.cat([q[3:8], q[45:]]), 64 ** -0.5, True)
            have = torch.cat([got[3:8], got[45:]]).cpu().double()
            assert ((have - want).abs() <= tol).all()
        else:
            assert (lse > -math.inf).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 30])
def test_attention_with_pages_missing(kind, new):
    """Entries outside the cache hold nothing: their keys are masked, wherever they lie in a tile; a sequence of none gives zeros."""
    st = Step([200, 64, 130, 48], [new] * 4, 2, 64, 16, kind, "f16")
    st.table[0, 3] = -1
    st.table[0, 12] = st.n_pages                         # the tile that ends the sequence
    st.table[1] = -1
    st.table[2, 0:4] = 1 << 30
    check_attention(st, 4, False)
    check_attention(st, 4, True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_never_uses_what_lies_behind(kind, new, dim):
    """NaN and the types' largest values in rows behind the sequences' ends, in unused pages and in their scales."""
    st = Step([75, 130, 97], [min(new, 70)] * 3, 2, dim, 32, kind, "bf16", spare=3)
    used = torch.zeros(st.n_pages, 32, dtype=torch.bool)
    for s, n in enumerate(st.lens):
        for p in range(n):
            used[int(st.table[s, p // 32]), p % 32] = True
    free = ~used[:, None].expand(-1, 2, -1)
    for t in (st.k, st.v):
        t[free] = {"same": math.nan, "e4m3": 0x7F, "int8": -128}[kind]
    for t in (st.ks, st.vs):
        if t is not None:
            t[free] = 255 if kind == "e4m3" else math.nan
    check_attention(st, 2, True)
    check_attention(st, 2, False)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_of_uneven_scales(kind, dt, new):
    """Key and value rows whose sizes differ by factors up to 2^12 from row to row, rising and falling: the running scale moves both ways; zero rows."""
    st = Step([180, 333], [new] * 2, 1, 64, 16, kind, dt)
    f = torch.exp2(torch.randint(-6, 7, (st.n_pages, 1, 16, 1), generator=st.g).float())
    f[:, :, 5] = 0
    (st.k, st.ks), (st.v, st.vs) = quantise((torch.randn(st.k.shape, generator=st.g) * f / 64).to(st.dt), kind), quantise((torch.randn(st.k.shape, generator=st.g) * f).to(st.dt), kind)
    check_attention(st, 3, True)


@pytest.mark.parametrize("kind", ["same", "int8"])
def test_attention_of_large_and_tiny_bf16_queries(kind):
    st = Step([100, 60], [1, 50], 2, 64, 16, kind, "bf16")
    q = torch.randn((51, 4, 64), generator=st.g)
    q[0] *= 2.0 ** 60
    q[1] *= 2.0 ** -60
    q[2, 1] = 0
    q = q.bfloat16()
    for scale in (2.0 ** -62, 2.0 ** 58 / 8):
        keep = [0, 2] if scale < 1 else [1, 2]           # rows whose scores are of order 1 to 2^-2
        st.cuda()
        want, tol, _ = st.attend(q, scale, True)
        got = ops.kv_attention(st.cache, st.batch, q.cuda(), scale=scale).cpu().double()
        assert ((got - want).abs() <= tol)[keep].all()


def test_attention_of_scores_far_apart():
    """Scores that rise by hundreds from tile to tile (every tile moves the maximum) and that fall: nothing overflows, the far keys vanish."""
    for rising in (True, False):
        for new in (1, 20):
            st = Step([400], [new], 1, 64, 16, "same", "f16")
            for p in range(400):
                st.k[int(st.table[0, p // 16]), 0, p % 16] = 0
                st.k[int(st.table[0, p // 16]), 0, p % 16, 0] = (p if rising else 400 - p) * 0.25
            q = torch.zeros(new, 2, 64, dtype=torch.float16)
            q[..., 0] = 2.0
            q[..., 1, 0] = -2.0
            st.cuda()
            want, tol, wl = st.attend(q, 1.0, False)
            got, lse = ops.kv_attention(st.cache, st.batch, q.cuda(), scale=1.0, causal=False, return_lse=True)
            # scores reach 200 = 2^8.2 in log2 units: their float32 steps are 2^-15, twice
            assert ((got.cpu().double() - want).abs() <= tol + 2.0 ** -14 * want.abs().max()).all()
            assert ((lse.cpu().double() - wl).abs() <= 2.0 ** -13).all()


def test_strides_views_and_orders():
    """Queries out of a fused projection, results into a transposed tensor, keys and values that are views of one pool, a padded page table."""
    st = Step([40, 70, 129], [1, 20, 129], 4, 64, 16, "same", "bf16")
    plain = check_attention(st, 8, True, q=(q := torch.randn((st.n, 8, 64), generator=st.g).bfloat16()))
    pool = torch.full((st.n_pages, 2, 4, 16, 64), math.nan, dtype=torch.bfloat16, device="cuda")
    cache = ops.KvCache(pool[:, 0], pool[:, 1])
    cache.k.copy_(st.k)
    cache.v.copy_(st.v)
    fused = torch.full((st.n, 3 * 8 * 64 + 8), math.nan, dtype=torch.bfloat16, device="cuda")
    fused[:, 8 * 64:2 * 8 * 64] = q.reshape(st.n, -1).cuda()
    out = torch.full((8, st.n, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    table = torch.full((3, st.table.shape[1] + 5), 1 << 30, dtype=torch.int32, device="cuda")[:, : st.table.shape[1]]
    table.copy_(st.table)
    b = ops.KvBatch(table, st.batch.q_start, st.batch.kv_len, n_tokens=st.n, max_new=129, min_new=1, max_len=129)
    ops.kv_attention(cache, b, fused[:, 8 * 64:2 * 8 * 64].unflatten(1, (8, 64)), out=out.transpose(0, 1))
    assert torch.equal(out.transpose(0, 1).cpu().double(), plain)
    # a query broadcast over the heads
    one = torch.randn((st.n, 1, 64), generator=st.g).bfloat16().cuda()
    assert torch.equal(ops.kv_attention(cache, b, one.expand(-1, 8, -1)), ops.kv_attention(cache, b, one.repeat(1, 8, 1)))
    # append and read through the same views
    k = torch.randn((st.n, 4, 3, 64), generator=st.g).bfloat16().cuda()
    ops.kv_append(cache, b, k[:, :, 1], k[:, :, 2])
    r = torch.full((4, 2, st.n, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.kv_read(cache, b, out=(r[:, 0].transpose(0, 1), r[:, 1].transpose(0, 1)))
    assert torch.equal(r[:, 0].transpose(0, 1), k[:, :, 1]) and torch.equal(r[:, 1].transpose(0, 1), k[:, :, 2])


def test_refusals_of_the_python_layer():
    c = ops.KvCache.empty(4, 2, 16, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    b = ops.KvBatch(torch.zeros((1, 2), **i32), torch.zeros(2, **i32), torch.zeros(1, **i32), n_tokens=3, max_new=3)
    h = lambda *s, dtype=torch.float16: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    for call in (lambda: ops.kv_append(c, b, h(3, 2, 64, dtype=torch.bfloat16), h(3, 2, 64)), lambda: ops.kv_append(c, b, h(2, 2, 64), h(3, 2, 64)),
                 lambda: ops.kv_append(c, b, h(3, 3, 64), h(3, 2, 64)), lambda: ops.kv_read(c, b, out=(h(3, 2, 64), h(3, 2, 128))), lambda: ops.kv_attention(c, b, h(3, 2, 64).cpu()),
                 lambda: ops.kv_attention(c, b, h(3, 64, 2).transpose(1, 2)), lambda: ops.kv_attention(b, c, h(3, 2, 64)),
                 lambda: ops.KvBatch(torch.zeros((1, 2), **i32), torch.zeros(3, **i32), torch.zeros(1, **i32), n_tokens=3, max_new=3),
                 lambda: ops.KvBatch(torch.zeros((1, 2), device="cuda"), torch.zeros(2, **i32), torch.zeros(1, **i32), n_tokens=3, max_new=3),
                 lambda: ops.KvBatch(torch.zeros((1, 2), **i32), torch.zeros(2, **i32), torch.zeros(1, **i32), n_tokens=-1, max_new=3),
                 lambda: ops.KvBatch(torch.zeros((1, 2), **i32), torch.zeros(2, **i32), torch.zeros(1, **i32), n_tokens=1 << 32, max_new=3),
                 lambda: ops.KvCache(h(4, 2, 64, 16).transpose(2, 3), h(4, 2, 16, 64)), lambda: ops.KvCache(h(4, 2, 16, 64), h(4, 2, 16, 64), kind="int8", dtype=torch.float16),
                 lambda: ops.KvCache(h(4, 2, 16, 64), h(4, 2, 16, 64), h(4, 2, 16), h(4, 2, 16)), lambda: ops.KvCache(h(4, 2, 16, 64, dtype=torch.float32), h(4, 2, 16, 64)),
                 lambda: ops.KvCache(h(4, 2, 16, 64, dtype=torch.int8), h(4, 2, 16, 64, dtype=torch.int8), h(4, 2, 16), h(4, 2, 16), kind="int8", dtype=torch.float16)):
        with pytest.raises(ValueError):
            call()
    from speaksense_amd.binding import SpeakSenseError
    for call in (lambda: ops.KvCache.empty(4, 2, 24, 64), lambda: ops.KvCache.empty(4, 2, 16, 80)):
        bad = call()
        with pytest.raises(SpeakSenseError):
            ops.kv_attention(bad, b, h(3, 2, bad.head_dim))
    with pytest.raises(SpeakSenseError, match="multiple"):
        ops.kv_attention(c, b, h(3, 3, 64))
    with pytest.raises(SpeakSenseError, match="overlap"):
        ops.kv_read(c, b, out=(h(1, 2, 64).expand(3, -1, -1), h(3, 2, 64)))
    with pytest.raises(SpeakSenseError, match="aligned"):
        ops.kv_attention(c, b, h(3 * 2 * 64 + 8)[1:1 + 3 * 2 * 64].view(3, 2, 64))


def test_empty_calls():
    c = ops.KvCache.empty(4, 2, 16, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    for n_seqs, n_tokens in ((0, 0), (0, 3), (2, 0), (2, 3)):
        b = ops.KvBatch(torch.zeros((n_seqs, 2), **i32), torch.zeros(n_seqs + 1, **i32), torch.zeros(n_seqs, **i32), n_tokens=n_tokens, max_new=0)
        x = torch.full((n_tokens, 2, 64), 7.0, dtype=torch.float16, device="cuda")
        ops.kv_append(c, b, x, x)
        ops.kv_read(c, b, out=(x, x.clone()))
        ops.kv_attention(c, b, x.clone(), out=x)
        assert (x == 7.0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_pages_beyond_32_bits(kind):
    """Pages that lie more than 2^32 bytes apart."""
    size = {"same": 2, "e4m3": 1, "int8": 1}[kind]
    n = 5 * (1 << 30) // (2 * 16 * 64 * size)
    shape = (n, 2, 16, 64)
    held = {"same": torch.float16, "e4m3": torch.uint8, "int8": torch.int8}[kind]
    k, v = (torch.empty(shape, dtype=held, device="cuda") for _ in "kv")
    sc = [None, None] if kind == "same" else [torch.empty(shape[:3], dtype=torch.uint8 if kind == "e4m3" else torch.float32, device="cuda") for _ in "kv"]
    cache = ops.KvCache(k, v, *sc, kind=kind, dtype=torch.float16)
    g = torch.Generator().manual_seed(3)
    table = torch.tensor([[n - 1, 0, n - 2, n // 2], [n // 2 + 1, n - 3, 1, 5]], dtype=torch.int32)
    lens, news = [50, 64], [50, 64]
    i = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    b = ops.KvBatch(table.cuda(), i([0, 50, 114]), i(lens), n_tokens=114, max_new=64)
    x = [torch.randn((114, 2, 64), generator=g).half() for _ in "kvq"]
    ops.kv_append(cache, b, x[0].cuda(), x[1].cuda())
    got = [t.cpu() for t in ops.kv_read(cache, b)]
    for t, src in zip(got, x):
        want = src if kind == "same" else values(*quantise(src, kind), kind).half()
        assert torch.equal(t, want)
    st = Step([50, 64], news, 2, 64, 16, kind, "f16")     # the same sequences in a small cache
    small = st.cuda()[0]
    ops.kv_append(small, st.batch, x[0].cuda(), x[1].cuda())
    assert torch.equal(ops.kv_attention(cache, b, x[2].cuda()), ops.kv_attention(small, ops.KvBatch(st.batch.page_table, st.batch.q_start, st.batch.kv_len, n_tokens=114, max_new=64), x[2].cuda()))
    del k, v, cache
    torch.cuda.empty_cache()


def test_results_repeat_and_do_not_depend_on_the_pages():
    """The same call twice, and over another placement of the same sequences: bit for bit."""
    for news in ([1, 1, 1], [40, 1, 200]):
        st = Step([700, 33, 200], news, 2, 64, 16, "e4m3", "f16")
        st.cuda()
        q = torch.randn((st.n, 6, 64), generator=st.g).half().cuda()
        a = ops.kv_attention(st.cache, st.batch, q)
        assert torch.equal(a, ops.kv_attention(st.cache, st.batch, q))
        order = torch.randperm(st.n_pages, generator=st.g)
        back = torch.empty_like(order)
        back[order] = torch.arange(st.n_pages)
        moved = ops.KvCache(*(t[order.cuda()].contiguous() for t in (st.cache.k, st.cache.v, st.cache.k_scale, st.cache.v_scale)), kind="e4m3", dtype=torch.float16)
        table = torch.where(st.table >= 0, back[st.table.clamp(min=0).long()].int(), st.table)
        b = ops.KvBatch(table.cuda(), st.batch.q_start, st.batch.kv_len, n_tokens=st.n, max_new=max(news), min_new=min(news), max_len=700)
        assert torch.equal(a, ops.kv_attention(moved, b, q))


def test_wrong_hints_cost_time_only():
    """max_len far too small or too large, min_new at 0: results stay within the bound; a span longer than max_new is covered up to max_new."""
    st = Step([900, 130], [3, 60], 1, 64, 16, "same", "f16")
    st.cuda()
    q = torch.randn((63, 4, 64), generator=st.g).half()
    want, tol, _ = st.attend(q, 0.125, True)
    for max_len in (0, 1, 130, 1 << 29):
        for min_new in (0, 3):
            b = ops.KvBatch(st.batch.page_table, st.batch.q_start, st.batch.kv_len, n_tokens=63, max_new=60, min_new=min_new, max_len=max_len)
            got = ops.kv_attention(st.cache, b, q.cuda()).cpu().double()
            assert ((got - want).abs() <= tol).all()
    b = ops.KvBatch(st.batch.page_table, st.batch.q_start, st.batch.kv_len, n_tokens=63, max_new=60, min_new=60)      # a lie: one span has 3
    assert ((ops.kv_attention(st.cache, b, q.cuda()).cpu().double() - want).abs() <= tol).all()


def test_joining_disjoint_keys_by_lse():
    """Two calls over halves of the keys joined with their lse equal one call over all of them."""
    st = Step([96, 160], [1, 30], 2, 64, 16, "same", "f16")
    st.cuda()
    q = torch.randn((31, 4, 64), generator=st.g).half()
    want, tol, _ = st.attend(q, 0.125, False)
    parts = []
    for a, b in ((0, 3), (3, 10)):
        t = torch.full_like(st.table, -1)
        t[:, a:b] = st.table[:, a:b]
        parts.append(ops.kv_attention(st.cache, ops.KvBatch(t.cuda(), st.batch.q_start, st.batch.kv_len, n_tokens=31, max_new=30), q.cuda(), causal=False, return_lse=True))
    lse = torch.stack([p[1] for p in parts]).double()
    w = torch.softmax(lse, 0)[..., None]
    got = (w[0] * parts[0][0].double() + w[1] * parts[1][0].double()).cpu()
    assert ((got - want).abs() <= 2 * tol + 2.0 ** -11 * want.abs() + 2.0 ** -12).all()


def test_streams_and_two_calls_at_once():
    """Launched on the current stream, whatever it is; two streams at work on one cache."""
    st = Step([2000, 1500], [1, 1], 2, 64, 16, "same", "f16")
    st.cuda()
    q = torch.randn((2, 4, 64), generator=st.g).half().cuda()
    want = ops.kv_attention(st.cache, st.batch, q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.kv_attention(st.cache, st.batch, q))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for g in got for x in g)
    with torch.cuda.stream(streams[0]):                   # ordered behind what runs there
        x = torch.zeros_like(q)
        torch.cuda._sleep(1000000)
        x.copy_(q)
        y = ops.kv_attention(st.cache, st.batch, x)
    streams[0].synchronize()
    assert torch.equal(y, want)


def test_captured_steps():
    """Two graphs of append + attention on one cache, replayed in turn with eager work in between; lengths and inputs change in place."""
    st = Step([300, 310], [1, 1], 2, 64, 16, "int8", "f16", extra_pages=2, spare=8)
    st.table[0, 19], st.table[1, 20] = [p for p in range(st.n_pages) if p not in st.table.flatten().tolist()][:2]
    cache, _ = st.cuda()
    lens = torch.tensor([300, 310], dtype=torch.int32).cuda()
    starts = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    b = ops.KvBatch(st.table.cuda(), starts, lens, n_tokens=2, max_new=1, max_len=2000)
    k, v, q = (torch.zeros((2, h, 64), dtype=torch.float16, device="cuda") for h in (2, 2, 4))

    def step():
        ops.kv_append(cache, b, k, v)
        return ops.kv_attention(cache, b, q)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for i in range(6):
        lens += 1
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=st.g))
        want = step().clone()                             # eager, on the same inputs: writes the same rows
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        assert torch.equal(outs[i % 2], want), i
        torch.randn(1000, device="cuda").sum().item()


def test_the_current_device_stays():
    """Raw calls: another device than the current one is an error without a launch when it does not exist, and leaves the current device alone."""
    c = ops.KvCache.empty(4, 2, 16, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    b = ops.KvBatch(torch.zeros((1, 2), **i32), torch.zeros(2, **i32), torch.zeros(1, **i32), n_tokens=1, max_new=1)
    x = torch.zeros((1, 2, 64), dtype=torch.float16, device="cuda")
    r = ops._rows(x, "x", c, b, 2)
    L = ops._lib()
    for device in (torch.cuda.device_count(), -1, 4096):
        assert L.ss_kv_append(c._c, b._c, r, r, device, None) == -4
    assert torch.cuda.current_device() == 0
    assert L.ss_kv_append(c._c, b._c, r, r, 0, None) == 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("kind", KINDS)
def test_a_cache_of_one_page(kind):
    """The stride over a single page says nothing: a slice of a pool with any stride is taken."""
    held = {"same": torch.float16, "e4m3": torch.uint8, "int8": torch.int8}[kind]
    pool = torch.zeros(2 * 2 * 16 * 64, dtype=held, device="cuda")
    k, v = (torch.as_strided(pool, (1, 2, 16, 64), (stride, 1024, 64, 1), at) for stride, at in ((7, 0), (1 << 33, 2048)))
    scales = [] if kind == "same" else [torch.as_strided(torch.zeros(32, dtype=torch.uint8 if kind == "e4m3" else torch.float32, device="cuda"), (1, 2, 16), (s, 16, 1)) for s in (3, 5)]
    c = ops.KvCache(k, v, *scales, kind=kind, dtype=torch.float16)
    t32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    b = ops.KvBatch(t32(0)[None], t32(0, 5), t32(5), n_tokens=5, max_new=5)
    x = torch.ones((5, 2, 64), dtype=torch.float16, device="cuda")
    ops.kv_append(c, b, x, 2 * x)
    rk, rv = ops.kv_read(c, b)
    tol = 0 if kind != "int8" else 2.0 ** -11                            # 127 * (1 / 127 in float32) rounded to f16
    assert float((rk - x).abs().max()) <= tol and float((rv - 2 * x).abs().max()) <= 2 * tol
    assert float((ops.kv_attention(c, b, x) - 2.0).abs().max()) <= 2 * 2.0 ** -9
