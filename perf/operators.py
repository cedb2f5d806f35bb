"""Cases of the decoder operators on paged caches and of the sampler: append, read, attention, sampling.

`own` false: the operators' plain forms in elementary torch operations.  `own` true: the calls a program makes of speaksense_amd.ops."""
import math

import torch

own = False

F16, BF16 = torch.float16, torch.bfloat16
TYPES = {"f16": F16, "bf16": BF16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of eight streams of the 20-head decoder into an e4m3 cache: a call that is all latency
        dict(name="append step e4m3", op="append", dtype="f16", kind="e4m3", seqs=8, new_lo=1, new_hi=1, len_lo=4, len_hi=448, heads=20, dim=64, page=16),
        # the prompts (up to half of the 448-position context) of 96 windows in flight, into an int8 cache
        dict(name="append prompts int8", op="append", dtype="bf16", kind="int8", seqs=96, new_lo=3, new_hi=224, len_lo=224, len_hi=448, heads=20, dim=64, page=32),
        # one short context of the 8-head decoder read back dense
        dict(name="read one context int8", op="read", dtype="bf16", kind="int8", seqs=1, new_lo=99, new_hi=99, len_lo=99, len_hi=99, heads=8, dim=64, page=16),
        # 32 encoder windows of 1500 keys read back from the cross cache's 8-bit form
        dict(name="read windows e4m3", op="read", dtype="f16", kind="e4m3", seqs=32, new_lo=1500, new_hi=1500, len_lo=1500, len_hi=1500, heads=20, dim=64, page=64),
        # a decoding step of eight streams of the 8-head decoder: the smallest attention
        dict(name="attend step f16", op="attend", dtype="f16", kind="same", seqs=8, new_lo=1, new_hi=1, len_lo=4, len_hi=448, heads=8, groups=1, dim=64, page=16, causal=True),
        # cross-attention of 96 decoders over 1500 encoder positions each, 8-bit cache: the decoder's largest stream
        dict(name="attend windows e4m3", op="attend", dtype="f16", kind="e4m3", seqs=96, new_lo=1, new_hi=1, len_lo=1500, len_hi=1500, heads=20, groups=1, dim=64, page=64, causal=False),
        # a few long contexts with grouped heads: little parallelism but along the keys
        dict(name="attend long bf16", op="attend", dtype="bf16", kind="same", seqs=4, new_lo=1, new_hi=1, len_lo=30001, len_hi=65536, heads=8, groups=4, dim=128, page=64, causal=True),
        # the prompt pass of 32 windows
        dict(name="attend prompts f16", op="attend", dtype="f16", kind="same", seqs=32, new_lo=3, new_hi=224, len_lo=224, len_hi=448, heads=20, groups=1, dim=64, page=16, causal=True),
        # chunks of a long prompt over what is cached of it, 8-bit cache, grouped heads: all arithmetic
        dict(name="attend chunk int8", op="attend", dtype="bf16", kind="int8", seqs=2, new_lo=2000, new_hi=2048, len_lo=15000, len_hi=16384, heads=8, groups=4, dim=128, page=64, causal=True),
        # the fallback's sampled step of eight windows: temperature alone over the whole vocabulary
        dict(name="sample step", op="sample", dtype="f32", rows=8, vocab=51866, filters="none"),
        # 32 windows of five sampled decoders each, with filters
        dict(name="sample decoders", op="sample", dtype="f32", rows=160, vocab=51866, filters="mixed"),
        # many rows of a larger vocabulary in 16 bits
        dict(name="sample wide", op="sample", dtype="bf16", rows=512, vocab=128000, filters="mixed"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "attend", "sample"])
    if op == "sample":
        rows, vocab = _log(rng, 1, 512), _log(rng, 999, 128000)
        return dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), rows=rows, vocab=vocab, filters=rng.choice(["none", "mixed", "mixed"]))
    dtype, kind = rng.choice(["f16", "bf16"]), rng.choice(["same", "e4m3", "int8"])
    dim, page = rng.choice([64, 64, 128]), rng.choice([16, 32, 64, 128])
    if op in ("append", "read"):
        seqs, heads = _log(rng, 1, 96), rng.choice([1, 4, 6, 8, 12, 16, 20])
        hi = _log(rng, 1, max(1, min(4000, 30000 // seqs)))
        lo = rng.choice([hi, (hi + 1) // 2, 1])
        return dict(op=op, dtype=dtype, kind=kind, seqs=seqs, new_lo=lo, new_hi=hi, len_lo=hi, len_hi=hi + _log(rng, 1, 500), heads=heads, dim=dim, page=page)
    heads, groups = rng.choice([1, 2, 4, 6, 8, 12, 20]), rng.choice([1, 1, 2, 4, 5, 8])
    causal = rng.random() < 0.7
    if rng.random() < 0.5:      # one token each, or a few
        seqs, hi = _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 5])
        most = 60000000 // (seqs * heads * dim)
        top = _log(rng, 16, max(16, min(65536, most)))
    else:                       # a chunk
        seqs = _log(rng, 1, 16)
        most = 2e11 / (seqs * heads * groups * dim * 4)         # new tokens x keys
        hi = _log(rng, 6, min(2048, int(most ** 0.5)))
        top = _log(rng, hi, max(hi, min(16384, int(most / hi))))
    lo = rng.choice([hi, (hi + 1) // 2, 1])
    return dict(op=op, dtype=dtype, kind=kind, seqs=seqs, new_lo=lo, new_hi=hi, len_lo=max(hi, top // rng.choice([1, 2, 8])), len_hi=top, heads=heads, groups=groups, dim=dim,
                page=page, causal=causal)


# ---------------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------------
def _between(gen, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=gen)


def _sizes(case):
    """New tokens and lengths of each sequence: host numbers, as a scheduler has them.  They belong to the case: its outputs have one shape."""
    gen = torch.Generator().manual_seed(case["seqs"] * 7919 + case["new_hi"] * 31 + case["len_hi"])
    new = _between(gen, case["new_lo"], case["new_hi"], case["seqs"])
    return new, torch.maximum(_between(gen, case["len_lo"], case["len_hi"], case["seqs"]), new)


def _rows(gen, shape, dtype):
    """Key / value rows: normal, each head at a size of its own, one large channel."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    x *= torch.exp(torch.randn(shape[-3:-2] + (1, 1) if len(shape) == 4 else (shape[1], 1), generator=gen, device="cuda") * 0.5)
    x[..., 5] *= 4.0
    return x.to(dtype)


def _exponent(amax):
    """The E8M0 byte of a row whose largest magnitude is amax: amax / 2^(byte - 127) <= 448."""
    bits = amax.contiguous().view(torch.int32)
    return (((bits >> 23) & 255) - 8 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32)).clamp(1, 253)


def _pow2(e):
    return ((e.to(torch.int32)) << 23).view(torch.float32)          # 2^(e - 127), 1 <= e <= 254


def _quantise(x, kind):
    """Codes and scales of 16-bit rows [..., D]."""
    x = x.float()
    amax = x.abs().amax(-1)
    if kind == "e4m3":
        e = _exponent(amax)
        return (x * _pow2(254 - e)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), e.to(torch.uint8)
    s = amax / 127.0
    q = torch.round(x / torch.where(s > 0, s, torch.ones_like(s))[..., None]).clamp(-127, 127)
    return q.to(torch.int8), s


def _values(codes, scale, kind, wide=torch.float32):
    if kind == "same":
        return codes.to(wide)
    if kind == "e4m3":
        return codes.view(torch.float8_e4m3fn).float().to(wide) * _pow2(scale).to(wide)[..., None]
    return codes.to(wide) * scale.to(wide)[..., None]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]
    s = dict(case=case, dt=dt)
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        x = torch.randn((n, v), generator=gen, device="cuda") * 2.5
        # a handful of likely ids, and ids that rules have masked
        at = torch.randint(0, v, (n, 12), generator=gen, device="cuda")
        x.scatter_add_(1, at, torch.rand((n, 12), generator=gen, device="cuda") * 14)
        x.masked_fill_(torch.rand((1, v), generator=gen, device="cuda") < 0.02, float("-inf"))
        s["logits"] = x.to(dt)
        s["u"] = torch.rand((n,), generator=gen, device="cuda", dtype=torch.float64)
        pick = torch.rand((4, n), generator=gen, device="cuda")
        s["temperature"] = (torch.floor(torch.rand((n,), generator=gen, device="cuda") * 5) + 1) * 0.2
        if case["filters"] == "mixed":      # requests of their own settings share a step
            s["temperature"] = torch.where(pick[0] < 0.1, torch.zeros_like(s["temperature"]), s["temperature"])
            k = torch.tensor([1, 5, 40, 50, 200, 1000], device="cuda")[torch.randint(0, 6, (n,), generator=gen, device="cuda")]
            s["top_k"] = torch.where(pick[1] < 0.5, k, torch.zeros_like(k)).to(torch.int32)
            s["top_p"] = torch.where(pick[2] < 0.6, 0.5 + 0.49 * torch.rand((n,), generator=gen, device="cuda"), torch.ones(n, device="cuda"))
            s["min_p"] = torch.where(pick[3] < 0.3, 0.1 * torch.rand((n,), generator=gen, device="cuda"), torch.zeros(n, device="cuda"))
        else:
            s["top_k"] = s["top_p"] = s["min_p"] = None
        return s

    new, length = _sizes(case)
    host = torch.Generator().manual_seed(seed)
    b, page, heads, dim = case["seqs"], case["page"], case["heads"], case["dim"]
    need = (length + page - 1) // page
    most, total = int(need.max()), int(need.sum())
    n_pages = total + 3
    order = torch.randperm(n_pages, generator=host)
    table = torch.full((b, most), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need.tolist()):
        table[i, :n] = order[at:at + n]
        at += n
    s["table"], s["kv_len"] = table.cuda(), length.to(torch.int32).cuda()
    s["q_start"] = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).to(torch.int32).cuda()
    s["n"], s["max_new"], s["min_new"], s["max_len"] = int(new.sum()), int(new.max()), int(new.min()), int(length.max())
    kind = case["kind"]
    shape = (n_pages, heads, page, dim)
    for name in ("k", "v"):
        x = _rows(gen, shape, dt)
        if kind == "same":
            s[name], s[name + "_scale"] = x, None
        else:
            s[name], s[name + "_scale"] = _quantise(x, kind)
    if case["op"] == "append":
        s["k_new"], s["v_new"] = (_rows(gen, (s["n"], heads, dim), dt) for _ in "kv")
    if case["op"] == "attend":
        q = torch.randn((s["n"], heads * case["groups"], dim), generator=gen, device="cuda")
        s["q"], s["scale"] = (q * 1.5).to(dt), dim ** -0.5
    if own:
        from speaksense_amd import ops
        s["cache"] = ops.KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"], kind=kind, dtype=dt)
        s["batch"] = ops.KvBatch(s["table"], s["q_start"], s["kv_len"], n_tokens=s["n"], max_new=s["max_new"], min_new=s["min_new"], max_len=s["max_len"])
    return s


# ---------------------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------------------
def _places(s):
    """Page and row of every new token."""
    start, length, page = s["q_start"].long(), s["kv_len"].long(), s["case"]["page"]
    t = torch.arange(s["n"], device="cuda")
    seq = torch.searchsorted(start, t, right=True) - 1
    pos = length[seq] - start[seq + 1] + t
    return seq, pos, s["table"].long()[seq, pos // page], pos % page


def _append(s):
    _, _, page, row = _places(s)
    kind = s["case"]["kind"]
    for name in ("k", "v"):
        if kind == "same":
            s[name][page, :, row] = s[name + "_new"]
        else:
            codes, scale = _quantise(s[name + "_new"], kind)
            s[name][page, :, row] = codes
            s[name + "_scale"][page, :, row] = scale


def _read(s):
    _, _, page, row = _places(s)
    kind = s["case"]["kind"]
    return [_values(s[n][page, :, row], None if kind == "same" else s[n + "_scale"][page, :, row], kind).to(s["dt"]) for n in ("k", "v")]


def _attend(s):
    c = s["case"]
    b, heads, g, dim, page = c["seqs"], c["heads"], c["groups"], c["dim"], c["page"]
    table, length = s["table"].long().clamp(min=0), s["kv_len"].long()
    keys = table.shape[1] * page

    def dense(name):        # [b, heads, keys, dim]
        scale = None if c["kind"] == "same" else s[name + "_scale"][table]
        return _values(s[name][table], scale, c["kind"]).permute(0, 2, 1, 3, 4).reshape(b, heads, keys, dim)

    seq, pos, _, _ = _places(s)
    at = torch.arange(s["n"], device="cuda") - s["q_start"].long()[seq]
    q = torch.zeros((b, s["max_new"], heads, g, dim), device="cuda")
    q[seq, at] = s["q"].float().view(s["n"], heads, g, dim)
    last = torch.full((b, s["max_new"]), -1, device="cuda")
    last[seq, at] = pos if c["causal"] else length[seq] - 1
    q = q.permute(0, 2, 3, 1, 4).reshape(b, heads, g * s["max_new"], dim)
    x = torch.matmul(q, dense("k").transpose(-1, -2)).view(b, heads, g, s["max_new"], keys)
    x *= s["scale"]
    x.masked_fill_((torch.arange(keys, device="cuda") > last[..., None])[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top > float("-inf"), top, torch.zeros_like(top))).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, heads, g * s["max_new"], keys), dense("v")).view(b, heads, g, s["max_new"], dim)
    o /= torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 3, 1, 2, 4)[seq, at].reshape(s["n"], heads * g, dim).to(s["dt"])


def _sample(s):
    """In 64 bits: a draw is a comparison with a running sum."""
    x = s["logits"].double()
    n, v = x.shape
    x = torch.where(torch.isnan(x), float("-inf"), x)
    top, best = x.max(-1, keepdim=True)
    best = torch.where(x == top, torch.arange(v, device="cuda"), v).amin(-1, keepdim=True)
    t = s["temperature"].double()[:, None]
    greedy = ~(t > 0)
    w = torch.where(x == top, 1.0, torch.exp((x - top) / torch.where(greedy, torch.ones_like(t), t)))
    whole = w.sum(-1, keepdim=True)
    keep = x > float("-inf")
    if s["top_k"] is not None:
        _, order = torch.sort(x, dim=-1, descending=True, stable=True)      # ties stay in order of their ids
        k = s["top_k"].long()[:, None]
        in_k = torch.arange(v, device="cuda") < torch.where((k > 0) & (k < v), k, torch.full_like(k, v))
        y = torch.where(in_k, w.gather(1, order), 0.0)
        p = s["top_p"].double()[:, None]
        cut = ((y.cumsum(-1) - y >= p * y.sum(-1, keepdim=True)) & (p < 1)) | (y < s["min_p"].double()[:, None]) | ~in_k
        cut[:, 0] = False
        keep &= torch.zeros_like(keep).scatter_(1, order, ~cut)
    kept = torch.where(keep, w, 0.0)
    run = kept.cumsum(-1)
    total = run[:, -1:]
    target = s["u"][:, None] * total
    first = torch.where((run > target) & (kept > 0), torch.arange(v, device="cuda"), v).amin(-1, keepdim=True)
    ids = torch.where(greedy, best, first)
    p = torch.where(greedy, 1.0, kept.gather(1, ids) / total)
    n_kept = torch.where(greedy, 1, keep.sum(-1, keepdim=True))
    return dict(id=ids[:, 0].int(), p=p[:, 0].float(), logprob=torch.log(w.gather(1, ids) / whole)[:, 0].float(), n_kept=n_kept[:, 0].int())


def run(s):
    op = s["case"]["op"]
    if own:
        from speaksense_amd import ops
        if op == "append":
            ops.kv_append(s["cache"], s["batch"], s["k_new"], s["v_new"])
            return (s["k"], s["v"]) if s["case"]["kind"] == "same" else ops.kv_read(s["cache"], s["batch"])
        if op == "read":
            return ops.kv_read(s["cache"], s["batch"])
        if op == "attend":
            return ops.kv_attention(s["cache"], s["batch"], s["q"], scale=s["scale"], causal=s["case"]["causal"])
        r = ops.sample_rows(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return dict(id=r.id, p=r.p, logprob=r.logprob, n_kept=r.n_kept)
    if op == "append":      # rows of 8 bits come back as the values that the cache holds of them
        _append(s)
        return (s["k"], s["v"]) if s["case"]["kind"] == "same" else _read(s)
    return {"read": _read, "attend": _attend, "sample": _sample}[op](s)


# ---------------------------------------------------------------------------------------------------------------------------------
# work, and the operators from their definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "sample":
        size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
        return dict(bytes=case["rows"] * (case["vocab"] * size + 40), flops=4 * case["rows"] * case["vocab"])
    new, length = (case["new_lo"] + case["new_hi"]) / 2, (case["len_lo"] + case["len_hi"]) / 2
    held = case["dim"] * (2 if case["kind"] == "same" else 1) + {"same": 0, "e4m3": 1, "int8": 4}[case["kind"]]
    rows = case["seqs"] * new * case["heads"]
    if case["op"] == "append":
        back = 0 if case["kind"] == "same" else held + case["dim"] * 2
        return dict(bytes=2 * rows * (case["dim"] * 2 + held + back), flops=4 * rows * case["dim"])
    if case["op"] == "read":
        return dict(bytes=2 * rows * (case["dim"] * 2 + held), flops=2 * rows * case["dim"])
    seen = length - (new - 1) / 2 if case["causal"] else length
    return dict(bytes=case["seqs"] * (2 * length * case["heads"] * held + 4 * new * case["heads"] * case["groups"] * case["dim"]),
                flops=4 * rows * case["groups"] * seen * case["dim"])


def _exact_rows(s, name, i):
    """Sequence i's rows [len, heads, dim] in 64 bits, gathered page by page."""
    n, kind = int(s["kv_len"][i]), s["case"]["kind"]
    pages = s["table"][i, : (n + s["case"]["page"] - 1) // s["case"]["page"]].long()
    x = s[name][pages]
    x = x.view(torch.float8_e4m3fn).double() if kind == "e4m3" else x.double()
    if kind != "same":
        f = s[name + "_scale"][pages].double()
        x = x * (_exact_pow2(f - 127) if kind == "e4m3" else f)[..., None]
    return x.transpose(1, 2).flatten(0, 1)[:n]


def _exact_pow2(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_held(x, kind):
    """What an 8-bit cache holds of rows [n, heads, dim]."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    if kind == "int8":
        f = torch.where(top > 0, top / 127, torch.ones_like(top))
        return torch.round(x / f) * f
    m, e = torch.frexp(torch.where(top > 0, top, torch.ones_like(top)) / 448)       # m in [1/2, 1): 2^(e - 1) only where m is 1/2
    f = _exact_pow2(e - (m == 0.5).to(e.dtype))
    y = x / f
    _, e = torch.frexp(y.abs().clamp(min=2.0 ** -6))
    step = _exact_pow2(e - 4)
    return torch.round(y / step) * step * f


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "sample":
        return _exact_sample(s)
    kind, starts, lens = case["kind"], s["q_start"].tolist(), s["kv_len"].tolist()
    if case["op"] == "append":
        if kind != "same":
            return [_exact_held(s[n + "_new"], kind) for n in ("k", "v")]
        out = [s["k"].double(), s["v"].double()]
        for x, new in zip(out, (s["k_new"], s["v_new"])):
            for i in range(case["seqs"]):
                p = torch.arange(lens[i] - (starts[i + 1] - starts[i]), lens[i], device="cuda")
                x[s["table"][i].long()[p // case["page"]], :, p % case["page"]] = new[starts[i]:starts[i + 1]].double()
        return out
    if case["op"] == "read":
        return [torch.cat([_exact_rows(s, n, i)[lens[i] - (starts[i + 1] - starts[i]):] for i in range(case["seqs"])]) for n in ("k", "v")]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i in range(case["seqs"]):
        a, b = starts[i], starts[i + 1]
        k, v = _exact_rows(s, "k", i), _exact_rows(s, "v", i)
        behind = torch.arange(lens[i], device="cuda") > torch.arange(lens[i] - (b - a), lens[i], device="cuda")[:, None]
        for h in range(case["heads"]):
            for j in range(h * case["groups"], (h + 1) * case["groups"]):
                x = s["q"][a:b, j].double() @ k[:, h].t().contiguous() * s["scale"]
                if case["causal"]:
                    x.masked_fill_(behind, float("-inf"))
                out[a:b, j] = torch.softmax(x, -1) @ v[:, h].contiguous()
    return out


def _exact_sample(s):
    """Row by row."""
    n, v = s["logits"].shape
    ids, p, logprob, kept_n = [], [], [], []
    temperature = s["temperature"].tolist()
    for i in range(n):
        x = s["logits"][i].double()
        t = temperature[i]
        if not t > 0:
            at = int((x == x.max()).nonzero()[0])
            ids.append(at), p.append(1.0), kept_n.append(1)
            logprob.append(torch.log_softmax(x, -1)[at].item())
            continue
        prob = torch.softmax(x / t, -1)
        keep = x > float("-inf")
        if s["top_k"] is not None:
            k, top_p, min_p = int(s["top_k"][i]), float(s["top_p"][i]), float(s["min_p"][i])
            order = torch.argsort(x, descending=True, stable=True)[: k if 0 < k < v else v]
            q = prob[order] / prob[order].sum()
            if top_p < 1:
                q = q[: 1 + int((q.cumsum(0) < top_p).sum())]
            q = q[q >= q[0] * min_p]
            keep = torch.zeros(v, dtype=torch.bool, device="cuda")
            keep[order[: len(q)]] = True
        held = torch.where(keep, prob, 0.0)
        held = held / held.sum()
        at = min(int((held.cumsum(0) <= s["u"][i]).sum()), int(keep.nonzero()[-1]))
        ids.append(at), p.append(held[at].item()), logprob.append(math.log(prob[at].item())), kept_n.append(int(keep.sum()))
    return dict(id=torch.tensor(ids, dtype=torch.int32), p=torch.tensor(p, dtype=torch.float64), logprob=torch.tensor(logprob, dtype=torch.float64), n_kept=torch.tensor(kept_n, dtype=torch.int32))
