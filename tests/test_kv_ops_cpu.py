"""Decoder operators without a GPU: every refusal of the C entry points happens before the device is touched, the workspace query is host arithmetic,
and the Python layer refuses what it is not given in device memory."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
from speaksense_amd import binding, ops  # noqa: E402

P = 1 << 20      # an aligned address that nothing dereferences: refusals come first


def _cache(**kw):
    d = dict(k=P, v=P, k_scale=None, v_scale=None, page_stride=8 * 16 * 64, scale_stride=0, n_pages=4, page_size=16, n_kv_heads=8, head_dim=64, dtype=binding.DTYPE_F16,
             kind=ops.KV_SAME)
    d.update(kw)
    return ops._Cache(**d)


def _cache8(**kw):
    return _cache(**dict(dict(k_scale=P, v_scale=P, scale_stride=8 * 16, kind=ops.KV_E4M3), **kw))


def _batch(**kw):
    d = dict(page_table=P, q_start=P, kv_len=P, table_stride=4, n_seqs=2, max_pages=4, n_tokens=3, max_new=2, min_new=1, max_len=64)
    d.update(kw)
    return ops._Batch(**d)


def _rows(**kw):
    d = dict(p=P, row_stride=8 * 64, head_stride=64)
    d.update(kw)
    return ops._Rows(**d)


BAD_CACHES = [dict(kind=3), dict(kind=-1), dict(dtype=2), dict(dtype=3), dict(head_dim=32), dict(head_dim=96), dict(head_dim=256), dict(page_size=8), dict(page_size=48),
              dict(page_size=512), dict(page_size=0), dict(n_pages=0), dict(n_pages=-1), dict(n_kv_heads=0), dict(page_stride=8 * 16 * 64 - 16), dict(page_stride=8 * 16 * 64 + 8),
              dict(k=None), dict(v=None), dict(k=P + 8), dict(v=P + 2)]
BAD_CACHES8 = [dict(k_scale=None), dict(v_scale=None), dict(k_scale=P + 4), dict(scale_stride=8 * 16 - 1), dict(scale_stride=8 * 16 + 4)]
BAD_BATCHES = [dict(n_seqs=-1), dict(n_tokens=-1), dict(max_new=-1), dict(min_new=-1), dict(max_len=-1), dict(max_pages=0), dict(max_pages=1 << 26), dict(table_stride=3),
               dict(page_table=None), dict(q_start=None), dict(kv_len=None), dict(q_start=P + 2), dict(min_new=3), dict(n_seqs=1 << 21), dict(n_tokens=(1 << 28) + 1)]
BAD_ROWS = [dict(p=None), dict(p=P + 8), dict(row_stride=8 * 64 + 4), dict(head_stride=68), dict(row_stride=-512), dict(head_stride=-64)]


def _refused(rc, part=""):
    assert rc == -1, rc
    msg = ops._lib().ss_last_error().decode()
    assert msg.startswith("ss_") and part in msg, msg


def _calls(c, b, r=None):
    L = ops._lib()
    r = r or _rows()
    yield L.ss_kv_append(c, b, r, r, 0, None)
    yield L.ss_kv_read(c, b, r, r, 0, None)
    yield L.ss_kv_attention(c, b, r, 8, 1.0, 1, r, None, None, 0, 0, None)


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_bad_caches_are_refused(kw):
    for rc in _calls(_cache(**kw), _batch()):
        _refused(rc)
    assert ops._lib().ss_kv_attention_workspace(_cache(**kw), _batch(), 8) == -1


@pytest.mark.parametrize("kw", BAD_CACHES8)
@pytest.mark.parametrize("kind", [ops.KV_E4M3, ops.KV_INT8])
def test_bad_scales_are_refused(kw, kind):
    for rc in _calls(_cache8(kind=kind, **kw), _batch()):
        _refused(rc)


@pytest.mark.parametrize("kw", BAD_BATCHES)
def test_bad_batches_are_refused(kw):
    for rc in _calls(_cache(), _batch(**kw)):
        _refused(rc)


@pytest.mark.parametrize("kw", BAD_ROWS)
def test_bad_rows_are_refused(kw):
    for rc in _calls(_cache(), _batch(), _rows(**kw)):
        _refused(rc)


@pytest.mark.parametrize("kw", [dict(row_stride=0), dict(head_stride=0), dict(row_stride=64, head_stride=64), dict(row_stride=8 * 64 - 8), dict(head_stride=56)])
def test_overlapping_results_are_refused(kw):
    L, c, b, r, bad = ops._lib(), _cache(), _batch(), _rows(), _rows(**kw)
    _refused(L.ss_kv_read(c, b, r, bad, 0, None), "overlap")
    _refused(L.ss_kv_read(c, b, bad, r, 0, None), "overlap")
    _refused(L.ss_kv_attention(c, b, r, 8, 1.0, 1, bad, None, None, 0, 0, None), "overlap")


def test_null_arguments_are_refused():
    L, c, b, r = ops._lib(), _cache(), _batch(), _rows()
    for rc in (L.ss_kv_append(None, b, r, r, 0, None), L.ss_kv_append(c, None, r, r, 0, None), L.ss_kv_append(c, b, None, r, 0, None), L.ss_kv_append(c, b, r, None, 0, None),
               L.ss_kv_read(None, b, r, r, 0, None), L.ss_kv_read(c, b, r, None, 0, None), L.ss_kv_attention(c, b, None, 8, 1.0, 1, r, None, None, 0, 0, None),
               L.ss_kv_attention(c, b, r, 8, 1.0, 1, None, None, None, 0, 0, None), L.ss_kv_attention_workspace(None, b, 8), L.ss_kv_attention_workspace(c, None, 8),
               L.ss_sample_rows(None, 0, None)):
        _refused(rc, "null")


@pytest.mark.parametrize("heads", [0, -8, 4, 12, 1 << 17])
def test_bad_heads_are_refused(heads):
    _refused(ops._lib().ss_kv_attention(_cache(), _batch(), _rows(), heads, 1.0, 1, _rows(), None, None, 0, 0, None), "n_heads")


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_bad_scale_is_refused(scale):
    _refused(ops._lib().ss_kv_attention(_cache(), _batch(), _rows(), 8, scale, 1, _rows(), None, None, 0, 0, None), "scale")


def test_workspace_is_host_arithmetic_and_enforced():
    L = ops._lib()
    c, r = _cache(n_pages=4096), _rows()
    short, long = _batch(max_len=40), _batch(max_pages=4096, table_stride=4096, max_len=60000)
    assert L.ss_kv_attention_workspace(c, short, 8) == 0
    need = L.ss_kv_attention_workspace(c, long, 8)
    assert need > 0 and need % 8 == 0 and need <= 3 * 8 * 64 * 66 * 4
    for empty in (dict(n_seqs=0), dict(n_tokens=0), dict(max_new=0, min_new=0)):
        assert L.ss_kv_attention_workspace(c, _batch(**empty), 8) == 0
    assert L.ss_kv_attention(c, long, r, 8, 1.0, 1, r, None, None, 0, 0, None) == -1                  # none
    assert L.ss_kv_attention(c, long, r, 8, 1.0, 1, r, None, P + 4, need, 0, None) == -1              # misaligned
    assert L.ss_kv_attention(c, long, r, 8, 1.0, 1, r, None, P, need - 1, 0, None) == -6              # too small: SS_ERR_BUFFER
    assert str(need) in L.ss_last_error().decode()


BAD_SAMPLES = [dict(dtype=2), dict(dtype=4), dict(n_rows=-1), dict(n_vocab=0), dict(n_vocab=(1 << 20) + 1, row_stride=1 << 21), dict(row_stride=99), dict(logits=None), dict(u=None),
               dict(id=None), dict(logits=P + 2), dict(u=P + 4), dict(temperature=P + 1), dict(top_k=P + 2), dict(top_p=P + 3), dict(min_p=P + 2), dict(id=P + 1), dict(p=P + 2),
               dict(logprob=P + 2), dict(n_kept=P + 2)]


@pytest.mark.parametrize("kw", BAD_SAMPLES)
def test_bad_sampling_arguments_are_refused(kw):
    d = dict(logits=P, u=P, temperature=None, top_k=None, top_p=None, min_p=None, id=P, p=None, logprob=None, n_kept=None, row_stride=100, n_rows=2, n_vocab=100, dtype=3, reserved=0)
    d.update(kw)
    _refused(ops._lib().ss_sample_rows(ops._Sample(**d), 0, None))


def test_structs_have_the_header_s_sizes():
    L = ops._lib()
    assert (L.ss_sizeof_kv_cache(), L.ss_sizeof_kv_batch(), L.ss_sizeof_kv_rows(), L.ss_sizeof_sample_rows_args()) == tuple(C.sizeof(s) for s in (ops._Cache, ops._Batch, ops._Rows, ops._Sample))


def test_host_tensors_are_refused():
    k = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="device memory"):
        ops.KvCache(k, k)
    with pytest.raises(ValueError, match="kind"):
        ops.KvCache(k, k, kind="int4")
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device memory"):
        ops.KvBatch(torch.zeros(1, 2, dtype=torch.int32), i, i[:1], n_tokens=1, max_new=1)
    with pytest.raises(ValueError, match="device memory"):
        ops.sample_rows(torch.zeros(2, 10), torch.zeros(2, dtype=torch.float64))


def test_sizes_that_are_no_grid_are_refused():
    """A launch holds less than 2^32 threads: one workgroup of 256 per token row at most, one of 1024 per row of logits."""
    for rc in _calls(_cache(), _batch(n_tokens=(1 << 24) + 1)):
        _refused(rc, "too many")
    d = dict(logits=P, u=P, temperature=None, top_k=None, top_p=None, min_p=None, id=P, p=None, logprob=None, n_kept=None, row_stride=100, n_rows=(1 << 21) + 1, n_vocab=100, dtype=3, reserved=0)
    _refused(ops._lib().ss_sample_rows(ops._Sample(**d), 0, None), "n_rows")
    # keys are cut only where a workgroup per query row is a grid
    b = _batch(n_tokens=1 << 20, max_new=1, n_seqs=1)
    need = lambda heads: ops._lib().ss_kv_attention_workspace(_cache(n_kv_heads=1, page_stride=256 * 64, page_size=256), b, heads)  # noqa: E731
    b.max_pages, b.table_stride, b.max_len = 64, 64, 0
    assert need(8) > 0 and need(16) == 0
