"""The 8-bit cache and the page operations refuse what their kernels do not take, before anything is launched."""
import ctypes as C

import pytest
import torch

from omnikv_amd import _lib, ops

PTR = 1 << 20  # an aligned address that nothing dereferences: every call here is refused on the host


def cache(**kw):
    c = _lib.KV8Cache(PTR, PTR, PTR, PTR, _lib.OKV_E4M3, _lib.OKV_BF16, 8, 128, 64, 1024)
    c.token_stride, c.head_stride, c.batch_stride = 128, 128 * 1024, 8 * 128 * 1024
    c.scale_block_stride, c.scale_head_stride, c.scale_batch_stride = 1, 16, 128
    c.open_k = c.open_v = PTR
    c.open_token_stride, c.open_head_stride, c.open_batch_stride = 128, 64 * 128, 8 * 64 * 128
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def append(c, starts=None, start=0, new_lens=None, n=4, close=0, batch=1, row=1024, k=PTR):
    return _lib.lib().okv_kv8_append(C.byref(c), k, row, 128, 0, PTR, 1024, 128, 0, starts, start, new_lens, n, close, batch, None)


def dense(c, hq=32, n=100, batch=1, ws=PTR, nbytes=1 << 40, scores=None, score_len=0, red=0, norm=0, q=PTR):
    return _lib.lib().okv_kv8_dense_attn(q, hq, C.byref(c), None, n, batch, 1.0, PTR, None, score_len, red, norm, scores,
                                         score_len, ws, nbytes, None)


def sparse(c, idx=PTR, stride=50, slots=0, n=50, tail=None, tail_len=0, hq=32, nbytes=1 << 40, tts=1024):
    return _lib.lib().okv_kv8_sparse_attn(PTR, hq, C.byref(c), idx, stride, slots, None, n, tail, tail, tts, 128, 0, None,
                                          tail_len, 1, 1.0, PTR, PTR, nbytes, None)


INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3


@pytest.mark.parametrize("field, value, code", [
    ("k_codes", None, INVALID), ("v_scale", None, INVALID), ("k_codes", PTR + 8, INVALID), ("k_scale", PTR + 2, INVALID),
    ("format", _lib.OKV_BF16, UNSUPPORTED), ("format", 7, UNSUPPORTED), ("dtype", _lib.OKV_F32, UNSUPPORTED),
    ("head_dim", 64, UNSUPPORTED), ("num_kv_heads", 0, INVALID), ("block_tokens", 8, UNSUPPORTED),
    ("block_tokens", 48, UNSUPPORTED), ("block_tokens", 256, UNSUPPORTED), ("capacity", 1000, INVALID), ("capacity", 0, INVALID),
    ("token_stride", 136, INVALID), ("token_stride", -128, UNSUPPORTED), ("head_stride", 8, INVALID), ("open_k", None, INVALID),
    ("open_v", PTR + 4, INVALID), ("open_token_stride", 4, INVALID)])
def test_every_call_checks_the_cache(field, value, code):
    c = cache(**{field: value})
    for rc in (append(c), dense(c), sparse(c),
               _lib.lib().okv_kv8_read(C.byref(c), None, 0, 10, None, 10, 1, PTR, PTR, 128, 1280, 0, None)):
        assert rc == code, _lib.lib().okv_last_error()


@pytest.mark.parametrize("kw, code", [
    ({"page_size": 72}, INVALID), ({"page_size": 32}, INVALID), ({"page_table_stride": 0}, INVALID), ({"num_pages": 0}, INVALID)])
def test_pages_hold_whole_blocks(kw, code):
    base = dict(page_table=PTR, page_size=64, page_table_stride=4, num_pages=9, page_stride=64 * 1024, scale_page_stride=8)
    assert dense(cache(**{**base, **kw})) == code


def test_append_refusals():
    assert append(cache(), n=-1) == INVALID
    assert append(cache(), batch=0) == INVALID
    assert append(cache(), start=-1) == INVALID
    assert append(cache(), start=1000, n=25) == INVALID  # 1024 tokens
    assert append(cache(), row=1028) == INVALID
    assert append(cache(), k=PTR + 8) == INVALID
    assert append(cache(), start=3, close=1) == INVALID
    assert append(cache(), starts=PTR, close=1) == INVALID
    closed = cache(open_k=None, open_v=None)
    assert append(closed, n=63) == INVALID
    assert append(closed, n=64, new_lens=PTR) == INVALID
    assert append(closed, n=64, starts=PTR) == INVALID
    assert append(cache(), n=0) == 0


def test_attention_refusals():
    assert dense(cache(), hq=31) == INVALID
    assert dense(cache(), hq=72) == UNSUPPORTED  # nine q heads per kv head
    assert dense(cache(num_kv_heads=64), hq=512) == UNSUPPORTED
    assert dense(cache(), n=0) == INVALID
    assert dense(cache(), n=1025) == INVALID
    assert dense(cache(), batch=0) == INVALID
    assert dense(cache(), q=PTR + 8) == INVALID
    assert dense(cache(), n=1000, ws=None) == INVALID
    assert dense(cache(), n=1000, nbytes=256) == WORKSPACE
    assert dense(cache(), scores=PTR, score_len=101) == INVALID
    assert dense(cache(), scores=PTR, score_len=50, red=2) == INVALID
    assert dense(cache(), scores=PTR, score_len=50, norm=2) == INVALID
    assert sparse(cache(), stride=49) == INVALID
    assert sparse(cache(), n=0) == INVALID
    assert sparse(cache(), idx=None, n=1025) == INVALID
    assert sparse(cache(), slots=1) == INVALID  # no page table
    assert sparse(cache(), tail_len=3) == INVALID
    assert sparse(cache(), tail=PTR, tail_len=3, tts=1028) == INVALID
    assert sparse(cache(), n=900, stride=900, nbytes=256) == WORKSPACE  # (one of up to 512 rows needs none)
    far = dict(page_table=PTR, page_size=128, page_table_stride=(1 << 24) - 1, num_pages=9, page_stride=1 << 17, scale_page_stride=16)
    assert dense(cache(**far), n=(1 << 31) - 65535) == UNSUPPORTED  # row numbers of a last step would pass 32 bits
    assert sparse(cache(**far), idx=None, n=(1 << 31) - 65600, tail=PTR, tail_len=128) == UNSUPPORTED
    gap = dict(page_table=PTR, page_size=64, page_table_stride=4, num_pages=9, page_stride=65 * 128 * 8, token_stride=1024)
    assert sparse(cache(**gap), slots=1) == INVALID
    n, c = C.c_size_t(0), cache()
    size = _lib.lib().okv_kv8_workspace_bytes
    assert size(C.byref(c), 32, 0, 10, 0, 0, C.byref(n)) == INVALID
    assert size(C.byref(c), 4, 1, 10, 0, 0, C.byref(n)) == INVALID
    assert size(C.byref(c), 32, 1, -1, 0, 0, C.byref(n)) == INVALID
    assert size(C.byref(c), 32, 1, 10, 0, 0, None) == INVALID
    assert size(None, 32, 1, 10, 0, 0, C.byref(n)) == INVALID
    assert size(C.byref(c), 32, 1, 100000, 0, 0, C.byref(n)) == 0 and n.value > 0


def test_page_refusals():
    l, pool = _lib.lib(), _lib.PagePool(PTR, PTR, PTR, 8, 4, 8, 100, 16)
    buf = (_lib.PageBuffer * 1)(_lib.PageBuffer(PTR, 4096))
    n = C.c_size_t(0)
    assert l.okv_pages_workspace_bytes(C.byref(pool), 3, C.byref(n)) == 0 and n.value > 0
    big = 1 << 40
    for field, value in (("table", None), ("refs", None), ("lens", None), ("num_seqs", 0), ("max_pages", 0), ("num_pages", 0),
                         ("page_size", 0), ("table_stride", 7)):
        bad = _lib.PagePool(PTR, PTR, PTR, 8, 4, 8, 100, 16)
        setattr(bad, field, value)
        assert l.okv_pages_free(C.byref(bad), PTR, 1, None, None) == INVALID
        assert l.okv_pages_fork(C.byref(bad), PTR, PTR, 1, buf, 1, None, 0, None, PTR, big, None) == INVALID
        assert l.okv_pages_extend(C.byref(bad), PTR, PTR, 1, None, None) == INVALID
        if field != "lens":
            assert l.okv_pages_compact(C.byref(bad), PTR, 8, PTR, None, buf, 1, PTR, big, None) == INVALID
    assert l.okv_pages_free(C.byref(pool), None, 1, None, None) == INVALID
    assert l.okv_pages_free(C.byref(pool), PTR, 0, None, None) == INVALID
    assert l.okv_pages_fork(C.byref(pool), PTR, None, 1, buf, 1, None, 0, None, PTR, big, None) == INVALID
    assert l.okv_pages_fork(C.byref(pool), PTR, PTR, 1, buf, 1, None, 0, None, PTR, 16, None) == WORKSPACE
    assert l.okv_pages_fork(C.byref(pool), PTR, PTR, 1, None, 1, None, 0, None, PTR, big, None) == INVALID
    assert l.okv_pages_fork(C.byref(pool), PTR, PTR, 1, buf, 1, None, 2, None, PTR, big, None) == INVALID
    assert l.okv_pages_extend(C.byref(pool), PTR, None, 1, None, None) == INVALID
    wide = _lib.PagePool(PTR, PTR, PTR, 1 << 21, 4, 1 << 21, 100, 16)
    assert l.okv_pages_extend(C.byref(wide), PTR, PTR, 1024, None, None) == UNSUPPORTED
    assert l.okv_pages_extend(C.byref(pool), PTR, PTR, 1025, None, None) == UNSUPPORTED
    assert l.okv_pages_fork(C.byref(pool), PTR, PTR, 1025, buf, 1, None, 0, None, PTR, big, None) == UNSUPPORTED
    assert l.okv_pages_copy(buf, 1, 100, None, PTR, None, 3, None) == INVALID
    assert l.okv_pages_copy(buf, 1, 100, None, None, None, 0, None) == 0
    assert l.okv_pages_compact(C.byref(pool), PTR, 7, PTR, None, buf, 1, PTR, big, None) == INVALID
    for base, size in ((PTR + 2, 4096), (PTR, 4098), (None, 4096), (PTR, 0)):
        odd = (_lib.PageBuffer * 1)(_lib.PageBuffer(base, size))
        assert l.okv_pages_copy(odd, 1, 100, PTR, PTR, None, 3, None) == INVALID


def test_python_front_end_refuses_cpu_tensors_and_shapes():
    k = torch.zeros((1, 2, 64, 128), dtype=torch.int8)
    s = torch.zeros((1, 2, 1))
    with pytest.raises(ValueError, match="one GPU"):
        ops.KV8(k, k, s, s, 64)
    with pytest.raises(ValueError, match="codes"):
        ops.KV8(k.to(torch.bfloat16), k, s, s, 64)
    with pytest.raises(ValueError, match="block"):
        ops.KV8(k, k, s, s, 48)
    with pytest.raises(ValueError, match="scales"):
        ops.KV8(k, k, s[:, :1], s, 64)
    with pytest.raises(ValueError, match="contiguous"):
        ops.PageBuffers([torch.zeros((4, 16))])
    with pytest.raises(ValueError, match="table"):
        ops.pages_free(torch.zeros((2, 4), dtype=torch.int32), torch.zeros(2), torch.zeros(4), torch.zeros(1), 16)


def cpu_cache(bsz=2, hkv=2, cap=1024):
    """A handle whose tensors are on the CPU: every check of a front end runs before anything is launched."""
    c = ops.KV8.__new__(ops.KV8)
    c.device, c.bsz, c.num_kv_heads, c.capacity, c.block, c.page_table = torch.device("cpu"), bsz, hkv, cap, 64, None
    c._c = {torch.bfloat16: cache(num_kv_heads=hkv, capacity=cap)}
    c._ref = {dt: C.byref(x) for dt, x in c._c.items()}
    c._ws_bytes, c._writable = {}, True
    return c


def test_select_refuses_an_output_that_does_not_fit():
    c, q = cpu_cache(), torch.zeros((2, 8, 128), dtype=torch.bfloat16)
    good = torch.zeros((2, 20), dtype=torch.int32)
    for out in (good.long(), good.float(), good[:1], good[:, :19], torch.zeros((2, 21), dtype=torch.int32), good[0],
                torch.zeros((20, 2), dtype=torch.int32).t(), torch.zeros((2, 40), dtype=torch.int32)[:, ::2],
                good[:1].expand(2, 20), torch.zeros((2, 20), dtype=torch.int32, device="meta")):
        with pytest.raises(ValueError, match="idx_out"):
            ops.kv8_dense_attn(q, c, seq_len=500, selector="last", score_len=400, select_k=20, idx_out=out)
    with pytest.raises(ValueError, match="idx_out"):  # no more entries than there are scores
        ops.kv8_dense_attn(q, c, seq_len=500, selector="last", score_len=10, select_k=20, idx_out=good)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("hkv, group, code", [(1, 9, UNSUPPORTED), (2, 72, UNSUPPORTED), (1, 129, UNSUPPORTED), (1, 256, UNSUPPORTED),
                                              (8, 1000, UNSUPPORTED), (64, 8, UNSUPPORTED)])
def test_scratch_of_unsupported_heads_is_refused_as_the_call_is(paged, hkv, group, code):
    c = cache(num_kv_heads=hkv, token_stride=128 * hkv, head_stride=128)
    if paged:
        for k, v in dict(page_table=PTR, page_size=64, page_table_stride=16, num_pages=20, page_stride=64 * 128 * hkv).items():
            setattr(c, k, v)
    n = C.c_size_t(0)
    for rows, score_len in ((1000, 500), (1000, 0), (100, 0)):
        assert _lib.lib().okv_kv8_workspace_bytes(C.byref(c), hkv * group, 1, rows, score_len, 0, C.byref(n)) == code
    assert dense(c, hq=hkv * group, n=1000, scores=PTR, score_len=500) == code


def test_scratch_of_other_bad_sizes_is_refused():
    size, c, n = _lib.lib().okv_kv8_workspace_bytes, cache(), C.c_size_t(0)
    assert size(C.byref(c), 31, 1, 1000, 500, 0, C.byref(n)) == INVALID
    assert size(C.byref(c), 32, 65536, 10, 0, 0, C.byref(n)) == UNSUPPORTED
    assert size(C.byref(c), 32, 3, 1 << 30, 0, 0, C.byref(n)) == UNSUPPORTED
    assert size(C.byref(c), 32, 1, (1 << 31) - 65536, 500, 0, C.byref(n)) == 0


def test_selecting_with_unsupported_heads_raises():
    c = cpu_cache(bsz=1, hkv=1)
    with pytest.raises(Exception, match="GQA group size 200"):
        ops.kv8_dense_attn(torch.zeros((1, 200, 128), dtype=torch.bfloat16), c, seq_len=1000, selector="last", select_k=5)


def test_scratch_of_an_indexed_call_is_enough_for_an_empty_index():
    """An array without entries has no address: such a call runs as one without an index."""
    n, size = [C.c_size_t(0), C.c_size_t(0)], _lib.lib().okv_kv8_workspace_bytes
    for hkv in (1, 2, 8):
        for page in (0, 64):
            c = cache(num_kv_heads=hkv, token_stride=128 * hkv, head_stride=128, page_table=PTR if page else None, page_size=page,
                      page_table_stride=16, num_pages=20, page_stride=64 * 128 * hkv)
            for batch in (1, 2, 3, 17):
                for rows in (1, 512, 600, 1400, 2049, 30000):
                    for indexed in (0, 1):
                        assert size(C.byref(c), 4 * hkv, batch, rows, 0, indexed, C.byref(n[indexed])) == 0
                    assert n[1].value >= n[0].value, (hkv, page, batch, rows)


def test_pools_and_lists_beyond_what_the_plans_count_are_refused():
    """Page, sequence and entry numbers run past the last one by a step of a workgroup, and stay in 32 bits."""
    l, most = _lib.lib(), (1 << 31) - 1
    buf = (_lib.PageBuffer * 1)(_lib.PageBuffer(PTR, 4096))
    big, n = 1 << 50, C.c_size_t(0)
    for field in ("num_pages", "max_pages", "num_seqs"):
        pool = _lib.PagePool(PTR, PTR, PTR, 1 << 32, 4, 8, 100, 16)
        setattr(pool, field, most)
        assert l.okv_pages_free(C.byref(pool), PTR, 1, None, None) == UNSUPPORTED
        assert l.okv_pages_fork(C.byref(pool), PTR, PTR, 1, buf, 1, None, 0, None, PTR, big, None) == UNSUPPORTED
        assert l.okv_pages_extend(C.byref(pool), PTR, PTR, 1, None, None) == UNSUPPORTED
        assert l.okv_pages_compact(C.byref(pool), PTR, 1 << 32, PTR, None, buf, 1, PTR, big, None) == UNSUPPORTED
        if field != "max_pages":
            assert l.okv_pages_workspace_bytes(C.byref(pool), 3, C.byref(n)) == UNSUPPORTED
    ok = _lib.PagePool(PTR, PTR, PTR, 8, 4, 8, 100, 16)
    assert l.okv_pages_workspace_bytes(C.byref(ok), most, C.byref(n)) == UNSUPPORTED
    assert l.okv_pages_free(C.byref(ok), PTR, most, None, None) == UNSUPPORTED
    assert l.okv_pages_copy(buf, 1, 100, PTR, PTR, None, most, None) == UNSUPPORTED
    assert l.okv_pages_copy(buf, 1, most, PTR, PTR, None, 3, None) == UNSUPPORTED
    meta = lambda *shape: torch.empty(shape, dtype=torch.int32, device="meta")  # noqa: E731
    with pytest.raises(ValueError, match="2\\^30"):  # (2^32 + 5 would arrive as 5)
        ops.pages_free(meta(4, 8), meta(4), meta((1 << 32) + 5), meta(1), 16)
    with pytest.raises(ValueError, match="2\\^30"):
        ops.PageBuffers([meta((1 << 32) + 5, 4)])


def test_calls_of_no_rows_need_no_arrays():
    """An array without rows has no address."""
    c, l = cache(), _lib.lib()
    assert l.okv_kv8_read(C.byref(c), None, 0, 0, None, 10, 1, None, None, 128, 1280, 0, None) == 0
    assert l.okv_kv8_read(C.byref(c), None, 0, 1, None, 10, 1, None, None, 128, 1280, 0, None) == INVALID
    assert l.okv_kv8_append(C.byref(c), None, 1024, 128, 0, None, 1024, 128, 0, None, 0, None, 0, 0, 1, None) == 0
    assert l.okv_kv8_append(C.byref(c), None, 1024, 128, 0, None, 1024, 128, 0, None, 0, None, 4, 0, 1, None) == INVALID
    assert append(c, start=2000, n=0) == INVALID
