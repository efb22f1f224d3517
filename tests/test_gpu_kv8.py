"""The 8-bit K/V cache on the GPU against plain 64-bit restatements (tests/kv8_reference.py).

Written rows are compared bit for bit: every rounding of the format is fixed.  Attention outputs and scores are held to
bounds that kv8_reference derives from the inputs (logit_error, output_bound)."""
import pytest
import torch

import kv8_reference as ref
from omnikv_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


def rows(g, *shape, dtype=BF, gain=1.0):
    x = torch.randn(*shape, 128, generator=g) * gain
    x[..., ::31] *= 5.0
    return x.to(dtype)


def make(g, fmt, dtype, block, page, lens, hkv, open_rows=True, spare=1):
    """A cache holding requests of the given lengths, filled by one append, and its exact contents: (cache, [k], [v])
    with k, v (hkv, len, 128) float64 per request."""
    bsz, n = len(lens), max(max(lens), 1)
    k, v = (rows(g, bsz, hkv, n, dtype=dtype) for _ in "kv")
    cap = (-(-n // block) + spare) * block
    if page:
        per = -(-cap // page)
        table = torch.randperm(bsz * per + 3, generator=g)[: bsz * per].to(torch.int32).view(bsz, per).to(DEV)
        cache = ops.KV8.empty_paged(table, bsz * per + 3, page, hkv, fmt, block, dtype if open_rows else None)
    else:
        cache = ops.KV8.empty(bsz, hkv, cap, fmt, block, dtype if open_rows else None, DEV)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ops.kv8_append(cache, k.to(DEV), v.to(DEV), 0, lens_t, close=not open_rows)
    return cache, [held(x[:, :m], fmt, block, open_rows) for x, m in zip(k, lens)], \
        [held(x[:, :m], fmt, block, open_rows) for x, m in zip(v, lens)]


def held(x, fmt, block, open_rows):
    """What the cache holds of rows x (hkv, n, 128): float64 values."""
    n = x.shape[1]
    full = n if not open_rows else n // block * block
    parts = []
    for lo in range(0, full, block):
        c, s = ref.quantise(x[:, lo: min(lo + block, full)], fmt)
        parts.append(c * s.double()[:, None, None])
    parts.append(x[:, full:].double())
    return torch.cat(parts, 1)


def read_back(cache, request, n, hkv):
    """codes * scale of the first n rows of a request, straight from its tensors."""
    out = []
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes, scale = codes.cpu().double(), scale.cpu().double()
        if cache.page_table is not None:
            pages = cache.page_table[request].cpu().long()
            c = codes[pages].flatten(0, 1).transpose(0, 1)
            s = scale[pages].flatten(0, 1).transpose(0, 1)
        else:
            c, s = codes[request], scale[request]
        out.append((c * s.repeat_interleave(cache.block, 1)[..., None])[:, :n])
    return out


# ------------------------------------------------------------------------------------------ append, read
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("block, page", [(16, 0), (64, 0), (128, 0), (16, 48), (32, 32), (64, 128)])
def test_append_in_pieces_equals_one_append(fmt, dtype, block, page):
    """A prompt, chunks that end inside blocks, single tokens, an empty append: the codes are those of one quantisation."""
    g = torch.Generator().manual_seed(1)
    bsz, hkv = 3, 2
    pieces = [5, block + 7, 1, 1, 2 * block - 14, 0, 3 * block + 1, 1]
    total = sum(pieces)
    k, v = rows(g, bsz, hkv, total, dtype=dtype), rows(g, bsz, hkv, total, dtype=dtype, gain=3e-3)
    cache, _, _ = make(g, fmt, dtype, block, page, [total + 2 * block] * bsz, hkv)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0x55)
    lens = torch.zeros(bsz, dtype=torch.int32, device=DEV)
    at = 0
    for n in pieces:
        ops.kv8_append(cache, k[:, :, at: at + n].to(DEV), v[:, :, at: at + n].to(DEV), lens)
        lens += n
        at += n
    full = total // block * block
    for b in range(bsz):
        for got, x in zip(read_back(cache, b, full, hkv), (k, v)):
            assert torch.equal(got, held(x[b, :, :full], fmt, block, True))
    for got, x in ((cache.open_k, k), (cache.open_v, v)):
        assert torch.equal(got[:, :, : total - full].cpu(), x[:, :, full:])
    # rows behind the last full block: left as they were
    codes = cache.k if page == 0 else cache.k[cache.page_table.long()].flatten(1, 2).transpose(1, 2)
    assert bool((codes.contiguous().view(torch.uint8)[:, :, full: full + block] == 0x55).all())
    rk, rv = ops.kv8_read(cache, dtype, seq_len=total + 1, seq_lens=lens)
    for got, x in ((rk, k), (rv, v)):
        for b in range(bsz):
            assert torch.equal(got[b, :, :total].cpu(), held(x[b], fmt, block, True).float().to(dtype))
        assert not got[:, :, total:].any()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("n", [1, 15, 64, 65, 200])
def test_append_closing_the_last_block(fmt, n):
    g = torch.Generator().manual_seed(2)
    cache, k, v = make(g, fmt, BF, 64, 0, [n], 3, open_rows=False)
    cache.k.view(torch.uint8)[:, :, n:].fill_(7)
    for got, want in zip(read_back(cache, 0, n, 3), (k[0], v[0])):
        assert torch.equal(got, want)
    x = rows(g, 1, 3, n)
    ops.kv8_append(cache, x.to(DEV), x.to(DEV), 0, close=True)
    assert torch.equal(read_back(cache, 0, n, 3)[0], held(x[0], fmt, 64, False))
    assert bool((cache.k.view(torch.uint8)[:, :, n:] == 7).all())


def test_append_strides_ragged_lengths_and_what_does_not_fit():
    g = torch.Generator().manual_seed(3)
    cache = ops.KV8.empty(4, 2, 96, "int8", 32, BF, DEV)
    x = rows(g, 4, 40, 2).transpose(1, 2)  # (b, heads, n, 128), token-major storage
    y = rows(g, 4, 2, 40)  # V in other strides than K
    starts = torch.tensor([0, 60, -1, 57], dtype=torch.int32, device=DEV)  # 60 + 40 and -1 do not fit
    lens = torch.tensor([33, 40, 40, 7], dtype=torch.int32, device=DEV)
    ops.kv8_append(cache, x.to(DEV), y.to(DEV), starts, lens)
    assert torch.equal(read_back(cache, 0, 32, 2)[0], held(x[0, :, :32], "int8", 32, True))
    assert torch.equal(cache.open_v[0, :, :1].cpu(), y[0, :, 32:33])
    for b in (1, 2):
        assert not cache.k_scale[b].any() and not cache.open_k[b].any()
    want = torch.zeros(2, 32, 128, dtype=BF)  # request 3: its rows 57 .. 64 complete block 1 behind open rows of zeros
    want[:, 25:32] = x[3, :, :7]
    c, s = ref.quantise(want, "int8")
    assert torch.equal(read_back(cache, 3, 64, 2)[0][:, 32:], c * s.double()[:, None, None])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_at_the_borders_of_the_format(fmt, dtype):
    """Zeros, the type's extremes, subnormals, exact ties, and NaN / infinity poisoning their block only."""
    g = torch.Generator().manual_seed(4)
    big = torch.finfo(dtype).max
    x = torch.zeros(1, 1, 16 * 8, 128, dtype=dtype)
    x[..., 16:32, :] = torch.linspace(-1, 1, 128).to(dtype) * big
    x[..., 32:48, :] = torch.finfo(dtype).smallest_normal * torch.arange(128).to(dtype) / 256
    x[..., 48:64, :] = (torch.arange(128) - 64).to(dtype)  # amax / 2, the tie of the integer format, among them
    x[..., 64:80, :] = (torch.arange(2048).view(16, 128) % 897 - 448).to(dtype)  # e4m3: every integer up to qmax, scale 1
    x[..., 80:96, :] = rows(g, 16, dtype=dtype)
    x[..., 85, 3] = float("inf")
    x[..., 96:112, :] = rows(g, 16, dtype=dtype)
    x[..., 100, 90] = float("nan")
    x[..., 112:, :] = rows(g, 16, dtype=dtype)
    cache = ops.KV8.empty(1, 1, 128, fmt, 16, dtype, DEV)
    ops.kv8_append(cache, x.to(DEV), x.to(DEV), 0)
    for lo in range(0, 128, 16):
        c, s = ref.quantise(x[0, :, lo: lo + 16], fmt)
        assert torch.equal(cache.k[0, :, lo: lo + 16].cpu().double(), c), lo
        assert torch.equal(cache.v_scale[0, :, lo // 16].cpu().nan_to_num(-1), s.nan_to_num(-1)), lo
    q = rows(g, 1, 2, dtype=dtype).to(DEV)
    assert bool(ops.kv8_dense_attn(q, cache, seq_len=96).isnan().all())
    # rows of the finite blocks; without the block of bfloat16's largest numbers (3.4e38), whose logits, sums of
    # 128 products with queries of order 1 to 5, are beyond fp32 in any arithmetic that forms them there
    at = torch.cat([torch.arange(0, 16), torch.arange(32, 80), torch.arange(112, 128)]).to(torch.int32).to(DEV)[None]
    assert bool(ops.kv8_sparse_attn(q, cache, idx=at).isfinite().all())


# ------------------------------------------------------------------------------------------ attention
def check_attention(got, q, ks, vs, scale, dtype):
    for b, (k, v) in enumerate(zip(ks, vs)):
        out, _, _, spread, mass = ref.attention(q[b], k, v, scale)
        bound = ref.output_bound(out, spread, mass, dtype)
        diff = (got[b].cpu().double() - out).abs()
        assert bool((diff <= bound).all()), (b, float((diff / bound).max()))


DENSE = [
    # fmt, dtype, block, page, hkv, group, lengths
    ("e4m3", BF, 64, 0, 2, 4, [1]),
    ("int8", BF, 16, 0, 1, 1, [17, 16, 15, 1, 0, 33]),
    ("e4m3", HF, 32, 0, 3, 7, [31, 32, 64, 95, 0]),
    ("int8", HF, 64, 0, 8, 8, [700]),
    ("e4m3", BF, 128, 0, 2, 2, [127, 128, 129, 515]),
    ("int8", BF, 16, 16, 8, 4, [1, 100, 257, 0, 512]),
    ("e4m3", HF, 16, 48, 5, 3, [1000, 47, 48, 49]),
    ("int8", HF, 32, 96, 2, 5, [95, 96, 97, 64]),
    ("e4m3", BF, 64, 64, 8, 4, [3001]),
    ("int8", BF, 64, 0, 4, 6, [5000, 1, 4097]),
]


@pytest.mark.parametrize("fmt, dtype, block, page, hkv, group, lens", DENSE)
def test_dense(fmt, dtype, block, page, hkv, group, lens):
    g = torch.Generator().manual_seed(11)
    cache, ks, vs = make(g, fmt, dtype, block, page, lens, hkv)
    q = rows(g, len(lens), hkv * group, dtype=dtype)
    t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = ops.kv8_dense_attn(q.to(DEV), cache, seq_lens=t, seq_len=max(lens))
    check_attention(out, q, ks, vs, 128 ** -0.5, dtype)
    for b, n in enumerate(lens):
        if n == 0:
            assert not out[b].any()
    # a longer bound on the lengths splits the rows otherwise
    more = ops.kv8_dense_attn(q.to(DEV)[:, :, None], cache, seq_lens=t, scale=0.3)
    check_attention(more, q, ks, vs, 0.3, dtype)


@pytest.mark.parametrize("fmt, dtype, block, page, hkv, group, lens", DENSE[1:])
@pytest.mark.parametrize("selector", ["last", "softmax_before_last", "softmax_sum_last"])
def test_dense_scores(fmt, dtype, block, page, hkv, group, lens, selector):
    """Scored lengths that end inside a block, at and behind the open rows, and beyond a request's own length."""
    g = torch.Generator().manual_seed(12)
    cache, ks, vs = make(g, fmt, dtype, block, page, lens, hkv)
    q = rows(g, len(lens), hkv * group, dtype=dtype)
    most = max(lens)
    want_len = [max(0, n - (0, 1, 13)[b % 3]) for b, n in enumerate(lens)]
    t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    tl = torch.tensor(want_len, dtype=torch.int32, device=DEV)
    buf = torch.full((len(lens), most + 5), 77.0, device=DEV)[:, :most]
    out, scores = ops.kv8_dense_attn(q.to(DEV), cache, seq_lens=t, seq_len=most, selector=selector, score_len=most,
                                     score_lens=tl, scores_out=buf)
    assert scores.data_ptr() == buf.data_ptr()
    check_attention(out, q, ks, vs, 128 ** -0.5, dtype)
    for b, n in enumerate(want_len):
        assert bool((scores[b, n:] == 77).all())
        if n == 0:
            continue
        _, x, p, _, mass = ref.attention(q[b], ks[b][:, :n], vs[b][:, :n], 128 ** -0.5)
        dl = ref.logit_error(mass)
        if selector == "last":
            y, bound = x.amax(0), dl.amax(0)
        else:
            # the logit's own error and the normaliser's; 2^-18 for exponentials and sums in fp32
            rel = torch.expm1(dl + dl.amax(1, keepdim=True)) * 2 + 2.0 ** -18
            y, bound = (p.amax(0), (p * rel).amax(0)) if selector == "softmax_before_last" else (p.sum(0), (p * rel).sum(0))
            bound = bound + 2.0 ** -120
        diff = (scores[b, :n].cpu().double() - y).abs()
        assert bool((diff <= bound).all()), (b, float((diff / bound).max()))


def test_dense_select_equals_topk_of_its_scores():
    g = torch.Generator().manual_seed(13)
    cache, _, _ = make(g, "e4m3", BF, 64, 0, [900, 500], 2)
    q = rows(g, 2, 8).to(DEV)
    t = torch.tensor([900, 500], dtype=torch.int32, device=DEV)
    out, scores, idx = ops.kv8_dense_attn(q, cache, seq_lens=t, seq_len=900, selector="softmax_before_last", score_len=900,
                                          score_lens=t, select_k=60)
    assert torch.equal(idx, ops.topk(scores, 60, t))
    assert torch.equal(out, ops.kv8_dense_attn(q, cache, seq_lens=t, seq_len=900, selector="last")[0])


@pytest.mark.parametrize("lens", [[900, 500, 30, 0], [20000, 150, 15000, 16384]])
def test_dense_select_ranks_the_requests_own_rows_alone(lens):
    """Ragged lengths without score_lens, with larger ones, and with smaller and larger ones: what a request has no rows
    for is never selected, whatever the buffer of the scores held."""
    g = torch.Generator().manual_seed(14)
    cache, _, _ = make(g, "int8", BF, 16, 0, lens, 1)
    q, n, k = rows(g, 4, 4).to(DEV), max(lens), 60
    t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for wanted in (None, t, t + 100, torch.tensor([n, 40, n, 40], dtype=torch.int32, device=DEV)):
        buf = torch.full((4, n), 1e9, device=DEV)
        out, scores, idx = ops.kv8_dense_attn(q, cache, seq_lens=t, seq_len=n, selector="last", score_len=n, score_lens=wanted,
                                              scores_out=buf, select_k=k)
        scored = t if wanted is None else torch.minimum(t, wanted)
        assert idx.shape == (4, k) and bool((scores.cpu() == 1e9).sum(1).eq(n - scored.cpu()).all())
        for b, m in enumerate(scored.tolist()):
            want = torch.full((k,), -1, dtype=torch.int32)
            if m:
                top = torch.sort(scores[b, :m].cpu(), descending=True, stable=True)[1][:k].sort()[0]
                want[: top.numel()] = top.to(torch.int32)
            assert torch.equal(idx[b].cpu(), want), (b, m)


SPARSE = [
    # fmt, dtype, block, page, hkv, group, lengths, selected rows, tails
    ("e4m3", BF, 64, 0, 2, 4, [300], [1], [0]),
    ("int8", BF, 16, 0, 8, 4, [500, 40, 7], [100, 40, 0], [5, 0, 3]),
    ("e4m3", HF, 32, 0, 3, 7, [1000, 1000], [333, 0], [0, 0]),
    ("int8", HF, 16, 16, 5, 2, [2000, 100, 33, 17], [1500, 99, 33, 1], [129, 0, 31, 16]),
    ("e4m3", BF, 16, 48, 8, 8, [700, 3], [70, 3], [1, 40]),
    ("int8", BF, 64, 0, 1, 1, [6000], [5999], [700]),
]


@pytest.mark.parametrize("fmt, dtype, block, page, hkv, group, lens, picks, tails", SPARSE)
def test_sparse(fmt, dtype, block, page, hkv, group, lens, picks, tails):
    g = torch.Generator().manual_seed(21)
    bsz = len(lens)
    cache, ks, vs = make(g, fmt, dtype, block, page, lens, hkv, open_rows=False)
    q = rows(g, bsz, hkv * group, dtype=dtype)
    idx = torch.full((bsz, max(picks) + 3), -1, dtype=torch.int32)
    tk, tv = (rows(g, bsz, max(tails) + 1, hkv, dtype=dtype).transpose(1, 2) for _ in "kv")
    wk, wv = [], []
    for b in range(bsz):
        at = torch.randperm(lens[b], generator=g)[: picks[b]].sort()[0]
        idx[b, : picks[b]] = at.to(torch.int32)
        wk.append(torch.cat([ks[b][:, at], tk[b, :, : tails[b]].double()], 1))
        wv.append(torch.cat([vs[b][:, at], tv[b, :, : tails[b]].double()], 1))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    kw = dict(tail_k=tk.to(DEV), tail_v=tv.to(DEV), tail_lens=i32(tails))
    di = idx.to(DEV)
    out = ops.kv8_sparse_attn(q.to(DEV), cache, idx=di, sel_lens=i32(picks), **kw)
    check_attention(out, q, wk, wv, 128 ** -0.5, dtype)
    padded = ops.kv8_sparse_attn(q.to(DEV), cache, idx=di, **kw)  # padding (-1) takes no part
    check_attention(padded, q, wk, wv, 128 ** -0.5, dtype)
    stray = torch.where(di < 0, 1 << 30, di)
    assert torch.equal(ops.kv8_sparse_attn(q.to(DEV), cache, idx=stray, **kw), padded)
    if page:
        slots = cache.slot_index(di)
        assert torch.equal(ops.kv8_sparse_attn(q.to(DEV), cache, slots=slots, sel_lens=i32(picks), **kw), out)
    if max(tails) == 0:
        none = ops.kv8_sparse_attn(q.to(DEV), cache, idx=di, sel_lens=i32(picks))
        check_attention(none, q, wk, wv, 128 ** -0.5, dtype)


@pytest.mark.parametrize("page", [0, 32])
def test_batch_of_many_ragged_requests(page):
    """More requests than a wave has lanes: the shares of all of them, scored and not, through an index and not."""
    g = torch.Generator().manual_seed(25)
    lens = [int(x) for x in torch.randint(0, 900, (131,), generator=g)]
    lens[0], lens[64], lens[130] = 2500, 0, 2900
    cache, ks, vs = make(g, "int8", BF, 16, page, lens, 1)
    q = rows(g, 131, 2)
    t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    check_attention(ops.kv8_dense_attn(q.to(DEV), cache, seq_lens=t, seq_len=2900), q, ks, vs, 128 ** -0.5, BF)
    out, raw = ops.kv8_dense_attn(q.to(DEV), cache, seq_lens=t, seq_len=2900, selector="last", score_len=2900, score_lens=t - 1)
    check_attention(out, q, ks, vs, 128 ** -0.5, BF)
    for b in (0, 1, 77, 130):
        _, x, _, _, mass = ref.attention(q[b], ks[b], vs[b], 128 ** -0.5)
        n = max(lens[b] - 1, 0)
        assert bool(((raw[b, :n].cpu().double() - x.amax(0)[:n]).abs() <= ref.logit_error(mass).amax(0)[:n]).all())
    closed = [n // 16 * 16 for n in lens]
    idx = torch.arange(0, 2900, 3, dtype=torch.int32, device=DEV).expand(131, -1).contiguous()
    picks = torch.tensor([(n + 2) // 3 for n in closed], dtype=torch.int32, device=DEV)
    got = ops.kv8_sparse_attn(q.to(DEV), cache, idx=idx, sel_lens=picks)
    check_attention(got, q, [k[:, :n:3] for k, n in zip(ks, closed)], [v[:, :n:3] for v, n in zip(vs, closed)], 128 ** -0.5, BF)


@pytest.mark.parametrize("bsz, hkv, most", [(1, 8, 512), (3, 2, 513), (70, 4, 500), (70, 4, 2047), (33, 8, 130)])
@pytest.mark.parametrize("page", [0, 48])
def test_short_requests_in_one_launch(bsz, hkv, most, page):
    """Around the sizes where a request is one share, few and many of them, one of no rows, one of a single open row."""
    g = torch.Generator().manual_seed(27)
    lens = [int(x) for x in torch.randint(2, most + 1, (bsz,), generator=g)]
    lens[0] = most
    if bsz > 2:
        lens[1], lens[2] = 0, 1
    cache, ks, vs = make(g, "int8", HF, 16, page, lens, hkv)
    q = rows(g, bsz, 2 * hkv, dtype=HF)
    t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    check_attention(ops.kv8_dense_attn(q.to(DEV), cache, seq_lens=t, seq_len=most), q, ks, vs, 128 ** -0.5, HF)
    closed = [n // 16 * 16 for n in lens]
    idx = torch.arange(0, most, dtype=torch.int32, device=DEV).flip(0).expand(bsz, -1).contiguous()
    idx[idx >= torch.tensor(closed, device=DEV)[:, None]] = -1  # padding in front of the request's own rows
    tk, tv = rows(g, bsz, hkv, 3, dtype=HF), rows(g, bsz, hkv, 3, dtype=HF)
    got = ops.kv8_sparse_attn(q.to(DEV), cache, idx=idx, tail_k=tk.to(DEV), tail_v=tv.to(DEV))
    check_attention(got, q, [torch.cat([k[:, :n].flip(1), x.double()], 1) for k, n, x in zip(ks, closed, tk)],
                    [torch.cat([v[:, :n].flip(1), x.double()], 1) for v, n, x in zip(vs, closed, tv)], 128 ** -0.5, HF)


def test_a_shared_prompt_can_be_read_by_several_requests_and_not_written():
    g = torch.Generator().manual_seed(26)
    one, ks, vs = make(g, "e4m3", BF, 32, 0, [600], 2, open_rows=False)
    ex = [t.expand(3, *t.shape[1:]) for t in (one.k, one.v, one.k_scale, one.v_scale)]
    cache = ops.KV8(*ex, 32)
    q = rows(g, 3, 8)
    check_attention(ops.kv8_dense_attn(q.to(DEV), cache, seq_len=600), q, ks * 3, vs * 3, 128 ** -0.5, BF)
    with pytest.raises(ValueError, match="read only"):
        ops.kv8_append(cache, q[:, :2, None].to(DEV), q[:, :2, None].to(DEV), 0, close=True)


def test_sparse_without_an_index_and_with_a_tail_alone():
    g = torch.Generator().manual_seed(22)
    cache, ks, vs = make(g, "int8", BF, 32, 0, [130, 77], 2, open_rows=False)
    q = rows(g, 2, 8)
    tk, tv = rows(g, 2, 2, 9), rows(g, 2, 2, 9)
    n = torch.tensor([130, 77], dtype=torch.int32, device=DEV)
    out = ops.kv8_sparse_attn(q.to(DEV), cache, sel_len=130, sel_lens=n, tail_k=tk.to(DEV), tail_v=tv.to(DEV))
    check_attention(out, q, [torch.cat([k, t.double()], 1) for k, t in zip(ks, tk)],
                    [torch.cat([v, t.double()], 1) for v, t in zip(vs, tv)], 128 ** -0.5, BF)
    out = ops.kv8_sparse_attn(q.to(DEV), cache, sel_len=0, tail_k=tk.to(DEV), tail_v=tv.to(DEV), tail_len=4)
    check_attention(out, q, tk[:, :, :4].double(), tv[:, :, :4].double(), 128 ** -0.5, BF)


@pytest.mark.parametrize("bsz", [1, 2, 5])
@pytest.mark.parametrize("page", [0, 32])
@pytest.mark.parametrize("tail", [1, 600, 2500])
def test_an_empty_selection_leaves_the_tail(bsz, page, tail):
    """An index without entries, contiguous, paged and by slots: the same as no selected rows at all."""
    g = torch.Generator().manual_seed(28)
    cache, _, _ = make(g, "int8", BF, 16, page, [80] * bsz, 2, open_rows=False)
    q, tk, tv = rows(g, bsz, 8), rows(g, bsz, 2, tail), rows(g, bsz, 2, tail)
    none = torch.empty((bsz, 0), dtype=torch.int32, device=DEV)
    kw = dict(tail_k=tk.to(DEV), tail_v=tv.to(DEV))
    for how in [dict(idx=none)] + ([dict(slots=none), dict(slots=cache.slot_index(none))] if page else []):
        check_attention(ops.kv8_sparse_attn(q.to(DEV), cache, **how, **kw), q, tk.double(), tv.double(), 128 ** -0.5, BF)
    some = torch.full((bsz, 4), 3, dtype=torch.int32, device=DEV)
    check_attention(ops.kv8_sparse_attn(q.to(DEV), cache, idx=some, sel_len=0, **kw), q, tk.double(), tv.double(), 128 ** -0.5, BF)
    with pytest.raises(Exception, match="no rows"):
        ops.kv8_sparse_attn(q.to(DEV), cache, idx=none)


def test_pages_outside_the_pool_take_no_part():
    g = torch.Generator().manual_seed(23)
    cache, ks, vs = make(g, "e4m3", BF, 16, 32, [200, 90], 2)
    q = rows(g, 2, 8)
    t = torch.tensor([200, 90], dtype=torch.int32, device=DEV)
    cache.page_table[0, 2], cache.page_table[0, 5] = -1, 1 << 30
    cache.page_table[1, :2] = -7
    keep = [[r for r in range(200) if r // 32 not in (2, 5)], [r for r in range(90) if r // 32 not in (0, 1)]]
    out, scores = ops.kv8_dense_attn(q.to(DEV), cache, seq_lens=t, seq_len=200, selector="softmax_sum_last", score_len=200,
                                     score_lens=t)
    check_attention(out, q, [k[:, i] for k, i in zip(ks, keep)], [v[:, i] for v, i in zip(vs, keep)], 128 ** -0.5, BF)
    assert not scores[0, 64:96].any() and not scores[0, 160:192].any() and bool(scores[0, :64].all())
    raw = ops.kv8_dense_attn(q.to(DEV), cache, seq_lens=t, seq_len=200, selector="last", score_len=200, score_lens=t)[1]
    assert bool((raw[0, 64:96] == float("-inf")).all()) and bool(raw[1, 64:90].isfinite().all())
    cache.page_table[:] = -1  # closed rows: none left
    only_open = ops.kv8_dense_attn(q.to(DEV), cache, seq_lens=t, seq_len=200)
    check_attention(only_open, q, [ks[0][:, 192:], ks[1][:, 80:]], [vs[0][:, 192:], vs[1][:, 80:]], 128 ** -0.5, BF)
    whole = torch.tensor([192, 80], dtype=torch.int32, device=DEV)
    out, scores = ops.kv8_dense_attn(q.to(DEV), cache, seq_lens=whole, seq_len=200, selector="softmax_before_last",
                                     score_len=192, score_lens=whole)
    assert not out.any() and not scores[0].any()
    x = rows(g, 2, 2, 1)
    before = [t.clone() for t in (cache.k.view(torch.uint8), cache.k_scale)]
    ops.kv8_append(cache, x.to(DEV), x.to(DEV), torch.tensor([207, 95], dtype=torch.int32, device=DEV))  # both fill a block
    assert torch.equal(cache.k.view(torch.uint8), before[0]) and torch.equal(cache.k_scale, before[1])


def test_large_values_and_a_lone_huge_logit():
    """Logits of thousands: the running maximum moves late, everything else underflows to nothing."""
    g = torch.Generator().manual_seed(24)
    cache, ks, vs = make(g, "int8", BF, 16, 0, [2000], 1)
    k = rows(g, 1, 1, 16, gain=300.0)
    v = rows(g, 1, 1, 16)
    ops.kv8_append(cache, k.to(DEV), v.to(DEV), 2000)
    ks[0], vs[0] = (torch.cat([a, held(x[0], "int8", 16, True)], 1) for a, x in ((ks[0], k), (vs[0], v)))
    q = rows(g, 1, 4, gain=8.0)
    out = ops.kv8_dense_attn(q.to(DEV), cache, seq_len=2016)
    # (2000 is a multiple of 16: the sixteen rows are one block)
    want, _, p, spread, mass = ref.attention(q[0], ks[0], vs[0], 128 ** -0.5)
    assert float(p.amax()) > 0.9
    dl = ref.logit_error(mass.amax())
    assert dl < 1  # else the bound says nothing
    assert bool(((out[0].cpu().double() - want).abs() <= ref.output_bound(want, spread, mass.amax(), BF)).all())


# ------------------------------------------------------------------------------------------ use together
def test_decode_loop_append_and_attend_in_a_replayed_graph():
    """A captured step (append one token, attend, score and select, attend to the selection) replayed with the lengths
    on the device, every replay against the eager step on a second cache, eager work and waits in between."""
    g = torch.Generator().manual_seed(31)
    lens0 = [125, 64, 1]
    caches = [make(torch.Generator().manual_seed(5), "e4m3", BF, 16, 32, lens0, 2, spare=8)[0] for _ in range(2)]
    steps = 40
    ks, vs = rows(g, steps, 3, 2, 1).to(DEV), rows(g, steps, 3, 2, 1).to(DEV)
    qs = rows(g, steps, 3, 8).to(DEV)
    bound = max(lens0) + steps

    def step(cache, q, k, v, lens):
        ops.kv8_append(cache, k, v, lens)
        lens += 1
        out, scores, idx = ops.kv8_dense_attn(q, cache, seq_lens=lens, seq_len=bound, selector="softmax_before_last",
                                              score_len=bound, score_lens=lens // 16 * 16, select_k=20)
        return out, idx, ops.kv8_sparse_attn(q, cache, idx=idx, tail_k=k, tail_v=v)

    q, k, v = qs[0].clone(), ks[0].clone(), vs[0].clone()
    lens = [torch.tensor(lens0, dtype=torch.int32, device=DEV) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        spare = make(torch.Generator().manual_seed(5), "e4m3", BF, 16, 32, lens0, 2, spare=8)[0]
        step(spare, q, k, v, torch.tensor(lens0, dtype=torch.int32, device=DEV))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0], q, k, v, lens[0])
    lens[0].copy_(torch.tensor(lens0))
    for i in range(steps):
        q.copy_(qs[i]), k.copy_(ks[i]), v.copy_(vs[i])
        graph.replay()
        want = step(caches[1], qs[i], ks[i], vs[i], lens[1])
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
        if i % 7 == 0:
            torch.cuda.synchronize()
    assert torch.equal(lens[0], lens[1])
    for name in ("k", "v"):
        assert torch.equal(getattr(caches[0], name).view(torch.uint8), getattr(caches[1], name).view(torch.uint8))


def test_two_graphs_and_another_stream_do_not_share_scratch():
    g = torch.Generator().manual_seed(32)
    cache, ks, vs = make(g, "int8", HF, 64, 0, [4000], 2)
    qa, qb = rows(g, 1, 8, dtype=HF).to(DEV), rows(g, 1, 8, dtype=HF).to(DEV)
    want = [ops.kv8_dense_attn(x, cache, seq_len=4000) for x in (qa, qb)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in (qa, qb):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.kv8_dense_attn(x, cache, seq_len=4000))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for s, gr in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                gr.replay()
        eager = ops.kv8_dense_attn(qa, cache, seq_len=4000)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])


def test_long_cache_offsets_pass_32_bits():
    """One request whose codes lie beyond 4 GiB from the base: every row attended through an index and densely."""
    g = torch.Generator().manual_seed(33)
    hkv, n = 2, 256
    far = (1 << 32) // 128 + 4096  # tokens between the two heads' rows: the second head starts behind 4 GiB
    base = [torch.zeros(far * 128 + n * 128, dtype=torch.uint8, device=DEV) for _ in "kv"]
    k, v = (torch.as_strided(t, (1, hkv, n, 128), (0, far * 128, 128, 1)).view(torch.int8) for t in base)
    s = torch.zeros((2, 1, hkv, n // 64), device=DEV)
    cache = ops.KV8(k, v, s[0], s[1], 64)
    x, y = rows(g, 1, hkv, n), rows(g, 1, hkv, n)
    ops.kv8_append(cache, x.to(DEV), y.to(DEV), 0, close=True)
    q = rows(g, 1, 8)
    kk, vv = [held(x[0], "int8", 64, False)], [held(y[0], "int8", 64, False)]
    check_attention(ops.kv8_dense_attn(q.to(DEV), cache), q, kk, vv, 128 ** -0.5, BF)
    idx = torch.arange(n, dtype=torch.int32, device=DEV)[None]
    check_attention(ops.kv8_sparse_attn(q.to(DEV), cache, idx=idx), q, kk, vv, 128 ** -0.5, BF)


@pytest.mark.parametrize("layout", ["head by head", "every other head", "token padded"])
def test_pages_in_other_layouts(layout):
    """Pools whose heads of a token do not lie back to back; rows behind the end hold codes that decode to NaN."""
    g = torch.Generator().manual_seed(37)
    pages, page, hkv, lens = 24, 32, 4, [333, 17, 250]
    if layout == "head by head":
        k, v = (torch.full((pages, hkv, page, 128), 0x7F, dtype=torch.uint8, device=DEV).transpose(1, 2) for _ in "kv")
    elif layout == "every other head":
        k, v = (torch.full((pages, page, 2 * hkv, 128), 0x7F, dtype=torch.uint8, device=DEV)[:, :, ::2] for _ in "kv")
    else:
        k, v = (torch.full((pages, page, hkv + 1, 128), 0x7F, dtype=torch.uint8, device=DEV)[:, :, :hkv] for _ in "kv")
    s = torch.full((2, pages, page // 16, hkv), float("nan"), device=DEV)
    order, table = torch.randperm(pages, generator=g).to(torch.int32).tolist(), torch.full((3, 11), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            table[b, i] = order.pop()
    table = table.to(DEV)
    cache = ops.KV8(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), s[0], s[1], 16, page_table=table)
    x, y = rows(g, 3, hkv, 333), rows(g, 3, hkv, 333)
    for b, n in enumerate(lens):
        one = ops.KV8(cache.k, cache.v, s[0], s[1], 16, page_table=table[b: b + 1])
        ops.kv8_append(one, x[b: b + 1, :, :n].to(DEV), y[b: b + 1, :, :n].to(DEV), 0, close=True)
    q = rows(g, 3, 4 * hkv)
    t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ks, vs = ([held(z[b, :, :n], "e4m3", 16, False) for b, n in enumerate(lens)] for z in (x, y))
    check_attention(ops.kv8_dense_attn(q.to(DEV), cache, seq_len=340, seq_lens=t), q, ks, vs, 128 ** -0.5, BF)
    out, raw = ops.kv8_dense_attn(q.to(DEV), cache, seq_len=340, seq_lens=t, selector="last", score_len=340, score_lens=t)
    check_attention(out, q, ks, vs, 128 ** -0.5, BF)
    for b, n in enumerate(lens):
        _, z, _, _, mass = ref.attention(q[b], ks[b], vs[b], 128 ** -0.5)
        assert bool(((raw[b, :n].cpu().double() - z.amax(0)).abs() <= ref.logit_error(mass).amax(0)).all())


def test_append_at_the_last_token_numbers():
    """A page table of almost 2^31 tokens whose last page alone lies in the pool: block numbers behind the end do not wrap."""
    g = torch.Generator().manual_seed(34)
    width = (1 << 24) - 1
    table = torch.full((1, width), -1, dtype=torch.int32, device=DEV)
    table[0, -1] = 2
    cache = ops.KV8.empty_paged(table, 4, 128, 1, "int8", 128, BF)
    x, y = rows(g, 1, 1, 128), rows(g, 1, 1, 128)
    room = width * 128
    ops.kv8_append(cache, x[:, :, :123].to(DEV), y[:, :, :123].to(DEV), torch.tensor([room - 128], dtype=torch.int32, device=DEV))
    ops.kv8_append(cache, x[:, :, 123:].to(DEV), y[:, :, 123:].to(DEV), torch.tensor([room - 5], dtype=torch.int32, device=DEV))
    for codes, scale, t in ((cache.k, cache.k_scale, x), (cache.v, cache.v_scale, y)):
        c, s = ref.quantise(t[0], "int8")
        assert torch.equal(codes[2, :, 0].cpu().double(), c[0].double()) and torch.equal(scale[2, 0].cpu().double(), s.double())
        assert not codes[[0, 1, 3]].view(torch.uint8).any() and not scale[[0, 1, 3]].any()
    # one row more than there is room for: left as it was
    before = [t.clone() for t in (cache.k, cache.k_scale, cache.open_k)]
    ops.kv8_append(cache, y[:, :, :6].to(DEV), x[:, :, :6].to(DEV), torch.tensor([room - 5], dtype=torch.int32, device=DEV))
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.k_scale, cache.open_k)))
    q = rows(g, 1, 4)
    idx = torch.arange(room - 128, room, dtype=torch.int32, device=DEV)[None]
    check_attention(ops.kv8_sparse_attn(q.to(DEV), cache, idx=idx), q, [held(x[0], "int8", 128, False)],
                    [held(y[0], "int8", 128, False)], 128 ** -0.5, BF)


def test_a_closed_short_block_is_read_without_the_open_buffers():
    g = torch.Generator().manual_seed(35)
    cache = ops.KV8.empty(1, 2, 128, "e4m3", 64, BF, DEV)
    x, y = rows(g, 1, 2, 100), rows(g, 1, 2, 100)
    ops.kv8_append(cache, x.to(DEV), y.to(DEV), 0, close=True)
    assert not cache.open_k.any() and not cache.open_v.any()
    closed = ops.KV8(cache.k, cache.v, cache.k_scale, cache.v_scale, 64)
    q = rows(g, 1, 8)
    check_attention(ops.kv8_dense_attn(q.to(DEV), closed, seq_len=100), q, [held(x[0], "e4m3", 64, False)],
                    [held(y[0], "e4m3", 64, False)], 128 ** -0.5, BF)


def test_single_entries_in_views_of_any_stride():
    """One request, one row: the strides of these dimensions say nothing."""
    g = torch.Generator().manual_seed(38)
    odd = lambda x: x.to(DEV).as_strided(x.shape, (131, 128, 3, 1))  # x: (1, heads, 1, 128)
    buf = torch.zeros(2 * 64 * 128, dtype=torch.uint8, device=DEV).view(torch.int8)
    codes = [buf.clone().as_strided((1, 2, 64, 128), (7, 64 * 128, 128, 1)) for _ in "kv"]
    s = torch.zeros((2, 1, 2, 4), device=DEV)
    cache = ops.KV8(codes[0], codes[1], s[0], s[1], 16)
    x, y, q = rows(g, 1, 2, 1), rows(g, 1, 2, 1), rows(g, 1, 8)
    ops.kv8_append(cache, odd(x), odd(y), 0, close=True)
    k, v = held(x[0], "int8", 16, False), held(y[0], "int8", 16, False)
    check_attention(ops.kv8_dense_attn(q.to(DEV), cache, seq_len=1), q, [k], [v], 128 ** -0.5, BF)
    out = ops.kv8_sparse_attn(q.to(DEV), cache, sel_len=1, tail_k=odd(y), tail_v=odd(x))
    check_attention(out, q, [torch.cat([k, y[0].double()], 1)], [torch.cat([v, x[0].double()], 1)], 128 ** -0.5, BF)


def test_a_single_kv_head_in_views_of_any_stride():
    """One kv head, in the new rows, the tail and the open buffers: the stride between heads says nothing."""
    g = torch.Generator().manual_seed(40)
    n, odd = 37, lambda x: x.to(DEV).as_strided(x.shape, (x.shape[2] * 128, 5, 128, 1))  # noqa: E731  x: (b, 1, n, 128)
    x, y, q, tk, tv = rows(g, 2, 1, n), rows(g, 2, 1, n), rows(g, 2, 4), rows(g, 2, 1, 9), rows(g, 2, 1, 9)
    whole = ops.KV8.empty(2, 1, 64, "int8", 16, BF, DEV)
    cache = ops.KV8(whole.k, whole.v, whole.k_scale, whole.v_scale, 16, odd(whole.open_k), odd(whole.open_v))
    ops.kv8_append(cache, odd(x), odd(y), 0)
    ks, vs = [held(r, "int8", 16, True) for r in x], [held(r, "int8", 16, True) for r in y]
    check_attention(ops.kv8_dense_attn(q.to(DEV), cache, seq_len=n), q, ks, vs, 128 ** -0.5, BF)
    idx = torch.arange(32, dtype=torch.int32, device=DEV).expand(2, -1).contiguous()
    out = ops.kv8_sparse_attn(q.to(DEV), cache, idx=idx, tail_k=odd(tk), tail_v=odd(tv))
    check_attention(out, q, [torch.cat([k[:, :32], t.double()], 1) for k, t in zip(ks, tk)],
                    [torch.cat([v[:, :32], t.double()], 1) for v, t in zip(vs, tv)], 128 ** -0.5, BF)


def test_scores_into_a_row_of_a_larger_tensor():
    """One request: the row's stride says nothing, whatever a view left there."""
    g = torch.Generator().manual_seed(36)
    cache, _, _ = make(g, "int8", BF, 32, 0, [700], 2)
    q = rows(g, 1, 8).to(DEV)
    want = ops.kv8_dense_attn(q, cache, seq_len=700, selector="last", score_len=600)[1]
    buf = torch.zeros(601, device=DEV)
    row = buf[:600].as_strided((1, 600), (1, 1))
    got = ops.kv8_dense_attn(q, cache, seq_len=700, selector="last", score_len=600, scores_out=row)[1]
    assert got.data_ptr() == buf.data_ptr() and torch.equal(got, want) and not buf[600:].any()


def test_front_end_refusals():
    cache = ops.KV8.empty(2, 2, 64, "int8", 32, BF, DEV)
    q = torch.zeros((2, 8, 128), dtype=BF, device=DEV)
    i = torch.zeros((2, 4), dtype=torch.int32, device=DEV)
    for bad in (lambda: ops.kv8_dense_attn(q.half(), cache), lambda: ops.kv8_dense_attn(q.float(), cache),
                lambda: ops.kv8_dense_attn(q[:1], cache), lambda: ops.kv8_dense_attn(q.cpu(), cache),
                lambda: ops.kv8_dense_attn(q, cache, select_k=3),
                lambda: ops.kv8_dense_attn(q, cache, seq_lens=torch.zeros(2, dtype=torch.int64, device=DEV)),
                lambda: ops.kv8_dense_attn(q, cache, seq_lens=torch.zeros(3, dtype=torch.int32, device=DEV)),
                lambda: ops.kv8_sparse_attn(q, cache, idx=i.long()), lambda: ops.kv8_sparse_attn(q, cache, idx=i[:1]),
                lambda: ops.kv8_sparse_attn(q, cache, idx=i, sel_len=5), lambda: ops.kv8_sparse_attn(q, cache, slots=i),
                lambda: ops.kv8_sparse_attn(q, cache, idx=i, tail_len=2), lambda: cache.slot_index(i),
                lambda: ops.kv8_append(cache, q[:, :2, None], q[:, :2, None].half(), 0),
                lambda: ops.kv8_append(cache, q[:, :3, None], q[:, :3, None], 0),
                lambda: ops.kv8_append(cache, q[:, :2, None], q[:, :2, None], 1 << 32),  # (no 32-bit number wraps round)
                lambda: ops.kv8_append(cache, q[:, :2, None], q[:, :2, None], -1),
                lambda: ops.kv8_dense_attn(q, cache, seq_len=(1 << 32) + 5),
                lambda: ops.kv8_dense_attn(q, cache, seq_len=5, selector="last", score_len=6),
                lambda: ops.kv8_sparse_attn(q, cache, sel_len=(1 << 32) + 5), lambda: ops.kv8_read(cache, BF, seq_len=(1 << 32) + 5),
                lambda: ops.kv8_append(cache, q[:, :2, None], q[:, :2, None], i[:, 0].long())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.kv8_dense_attn(q, cache, seq_len=65), lambda: ops.kv8_dense_attn(q, cache, seq_len=0),
                lambda: ops.kv8_append(cache, q[:, :2, None], q[:, :2, None], 64),
                lambda: ops.kv8_append(cache, q[:, :2, None], q[:, :2, None], 5, close=True)):
        with pytest.raises(Exception, match="invalid"):
            bad()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("top", [12.0, 18.0, 24.0])
def test_small_probabilities_of_16_bit_rows_keep_their_bits(dtype, top):
    """An 8-bit block takes almost all the weight and has V = 0: what is left of the output are the 16-bit rows, with
    probabilities around exp(-top), down to 2^-37: below half the smallest float16."""
    g = torch.Generator().manual_seed(39)
    k, v = torch.zeros(1, 1, 31, 128), torch.rand(1, 1, 31, 128, generator=g) * 4e4
    k[:, :, :16] = top * 128 ** -0.5
    v[:, :, :16] = 0
    k[:, :, 16:] = torch.randn(1, 1, 15, 128, generator=g) * 0.05
    k, v = k.to(dtype), v.to(dtype)
    cache = ops.KV8.empty(1, 1, 64, "int8", 16, dtype, DEV)
    ops.kv8_append(cache, k.to(DEV), v.to(DEV), 0)
    q = (1 + 0.1 * torch.randn(1, 4, 128, generator=g)).to(dtype)
    check_attention(ops.kv8_dense_attn(q.to(DEV), cache, seq_len=31), q, [held(k[0], "int8", 16, True)],
                    [held(v[0], "int8", 16, True)], 128 ** -0.5, dtype)
    closed = [held(x[0, :, :16], "int8", 16, True) for x in (k, v)]
    tk = (torch.randn(1, 1, 700, 128, generator=g) * 0.05).to(dtype)
    tv = (torch.rand(1, 1, 700, 128, generator=g) * 4e4).to(dtype)
    idx = torch.arange(16, dtype=torch.int32, device=DEV)[None]
    out = ops.kv8_sparse_attn(q.to(DEV), cache, idx=idx, tail_k=tk.to(DEV), tail_v=tv.to(DEV))
    check_attention(out, q, [torch.cat([closed[0], tk[0].double()], 1)], [torch.cat([closed[1], tv[0].double()], 1)],
                    128 ** -0.5, dtype)


@pytest.mark.parametrize("page", [0, 32])
def test_a_selection_and_the_open_rows_as_its_tail(page):
    """A filter layer scores the rows that are codes, a sparse layer reads those it selects and its own open rows as the
    tail: with every code selected, attention over the whole request."""
    g = torch.Generator().manual_seed(41)
    lens, hkv, block = [333, 31, 160, 7], 2, 16
    (one, k1, v1), (two, k2, v2) = (make(g, "e4m3", BF, block, page, lens, hkv) for _ in range(2))
    for codes in (one.k, one.v, two.k, two.v) if not page else ():
        for b, n in enumerate(lens):  # behind the last full block: whatever was there before
            codes.view(torch.uint8)[b, :, n // block * block:].fill_(0x66)
    q, q2 = rows(g, 4, 8), rows(g, 4, 8)
    t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    closed = t // block * block
    for k in (333, 20):
        out, scores, idx = ops.kv8_dense_attn(q.to(DEV), one, seq_lens=t, seq_len=333, selector="last", score_len=333,
                                              score_lens=closed, select_k=k)
        check_attention(out, q, k1, v1, 128 ** -0.5, BF)
        how = dict(slots=two.slot_index(idx)) if page else dict(idx=idx)
        got = ops.kv8_sparse_attn(q2.to(DEV), two, tail_k=two.open_k, tail_v=two.open_v, tail_lens=t - closed, **how)
        at = [torch.cat([i[i >= 0].long().cpu(), torch.arange(n // block * block, n)]) for i, n in zip(idx, lens)]
        assert all(a.numel() == min(k, n // block * block) + n % block for a, n in zip(at, lens))
        check_attention(got, q2, [x[:, a] for x, a in zip(k2, at)], [x[:, a] for x, a in zip(v2, at)], 128 ** -0.5, BF)


def test_a_selection_uses_scratch_of_its_own(monkeypatch):
    """None of the buffers that the 16-bit calls of a stream share: two captured graphs, replayed side by side, and eager
    calls next to them select what each selects alone."""
    g = torch.Generator().manual_seed(42)
    n, k = 40000, 2700
    cache, _, _ = make(g, "int8", BF, 64, 0, [n], 1)
    qs = [rows(g, 1, 4).to(DEV) for _ in range(3)]

    def call(q):
        return ops.kv8_dense_attn(q, cache, seq_len=n, selector="last", score_len=n, select_k=k)[2]

    with monkeypatch.context() as mp:
        mp.setattr(ops, "_workspace", lambda *a: pytest.fail("shared scratch"))
        want = [call(q) for q in qs]
    for q, idx in zip(qs, want):
        assert torch.equal(idx, ops.topk(ops.kv8_dense_attn(q, cache, seq_len=n, selector="last", score_len=n)[1], k))
    torch.cuda.synchronize()
    graphs, got = [], []
    for q in qs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(call(q))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for idx in got:
            idx.fill_(-1)
        for s, graph in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        eager = call(qs[2])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got + [eager], want))
