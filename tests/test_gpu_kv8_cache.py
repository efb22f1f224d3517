"""The multi-stage cache and the model with K and V in 8 bits: what they attend to is what update() says they hold, and the
static (captured) path equals the eager one."""
import pytest
import torch

import kv8_reference as ref
from omnikv_amd import ops
from omnikv_amd.cache import OmniKVLazyCache, OmniKVMultiStageCache, WOPackCache
from omnikv_amd.config import OmniKVConfig
from omnikv_amd.model import LlamaShape, OmniKVMulLM

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HQ, HKV, D = 8, 2, 128
SHAPE = LlamaShape(hidden_size=256, intermediate_size=512, vocab_size=1000, num_hidden_layers=7, num_attention_heads=HQ,
                   num_key_value_heads=HKV, head_dim=D)


def rows(g, n, dtype, heads=HKV):
    return torch.randn((1, heads, n, D), generator=g).to(dtype).to(DEV)


def config(**kw):
    return OmniKVConfig(model_cls="multi", cache_cls="multi", do_select_layers="1,4", num_wait_load_layers=1, real_offload=False,
                        dense_more=True, num_of_selected_tokens=0.1, selector_cls="softmax_before_last", **kw)


def within(out, q, k, v, dtype):
    """An attention output against 64 bits over the 16-bit tensors k, v that update() handed out.  update() rounds a stored
    value (code times scale) to 16 bits where the kernel does not: half a step of every K and V element on top."""
    want, _, _, spread, mass = ref.attention(q[0, :, 0].cpu(), k[0].cpu(), v[0].cpu(), D ** -0.5)
    half = torch.finfo(dtype).eps / 2
    extra = (torch.expm1(2 * half * mass.amax()) * 2 + half) * spread
    assert bool(((out[0].cpu().double() - want).abs() <= ref.output_bound(want, spread, mass, dtype) + extra).all())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cls", [OmniKVMultiStageCache, WOPackCache, OmniKVLazyCache])
@pytest.mark.parametrize("n, block", [(300, 64), (256, 32), (17, 16)])
def test_attend_equals_attention_over_what_update_returns(fmt, dtype, cls, n, block):
    g = torch.Generator().manual_seed(1)
    kw = {"skip_threshold": 2.0} if cls is OmniKVLazyCache else {}
    cache = cls([0, 1, 4, 7], 7, 1, False, max_new_tokens=8, kv_format=fmt, kv_block=block, **kw)
    twin = cls([0, 1, 4, 7], 7, 1, False, max_new_tokens=8, kv_format=fmt, kv_block=block, **kw)
    sparse = {i for i, s in cache.layer_state.items() if s[0]}
    assert sparse == {3, 6}
    for i in range(7):
        k, v = rows(g, n, dtype), rows(g, n, dtype)
        for c in (cache, twin):
            pk, pv = c.update(k, v, i)
        if i in sparse:
            assert torch.equal(pk, k) and torch.equal(pv, v)
        else:  # whole blocks as stored, the rest as it came
            assert torch.equal(pk[:, :, n // block * block:], k[:, :, n // block * block:]) and pk.shape == k.shape
    for step in range(20):  # past max_new_tokens: the stores grow
        for c in (cache, twin):
            c.stage = "decoding"
        for i in range(7):
            k, v, q = rows(g, 1, dtype), rows(g, 1, dtype), rows(g, 1, dtype, HQ)
            cache.append(k, v, i)
            if i in (1, 4):
                out, idx = cache.attend_and_select(q, i, max(1, n // 10), n, "softmax_before_last")
                twin.set_idx_on_gpu(idx, i)
            else:
                out = cache.attend(q, i)
            kk, vv = twin.update(k, v, i)
            within(out, q, kk, vv, dtype)
    assert cache.get_seq_length() == n + 20


def test_refusals():
    with pytest.raises(NotImplementedError, match="host tier"):
        OmniKVMultiStageCache([0, 1, 4, 7], 7, 1, True, kv_format="int8")
    with pytest.raises(ValueError, match="kv_format"):
        OmniKVMultiStageCache([0, 1, 4, 7], 7, 1, False, kv_format="fp4")
    g = torch.Generator().manual_seed(2)
    cache = OmniKVMultiStageCache([0, 1, 4, 7], 7, 1, False, kv_format="int8")
    x = rows(g, 40, torch.bfloat16)
    for i in range(7):
        cache.append(x, x, i)
    with pytest.raises(NotImplementedError, match="16-bit keys"):
        cache.attend_and_select_window(rows(g, 1, torch.bfloat16, HQ), rows(g, 4, torch.bfloat16, HQ), 1, 4, 40, "uniform")
    with pytest.raises(NotImplementedError, match="one prefill"):
        cache.append(x, x, 3)
    with pytest.raises(ValueError):
        cache.append(x.float(), x.float(), 0)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_model_static_decode_and_graph_replays_equal_eager_static_steps(fmt):
    torch.manual_seed(0)
    torch.set_default_dtype(torch.bfloat16)
    try:
        with torch.device(DEV):
            lm = OmniKVMulLM(SHAPE, config(kv_format=fmt, kv_block=16))
    finally:
        torch.set_default_dtype(torch.float32)
    lm.init_weights(seed=3, std=0.08)
    ids = torch.randint(0, SHAPE.vocab_size, (1, 333), generator=torch.Generator().manual_seed(1)).to(DEV)
    steps, warm = 40, 2
    logits, eager = lm.forward(ids, None, max_new_tokens=steps + 8)
    tok = logits[:, -1].argmax(-1, keepdim=True)
    _, cache = lm.forward(ids, None, max_new_tokens=steps + 8)
    graph, token, glogits = lm.capture_decode(cache, tok, warmup=warm)
    eager.enable_static_decode()
    for _ in range(warm):
        out, _ = lm.forward(tok, eager)
        tok = out[:, -1].argmax(-1, keepdim=True)
    assert torch.equal(token, tok)
    for i in range(steps):  # blocks of 16 fill on the way
        out, _ = lm.forward(tok, eager)
        tok = out[:, -1].argmax(-1, keepdim=True)
        graph.replay()
        assert torch.equal(glogits, out) and torch.equal(token, tok), i
        if i % 9 == 0:
            torch.cuda.synchronize()
    # the ordinary eager path: the same model, lengths on the host; bf16 activations rounded at other places
    logits, plain = lm.forward(ids, None, max_new_tokens=steps + 8)
    first = logits[:, -1].argmax(-1, keepdim=True)
    a, _ = lm.forward(first, plain)
    _, again = lm.forward(ids, None, max_new_tokens=steps + 8)
    again.enable_static_decode()
    b, _ = lm.forward(first, again)
    assert float((a - b).abs().max()) <= 2 ** -6 * float(a.abs().max())


def test_selection_tracing_is_refused():
    from omnikv_amd import trace

    with torch.device(DEV):
        lm = OmniKVMulLM(SHAPE, config(kv_format="int8")).to(torch.bfloat16)
    ids = torch.zeros((1, 40), dtype=torch.int64, device=DEV)
    _, cache = lm.forward(ids, None)
    trace.set_tracer(trace.SelectedIndexTracer(desc="x", num_selected_tokens=0.1))
    try:
        with pytest.raises(NotImplementedError, match="16-bit keys"):
            lm.forward(ids[:, :1], cache)
    finally:
        trace.set_tracer(None)


def test_model_generates_with_an_8_bit_cache():
    """16-bit and 8-bit caches side by side: same first token (the prefill attends in 16 bits), close logits after it."""
    lms = []
    for kw in ({}, {"kv_format": "int8", "kv_block": 16}):
        torch.set_default_dtype(torch.bfloat16)
        try:
            with torch.device(DEV):
                lm = OmniKVMulLM(SHAPE, config(**kw))
        finally:
            torch.set_default_dtype(torch.float32)
        lms.append(lm.init_weights(seed=5, std=0.05))
    ids = torch.randint(0, SHAPE.vocab_size, (1, 400), generator=torch.Generator().manual_seed(4)).to(DEV)
    got = [lm.generate_greedy(ids, 12) for lm in lms]
    assert torch.equal(got[0][0][:, :1], got[1][0][:, :1]) and torch.equal(got[0][1][0], got[1][1][0])
    assert got[1][0].shape == (1, 12) and all(bool(l.isfinite().all()) for l in got[1][1])


def test_a_prompt_too_short_for_a_selection():
    """A ratio that selects no row of a short prompt: the sparse layers attend to the generated tokens alone."""
    g = torch.Generator().manual_seed(7)
    cache, twin = (OmniKVMultiStageCache([0, 1, 4, 7], 7, 1, False, max_new_tokens=8, kv_format="int8", kv_block=16) for _ in "ab")
    for i in range(7):
        k, v = rows(g, 5, torch.bfloat16), rows(g, 5, torch.bfloat16)
        for c in (cache, twin):
            c.append(k, v, i)
    for step in range(12):
        cache.stage = twin.stage = "decoding"
        for i in range(7):
            k, v, q = rows(g, 1, torch.bfloat16), rows(g, 1, torch.bfloat16), rows(g, 1, torch.bfloat16, HQ)
            cache.append(k, v, i)
            if i in (1, 4):
                out, idx = cache.attend_and_select(q, i, 0, 5, "softmax_before_last")
                assert idx.shape == (1, 0)
                twin.set_idx_on_gpu(idx, i)
            else:
                out = cache.attend(q, i)
            kk, vv = twin.update(k, v, i)
            assert kk.shape[2] == (step + 1 if i in (3, 6) else 5 + step + 1)
            within(out, q, kk, vv, torch.bfloat16)
