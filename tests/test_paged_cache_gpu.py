"""The paged cache behind the layer loops: decode steps of the small model over pages against the same steps over the
contiguous cache, eager and captured, over all pages and over selected ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(paged_kv, seed=3, layers=2, dtype=torch.bfloat16):
    from longcontext_sqattn_paddle_b200.model_hub import DecoderConfig, RandomInitDecoder
    cfg = DecoderConfig(num_hidden_layers=layers, hidden_size=512, num_attention_heads=4, num_key_value_heads=2,
                        intermediate_size=1024, vocab_size=2048, model_size_b=0)
    return RandomInitDecoder(cfg, max_length=1024, dtype=dtype, device="cuda:0", seed=seed, paged_kv=paged_kv)


def _prefill(m, ids, new, valid_start=None):
    m.batch_size, m.max_new_length = ids.shape[0], new
    m.init_kv_cache(ids.shape[1], (0,) * ids.shape[0] if valid_start is None else valid_start)
    logits = m.prefill_forward(ids)
    m.move()
    return logits


def _steps(m, ids, n, graph=False):
    if graph:
        m.capture_decode_step(ids.shape[0])
    tok, out = torch.full((ids.shape[0], 1), 5, device="cuda"), []
    for t in range(n):
        logits = (m.decode_forward_graph(tok) if graph else m.decode_forward(tok)).clone()
        out.append(logits)
        tok = torch.full_like(tok, 7 + 3 * t)
    return out


# The 16-bit hidden states carry their own rounding (2^-9 a tensor, a dozen tensors a layer) through both models alike where the
# attention agrees; 8-bit rows add 1/254 of a row's largest, 4-bit rows 1/14, to what each key and value contributes.
@pytest.mark.parametrize("fmt,page,tol", [("native", 16, 0.03), ("native", 64, 0.03), ("int8", 32, 0.05), ("int4", 128, 0.5)])
def test_decode_over_pages_follows_the_contiguous_cache(fmt, page, tol):
    g = torch.Generator().manual_seed(21)
    ids = torch.randint(0, 2048, (2, 200), generator=g).cuda()
    ref, got = _model(None), _model(dict(kv_format=fmt, page_size=page))
    a, b = _prefill(ref, ids, 8), _prefill(got, ids, 8)
    assert torch.equal(a, b)       # the prompt's attention does not read the cache
    for x, y in zip(_steps(ref, ids, 6), _steps(got, ids, 6)):
        assert (x - y).abs().max().item() < tol * x.abs().max().item()
    assert got.kv_cache.valid_length_host == ref.kv_cache.valid_length_host == [206, 206]
    assert got.kv_cache.valid_length.tolist() == [206, 206] and got.kv_cache.context == ref.kv_cache.context
    key, value = got.kv_cache.read(1, 1)
    want = ref.kv_cache.key_cache[1][1, :206].float()
    step = {"native": 2.0 ** -6, "int8": 1 / 100, "int4": 1 / 5}[fmt]
    assert key.shape == (1, 206, 2, 128) and value.shape == key.shape
    assert ((key[0, :200].float() - want[:200]).abs() <= step * want[:200].abs().amax(-1, keepdim=True) + 1e-6).all()


def test_left_padded_prompts_keep_their_valid_part():
    """(The dense prefill operator takes no padded prompts, so the caches are called directly.)"""
    from longcontext_sqattn_paddle_b200.cache_hub import PagedKVCache, flash_attn_cache
    args = ((0, 37), 1, 2, 200, 2, 4, 128, torch.bfloat16)
    ref, got = flash_attn_cache(*args, force_host=False), PagedKVCache(*args, kv_format="native", page_size=16)
    g = torch.Generator().manual_seed(22)
    for b in range(2):
        k, v = (torch.randn(1, 150, 2, 128, generator=g).bfloat16().cuda() for _ in range(2))
        for x, y in zip(ref.prefill_update_kv_cache(None, k, v, 0, b), got.prefill_update_kv_cache(None, k, v, 0, b)):
            assert torch.equal(x, y)
    ref.sync(0)
    assert got.valid_length_host == [150, 113] and got.context == ref.context
    for b, n in ((0, 150), (1, 113)):
        key, value = got.read(0, b)
        assert torch.equal(key[0], ref.key_cache[0][b, :n]) and torch.equal(value[0], ref.value_cache[0][b, :n])


@pytest.mark.parametrize("options", [dict(kv_format="int8", page_size=16), dict(kv_format="int8", page_size=16, select_pages=4)])
def test_captured_steps_are_the_eager_ones(options):
    g = torch.Generator().manual_seed(23)
    ids = torch.randint(0, 2048, (1, 90), generator=g).cuda()
    eager, graphed = _model(options), _model(options)
    _prefill(eager, ids, 40), _prefill(graphed, ids, 40)
    for x, y in zip(_steps(eager, ids, 30), _steps(graphed, ids, 30, graph=True)):
        assert (x - y).abs().max().item() < 0.03 * x.abs().max().item()     # other key ranges in the captured launch
    assert torch.equal(eager.kv_cache.valid_length, graphed.kv_cache.valid_length)
    assert graphed.kv_cache.context == eager.kv_cache.context


def test_selecting_every_page_is_attending_to_all():
    g = torch.Generator().manual_seed(24)
    ids = torch.randint(0, 2048, (1, 130), generator=g).cuda()
    every, some = _model(dict(kv_format="native", page_size=16)), _model(dict(kv_format="native", page_size=16, select_pages=9))
    _prefill(every, ids, 4), _prefill(some, ids, 4)
    for x, y in zip(_steps(every, ids, 4), _steps(some, ids, 4)):
        assert (x - y).abs().max().item() < 0.03 * x.abs().max().item()


def test_generate_with_pages():
    ids = torch.randint(0, 2048, (1, 100), generator=torch.Generator().manual_seed(25)).cuda()
    out = _model(dict(kv_format="int8")).generate("SQAttn", ids, None, 5)
    assert len(out) == 1 and len(out[0]) == 5


def test_pages_come_back_and_the_pool_can_run_out():
    from longcontext_sqattn_paddle_b200.cache_hub import PagedKVCache
    kc = PagedKVCache(0, 1, 3, 256, 2, 4, 64, torch.float16, kv_format="int4", page_size=16, num_pages=20)
    rows = lambda n: torch.randn(1, n, 2, 64, device="cuda").half()  # noqa: E731
    for b, n in ((0, 100), (1, 200)):
        kc.prefill_update_kv_cache(None, rows(n), rows(n), 0, b)
    with pytest.raises(RuntimeError, match="exhausted"):
        kc.prefill_update_kv_cache(None, rows(17), rows(17), 0, 2)
    kept = kc.read(0, 0)[0].clone()
    kc.release(1)
    assert kc.valid_length.tolist() == [100, 0, 0] and (kc.block_table[1] == -1).all()
    kc.prefill_update_kv_cache(None, rows(180), rows(180), 0, 2)
    assert torch.equal(kc.read(0, 0)[0], kept)               # the others' pages are theirs
    with pytest.raises(ValueError, match="the block table has"):
        kc.reserve(0, 300)
    out = kc.decode_update_kv_cache(rows(1).expand(3, -1, -1, -1), rows(1).expand(3, -1, -1, -1), 0)
    assert out is None and kc.valid_length.tolist() == [101, 1, 181]
    o = kc.decode_attention(torch.randn(3, 1, 4, 64, device="cuda").half(), 0)
    assert o.shape == (3, 1, 4, 64) and o.isfinite().all()
