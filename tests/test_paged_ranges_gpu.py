"""The paged cache away from the middle of its range: queries, values and scores of unlike size, infinities and NaN, outputs of
another type, the forms that only large calls take; against the definitions in 64 bits."""
import math

import pytest
import torch

from oracle import paged_oracle as PO
from test_paged_gpu import DTYPES, FORMATS, _cuda, _decode, _empty, _full, _gen, _handle, _i32, _ops, _same, _table

pytestmark = pytest.mark.gpu


def _bounds(q, pool, fmt, table, lens, out_dtype, pages=None, one_part=False):
    """(o, lse, tolerance of o, tolerance of lse) from the definition.  Half a step of the output's type; of the weights,
    their rounding (one part of 11 bits where `one_part`, else two parts, 2^-15 at most) and twice the scores' error, as numerator
    and denominator both have it; sums of n terms in fp32.  A score is off by D fp32 steps of sum |q k| and by the query's
    conversion, 2^-23 of its largest channel in every one.  Weights below f16's normal numbers: n 2^-39 max |v|."""
    d, n = q.shape[-1], max(list(lens) + [1])
    o, lse, spread, size, vmax = PO.attention(q, pool, fmt, table, lens, pages)
    score = d * 2.0 ** -23 * size
    if fmt != "native":
        largest = max(PO.values(pool, "k", fmt, int(page), h, slice(None)).abs().sum(-1).max().item()
                      for page in table.unique() if 0 <= page < pool["k_pages"].shape[0] for h in range(pool["k_pages"].shape[1]))
        score = score + 2.0 ** -23 * q.double().abs().amax(-1) * largest / math.sqrt(d)
    weight = (2.0 ** -11 if one_part else 2.0 ** -15) + 2 * score + n * 2.0 ** -23
    tol = torch.finfo(out_dtype).eps / 2 * o.abs() + weight[..., None] * spread + n * 2.0 ** -39 * vmax[..., None] + torch.finfo(out_dtype).tiny
    return o, lse, tol, (score + n * 2.0 ** -23) * 1.4427 + 2.0 ** -22 * (1 + lse.abs())


def _within(got, want, tol):
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() / tol).max()


# ---- queries ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("ratio", [1, 16, 64, 256])
@pytest.mark.parametrize("d,n", [(128, 100), (64, 5)])
def test_decode_of_queries_with_a_large_channel(dtype, fmt, ratio, d, n):
    """One channel of every query is many times the others, and the keys have little in it: the other channels decide."""
    ref = _empty(fmt, dtype, 2, 2, 64, d)
    g = _gen(201)
    key, value = (torch.randn(1, n, 2, d, generator=g) for _ in range(2))
    key[..., 7] *= 1e-2 / ratio
    table = torch.arange(2, dtype=torch.int32)[None]
    PO.write(ref, fmt, key.to(dtype), value.to(dtype), table, [0], [n])
    q = torch.randn(1, 16, d, generator=g)
    q[..., 7] = 3.3 * ratio
    q = q.to(dtype).cuda()
    pool = _cuda(ref)
    out, lse = _decode(q, pool, dtype, table, [n])
    o, l, tol, tol_l = _bounds(q, pool, fmt, table, [n], dtype, one_part=dtype == torch.bfloat16)
    _within(lse, l, tol_l)
    _within(out, o, tol)


# ---- outputs of another type -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.float16), (torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("group,lens", [(4, [3, 1, 5]), (12, [700])])
def test_decode_is_as_exact_as_its_outputs_type(fmt, dtype, out_dtype, group, lens):
    """(Small queries: the scores' own error stays below the weights'.)"""
    d, hkv, ps = 128, 2, 32
    per = (max(lens) + ps - 1) // ps
    pool = _cuda(_full(fmt, dtype, per * len(lens), hkv, ps, d, 211))
    table = _table(len(lens), per, per * len(lens), 212)
    q = (torch.randn(len(lens), hkv * group, d, generator=_gen(213)) / 32).to(dtype).cuda()
    out, lse = _decode(q, pool, dtype, table, lens, out_dtype=out_dtype)
    o, l, tol, tol_l = _bounds(q, pool, fmt, table, lens, out_dtype, one_part=fmt != "native" and out_dtype == torch.bfloat16)
    assert out.dtype == out_dtype
    _within(lse, l, tol_l)
    _within(out, o, tol)


# ---- infinities ------------------------------------------------------------------------------------------------------
# (KV heads, lengths): clusters of CTAs; whole segments of one warp; segments cut between CTAs, joined by cuts and by rows
FORMS = [(2, [100, 33, 1, 700]), (8, [20, 700, 9, 64] * 10), (1, [30000]), (4, [9000, 20, 8193])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,lens", FORMS)
def test_infinite_values_of_keys_that_count(dtype, hkv, lens):
    """An infinite value makes its channel infinite, however small the key's weight and whatever the parts it is split into;
    two of unlike sign, or a NaN, make it NaN; every other channel is as without them."""
    d, ps, group = 128, 64, 3
    per = (max(lens) + ps - 1) // ps
    pages = per * len(lens)
    clean = _full("native", dtype, pages, hkv, ps, d, 221)
    table = _table(len(lens), per, pages, 222)
    q = (torch.randn(len(lens), hkv * group, d, generator=_gen(223)) * 6).to(dtype).cuda()
    host = {n: None if t is None else t.clone() for n, t in clean.items()}
    inf = float("inf")
    for i, n in enumerate(lens):
        for c, (key, x) in enumerate([(0, inf), (n - 1, -inf), (n // 2, float("nan")), (n // 3, inf), (n // 4, -inf), (n // 3, inf)]):
            page, row = int(table[i, key // ps]), key % ps
            host["v_pages"][page, :, row, 5 + c % 5], clean["v_pages"][page, :, row, 5 + c % 5] = x, 0.0
    for i, n in enumerate(lens):   # and one channel with both signs
        for key, x in ((0, inf), (n - 1, -inf if n > 1 else inf)):
            host["v_pages"][int(table[i, key // ps]), :, key % ps, 90], clean["v_pages"][int(table[i, key // ps]), :, key % ps, 90] = x, 0.0
    pool, dev = _cuda(host), table.cuda()
    out, lse = _decode(q, pool, dtype, table, lens)
    want = PO.attention(q, pool, "native", dev, lens)[0]
    o, l, tol, tol_l = _bounds(q, _cuda(clean), "native", dev, lens, dtype)
    odd = ~want.isfinite()
    assert odd.any(-1).all() and not odd.all(-1).any()
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isinf(), want.isinf()) and torch.equal(out[odd] > 0, want[odd] > 0)
    _within(out[~odd], o[~odd], tol[~odd])
    _within(lse, l, tol_l)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,lens", FORMS)
@pytest.mark.parametrize("first", [0, 1])
def test_scores_of_minus_infinity(dtype, hkv, lens, first):
    """Keys whose score is -inf have no weight beside others; where no other is left the softmax is NaN and the LSE -inf, unlike
    that of a sequence without keys."""
    d, ps, group = 64, 64, 3
    lens = lens + [0]
    per = (max(lens) + ps - 1) // ps
    pages = per * len(lens)
    host = _full("native", dtype, pages, hkv, ps, d, 231)
    table = _table(len(lens), per, pages, 232)
    q = torch.randn(len(lens), hkv * group, d, generator=_gen(233)).to(dtype)
    q[..., 3] = q[..., 3].abs() + 1
    host["k_pages"][..., 3] = -float("inf")            # of every key, but of every second sequence the last three are spared
    spared = list(range(first, len(lens) - 1, 2))
    for b in spared:
        for key in range(max(0, lens[b] - 3), lens[b]):
            host["k_pages"][int(table[b, key // ps]), :, key % ps, 3] = 0.5
    out, lse = _decode(q.cuda(), _cuda(host), dtype, table, lens)
    for b, n in enumerate(lens):
        if b in spared:
            assert out[b].isfinite().all() and lse[b].isfinite().all()
        else:
            assert (lse[b] == -float("inf")).all() and (out[b].isnan().all() if n else (out[b] == 0).all())
    if not spared:
        return
    few = {n: None if t is None else torch.zeros_like(t) for n, t in host.items()}   # the spared keys by themselves
    short = torch.arange(len(lens), dtype=torch.int32)[:, None]
    for b in spared:
        for i, key in enumerate(range(max(0, lens[b] - 3), lens[b])):
            for t in ("k_pages", "v_pages"):
                few[t][b, :, i] = host[t][int(table[b, key // ps]), :, key % ps]
    rows = torch.tensor(spared)
    counts = [min(3, lens[b]) for b in spared]
    o, l, tol, tol_l = _bounds(q[rows].cuda(), _cuda(few), "native", short[rows].cuda(), counts, dtype)
    _within(out[rows.cuda()], o, tol)
    _within(lse[rows.cuda()], l, tol_l)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_bounds_of_keys_that_are_nan(dtype, fmt):
    """NaN in one key, in every key of a page, in rows appended to a page begun before: the channel's bounds are NaN and the page
    is chosen last."""
    ops = _ops()
    d, ps, n = 64, 16, 16 * 12
    key = torch.randn(1, n, 1, d, generator=_gen(241)).to(dtype)
    key[0, 3 * ps + 5, 0, 9] = float("nan")
    key[0, 5 * ps:6 * ps, 0, 11] = float("nan")
    key[0, 8 * ps + 4, 0, 2] = float("nan")            # the page's first four rows come before
    key[0, 10 * ps + 1, 0, 30] = float("inf")
    value = torch.randn(1, n, 1, d, generator=_gen(242)).to(dtype)
    ref = _empty(fmt, dtype, 12, 1, ps, d)
    got = _cuda(ref)
    pool, table = _handle(got, dtype), torch.arange(12, dtype=torch.int32)[None]
    cut = 8 * ps + 4
    for a, b in ((0, cut), (cut, n)):
        ops.paged_write(pool, key[:, a:b].cuda(), value[:, a:b].cuda(), table.cuda(), _i32([a]))
        PO.write(ref, fmt, key[:, a:b], value[:, a:b], table, [a], [b - a])
    assert _same(got["k_bounds"], ref["k_bounds"]) and ref["k_bounds"].isnan().any(-1).any(-1).sum() == 3
    q = torch.randn(1, 1, 2, d, generator=_gen(243)).to(dtype).cuda()
    most = ops.paged_select(q, pool, table.cuda(), _i32([n]), 9, sink_pages=0, recent_pages=0)
    assert most[0, 0].tolist() == [i for i in range(12) if i not in (3, 5, 8)]


# ---- calls side by side ----------------------------------------------------------------------------------------------
def test_calls_of_several_threads_with_unlike_batches():
    """The calls of one kernel need unlike amounts of shared memory; each gets its own, whatever other threads call meanwhile.
    (Through the C ABI, which runs without the interpreter's lock.)"""
    import ctypes as C
    import threading
    from longcontext_sqattn_paddle_b200 import _lib as L
    ops = _ops()
    dtype, d, n = torch.bfloat16, 64, 4
    pool = _handle(_cuda(_full("int8", dtype, 8, 1, 16, d, 251)), dtype)
    calls, kept, want = [], [], []
    for b in [1024] + [20] * (n - 1):
        q = torch.randn(b, 1, 4, d, generator=_gen(252)).to(dtype).cuda()
        table, lens = torch.arange(8, dtype=torch.int32).expand(b, 8).contiguous().cuda(), _i32([1] * b)
        out = torch.empty_like(q)
        a = L.PagedDecodeArgs(pool=pool._address, q=L.Tensor(q.data_ptr(), 4 * d, d, 4 * d), o=L.Tensor(out.data_ptr(), 4 * d, d, 4 * d),
                              block_table=table.data_ptr(), table_stride=8, kv_lens=lens.data_ptr(), batch=b, num_q_heads=4, max_pages=8,
                              o_dtype=L.BF16)
        ws = torch.empty(L.lib.sqattn_paged_decode_workspace_bytes(C.byref(a)), dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        calls.append(a)
        kept.append((q, table, lens, out, ws, torch.cuda.Stream()))
        want.append(ops.paged_decode(q, pool, table, lens))
    refused = set()

    def run(i):
        stream = kept[i][5].cuda_stream
        torch.zeros(1, device="cuda")
        for _ in range(4000):
            if L.lib.sqattn_paged_decode(C.byref(calls[i]), stream):
                refused.add(L.lib.sqattn_last_error_string())

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not refused
    for k, w in zip(kept, want):
        assert torch.equal(k[3], w)


def test_the_first_call_of_a_host_thread():
    """A thread that has called nothing of CUDA before."""
    import ctypes as C
    import threading
    from longcontext_sqattn_paddle_b200 import _lib as L
    ops = _ops()
    dtype, d = torch.bfloat16, 64
    pool = _handle(_cuda(_full("int8", dtype, 8, 1, 16, d, 261)), dtype)
    q = torch.randn(1, 1, 4, d, generator=_gen(262)).to(dtype).cuda()
    table, lens, out = torch.arange(8, dtype=torch.int32)[None].cuda(), _i32([100]), torch.zeros_like(q)
    a = L.PagedDecodeArgs(pool=pool._address, q=L.Tensor(q.data_ptr(), 4 * d, d, 4 * d), o=L.Tensor(out.data_ptr(), 4 * d, d, 4 * d),
                          block_table=table.data_ptr(), table_stride=8, kv_lens=lens.data_ptr(), batch=1, num_q_heads=4, max_pages=8, o_dtype=L.BF16)
    ws = torch.empty(L.lib.sqattn_paged_decode_workspace_bytes(C.byref(a)), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    stream, said = torch.cuda.current_stream().cuda_stream, []
    thread = threading.Thread(target=lambda: said.append((L.lib.sqattn_paged_decode(C.byref(a), stream), L.lib.sqattn_last_error_string())))
    torch.cuda.synchronize()
    thread.start()
    thread.join()
    assert said[0][0] == L.OK, said
    assert torch.equal(out, ops.paged_decode(q, pool, table, lens))


# ---- forms of the decode ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("b,hkv", [(1, 14), (5, 3), (2, 8), (1, 17)])
@pytest.mark.parametrize("n", [100, 4609, 6657, 8193])
def test_decode_on_either_side_of_the_lines_between_its_forms(fmt, b, hkv, n):
    """As many segments as there are places for clusters, one more; lengths at which the form changes; bounds of the lengths too."""
    dtype, d, ps = torch.bfloat16, 128, 128
    per = (n + ps - 1) // ps
    pool = _cuda(_full(fmt, dtype, per + 2, hkv, ps, d, 271))
    table = torch.stack([torch.randperm(per + 2, generator=_gen(272 + i))[:per] for i in range(b)]).to(torch.int32).cuda()
    q = torch.randn(b, hkv, d, generator=_gen(273)).to(dtype).cuda()
    lens = [n - 7 * i for i in range(b)]
    o, l, tol, tol_l = _bounds(q, pool, fmt, table, lens, dtype, one_part=True)
    for bound in (0, n):
        out, lse = _decode(q, pool, dtype, table, lens, max_kv_len=bound)
        _within(lse, l, tol_l)
        _within(out, o, tol)


# ---- the cache -------------------------------------------------------------------------------------------------------
def _cache(**kw):
    from longcontext_sqattn_paddle_b200.cache_hub import PagedKVCache
    return PagedKVCache(0, 1, 3, 256, 2, 4, 64, torch.float16, **{**dict(kv_format="int8", page_size=16), **kw})


def _rows(b, n, seed):
    return torch.randn(b, n, 2, 64, generator=_gen(seed)).half().cuda()


def test_an_ended_sequence_takes_no_part_in_steps():
    """It takes no pages, its length stays 0 and its attention is zeros, while the others go on; a prefill begins another in its
    place."""
    kc = _cache(num_pages=16)
    for b, n in ((0, 40), (1, 100), (2, 48)):           # 3, 7 and 3 of the 16 pages
        kc.prefill_update_kv_cache(None, _rows(1, n, b), _rows(1, n, 10 + b), 0, b)
    kc.end(1)
    q = torch.randn(3, 1, 4, 64, generator=_gen(281)).half().cuda()
    for t in range(70):                                 # the two others need 13 pages in the end
        kc.decode_update_kv_cache(_rows(3, 1, 100 + t), _rows(3, 1, 200 + t), 0)
        out = kc.decode_attention(q, 0)
        assert (out[1] == 0).all() and (out[0] != 0).any() and (out[2] != 0).any()
    assert kc.valid_length.tolist() == kc.valid_length_host == [110, 0, 118]
    assert kc.allocator.pages[1] == [] and (kc.block_table[1] == -1).all() and len(kc.allocator.free) == 16 - 7 - 8
    key = kc.read(0, 0, 40, 70)[0][0].float()
    want = torch.cat([_rows(3, 1, 100 + t)[0] for t in range(70)]).float()
    assert ((key - want).abs() <= want.abs().amax(-1, keepdim=True) / 100).all()
    kc.prefill_update_kv_cache(None, _rows(1, 10, 5), _rows(1, 10, 6), 0, 1)
    kc.decode_update_kv_cache(_rows(3, 1, 7), _rows(3, 1, 8), 0)
    assert kc.valid_length.tolist() == kc.valid_length_host == [111, 11, 119]
    assert (kc.decode_attention(q, 0)[1] != 0).any()


def test_a_sequence_ends_between_captured_steps():
    from test_paged_cache_gpu import _model, _prefill
    m = _model(dict(kv_format="int8", page_size=16))
    ids = torch.randint(0, 2048, (2, 90), generator=_gen(282)).cuda()
    _prefill(m, ids, 40)
    m.capture_decode_step(2)
    tok = torch.full((2, 1), 5, device="cuda")
    m.decode_forward_graph(tok)
    m.kv_cache.end(0)
    for _ in range(3):
        logits = m.decode_forward_graph(tok)
    assert logits.isfinite().all()
    kc = m.kv_cache
    assert kc.valid_length.tolist() == kc.valid_length_host == [0, 94] and kc.context == 94
    assert kc.allocator.pages[0] == []


def test_captured_steps_take_pages_as_they_go():
    """A pool smaller than all sequences at their longest; a sequence that is prefilled anew after the capture; a pool that runs out
    refuses the step before it has run."""
    from test_paged_cache_gpu import _model, _prefill
    options = dict(kv_format="int8", page_size=16, num_pages=12)
    ids = torch.randint(0, 2048, (2, 60), generator=_gen(291)).cuda()
    eager, graphed = _model(options), _model(options)
    _prefill(eager, ids, 200), _prefill(graphed, ids, 200)      # 17 pages a sequence at the longest
    graphed.capture_decode_step(2)
    assert len(graphed.kv_cache.allocator.free) == 4
    tok = torch.full((2, 1), 5, device="cuda")
    for t in range(36):                                         # to 96 tokens, all twelve pages
        a, b = eager.decode_forward(tok), graphed.decode_forward_graph(tok)
        assert (a - b).abs().max().item() < 0.03 * a.abs().max().item()
        tok = torch.full_like(tok, 7 + 3 * t)
    assert graphed.kv_cache.allocator.free == [] and graphed.kv_cache.valid_length.tolist() == [96, 96]
    with pytest.raises(RuntimeError, match="exhausted"):
        graphed.decode_forward_graph(tok)
    kc = graphed.kv_cache
    assert kc.valid_length.tolist() == kc.valid_length_host == [96, 96]
    kc.end(0)
    g = _gen(292)
    k, v = (torch.randn(1, 14, 2, 128, generator=g).bfloat16().cuda() for _ in range(2))
    for layer in range(2):
        kc.prefill_update_kv_cache(None, k, v, layer, 0)
    for _ in range(5):                                          # the third step's token needs a second page
        graphed.decode_forward_graph(tok)
    assert kc.valid_length.tolist() == kc.valid_length_host == [19, 101] and len(kc.allocator.pages[0]) == 2
    key = kc.read(1, 0)[0][0].float()
    assert ((key[:14] - k[0].float()).abs() <= k[0].float().abs().amax(-1, keepdim=True) / 100).all() and (key[14:].abs().amax(-1) > 0).all()


def test_known_workspace_sizes_do_not_pile_up():
    """Neither over the steps of a cache nor with a bound or a table that changes in every call."""
    ops = _ops()
    kc = _cache(num_pages=48, kv_format="native")
    for b in range(3):
        kc.prefill_update_kv_cache(None, _rows(1, 20, b), _rows(1, 20, b), 0, b)
    q = torch.randn(3, 1, 4, 64, generator=_gen(301)).half().cuda()
    for t in range(100):
        kc.decode_update_kv_cache(_rows(3, 1, 0), _rows(3, 1, 1), 0)
        kc.decode_attention(q, 0)
    assert len(kc.pools[0]._scratch) == 1
    want = kc.decode_attention(q, 0)
    for bound in range(121, 400):
        assert torch.equal(ops.paged_decode(q, kc.pools[0], kc.block_table, kc.after, max_kv_len=bound), want)
    assert len(kc.pools[0]._scratch) <= 64


def _stretch(fmt, dtype, hkv, group, lens, ps, seed, d=128, distinct=None, pages=None):
    """Against the definition, over a pool of ``distinct`` pages that sequences share."""
    per = (max(lens) + ps - 1) // ps
    distinct = distinct or per * len(lens)
    pool = _cuda(_full(fmt, dtype, distinct, hkv, ps, d, seed))
    table = torch.randint(0, distinct, (len(lens), per), generator=_gen(seed + 1), dtype=torch.int32).cuda()
    q = torch.randn(len(lens), hkv * group, d, generator=_gen(seed + 2)).to(dtype).cuda()
    o, l, tol, tol_l = _bounds(q, pool, fmt, table, lens, dtype, pages=pages, one_part=fmt != "native" and dtype == torch.bfloat16)
    out, lse = _decode(q, pool, dtype, table, lens, **({} if pages is None else {"pages": _i32(pages)}))
    empty = l == -float("inf")                               # no keys: no tokens, or none of the listed pages is held
    assert (out[empty] == 0).all() and (lse[empty] == -float("inf")).all()
    _within(lse[~empty], l[~empty], tol_l[~empty])
    _within(out, o, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hkv,group,ps,lens", [
    (1, 7, 64, [20001]),                                     # all CTAs on one segment, their parts joined by rows
    (1, 16, 128, [12000]),
    (4, 12, 32, [9001, 8200]),
    (3, 8, 16, [30000, 1, 0, 8193, 77]),                     # the same beside segments that lie in one warp
])
def test_stretches_of_few_long_sequences(dtype, fmt, hkv, group, ps, lens):
    _stretch(fmt, dtype, hkv, group, lens, ps, 311)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hkv,group,ps,lens", [
    (8, 4, 32, [3000, 10, 0, 700, 64, 1500, 33, 2049] * 3),  # 192 segments: several tiles a warp, whole ones and cut ones, joined by cuts
    (8, 16, 64, [900, 2500, 1, 4000] * 5),
    (1, 9, 16, [1200 + 37 * i for i in range(160)]),
])
def test_stretches_of_many_sequences(dtype, fmt, hkv, group, ps, lens):
    _stretch(fmt, dtype, hkv, group, lens, ps, 321, distinct=300)


@pytest.mark.parametrize("fmt,n", [("native", 170001), ("int8", 170001), ("int4", 500003)])
def test_stretches_of_more_tiles_than_a_warp_looks_up_at_once(fmt, n):
    """More than 32 tiles a warp."""
    _stretch(fmt, torch.bfloat16, 8, 4, [n], 128, 331, distinct=40)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("group", [5, 16])
def test_stretches_over_listed_pages(fmt, group):
    """Lists of 20 pages for 24 segments, holes and pages past the end among them."""
    g = _gen(341)
    lens = [4000, 90, 2222]
    pages = [[torch.where(torch.rand(20, generator=g) < 0.2, -1, torch.randperm(70, generator=g)[:20]).tolist() for _ in range(8)] for _ in lens]
    _stretch(fmt, torch.float16, 8, group, lens, 64, 342, pages=pages)


# ---- selection over many pages ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("held,budget,sink,recent,distinct", [
    (16384, 100, 1, 1, 16384),                               # as many as stay in registers
    (16385, 100, 1, 1, 16385),                               # one more: the keys are read again in every round
    (40000, 3000, 4, 7, 40000),
    (40000, 17000, 1, 2, 3),                                 # pages of three kinds: the budget ends among equal ones, past the first 16384
    (40000, 9, 4, 5, 40000),                                 # nothing left to choose
    (131072, 1, 0, 0, 1),                                    # the most pages there may be, all alike
    (131072, 70000, 0, 1, 90000),
])
def test_select_over_many_pages(held, budget, sink, recent, distinct):
    ops = _ops()
    dtype, d, hkv, group = torch.bfloat16, 64, 2, 3
    g = _gen(351)
    bounds = torch.randn(distinct, hkv, 2, d, generator=g).to(dtype).sort(dim=2).values
    pool = _empty("int8", dtype, 1, hkv, 16, d)
    pool = {n: t.expand(distinct, *t.shape[1:]).contiguous() for n, t in pool.items()}
    pool["k_bounds"] = bounds
    table = torch.cat((torch.randperm(distinct, generator=g), torch.randint(0, distinct, (held - distinct,), generator=g))).to(torch.int32)[None]
    if held > 20000 and distinct > 3:
        table[0, 16390], table[0, 5] = -1, distinct          # pages that are not there
    q = torch.randn(1, hkv * group, d, generator=g).to(dtype)
    got = ops.paged_select(q[:, None].cuda(), _handle(_cuda(pool), dtype), table.cuda(), _i32([held * 16 - 3]), budget, sink_pages=sink, recent_pages=recent)
    u = q.view(hkv, group, d).double().sum(1)
    at = torch.arange(held)
    there = (table[0] >= 0) & (table[0] < distinct)
    for h in range(hkv):
        low, high = bounds[table[0].long().clamp(0, distinct - 1), h].double().unbind(1)
        score = torch.where(there, torch.maximum(u[h] * low, u[h] * high).sum(-1), -float("inf"))
        score[(at < sink) | (at >= held - recent)] = float("inf")
        best = torch.sort(score, descending=True, stable=True).indices[:budget].sort().values
        assert got[0, h].tolist() == best.tolist()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("group,lens", [(8, [500]), (3, [20, 9000])])
def test_decode_of_keys_near_the_types_range(fmt, group, lens):
    """bf16 keys of up to 2^119, scores of ordinary size."""
    dtype, d, hkv, ps = torch.bfloat16, 128, 1, 64
    per = (max(lens) + ps - 1) // ps
    g = _gen(361)
    table = torch.arange(per * len(lens), dtype=torch.int32).view(len(lens), per)
    got = _cuda(_empty(fmt, dtype, per * len(lens), hkv, ps, d))
    pool = _handle(got, dtype)
    key, value = torch.randn(len(lens), max(lens), hkv, d, generator=g) * 2.0 ** 117, torch.randn(len(lens), max(lens), hkv, d, generator=g)
    _ops().paged_write(pool, key.to(dtype).cuda(), value.to(dtype).cuda(), table.cuda(), _i32([0] * len(lens)))
    q = (torch.randn(len(lens), group, d, generator=g) * 2.0 ** -97).to(dtype).cuda()
    scale = 2.0 ** -23
    out, lse = _decode(q, got, dtype, table, lens, sm_scale=scale)
    o, l, spread, size, vmax = PO.attention(q, got, fmt, table.cuda(), lens, sm_scale=scale)
    n = max(lens)
    score = d * 2.0 ** -23 * size + (0.0 if fmt == "native" else 2.0 ** -23 * q.double().abs().amax(-1) * 2.0 ** 120 * d * scale)   # (as in _bounds)
    tol = 2.0 ** -8 * o.abs() + (2.0 ** -11 + 2 * score + n * 2.0 ** -23)[..., None] * spread + n * 2.0 ** -39 * vmax[..., None]
    assert 1 < size.max() < 100
    _within(lse, l, (score + n * 2.0 ** -23) * 1.4427 + 2.0 ** -22 * (1 + l.abs()))
    _within(out, o, tol)
