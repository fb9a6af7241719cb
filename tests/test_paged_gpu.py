"""The paged key/value cache: writing (quantising), reading back, decoding over all pages and over selected ones, against
the definitions in 64 bits."""
import math

import pytest
import torch

from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu

FORMATS = ["native", "int8", "int4"]
DTYPES = [torch.bfloat16, torch.float16]


def _ops():
    from longcontext_sqattn_paddle_b200 import ops
    return ops


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _empty(fmt, dtype, pages, hkv, ps, d):
    kind = {"native": dtype, "int8": torch.int8, "int4": torch.uint8}[fmt]
    row = d // 2 if fmt == "int4" else d
    pool = {"k_pages": torch.zeros(pages, hkv, ps, row, dtype=kind), "v_pages": torch.zeros(pages, hkv, ps, row, dtype=kind)}
    for n in ("k_scale", "v_scale"):
        pool[n] = None if fmt == "native" else torch.zeros(pages, hkv, ps)
    pool["k_bounds"] = torch.zeros(pages, hkv, 2, d, dtype=dtype)
    return pool


def _full(fmt, dtype, pages, hkv, ps, d, seed):
    """A pool whose every row is written."""
    g = _gen(seed)
    pool = _empty(fmt, dtype, pages, hkv, ps, d)
    for t in "kv":
        x = torch.randn(pages, hkv, ps, d, generator=g).to(dtype)
        if t == "k":
            pool["k_bounds"][:, :, 0], pool["k_bounds"][:, :, 1] = x.amin(2), x.amax(2)
        if fmt == "native":
            pool[t + "_pages"] = x
        else:
            codes, scale = PO.quantise(x, fmt)
            pool[t + "_pages"] = PO.pack4(codes) if fmt == "int4" else codes.to(torch.int8)
            pool[t + "_scale"] = scale
    return pool


def _cuda(pool):
    return {n: None if t is None else t.cuda() for n, t in pool.items()}


def _handle(pool, dtype):
    return _ops().PagedPool(dtype=dtype, **pool)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def _same(a, b):
    return torch.equal(torch.nan_to_num(a.float().cpu(), nan=1e30), torch.nan_to_num(b.float().cpu(), nan=1e30))


def _table(batch, per, pages, seed):
    return torch.randperm(pages, generator=_gen(seed))[:batch * per].to(torch.int32).view(batch, per)


# ---- write and read --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,hkv,ps,n,starts,counts", [
    (128, 4, 64, 1, [0, 63, 64, 100], None),                 # single tokens: a page's first and last row, the next page's first
    (64, 1, 16, 1, [15, 16, 31], None),
    (128, 2, 16, 50, [0, 5, 31, 160], None),                 # pages begun and ended anywhere
    (64, 3, 32, 77, [1, 32, 40], [77, 0, 3]),                # a padded batch, one of its sequences without rows
    (128, 8, 128, 130, [127, 3], [130, 129]),
])
def test_write_and_read_back(dtype, fmt, d, hkv, ps, n, starts, counts):
    ops = _ops()
    batch, per = len(starts), 4 if ps > 16 else 14
    pages = batch * per + 2
    ref = _full(fmt, dtype, pages, hkv, ps, d, 1)
    table = _table(batch, per, pages, 2)
    g = _gen(3)
    key = (torch.randn(batch, n, hkv, d, generator=g) * torch.logspace(-3, 2, n)[None, :, None, None]).to(dtype)
    value = torch.randn(batch, n, hkv, d, generator=g).to(dtype)
    key[:, ::3, :, 5] = key.abs().amax(-1)[:, ::3] / 2      # half the largest: the quotient is next to a half-integer
    key[:, ::7] = 0.0
    got = _cuda(ref)
    pool = _handle(got, dtype)
    ops.paged_write(pool, key.cuda(), value.cuda(), table.cuda(), _i32(starts), None if counts is None else _i32(counts))
    lens = [n] * batch if counts is None else counts
    PO.write(ref, fmt, key, value, table, starts, lens)
    for name, t in ref.items():
        if t is not None:
            assert torch.equal(got[name].cpu(), t), name     # codes, scales and bounds to the last bit; every other row as it was
    ends = [s + c for s, c in zip(starts, lens)]
    k, v = ops.paged_read(pool, table.cuda(), _i32(starts), n, _i32(ends))
    rk, rv = PO.read(ref, fmt, dtype, table, starts, n, ends)
    assert torch.equal(k.cpu(), rk) and torch.equal(v.cpu(), rv)


@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_are_the_nearest_multiples_of_the_scale(dtype, fmt):
    """Every 16-bit value against rows whose largest value makes ties and near ties: 254/256 and its neighbours, powers of two,
    the smallest and largest normal numbers and subnormal ones."""
    ops = _ops()
    tops = [1.0, 1.9844, 1.9922, 1.9766, 3.0, 0.0078, 254.0, 127.0, 7.0, 3.5, float(torch.finfo(dtype).max), float(torch.finfo(dtype).tiny),
            float(torch.finfo(dtype).tiny) / 8]
    if dtype == torch.bfloat16:
        tops += [1e-30, 1e-36, 1e30]
    d, rows = 128, []
    for t in tops:
        top = torch.tensor(t).to(dtype)
        half = (torch.arange(-254, 255).double() / 254.0 * float(top)).to(dtype)   # multiples of half a step, rounded
        half = half[half.abs() <= top]
        half = torch.cat((half, half.new_zeros(-len(half) % (d - 1)))).view(-1, d - 1)
        rows.append(torch.cat((top.expand(len(half), 1), half), 1))
    x = torch.cat(rows)
    n = len(x)
    ref = _empty(fmt, dtype, (n + 15) // 16, 1, 16, d)
    table = torch.arange((n + 15) // 16, dtype=torch.int32)[None]
    key = x.view(1, n, 1, d)
    got = _cuda(ref)
    ops.paged_write(_handle(got, dtype), key.cuda(), key.flip(1).cuda(), table.cuda(), _i32([0]))
    PO.write(ref, fmt, key, key.flip(1), table, [0], [n])
    for name, t in ref.items():
        assert torch.equal(got[name].cpu(), t), name


@pytest.mark.parametrize("fmt", ["int8", "int4"])
def test_rows_that_are_not_finite_read_back_as_nan(fmt):
    ops = _ops()
    dtype, d = torch.bfloat16, 64
    key = torch.randn(1, 5, 2, d, generator=_gen(1)).to(dtype)
    key[0, 1, 0, 3], key[0, 3, 1, 9] = float("inf"), float("nan")
    value = torch.randn(1, 5, 2, d, generator=_gen(2)).to(dtype)
    value[0, 2, 0, 63] = -float("inf")
    ref = _empty(fmt, dtype, 1, 2, 16, d)
    got = _cuda(ref)
    pool = _handle(got, dtype)
    table = torch.zeros(1, 1, dtype=torch.int32)
    ops.paged_write(pool, key.cuda(), value.cuda(), table.cuda(), _i32([0]))
    PO.write(ref, fmt, key, value, table, [0], [5])
    k, v = ops.paged_read(pool, table.cuda(), _i32([0]), 5)
    rk, rv = PO.read(ref, fmt, dtype, table, [0], 5, None)
    assert _same(k, rk) and _same(v, rv)
    assert k[0, 1, 0].isnan().all() and v[0, 2, 0].isnan().all() and not k[0, 1, 1].isnan().any()


@pytest.mark.parametrize("fmt", FORMATS)
def test_write_skips_what_the_table_does_not_hold(fmt):
    """Ids outside the pool, positions past the table or below zero: nothing is written, nothing faults, reads are zeros."""
    ops = _ops()
    dtype, hkv, ps, d, n = torch.float16, 2, 16, 128, 40
    ref = _full(fmt, dtype, 6, hkv, ps, d, 5)
    table = torch.tensor([[0, -1, 1], [6, 2, 2147483647], [3, 4, 5], [5, 4, 3]], dtype=torch.int32)
    starts = [8, 0, 30, -3]
    g = _gen(6)
    key, value = (torch.randn(4, n, hkv, d, generator=g).to(dtype) for _ in range(2))
    got = _cuda(ref)
    pool = _handle(got, dtype)
    ops.paged_write(pool, key.cuda(), value.cuda(), table.cuda(), _i32(starts))
    PO.write(ref, fmt, key, value, table, starts, [n] * 4)
    for name, t in ref.items():
        if t is not None:
            assert torch.equal(got[name].cpu(), t), name
    starts = [-5, 0, 20, 2147483640]
    k, v = ops.paged_read(pool, table.cuda(), _i32(starts), 60, _i32([40, 60, 30, 2147483647]))
    rk, rv = PO.read(ref, fmt, dtype, table, starts, 60, [40, 60, 30, 2147483647])
    assert torch.equal(k.cpu(), rk) and torch.equal(v.cpu(), rv)


def test_write_and_read_take_strided_and_unaligned_tensors():
    """Views of a fused projection, heads before tokens, odd offsets; a read into a larger buffer leaves the rest of it."""
    ops = _ops()
    dtype, hkv, ps, d, n, b = torch.bfloat16, 2, 32, 64, 45, 2
    fused = torch.randn(b, n, 3 * hkv * d + 4, generator=_gen(7)).to(dtype)
    table = _table(b, 2, 5, 8)
    ref = _empty("int8", dtype, 5, hkv, ps, d)
    PO.write(ref, "int8", fused[..., hkv * d:2 * hkv * d].reshape(b, n, hkv, d), fused[..., 3:3 + hkv * d].reshape(b, n, hkv, d), table, [3, 9], [n, n])
    got = _cuda(ref)
    for t in got.values():
        t.zero_()
    pool = _handle(got, dtype)
    dev = fused.cuda()
    key = dev[..., hkv * d:2 * hkv * d].unflatten(-1, (hkv, d))
    value = dev[..., 3:3 + hkv * d].unflatten(-1, (hkv, d))                    # rows that no 16-byte load can take
    key = key.transpose(1, 2).contiguous().transpose(1, 2)                     # [B, Hkv, N, D] storage
    ops.paged_write(pool, key, value, table.cuda(), _i32([3, 9]))
    for name, t in ref.items():
        assert torch.equal(got[name].cpu(), t), name
    big = torch.full((2, b, n + 7, hkv + 1, d), 3.0, dtype=dtype, device="cuda")
    ops.paged_read(pool, table.cuda(), _i32([3, 9]), n, out=(big[0, :, 2:n + 2, 1:], big[1, :, 2:n + 2, 1:]))
    rk, rv = PO.read(ref, "int8", dtype, table, [3, 9], n, None)
    assert torch.equal(big[0, :, 2:n + 2, 1:].cpu(), rk) and torch.equal(big[1, :, 2:n + 2, 1:].cpu(), rv)
    assert (big[:, :, :2] == 3).all() and (big[:, :, n + 2:] == 3).all() and (big[:, :, :, 0] == 3).all()


# ---- attention -------------------------------------------------------------------------------------------------------
def _check_attention(q, pool, fmt, table, lens, out, lse, pages=None, sm_scale=None):
    """|o - ref| <= half a step of the output's type + errors of the weights: their rounding to 11 bits, of the scores
    (sums of D products in fp32, so D steps of 2^-23 of sum |q k|; both numerator and denominator have it) and of sums of n
    terms in fp32.  The LSE has the scores' and the sum's.

    A weight p s_j (s_j the value's scale, p <= 1) is rounded to f16 as p s_j 2^14 / 2^e with 2^e <= max s, so below f16's
    normal numbers the step is 2^-24 in those units: an error of up to 2^-25 2^-14 2^e a key, times its code, |code| <= Q.  All
    keys together: n 2^-39 Q max s, and Q max s is the largest |v| (every row has a code of Q).  Native f16 weights have the
    same step, with 2^e = 1."""
    d, n = q.shape[-1], max(lens + [1])
    o, l, spread, size, vmax = PO.attention(q, pool, fmt, table, lens, pages, sm_scale)
    out, lse = out.double().cpu(), lse.double().cpu()
    o, l, spread, size, vmax = (t.cpu() for t in (o, l, spread, size, vmax))
    rel = 2.0 ** -11 + 2 * d * 2.0 ** -23 * size + n * 2.0 ** -23
    tol = torch.finfo(q.dtype).eps / 2 * o.abs() + rel[..., None] * spread + n * 2.0 ** -39 * vmax[..., None]
    tiny = torch.finfo(q.dtype).tiny
    assert ((out - o).abs() <= tol + tiny).all(), ((out - o).abs() / (tol + tiny)).max()
    empty = l == -float("inf")
    assert torch.equal(lse == -float("inf"), empty)
    err = (lse - l).abs()[~empty]
    assert (err <= (d * 2.0 ** -23 * size[~empty] + n * 2.0 ** -23) * 1.4427 + 2.0 ** -22 * (1 + l[~empty].abs())).all()


def _decode(q, pool, dtype, table, lens, **kw):
    """q [B, Hq, D]"""
    out, lse = _ops().paged_decode(q[:, None].cuda(), _handle(pool, dtype), table.cuda(), _i32(lens), return_lse=True, **kw)
    return out[:, 0], lse[:, :, 0]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,hkv,group,ps,lens", [
    (128, 4, 7, 64, [1000]),
    (128, 2, 1, 16, [1, 2, 15, 16, 17, 33, 0, 300]),         # lengths around a page and a tile, one of them zero
    (64, 1, 16, 32, [31, 32, 33, 2047]),
    (64, 8, 4, 128, [127, 128, 129, 700]),
    (128, 1, 8, 16, [4099]),
    (128, 3, 9, 32, [513, 95]),
    (64, 2, 5, 64, [63, 1, 3000]),
])
def test_decode_against_the_definition(dtype, fmt, d, hkv, group, ps, lens):
    per = max(1, (max(lens) + ps - 1) // ps)
    pages = len(lens) * per + 2
    host = _full(fmt, dtype, pages, hkv, ps, d, 11)
    pool = _cuda(host)
    table = _table(len(lens), per, pages, 12)
    q = torch.randn(len(lens), hkv * group, d, generator=_gen(13)).to(dtype)
    out, lse = _decode(q, pool, dtype, table, lens)
    assert out.dtype == dtype
    _check_attention(q.cuda(), pool, fmt, table, lens, out, lse)
    for i, n in enumerate(lens):
        if n == 0:
            assert (out[i] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("sm_scale,mag", [(0.0, 12.0), (1.0, 1.0), (0.02, 1e-3)])
def test_decode_with_sharp_and_flat_softmaxes(fmt, sm_scale, mag):
    """Scores that one key dominates, and ones that hardly differ; a key with tiny values takes nearly all the weight (the
    values' scales differ by orders of magnitude)."""
    dtype, d, hkv, ps, lens = torch.bfloat16, 128, 2, 32, [1500, 40]
    host = _full(fmt, dtype, 100, hkv, ps, d, 21)
    q = (torch.randn(2, 8, d, generator=_gen(22)) * mag).to(dtype)
    table = _table(2, 47, 100, 23)
    page = int(table[0, 0])
    if fmt == "native":
        host["k_pages"][page, 0, 0] = q[0, 0] * 2
        host["v_pages"][page, 0, 0] *= 1e-3
    else:
        host["v_scale"][page, 0, 0] *= 1e-3
        host["v_scale"][int(table[0, 3])] *= 1e3
        host["k_scale"][page, 0, 0] *= 5
    pool = _cuda(host)
    out, lse = _decode(q, pool, dtype, table, lens, sm_scale=sm_scale)
    _check_attention(q.cuda(), pool, fmt, table, lens, out, lse, sm_scale=sm_scale or None)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("ps", [16, 128])
def test_decode_ignores_what_lies_behind_a_sequence(fmt, ps):
    """NaN, infinities and the lowest values in the rows behind the last token, in pages of nobody and behind the table's
    bad ids change nothing."""
    dtype, d, hkv, lens = torch.float16, 128, 2, [ps * 3 + 5, 7, 1]
    host = _full(fmt, dtype, 16, hkv, ps, d, 31)
    table = torch.full((3, 5), -1, dtype=torch.int32)
    table[0, :4], table[1, 0], table[2, 0] = torch.tensor([3, 9, 0, 12]), 5, 7
    q = torch.randn(3, 8, d, generator=_gen(32)).to(dtype)
    clean, _ = _decode(q, _cuda(host), dtype, table, lens)
    used = {3: ps, 9: ps, 0: ps, 12: 5, 5: 7, 7: 1}
    for page in range(16):
        r = used.get(page, 0)
        if fmt == "native":
            host["k_pages"][page, :, r:] = float("nan")
            host["v_pages"][page, :, r:] = float("inf")
            host["v_pages"][page, :, r + 1:] = torch.finfo(dtype).min
        else:
            host["k_scale"][page, :, r:], host["v_scale"][page, :, r:] = float("nan"), float("inf")
            host["v_pages"][page, :, r:] = 127
    dirty, lse = _decode(q, _cuda(host), dtype, table, lens)
    assert torch.equal(clean, dirty) and lse.isfinite().all()
    table[0, 1], table[1, 0] = 16, -7          # a page lost in the middle, and a whole sequence
    out, lse = _decode(q, _cuda(host), dtype, table, lens)
    _check_attention(q.cuda(), _cuda(host), fmt, table, lens, out, lse)
    assert (out[1] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_hands_on_nan_of_rows_that_count(fmt):
    dtype, d = torch.bfloat16, 64
    host = _full(fmt, dtype, 8, 2, 16, d, 41)
    name = "v_pages" if fmt == "native" else "v_scale"
    host[name][2, 0, 3] = float("nan")
    table = torch.arange(8, dtype=torch.int32)[None]
    q = torch.randn(1, 4, d, generator=_gen(42)).to(dtype)
    out, _ = _decode(q, _cuda(host), dtype, table, [100])
    assert out[0, :2].isnan().all() and out[0, 2:].isfinite().all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n", [20, 500])
def test_decode_of_values_near_the_types_range(fmt, n):
    """bf16 values of up to 2^118, one warp's and several warps' keys: sums of weights times values stay in fp32's range."""
    dtype, d = torch.bfloat16, 128
    g = _gen(46)
    table = torch.arange(8, dtype=torch.int32)[None]
    ref = _empty(fmt, dtype, 8, 1, 64, d)
    key, value = torch.randn(1, n, 1, d, generator=g).to(dtype), (torch.rand(1, n, 1, d, generator=g) * 2.0 ** 118).to(dtype)
    PO.write(ref, fmt, key, value, table, [0], [n])
    q = torch.randn(1, 8, d, generator=g).to(dtype)
    pool = _cuda(ref)
    out, lse = _decode(q, pool, dtype, table, [n])
    assert out.isfinite().all()
    _check_attention(q.cuda(), pool, fmt, table, [n], out, lse)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shift", [1, 2])
def test_decode_of_queries_at_any_address(fmt, shift):
    ops = _ops()
    dtype, d = torch.float16, 64
    pool = _handle(_cuda(_full(fmt, dtype, 8, 2, 16, d, 47)), dtype)
    table, lens = torch.arange(8, dtype=torch.int32)[None].cuda(), _i32([100])
    q = torch.randn(1, 1, 6, d, generator=_gen(48)).to(dtype).cuda()
    odd = torch.zeros(1, 1, 6, d + shift, dtype=dtype, device="cuda")
    odd[..., shift:] = q
    assert torch.equal(ops.paged_decode(odd[..., shift:], pool, table, lens), ops.paged_decode(q, pool, table, lens))
    pages = ops.paged_select(odd[..., shift:], pool, table, lens, 3)
    assert torch.equal(pages, ops.paged_select(q, pool, table, lens, 3))


def test_decode_layouts_types_bounds_and_table_strides():
    ops = _ops()
    dtype, d, hkv, ps, lens = torch.bfloat16, 128, 2, 32, [100, 257]
    host = _full("int8", dtype, 30, hkv, ps, d, 51)
    pool = _cuda(host)
    h = _handle(pool, dtype)
    table = _table(2, 9, 30, 52)
    wide = torch.full((2, 13), -1, dtype=torch.int32)
    wide[:, :9] = table
    q = torch.randn(2, 6, d, generator=_gen(53)).to(dtype)
    ref, rl = _decode(q, pool, dtype, table, lens)
    nhd = ops.paged_decode(q[:, None].cuda(), h, wide.cuda()[:, :9], _i32(lens))
    assert torch.equal(nhd[:, 0], ref)
    odd = torch.zeros(2, 6, 2 * d + 1, dtype=dtype, device="cuda")            # rows at odd addresses
    odd[:, :, 1:d + 1] = q.cuda()
    hnd = ops.paged_decode(odd[:, :, None, 1:d + 1], h, table.cuda(), _i32(lens), layout="HND", out_dtype=torch.float16)
    assert hnd.shape == (2, 6, 1, d) and hnd.dtype == torch.float16
    assert torch.equal(hnd[:, :, 0].to(dtype), ref) or (hnd[:, :, 0].float() - ref.float()).abs().max() < 2.0 ** -7
    cut, cl = ops.paged_decode(q[:, None].cuda(), h, table.cuda(), _i32(lens), max_kv_len=150, return_lse=True)
    _check_attention(q.cuda(), pool, "int8", table, [100, 150], cut[:, 0], cl[:, :, 0])
    cap, pl = ops.paged_decode(q[:, None].cuda(), h, table.cuda(), _i32([10 ** 9, -5]), return_lse=True)   # past the table; below zero
    _check_attention(q.cuda(), pool, "int8", table, [288, 0], cap[:, 0], pl[:, :, 0])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
def test_decode_over_listed_pages(fmt, ps):
    """Lists of each KV head: in any order, with holes, with a page that the sequence does not hold, the last page among them."""
    ops = _ops()
    dtype, d, hkv, lens = torch.bfloat16, 128, 2, [9 * ps + 3, ps // 2]
    host = _full(fmt, dtype, 30, hkv, ps, d, 61)
    pool = _cuda(host)
    table = _table(2, 12, 30, 62)
    lists = [[[0, 9, 4, -1, 2, 11], [3, 10, 5, 2147483647, 1, 8]], [[0, -1, 1, -2147483648, 5, 2], [-1, -1, -1, -1, -1, -1]]]
    q = torch.randn(2, 14, d, generator=_gen(63)).to(dtype)
    out, lse = ops.paged_decode(q[:, None].cuda(), _handle(pool, dtype), table.cuda(), _i32(lens), pages=_i32(lists), return_lse=True)
    _check_attention(q.cuda(), pool, fmt, table, lens, out[:, 0], lse[:, :, 0], pages=lists)
    assert (out[1, 0, 7:] == 0).all() and (lse[1, 7:] == -float("inf")).all()


def test_listing_every_page_is_decoding_over_all():
    ops = _ops()
    dtype, d, hkv, ps, lens = torch.float16, 128, 4, 64, [3000, 1, 999]
    pool = _cuda(_full("int8", dtype, 150, hkv, ps, d, 71))
    h, table = _handle(pool, dtype), _table(3, 47, 150, 72).cuda()
    q = torch.randn(3, 1, 28, d, generator=_gen(73)).to(dtype).cuda()
    every = torch.arange(47, dtype=torch.int32, device="cuda").expand(3, hkv, 47).contiguous()
    a, la = ops.paged_decode(q, h, table, _i32(lens), return_lse=True)
    b, lb = ops.paged_decode(q, h, table, _i32(lens), pages=every, return_lse=True)
    # other key ranges, so other orders of the same sums: a step of the output's type at most where it is not tiny
    assert (a.float() - b.float()).abs().max() <= 2.0 ** -10 * max(1.0, a.abs().max().item())
    assert (la - lb).abs().max() < 1e-4


# ---- selection -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,hkv,group,ps,lens,budget,sink,recent", [
    (128, 4, 7, 64, [6400, 64, 100, 1, 0], 16, 1, 2),
    (64, 2, 1, 16, [1600, 1599], 30, 0, 0),
    (128, 1, 16, 32, [9000], 5, 2, 3),                       # nothing left to choose
    (64, 3, 4, 128, [20000, 300], 200, 1, 1),                # more than the sequence holds
    (128, 2, 2, 16, [33000], 700, 1, 4),
])
def test_select_against_the_definition(dtype, d, hkv, group, ps, lens, budget, sink, recent):
    ops = _ops()
    per = max(1, (max(lens) + ps - 1) // ps)
    pages = len(lens) * per
    pool = _empty("native", dtype, pages, hkv, ps, d)
    g = _gen(81)
    lo = torch.randn(pages, hkv, d, generator=g).to(dtype)
    pool["k_bounds"][:, :, 0] = lo
    pool["k_bounds"][:, :, 1] = lo + torch.rand(pages, hkv, d, generator=g).to(dtype)
    pool["k_bounds"][1::2] = pool["k_bounds"][: len(pool["k_bounds"][1::2])]        # pairs of equal scores
    table = _table(len(lens), per, pages, 82)
    if per > 20:
        table[0, 7], table[0, 11] = -1, pages
    q = torch.randn(len(lens), hkv * group, d, generator=g).to(dtype)
    got = ops.paged_select(q[:, None].cuda(), _handle(_cuda(pool), dtype), table.cuda(), _i32(lens), budget, sink_pages=sink, recent_pages=recent)
    assert got.tolist() == PO.select(q, pool, table, lens, budget, sink, recent)


def test_select_with_all_scores_equal_takes_the_lowest_pages():
    ops = _ops()
    pool = _empty("int8", torch.bfloat16, 500, 2, 16, 64)
    table = torch.arange(500, dtype=torch.int32)[None].cuda()
    q = torch.ones(1, 1, 4, 64, dtype=torch.bfloat16, device="cuda")
    got = ops.paged_select(q, _handle(_cuda(pool), torch.bfloat16), table, _i32([16 * 400]), 20, sink_pages=2, recent_pages=3)
    assert got[0, 0].tolist() == list(range(17)) + [397, 398, 399] and torch.equal(got[0, 0], got[0, 1])


def test_select_with_bounds_that_are_not_finite():
    """An infinite bound puts a page first or last, a NaN behind all others; zeros times infinities are NaN."""
    ops = _ops()
    dtype = torch.bfloat16
    pool = _empty("int8", dtype, 40, 1, 16, 64)
    pool["k_bounds"][:, 0, 1] = torch.randn(40, 64, generator=_gen(91)).to(dtype)
    pool["k_bounds"][9, 0, 1, 0], pool["k_bounds"][13, 0, 1, 1], pool["k_bounds"][21, 0, 1, 2] = float("inf"), float("nan"), -float("inf")
    pool["k_bounds"][21, 0, 0, 2] = -float("inf")
    q = torch.ones(1, 1, 1, 64, dtype=dtype, device="cuda")
    table = torch.arange(40, dtype=torch.int32)[None].cuda()
    h = _handle(_cuda(pool), dtype)
    first = ops.paged_select(q, h, table, _i32([640]), 1, sink_pages=0, recent_pages=0)
    assert first.tolist() == [[[9]]]
    most = ops.paged_select(q, h, table, _i32([640]), 39, sink_pages=0, recent_pages=0)
    assert most[0, 0].tolist() == [i for i in range(40) if i != 13]
    most = ops.paged_select(q, h, table, _i32([640]), 38, sink_pages=0, recent_pages=0)
    assert most[0, 0].tolist() == [i for i in range(40) if i not in (13, 21)]


# ---- together, streams, graphs ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
def test_prompt_then_steps_then_sparse(fmt):
    """A prompt goes into pages, tokens are appended one by one, each step attends over everything and over selected pages."""
    ops = _ops()
    dtype, d, hkv, hq, ps, n, steps = torch.bfloat16, 128, 2, 8, 16, 150, 40
    ref = _empty(fmt, dtype, 40, hkv, ps, d)
    got = _cuda(ref)
    pool = _handle(got, dtype)
    table = _table(2, 13, 40, 101)
    g = _gen(102)
    key, value = (torch.randn(2, n + steps, hkv, d, generator=g).to(dtype) for _ in range(2))
    counts = [n, n - 37]
    dev = table.cuda()
    ops.paged_write(pool, key[:, :n].cuda(), value[:, :n].cuda(), dev, _i32([0, 0]), _i32(counts))
    PO.write(ref, fmt, key[:, :n], value[:, :n], table, [0, 0], counts)
    lens = _i32(counts)
    for t in range(steps):
        new = slice(n + t, n + t + 1)
        ops.paged_write(pool, key[:, new].cuda(), value[:, new].cuda(), dev, lens)
        PO.write(ref, fmt, key[:, new], value[:, new], table, [c + t for c in counts], [1, 1])
        lens += 1
        if t % 13 and t != steps - 1:
            continue
        host = [c + t + 1 for c in counts]
        q = torch.randn(2, hq, d, generator=g).to(dtype)
        out, lse = ops.paged_decode(q[:, None].cuda(), pool, dev, lens, return_lse=True)
        _check_attention(q, ref, fmt, table, host, out[:, 0], lse[:, :, 0])
        pages = ops.paged_select(q[:, None].cuda(), pool, dev, lens, 5, sink_pages=1, recent_pages=1)
        assert pages.tolist() == PO.select(q, ref, table, host, 5, 1, 1)
        out, lse = ops.paged_decode(q[:, None].cuda(), pool, dev, lens, pages=pages, return_lse=True)
        _check_attention(q, ref, fmt, table, host, out[:, 0], lse[:, :, 0], pages=pages.tolist())


def test_captured_step_follows_the_lengths():
    """Append, select and attend captured once: replays read positions, lengths and pages when they run."""
    ops = _ops()
    dtype, d, hkv, hq, ps = torch.bfloat16, 128, 2, 8, 32
    pool_t = _cuda(_full("int8", dtype, 64, hkv, ps, d, 111))
    pool = _handle(pool_t, dtype)
    table = _table(1, 60, 64, 112).cuda()
    lens, q = _i32([100]), torch.zeros(1, 1, hq, d, dtype=dtype, device="cuda")
    key, value = (torch.zeros(1, 1, hkv, d, dtype=dtype, device="cuda") for _ in range(2))

    def step():
        ops.paged_write(pool, key, value, table, lens)
        after = lens + 1
        pages = ops.paged_select(q, pool, table, after, 6, recent_pages=2)
        return pages, ops.paged_decode(q, pool, table, after), ops.paged_decode(q, pool, table, after, pages=pages)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    g = _gen(113)
    for n in (100, 101, 1800, 0, 31):
        lens.fill_(n)
        q.copy_(torch.randn(1, 1, hq, d, generator=g))
        key.copy_(torch.randn(1, 1, hkv, d, generator=g))
        value.copy_(torch.randn(1, 1, hkv, d, generator=g))
        graph.replay()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_batches_at_the_limits():
    """One head of one short sequence; as many sequences as a call takes, empty ones among them; one more is refused."""
    ops = _ops()
    dtype, d = torch.bfloat16, 64
    host = _full("int4", dtype, 64, 1, 16, d, 141)
    pool_t = _cuda(host)
    pool = _handle(pool_t, dtype)
    b = 1024
    table = torch.randint(0, 64, (b, 3), generator=_gen(142), dtype=torch.int32)
    lens = torch.randint(-1, 49, (b,), generator=_gen(143)).tolist()
    q = torch.randn(b, 2, d, generator=_gen(144)).to(dtype)
    out, lse = _decode(q, pool_t, dtype, table, lens)
    _check_attention(q.cuda(), pool_t, "int4", table, lens, out, lse)
    one, l1 = _decode(q[:1, :1], pool_t, dtype, table[:1], [1])
    _check_attention(q[:1, :1].cuda(), pool_t, "int4", table[:1], [1], one, l1)
    with pytest.raises(ValueError, match="1024"):
        ops.paged_decode(torch.zeros(b + 1, 1, 2, d, dtype=dtype, device="cuda"), pool, torch.zeros(b + 1, 3, dtype=torch.int32, device="cuda"), _i32([1] * (b + 1)))
    none = ops.paged_decode(torch.zeros(0, 1, 2, d, dtype=dtype, device="cuda"), pool, table[:0].cuda(), _i32([]))
    assert none.shape == (0, 1, 2, d)


def test_wrong_tensors_are_refused():
    ops = _ops()
    dtype, d = torch.bfloat16, 64
    pool = _handle(_cuda(_full("int8", dtype, 4, 2, 16, d, 151)), dtype)
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), _i32([3, 4])
    q = torch.zeros(2, 1, 4, d, dtype=dtype, device="cuda")
    rows = torch.zeros(2, 3, 2, d, dtype=dtype, device="cuda")
    bad_calls = [
        lambda: ops.paged_decode(q.half(), pool, table, lens), lambda: ops.paged_decode(q.cpu(), pool, table, lens),
        lambda: ops.paged_decode(q[..., :32], pool, table, lens), lambda: ops.paged_decode(q.expand(2, 2, 4, d), pool, table, lens),
        lambda: ops.paged_decode(q, pool, table.long(), lens), lambda: ops.paged_decode(q, pool, table[:1], lens),
        lambda: ops.paged_decode(q, pool, table.cpu(), lens), lambda: ops.paged_decode(q, pool, table, lens.long()),
        lambda: ops.paged_decode(q, pool, table, lens[:1]), lambda: ops.paged_decode(q, pool, table.t().contiguous().t(), lens),
        lambda: ops.paged_decode(q, pool, table, lens, layout="HND"), lambda: ops.paged_decode(q, pool, table, lens, out_dtype=torch.float32),
        lambda: ops.paged_decode(q, pool, table, lens, pages=torch.zeros(2, 2, 0, dtype=torch.int32, device="cuda")),
        lambda: ops.paged_decode(q, pool, table, lens, pages=torch.zeros(2, 1, 3, dtype=torch.int32, device="cuda")),
        lambda: ops.paged_decode(q, pool, table, lens, sm_scale=float("nan")), lambda: ops.paged_decode(q, pool, table, lens, max_kv_len=-1),
        lambda: ops.paged_decode(q[:, :, :3], pool, table, lens),
        lambda: ops.paged_select(q, pool, table, lens, 0), lambda: ops.paged_select(q, pool, table, lens, 2, sink_pages=2, recent_pages=1),
        lambda: ops.paged_write(pool, rows.float(), rows.float(), table, lens), lambda: ops.paged_write(pool, rows, rows[:, :2], table, lens),
        lambda: ops.paged_write(pool, rows[:, :, :1], rows[:, :, :1], table, lens), lambda: ops.paged_write(pool, rows, rows, table, lens, lens[:1]),
        lambda: ops.paged_read(pool, table, lens, -1), lambda: ops.paged_read(pool, table, lens, 3, out=(rows, rows.half())),
        lambda: ops.paged_read(pool, table, lens, 3, out=(rows, rows[:1, :1].expand(2, 3, 2, d))),
    ]
    for i, call in enumerate(bad_calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_after_a_wait_that_ran_out_results_are_nan_until_it_is_cleared():
    """The failure is a wait of the cross-GPU merge for a flag that nothing sets: it gives up after a second.  While its word is set
    every form of the paged decode (clusters, stretches joined by rows and by cuts) returns NaN; then the old results again."""
    import ctypes as C
    from longcontext_sqattn_paddle_b200 import _lib as L
    ops = _ops()
    dtype, d = torch.bfloat16, 128
    forms = []
    for fmt, b, hkv, lens in (("native", 1, 2, [300]), ("int8", 1, 4, [20000]), ("int4", 40, 8, [700] * 40)):
        per = (max(lens) + 63) // 64
        pool = _handle(_cuda(_full(fmt, dtype, per + 3, hkv, 64, d, 161)), dtype)
        table = torch.arange(per, dtype=torch.int32).expand(b, per).contiguous().cuda()
        q = torch.randn(b, 1, 4 * hkv, d, generator=_gen(162)).to(dtype).cuda()
        forms.append((q, pool, table, _i32(lens)))
    clean = [ops.paged_decode(*f, return_lse=True) for f in forms]
    dev, rows, world = torch.device("cuda", 0), 8, 2
    ops.poll_device_status(dev)
    data = [torch.zeros(L.lib.sqattn_peer_merge_data_bytes(world, rows, d) // 4, dtype=torch.int32, device=dev) for _ in range(world)]
    flags = [torch.zeros(L.lib.sqattn_peer_merge_flag_bytes(world, rows) // 4, dtype=torch.int32, device=dev) for _ in range(world)]
    epoch, po, pl = torch.zeros(1, dtype=torch.int32, device=dev), torch.randn(rows, d, device=dev), torch.randn(rows, device=dev)
    out = torch.zeros(rows, d, dtype=dtype, device=dev)
    a = L.PeerMergeArgs()
    for i in range(world):
        a.peer_data[i], a.peer_flags[i] = data[i].data_ptr(), flags[i].data_ptr()
    a.rank, a.world, a.rows, a.rows_cap, a.head_dim = 0, world, rows, rows, d
    a.epoch, a.part_o, a.part_lse, a.out, a.o_dtype = epoch.data_ptr(), po.data_ptr(), pl.data_ptr(), out.data_ptr(), L.BF16
    L.check(L.lib.sqattn_decode_peer_merge(C.byref(a), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    with pytest.raises(L.SqattnError):
        ops.paged_decode(*forms[0])
    ops._MIRRORS[0][1].value = 0               # a caller that ignored the mirror and carried on
    for f in forms:
        o, l = ops.paged_decode(*f, return_lse=True)
        assert o.isnan().all() and l.isnan().all()
    with pytest.raises(L.SqattnError):
        ops.check_device_status()
    ops.check_device_status()
    for f, (o, l) in zip(forms, clean):
        o2, l2 = ops.paged_decode(*f, return_lse=True)
        assert torch.equal(o, o2) and torch.equal(l, l2)


def test_calls_on_two_streams_do_not_share_scratch():
    ops = _ops()
    dtype, d, hkv, hq, ps, lens = torch.bfloat16, 128, 4, 28, 64, [30000]
    pools = [_handle(_cuda(_full("int8", dtype, 480, hkv, ps, d, 121 + i)), dtype) for i in range(2)]
    table, kv = torch.arange(480, dtype=torch.int32)[None].cuda(), _i32(lens)
    q = torch.randn(1, 1, hq, d, generator=_gen(123)).to(dtype).cuda()
    alone = [ops.paged_decode(q, p, table, kv, pages=ops.paged_select(q, p, table, kv, 100)) for p in pools]
    full = [ops.paged_decode(q, p, table, kv) for p in pools]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = []
        for s, p in zip(streams, pools):
            with torch.cuda.stream(s):
                got.append((ops.paged_decode(q, p, table, kv, pages=ops.paged_select(q, p, table, kv, 100)), ops.paged_decode(q, p, table, kv)))
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(got[i][0], alone[i]) and torch.equal(got[i][1], full[i])


def test_offsets_beyond_32_bits():
    """Pages whose rows begin past 2^31 bytes and past 2^32 elements of the pool."""
    ops = _ops()
    dtype, d, hkv, ps = torch.bfloat16, 128, 8, 128
    pages = 35000                                             # 35000 * 8 * 128 * 128 = 4.6e9 elements, 9.2 GB a tensor
    pool = {n: torch.empty(pages, hkv, ps, d, dtype=dtype, device="cuda") for n in ("k_pages", "v_pages")}
    bounds = torch.empty(pages, hkv, 2, d, dtype=dtype, device="cuda")
    h = ops.PagedPool(k_bounds=bounds, **pool)
    table = torch.tensor([[34999, 16400, 0, 33000, 34998]], dtype=torch.int32)
    g = _gen(131)
    key, value = (torch.randn(1, 5 * ps, hkv, d, generator=g).to(dtype) for _ in range(2))
    ops.paged_write(h, key.cuda(), value.cuda(), table.cuda(), _i32([0]))
    for i, page in enumerate(table[0].tolist()):
        assert torch.equal(pool["k_pages"][page].transpose(0, 1).cpu(), key[0, i * ps:(i + 1) * ps])
    k, v = ops.paged_read(h, table.cuda(), _i32([0]), 5 * ps)
    assert torch.equal(k.cpu(), key) and torch.equal(v.cpu(), value)
    small = {n: torch.stack([pool[n][p] for p in table[0].tolist()]) for n in pool}
    small["k_bounds"] = torch.stack([bounds[p] for p in table[0].tolist()])
    q = torch.randn(1, 16, d, generator=g).to(dtype)
    order = torch.arange(5, dtype=torch.int32)[None]
    out, lse = ops.paged_decode(q[:, None].cuda(), h, table.cuda(), _i32([600]), return_lse=True)
    _check_attention(q.cuda(), small, "native", order, [600], out[:, 0], lse[:, :, 0])
    got = ops.paged_select(q[:, None].cuda(), h, table.cuda(), _i32([600]), 3)
    assert got.tolist() == PO.select(q.cuda(), small, order, [600], 3, 1, 1)
