"""The paged key/value cache of single-token decoding, and what is measured of it: quantising new rows into pages and
reading them back, attention of one new token over the pages, and the same over the pages that a cheap score selects.

Every operator is written here in its plain form (elementary tensor operations); with ``own`` the calls are the library's.
Geometries are those the repository's configurations name (28 query / 4 KV heads and 32 / 8, head_dim 128) and generic ones.
A layer's pool holds ``k_pages`` / ``v_pages`` [pages, Hkv, page_size, D] as 16-bit values ("native"), int8 codes or two 4-bit
codes a byte (even channel in the low half), one fp32 scale a row for codes, and ``k_bounds`` [pages, Hkv, 2, D], the channel
minima and maxima of the keys of every page."""
import math

import torch

own = False

SINK_PAGES, RECENT_PAGES = 1, 2
_TOP = {"int8": 127, "int4": 7}
_SMALLEST_SCALE = 2.0 ** -100


# ---- cases -----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one layer's keys and values of a 128K prompt go into 8-bit pages after its prefill
        dict(name="store_131072_int8", kind="store", batch=1, n=131072, ragged=False, start=0, hkv=4, d=128, page=64, fmt="int8", dtype="bf16"),
        # a padded batch of second turns is appended behind what the cache already holds, pages begun and ended anywhere
        dict(name="store_8x2001_int4", kind="store", batch=8, n=2001, ragged=True, start=1000, hkv=8, d=128, page=32, fmt="int4", dtype="fp16"),
        # the append of one decode step of a serving batch: pure latency
        dict(name="append_32_int8", kind="store", batch=32, n=1, ragged=False, start=9000, hkv=8, d=128, page=16, fmt="int8", dtype="bf16"),
        # a cached document is read back so that a prefill can attend to it
        dict(name="read_100003_int8", kind="read", batch=1, n=100003, start=0, hkv=4, d=128, page=64, fmt="int8", dtype="bf16"),
        # a few hundred rows from the middle of several short sequences
        dict(name="read_4x777_int4", kind="read", batch=4, n=777, start=300, hkv=2, d=64, page=16, fmt="int4", dtype="fp16"),
        # one token of one chat against a short cache: pure latency
        dict(name="decode_1000", kind="decode", batch=1, min_len=1000, max_len=1000, hq=28, hkv=4, d=128, page=64, fmt="native", dtype="bf16"),
        # one layer of a step at a million tokens of context, unquantised
        dict(name="decode_1048576", kind="decode", batch=1, min_len=1048576, max_len=1048576, hq=28, hkv=4, d=128, page=64, fmt="native", dtype="bf16"),
        # a serving batch whose contexts differ by a factor of thirty, 8-bit pages
        dict(name="decode_16_ragged_int8", kind="decode", batch=16, min_len=2000, max_len=65536, hq=32, hkv=8, d=128, page=32, fmt="int8", dtype="bf16"),
        # many short chats, 4-bit pages of the smallest size
        dict(name="decode_64_ragged_int4", kind="decode", batch=64, min_len=400, max_len=8191, hq=32, hkv=8, d=128, page=16, fmt="int4", dtype="fp16"),
        # half a million tokens in 4 bits
        dict(name="decode_524288_int4", kind="decode", batch=1, min_len=524288, max_len=524288, hq=28, hkv=4, d=128, page=64, fmt="int4", dtype="bf16"),
        # a million tokens of which each KV head attends to 4096
        dict(name="sparse_1048576_int8", kind="sparse", batch=1, min_len=1048576, max_len=1048576, hq=28, hkv=4, d=128, page=64, fmt="int8", dtype="bf16", top=64),
        # a ragged batch over unquantised pages, the budget above some of the lengths
        dict(name="sparse_16_ragged", kind="sparse", batch=16, min_len=3001, max_len=65536, hq=32, hkv=8, d=128, page=32, fmt="native", dtype="bf16", top=128),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "read", "decode", "decode", "sparse"])
    hkv, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128])
    c = dict(kind=kind, hkv=hkv, d=d, page=rng.choice([16, 32, 64, 128]), fmt=rng.choice(["native", "int8", "int4"]),
             dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind in ("store", "read"):
        c.update(batch=_log_uniform(rng, 1, 32), start=rng.choice([0, 0, rng.randint(1, 5000)]))
        c.update(n=_log_uniform(rng, 1, 524288 // (c["batch"] * hkv)))
        if kind == "store":
            c.update(ragged=rng.random() < 0.5)
        return c
    c.update(batch=_log_uniform(rng, 1, 64), hq=hkv * rng.choice([1, 2, 4, 5, 7, 8, 12, 16]))
    top = min(1048576, 2097152 // (c["batch"] * hkv))
    c.update(max_len=_log_uniform(rng, 16, top))
    c.update(min_len=_log_uniform(rng, 1, c["max_len"]))
    if kind == "sparse":
        c.update(top=_log_uniform(rng, 4, 256))
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _channels(case, dev):
    """Keys have a few channels that are much larger than the others."""
    w = torch.ones(case["d"], device=dev)
    w[:: case["d"] // 4] = 8.0
    return w


def _rows(g, shape, case, keys):
    x = torch.randn(*shape, device="cuda", generator=g)
    return (x * _channels(case, "cuda") if keys else x).to(_dtype(case))


def _lengths(case, seed):
    """Spread over the range's logarithm, the longest always among them."""
    r = torch.rand(case["batch"], generator=torch.Generator().manual_seed(seed + 77), dtype=torch.float64)
    r[0] = 1.0
    lo, hi = math.log(case["min_len"]), math.log(case["max_len"])
    return [max(1, min(case["max_len"], int(round(math.exp(lo + x * (hi - lo)))))) for x in r.tolist()]


def _empty_pool(case, pages):
    h, ps, d, fmt = case["hkv"], case["page"], case["d"], case["fmt"]
    kind = {"native": _dtype(case), "int8": torch.int8, "int4": torch.uint8}[fmt]
    width = d // 2 if fmt == "int4" else d
    pool = {n: torch.zeros(pages, h, ps, width, dtype=kind, device="cuda") for n in ("k_pages", "v_pages")}
    for n in ("k_scale", "v_scale"):
        pool[n] = None if fmt == "native" else torch.zeros(pages, h, ps, device="cuda")
    pool["k_bounds"] = torch.zeros(pages, h, 2, d, dtype=_dtype(case), device="cuda")
    return pool


def _fill(pool, case, g):
    """Every page full of rows as a model produces them."""
    for p0 in range(0, pool["k_pages"].shape[0], 2048):
        part = slice(p0, p0 + 2048)
        for t in ("k", "v"):
            n = pool["k_pages"][part].shape[0]
            x = _rows(g, (n, case["hkv"], case["page"], case["d"]), case, t == "k")
            if t == "k":
                pool["k_bounds"][part, :, 0], pool["k_bounds"][part, :, 1] = x.amin(dim=2), x.amax(dim=2)
            if case["fmt"] == "native":
                pool[t + "_pages"][part] = x
            else:
                codes, scale = _quantise(x, case["fmt"])
                pool[t + "_pages"][part] = _pack(codes) if case["fmt"] == "int4" else codes
                pool[t + "_scale"][part] = scale


def _handle(pool, case):
    """What a user of the library keeps for a layer: its pool."""
    from longcontext_sqattn_paddle_b200 import ops
    return ops.PagedPool(dtype=_dtype(case), **pool)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ps, batch = case["page"], case["batch"]
    s = dict(case=case)
    if case["kind"] in ("store", "read"):
        ends = [case["start"] + case["n"]] * batch
    else:
        ends = _lengths(case, seed)
    per = (max(ends) + ps - 1) // ps
    pages = batch * per + 3
    s["table"] = torch.randperm(pages, device="cuda", generator=g)[: batch * per].to(torch.int32).view(batch, per)   # pages of a sequence lie anywhere
    s["pool"] = _empty_pool(case, pages)
    if case["kind"] == "store":
        n = case["n"]
        s["key"] = _rows(g, (batch, n, case["hkv"], case["d"]), case, True)
        s["value"] = _rows(g, (batch, n, case["hkv"], case["d"]), case, False)
        s["start"] = torch.full((batch,), case["start"], dtype=torch.int32, device="cuda")
        s["count"] = torch.full((batch,), n, dtype=torch.int32, device="cuda")
        if case["ragged"]:
            s["count"] = torch.randint(1, n + 1, (batch,), device="cuda", generator=g, dtype=torch.int32)
        s["end"] = s["start"] + s["count"]
        if case["start"] % ps:
            _fill(s["pool"], case, g)   # the first pages are begun
    else:
        _fill(s["pool"], case, g)
        s["end"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        if case["kind"] == "read":
            s["start"] = torch.full((batch,), case["start"], dtype=torch.int32, device="cuda")
        else:
            s["q"] = torch.randn(batch, 1, case["hq"], case["d"], device="cuda", generator=g).to(_dtype(case))
            s["max_len"] = max(ends)
    if own:
        s["handle"] = _handle(s["pool"], case)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from longcontext_sqattn_paddle_b200 import ops
    case, pool, table = s["case"], s["handle"], s["table"]
    if case["kind"] == "store":
        ops.paged_write(pool, s["key"], s["value"], table, s["start"], s["count"] if case["ragged"] else None)
        key, value = ops.paged_read(pool, table, s["start"], case["n"], s["end"])
        return _stored(s["pool"], key, value)
    if case["kind"] == "read":
        return dict(zip(("key", "value"), ops.paged_read(pool, table, s["start"], case["n"], s["end"])))
    if case["kind"] == "decode":
        return dict(out=ops.paged_decode(s["q"], pool, table, s["end"], max_kv_len=s["max_len"]))
    pages = ops.paged_select(s["q"], pool, table, s["end"], case["top"], sink_pages=SINK_PAGES, recent_pages=RECENT_PAGES)
    return dict(pages=pages, out=ops.paged_decode(s["q"], pool, table, s["end"], pages=pages))


def _stored(pool, key, value):
    out = dict(key=key, value=value, k_bounds=pool["k_bounds"])
    if pool["k_scale"] is not None:
        out.update(k_scale=pool["k_scale"], v_scale=pool["v_scale"])
    return out


def _run_plain(s):
    case, pool, table, ps = s["case"], s["pool"], s["table"].long(), s["case"]["page"]
    if case["kind"] == "store":
        _plain_write(s, case, pool, table, ps)
    if case["kind"] in ("store", "read"):
        pos = s["start"].long()[:, None] + torch.arange(case["n"], device="cuda")
        inside = (pos < s["end"][:, None])[:, :, None, None]
        page, off = table.gather(1, pos // ps), pos % ps
        key, value = (torch.where(inside, _values(pool, t, case, (page, slice(None), off)), 0.0).to(_dtype(case)) for t in ("k", "v"))
        return _stored(pool, key, value) if case["kind"] == "store" else dict(key=key, value=value)
    count = torch.arange(table.shape[1], device="cuda")[None, None].expand(case["batch"], case["hkv"], -1)
    pages = _plain_select(s, case, pool, table, ps) if case["kind"] == "sparse" else None
    chosen = count if pages is None else pages
    out = _plain_attention(s, case, pool, table, ps, chosen)
    return dict(out=out) if pages is None else dict(pages=pages.to(torch.int32), out=out)


def _quantise(x, fmt):
    """Codes and scales of rows over the last dimension: the nearest multiple of the stored scale, ties to even (the quotient
    in 64 bits: a code next to a border depends on it)."""
    top = _TOP[fmt]
    scale = (x.float().abs().amax(dim=-1) / top).clamp(min=_SMALLEST_SCALE)
    codes = (x.double() / scale.double()[..., None]).round().clamp(-top, top)
    return codes.to(torch.int8), scale


def _pack(codes):
    c = codes.to(torch.int32) & 15
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)


def _values(pool, t, case, at):
    """The rows ``at`` of the pool's keys or values, in 32 bits."""
    x = pool[t + "_pages"][at]
    if case["fmt"] == "native":
        return x.float()
    if case["fmt"] == "int4":
        x = torch.stack((x & 15, x >> 4), dim=-1).flatten(-2).to(torch.int8)
        x = torch.where(x > 7, x - 16, x)
    return x.float() * pool[t + "_scale"][at][..., None]


def _plain_write(s, case, pool, table, ps):
    b, n = s["key"].shape[:2]
    pos = s["start"].long()[:, None] + torch.arange(n, device="cuda")
    rows = (torch.arange(n, device="cuda") < s["count"][:, None]).flatten().nonzero()[:, 0]
    page, off = table.gather(1, pos // ps).flatten()[rows], (pos % ps).flatten()[rows]
    for t, x in (("k", s["key"]), ("v", s["value"])):
        x = x.flatten(0, 1)[rows]                                    # [rows, Hkv, D]
        if t == "k":
            new = page[off == 0]                                     # pages that begin with these rows
            low, high = pool["k_bounds"][:, :, 0].float(), pool["k_bounds"][:, :, 1].float()
            low[new], high[new] = float("inf"), -float("inf")
            at = page[:, None, None].expand_as(x)
            pool["k_bounds"][:, :, 0] = low.scatter_reduce(0, at, x.float(), "amin").to(x.dtype)
            pool["k_bounds"][:, :, 1] = high.scatter_reduce(0, at, x.float(), "amax").to(x.dtype)
        if case["fmt"] == "native":
            pool[t + "_pages"][page, :, off] = x
        else:
            codes, scale = _quantise(x, case["fmt"])
            pool[t + "_pages"][page, :, off] = _pack(codes) if case["fmt"] == "int4" else codes
            pool[t + "_scale"][page, :, off] = scale


def _plain_select(s, case, pool, table, ps):
    """[B, Hkv, top] pages of each sequence in ascending order, -1 behind them; scores in 64 bits, since they decide."""
    b, h, d = case["batch"], case["hkv"], case["d"]
    q = s["q"].double().view(b, h, -1, d).sum(dim=2)
    bounds = pool["k_bounds"][table].double()                       # [B, pages, Hkv, 2, D]
    score = torch.maximum(bounds[:, :, :, 0] * q[:, None], bounds[:, :, :, 1] * q[:, None]).sum(dim=-1).transpose(1, 2)
    held = (s["end"].long() + ps - 1) // ps
    index = torch.arange(table.shape[1], device="cuda")
    always = (index < SINK_PAGES) | (index >= held[:, None] - RECENT_PAGES)
    score = torch.where(always[:, None], float("inf"), score)
    score = torch.where((index < held[:, None])[:, None], score, -float("inf"))
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., : case["top"]]
    best = torch.where(best < held[:, None, None], best, table.shape[1]).sort(dim=-1).values
    best = torch.where(best < table.shape[1], best, -1)
    return torch.cat((best, best.new_full((b, h, max(0, case["top"] - best.shape[-1])), -1)), dim=-1)


def _plain_attention(s, case, pool, table, ps, chosen):
    """chosen [B, Hkv, pages]: the pages of the sequence that each KV head attends to, -1 for none."""
    b, h, d = case["batch"], case["hkv"], case["d"]
    page = table[:, None].expand(-1, h, -1).gather(2, chosen.clamp(min=0))
    at = (page, torch.arange(h, device="cuda")[None, :, None])
    pos = chosen[..., None] * ps + torch.arange(ps, device="cuda")
    inside = ((chosen[..., None] >= 0) & (pos < s["end"].long()[:, None, None, None])).flatten(2)
    k, v = (_values(pool, t, case, at).flatten(2, 3) for t in ("k", "v"))   # [B, Hkv, keys, D]
    q = s["q"].float().view(b, h, -1, d)
    x = (q @ k.transpose(2, 3)) / math.sqrt(d)
    x = torch.where(inside[:, :, None], x, -float("inf"))
    p = torch.exp(x - x.amax(dim=-1, keepdim=True))
    return ((p @ v) / p.sum(dim=-1, keepdim=True)).view(b, 1, -1, d).to(_dtype(case))


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def _row_bytes(case):
    return {"native": 2 * case["d"], "int8": case["d"] + 4, "int4": case["d"] // 2 + 4}[case["fmt"]]


def work(case):
    h, d, ps = case["hkv"], case["d"], case["page"]
    if case["kind"] in ("store", "read"):
        rows = case["batch"] * case["n"] * h * (0.5 if case.get("ragged") else 1.0)
        bounds = rows / ps * 4 * d
        if case["kind"] == "read":
            return dict(bytes=2 * rows * (_row_bytes(case) + 2 * d), flops=2 * rows * d)
        # the new rows in, codes out; the codes back in, values out
        return dict(bytes=2 * rows * (2 * d + _row_bytes(case)) + bounds + 2 * rows * (_row_bytes(case) + 2 * d), flops=8 * rows * d)
    # lengths are spread over a logarithm: their mean
    lo, hi = case["min_len"], case["max_len"]
    mean = hi if hi == lo or case["batch"] == 1 else (hi + (case["batch"] - 1) * (hi - lo) / math.log(hi / lo)) / case["batch"]
    tokens, q = case["batch"] * mean * h, case["batch"] * case["hq"] * d
    if case["kind"] == "decode":
        return dict(bytes=2 * tokens * _row_bytes(case) + 4 * q, flops=4 * tokens * case["hq"] / h * d)
    kept = case["batch"] * h * min(mean, case["top"] * ps)
    return dict(bytes=2 * kept * _row_bytes(case) + tokens / ps * 4 * d + 6 * q,
                flops=4 * kept * case["hq"] / h * d + 2 * tokens / ps * d)


# ---- the definition in 64 bits, one sequence and head at a time -------------------------------------------------------
def _exact_codes(x, fmt):
    top = float(_TOP[fmt])
    largest, _ = torch.max(torch.abs(x.double()), dim=-1, keepdim=True)
    scale = torch.clamp((largest.float() / top), min=_SMALLEST_SCALE).double()
    return torch.clamp(torch.round(x.double() / scale), -top, top), scale


def _exact_held(s, t, b, h, pos):
    """Rows ``pos`` of sequence b and head h as the pool holds them."""
    case, ps = s["case"], s["case"]["page"]
    page, off = s["table"][b].long()[torch.div(pos, ps, rounding_mode="floor")], torch.remainder(pos, ps)
    x = s["pool"][t + "_pages"][:, h][page, off]
    if case["fmt"] == "native":
        return x.double()
    if case["fmt"] == "int4":
        both = x.to(torch.int64)
        both = torch.stack((both % 16, both // 16), dim=2).reshape(both.shape[0], -1)
        x = torch.remainder(both + 8, 16) - 8
    return x.double() * s["pool"][t + "_scale"][:, h][page, off].double().unsqueeze(1)


def _exact_store(s):
    case, ps, pool = s["case"], s["case"]["page"], s["pool"]
    n, ends = case["n"], s["end"].tolist()
    out = {t: torch.zeros(case["batch"], n, case["hkv"], case["d"], dtype=torch.float64, device="cuda") for t in ("key", "value")}
    bounds = pool["k_bounds"].double()
    scales = {t: None if case["fmt"] == "native" else pool[t + "_scale"].double() for t in ("k", "v")}
    for b in range(case["batch"]):
        pos = torch.arange(case["start"], ends[b], device="cuda")
        page, off = s["table"][b].long()[torch.div(pos, ps, rounding_mode="floor")], torch.remainder(pos, ps)
        for t, name in (("k", "key"), ("v", "value")):
            x = s[name][b, : len(pos)]
            if case["fmt"] == "native":
                out[name][b, : len(pos)] = x.double()
            else:
                codes, scale = _exact_codes(x, case["fmt"])
                out[name][b, : len(pos)] = codes * scale
                scales[t][page, :, off] = scale[..., 0]
        first, last = case["start"] // ps, (ends[b] - 1) // ps
        padded = torch.full(((last - first + 1) * ps, case["hkv"], case["d"]), float("nan"), dtype=torch.float64, device="cuda")
        padded[case["start"] - first * ps: ends[b] - first * ps] = s["key"][b, : len(pos)].double()
        padded = padded.view(last - first + 1, ps, case["hkv"], case["d"])
        low = torch.where(padded.isnan(), float("inf"), padded).amin(dim=1)
        high = torch.where(padded.isnan(), -float("inf"), padded).amax(dim=1)
        ids = s["table"][b, first: last + 1].long()
        if case["start"] % ps:
            low[0], high[0] = torch.minimum(low[0], bounds[ids[0], :, 0]), torch.maximum(high[0], bounds[ids[0], :, 1])
        bounds[ids, :, 0], bounds[ids, :, 1] = low, high
    res = dict(key=out["key"], value=out["value"], k_bounds=bounds)
    if case["fmt"] != "native":
        res.update(k_scale=scales["k"], v_scale=scales["v"])
    return res


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "store":
        return _exact_store(s)
    b, h, d = case["batch"], case["hkv"], case["d"]
    if case["kind"] == "read":
        pos = torch.arange(case["start"], case["start"] + case["n"], device="cuda")
        return {name: torch.stack([torch.stack([_exact_held(s, t, i, j, pos) for j in range(h)], dim=1) for i in range(b)])
                for t, name in (("k", "key"), ("v", "value"))}
    out = torch.zeros(b, 1, case["hq"], d, dtype=torch.float64, device="cuda")
    ps, group, ends = case["page"], case["hq"] // h, s["end"].tolist()
    for i in range(b):
        for j in range(h):
            pos = torch.arange(ends[i], device="cuda")
            q = s["q"][i, 0, j * group: (j + 1) * group].double()
            if case["kind"] == "sparse":
                held = (ends[i] + ps - 1) // ps
                total = q.sum(dim=0)
                bound = s["pool"]["k_bounds"][:, j][s["table"][i, :held].long()].double()
                # the larger product is the one with the bound of the sum's sign
                score = bound[:, 1] @ total.clamp(min=0) + bound[:, 0] @ total.clamp(max=0)
                score[:SINK_PAGES] = float("inf")
                score[max(0, held - RECENT_PAGES):] = float("inf")
                order = torch.argsort(-score, stable=True)[: case["top"]]
                pos = (order.sort().values[:, None] * ps + torch.arange(ps, device="cuda")).flatten()
                pos = pos[pos < ends[i]]
            w = torch.softmax((_exact_held(s, "k", i, j, pos) @ q.T) / math.sqrt(d), dim=0)
            out[i, 0, j * group: (j + 1) * group] = w.T @ _exact_held(s, "v", i, j, pos)
    return dict(out=out) if case["kind"] == "decode" else dict(pages=None, out=out)
