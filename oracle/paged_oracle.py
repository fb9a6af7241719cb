"""TEST INFRASTRUCTURE ONLY — the paged key/value cache's operators from their definitions, in 64 bits, on any device.

Nothing shipped imports this file.  A pool here is a dict of the tensors of a layer (``k_pages``, ``v_pages``, ``k_scale``,
``v_scale``, ``k_bounds``); loops go over sequences, heads and rows, so sizes stay small."""
from __future__ import annotations

import math

import torch

TOP = {"int8": 127, "int4": 7}
SMALLEST_SCALE = 2.0 ** -100


def quantise(x, fmt):
    """Rows over the last dimension -> (integer codes, fp32 scales): the nearest multiple of the scale, ties to even."""
    top = TOP[fmt]
    step = torch.tensor(1.0, device=x.device) / torch.tensor(float(top), device=x.device)   # fp32
    scale = torch.clamp(x.float().abs().amax(-1) * step, min=SMALLEST_SCALE)
    finite = torch.isfinite(x.double()).all(-1)
    scale = torch.where(finite, scale, float("nan"))
    codes = torch.where(finite[..., None], (x.double() / scale.double()[..., None]).round(), 0.0)
    return codes.to(torch.int64), scale


def pack4(codes):
    return ((codes[..., 0::2] & 15) | ((codes[..., 1::2] & 15) << 4)).to(torch.uint8)


def unpack4(b):
    c = torch.stack((b & 15, b >> 4), -1).flatten(-2).to(torch.int64)
    return torch.where(c > 7, c - 16, c)


def values(pool, t, fmt, page, head, rows):
    """fp64 rows of one page and head as the attention sees them."""
    x = pool[t + "_pages"][page, head, rows]
    if fmt == "native":
        return x.double()
    x = unpack4(x) if fmt == "int4" else x
    return x.double() * pool[t + "_scale"][page, head, rows].double()[..., None]


def write(pool, fmt, key, value, table, positions, counts):
    """In place, row by row."""
    num_pages, ps = pool["k_pages"].shape[0], pool["k_pages"].shape[2]
    for b in range(key.shape[0]):
        for i in range(counts[b]):
            pos = positions[b] + i
            if positions[b] < 0 or pos // ps >= table.shape[1]:
                continue
            page, off = int(table[b, pos // ps]), pos % ps
            if not 0 <= page < num_pages:
                continue
            for t, x in (("k", key[b, i]), ("v", value[b, i])):
                if fmt == "native":
                    pool[t + "_pages"][page, :, off] = x
                else:
                    codes, scale = quantise(x, fmt)
                    pool[t + "_pages"][page, :, off] = pack4(codes) if fmt == "int4" else codes.to(torch.int8)
                    pool[t + "_scale"][page, :, off] = scale
            if pool.get("k_bounds") is not None:
                x = key[b, i]
                if off == 0:
                    pool["k_bounds"][page, :, 0], pool["k_bounds"][page, :, 1] = x, x
                else:
                    pool["k_bounds"][page, :, 0] = torch.minimum(pool["k_bounds"][page, :, 0], x)
                    pool["k_bounds"][page, :, 1] = torch.maximum(pool["k_bounds"][page, :, 1], x)


def read(pool, fmt, dtype, table, starts, n, ends):
    num_pages, hkv, ps = pool["k_pages"].shape[:3]
    d = pool["k_pages"].shape[3] * (2 if fmt == "int4" else 1)
    out = {t: torch.zeros(len(starts), n, hkv, d, dtype=dtype, device=table.device) for t in "kv"}
    for b, s in enumerate(starts):
        for i in range(n):
            pos = s + i
            if pos < 0 or pos // ps >= table.shape[1] or (ends is not None and pos >= ends[b]):
                continue
            page = int(table[b, pos // ps])
            if 0 <= page < num_pages:
                for t in "kv":
                    x = pool[t + "_pages"][page, :, pos % ps]
                    if fmt != "native":   # the value is rounded to fp32, then to the 16-bit type
                        x = (unpack4(x) if fmt == "int4" else x).float() * pool[t + "_scale"][page, :, pos % ps, None]
                    out[t][b, i] = x.to(dtype)
    return out["k"], out["v"]


def attention(q, pool, fmt, table, lens, pages=None, sm_scale=None):
    """q [B, Hq, D] -> (o [B, Hq, D] fp64, lse [B, Hq] fp64 base 2, spread [B, Hq, D] = sum_j p_j |v_j|, size [B, Hq] =
    max_j sm_scale sum_d |q_d k_jd|, vmax [B, Hq] = max |v|): the last three are what error bounds are made of."""
    b, hq, d = q.shape
    num_pages, hkv, ps = pool["k_pages"].shape[:3]
    g = hq // hkv
    sm_scale = 1.0 / math.sqrt(d) if sm_scale is None else sm_scale
    o = torch.zeros(b, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((b, hq), -float("inf"), dtype=torch.float64, device=q.device)
    spread, size, vmax = torch.zeros_like(o), torch.zeros_like(lse), torch.zeros_like(lse)
    for i in range(b):
        n = max(0, min(lens[i], table.shape[1] * ps))
        held = (n + ps - 1) // ps
        for h in range(hkv):
            listed = range(held) if pages is None else pages[i][h]
            k, v = [], []
            for e in listed:
                if not 0 <= e < held or not 0 <= int(table[i, e]) < num_pages:
                    continue
                rows = slice(0, min(ps, n - e * ps))
                k.append(values(pool, "k", fmt, int(table[i, e]), h, rows))
                v.append(values(pool, "v", fmt, int(table[i, e]), h, rows))
            if not k:
                continue
            k, v, x = torch.cat(k), torch.cat(v), q[i, h * g:(h + 1) * g].double()
            s = x @ k.T * sm_scale
            w = torch.softmax(s, -1)
            o[i, h * g:(h + 1) * g] = w @ v
            spread[i, h * g:(h + 1) * g] = w @ v.abs()
            size[i, h * g:(h + 1) * g] = (x.abs() @ k.abs().T * sm_scale).amax(-1)
            vmax[i, h * g:(h + 1) * g] = v.abs().amax()
            lse[i, h * g:(h + 1) * g] = torch.logsumexp(s, -1) / math.log(2.0)
    return o, lse, spread, size, vmax


def select(q, pool, table, lens, budget, sink, recent):
    """q [B, Hq, D] -> lists [B][Hkv] of `budget` pages, ascending, -1 behind the last."""
    b, hq, d = q.shape
    num_pages, hkv, ps = pool["k_pages"].shape[:3]
    res = []
    for i in range(b):
        held = min((max(lens[i], 0) + ps - 1) // ps, table.shape[1])
        res.append([])
        for h in range(hkv):
            u = q[i, h * (hq // hkv):(h + 1) * (hq // hkv)].double().sum(0)
            score = []
            for e in range(held):
                page = int(table[i, e])
                if e < sink or e >= held - recent:
                    score.append(float("inf"))
                elif not 0 <= page < num_pages:
                    score.append(-float("inf"))
                else:
                    lo, hi = pool["k_bounds"][page, h].double()
                    score.append(float(torch.maximum(u * lo, u * hi).sum()))
            best = sorted(sorted(range(held), key=lambda e: (-score[e], e))[:budget])
            res[-1].append(best + [-1] * (budget - len(best)))
    return res
