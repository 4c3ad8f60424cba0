"""Plain restatements of libserving_ops' operators (include/serving_ops.h) - TEST INFRASTRUCTURE ONLY.

The stored bytes are defined by fp32 operations, so the cache's format is restated in fp32 and compared bit for bit;
everything else is computed in 64 bits.  All on the CPU, one sequence and head at a time, byte by byte.
"""
from __future__ import annotations

import torch


def rotate32(x, cos_sin, positions, interleaved):
    """fp32 rotation of heads x [T, H, D], every product rounded before the sum."""
    n = cos_sin.shape[1] // 2
    x = x.float().clone()
    known = (positions >= 0) & (positions < cos_sin.shape[0])
    rows = cos_sin[positions.clamp(0, max(0, cos_sin.shape[0] - 1))].clone() if cos_sin.shape[0] else torch.zeros(len(positions), 2 * n)
    rows[~known] = float("nan")
    cos, sin = rows[:, None, :n], rows[:, None, n:]
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    p, q = x[..., a].clone(), x[..., b].clone()
    x[..., a] = p * cos - q * sin
    x[..., b] = q * cos + p * sin
    return x


def rotate64(x, cos_sin, positions, interleaved):
    """The same in 64 bits, and the size |a cos| + |b sin| that an fp32 rotation's error is relative to."""
    n = cos_sin.shape[1] // 2
    x = x.double().clone()
    size = x.abs()
    cos, sin = cos_sin[positions, None, :n].double(), cos_sin[positions, None, n:].double()
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    p, q = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = p * cos - q * sin, q * cos + p * sin
    size[..., a], size[..., b] = (p * cos).abs() + (q * sin).abs(), (q * cos).abs() + (p * sin).abs()
    return x, size


def quantise(x):
    """fp32 heads [..., D] -> codes (int), scale and least (fp16), by the format's definition."""
    least = x.amin(-1).half()
    scale = ((x.amax(-1) - least.float()) * torch.tensor(1 / 15, dtype=torch.float32)).half()
    held = torch.isfinite(least) & torch.isfinite(scale) & torch.isfinite(x).all(-1)
    codes = torch.zeros(x.shape, dtype=torch.int64)
    on = held & (scale > 0)
    codes[on] = torch.round((x[on] - least[on].float()[..., None]) / scale[on].float()[..., None]).clamp(0, 15).long()
    nan = torch.tensor(float("nan"), dtype=torch.float16)
    return codes, torch.where(held, scale, nan), torch.where(held, least, nan)


def store(cache, head_size, slots, key, value):
    """Writes fp32 heads key, value [T, H, D] into the slots of a CPU cache, byte by byte."""
    blocks, heads, size = cache.shape
    p = size // (head_size + 8)
    raw = cache.numpy()
    halves = cache.view(torch.float16).numpy()
    for which, x in enumerate((key, value)):
        codes, scale, least = quantise(x)
        codes, scale, least = codes.numpy(), scale.numpy(), least.numpy()
        for t, slot in enumerate(slots.tolist()):
            if not 0 <= slot < blocks * p:
                continue
            block, at = divmod(slot, p)
            for h in range(heads):
                pairs = codes[t, h, 0::2] | (codes[t, h, 1::2] << 4)
                if which == 0:
                    raw[block, h, at * (head_size // 2):(at + 1) * (head_size // 2)] = pairs
                else:
                    for piece in range(head_size // 8):
                        start = p * head_size // 2 + (at // 16) * 8 * head_size + piece * 64 + (at % 16) * 4
                        raw[block, h, start:start + 4] = pairs[4 * piece:4 * piece + 4]
                word = (p * head_size + which * 4 * p) // 2 + 2 * at
                halves[block, h, word], halves[block, h, word + 1] = scale[t, h], least[t, h]


def values(cache, head_size, slots, code=None):
    """What slots stand for, in 64 bits: key, value [n, H, D], and the values' scales [n, H] (zeros outside the cache);
    what they would with `code` in every element, if given."""
    blocks, heads, size = cache.shape
    p = size // (head_size + 8)
    inside = (slots >= 0) & (slots < blocks * p)
    s = torch.where(inside, slots, torch.zeros_like(slots))
    block, at = s // p, s % p
    el = torch.arange(head_size)
    h = torch.arange(heads)
    k_byte = at[:, None] * (head_size // 2) + el // 2
    v_byte = p * head_size // 2 + (at[:, None] // 16) * 8 * head_size + (el // 8) * 64 + (at[:, None] % 16) * 4 + (el % 8) // 2
    halves = cache.view(torch.float16)
    found, scales = [], []
    for which, byte in enumerate((k_byte, v_byte)):
        raw = cache[block[:, None, None], h[None, :, None], byte[:, None, :]].long()
        stored = (raw >> (4 * (el % 2))) & 15
        word = (p * head_size + which * 4 * p) // 2 + 2 * at
        scale = halves[block[:, None], h[None], word[:, None]].double()
        least = halves[block[:, None], h[None], word[:, None] + 1].double()
        x = least[..., None] + (stored.double() if code is None else code) * scale[..., None]
        x = x.expand(stored.shape)
        found.append(torch.where(inside[:, None, None], x, torch.zeros_like(x)))
        scales.append(scale)
    return found[0], found[1], scales[1]


def attend(query, cache, tables, lens, start, scale, window, repaired):
    """64-bit attention and, for each output element, how far a kernel may be from it that
      rounds p_j vscale_j to fp16 once (a half step: 2^-11 of it; below fp16's normal numbers 2^-25 of 2^-15 of twice the
      largest vscale), times at most 15 codes, or 7.5 where what the roundings took is given back at the middle,
      sums products of a head in fp32: D + 8 roundings of at most scale * sum |q| (15 kscale + |kleast|) each, which
      moves every probability by twice that relatively, and the exponential by a few steps of it,
      and rounds the result once.
    (tables, lens, start: CPU int tensors; rows of no sequence are NaN in both.)"""
    t, heads, d = query.shape
    kv = cache.shape[1]
    p = cache.shape[2] // (d + 8)
    group = heads // kv
    eps = torch.finfo(query.dtype).eps / 2
    out = torch.full((t, heads, d), float("nan"), dtype=torch.float64)
    tol = out.clone()
    for b in range(len(lens)):
        n, r0 = min(int(lens[b]), tables.shape[1] * p), int(start[b])
        m = int(start[b + 1]) - r0
        if m == 0:
            continue
        j = torch.arange(max(n, 0))
        slots = tables[b].long()[j // p] * p + j % p
        k, v, vs = values(cache, d, slots)
        i = torch.arange(m)[:, None] + (n - m)
        sees = j[None] <= i
        if window:
            sees &= j[None] > i - window
        for h in range(heads):
            q = query[r0:r0 + m, h].double()
            kk, vv = k[:, h // group], v[:, h // group]
            x = torch.where(sees, (q @ kk.T) * scale, torch.tensor(-float("inf"), dtype=torch.float64))
            top = x.amax(1, keepdim=True) if n else torch.zeros(m, 1, dtype=torch.float64)
            top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
            e = torch.where(sees, torch.exp(x - top), torch.zeros_like(x))
            z = e.sum(1, keepdim=True)
            any_ = sees.any(1, keepdim=True) if n else torch.zeros(m, 1, dtype=torch.bool)
            o = torch.zeros(m, d, dtype=torch.float64)
            for r in range(m):  # (row by row: what a row does not see may be NaN)
                if any_[r]:
                    o[r] = e[r, sees[r]] @ vv[sees[r]] / z[r]
            out[r0:r0 + m, h] = o
            if n:
                size = abs(scale) * q.abs().sum(1, keepdim=True) * torch.where(sees, kk.abs().amax(1)[None], torch.zeros_like(x)).amax(1, keepdim=True)
                moved = 2 * (2 * (d + 8) * 2.0**-24 * 3 * size + 2.0**-20)
                seen = torch.where(sees, vs[None, :, h // group], torch.zeros_like(x))
                rounded = (e * seen).sum(1, keepdim=True) / z * 2.0**-11 + n * 2.0**-39 * seen.amax(1, keepdim=True) / z
                spread = torch.where(sees, vv.abs().amax(1)[None], torch.zeros_like(x)).amax(1, keepdim=True)
                err = moved * 2 * spread + rounded * (7.5 if repaired else 15.0) + 2.0**-20 * spread
                tol[r0:r0 + m, h] = err + eps * (o.abs() + err) + 2.0**-25
            else:
                tol[r0:r0 + m, h] = 0
    return out, tol


def attend_counted(query, cache, tables, lens, start, scale, window):
    """64-bit attention and how far a kernel may be from it, counted key by key, so that keys of very different values
    may stand beside each other.  The kernel
      has e_j (the exponential of score j) off by 2 (d + 8) roundings of fp32 of a score's parts, and by 2^-18 for the
      exponential and for the sum of a score and what it is held against: sum_j p_j |v_j - o| of that,
      holds w_j = e_j vscale_j in fp16, in a unit that has the largest w_j of the row at 2^6 or more: half a step, 2^-11 of
      w_j, or 2^-25 of the unit below fp16's normal numbers, times its code; for fp16 results times the code's distance from one that
      stands between the least value and 0, with which the rounded weight is taken off again.  A product with a code may
      lose 2^-21 of it,
      takes sums in fp32: of 64 matrix instructions, of what is set aside every 1024 keys, of 40 waves and pieces, each
      off by a step of 2^-23 of the sum of absolute values,
      and rounds the result once.
    (Rows of no sequence are NaN in both.)"""
    t, heads, d = query.shape
    p = cache.shape[2] // (d + 8)
    group = heads // cache.shape[1]
    half = query.dtype == torch.float16
    eps, least_step = torch.finfo(query.dtype).eps / 2, 2.0**-25 if half else 2.0**-60
    out = torch.full((t, heads, d), float("nan"), dtype=torch.float64)
    tol = out.clone()
    for b in range(len(lens)):
        n, r0 = min(int(lens[b]), tables.shape[1] * p), int(start[b])
        m = int(start[b + 1]) - r0
        j = torch.arange(max(n, 0))
        slots = tables[b].long()[j // p] * p + j % p
        keys, values_, scales = values(cache, d, slots)
        leasts = values(cache, d, slots, 0.0)[1]
        for r in range(m):
            last = n - m + r
            see = j[max(0, last + 1 - window if window else 0):max(0, last + 1)]
            if not len(see):
                out[r0 + r] = tol[r0 + r] = 0
                continue
            for h in range(heads):
                q = query[r0 + r, h].double()
                k, v, vs, least = (x[see, h // group] for x in (keys, values_, scales, leasts))
                pr = torch.softmax((k @ q) * scale, 0)
                o = pr @ v
                size = abs(scale) * q.abs().sum() * k.abs().max()
                moved = 2 * (2 * (d + 8) * 2.0**-24 * 3 * size + 2.0**-18)
                codes = pr @ (v - least)
                apart = pr @ torch.minimum(v.abs() + least.abs(), 15 * vs[:, None]) if half else codes
                sums = codes + 3 * (pr @ least.abs())
                err = moved * (pr @ (v - o).abs()) + 2.0**-11 * apart + 2.0**-21 * codes
                err += 15 * len(see) * (2.0**-31 * (pr * vs).max() + 2.0**-55)
                err += (104 + len(see) / 1024) * 2.0**-23 * (sums + o.abs())
                out[r0 + r, h] = o
                tol[r0 + r, h] = err + eps * (o.abs() + err) + least_step
    return out, tol


def logprobs(logits, tokens, top):
    """64-bit log probabilities, entropy, the most likely tokens (a stable order: the lowest index first)."""
    x = logits.double()
    logp = torch.log_softmax(x, 1)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
    entropy = torch.where(torch.isnan(logp).any(1), torch.full_like(entropy, float("nan")), entropy)
    rank = torch.where(torch.isnan(x), torch.full_like(x, float("inf")), x)
    # a NaN above +inf: two stable sorts, the finer order first
    at = torch.sort(rank, dim=1, descending=True, stable=True).indices
    nan = torch.isnan(x).gather(1, at)
    at = at.gather(1, torch.sort(nan.int(), dim=1, descending=True, stable=True).indices)[:, :top]
    inside = (tokens >= 0) & (tokens < x.shape[1])
    given = logp.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    given = torch.where(inside, given, torch.full_like(given, float("nan")))
    return given, entropy, at, logp.gather(1, at)
