"""What is timed of the operators that a generating step needs around its W4A16 products: appending rotated keys and
values to a paged cache that holds them in 4 bits, attention over that cache, and log probabilities of given tokens.

The cache is one uint8 tensor [blocks, kv heads, P (D + 8)] with P tokens a block and D elements a head.  A block's
part of one head holds, one behind the other,
  the keys    [P][D / 2]          element d of a token in bits 4 (d % 2) .. of byte d / 2,
  the values  [P / 16][D / 8][16][4]   the same bytes, cut into pieces of 4 (8 elements), 16 tokens of a piece together,
  parameters  [2 (keys, values)][P][2 (scale, least)] fp16,
and an element stands for `least + code * scale`.
"""
import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SPARE = 3  # blocks of a pool that no sequence uses


def listed():
    return [
        # one token of one sequence, the shape of a 7B layer with a head of keys for each head of queries
        dict(name="append 1", op="append", dtype="fp16", tokens=1, prompts=0, heads=32, kv=32, head=128, page=16, rotary=128,
             interleaved=False, padded=0, positions=4096),
        # a decode batch padded to a captured size, a 70B layer's grouped heads
        dict(name="append batch 64", op="append", dtype="fp16", tokens=64, prompts=0, heads=64, kv=8, head=128, page=16,
             rotary=128, interleaved=False, padded=5, positions=8192),
        # short prompts of odd lengths, small heads, neighbouring pairs rotated over half a head
        dict(name="append short prompts", op="append", dtype="bf16", tokens=777, prompts=5, heads=12, kv=4, head=64, page=32,
             rotary=32, interleaved=True, padded=0, positions=2048),
        # a chunk of a long prompt
        dict(name="append prompt 8192", op="append", dtype="bf16", tokens=8192, prompts=1, heads=64, kv=8, head=128, page=64,
             rotary=128, interleaved=False, padded=0, positions=32768),
        # the first step behind a short prompt: one sequence, every head with keys of its own
        dict(name="attend 1 x 129", op="attend", dtype="fp16", seqs=1, queries=1, shortest=129, longest=129, heads=32, kv=32,
             head=128, page=16, window=0),
        # a decode batch of mixed lengths, heads of keys not shared
        dict(name="attend 64 x 4096", op="attend", dtype="fp16", seqs=64, queries=1, shortest=97, longest=4096, heads=32, kv=32,
             head=128, page=16, window=0),
        # few long sequences, grouped heads
        dict(name="attend 8 x 65536", op="attend", dtype="bf16", seqs=8, queries=1, shortest=30011, longest=65536, heads=64,
             kv=8, head=128, page=64, window=0),
        # drafted tokens checked together, a sliding window, small heads
        dict(name="attend drafts", op="attend", dtype="bf16", seqs=16, queries=5, shortest=37, longest=2999, heads=28, kv=4,
             head=64, page=32, window=1024),
        # chunks of two prompts behind what the cache holds of them
        dict(name="attend prompt 2048", op="attend", dtype="bf16", seqs=2, queries=2048, shortest=2500, longest=8192, heads=64,
             kv=8, head=128, page=64, window=0),
        # greedy decoding of one sequence
        dict(name="logprobs 1", op="logprobs", dtype="fp16", rows=1, vocab=32000, top=1),
        # a decode batch over a large odd vocabulary, alternatives asked for
        dict(name="logprobs 64", op="logprobs", dtype="bf16", rows=64, vocab=128011, top=5),
        # a prompt scored token by token
        dict(name="logprobs 4096", op="logprobs", dtype="fp32", rows=4096, vocab=32000, top=20),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    head = rng.choice([64, 128])
    kv = rng.choice([1, 2, 3, 4, 8, 16, 32])
    group = rng.choice([g for g in (1, 2, 3, 4, 6, 7, 8, 16) if g * kv <= 64])
    return dict(heads=kv * group, kv=kv, head=head, page=rng.choice([16, 32, 64, 128]))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "logprobs"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "append":
        c = dict(op=op, dtype=dtype, **_heads(rng))
        most = 8192 * 80 * 128 // ((c["heads"] + 2 * c["kv"]) * c["head"])
        tokens = _spread(rng, 1, min(8192, most))
        prompts = rng.choice([0, rng.randint(1, 8)]) if tokens <= 256 else rng.randint(1, 8)
        c.update(tokens=tokens, prompts=min(prompts, tokens), rotary=rng.choice([c["head"], c["head"] // 2]),
                 interleaved=rng.random() < 0.25, padded=rng.randint(0, tokens // 4) if not prompts else 0,
                 positions=rng.choice([16384, 32768]))
        return c
    if op == "logprobs":
        vocab = _spread(rng, 1000, 131072)
        rows = _spread(rng, 1, min(4096, 4096 * 32000 // vocab))
        return dict(op=op, dtype=rng.choice(["fp16", "bf16", "fp32"]), rows=rows, vocab=vocab, top=rng.randint(0, 20))
    c = dict(op=op, dtype=dtype, **_heads(rng))
    kind = rng.choice(["decode", "decode", "drafts", "prompt"])
    longest = _spread(rng, 1, 65536)
    if kind == "prompt":
        queries = _spread(rng, 33, 2048)
        longest = max(queries, min(longest, 8192))
        queries = min(queries, max(17, int(5e11 / (4.0 * longest * c["heads"] * c["head"]))))
        one = 4.0 * queries * longest * c["heads"] * c["head"]
        seqs = _spread(rng, 1, max(1, min(8, int(5e11 / one))))
    else:
        queries = 1 if kind == "decode" else rng.randint(2, 16)
        longest = max(longest, queries)
        one = longest * c["kv"] * (c["head"] + 8) * max(1.0, queries * c["heads"] / c["kv"] / 16)
        seqs = _spread(rng, 1, max(1, min(128, int(4.0e8 / one))))
    shortest = max(queries, int(longest * rng.uniform(0.05, 1.0)))
    window = rng.choice([0, 0, 0, _spread(rng, 16, 4096)])
    c.update(seqs=seqs, queries=queries, shortest=shortest, longest=longest, window=window)
    return c


def _lengths(c):
    """Lengths of the sequences (the last one the longest) and how many queries each has, from the case alone."""
    n = c["seqs"]
    lens = [c["shortest"] + int((c["longest"] - c["shortest"]) * ((i * 0.6180339887) % 1.0)) for i in range(n - 1)] + [c["longest"]]
    if c["queries"] <= 16:
        return lens, [c["queries"]] * n
    return lens, [max(1, int(c["queries"] * (0.5 + 0.5 * ((i * 0.7548776662) % 1.0)))) for i in range(n - 1)] + [c["queries"]]


def _seen(c):
    """Pairs of a query and a key that it sees, and keys that some query of their sequence sees."""
    pairs = keys = 0
    for n, q in zip(*_lengths(c)):
        first = n - q + 1  # how many keys the first query sees without a window
        w = c["window"] or n
        short = max(0, min(q, w - first + 1))  # queries that see less than a window
        pairs += short * first + short * (short - 1) // 2 + (q - short) * w
        keys += min(n, q - 1 + w)
    return pairs, keys


def work(c):
    if c["op"] == "append":
        size = 2
        live = c["tokens"] - c["padded"]
        rows = c["tokens"] * 2 * c["heads"] * c["head"] * size  # queries in and out
        rows += live * 2 * c["kv"] * c["head"] * size  # keys and values in
        stored = live * c["kv"] * (c["head"] + 8)
        back = c["tokens"] * 2 * c["kv"] * c["head"] * size  # read back as values
        tables = c["tokens"] * (16 + 4 * c["rotary"])
        return {"bytes": rows + 2 * stored + back + tables,
                "flops": c["tokens"] * (c["heads"] + c["kv"]) * c["rotary"] * 3 + live * 2 * c["kv"] * c["head"] * 6}
    if c["op"] == "attend":
        pairs, keys = _seen(c)
        queries = sum(_lengths(c)[1])
        return {"bytes": keys * c["kv"] * (c["head"] + 8) + 4 * queries * c["heads"] * c["head"],
                "flops": 4 * pairs * c["heads"] * c["head"]}
    size = 4 if c["dtype"] == "fp32" else 2
    return {"bytes": c["rows"] * (c["vocab"] * size + 8 + 8 + 12 * c["top"]), "flops": 6 * c["rows"] * c["vocab"]}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _quantise(x):
    """fp32 [..., D] -> codes, scale, least of the cache's format (fp32 arithmetic, parameters rounded to fp16)."""
    least = x.amin(-1).half().float()
    scale = ((x.amax(-1) - least) / 15.0).half().float()
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    codes = torch.round((x - least[..., None]) / safe[..., None]).clamp(0, 15)
    codes = torch.where(scale[..., None] > 0, codes, torch.zeros_like(codes))
    return codes.to(torch.uint8), scale, least


def _parts(cache, head):
    """Views of a cache: keys [N, H, P, D / 2], values [N, H, P / 16, D / 8, 16, 4], parameters [N, H, 2, P, 2]."""
    n, h, size = cache.shape
    p = size // (head + 8)
    half = p * head // 2
    keys = cache[:, :, :half].view(n, h, p, head // 2)
    values = cache[:, :, half:2 * half].view(n, h, p // 16, head // 8, 16, 4)
    params = cache.view(torch.float16)[:, :, half:].view(n, h, 2, p, 2)
    return keys, values, params


def _unpack(b):
    """bytes [..., n] -> codes [..., 2 n]"""
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _store(cache, head, slots, k, v):
    """Quantises fp32 rows k, v [T, H, D] into the cache's slots."""
    keys, values, params = _parts(cache, head)
    p = params.shape[3]
    block, at = slots // p, slots % p
    kc, ks, kl = _quantise(k)
    vc, vs, vl = _quantise(v)
    pack = lambda c: c[..., 0::2] | (c[..., 1::2] << 4)  # noqa: E731
    keys[block, :, at] = pack(kc)
    values[block, :, at // 16, :, at % 16] = pack(vc).view(*vc.shape[:2], head // 8, 4)
    params[block, :, 0, at] = torch.stack([ks, kl], -1).half()
    params[block, :, 1, at] = torch.stack([vs, vl], -1).half()


def prepare(c, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = TYPES[c["dtype"]]
    if c["op"] == "logprobs":
        logits = torch.randn(c["rows"], c["vocab"], generator=gen, device=dev) * 2.5
        # a few likely tokens in each row, as a trained model has them, and the rows' own sharpness
        likely = torch.randint(c["vocab"], (c["rows"], 8), generator=gen, device=dev)
        lift = torch.rand(c["rows"], 8, generator=gen, device=dev) * 14
        logits.scatter_add_(1, likely, lift)
        tokens = torch.where(torch.rand(c["rows"], generator=gen, device=dev) < 0.7, likely[:, 0],
                             torch.randint(c["vocab"], (c["rows"], ), generator=gen, device=dev))
        return dict(case=c, logits=logits.to(dtype), tokens=tokens)
    d, p, kv = c["head"], c["page"], c["kv"]
    if c["op"] == "append":
        t = c["tokens"]
        qkv = torch.randn(t, (c["heads"] + 2 * kv) * d, generator=gen, device=dev) * torch.exp(
            0.7 * torch.randn((c["heads"] + 2 * kv) * d, generator=gen, device=dev))
        qkv = qkv.to(dtype)
        q, k, v = qkv.split([c["heads"] * d, kv * d, kv * d], 1)
        inv = 10000.0**(-torch.arange(0, c["rotary"], 2, device=dev, dtype=torch.float64) / c["rotary"])
        angle = torch.arange(c["positions"], device=dev, dtype=torch.float64)[:, None] * inv
        cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float()
        if c["prompts"]:  # whole chunks of sequences: consecutive positions in blocks of their own
            each = [t // c["prompts"] + (i < t % c["prompts"]) for i in range(c["prompts"])]
            starts = torch.randint(0, c["positions"] - max(each) + 1, (len(each), ), generator=gen, device=dev)
            of = torch.repeat_interleave(torch.arange(len(each), device=dev), torch.tensor(each, device=dev))
            first = torch.cumsum(torch.tensor([0] + each[:-1], device=dev), 0)
            positions = starts[of] + torch.arange(t, device=dev) - first[of]
            wide = max(each) // p + 2
            table = torch.randperm(len(each) * wide + SPARE, generator=gen, device=dev)[:len(each) * wide].view(len(each), wide)
            blocks = len(each) * wide + SPARE
            slots = table[of, positions // p - starts[of] // p] * p + positions % p
        else:  # one token for each sequence; the last `padded` rows belong to none
            positions = torch.randint(0, c["positions"], (t, ), generator=gen, device=dev)
            blocks = 4 * t + SPARE
            slots = torch.randperm(blocks, generator=gen, device=dev)[:t] * p + positions % p
            slots[t - c["padded"]:] = -1
        cache = torch.zeros(blocks, kv, p * (d + 8), dtype=torch.uint8, device=dev)
        live = torch.arange(t - c["padded"], device=dev)
        return dict(case=c, query=q.view(t, c["heads"], d), key=k.view(t, kv, d), value=v.view(t, kv, d), cos_sin=cos_sin,
                    positions=positions, slots=slots, cache=cache, live=live)
    lens, queries = _lengths(c)
    wide = -(-c["longest"] // p)
    used = [-(-n // p) for n in lens]
    blocks = sum(used) + SPARE
    order = torch.randperm(blocks, generator=gen, device=dev).to(torch.int32)
    col = torch.arange(wide, device=dev)[None]
    first = torch.cumsum(torch.tensor([0] + used[:-1], device=dev), 0)[:, None]
    inside = col < torch.tensor(used, device=dev)[:, None]
    tables = torch.where(inside, order[(first + col).clamp_(max=blocks - 1)], torch.zeros((), dtype=torch.int32, device=dev))
    cache = torch.zeros(blocks, kv, p * (d + 8), dtype=torch.uint8, device=dev)
    gain = torch.exp(0.7 * torch.randn(2, kv, d, generator=gen, device=dev))
    gain[0] *= 0.7
    step = max(1, (1 << 26) // (p * kv * d))
    for b in range(0, blocks, step):  # (quantised in pieces: a whole cache in 32 bits would not fit three times)
        e = min(blocks, b + step)
        kk, vv = torch.randn(2, (e - b) * p, kv, d, generator=gen, device=dev) * gain[:, None]
        _store(cache, d, torch.arange(b * p, e * p, device=dev), kk, vv)
    total = sum(queries)
    query = (torch.randn(total, c["heads"], d, generator=gen, device=dev) * 1.2).to(dtype)
    start = torch.cumsum(torch.tensor([0] + queries, device=dev), 0).to(torch.int32)
    return dict(case=c, query=query, cache=cache, tables=tables.contiguous(), lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                start=start, scale=d**-0.5)


# ---------------------------------------------------------------------------------------------------------------
# the operators in their plain form
# ---------------------------------------------------------------------------------------------------------------
def _rotate(x, cos, sin, interleaved):
    """Rotates the first 2 n elements of fp32 heads x [T, H, D]; cos, sin [T, 1, n]."""
    n = cos.shape[-1]
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _plain_append(s):
    c = s["case"]
    cos, sin = s["cos_sin"][s["positions"]][:, None].chunk(2, -1)
    query = _rotate(s["query"].float(), cos, sin, c["interleaved"]).to(s["query"].dtype)
    live = s["live"]
    slots = s["slots"][live]
    key = _rotate(s["key"].float(), cos, sin, c["interleaved"])[live]
    _store(s["cache"], c["head"], slots, key, s["value"].float()[live])
    keys, values, params = _parts(s["cache"], c["head"])
    block, at = slots // c["page"], slots % c["page"]
    back = []
    for i, codes in enumerate((keys[block, :, at], values[block, :, at // 16, :, at % 16].flatten(2))):
        scale, least = params[block, :, i, at].float().unbind(-1)
        rows = torch.zeros_like(s["key"], memory_format=torch.contiguous_format)
        rows[live] = (least[..., None] + _unpack(codes).float() * scale[..., None]).to(rows.dtype)
        back.append(rows)
    return query, back[0], back[1]


def _plain_attend(s):
    c = s["case"]
    d, kv, group = c["head"], c["kv"], c["heads"] // c["kv"]
    keys, values, params = _parts(s["cache"], d)
    tables, lens = s["tables"].long(), s["lens"].long()
    b, most = tables.shape[0], tables.shape[1] * c["page"]
    scale, least = params[tables].float().unbind(-1)  # [B, W, H, 2, P]
    flat = lambda t: t.transpose(1, 2).reshape(b, kv, most, -1)  # noqa: E731
    k = _unpack(keys[tables]).float() * scale[:, :, :, 0, :, None] + least[:, :, :, 0, :, None]
    v = _unpack(values[tables].transpose(-2, -3).flatten(-2)).flatten(3, 4).float()  # [B, W, H, P, D]
    v = v * scale[:, :, :, 1, :, None] + least[:, :, :, 1, :, None]
    k, v = flat(k), flat(v)
    start = s["start"].long()
    many = start[1:] - start[:-1]
    i = torch.arange(c["queries"], device=k.device)
    rows = (start[:-1, None] + i).clamp(max=s["query"].shape[0] - 1)
    q = s["query"][rows].float().view(b, -1, kv, group, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)
    at = (lens - many)[:, None] + i  # the position of each query
    j = torch.arange(most, device=k.device)
    sees = (j <= at[..., None]) & (j < lens[:, None, None])
    if c["window"]:
        sees &= j > at[..., None] - c["window"]
    x = (torch.matmul(q, k.transpose(2, 3)) * s["scale"]).view(b, kv, group, -1, most)
    x.masked_fill_(~sees[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True).clamp(min=-1e30)
    x.exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, kv, -1, most), v).view(b, kv, group, -1, d) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, -1, c["heads"], d).to(s["query"].dtype)
    of = torch.repeat_interleave(torch.arange(b, device=k.device), many, output_size=s["query"].shape[0])
    return o[of, torch.arange(s["query"].shape[0], device=k.device) - start[of]]


def _ranked(x, n):
    """Where the n largest of each row stand, the largest first: the lowest index first among equals."""
    bits = x.float().view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))  # rises with the number; both zeros alike
    key = order * (1 << 20) + ((1 << 20) - 1 - torch.arange(x.shape[1], device=x.device))
    return ((1 << 20) - 1) - (torch.topk(key, n, dim=1).values & ((1 << 20) - 1))


def _plain_logprobs(s):
    x = s["logits"].float()
    y = x - x.amax(1, keepdim=True)
    p = y.exp()
    total = p.sum(1, dtype=torch.float64)  # (next to 1 where one token has nearly all: 32 bits lose the rest)
    log_total = total.log()
    entropy = (log_total - (p * y).sum(1) / total).float()
    given = (y.gather(1, s["tokens"][:, None])[:, 0] - log_total).float()
    at = _ranked(x, s["case"]["top"])
    return given, entropy, at, (y.gather(1, at) - log_total[:, None]).float()


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        from vllm_quick_amd import ops
        if c["op"] == "append":
            query = ops.rope_append_kv4(s["positions"], s["query"], s["key"], s["value"], s["cos_sin"], s["cache"], s["slots"],
                                        interleaved=c["interleaved"])
            return (query, *ops.kv4_read(s["cache"], s["slots"], c["head"], s["query"].dtype))
        if c["op"] == "attend":
            return ops.paged_attention_kv4(s["query"], s["cache"], s["tables"], s["lens"], s["scale"], c["longest"],
                                           query_start=s["start"] if c["queries"] > 1 else None, max_query_len=c["queries"],
                                           window=c["window"])
        return ops.token_logprobs(s["logits"], s["tokens"], c["top"])
    if c["op"] == "append":
        return _plain_append(s)
    return _plain_attend(s) if c["op"] == "attend" else _plain_logprobs(s)


# ---------------------------------------------------------------------------------------------------------------
# what the definition gives in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _values_of(cache, head, block, at):
    """The keys and values that slots (block, at) [n] stand for: two [n, H, D] in 64 bits, byte by byte."""
    p = cache.shape[2] // (head + 8)
    el = torch.arange(head, device=cache.device)
    base = block[:, None, None]
    heads = torch.arange(cache.shape[1], device=cache.device)[None, :, None]
    k_byte = at[:, None, None] * (head // 2) + el // 2
    v_byte = p * head // 2 + (at[:, None, None] // 16) * (8 * head) + (el // 8) * 64 + (at[:, None, None] % 16) * 4 + (el % 8) // 2
    found = []
    for which, byte in enumerate((k_byte, v_byte)):
        code = (cache[base, heads, byte] >> (4 * (el % 2))) & 15
        word = (p * head + which * 4 * p) // 2 + 2 * at[:, None, None]
        halves = cache.view(torch.float16)
        scale, least = (halves[base, heads, word + i].double() for i in (0, 1))
        found.append(least + code.double() * scale)
    return found


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "logprobs":
        x = s["logits"].double()
        logp = torch.log_softmax(x, 1)
        entropy = -(logp.exp() * logp).sum(1)
        at = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["top"]]
        return logp.gather(1, s["tokens"][:, None])[:, 0], entropy, at, logp.gather(1, at)
    if c["op"] == "append":
        n = c["rotary"] // 2
        unit = torch.complex(*(s["cos_sin"][s["positions"]].double()[:, None, i * n:(i + 1) * n] for i in (0, 1)))

        def turn(x):
            x = x.double().clone()
            a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if c["interleaved"] else (slice(0, n), slice(n, 2 * n))
            z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * unit
            x[..., a], x[..., b] = z.real, z.imag
            return x

        back = []
        for x in (turn(s["key"]), s["value"].double()):
            least = x.amin(-1, keepdim=True).half().double()
            scale = ((x.amax(-1, keepdim=True) - least) / 15).half().double()
            code = ((x - least) / scale).round().clamp(0, 15)
            stood = torch.where(scale > 0, least + code * scale, least)
            stood[c["tokens"] - c["padded"]:] = 0
            back.append(stood)
        return turn(s["query"]), back[0], back[1]
    lens, queries = _lengths(c)
    group = c["heads"] // c["kv"]
    out = torch.empty(s["query"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, m) in enumerate(zip(lens, queries)):
        j = torch.arange(n, device="cuda")
        low = max(0, n - m + 1 - c["window"]) if c["window"] else 0
        j = j[low:]
        k, v = _values_of(s["cache"], c["head"], s["tables"][b].long()[j // c["page"]], j % c["page"])
        at = torch.arange(n - m, n, device="cuda")[:, None]
        hidden = (j[None] > at) | ((at - j[None] >= c["window"]) if c["window"] else False)
        for h in range(c["kv"]):
            q = s["query"][row:row + m, h * group:(h + 1) * group].double().transpose(0, 1)  # [group, m, D]
            x = torch.matmul(q, k[:, h].t().contiguous()) * s["scale"]
            x = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            out[row:row + m, h * group:(h + 1) * group] = torch.matmul(x, v[:, h].contiguous()).transpose(0, 1)
        row += m
    return out
