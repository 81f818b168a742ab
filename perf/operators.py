"""The serving operators around the quantized GEMMs, as cases to run and time:

* ``rope``       rotary positions with several axes on the queries and keys of a step;
* ``append``     quantizing a step's keys and values into the paged 4-bit cache;
* ``attention``  attention of a step's queries over that cache (single tokens, a few
                 speculated tokens, whole prompts), optionally adding every cached token's
                 attention weight to a running sum;
* ``evict``      keeping the tokens of largest accumulated weight and compacting the cache.

``run`` computes them in plain torch (32-bit arithmetic) or, with ``own`` set, through
``busfill_b200``. The head layout of most cases (64 query heads, 8 key/value heads of 128) is the
one of the decoder layer whose GEMMs ``bench.py`` times: a fused QKV of 10240 columns and an
8192-deep O projection.

The cache. A page holds 64 tokens of one key/value head; ``pages`` is uint8
[num_pages, kv_heads, 72 * D] for head dimension D, in four parts: key codes (64 rows of D/2
bytes), key scales, value codes (64 rows), value scales. Every 32 channels of a token share an
fp16 scale d; a code c in 0..15 stands for (c - 8) * d. `_layout` says where the code of a
channel and the scale of a block sit.
"""
import math
import random

import torch

own = False

PAGE = 64          # tokens of one head in a page
BLOCK = 32         # channels that share a scale
MAX_SCALE = 896.0  # largest |scale| of the format

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 8 sequences, each token with its own text position: launch latency
        dict(name="rope-decode8", kind="rope", tokens=8, heads=64, kv_heads=8, dim=128, rot=128, axes=3,
             pairs="halves", dtype="fp16", shape_seed=1),
        # a prompt of text and image patches (time, height, width positions), partial rotation
        dict(name="rope-prompt-8190-bf16", kind="rope", tokens=8190, heads=64, kv_heads=8, dim=128, rot=96, axes=3,
             pairs="adjacent", dtype="bf16", shape_seed=2),
        # the step's keys and values of 33 sequences, one token each, at odd places in their last pages
        dict(name="append-decode33", kind="append", batch=33, new=1, ctx=5000, ragged=True, kv_heads=8, dim=128,
             dtype="fp16", shape_seed=3),
        # prompts of four requests of uneven length, written behind what their cache holds
        dict(name="append-prompt-4x4099-bf16", kind="append", batch=4, new=4099, ctx=700, ragged=True, kv_heads=8,
             dim=128, dtype="bf16", shape_seed=4),
        # one request, one token, a short chat: the smallest attention call
        dict(name="attn-decode-1x300", kind="attention", batch=1, new=1, ctx=300, ragged=False, heads=64, kv_heads=8,
             dim=128, window=0, weights=False, dtype="fp16", shape_seed=5),
        # ordinary serving: a batch of 32 at uneven lengths up to 16K
        dict(name="attn-decode-32x16000", kind="attention", batch=32, new=1, ctx=16000, ragged=True, heads=64,
             kv_heads=8, dim=128, window=0, weights=False, dtype="fp16", shape_seed=6),
        # one long document, with the weights that eviction needs
        dict(name="attn-decode-1x131071-weights-bf16", kind="attention", batch=1, new=1, ctx=131071, ragged=False,
             heads=64, kv_heads=8, dim=128, window=0, weights=True, dtype="bf16", shape_seed=7),
        # checking four speculated tokens of 8 sequences; head dimension 64, sliding window
        dict(name="attn-verify-8x4-d64", kind="attention", batch=8, new=4, ctx=9000, ragged=True, heads=32,
             kv_heads=8, dim=64, window=4096, weights=False, dtype="fp16", shape_seed=8),
        # uneven prompts of three requests behind cached prefixes, with the weights
        dict(name="attn-prompt-3x1000-weights", kind="attention", batch=3, new=1000, ctx=2500, ragged=True, heads=64,
             kv_heads=8, dim=128, window=0, weights=True, dtype="bf16", shape_seed=9),
        # a long prompt in one piece: the largest call
        dict(name="attn-prompt-1x8000", kind="attention", batch=1, new=8000, ctx=8000, ragged=False, heads=64,
             kv_heads=8, dim=128, window=0, weights=False, dtype="fp16", shape_seed=10),
        # one request over its budget by a little
        dict(name="evict-1x1100-1024", kind="evict", batch=1, ctx=1100, ragged=False, keep=1024, recent=256,
             kv_heads=8, dim=128, shape_seed=11),
        # a batch of long requests brought down to a quarter
        dict(name="evict-8x32000-8000", kind="evict", batch=8, ctx=32000, ragged=True, keep=8000, recent=1000,
             kv_heads=8, dim=128, shape_seed=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attention", "attention", "attention", "evict"])
    kv_heads = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 128, 128, 256])
    dtype = rng.choice(["fp16", "bf16"])
    case = dict(kind=kind, kv_heads=kv_heads, dim=dim, shape_seed=rng.randrange(1 << 30))
    if kind == "rope":
        case.update(tokens=_log(rng, 1, 8190), heads=kv_heads * rng.choice([1, 3, 4, 8]),
                    rot=rng.choice([dim, dim // 2, dim - 16]), axes=rng.choice([1, 2, 3, 4]),
                    pairs=rng.choice(["halves", "adjacent"]), dtype=dtype)
        case["tokens"] = max(1, min(case["tokens"], 8190 * 72 * 128 // ((case["heads"] + kv_heads) * dim)))
    elif kind == "append":
        batch = _log(rng, 1, 64)
        case.update(batch=batch, new=_log(rng, 1, max(1, 16000 // batch)), ctx=_log(rng, 1, 20000),
                    ragged=rng.random() < 0.7, dtype=dtype)
    elif kind == "attention":
        group = rng.choice([1, 4, 7, 8, 16])
        case.update(heads=kv_heads * group, dtype=dtype, ragged=rng.random() < 0.7, weights=rng.random() < 0.3)
        form = rng.choice(["decode", "decode", "verify", "prompt"])
        if form == "prompt":
            case.update(batch=rng.choice([1, 2, 3, 5]), new=_log(rng, 9, 4000))
            case["ctx"] = case["new"] + rng.choice([0, _log(rng, 1, 4000)])
        else:
            batch = _log(rng, 1, 64)
            case.update(batch=batch, new=1 if form == "decode" else rng.randint(2, 8),
                        ctx=_log(rng, 8, max(16, min(131072, 500000 // batch))))
        case["window"] = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
        most = work(listed()[9])["flops"]
        while work(case)["flops"] > most:
            case["new"] = max(1, case["new"] // 2)
            case["ctx"] = max(case["new"], case["ctx"] // 2)
    else:
        batch = _log(rng, 1, 16)
        ctx = _log(rng, 16, max(16, 250000 // batch))
        keep = max(2, int(ctx * rng.uniform(0.1, 1.1)))
        case.update(batch=batch, ctx=ctx, ragged=rng.random() < 0.7, keep=keep, recent=int(keep * rng.uniform(0, 0.6)))
    return case


def _lengths(case):
    """(cached tokens, new tokens) of every sequence; the cached count includes the new ones."""
    rng = random.Random(case["shape_seed"])
    ctx, new = [], []
    for _ in range(case["batch"]):
        n = case.get("new", 0)
        if case["ragged"] and n > 8:
            n = rng.randint(max(1, n // 4), n)
        c = case["ctx"]
        if case["ragged"]:
            c = rng.randint(max(1, c // 8), c)
        if case["kind"] == "append":
            c += n
        ctx.append(max(c, n))
        new.append(n)
    return ctx, new


def _pages_of(length):
    return (length + PAGE - 1) // PAGE


def work(case):
    kv, dim = case["kv_heads"], case["dim"]
    token = kv * dim * 9 // 8          # bytes of one cached token: codes and scales of K and V
    if case["kind"] == "rope":
        t, heads = case["tokens"], case["heads"] + kv
        # queries and keys in and out, positions, and the rows of the angle tables once a token and axis
        return {"bytes": 4 * t * heads * dim + 4 * t * case["axes"] + 4 * t * case["rot"],
                "flops": 3 * t * heads * case["rot"]}
    ctx, new = _lengths(case)
    if case["kind"] == "append":
        t = sum(new)
        # keys and values in, codes and scales out, and the values they stand for
        return {"bytes": 4 * t * kv * dim + t * token + 4 * t * kv * dim, "flops": 8 * t * kv * dim}
    if case["kind"] == "evict":
        keep = [min(c, case["keep"]) for c in ctx]
        # the weights in, the kept ones out with their indices, the kept tokens in and out, and their values
        return {"bytes": 4 * kv * sum(ctx) + 8 * kv * sum(keep) + 2 * sum(keep) * token + 4 * sum(keep) * kv * dim,
                "flops": kv * sum(ctx)}
    seen = read = 0                    # (query, key) pairs and cached tokens that some query sees
    for c, n in zip(ctx, new):
        for e in (range(c - n + 1, c + 1) if n <= 64 else ()):
            seen += min(e, case["window"]) if case["window"] else e
        if n > 64:
            w = case["window"] or c
            full = max(0, min(n, c - w))          # queries that see w keys
            part = n - full                       # the others see their whole past
            first = c - n + 1
            seen += full * w + part * first + part * (part - 1) // 2
        read += min(c, case["window"] + n - 1) if case["window"] else c
    t = sum(new)
    io = 4 * t * case["heads"] * dim + (8 * kv * sum(ctx) if case["weights"] else 0)
    return {"bytes": read * token + io, "flops": 4 * seen * case["heads"] * dim}


# ---------------------------------------------------------------------------
# the cache format, in torch
# ---------------------------------------------------------------------------
def _layout(dim, device):
    """Where things sit in a page: for keys, the nibble of each channel in its row [D]; for values,
    the nibble of each channel by token [64, D]; for value scales, the column of each token [64]."""
    nb = dim // BLOCK
    ch = torch.arange(dim, device=device)
    b, j, n = ch // 32, ch % 32 // 8, ch % 8
    key = (j * nb + b) * 8 + n // 2 + 4 * (n % 2)
    t = torch.arange(PAGE, device=device)[:, None]
    swizzle = {64: t * 0, 128: 4 * (t // 4 % 2), 256: 2 * (t // 2 % 4)}[dim]
    value = (((2 * j + n % 2)[None] ^ swizzle) * nb + b) * 4 + n // 2
    column = t[:, 0] ^ (t[:, 0] // 2 % 2)
    return key, value, column


def _quantize(x):
    """x [..., D] -> codes uint8 [..., D] and scales fp16 [..., D/32]: a block's scale is its value of
    largest magnitude (the first of equals) over -8, rounded to 7 significant bits; a code is the
    nearest step, ties up. Infinities saturate, NaN counts as zero."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=65504.0, neginf=-65504.0)
    blocks = x.unflatten(-1, (-1, BLOCK))
    mag = blocks.abs()
    lane = torch.arange(BLOCK, device=x.device)
    first = torch.where(mag == mag.amax(-1, keepdim=True), lane, BLOCK).amin(-1, keepdim=True)
    top = blocks.gather(-1, first) / -8.0
    bits = top.view(torch.int32)
    bits = (bits + 0xFFFF + ((bits >> 17) & 1)) & ~0x1FFFF
    d = bits.view(torch.float32).clamp(-MAX_SCALE, MAX_SCALE).half().float()
    codes = torch.where(d == 0, 8.0, torch.floor(blocks / torch.where(d == 0, 1.0, d) + 8.5)).clamp(0, 15)
    return codes.to(torch.uint8).flatten(-2), d.squeeze(-1).half()


def _pack(k, v):
    """Keys and values [tokens, kv_heads, D], tokens a multiple of 64 -> pages uint8 [n, kv_heads, 72 D]."""
    tokens, heads, dim = k.shape
    n = tokens // PAGE
    key, value, column = _layout(dim, k.device)

    def rows(codes, where):
        codes = codes.view(n, PAGE, heads, dim).transpose(1, 2)
        row = torch.empty_like(codes)
        row.scatter_(-1, where.expand_as(codes), codes)
        return (row[..., 0::2] | row[..., 1::2] << 4).reshape(n, heads, -1)

    kc, kd = _quantize(k)
    vc, vd = _quantize(v)
    kd = kd.view(n, PAGE, heads, -1).transpose(1, 2).reshape(n, heads, -1)
    vd = vd.view(n, PAGE, heads, -1).permute(0, 2, 3, 1)
    placed = torch.empty_like(vd)
    placed[..., column] = vd
    return torch.cat([rows(kc, key), kd.contiguous().view(torch.uint8), rows(vc, value),
                      placed.reshape(n, heads, -1).view(torch.uint8)], dim=-1)


def _unpack(pages, dim):
    """pages uint8 [n, kv_heads, 72 D] -> the keys and values they stand for, fp32 [kv_heads, n * 64, D]."""
    n, heads = pages.shape[:2]
    key, value, column = _layout(dim, pages.device)
    nb = dim // BLOCK
    kc, kd, vc, vd = pages.split([32 * dim, 4 * dim, 32 * dim, 4 * dim], dim=-1)

    def codes(part, where):
        part = part.reshape(n, heads, PAGE, dim // 2)
        nibbles = torch.stack([part & 15, part >> 4], dim=-1).flatten(-2)
        return nibbles.gather(-1, where.expand(n, heads, PAGE, dim)).float() - 8.0

    kd = kd.contiguous().view(torch.float16).view(n, heads, PAGE, nb).float()
    vd = vd.contiguous().view(torch.float16).view(n, heads, nb, PAGE)[..., column].transpose(2, 3).float()
    k = codes(kc, key).unflatten(-1, (nb, BLOCK)) * kd[..., None]
    v = codes(vc, value).unflatten(-1, (nb, BLOCK)) * vd[..., None]
    return (k.flatten(-2).transpose(0, 1).reshape(heads, n * PAGE, dim),
            v.flatten(-2).transpose(0, 1).reshape(heads, n * PAGE, dim))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _keys_values(tokens, heads, dim, gen, dev):
    """Keys with a few strong channels (as rotary models have them) and plain values."""
    k = torch.randn((tokens, heads, dim), generator=gen, device=dev)
    k *= 1.0 + 4.0 * (torch.rand((1, heads, dim), generator=gen, device=dev) > 0.96)
    return k, torch.randn((tokens, heads, dim), generator=gen, device=dev)


def _tables(batch, pages, gen, dev):
    """A page table with the sequences' pages scattered over the pool (unused entries: page 0)."""
    cols = max(pages)
    order = torch.randperm(sum(pages), generator=gen, device=dev).int()
    table = torch.zeros((batch, cols), dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    return table


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 1000003 + 17)
    kind, kv, dim = case["kind"], case["kv_heads"], case["dim"]
    state = {"case": case}
    if kind == "rope":
        dtype, t, half = _DTYPES[case["dtype"]], case["tokens"], case["rot"] // 2
        qkv = torch.randn((t, case["heads"] + 2 * kv, dim), generator=gen, device=dev).to(dtype)
        state["q"], state["k"] = qkv[:, :case["heads"]], qkv[:, case["heads"]:case["heads"] + kv]
        # positions: text runs forward on every axis, an image holds time and walks height and width
        if t <= 64:
            pos = torch.randint(0, 30000, (1, t), generator=gen, device=dev).expand(case["axes"], t).clone()
        else:
            i = torch.arange(t, device=dev)
            pos = i.expand(case["axes"], t).clone()
            start, stop = t // 5, t // 5 + t // 2
            side = max(1, math.isqrt(stop - start))
            for axis in range(case["axes"]):
                walk = [i * 0, (i - start) // side, (i - start) % side, i * 0][axis]
                pos[axis, start:stop] = start + walk[start:stop]
            pos += torch.randint(0, 1000, (1, 1), generator=gen, device=dev)
        state["positions"] = pos.int()
        freq = 1e6 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
        angle = torch.arange(32768, device=dev, dtype=torch.float64)[:, None] * freq
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        # frequencies dealt to the axes in runs
        state["axis"] = [i * case["axes"] // half for i in range(half)]
        return state

    ctx, new = _lengths(case)
    pages = [_pages_of(c) for c in ctx]
    state["ctx"], state["new"] = ctx, new
    state["kv_len"] = torch.tensor(ctx, dtype=torch.int32, device=dev)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    state["q_start"] = torch.tensor(start, dtype=torch.int32, device=dev)
    state["table"] = _tables(case["batch"], pages, gen, dev)
    if kind == "append":
        dtype = _DTYPES[case["dtype"]]
        k, v = _keys_values(start[-1], kv, dim, gen, dev)
        state["k"], state["v"] = k.to(dtype), v.to(dtype)
        state["pages"] = torch.zeros((sum(pages), kv, 72 * dim), dtype=torch.uint8, device=dev)
        return state
    total = sum(pages)
    store = torch.empty((total, kv, 72 * dim), dtype=torch.uint8, device=dev)
    for at in range(0, total, 2048):
        n = min(2048, total - at)
        store[at:at + n] = _pack(*_keys_values(n * PAGE, kv, dim, gen, dev))
    state["pages"] = store
    if kind == "attention":
        dtype = _DTYPES[case["dtype"]]
        state["q"] = torch.randn((start[-1], case["heads"], dim), generator=gen, device=dev).to(dtype)
        state["scale"] = dim ** -0.5
        if case["weights"]:
            state["weights"] = torch.rand((case["batch"], kv, max(pages) * PAGE), generator=gen, device=dev)
    else:
        # accumulated weights: heavy-tailed, many tokens that nothing has looked at yet
        w = torch.randn((case["batch"], kv, max(pages) * PAGE), generator=gen, device=dev).mul(2.0).exp()
        state["weights"] = torch.where(w < 0.1, 0.0, w)
        kept = [min(c, case["keep"]) for c in ctx]
        state["kept"] = kept
        room = [_pages_of(c) for c in kept]
        state["room"] = _tables(case["batch"], room, gen, dev) + total
        for i, n in enumerate(room):
            state["room"][i, n:] = 0
        state["pages"] = torch.cat([store, torch.zeros((sum(room), kv, 72 * dim), dtype=torch.uint8, device=dev)])
        state["kept_len"] = torch.tensor(kept, dtype=torch.int32, device=dev)
        kept_start = [0]
        for n in kept:
            kept_start.append(kept_start[-1] + n)
        state["kept_start"] = torch.tensor(kept_start, dtype=torch.int32, device=dev)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return {"rope": _rope, "append": _append, "attention": _attention, "evict": _evict}[state["case"]["kind"]](state)


def _rope(s):
    case = s["case"]
    if own:
        import busfill_b200 as bf
        return bf.rope_axes(s["q"], s["k"], s["positions"], s["cos"], s["sin"], s["axis"],
                            adjacent=case["pairs"] == "adjacent")
    half = case["rot"] // 2
    axis = torch.tensor(s["axis"], device=s["q"].device)
    col = torch.arange(half, device=s["q"].device)
    at = s["positions"].long()[axis].t()
    cos, sin = s["cos"][at, col][:, None], s["sin"][at, col][:, None]

    def turn(x):
        y = x.float().clone()
        if case["pairs"] == "halves":
            a, b = slice(0, half), slice(half, 2 * half)
        else:
            a, b = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
        x0, x1 = y[..., a].clone(), y[..., b].clone()
        y[..., a] = x0 * cos - x1 * sin
        y[..., b] = x1 * cos + x0 * sin
        return y.to(x.dtype)

    return turn(s["q"]), turn(s["k"])


def _append(s):
    if own:
        import busfill_b200 as bf
        bf.kv4_append(s["pages"], s["table"], s["kv_len"], s["k"], s["v"], q_start=s["q_start"])
        return bf.kv4_read(s["pages"], s["table"], s["kv_len"], s["q_start"], s["k"].shape[0])
    out = []
    for x in (s["k"], s["v"]):
        codes, d = _quantize(x)
        x = (codes.float().unflatten(-1, (-1, BLOCK)) - 8.0) * d.float()[..., None]
        out.append(x.flatten(-2).half())
    return tuple(out)


def _attention(s):
    case = s["case"]
    weights = s["weights"].clone() if case["weights"] else None
    if own:
        import busfill_b200 as bf
        out = bf.attn_kv4(s["q"], s["pages"], s["table"], s["kv_len"], q_start=s["q_start"], max_q=max(s["new"]),
                          scale=s["scale"], causal=True, window=case["window"], weights=weights)
        return (out, weights) if case["weights"] else out
    group, dim = case["heads"] // case["kv_heads"], case["dim"]
    out = torch.empty_like(s["q"])
    at = 0
    for i, (c, n) in enumerate(zip(s["ctx"], s["new"])):
        k, v = _unpack(s["pages"][s["table"][i, :_pages_of(c)].long()], dim)
        slot = torch.arange(c, device=out.device)
        last = torch.arange(c - n, c, device=out.device)[:, None]
        unseen = slot > last
        if case["window"]:
            unseen |= slot <= last - case["window"]
        for h in range(case["kv_heads"]):
            q = s["q"][at:at + n, h * group:(h + 1) * group].float().transpose(0, 1)
            p = q @ k[h, :c].t() * s["scale"]
            p.masked_fill_(unseen, float("-inf"))
            p -= p.amax(-1, keepdim=True)
            p.exp_()
            p /= p.sum(-1, keepdim=True)
            out[at:at + n, h * group:(h + 1) * group] = (p @ v[h, :c]).transpose(0, 1).to(out.dtype)
            if weights is not None:
                weights[i, h, :c] += p.sum((0, 1))
        at += n
    return (out, weights) if case["weights"] else out


def _evict(s):
    case = s["case"]
    if own:
        import busfill_b200 as bf
        index, weights, kv_len = bf.kv4_evict(s["pages"], s["table"], s["kv_len"], s["weights"], case["keep"],
                                              case["recent"], out_table=s["room"])
        k, v = bf.kv4_read(s["pages"], s["room"], kv_len, s["kept_start"], sum(s["kept"]))
        return index, weights, kv_len, k, v
    kv, dim, dev = case["kv_heads"], case["dim"], s["pages"].device
    index = torch.full((case["batch"], kv, case["keep"]), -1, dtype=torch.int32, device=dev)
    weights = torch.zeros_like(s["weights"])
    ks, vs = [], []
    for i, c in enumerate(s["ctx"]):
        keep = min(c, case["keep"])
        recent = min(case["recent"], keep)
        order = torch.sort(s["weights"][i, :, :c - recent], dim=-1, descending=True, stable=True).indices
        tail = torch.arange(c - recent, c, device=dev).expand(kv, recent)
        kept = torch.cat([order[:, :keep - recent].sort(-1).values, tail], dim=-1)
        index[i, :, :keep] = kept.int()
        weights[i, :, :keep] = s["weights"][i].gather(-1, kept)
        for x, store in zip(_unpack(s["pages"][s["table"][i, :_pages_of(c)].long()], dim), (ks, vs)):
            store.append(x.gather(1, kept[..., None].expand(kv, keep, dim)).transpose(0, 1).half())
    return index, weights, s["kept_len"].clone(), torch.cat(ks), torch.cat(vs)


# ---------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------
def _page_values(page, dim):
    """Keys and values of one head's pages uint8 [n, 72 D], fp64 [n * 64, D], channel by channel."""
    n, nb = page.shape[0], dim // BLOCK
    rows = torch.empty((2, n * PAGE, dim), dtype=torch.float64, device=page.device)
    tok = torch.arange(PAGE, device=page.device)
    for ch in range(dim):
        b, r = divmod(ch, BLOCK)
        j, m = divmod(r, 8)
        # keys: 32-bit word (j, b); its low half has the even channels, its high half the odd ones
        byte = tok * (dim // 2) + 4 * (j * nb + b) + 2 * (m & 1) + (m >> 2)
        code = (page[:, byte] >> (4 * ((m >> 1) & 1))) & 15
        d = page[:, 32 * dim:36 * dim].contiguous().view(torch.float16)[:, tok * nb + b].double()
        rows[0, :, ch] = ((code.double() - 8) * d).flatten()
        # values: 16-bit word (c, b), c exchanged among the tokens of a page
        c = torch.full_like(tok, 2 * j + (m & 1))
        if dim == 128:
            c = torch.where((tok & 4) != 0, c ^ 4, c)
        if dim == 256:
            c = c ^ (tok & 6)
        byte = 36 * dim + tok * (dim // 2) + 2 * (c * nb + b) + (m >> 2)
        code = (page[:, byte] >> (4 * ((m >> 1) & 1))) & 15
        place = tok - (tok & 1) + ((tok & 1) ^ ((tok >> 1) & 1))
        d = page[:, 68 * dim:].contiguous().view(torch.float16)[:, b * PAGE + place].double()
        rows[1, :, ch] = ((code.double() - 8) * d).flatten()
    return rows[0], rows[1]


def _nearest(x):
    """The cached values of x [tokens, heads, D] in fp64: 32-channel blocks, one scale each."""
    x = x.double().unflatten(-1, (-1, BLOCK))
    largest = x.abs() == x.abs().amax(-1, keepdim=True)
    step = torch.where(largest & (largest.cumsum(-1) == 1), x, 0.0).sum(-1, keepdim=True) / -8
    wide = step * (2.0 ** 46 + 1)      # the upper 53 - 46 = 7 significant bits, to nearest
    step = (wide - (wide - step)).clamp(-MAX_SCALE, MAX_SCALE).half().double()
    code = torch.floor(x / torch.where(step == 0, 1.0, step) + 0.5).clamp(-8, 7)
    return (code * step).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    kind, kv, dim = case["kind"], case["kv_heads"], case["dim"]
    if kind == "rope":
        half, out = case["rot"] // 2, []
        pos = s["positions"].long()
        c = torch.stack([s["cos"][pos[s["axis"][i]], i] for i in range(half)], -1).double()[:, None]
        sn = torch.stack([s["sin"][pos[s["axis"][i]], i] for i in range(half)], -1).double()[:, None]
        for x in (s["q"], s["k"]):
            y = x.double()
            shape = (2, half) if case["pairs"] == "halves" else (half, 2)
            z = y[..., :2 * half].unflatten(-1, shape)
            if case["pairs"] == "adjacent":
                z = z.transpose(-1, -2)
            re, im = z[..., 0, :] * c - z[..., 1, :] * sn, z[..., 0, :] * sn + z[..., 1, :] * c
            z = torch.stack([re, im], -2 if case["pairs"] == "halves" else -1).flatten(-2)
            out.append(torch.cat([z, y[..., 2 * half:]], -1))
        return tuple(out)
    if kind == "append":
        return _nearest(s["k"]), _nearest(s["v"])
    if kind == "evict":
        kept_all, new_w, ks, vs = [], torch.zeros_like(s["weights"], dtype=torch.float64), [], []
        for i, c in enumerate(s["ctx"]):
            keep = min(c, case["keep"])
            recent = min(case["recent"], keep)
            page = s["pages"][s["table"][i, :_pages_of(c)].long()]
            heads = []
            for h in range(kv):
                w = s["weights"][i, h, :c].double()
                # strictly larger weights first, then the lowest indices among equals
                need, old = keep - recent, w[:c - recent]
                mark = torch.zeros(c, dtype=torch.bool, device=w.device)
                mark[c - recent:] = True
                if need > 0:
                    edge = old.kthvalue(old.numel() - need + 1).values
                    mark[:c - recent] = old > edge
                    equal = (old == edge).nonzero().flatten()
                    mark[equal[:need - int((old > edge).sum())]] = True
                at = mark.nonzero().flatten()
                heads.append(torch.nn.functional.pad(at, (0, case["keep"] - keep), value=-1))
                new_w[i, h, :keep] = w[at]
                k, v = _page_values(page[:, h], dim)
                ks.append((i, h, k[at]))
                vs.append((i, h, v[at]))
            kept_all.append(torch.stack(heads))
        k = torch.cat([torch.stack([x for a, _, x in ks if a == i], 1) for i in range(case["batch"])])
        v = torch.cat([torch.stack([x for a, _, x in vs if a == i], 1) for i in range(case["batch"])])
        return torch.stack(kept_all).int(), new_w, s["kept_len"].clone(), k, v
    # softmax attention, one query head after another
    heads, group = case["heads"], case["heads"] // kv
    out = torch.zeros((sum(s["new"]), heads, dim), dtype=torch.float64, device=s["q"].device)
    weights = s["weights"].double() if case["weights"] else None
    base = 0
    for i, (c, n) in enumerate(zip(s["ctx"], s["new"])):
        page = s["pages"][s["table"][i, :_pages_of(c)].long()]
        for h in range(kv):
            k, v = _page_values(page[:, h], dim)
            k, v = k[:c], v[:c]
            for g in range(group):
                for lo in range(0, n, 2048):
                    hi = min(n, lo + 2048)
                    score = s["q"][base + lo:base + hi, h * group + g].double() @ k.t() * s["scale"]
                    row = torch.arange(c - n + lo, c - n + hi, device=score.device)
                    gap = row[:, None] - torch.arange(c, device=score.device)[None]
                    hide = gap < 0
                    if case["window"] > 0:
                        hide = hide | (gap >= case["window"])
                    p = torch.softmax(score.masked_fill(hide, -math.inf), -1)
                    out[base + lo:base + hi, h * group + g] = p @ v
                    if weights is not None:
                        weights[i, h, :c] += p.sum(0)
        base += n
    return (out, weights) if case["weights"] else out
