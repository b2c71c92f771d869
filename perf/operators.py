"""The 8-bit prefix cache and the block-sparse attention: the work whose speed is watched.

Families (``kind``), each through ``diffusorrt_amd.kernels.PrefixKVCache``:

  store   ``store`` of new rows into an 8-bit cache, then ``load`` of the blocks they touch
  attend  ``attention`` over a filled 8-bit cache
  select  ``select_blocks``: the blocks of keys that each query reads, by a cheap score
  sparse  ``sparse_attention`` over given blocks
  step    the three of a layer's step: ``store`` of its rows, ``select_blocks``,
          ``sparse_attention``

An 8-bit cache holds, for each 32 keys of a K/V head (a tile), K and V as whole numbers of
[-127, 127] times one power of two each, the least that holds the tile (2^-40 at least). A
store quantizes a tile it touches as a whole: the rows it keeps, as they read, and the new.

Heads are those of the two architectures the framework serves (16 over 8 and 28 over 4, head
dimension 128); positions under the ``d2f`` mask see whole blocks of 32 up to their own.
"""
from __future__ import annotations

import math

import torch

own = False

HD = 128
TILE = 32   # keys that share a scale
MASK = 32   # the d2f mask's block
HEADS = {"bd3": (16, 8), "dream": (28, 4)}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # a denoised block joins a long prefix: the smallest call, all latency
        {"name": "store_block", "kind": "store", "arch": "bd3", "pos0": 8192, "rows": 32,
         "src": "bf16"},
        # a prompt's second chunk, off the tile grid at both ends
        {"name": "store_prompt", "kind": "store", "arch": "dream", "pos0": 1005, "rows": 2000,
         "src": "f32"},
        # one token of the large model over a long prefix
        {"name": "attend_token", "kind": "attend", "arch": "dream", "rows": 1, "keys": 8192,
         "q": "f16", "mask": "full"},
        # a block of the small model over a long prefix
        {"name": "attend_block", "kind": "attend", "arch": "bd3", "rows": 32, "keys": 8224,
         "q": "bf16", "mask": "d2f"},
        # an 8-token block and the row before it, a short ragged prefix
        {"name": "attend_rows9", "kind": "attend", "arch": "dream", "rows": 9, "keys": 1337,
         "q": "bf16", "mask": "full"},
        # a block over a prefix of a whole book
        {"name": "attend_book", "kind": "attend", "arch": "bd3", "rows": 32, "keys": 131072,
         "q": "f16", "mask": "full"},
        # a prompt's second chunk of 2048 rows
        {"name": "attend_prompt", "kind": "attend", "arch": "bd3", "rows": 2048, "keys": 4096,
         "q": "bf16", "mask": "d2f"},
        # the blocks a denoised block reads of a long prefix
        {"name": "select_block", "kind": "select", "arch": "bd3", "rows": 32, "keys": 32768,
         "q": "f16", "cache": "i8", "mask": "d2f", "block": 64, "count": 16},
        # the same of a prompt's rows, small blocks of an unquantized cache
        {"name": "select_prompt", "kind": "select", "arch": "dream", "rows": 1000, "keys": 16000,
         "q": "bf16", "cache": "bf16", "mask": "d2f", "block": 32, "count": 24},
        # a block over the chosen part of a book
        {"name": "sparse_block", "kind": "sparse", "arch": "bd3", "rows": 32, "keys": 131072,
         "q": "bf16", "cache": "i8", "mask": "d2f", "block": 64, "count": 32},
        # a prompt's last chunk over the chosen part of what comes before
        {"name": "sparse_prompt", "kind": "sparse", "arch": "bd3", "rows": 2048, "keys": 32768,
         "q": "f16", "cache": "i8", "mask": "d2f", "block": 64, "count": 16},
        # a layer's step of the large model: an 8-token block and the row before it
        {"name": "step_rows9", "kind": "step", "arch": "dream", "rows": 9, "keys": 20000,
         "q": "f16", "cache": "f16", "mask": "full", "block": 64, "count": 16},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "select", "sparse", "sparse", "step"])
    case = {"kind": kind, "arch": rng.choice(["bd3", "dream"])}
    if kind == "store":
        return case | {"pos0": rng.randint(0, 8192), "rows": _log_int(rng, 1, 2048),
                       "src": rng.choice(["f32", "bf16"])}
    # rows and keys together cost no more than the largest listed case
    rows = 9 if kind == "step" else _log_int(rng, 1, 2048)
    most = {"attend": 1 << 22, "select": 1 << 25, "sparse": 1 << 25, "step": 1 << 25}[kind]
    size, count = rng.choice([32, 64, 96, 128]), rng.randint(4, 32)
    least = 2 * size * count if kind == "select" else 64  # (a choice that the inputs decide)
    keys = _log_int(rng, max(rows, least), min(131072, max(2 * rows, 2 * least, most // rows)))
    case |= {"rows": rows, "keys": keys, "q": rng.choice(["f16", "bf16"]),
             "mask": rng.choice(["full", "d2f"])}
    if kind == "attend":
        return case
    cache = rng.choice(["i8", "i8", case["q"]])  # a 16-bit cache takes queries of its own type
    return case | {"cache": cache, "block": size, "count": count}


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _topics(gen, keys, hkv):
    """What passages of about 200 tokens have in common: a direction for each and head."""
    n = keys // 200 + 1
    return 0.5 * _randn(gen, n, hkv, HD), torch.arange(keys, device="cuda") * n // keys


def _kv(gen, keys, hkv, topics):
    chan = torch.exp(0.4 * _randn(gen, 1, hkv, HD))  # some channels of K are larger
    k = (_randn(gen, keys, hkv, HD) + topics[0][topics[1]]) * chan
    v = _randn(gen, keys, hkv, HD) * (0.2 + 0.6 * torch.rand(1, hkv, 1, generator=gen,
                                                             device="cuda"))
    return k.bfloat16(), v.bfloat16(), chan


def _queries(gen, rows, hq, hkv, topics, chan, dtype):
    """Neighbouring queries ask after the same passage, each with a part of its own."""
    at = torch.randint(0, topics[0].shape[0], (rows // 16 + 1,), generator=gen, device="cuda")
    about = topics[0][at].repeat_interleave(16, 0)[:rows].repeat_interleave(hq // hkv, 1)
    q = (_randn(gen, rows, hq, HD) + 2.0 * about) / chan.repeat_interleave(hq // hkv, 1)
    return q.to(dtype)


def _exponents(most):
    """The least e >= -40 with most <= 127 * 2^e, from the bits of a float32."""
    bits = most.contiguous().view(torch.int32)
    e = (bits >> 23) - 133 + ((bits & 0x7FFFFF) > 0x7E0000).int()
    return e.clamp_min(-40)


def _tiles(x):
    """[n, hkv, 128] as whole tiles [t, 32, hkv, 128], zeros behind the last row."""
    t = -(-x.shape[0] // TILE)
    out = torch.zeros((t * TILE,) + x.shape[1:], dtype=torch.float32, device=x.device)
    out[:x.shape[0]] = x.float()
    return out.view(t, TILE, *x.shape[1:])


def _quantized(x):
    """(codes int8 [t, 32, hkv, 128], scales float32 [t, hkv]) of float32 tiles."""
    e = _exponents(x.abs().amax((1, 3)))
    scale = ((e + 127) << 23).view(torch.float32)
    return torch.round(x / scale[:, None, :, None]).to(torch.int8), scale


def _values(codes, scale):
    return codes.float() * scale[:, None, :, None]


def _held(x, kind):
    """A cache's rows as the plain form keeps them."""
    if kind == "i8":
        return _quantized(_tiles(x))
    return (_tiles(x).to(TYPES[kind]), None)


def _read(held):
    """Its rows as float32 values [keys rounded up to tiles, hkv, 128]."""
    x = held[0].float() if held[1] is None else _values(*held)
    return x.flatten(0, 1)


def _ends(case, device="cuda"):
    """The number of keys each row sees, always the first ones."""
    keys, rows = case["keys"], case["rows"]
    p = torch.arange(keys - rows, keys, device=device)
    if case["mask"] == "full":
        return torch.full_like(p, keys)
    return ((p // MASK + 1) * MASK).clamp_max(keys)


def _any_blocks(gen, case, hkv):
    """Blocks for a case that takes them as given: those of a few passages that neighbouring
    rows share, the row's last block among them, ascending, -1 behind the last."""
    rows, count, size = case["rows"], case["count"], case["block"]
    last = (_ends(case) - 1) // size                                    # [rows]
    n = (case["keys"] + size - 1) // size
    score = torch.rand((rows // 16 + 1, hkv, n), generator=gen, device="cuda")
    score = score.repeat_interleave(16, 0)[:rows] + 0.05 * torch.rand(
        (rows, hkv, n), generator=gen, device="cuda")
    b = torch.arange(n, device="cuda")
    score = torch.where(b == last[:, None, None], 2.0, score)
    score = torch.where(b > last[:, None, None], -1.0, score)
    if n < count:
        score = torch.nn.functional.pad(score, (0, count - n), value=-1.0)
    top, at = score.topk(count, -1)
    at = torch.where(top >= 0, at, 1 << 30).sort(-1).values
    return torch.where(at < (1 << 30), at, -1).int()


def _raw(case, seed):
    """(k, v, queries or None, given blocks or None): what the inputs are made of."""
    gen = _gen(seed)
    hq, hkv = HEADS[case["arch"]]
    if case["kind"] == "store":
        keys = case["pos0"] + case["rows"]
        k, v, _ = _kv(gen, keys, hkv, _topics(gen, keys, hkv))
        return k, v, None, None
    topics = _topics(gen, case["keys"], hkv)
    k, v, chan = _kv(gen, case["keys"], hkv, topics)
    q = _queries(gen, case["rows"], hq, hkv, topics, chan, TYPES[case["q"]])
    return k, v, q, _any_blocks(gen, case, hkv) if case["kind"] == "sparse" else None


def _first_new(case):
    """The first row that the pass itself stores (all are there already otherwise)."""
    return {"store": case.get("pos0"), "step": case.get("keys", 0) - case["rows"]}.get(
        case["kind"], case.get("keys"))


def prepare(case, seed):
    k, v, q, blocks = _raw(case, seed)
    n, kind = _first_new(case), case.get("cache", "i8")
    src = TYPES[case.get("src", "bf16")]
    state = {"case": case, "q": q, "blocks": blocks, "k": k[n:].to(src), "v": v[n:].to(src)}
    if own:  # the cache that a program keeps
        from diffusorrt_amd.kernels import PrefixKVCache

        state["cache"] = PrefixKVCache(1, k.shape[1], k.shape[0], dtype=kind,
                                       block_sums=case["kind"] != "attend")
        if n:
            state["cache"].store(0, k[:n], v[:n], 0)
    else:  # its rows in a plain order
        total = -(-k.shape[0] // TILE) * TILE
        state["held"] = []
        for x in (k, v):
            rows = torch.zeros((total,) + x.shape[1:], device="cuda")
            rows[:n] = x[:n].float()
            state["held"].append(_held(rows, kind))
    return state


# ---------------------------------------------------------------- one pass, plain form

def _stored(held, x, pos0, kind):
    """The tiles from the first that rows x at pos0 touch to the last, as a cache holds them
    with the new rows: (first tile, tiles as _held gives them)."""
    t0, t1 = pos0 // TILE, (pos0 + x.shape[0] - 1) // TILE + 1
    part = (held[0][t0:t1], None if held[1] is None else held[1][t0:t1])
    rows = _read(part)
    rows[pos0 - t0 * TILE:pos0 - t0 * TILE + x.shape[0]] = x.float()
    return t0, _held(rows, kind)


def _with(held, t0, new):
    return tuple(None if a is None else torch.cat([a[:t0], b, a[t0 + b.shape[0]:]])
                 for a, b in zip(held, new))


def _tile_sums(k):
    """Each tile's keys added up: [t, hkv, 128], summed in 64 bits and rounded once."""
    return k.view(-1, TILE, *k.shape[1:]).double().sum(1).float()


def _plain_select(case, q, k):
    """Each row's blocks for each K/V head: its last, and those whose keys' sum has the largest
    products with the sum of the head's queries; [rows, hkv, count], ascending, -1 behind."""
    size, count, hkv = case["block"], case["count"], k.shape[1]
    rows = q.shape[0]
    n = (case["keys"] + size - 1) // size
    sums = _tile_sums(k)
    pad = n * (size // TILE) - sums.shape[0]
    sums = torch.nn.functional.pad(sums, (0, 0, 0, 0, 0, pad)).double()
    sums = sums.view(n, size // TILE, hkv, HD).sum(1)                      # [n, hkv, 128]
    qs = q.double().view(rows, hkv, -1, HD).sum(2)                        # [rows, hkv, 128]
    score = torch.matmul(qs.transpose(0, 1).contiguous(), sums.permute(1, 2, 0).contiguous())
    score = score.transpose(0, 1)                                         # [rows, hkv, n]
    last = ((_ends(case) - 1) // size)[:, None, None]
    b = torch.arange(n, device=q.device)
    score = score.masked_fill(b == last, math.inf).masked_fill(b > last, -math.inf)
    at = score.sort(dim=-1, descending=True, stable=True).indices[..., :count]
    at = torch.where(at <= last, at, 1 << 30).sort(dim=-1).values
    if at.shape[-1] < count:
        at = torch.nn.functional.pad(at, (0, count - at.shape[-1]), value=1 << 30)
    return torch.where(at < (1 << 30), at, -1).int()


def _plain_attention(case, q, k, v, blocks=None):
    """softmax(q k^T / sqrt(128)) v over the keys a row sees (of its blocks, where given)."""
    rows, hq, _ = q.shape
    keys, hkv = case["keys"], k.shape[1]
    k, v = k[:keys].transpose(0, 1).contiguous(), v[:keys].transpose(0, 1).contiguous()
    qg = q.float().view(rows, hkv, hq // hkv, HD).permute(1, 0, 2, 3).reshape(hkv, -1, HD)
    s = torch.matmul(qg, k.transpose(1, 2).contiguous()) / math.sqrt(HD)
    s = s.view(hkv, rows, hq // hkv, keys)
    seen = (torch.arange(keys, device=q.device) < _ends(case)[:, None])[None, :, None, :]
    if blocks is not None:
        n = (keys + case["block"] - 1) // case["block"]
        of = torch.zeros((rows, hkv, n + 1), dtype=torch.bool, device=q.device)
        of.scatter_(2, torch.where(blocks >= 0, blocks, n).long(), True)
        of = of[..., :n].repeat_interleave(case["block"], 2)[..., :keys]
        seen = seen & of.transpose(0, 1)[:, :, None, :]
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(hkv, -1, keys), v).view(hkv, rows, hq // hkv, HD)
    return o.permute(1, 0, 2, 3).reshape(rows, hq * HD).bfloat16()


def _run_plain(st):
    case, kind = st["case"], st["case"]["kind"]
    cache = case.get("cache", "i8")
    if kind == "store":
        t0, k = _stored(st["held"][0], st["k"], case["pos0"], cache)
        _, v = _stored(st["held"][1], st["v"], case["pos0"], cache)
        return {"k": _read(k), "v": _read(v), "sums": _tile_sums(_read(k)).transpose(0, 1)}
    held = st["held"]
    if kind == "step":
        n = _first_new(case)
        held = [_with(h, *_stored(h, st[x], n, cache)) for h, x in zip(held, ("k", "v"))]
    k = _read(held[0])
    if kind == "select":
        return _plain_select(case, st["q"], k)
    blocks = _plain_select(case, st["q"], k) if kind == "step" else st["blocks"]
    out = _plain_attention(case, st["q"], k, _read(held[1]), blocks)
    return {"blocks": blocks, "out": out} if kind == "step" else out


# ---------------------------------------------------------------- one pass, the framework's

def _where(case):
    return {"n_keys": case["keys"], "row_pos0": case["keys"] - case["rows"],
            "kind": "full" if case["mask"] == "full" else "d2f_hybrid",
            "mask_geometry": None if case["mask"] == "full" else (0, MASK)}


def _run_own(st):
    case, kind, cache = st["case"], st["case"]["kind"], st["cache"]
    if kind == "store":
        pos0, n = case["pos0"], case["rows"]
        cache.store(0, st["k"], st["v"], pos0)
        t0, t1 = pos0 // TILE, (pos0 + n - 1) // TILE + 1
        k, v = cache.load(0, t0 * TILE, (t1 - t0) * TILE)
        return {"k": k, "v": v, "sums": cache.sums[0, :, t0:t1]}
    if kind == "attend":
        return cache.attention(0, st["q"], out_dtype=torch.bfloat16, **_where(case))
    if kind == "step":
        cache.store(0, st["k"], st["v"], _first_new(case))
    blocks = st["blocks"]
    if kind != "sparse":
        blocks = cache.select_blocks(0, st["q"], block_size=case["block"], count=case["count"],
                                     **_where(case))
        if kind == "select":
            return blocks
    out = cache.sparse_attention(0, st["q"], blocks, block_size=case["block"],
                                 out_dtype=torch.bfloat16, **_where(case))
    return {"blocks": blocks, "out": out} if kind == "step" else out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    hq, hkv = HEADS[case["arch"]]
    rows, kind = case["rows"], case["kind"]
    row = hkv * HD
    if kind == "store":
        tiles = (case["pos0"] + rows - 1) // TILE - case["pos0"] // TILE + 1
        src = 4 if case["src"] == "f32" else 2
        return {"bytes": 2 * rows * row * (src + 1) + tiles * row * (2 * TILE * (1 + 4) + 8),
                "flops": 4 * rows * row}
    keys, w = case["keys"], 1 if case.get("cache", "i8") == "i8" else 2
    q = rows * hq * HD * 2
    if kind == "attend":
        return {"bytes": 2 * q + 2 * keys * row * w,
                "flops": 4.0 * HD * hq * float(_ends(case, "cpu").sum())}
    n, size, count = -(-keys // case["block"]), case["block"], case["count"]
    pairs = float((_ends(case, "cpu") + size - 1).div(size, rounding_mode="floor")
                  .clamp_max(count).sum())  # (row, block) pairs for each K/V head
    lists = rows * hkv * count * 4
    select = {"bytes": q + (keys // TILE) * row * 4 + lists, "flops": 2.0 * rows * n * row}
    read = min(keys, pairs * size)  # keys of each head at most
    sparse = {"bytes": 2 * q + 2 * read * row * w + lists,
              "flops": 4.0 * HD * hq * pairs * size}
    if kind == "select":
        return select
    if kind == "sparse":
        return sparse
    return {"bytes": select["bytes"] + sparse["bytes"] + 2 * rows * row * (2 + w),
            "flops": select["flops"] + sparse["flops"]}


# ---------------------------------------------------------------- in 64 bits, from the definitions

def _power(e):
    """2^e in 64 bits, from its bits (a library's power may be off by one in the last)."""
    return ((e + 1023) << 52).view(torch.float64)


def _exact_tile(x, kind):
    """One (tile, head)'s rows [.., 32, hkv, 128] in 64 bits as a cache gives them back."""
    if kind != "i8":
        return x.to(TYPES[kind]).double()
    most = x.abs().amax((-3, -1), keepdim=True)
    e = torch.ceil(torch.log2(most / 127)).clamp_min(-40).long()
    e = torch.where(127 * _power(e) < most, e + 1, e)
    e = torch.where((e > -40) & (127 * _power(e - 1) >= most), e - 1, e)
    step = _power(e)
    return torch.round(x / step) * step


def _exact_cache(x, n, kind):
    """Rows [0, n) stored first, the others after them; [tiles, 32, hkv, 128]."""
    full = torch.zeros((-(-x.shape[0] // TILE) * TILE,) + x.shape[1:], dtype=torch.float64,
                       device=x.device)
    full[:n] = x[:n].double()
    full = _exact_tile(full.view(-1, TILE, *x.shape[1:]), kind).view_as(full)
    if n < x.shape[0]:
        full[n:x.shape[0]] = x[n:].double()
        t0 = n // TILE
        full[t0 * TILE:] = _exact_tile(full[t0 * TILE:].view(-1, TILE, *x.shape[1:]),
                                       kind).view_as(full[t0 * TILE:])
    return full


def _exact_select(case, q, k):
    """For each row and K/V head the last block and the best others, in any order."""
    rows, hkv, size = q.shape[0], k.shape[1], case["block"]
    ends = _ends(case)
    blocks = torch.full((rows, hkv, case["count"]), -1, dtype=torch.int32, device=q.device)
    for r in range(rows):
        last = (int(ends[r]) - 1) // size
        whole = k[:last * size].view(last, size, hkv, HD).sum(1)
        for h in range(hkv):
            g = q.shape[1] // hkv
            score = whole[:, h] @ q[r, h * g:(h + 1) * g].double().sum(0)
            best = torch.argsort(-score, stable=True)[:case["count"] - 1]
            blocks[r, h, :best.numel()] = best.int()
            blocks[r, h, best.numel()] = last
    return blocks


def exact(case, seed):
    k, v, q, blocks = _raw(case, seed)
    kind, n = case.get("cache", "i8"), _first_new(case)
    k, v = _exact_cache(k, n, kind), _exact_cache(v, n, kind)
    if case["kind"] == "store":
        t0 = n // TILE
        return {"k": k[t0 * TILE:], "v": v[t0 * TILE:],
                "sums": k[t0 * TILE:].view(-1, TILE, *k.shape[1:]).sum(1).transpose(0, 1)}
    if case["kind"] == "select":
        return None
    hkv, keys = k.shape[1], case["keys"]
    g = q.shape[1] // hkv
    ends = _ends(case)
    key = torch.arange(keys, device=q.device)
    if case["kind"] == "step":
        blocks = _exact_select(case, q, k)
    out = torch.empty((q.shape[0], hkv, g, HD), dtype=torch.float64, device=q.device)
    for r0 in range(0, q.shape[0], 64):
        for h in range(hkv):
            seen = key[None] < ends[r0:r0 + 64, None]
            if blocks is not None:
                mine = blocks[r0:r0 + 64, h]
                hit = (mine[:, :, None] == torch.arange(-(-keys // case["block"]),
                                                        device=q.device)).any(1)
                seen = seen & hit[:, key // case["block"]]
            for j in range(g):
                s = q[r0:r0 + 64, h * g + j].double() @ k[:keys, h].t() * HD ** -0.5
                out[r0:r0 + 64, h, j] = torch.softmax(s.masked_fill(~seen, -math.inf),
                                                      -1) @ v[:keys, h]
    out = out.reshape(q.shape[0], -1)
    return {"blocks": None, "out": out} if case["kind"] == "step" else out
