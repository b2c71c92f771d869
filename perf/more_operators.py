"""Rotary positions, the paged K/V cache and attention over it: the work whose speed is watched.

Families (``kind``):

  rotate  ``diffusorrt_amd.rotary.RotaryPositions.rotate`` of rows of heads at given positions
  append  ``diffusorrt_amd.paged.PagedKVCache.append``: new rows of several sequences into their
          pages, keys (and the queries beside them) rotated on the way, then ``load`` of them
  attend  ``PagedKVCache.attention``: each sequence's new rows over all its keys in the pages
  step    a layer's step: ``append`` of its rows, ``attention`` of them, ``load``

A sequence's keys lie in pages of a pool that all sequences share; its list of pages gives their
order. Its new rows are its last positions. A row at position p sees all of the sequence's keys
(``full``), those up to p (``causal``), or whole blocks of 32 up to its own (``d2f``).

Rotation at position p turns pair i of a head's first ``dim`` elements by p f_i, with
f_i = theta^(-2 i / dim) or one of the scaled forms in ``_frequencies``; a pair is elements
(i, i + dim / 2) of the ``half`` layout, (2 i, 2 i + 1) of the ``interleaved`` one.

Heads are those of the two architectures the framework serves (16 over 8 and 28 over 4, head
dimension 128, theta 10^6).
"""
from __future__ import annotations

import math
import random

import torch

own = False

HD = 128
THETA = 1e6
MASK = 32   # the d2f mask's block
HEADS = {"bd3": (16, 8), "dream": (28, 4)}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ORIGINAL = 32768  # positions that a model with scaled frequencies was trained on


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one token's queries far into a sequence: the smallest call, all latency
        {"name": "rotate_token", "kind": "rotate", "arch": "bd3", "rows": 1, "type": "bf16",
         "dim": 128, "layout": "half", "scaling": "none", "far": 131071, "fused": False},
        # queries as a fused projection leaves them, half of each head, neighbours paired
        {"name": "rotate_rows", "kind": "rotate", "arch": "dream", "rows": 1000, "type": "f32",
         "dim": 64, "layout": "interleaved", "scaling": "linear", "far": 100000, "fused": True},
        # a long prompt's queries, frequencies stretched by parts
        {"name": "rotate_prompt", "kind": "rotate", "arch": "bd3", "rows": 8192, "type": "bf16",
         "dim": 128, "layout": "half", "scaling": "yarn", "far": 120000, "fused": False},
        # the next token of 64 sequences
        {"name": "append_tokens", "kind": "append", "arch": "dream", "seqs": 64, "rows": 1,
         "chunk": 0, "keys": 4096, "least": 64, "ragged": False, "salt": 1, "cache": "f16",
         "src": "f32", "page": 64, "layout": "half", "scaling": "none"},
        # three prompts of up to 2048 rows, the first a later chunk of a longer one
        {"name": "append_prompts", "kind": "append", "arch": "bd3", "seqs": 3, "rows": 2048,
         "chunk": 0, "keys": 6000, "least": 700, "ragged": True, "salt": 2, "cache": "bf16",
         "src": "bf16", "page": 128, "layout": "half", "scaling": "yarn"},
        # one token of one short sequence
        {"name": "attend_token", "kind": "attend", "arch": "bd3", "seqs": 1, "rows": 1,
         "chunk": 0, "keys": 1337, "least": 1, "ragged": False, "salt": 3, "cache": "f16",
         "page": 64, "mask": "causal"},
        # a token each of 32 sequences from a few hundred to 16384 keys
        {"name": "attend_tokens", "kind": "attend", "arch": "dream", "seqs": 32, "rows": 1,
         "chunk": 0, "keys": 16384, "least": 200, "ragged": False, "salt": 4, "cache": "bf16",
         "page": 64, "mask": "causal"},
        # a token over a whole book
        {"name": "attend_book", "kind": "attend", "arch": "bd3", "seqs": 1, "rows": 1,
         "chunk": 0, "keys": 131072, "least": 1, "ragged": False, "salt": 5, "cache": "f16",
         "page": 256, "mask": "causal"},
        # a block of 32 tokens each of 16 sequences
        {"name": "attend_blocks", "kind": "attend", "arch": "bd3", "seqs": 16, "rows": 32,
         "chunk": 0, "keys": 8224, "least": 320, "ragged": False, "salt": 6, "cache": "f16",
         "page": 32, "mask": "d2f"},
        # a prompt's last chunk of 2048 rows
        {"name": "attend_prompt", "kind": "attend", "arch": "dream", "seqs": 1, "rows": 2048,
         "chunk": 0, "keys": 10240, "least": 2048, "ragged": False, "salt": 7, "cache": "bf16",
         "page": 128, "mask": "causal"},
        # one sequence's chunk of 500 rows beside the next token of 31 others
        {"name": "attend_mixed", "kind": "attend", "arch": "bd3", "seqs": 32, "rows": 1,
         "chunk": 500, "keys": 4097, "least": 100, "ragged": False, "salt": 8, "cache": "bf16",
         "page": 64, "mask": "causal"},
        # a layer's step of the large model: 8 sequences' block of 8 and the row before it
        {"name": "step_rows9", "kind": "step", "arch": "dream", "seqs": 8, "rows": 9,
         "chunk": 0, "keys": 2500, "least": 300, "ragged": False, "salt": 9, "cache": "f16",
         "src": "f32", "page": 64, "mask": "full", "layout": "half", "scaling": "none"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["rotate", "rotate", "append", "append", "attend", "attend", "attend",
                       "attend", "step"])
    case = {"kind": kind, "arch": rng.choice(["bd3", "dream"])}
    layout = rng.choice(["half", "interleaved"])
    scaling = rng.choice(["none", "linear", "ntk", "yarn"])
    if kind == "rotate":
        kinds = rng.choice(["f32", "f16", "bf16"])
        most = 2048 if kinds == "f32" else 4096  # no more than the largest listed case
        return case | {"rows": _log_int(rng, 1, most), "type": kinds,
                       "dim": rng.choice([32, 64, 96, 128]), "layout": layout,
                       "scaling": scaling, "far": _log_int(rng, 8192, 1 << 20),
                       "fused": rng.random() < 0.5}
    case |= {"cache": rng.choice(["f16", "bf16"]), "page": rng.choice([32, 64, 128, 256]),
             "salt": rng.randrange(1 << 30)}
    if kind in ("append", "step"):
        case |= {"src": rng.choice(["f32", "f16", "bf16"]), "layout": layout, "scaling": scaling}
    seqs = 1 if rng.random() < 0.25 else _log_int(rng, 2, 64)
    if kind == "append":
        rows = _log_int(rng, 1, max(1, 4096 // seqs))
        keys = rows + _log_int(rng, 1, 4096)
        return case | {"seqs": seqs, "rows": rows, "chunk": 0, "keys": keys,
                       "least": rng.randint(1, keys), "ragged": rng.random() < 0.5}
    rows = rng.choice([1, 1, 9, 32, _log_int(rng, 1, max(1, 2048 // seqs))])
    if kind == "step":
        rows = min(rows, 32)
    chunk = _log_int(rng, 32, 1000) if seqs > 1 and rows == 1 and rng.random() < 0.3 else 0
    # keys in all, and keys times rows, no more than the largest listed cases'
    most = min(131072 // seqs, (1 << 24) // (seqs * rows + chunk))
    keys = _log_int(rng, max(rows, chunk, 1), max(rows, chunk, 1, most))
    return case | {"seqs": seqs, "rows": rows, "chunk": chunk, "keys": keys,
                   "least": rng.randint(1, keys), "ragged": rng.random() < 0.5,
                   "mask": rng.choice(["full", "causal", "d2f"])}


def _lengths(case):
    """(rows, keys) of every sequence: the first has the most keys, the others any number from
    ``least`` on; ``ragged``: any number of rows up to ``rows``."""
    rng = random.Random(case["salt"])
    rows, keys = [], []
    for s in range(case["seqs"]):
        n = case["rows"] if not case["ragged"] else rng.randint(1, case["rows"])
        if s == 0 and case["chunk"]:
            n = case["chunk"]
        k = case["keys"] if s == 0 else _log_int(rng, min(case["least"], case["keys"]),
                                                  case["keys"])
        rows.append(n)
        keys.append(max(n, k))
    return rows, keys


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _scaling(case):
    """What a model's configuration says of its frequencies."""
    if case["scaling"] == "none":
        return None
    out = {"rope_type": case["scaling"], "factor": 4.0}
    if case["scaling"] == "yarn":
        out["original_max_position_embeddings"] = ORIGINAL
    return out


def _fresh(case, gen, rows):
    """q, k, v [rows, heads, 128] of the new rows, views of one fused projection."""
    hq, hkv = HEADS[case["arch"]]
    fused = _randn(gen, rows, hq + 2 * hkv, HD)
    fused = fused * torch.exp(0.4 * _randn(gen, 1, hq + 2 * hkv, HD))  # channels differ in size
    fused = fused.to(TYPES[case["src"]])
    return fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:]


def _pool(case, seed):
    """What the sequences have: their pages, the keys and values there, and the new rows'
    queries (and, where the pass appends them, keys and values)."""
    gen = _gen(seed)
    hq, hkv = HEADS[case["arch"]]
    rows, keys = _lengths(case)
    size, dtype = case["page"], TYPES[case["cache"]]
    need = [-(-k // size) for k in keys]
    order = torch.randperm(sum(need) + 3, generator=torch.Generator().manual_seed(int(seed)))
    table = torch.full((len(keys), max(need)), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n].int()
        at += n
    total = sum(keys)
    # passages of about 200 tokens have a direction in common that queries ask after
    topics = 0.5 * _randn(gen, total // 200 + 1, hkv, HD)
    of = torch.arange(total, device="cuda") * topics.shape[0] // total
    chan = torch.exp(0.4 * _randn(gen, 1, hkv, HD))
    k = ((_randn(gen, total, hkv, HD) + topics[of]) * chan).to(dtype)
    v = (_randn(gen, total, hkv, HD) * (0.2 + 0.6 * torch.rand(
        1, hkv, 1, generator=gen, device="cuda"))).to(dtype)
    n = sum(rows)
    state = {"case": case, "rows": rows, "keys": keys, "table": table, "pages": order.numel(),
             "old_k": k, "old_v": v}
    if case["kind"] == "attend":
        about = topics[torch.randint(0, topics.shape[0], (n,), generator=gen, device="cuda")]
        q = _randn(gen, n, hq, HD) + 2.0 * about.repeat_interleave(hq // hkv, 1)
        return state | {"q": (q / chan.repeat_interleave(hq // hkv, 1)).to(dtype)}
    q, k, v = _fresh(case, gen, n)
    return state | {"q": q, "k": k, "v": v}


def _heads(case, seed):
    """x and positions of a rotation."""
    gen = _gen(seed)
    hq, hkv = HEADS[case["arch"]]
    if case["fused"]:
        x = _fresh(case | {"src": case["type"]}, gen, case["rows"])[0]
    else:
        x = _randn(gen, case["rows"], hq, HD).to(TYPES[case["type"]])
    first = case["far"] - case["rows"] + 1
    positions = torch.arange(first, case["far"] + 1, device="cuda", dtype=torch.int32)
    if case["rows"] > 1:  # rows of several sequences, one after another
        positions = torch.where(torch.arange(case["rows"], device="cuda") < case["rows"] // 3,
                                positions - first, positions)
    return x, positions.int()


def prepare(case, seed):
    if case["kind"] == "rotate":
        x, positions = _heads(case, seed)
        state = {"case": case, "x": x, "positions": positions}
    else:
        state = _pool(case, seed)
    if own:
        return _prepare_own(state)
    if case["kind"] == "rotate":
        return state
    # the pool in a plain order, [pages, page, hkv, 128]; where each row of each sequence lies
    size, hkv = case["page"], HEADS[case["arch"]][1]
    state["pool"] = [torch.zeros((state["pages"], size, hkv, HD), dtype=TYPES[case["cache"]],
                                 device="cuda") for _ in range(2)]
    state["where"] = []
    at = 0
    for s, n in enumerate(state["keys"]):
        p = torch.arange(n)
        slot = (state["table"][s].long()[p // size] * size + p % size).cuda()
        state["where"].append(slot)
        for pool, old in zip(state["pool"], (state["old_k"], state["old_v"])):
            pool.view(-1, hkv, HD)[slot] = old[at:at + n]
        at += n
    state["new"] = torch.cat([w[len(w) - n:] for w, n in zip(state["where"], state["rows"])])
    state["positions"] = _positions(state)
    return state


def _positions(state):
    return torch.cat([torch.arange(k - n, k, device="cuda")
                      for n, k in zip(state["rows"], state["keys"])])


# ---------------------------------------------------------------- one pass, plain form

def _frequencies(dim, scaling, device):
    """(f_i [dim / 2] in 64 bits, what cosine and sine are multiplied by).

    linear: f / factor. ntk: a base of theta factor^(dim / (dim - 2)), which leaves the first pair
    and divides the last by the factor. yarn: pair i makes r = original f_i / 2 pi turns over the
    original positions; f is left where r >= 32, divided by the factor where r <= 1 and between the
    two in proportion to r; magnitude 0.1 ln(factor) + 1."""
    i = torch.arange(dim // 2, dtype=torch.float64, device=device)
    f = THETA ** (-2 * i / dim)
    if scaling is None:
        return f, 1.0
    factor = scaling["factor"]
    if scaling["rope_type"] == "linear":
        return f / factor, 1.0
    if scaling["rope_type"] == "ntk":
        return (THETA * factor ** (dim / (dim - 2))) ** (-2 * i / dim), 1.0
    r = scaling["original_max_position_embeddings"] * f / (2 * math.pi)
    keep = ((r - 1) / 31).clamp(0, 1)
    return f * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1


def _plain_rotate(x, positions, dim, layout, scaling):
    """x [rows, heads, 128] turned, in 32 bits (its angles in 64)."""
    f, magnitude = _frequencies(dim, scaling, x.device)
    angle = positions.double()[:, None, None] * f
    c, s = (torch.cos(angle) * magnitude).float(), (torch.sin(angle) * magnitude).float()
    y = x.float().clone()
    head = y[..., :dim]
    a, b = (head[..., :dim // 2], head[..., dim // 2:]) if layout == "half" else \
        (head[..., ::2], head[..., 1::2])
    a2, b2 = a * c - b * s, b * c + a * s
    a.copy_(a2)
    b.copy_(b2)
    return y


def _ends(kind, first, rows, keys, device):
    """How many of the sequence's keys each row sees, always the first ones."""
    p = torch.arange(first, first + rows, device=device)
    if kind == "full":
        return torch.full_like(p, keys)
    block = 1 if kind == "causal" else MASK
    return ((p // block + 1) * block).clamp_max(keys)


def _plain_append(st):
    case = st["case"]
    k = _plain_rotate(st["k"], st["positions"], HD, case["layout"], _scaling(case))
    q = _plain_rotate(st["q"], st["positions"], HD, case["layout"], _scaling(case))
    for pool, x in zip(st["pool"], (k, st["v"])):
        pool.view(-1, pool.shape[2], HD)[st["new"]] = x.to(pool.dtype)
    return q.to(TYPES[case["cache"]])


def _plain_load(st):
    return [pool.view(-1, pool.shape[2], HD)[st["new"]] for pool in st["pool"]]


def _plain_attention(st, q):
    """softmax(q k^T / sqrt(128)) v of each sequence's rows over the keys that they see."""
    case = st["case"]
    hq, hkv = HEADS[case["arch"]]
    outs, r0 = [], 0
    for rows, keys, where in zip(st["rows"], st["keys"], st["where"]):
        k, v = (pool.view(-1, hkv, HD)[where].float().transpose(0, 1).contiguous()
                for pool in st["pool"])
        qg = q[r0:r0 + rows].float().view(rows, hkv, hq // hkv, HD).permute(1, 0, 2, 3)
        qg = qg.reshape(hkv, -1, HD)
        s = torch.matmul(qg, k.transpose(1, 2).contiguous()) / math.sqrt(HD)
        s = s.view(hkv, rows, hq // hkv, keys)
        ends = _ends(case["mask"], keys - rows, rows, keys, q.device)
        seen = torch.arange(keys, device=q.device) < ends[:, None]
        s = s.masked_fill(~seen[None, :, None, :], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o = torch.matmul(p.view(hkv, -1, keys), v).view(hkv, rows, hq // hkv, HD)
        outs.append(o.permute(1, 0, 2, 3).reshape(rows, hq * HD).bfloat16())
        r0 += rows
    return torch.cat(outs)


def _run_plain(st):
    case, kind = st["case"], st["case"]["kind"]
    if kind == "rotate":
        y = _plain_rotate(st["x"], st["positions"], case["dim"], case["layout"], _scaling(case))
        return y.to(st["x"].dtype)
    if kind == "attend":
        return _plain_attention(st, st["q"])
    q = _plain_append(st)
    out = {"q": q} if kind == "append" else {"q": q, "out": _plain_attention(st, q)}
    k, v = _plain_load(st)
    return out | {"k": k, "v": v}


# ---------------------------------------------------------------- one pass, the framework's

def _prepare_own(state):
    from diffusorrt_amd.paged import PagedKVCache
    from diffusorrt_amd.rotary import RotaryPositions, rotary_frequencies

    case = state["case"]
    if case["kind"] != "attend":  # the frequencies that a model keeps (yarn's by turns, as above)
        dim = case.get("dim", HD)
        frequencies, magnitude = rotary_frequencies(dim, THETA, _scaling(case))
        state["rotary"] = RotaryPositions(dim, layout=case["layout"], frequencies=frequencies,
                                          magnitude=magnitude)
    if case["kind"] == "rotate":
        return state
    hq, hkv = HEADS[case["arch"]]
    cache = PagedKVCache(1, hkv, state["pages"], page_size=case["page"], dtype=case["cache"])
    mask = case.get("mask", "causal")
    # what was appended before, and the plan of a step, which serves all layers
    keys, rows = state["keys"], state["rows"]
    cache.append(0, state["old_k"], state["old_v"],
                 cache.batch(state["table"], keys, keys, heads=hq, kind="full"))
    state["batch"] = cache.batch(state["table"], keys, rows, heads=hq,
                                 kind="d2f_hybrid" if mask == "d2f" else mask,
                                 mask_geometry=(0, MASK) if mask == "d2f" else None)
    del state["old_k"], state["old_v"]
    return state | {"cache": cache}


def _run_own(st):
    kind = st["case"]["kind"]
    if kind == "rotate":
        return st["rotary"].rotate(st["x"], st["positions"])
    cache, batch = st["cache"], st["batch"]
    if kind == "attend":
        return cache.attention(0, st["q"], batch, out_dtype=torch.bfloat16)
    q = cache.append(0, st["k"], st["v"], batch, rotary=st["rotary"], q=st["q"])
    out = {"q": q}
    if kind == "step":
        out["out"] = cache.attention(0, q, batch, out_dtype=torch.bfloat16)
    k, v = cache.load(0, batch)
    return out | {"k": k, "v": v}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    hq, hkv = HEADS[case["arch"]]
    if case["kind"] == "rotate":
        n = case["rows"] * hq
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": 2 * n * HD * size + 4 * case["rows"], "flops": 3 * n * case["dim"]}
    rows, keys = _lengths(case)
    n, pages = sum(rows), sum(-(-k // case["page"]) for k in keys)
    out = {"bytes": 0, "flops": 0}
    if case["kind"] != "attend":  # rows in, q and k and v out; load reads k and v and gives them
        src = 4 if case["src"] == "f32" else 2
        out["bytes"] += n * (hq + 2 * hkv) * HD * (src + 2) + 8 * n * hkv * HD
        out["flops"] += 3 * n * (hq + hkv) * HD
    if case["kind"] != "append":
        pairs = sum(int(_ends(case["mask"], k - r, r, k, "cpu").sum())
                    for r, k in zip(rows, keys))
        out["bytes"] += 4 * n * hq * HD + 4 * sum(keys) * hkv * HD + 4 * pages
        out["flops"] += 4 * HD * hq * pairs
    return out


# ---------------------------------------------------------------- in 64 bits, from the definitions

def _exact_rotate(x, positions, dim, layout, scaling):
    """As products of complex numbers."""
    inv = []
    for i in range(dim // 2):
        theta = THETA
        if scaling is not None and scaling["rope_type"] == "ntk":
            theta *= scaling["factor"] ** (dim / (dim - 2))
        f = theta ** (-2.0 * i / dim)
        if scaling is not None and scaling["rope_type"] == "linear":
            f /= scaling["factor"]
        if scaling is not None and scaling["rope_type"] == "yarn":
            turns = scaling["original_max_position_embeddings"] * f / (2 * math.pi)
            share = min(1.0, max(0.0, (turns - 1) / 31))
            f = share * f + (1 - share) * f / scaling["factor"]
        inv.append(f)
    size = 1.0
    if scaling is not None and scaling["rope_type"] == "yarn":
        size = 0.1 * math.log(scaling["factor"]) + 1
    turn = positions.double()[:, None] * torch.tensor(inv, dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.full_like(turn, size), turn)[:, None, :]
    x = x.double()
    head = x[..., :dim].unflatten(-1, (2, dim // 2) if layout == "half" else (dim // 2, 2))
    axis = -2 if layout == "half" else -1
    z = torch.complex(head.select(axis, 0), head.select(axis, 1)) * turn
    return torch.cat([torch.stack([z.real, z.imag], axis).flatten(-2), x[..., dim:]], -1)


def exact(case, seed):
    if case["kind"] == "rotate":
        x, positions = _heads(case, seed)
        return _exact_rotate(x, positions, case["dim"], case["layout"], _scaling(case))
    st = _pool(case, seed)
    hq, hkv = HEADS[case["arch"]]
    q, out = st["q"], {}
    if case["kind"] != "attend":
        positions = _positions(st)
        q = _exact_rotate(q, positions, HD, case["layout"], _scaling(case))
        new = (_exact_rotate(st["k"], positions, HD, case["layout"], _scaling(case)),
               st["v"].double())
        out = {"q": q, "k": new[0], "v": new[1]}
        if case["kind"] == "append":
            return out
        held = TYPES[case["cache"]]  # the cache holds its type's values, and so does q
        q, new = q.to(held), [x.to(held) for x in new]
    o = torch.empty((q.shape[0], hkv, hq // hkv, HD), dtype=torch.float64, device=q.device)
    r0 = k0 = 0
    for rows, keys in zip(st["rows"], st["keys"]):
        k, v = st["old_k"][k0:k0 + keys], st["old_v"][k0:k0 + keys]
        if case["kind"] == "step":
            k, v = (torch.cat([a[:keys - rows], b[r0:r0 + rows]]) for a, b in zip((k, v), new))
        k, v, at = k.double(), v.double(), torch.arange(keys, device=q.device)
        p = torch.arange(keys - rows, keys, device=q.device)[:, None]
        unseen = {"full": at[None] < 0, "causal": at[None] > p,
                  "d2f": at[None] // MASK > p // MASK}[case["mask"]]
        for h in range(hkv):
            for j in range(hq // hkv):
                s = q[r0:r0 + rows, h * (hq // hkv) + j].double() @ k[:, h].t() * HD ** -0.5
                s = torch.softmax(s.masked_fill(unseen, -math.inf), -1)
                o[r0:r0 + rows, h, j] = s @ v[:, h]
        r0, k0 = r0 + rows, k0 + keys
    o = o.reshape(q.shape[0], -1)
    return out | {"out": o} if case["kind"] == "step" else o
