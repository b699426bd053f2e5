"""Cases and plain forms of the decode-step operators: the 4-bit paged cache of
keys and values (append, read, attention, page turnover) and token sampling.

`own = False` computes the plain form with elementary torch operations in 32
bits; `own = True` makes the calls that a user makes of sion_b200. Both take
the state that `prepare` gives.

The cache. A pool is a uint8 tensor [pages, page bytes]; a page holds
`page_size` tokens of every key/value head as [head][block of 16 tokens][K codes
16 x D/2 | V codes 16 x D/2 | K (scale, base) 16 x 2 fp16 | V (scale, base)
16 x 2 fp16]. A token's head vector x is held as x ~ base + scale * (code - 8),
code in 0..15. K codes are row-major, even dimension in the low nibble; the V
code of token 8h + 2t + o and dimension g * D/8 + 4w + i lies in byte
h * 4D + g * D/2 + t * D/8 + 4w + 2o + i // 2, nibble i % 2. `table` [slots,
pages a slot] names each slot's pages, `lens` its tokens, `refs` how many slots
hold a page (0: the page is free).
"""
import math
import random

import numpy as np
import torch

own = False

BLOCK = 16  # tokens of one block of a page


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one conversation answered alone: latency
        {"name": "attend_one", "kind": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "length": 1037, "ragged": False, "rows": 1, "dtype": "f16", "lse": False},
        # a full decode batch of conversations of every length, empty slots among them
        {"name": "attend_batch", "kind": "attend", "batch": 96, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "length": 12288, "ragged": True, "rows": 1, "dtype": "f16",
         "lse": False},
        # long documents, five drafted tokens verified at once, heads of 64 in bf16
        {"name": "attend_long", "kind": "attend", "batch": 4, "heads": 64, "kv_heads": 8, "dim": 64,
         "page": 128, "length": 131071, "ragged": False, "rows": 5, "dtype": "bf16", "lse": True},
        # the tokens of one decode step enter the cache
        {"name": "append_step", "kind": "append", "batch": 64, "kv_heads": 8, "dim": 128,
         "page": 64, "length": 4096, "rows": 1, "dtype": "f16"},
        # prompts of several requests enter the cache
        {"name": "append_prompts", "kind": "append", "batch": 8, "kv_heads": 8, "dim": 128,
         "page": 16, "length": 4096, "rows": 2047, "dtype": "bf16"},
        # between two decode steps: answers that ended leave, others are forked, all get room
        {"name": "turn_small", "kind": "turn", "slots": 16, "pages": 1024, "kv_heads": 8,
         "dim": 128, "page": 64, "length": 2048, "moved": 3},
        # the same for a large pool of small pages
        {"name": "turn_large", "kind": "turn", "slots": 512, "pages": 65536, "kv_heads": 4,
         "dim": 64, "page": 16, "length": 3000, "moved": 129},
        # a fragmented pool is made dense so that its upper part can be given back
        {"name": "compact", "kind": "compact", "slots": 256, "pages": 6007, "kv_heads": 8,
         "dim": 128, "page": 64, "length": 2500},
        # finished prompts move from one pool to another
        {"name": "copy", "kind": "copy", "pages": 2048, "moved": 515, "kv_heads": 8, "dim": 128,
         "page": 32},
        # one answer, all filters
        {"name": "sample_one", "kind": "sample", "batch": 1, "vocab": 32000, "dtype": "f16",
         "top_k": 50, "top_p": 0.95, "min_p": 0.02},
        # a batch with a nucleus only, and an odd vocabulary
        {"name": "sample_nucleus", "kind": "sample", "batch": 33, "vocab": 50021, "dtype": "bf16",
         "top_k": 0, "top_p": 0.9, "min_p": 0.0},
        # a large batch over a large vocabulary
        {"name": "sample_batch", "kind": "sample", "batch": 256, "vocab": 131072, "dtype": "f32",
         "top_k": 1000, "top_p": 0.95, "min_p": 0.0},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    kind = rng.choice(["attend", "attend", "append", "turn", "compact", "copy", "sample", "sample"])
    kv_heads = rng.choice([1, 2, 4, 8])
    dim, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["f16", "bf16"])
    while True:
        if kind == "attend":
            case = {"kind": kind, "batch": _spread(rng, 1, 128),
                    "heads": kv_heads * rng.choice([1, 2, 4, 6, 8]), "kv_heads": kv_heads,
                    "dim": dim, "page": page, "length": _spread(rng, 1, 131071),
                    "ragged": rng.random() < 0.6, "rows": rng.choice([1, 1, 1, 2, 3, 5, 8]),
                    "dtype": dtype, "lse": rng.random() < 0.5}
            slots = case["batch"] * case["length"] * kv_heads * dim
        elif kind == "append":
            case = {"kind": kind, "batch": _spread(rng, 1, 128), "kv_heads": kv_heads, "dim": dim,
                    "page": page, "length": _spread(rng, 4000, 8000),
                    "rows": _spread(rng, 1, 3000), "dtype": dtype}
            slots = case["batch"] * case["length"] * kv_heads * dim
        elif kind in ("turn", "compact"):
            count = _spread(rng, 4, 512)
            length = _spread(rng, 100, 4000)
            case = {"kind": kind, "slots": count,
                    "pages": count * (length // page + 2) + rng.randrange(100), "kv_heads": kv_heads,
                    "dim": dim, "page": page, "length": length}
            if kind == "turn":
                case["moved"] = max(1, count // 4)
            slots = case["pages"] * page * kv_heads * dim
        elif kind == "copy":
            pages = _spread(rng, 8, 4096)
            case = {"kind": kind, "pages": pages, "moved": rng.randrange(1, pages // 2 + 1),
                    "kv_heads": kv_heads, "dim": dim, "page": page}
            slots = pages * page * kv_heads * dim
        else:
            case = {"kind": kind, "batch": _spread(rng, 1, 256), "vocab": _spread(rng, 1000, 200000),
                    "dtype": rng.choice(["f16", "bf16", "f32"]),
                    "top_k": rng.choice([0, 1, 20, 50, 1000]), "top_p": rng.choice([1.0, 0.9, 0.5]),
                    "min_p": rng.choice([0.0, 0.05])}
            slots = 0
        # the padded plain form and the pool have to stay small next to the card
        if _cost(case) <= most and slots <= 96 * 12288 * 8 * 128:
            return case


# ------------------------------------------------- what follows from the case
def _lengths(case, count):
    """Tokens of each slot, from the case alone: one empty slot and one of a
    single token among the ragged ones."""
    rng = random.Random("%s %s" % (case["length"], count))
    if not case.get("ragged", True):
        return [case["length"]] * count
    lens = [rng.randint(1, case["length"]) for _ in range(count)]
    if count > 3:
        lens[count // 2], lens[count // 3], lens[0] = 0, 1, case["length"]
    return lens


def _counts(case, lens):
    """New tokens of each slot: all rows, fewer where the slot has fewer."""
    rng = random.Random("counts %s" % case["rows"])
    counts = [min(n, case["rows"]) for n in lens]
    if case["kind"] == "append" and len(lens) > 2 and case["rows"] > 1:
        counts = [rng.randint(c // 2, c) for c in counts]
    return counts


def _token_bytes(case):
    return case["kv_heads"] * (case["dim"] + 8)


def _page_bytes(case):
    return case["page"] * _token_bytes(case)


def _turn_lists(case):
    """Slots that leave, and (parent, child) pairs that take their places."""
    rng = random.Random("turn %s %s" % (case["slots"], case["moved"]))
    order = list(range(case["slots"]))
    rng.shuffle(order)
    gone, stay = order[:case["moved"]], order[case["moved"]:]
    return gone, [rng.choice(stay) for _ in gone], list(gone)


def _slot_lengths(case):
    """Lengths for the page operations, such that every slot fits the pool."""
    lens = _lengths(case, case["slots"])
    room, page = case["pages"] - case["slots"] - 2, case["page"]
    while sum(-(-n // page) for n in lens) > room:
        lens = [n // 2 for n in lens]
    return lens


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def work(case):
    kind = case["kind"]
    if kind == "attend":
        lens = _lengths(case, case["batch"])
        counts = _counts(case, lens)
        rows = case["batch"] * case["heads"] * case["rows"]
        seen = sum(c * n - c * (c - 1) // 2 for n, c in zip(lens, counts))
        return {"bytes": sum(lens) * _token_bytes(case) + 4 * rows * case["dim"] +
                (4 * rows if case["lse"] else 0) + 4 * sum(-(-n // case["page"]) for n in lens),
                "flops": 4.0 * seen * case["heads"] * case["dim"]}
    if kind == "append":
        counts = _counts(case, [case["length"]] * case["batch"])
        n = sum(counts) * case["kv_heads"]
        # both inputs, the cache written and read back, both outputs and their padding
        return {"bytes": n * (4 * case["dim"] + 2 * (case["dim"] + 8)) +
                4 * case["batch"] * case["rows"] * case["kv_heads"] * case["dim"],
                "flops": 8.0 * n * case["dim"]}
    if kind in ("turn", "compact"):
        lens = _slot_lengths(case)
        width = max(1, -(-(max(lens) + 1) // case["page"]))
        meta = 4 * (2 * case["slots"] * width + 2 * case["pages"] + 2 * case["slots"])
        if kind == "turn":
            _, parents, _ = _turn_lists(case)
            moved = sum(1 for p in parents if lens[p] % case["page"])
        else:
            live = sum(-(-n // case["page"]) for n in lens)
            moved = live * (case["pages"] - live) // case["pages"]
        return {"bytes": meta + 2 * moved * _page_bytes(case), "flops": 0.0}
    if kind == "copy":
        return {"bytes": case["moved"] * (2 * _page_bytes(case) + 8), "flops": 0.0}
    size = 4 if case["dtype"] == "f32" else 2
    n = case["batch"] * case["vocab"]
    return {"bytes": n * size + 28 * case["batch"], "flops": 4.0 * n}


# ----------------------------------------------------------------- the inputs
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _quantise(x):
    """(codes uint8, scale fp16, base fp16) of fp32 head vectors [..., D]."""
    x = x.clamp(-65504.0, 65504.0)
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((hi - lo) / 15).half()
    s = scale.float()
    base = (lo + 8 * s).half()
    code = torch.round((x - base.float()) / s) + 8
    code = torch.where(s > 0, code.clamp(0, 15), torch.full_like(x, 8.0))
    return code.to(torch.uint8), scale, base


def _pack_pages(k, v, pool, first):
    """Writes fp16 K, V [pages, heads, tokens, D] into pool[first:...]."""
    n, heads, page, dim = k.shape
    out = pool[first:first + n].view(n, heads, page // BLOCK, BLOCK * (dim + 8))
    half = BLOCK * dim // 2
    ck, sk, bk = _quantise(k.float())
    cv, sv, bv = _quantise(v.float())
    ck = ck.view(n, heads, page // BLOCK, BLOCK * dim // 2, 2)
    out[..., :half] = ck[..., 0] | (ck[..., 1] << 4)
    cv = cv.view(n, heads, page // BLOCK, 2, 4, 2, 8, dim // 32, 4)  # h t o g w i
    cv = cv.permute(0, 1, 2, 3, 6, 4, 7, 5, 8).reshape(n, heads, page // BLOCK, half, 2)
    out[..., half:2 * half] = cv[..., 0] | (cv[..., 1] << 4)
    for at, s, b in ((2 * half, sk, bk), (2 * half + 4 * BLOCK, sv, bv)):
        par = torch.cat([s, b], -1).view(n, heads, page // BLOCK, 2 * BLOCK)
        out[..., at:at + 4 * BLOCK] = par.view(torch.uint8)


def _fill(pool, case, gen):
    """Keys with a few strong channels and an offset, values around zero."""
    heads, page, dim = case["kv_heads"], case["page"], case["dim"]
    gain = torch.ones(heads, 1, dim, device="cuda")
    gain[..., ::17] = 3.0
    shift = torch.randn(heads, 1, dim, generator=gen, device="cuda") * 0.5
    step = max(1, (1 << 25) // (heads * page * dim))
    for first in range(0, pool.shape[0], step):
        n = min(step, pool.shape[0] - first)
        k = torch.randn(n, heads, page, dim, generator=gen, device="cuda") * gain + shift
        v = torch.randn(n, heads, page, dim, generator=gen, device="cuda") * 0.7
        _pack_pages(k.half(), v.half(), pool, first)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(lens, page, spare, rs):
    """Slots' pages in a random order of the pool, -1 past each slot's end."""
    need = [-(-n // page) for n in lens]
    width = max(1, max(need))
    order = rs.permutation(sum(need) + spare).astype(np.int32)
    table = np.full((len(lens), width), -1, np.int32)
    table[np.arange(width)[None] < np.array(need)[:, None]] = order[:sum(need)]
    return torch.from_numpy(table).cuda(), sum(need) + spare


def _slots_state(case, seed, gen):
    """Slots over a fragmented pool; neighbouring slots share their first pages
    (a common prompt) where both are long enough."""
    rs = np.random.RandomState(seed % (1 << 31))
    lens = _slot_lengths(case)
    page = case["page"]
    need = np.array([-(-n // page) for n in lens])
    width = int(max(1, -(-(max(lens) + 1) // page)))
    order = rs.permutation(case["pages"]).astype(np.int32)
    table = np.full((len(lens), width), -1, np.int32)
    table[np.arange(width)[None] < need[:, None]] = order[:need.sum()]
    if case["kind"] == "turn":
        for s in range(1, len(lens), 2):
            shared = int(min(lens[s - 1], lens[s]) // page // 2)
            table[s, :shared] = table[s - 1, :shared]
    refs = np.bincount(table[table >= 0], minlength=case["pages"]).astype(np.int32)
    pool = torch.randint(0, 256, (case["pages"], _page_bytes(case)), dtype=torch.uint8,
                         device="cuda", generator=gen)
    return {"pages": pool, "table": torch.from_numpy(table).cuda(), "lens": _ints(lens),
            "refs": torch.from_numpy(refs).cuda(), "page": page}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 31))
    kind = case["kind"]
    if kind in ("turn", "compact"):
        s = _slots_state(case, seed, gen)
        if kind == "turn":
            gone, parents, children = _turn_lists(case)
            s.update(gone=_ints(gone), parents=_ints(parents), children=_ints(children),
                     counts=_ints([1] * case["slots"]))
    elif kind == "copy":
        size = (case["pages"], _page_bytes(case))
        s = {"from": torch.randint(0, 256, size, dtype=torch.uint8, device="cuda", generator=gen),
             "to": torch.zeros(size, dtype=torch.uint8, device="cuda"),
             "src": _ints(rs.permutation(case["pages"])[:case["moved"]].tolist()),
             "dst": _ints(rs.permutation(case["pages"])[:case["moved"]].tolist())}
    elif kind == "sample":
        rows, vocab = case["batch"], case["vocab"]
        x = torch.randn(rows, vocab, generator=gen, device="cuda") * 2.0
        # a few likely tokens stand out, and some are forbidden
        x += 9.0 * (torch.rand(rows, vocab, generator=gen, device="cuda") < 20.0 / vocab)
        x[:, 3::101] = float("-inf")
        temp = 0.6 + 0.6 * torch.rand(rows, generator=gen, device="cuda")
        if rows > 4:
            temp[rows // 3] = 0.0  # one greedy row among the others
        s = {"logits": x.to(_TYPES[case["dtype"]]), "temperature": temp,
             "uniform": torch.rand(rows, generator=gen, device="cuda"),
             "top_k": _ints([case["top_k"]] * rows) if case["top_k"] else None,
             "top_p": torch.full((rows,), case["top_p"], device="cuda") if case["top_p"] < 1 else None,
             "min_p": torch.full((rows,), case["min_p"], device="cuda") if case["min_p"] else None}
    else:
        lens = _lengths(case, case["batch"]) if kind == "attend" else [case["length"]] * case["batch"]
        table, total = _table(lens, case["page"], 3, rs)
        pool = torch.zeros(total, _page_bytes(case), dtype=torch.uint8, device="cuda")
        s = {"pages": pool, "table": table, "lens": _ints(lens),
             "counts": _ints(_counts(case, lens)), "kv_heads": case["kv_heads"],
             "dim": case["dim"], "page": case["page"], "rows": case["rows"]}
        if kind == "attend":
            _fill(pool, case, gen)
            q = torch.randn(case["batch"], case["heads"], case["rows"], case["dim"], generator=gen,
                            device="cuda")
            s.update(q=q.to(_TYPES[case["dtype"]]), lse=case["lse"])
        else:
            shape = (case["batch"], case["rows"], 2, case["kv_heads"], case["dim"])
            kv = torch.randn(shape, generator=gen, device="cuda").to(_TYPES[case["dtype"]])
            # K and V as one projection gives them: views [batch, heads, rows, dim]
            s.update(k=kv[:, :, 0].transpose(1, 2), v=kv[:, :, 1].transpose(1, 2))
    s["kind"] = kind
    return s


# ------------------------------------------------------------ the plain forms
def _unpack(raw, dim):
    """fp32 K, V [..., 16, D] of blocks' bytes [..., 16 * (D + 8)]."""
    half = BLOCK * dim // 2
    lead = raw.shape[:-1]

    def params(at):
        p = raw[..., at:at + 4 * BLOCK].contiguous().view(torch.float16).view(*lead, BLOCK, 2)
        return p[..., :1].float(), p[..., 1:].float()

    def codes(b):
        return torch.stack([b & 15, b >> 4], -1).float() - 8

    ks, kb = params(2 * half)
    vs, vb = params(2 * half + 4 * BLOCK)
    k = codes(raw[..., :half]).view(*lead, BLOCK, dim)
    v = codes(raw[..., half:2 * half]).view(*lead, 2, 8, 4, dim // 32, 2, 4)  # h g t w o i
    n = len(lead)
    v = v.permute(*range(n), n, n + 2, n + 4, n + 1, n + 3, n + 5).reshape(*lead, BLOCK, dim)
    return kb + ks * k, vb + vs * v


def _gather(s):
    """fp32 K, V [batch, kv heads, tokens, D] of the tables' pages."""
    b, width = s["table"].shape
    raw = s["pages"][s["table"].clamp(min=0).long()]
    raw = raw.view(b, width, s["kv_heads"], s["page"] // BLOCK, BLOCK * (s["dim"] + 8))
    k, v = _unpack(raw.transpose(1, 2), s["dim"])
    shape = (b, s["kv_heads"], width * s["page"], s["dim"])
    return k.reshape(shape), v.reshape(shape)


def _attend(s):
    q = s["q"].float()
    b, heads, rows, dim = q.shape
    k, v = _gather(s)
    group = heads // s["kv_heads"]
    q = q.view(b, s["kv_heads"], group * rows, dim)
    scores = torch.matmul(q, k.transpose(2, 3)).view(b, s["kv_heads"], group, rows, -1)
    scores *= 1 / math.sqrt(dim)
    row = torch.arange(rows, device=q.device)[None]
    lens, counts = s["lens"][:, None], s["counts"][:, None]
    last = torch.where(row < counts, lens - counts + row, -1)  # the last token a row sees
    seen = torch.arange(scores.shape[-1], device=q.device) <= last[..., None]
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == float("-inf"), 0.0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, s["kv_heads"], group * rows, -1), v)
    o = o.view(b, heads, rows, dim) / total.view(b, heads, rows, 1).clamp(min=1e-30)
    lse = (top + torch.log(total)).view(b, heads, rows)
    return o.to(s["q"].dtype), lse


def _places(s):
    """Byte offset of each row's token block [batch, rows, heads], its place in
    the block, and which rows are tokens."""
    b, rows = s["table"].shape[0], s["rows"]
    row = torch.arange(rows, device=s["lens"].device)[None]
    at = (s["lens"] - s["counts"])[:, None] + row
    valid = row < s["counts"][:, None]
    at = torch.where(valid, at, 0).long()
    page = torch.gather(s["table"].long(), 1, at // s["page"])
    inside, size = at % s["page"], BLOCK * (s["dim"] + 8)
    head = torch.arange(s["kv_heads"], device=at.device)
    block = page[..., None] * s["pages"].shape[1] + \
        (head * (s["page"] // BLOCK) + (inside // BLOCK)[..., None]) * size
    return block.view(b, rows, -1), (inside % BLOCK)[..., None], valid


def _byte_order(dim, r, device):
    """Offsets in a block of the D/2 K bytes and the D/2 V bytes of token r."""
    j = torch.arange(dim // 2, device=device)
    d = 2 * j
    g, w, i = d // (dim // 8), d % (dim // 8) // 4, d % 4
    r = r[..., None]
    k = r * (dim // 2) + j
    v = BLOCK * dim // 2 + (r // 8) * 4 * dim + g * (dim // 2) + (r % 8 // 2) * (dim // 8) + \
        4 * w + 2 * (r % 2) + i // 2
    return k, v


def _append(s):
    dim, flat = s["dim"], s["pages"].view(-1)
    block, r, valid = _places(s)
    put = []
    orders = _byte_order(dim, r, flat.device)
    for n, x in enumerate((s["k"], s["v"])):
        code, scale, base = _quantise(x.transpose(1, 2).float())
        put.append((block[..., None] + orders[n], code[..., 0::2] | (code[..., 1::2] << 4)))
        par = torch.cat([scale, base], -1).view(torch.uint8)
        at = BLOCK * dim + n * 4 * BLOCK + 4 * r
        put.append((block[..., None] + at[..., None] + torch.arange(4, device=flat.device), par))
    for at, what in put:
        flat[at[valid]] = what[valid]
    out = []
    for n in range(2):  # what the cache now holds for these tokens
        codes, par = flat[put[2 * n][0]], flat[put[2 * n + 1][0]].view(torch.float16).float()
        c = torch.stack([codes & 15, codes >> 4], -1).float().view(*codes.shape[:-1], dim) - 8
        x = par[..., 1:] + par[..., :1] * c
        x = torch.where(valid[..., None, None], x, 0.0)
        out.append(x.half().transpose(1, 2).contiguous())
    return tuple(out)


def _pages_of(n, page):
    return (n + page - 1) // page


def _free(table, lens, refs, gone, page):
    leave = torch.zeros_like(lens, dtype=torch.bool)
    leave[gone.long()] = True
    col = torch.arange(table.shape[1], device=table.device)[None]
    held = leave[:, None] & (col < _pages_of(lens, page)[:, None])
    drop = torch.zeros_like(refs).scatter_add_(
        0, table.clamp(min=0).long().view(-1), held.to(refs.dtype).view(-1))
    return (torch.where(leave[:, None], -1, table), torch.where(leave, 0, lens), refs - drop)


def _free_pages(refs):
    """Page numbers, the free ones first, each part in ascending order."""
    return torch.argsort((refs != 0).to(torch.uint8), stable=True).to(torch.int32)


def _fork(pages, table, lens, refs, parents, children, page):
    p, c = parents.long(), children.long()
    earlier = torch.tril(c[:, None] == c[None], -1).any(1)
    valid = (p != c) & (lens[c] == 0) & ~earlier
    skipped = (~valid).sum()
    need = valid & (lens[p] % page != 0)
    rank = torch.cumsum(need, 0) - 1
    total, room = need.sum(), (refs == 0).sum()
    fits = total <= room
    valid, need = valid & fits, need & fits
    fresh = _free_pages(refs)[rank.clamp(0, refs.numel() - 1)]
    col = torch.arange(table.shape[1], device=table.device)[None]
    whole = lens[p] // page
    shared = valid[:, None] & (col < whole[:, None])
    rows = torch.where(shared, table[p], -1)
    rows = torch.where(need[:, None] & (col == whole[:, None]), fresh[:, None], rows)
    add = torch.zeros_like(refs).scatter_add_(
        0, table[p].clamp(min=0).long().view(-1), shared.to(refs.dtype).view(-1))
    refs = refs + add
    refs[fresh[need].long()] = 1
    table, new_lens = table.clone(), lens.clone()
    last = table[p, (whole.clamp(max=table.shape[1] - 1)).long()]
    table[c[valid]] = rows[valid]
    new_lens[c[valid]] = lens[p][valid]
    pages[fresh[need].long()] = pages[last[need].long()]
    status = torch.stack([(total - room).clamp(min=0), skipped]).to(torch.int32)
    return table, new_lens, refs, status


def _reserve(table, lens, refs, counts, page):
    old, new = _pages_of(lens, page), _pages_of(lens + counts, page)
    need = new - old
    start = torch.cumsum(need, 0) - need
    total, room = need.sum(), (refs == 0).sum()
    fits = total <= room
    col = torch.arange(table.shape[1], device=table.device)[None]
    given = fits & (col >= old[:, None]) & (col < new[:, None])
    rank = (start[:, None] + col - old[:, None]).clamp(0, refs.numel() - 1)
    order = _free_pages(refs)
    refs = torch.where(torch.arange(refs.numel(), device=refs.device) < torch.where(fits, total, 0),
                       1, refs[order.long()])
    refs = torch.empty_like(refs).scatter_(0, order.long(), refs)
    table = torch.where(given, order[rank.long()], table)
    status = torch.stack([(total - room).clamp(min=0), torch.zeros_like(total)]).to(torch.int32)
    return table, torch.where(fits, lens + counts, lens).to(torch.int32), refs.to(torch.int32), status


def _compact(pages, table, refs):
    live = refs > 0
    count = live.sum()
    at = torch.arange(refs.numel(), device=refs.device)
    src, dst = at[live & (at >= count)], at[~live & (at < count)]
    to = at.to(torch.int32)
    to[src] = dst.to(torch.int32)
    pages[dst] = pages[src]
    out = torch.zeros_like(refs)
    out[to[live].long()] = refs[live]
    return torch.where(table >= 0, to[table.clamp(min=0).long()], -1), out


def _sample(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    x = torch.where(torch.isnan(x), float("-inf"), x)
    temp = s["temperature"][:, None]
    top = x.amax(-1, keepdim=True)
    z = torch.where(x == top, 0.0, x - top) / torch.where(temp > 0, temp, 1.0)
    w = torch.exp(z)
    mass = torch.round(w * 2.0 ** 31).to(torch.int64)  # probabilities in fixed point
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ranked = torch.gather(mass, 1, order)
    keep = torch.arange(vocab, device=x.device)[None].expand(rows, vocab)
    k = vocab if s["top_k"] is None else torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    keep = keep < k
    if s["top_p"] is not None:
        ranked = torch.where(keep, ranked, 0)
        before = torch.cumsum(ranked, 1) - ranked
        p = s["top_p"].double()[:, None]
        keep = keep & ((before < p * ranked.sum(1, keepdim=True)) | (p >= 1))
    if s["min_p"] is not None:
        keep = keep & (torch.gather(w, 1, order) >= s["min_p"][:, None])
    keep[:, 0] = True
    mass = torch.where(torch.empty_like(keep).scatter_(1, order, keep), mass, 0)
    upto = torch.cumsum(mass, 1)
    total = upto[:, -1:]
    target = (s["uniform"].double()[:, None] * total).floor().to(torch.int64)
    token = torch.searchsorted(upto, torch.minimum(target, total - 1), right=True)
    greedy = (x == top).to(torch.uint8).argmax(1, keepdim=True)
    token = torch.where(temp > 0, token, greedy)
    logprob = torch.gather(z, 1, token) - torch.log(total.float() * 2.0 ** -31)
    logprob = torch.where(temp > 0, logprob, 0.0)
    none = top == float("-inf")
    token = torch.where(none, -1, token).to(torch.int32)
    return token[:, 0], torch.where(none, float("-inf"), logprob)[:, 0]


# ------------------------------------------------------------------- one pass
def run(state):
    s, kind = state, state["kind"]
    if own:
        import sion_b200 as sion
        if kind == "attend":
            if s["lse"]:
                return sion.kv4_attention_lse(s["q"], s["pages"], s["table"], s["lens"],
                                              s["kv_heads"], counts=s["counts"])
            return sion.kv4_attention(s["q"], s["pages"], s["table"], s["lens"], s["kv_heads"],
                                      counts=s["counts"])
        if kind == "append":
            sion.kv4_append(s["pages"], s["table"], s["lens"], s["k"], s["v"], counts=s["counts"])
            return sion.kv4_read(s["pages"], s["table"], s["lens"], s["rows"], s["kv_heads"],
                                 s["dim"], counts=s["counts"])
        if kind == "turn":
            table, lens, refs = sion.kv4_free(s["table"], s["lens"], s["refs"], s["gone"], s["page"])
            table, lens, refs, forked = sion.kv4_fork(s["pages"], table, lens, refs, s["parents"],
                                                      s["children"], s["page"])
            table, lens, refs, given = sion.kv4_reserve(table, lens, refs, s["counts"], s["page"])
            return table, lens, refs, forked, given, s["pages"]
        if kind == "compact":
            table, refs = sion.kv4_compact(s["pages"], s["table"], s["refs"])
            return table, refs, s["pages"]
        if kind == "copy":
            sion.kv4_copy_pages(s["from"], s["to"], s["src"], s["dst"])
            return s["to"]
        return sion.sample(s["logits"], s["uniform"], temperature=s["temperature"],
                           top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    if kind == "attend":
        o, lse = _attend(s)
        return (o, lse) if s["lse"] else o
    if kind == "append":
        return _append(s)
    if kind == "turn":
        table, lens, refs = _free(s["table"], s["lens"], s["refs"], s["gone"], s["page"])
        table, lens, refs, forked = _fork(s["pages"], table, lens, refs, s["parents"],
                                          s["children"], s["page"])
        table, lens, refs, given = _reserve(table, lens, refs, s["counts"], s["page"])
        return table, lens, refs, forked, given, s["pages"]
    if kind == "compact":
        table, refs = _compact(s["pages"], s["table"], s["refs"])
        return table, refs, s["pages"]
    if kind == "copy":
        s["to"][s["dst"].long()] = s["from"][s["src"].long()]
        return s["to"]
    return _sample(s)


# ------------------------------------------- the definitions in 64 bits
def _exact_attend(case, s):
    dim, page, kvh = s["dim"], s["page"], s["kv_heads"]
    d = torch.arange(dim, device="cuda")
    lens, counts = s["lens"].tolist(), s["counts"].tolist()
    b, heads, rows, _ = s["q"].shape
    o = torch.zeros(b, heads, rows, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((b, heads, rows), -math.inf, dtype=torch.float64, device="cuda")
    unit = BLOCK * (dim + 8)
    for i in range(b):
        if not lens[i]:
            continue
        at = torch.arange(lens[i], device="cuda")
        raw = s["pages"][s["table"][i].clamp(min=0).long()].view(-1, kvh, page // BLOCK, unit)
        r = at % BLOCK
        kat = (r * (dim // 2))[:, None] + d // 2
        e = d % (dim // 8)
        vat = 8 * dim + ((r // 8) * 4 * dim + (r % 8 // 2) * (dim // 8) + 2 * (r % 2))[:, None] + \
            d // (dim // 8) * (dim // 2) + e // 4 * 4 + e % 4 // 2
        for h in range(kvh):
            blocks = raw[:, h].reshape(-1, unit)[:-(-lens[i] // BLOCK)]
            vectors = []
            for place, odd, par in ((kat, d % 2, 16 * dim), (vat, e % 2, 16 * dim + 64)):
                code = blocks.view(-1)[(at // BLOCK * unit)[:, None] + place].to(torch.int32)
                code = (code >> (4 * odd)) & 15
                sb = blocks[:, par:par + 64].contiguous().view(torch.float16).double().view(-1, 2)
                sb = sb[:lens[i]]
                vectors.append(sb[:, 1:] + sb[:, :1] * (code.double() - 8))
            k, v = vectors
            group = heads // kvh
            for j in range(counts[i]):
                end = lens[i] - counts[i] + j + 1
                x = s["q"][i, h * group:(h + 1) * group, j].double() @ k[:end].T / math.sqrt(dim)
                lse[i, h * group:(h + 1) * group, j] = torch.logsumexp(x, -1)
                o[i, h * group:(h + 1) * group, j] = torch.softmax(x, -1) @ v[:end]
    return (o, lse) if case["lse"] else o


def _exact_append(s):
    out = []
    rows, counts = s["rows"], s["counts"]
    valid = torch.arange(rows, device="cuda")[None] < counts[:, None]
    for x in (s["k"], s["v"]):
        x = x.double()
        lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
        # scale and base are what the cache stores: fp16 values
        scale = ((hi - lo) / 15).half().double()
        base = (lo + 8 * scale).half().double()
        code = (torch.round((x - base) / scale) + 8).clamp(0, 15)
        out.append((base + scale * (code - 8)) * valid[:, None, :, None])
    return tuple(out)


def _exact_sample(s):
    x = s["logits"].double().cpu().numpy()
    got = []
    for i in range(x.shape[0]):
        temp, u = float(s["temperature"][i]), float(s["uniform"][i])
        if temp <= 0:
            got.append(0.0)
            continue
        row = (x[i] - x[i].max()) / temp
        order = np.argsort(-row, kind="stable")
        w = np.exp(row)
        k = int(s["top_k"][i]) if s["top_k"] is not None else 0
        n = k if k > 0 else len(row)
        if s["top_p"] is not None:
            upto = np.cumsum(w[order[:n]])
            n = min(n, 1 + int(np.sum(upto < float(s["top_p"][i]) * upto[-1])))
        kept = np.zeros(len(row), bool)
        kept[order[:n]] = True
        if s["min_p"] is not None:
            kept &= w >= float(s["min_p"][i])
        w = np.where(kept, w, 0.0)
        upto = np.cumsum(w)
        token = min(int(np.searchsorted(upto, u * upto[-1], side="right")), len(row) - 1)
        got.append(row[token] - math.log(upto[-1]))
    return None, torch.tensor(got, dtype=torch.float64)


def exact(case, seed):
    if case["kind"] in ("turn", "compact", "copy"):
        return None  # page numbers, counts and bytes only
    s = prepare(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(case, s)
    if case["kind"] == "append":
        return _exact_append(s)
    return _exact_sample(s)
