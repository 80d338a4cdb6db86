"""The paged 8-bit key/value cache and the attention over it, as timed cases with their plain forms.

A case is one pass through what a serving program does with the cache (`kaio_b200.kv_cache.PagedKvInt8`):
rotating and appending a step's keys and values and reading them back, reading a cache back as dense
rows, or attending to it.  Head layouts are those of the 7B (32 heads of 128) and 70B (64 query heads
over 8 key/value heads) layers the benchmark uses and of the small shapes the tests carry; `draw`
spreads the same operations over batch, lengths, head layouts, head sizes and page sizes.
"""
import math
import random

import torch

own = False

BLOCK = 16                 # tokens that share a scale
SCALE_MIN = 2.0 ** -40     # the smallest scale
LARGEST = 131008.0         # what an infinite value is held as: twice the largest f16


def listed():
    return [
        # one sequence's next token, 7B heads: the smallest append, where the launch counts
        {"name": "append step b1", "kind": "append", "batch": 1, "new": 1, "kv": 21, "ragged": False, "heads": 32, "kv_heads": 32,
         "d": 128, "page": 16, "rot": 128, "interleaved": False, "mix": 1},
        # the next token of 64 short conversations, 70B heads: old tokens of a block may have to be scaled down
        {"name": "append step b64", "kind": "append", "batch": 64, "new": 1, "kv": 120, "ragged": True, "heads": 64, "kv_heads": 8,
         "d": 128, "page": 64, "rot": 128, "interleaved": False, "mix": 2},
        # three ragged prompts, 70B heads: every block is written whole
        {"name": "append prompts", "kind": "append", "batch": 3, "new": 1777, "kv": 1777, "ragged": True, "heads": 64, "kv_heads": 8,
         "d": 128, "page": 64, "rot": 128, "interleaved": False, "mix": 3},
        # a short prefix read back, head size 64
        {"name": "gather small", "kind": "gather", "batch": 1, "kv": 333, "ragged": False, "heads": 16, "kv_heads": 8, "d": 64,
         "page": 16, "mix": 4},
        # the caches of eight ragged sequences read back, 7B heads
        {"name": "gather b8", "kind": "gather", "batch": 8, "kv": 2000, "ragged": True, "heads": 32, "kv_heads": 32, "d": 128,
         "page": 64, "mix": 5},
        # one sequence's next token over a short cache, 7B heads: the smallest attention
        {"name": "attend step b1", "kind": "attend", "batch": 1, "new": 1, "kv": 500, "ragged": False, "heads": 32, "kv_heads": 32,
         "d": 128, "page": 64, "causal": True, "mix": 6},
        # one token of eight sequences over 2000 cached ones, 7B heads: the decode step of the benchmark's attention
        {"name": "attend step b8", "kind": "attend", "batch": 8, "new": 1, "kv": 2000, "ragged": False, "heads": 32, "kv_heads": 32,
         "d": 128, "page": 64, "causal": True, "mix": 7},
        # one token of 64 ragged sequences, 70B heads: a serving batch
        {"name": "attend step b64 ragged", "kind": "attend", "batch": 64, "new": 1, "kv": 7000, "ragged": True, "heads": 64,
         "kv_heads": 8, "d": 128, "page": 64, "causal": True, "mix": 8},
        # one token over a long document, 70B heads: few rows, one long axis
        {"name": "attend long b1", "kind": "attend", "batch": 1, "new": 1, "kv": 100001, "ragged": False, "heads": 64,
         "kv_heads": 8, "d": 128, "page": 128, "causal": True, "mix": 9},
        # three drafted tokens of twelve sequences to be verified, head size 64, four query heads to a key head
        {"name": "attend verify b12 d64", "kind": "attend", "batch": 12, "new": 3, "kv": 1111, "ragged": True, "heads": 16,
         "kv_heads": 4, "d": 64, "page": 16, "causal": True, "mix": 10},
        # a 512-token chunk of a prompt whose first 8192 tokens are cached, 70B heads
        {"name": "attend chunk 512", "kind": "attend", "batch": 1, "new": 512, "kv": 8704, "ragged": False, "heads": 64,
         "kv_heads": 8, "d": 128, "page": 64, "causal": True, "mix": 11},
        # four ragged prompts at once, 7B heads
        {"name": "attend prompts b4", "kind": "attend", "batch": 4, "new": 2048, "kv": 2048, "ragged": True, "heads": 32,
         "kv_heads": 32, "d": 128, "page": 64, "causal": True, "mix": 12},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads, kv_heads = rng.choice([(32, 32), (64, 8), (64, 8), (32, 8), (16, 4), (8, 8), (16, 1), (12, 4)])
    case = {"kind": rng.choice(["append", "append", "gather", "attend", "attend", "attend", "attend"]), "batch": _log(rng, 1, 64), "ragged": rng.random() < 0.6,
            "heads": heads, "kv_heads": kv_heads, "d": rng.choice([64, 128, 128]), "page": rng.choice([16, 32, 64, 128]),
            "mix": rng.randrange(1 << 20)}
    width = kv_heads * case["d"]
    if case["kind"] == "gather":
        case["kv"] = min(_log(rng, 1, 16384), max(1, 65_000_000 // (width * case["batch"])))
        return case
    if case["kind"] == "append":
        case["new"] = 1 if rng.random() < 0.5 else min(_log(rng, 2, 4096), max(2, 5000 // case["batch"]))
        # what was there before stays short: a pass reads the cache back
        case["kv"] = case["new"] + rng.choice([0, rng.randrange(64)])
        case["rot"] = rng.choice([case["d"], case["d"], case["d"] // 2, 32])
        case["interleaved"] = rng.random() < 0.3
        return case
    form = rng.choice(["one", "one", "few", "chunk"])
    case["causal"] = rng.random() < 0.85
    case["new"] = 1 if form == "one" else rng.randrange(2, 9) if form == "few" else _log(rng, 16, 1024)
    if form == "chunk":
        case["batch"] = min(case["batch"], max(1, 2048 // case["new"]))
    room = min(230_000_000 // (width * case["batch"]), 60_000_000_000 // (4 * case["d"] * heads * case["batch"] * case["new"]),
               400_000_000 // (heads * case["batch"] * case["new"]))
    case["kv"] = max(case["new"], min(_log(rng, case["new"], 65536), room))
    return case


def lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence; they are the case's, not the seed's."""
    r = random.Random(case["mix"])
    new, kv = case.get("new", 0), case["kv"]
    got = []
    for _ in range(case["batch"]):
        n, old = new, kv - new
        if case["ragged"]:
            n = n if n <= 8 else r.randint(max(1, n // 4), n)
            old = r.randint(old // 8, old) if old else 0
        got.append((n, n + old))
    return got


def _sizes(case):
    return case["batch"], case["heads"], case["kv_heads"], case["d"], case["page"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    b, h, hk, d, page = _sizes(case)
    lens = lengths(case)
    new, kv = [n for n, _ in lens], [k for _, k in lens]
    pages = [-(-k // page) for k in kv]
    s = {"case": case, "tokens": sum(new), "max_new": max(new), "total": sum(kv), "num_pages": sum(pages) + 3}

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    def starts(v):
        return ints([sum(v[:i]) for i in range(len(v) + 1)])

    s["q_start"], s["kv_start"], s["kv_len"] = starts(new), starts(kv), ints(kv)
    # the pages of a server that has run for a while: in no order, entries past the end left from before
    order = torch.randperm(s["num_pages"], generator=gen, device="cuda").to(torch.int32)
    table = torch.full((b, max(pages)), s["num_pages"] - 1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    s["table"] = table
    shape = (s["num_pages"], hk, page, d)
    # what normally distributed keys and values leave behind: the largest of each block of 16 tokens at 127
    for name in ("k", "v"):
        s[name + "_cache"] = torch.empty(shape, dtype=torch.int8, device="cuda")
        for i in range(0, s["num_pages"], 4096):
            part = s[name + "_cache"][i:i + 4096]
            part.copy_(torch.randn(part.shape, generator=gen, device="cuda").mul_(36.0).round_().clamp_(-127, 127))
        s[name + "_scale"] = torch.rand((s["num_pages"], hk, page // BLOCK), generator=gen, device="cuda").mul_(0.02).add_(0.018)
    t = s["tokens"]
    if case["kind"] != "gather":
        s["q"] = torch.randn(t, h * d, generator=gen, device="cuda").half()
    if case["kind"] == "append":
        s["k"], s["v"] = [torch.randn(t, hk * d, generator=gen, device="cuda").half() for _ in range(2)]
        # a channel or two of the keys is far larger than the rest, as in trained models
        s["k"].view(t, hk, d)[:, :, 5] *= 6.0
        half = case["rot"] // 2
        angle = torch.arange(max(kv), dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    if own:
        from kaio_b200 import ops
        from kaio_b200.kv_cache import PagedKvInt8
        dev = ops.KaioDevice(0)
        s["cache"] = PagedKvInt8(ops, dev, s["num_pages"], h, hk, d, page, storage=(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]))
        if case["kind"] != "gather":
            s["out"] = torch.empty(t, h * d, dtype=torch.float16, device="cuda")
        if case["kind"] == "attend":
            s["scratch"] = s["cache"].scratch(b, t, s["max_new"])
        else:
            s["k_out"], s["v_out"] = [torch.empty(s["total"], hk * d, dtype=torch.float16, device="cuda") for _ in range(2)]
    return s


# ---------------------------------------------------------------- plain forms

def _places(s, start, rows, first):
    """For each row of a ragged batch (start: rows before each sequence): its sequence, its position, and the page, scale
    block and slot that hold it; `first`: the position of each sequence's first row."""
    page = s["case"]["page"]
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(start[1:].long(), row, right=True)
    pos = row - start[seq] + first[seq]
    return pos, s["table"][seq, pos // page].long(), pos % page // BLOCK, pos % BLOCK


def _rotate(x, cos, sin, rot, interleaved):
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    c, n = cos[:, None], sin[:, None]
    y0, y1 = a * c - b * n, b * c + a * n
    y = torch.stack((y0, y1), -1).flatten(-2) if interleaved else torch.cat((y0, y1), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _store(s, name, x, first, page, block, slot):
    """x f32 [tokens, kv_heads, d] into the cache: a block's scale may grow, its older tokens are scaled down to it."""
    _, _, hk, d, size = _sizes(s["case"])
    cache, scale = s[name + "_cache"], s[name + "_scale"]
    # the blocks that get new tokens, as many for each sequence as the longest may touch: the last one stands for the rest
    at = torch.minimum((first // BLOCK)[:, None] + torch.arange((s["max_new"] + 2 * BLOCK - 2) // BLOCK, device="cuda"),
                       ((s["kv_len"] - 1) // BLOCK)[:, None])
    inside = at % (size // BLOCK)
    where = s["table"].gather(1, (at // (size // BLOCK)).long()).long()
    top = torch.nan_to_num(x.abs(), nan=0.0).clamp(max=LARGEST).amax(-1)
    cells = torch.zeros(s["num_pages"] * (size // BLOCK), hk, device="cuda")
    largest = cells.scatter_reduce(0, (page * (size // BLOCK) + block)[:, None].expand(-1, hk), top, "amax")
    old = torch.where((at * BLOCK >= first[:, None])[..., None], 0.0, scale[where, :, inside])
    new = torch.maximum(largest[where * (size // BLOCK) + inside] / 127.0, old).clamp(min=SCALE_MIN)
    held = cache.view(s["num_pages"], hk, size // BLOCK, BLOCK, d)
    ratio = torch.where(new > old, old / new, 1.0)
    held[where, :, inside] = torch.round(held[where, :, inside].float() * ratio[..., None, None]).to(torch.int8)
    scale[where, :, inside] = new
    q = torch.nan_to_num(x * (1.0 / scale[page, :, block])[..., None], nan=0.0).clamp(-127.0, 127.0)
    cache[page, :, block * BLOCK + slot] = q.round().to(torch.int8)


def _read(s, name, page, block, slot):
    x = s[name + "_cache"][page, :, block * BLOCK + slot].float()
    return x * s[name + "_scale"][page, :, block].clamp(min=SCALE_MIN)[..., None]


def _plain_append(s):
    case = s["case"]
    _, h, hk, d, _ = _sizes(case)
    first = s["kv_len"] - (s["q_start"][1:] - s["q_start"][:-1])
    pos, *at = _places(s, s["q_start"], s["tokens"], first)
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotate(s["q"].view(-1, h, d).float(), cos, sin, case["rot"], case["interleaved"]).half()
    _store(s, "k", _rotate(s["k"].view(-1, hk, d).float(), cos, sin, case["rot"], case["interleaved"]), first, *at)
    _store(s, "v", s["v"].view(-1, hk, d).float(), first, *at)
    return {"q": q.view(-1, h * d), **_plain_gather(s)}


def _plain_gather(s):
    _, *at = _places(s, s["kv_start"], s["total"], torch.zeros_like(s["kv_len"]))
    return {n: _read(s, n, *at).half().flatten(1) for n in ("k", "v")}


def _plain_attend(s):
    case = s["case"]
    _, h, hk, d, page = _sizes(case)
    new = s["q_start"][1:] - s["q_start"][:-1]
    longest = s["table"].shape[1] * page
    j = torch.arange(longest, device="cuda")
    where = s["table"][:, j // page].long()
    # [batch, keys, kv_heads, d] with keys past a sequence's end masked below
    k, v = [s[n + "_cache"][where, :, j % page].float() * s[n + "_scale"][where, :, j % page // BLOCK].clamp(min=SCALE_MIN)[..., None]
            for n in ("k", "v")]
    i = torch.arange(s["max_new"], device="cuda")
    row = s["q_start"][:-1, None] + i
    q = s["q"].view(-1, hk, h // hk, d)[row.clamp(max=s["tokens"] - 1)].float()
    x = torch.einsum("bihgd,bjhd->bhgij", q, k) / math.sqrt(d)
    last = s["kv_len"][:, None] - (new[:, None] - i if case["causal"] else 0 * i)
    end = last + 1 if case["causal"] else last
    seen = j < end[:, :, None]
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1)
    o = torch.einsum("bhgij,bjhd->bihgd", p, v) / total.clamp(min=1e-30).permute(0, 3, 1, 2)[..., None]
    token = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["q_start"][1:].long(), token, right=True)
    return o[seq, token - s["q_start"][seq]].half().flatten(1)


def run(s):
    case = s["case"]
    if own:
        cache = s["cache"]
        if case["kind"] == "append":
            cache.append(s["q"], s["k"], s["v"], s["out"], s["cos"], s["sin"], s["table"], s["q_start"], s["kv_len"],
                         rot_dim=case["rot"], interleaved=case["interleaved"])
        if case["kind"] == "attend":
            cache.attend(s["q"], s["out"], s["table"], s["q_start"], s["kv_len"], s["max_new"], causal=case["causal"], scratch=s["scratch"])
            return {"out": s["out"]}
        cache.gather(s["k_out"], s["v_out"], s["table"], s["kv_start"])
        got = {"k": s["k_out"], "v": s["v_out"]}
        return {"q": s["out"], **got} if case["kind"] == "append" else got
    if case["kind"] == "append":
        return _plain_append(s)
    return _plain_gather(s) if case["kind"] == "gather" else {"out": _plain_attend(s)}


# ---------------------------------------------------------------- from the definition, in 64 bits

def _exact_block(x, old_q, old_scale):
    """What a block holds after the rows x [n, heads, d] join the rows old_q [m, heads, d] with scales old_scale [heads]."""
    a = x.abs().amax((0, 2)) / 127.0
    scale = a.clamp(min=SCALE_MIN)
    if old_q.shape[0]:
        scale = torch.maximum(scale, old_scale)
        ratio = torch.where(scale > old_scale, old_scale / scale, torch.ones_like(scale))
        old_q = torch.round(old_q * ratio[None, :, None])
    q = torch.cat((old_q, torch.round(x / scale[None, :, None]).clamp(-127, 127)))
    return q * scale[None, :, None]


def exact(case, seed):
    s = prepare(case, seed)
    b, h, hk, d, page = _sizes(case)
    lens, table = lengths(case), s["table"].cpu()
    outs = {"q": [], "k": [], "v": [], "out": []}
    row = 0
    for i, (n, kv) in enumerate(lens):
        pages = table[i, :-(-kv // page)].long().cuda()
        held, scales = {}, {}
        for name in ("k", "v"):
            c = s[name + "_cache"][pages].double().transpose(1, 2).reshape(-1, hk, d)
            z = s[name + "_scale"][pages].double().clamp(min=SCALE_MIN).transpose(1, 2).reshape(-1, hk)
            held[name], scales[name] = c, z
        if case["kind"] == "append":
            pos = torch.arange(kv - n, kv, device="cuda")
            fresh = {"v": s["v"][row:row + n].double().view(n, hk, d)}
            for name, heads in (("q", h), ("k", hk)):
                x = s[name][row:row + n].double().view(n, heads, d)
                y, half = x.clone(), case["rot"] // 2
                e = torch.arange(half, device="cuda")
                one, two = (2 * e, 2 * e + 1) if case["interleaved"] else (e, e + half)
                c, z = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
                y[:, :, one], y[:, :, two] = x[:, :, one] * c - x[:, :, two] * z, x[:, :, two] * c + x[:, :, one] * z
                fresh[name] = y
            outs["q"].append(fresh["q"].reshape(n, h * d))
            for name in ("k", "v"):
                values = held[name][:kv] * scales[name].repeat_interleave(BLOCK, 0)[:kv, :, None]
                for block in range((kv - n) // BLOCK, -(-kv // BLOCK)):
                    lo, hi, mid = block * BLOCK, min(kv, (block + 1) * BLOCK), max(kv - n, block * BLOCK)
                    values[lo:hi] = _exact_block(fresh[name][mid - (kv - n):hi - (kv - n)], held[name][lo:mid], scales[name][block])
                outs[name].append(values.reshape(kv, hk * d))
        else:
            k, v = [held[name][:kv] * scales[name].repeat_interleave(BLOCK, 0)[:kv, :, None] for name in ("k", "v")]
            if case["kind"] == "gather":
                outs["k"].append(k.reshape(kv, hk * d))
                outs["v"].append(v.reshape(kv, hk * d))
            else:
                o = torch.empty(n, h, d, dtype=torch.float64, device="cuda")
                hidden = torch.arange(kv, device="cuda") > torch.arange(kv - n, kv, device="cuda")[:, None]
                for head in range(h):
                    at = head // (h // hk)
                    x = s["q"][row:row + n].view(n, h, d)[:, head].double() @ k[:, at].T / math.sqrt(d)
                    if case["causal"]:
                        x = x.masked_fill(hidden, -math.inf)
                    o[:, head] = torch.softmax(x, 1) @ v[:, at]
                outs["out"].append(o.reshape(n, h * d))
        row += n
    return {name: torch.cat(v) for name, v in outs.items() if v}


def work(case):
    b, h, hk, d, page = _sizes(case)
    lens = lengths(case)
    new, kv = sum(n for n, _ in lens), sum(k for _, k in lens)
    blocks = sum(-(-k // BLOCK) for _, k in lens)
    cache = 2 * hk * (kv * d + 4 * blocks)  # keys and values with their scales, each read once
    if case["kind"] == "gather":
        return {"bytes": cache + 4 * kv * hk * d, "flops": 2 * kv * hk * d}
    if case["kind"] == "append":
        # q read and written, k and v read in f16 and written in 8 bits, the table's rows; then all of it read back
        step = 4 * new * h * d + 6 * new * hk * d + 4 * new * case["rot"]
        return {"bytes": step + cache + 4 * kv * hk * d, "flops": 3 * new * (h + hk) * case["rot"] + 4 * new * hk * d + 2 * kv * hk * d}
    pairs = sum(n * k - (n * (n - 1) // 2 if case["causal"] else 0) for n, k in lens)
    return {"bytes": cache + 4 * new * h * d, "flops": 4 * h * d * pairs}
