"""Cases of the operators on a paged KV cache held in 4 bits: attention over it, appending to it
with the query / key norms and the position rotation on the way, storing to it and loading from it.

The cache (one layer) is uint8 ``[pages, kv heads, 160 * P]`` for pages of P tokens: P / 8 blocks of
8 tokens, 1280 bytes each. A row of 128 values is held in four groups of 32 as
``mid + scale * (code - 7.5)`` with codes 0..15 and bf16 ``scale`` and ``mid``. Inside a block:

* bytes 0..511: key codes; token i at 64 i, then 16 t + 4 g: a 32-bit word whose nibble j is the code
  of value 32 g + 8 t + j;
* bytes 512..639: token i, group g at 16 i + 4 g: scale, mid;
* bytes 640..1151: value codes; token pair p at 128 p, unit u (0..7) at 16 (u ^ 2p), then 4 g: a
  16-bit half for each token of the pair whose nibble j is the code of value 32 g + 4 u + j;
* bytes 1152..1279: the values' scale, mid.
"""

import random

import torch

own = False

HD, GROUP, BLOCK_BYTES, EPS, THETA = 128, 32, 1280, 1e-6, 1e6


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    attend = {"op": "attend", "heads": 32, "kv_heads": 8, "q_len": 1, "page": 16, "spread": 1}
    append = {"op": "append", "heads": 32, "kv_heads": 8, "page": 16, "pad": 0}
    return [
        # one sequence early in a chat: where a call is all latency
        dict(attend, name="attend 1 x 1000", batch=1, context=1000),
        # the paged context of the repository's own benchmark, one token
        dict(attend, name="attend 1 x 16384", batch=1, context=16384),
        # a serving batch whose sequences are at very different lengths
        dict(attend, name="attend 48 ragged to 8111", batch=48, context=8111, spread=64),
        # speculative verification: 5 rows a sequence, the smaller model's 16 query heads
        dict(attend, name="verify 8 x 5 rows x 4099", heads=16, batch=8, context=4099, q_len=5, spread=2),
        # one long document, large pages
        dict(attend, name="attend 1 x 131072", batch=1, context=131072, page=64),
        # one token of one sequence: the append of every decode step
        dict(append, name="append 1 token", tokens=1, context=700, batch=1),
        # a decode batch padded to its captured size
        dict(append, name="append 61 of 64 sequences", tokens=64, context=5000, batch=64, pad=3),
        # a long prompt's rows
        dict(append, name="append prompt of 8190", tokens=8190, context=8190, batch=1),
        # rows mirrored from a forward that ran elsewhere: a few, and a prompt
        {"op": "store", "name": "store 5 rows", "kv_heads": 8, "page": 16, "tokens": 5},
        {"op": "store", "name": "store 16380 rows", "kv_heads": 8, "page": 16, "tokens": 16380},
        # a cached prefix read back for the prompt kernel: short and long
        {"op": "load", "name": "load 333 rows", "kv_heads": 8, "page": 16, "tokens": 333},
        {"op": "load", "name": "load 32001 rows", "kv_heads": 8, "page": 16, "tokens": 32001},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "store", "load"])
    page = rng.choice([8, 16, 16, 32, 64])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    if op == "attend":
        batch = _log(rng, 1, 64)
        group = rng.choice([1, 2, 4, 4, 5, 7, 8])
        q_len = rng.choice([1, 1, 1, 2, 3, 5, 8])
        most = 131072 * 8 // (batch * kv_heads * (2 if q_len * group > 8 else 1))
        context = _log(rng, max(q_len, 3), min(131072, most))
        return {"op": op, "heads": group * kv_heads, "kv_heads": kv_heads, "q_len": q_len, "page": page,
                "batch": batch, "context": context, "spread": rng.choice([1, 2, 16])}
    if op == "append":
        heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
        if rng.random() < 0.5:
            batch = _log(rng, 1, 256)
            return {"op": op, "heads": heads, "kv_heads": kv_heads, "page": page, "tokens": batch,
                    "context": _log(rng, 2, 20000), "batch": batch, "pad": min(batch - 1, rng.choice([0, 1, 5]))}
        tokens = _log(rng, 2, min(8190, 8190 * 48 // (heads + 2 * kv_heads)))
        return {"op": op, "heads": heads, "kv_heads": kv_heads, "page": page, "tokens": tokens,
                "context": tokens + rng.randrange(0, 1000), "batch": 1, "pad": 0}
    return {"op": op, "kv_heads": kv_heads, "page": page,
            "tokens": _log(rng, 2, (16380 if op == "store" else 32001) * 8 // max(kv_heads, 2))}


def _lengths(case):
    """Keys of each sequence: from ``context / spread`` to ``context`` in even steps of the logarithm."""
    n, top, spread = case["batch"], case["context"], case["spread"]
    least = max(case["q_len"], top // spread)
    return [max(least, int(round(top * (least / top) ** (i / max(1, n - 1))))) for i in range(n)]


def work(case):
    row = case["kv_heads"] * 160  # keys and values of one token, in 4 bits
    if case["op"] == "attend":
        keys, rows = sum(_lengths(case)), case["heads"] * case["q_len"]
        pages = sum(-(-n // case["page"]) for n in _lengths(case))
        return {"bytes": keys * row + case["batch"] * (rows * HD * 4 + 8) + pages * 4,
                "flops": 4 * HD * rows * keys}
    if case["op"] == "append":
        live, h, k = case["tokens"] - case["pad"], case["heads"], case["kv_heads"]
        positions = case["tokens"] if case["batch"] == 1 else live
        rows = (h + 2 * k) * HD * 2 + h * HD * 2 + row + k * HD * 4 + 16  # the rows held come back in bf16
        return {"bytes": live * rows + positions * HD * 4, "flops": live * (h + 2 * k) * HD * 8}
    back = case["kv_heads"] * HD * 4 * (2 if case["op"] == "store" else 1)
    return {"bytes": case["tokens"] * (row + back + 8), "flops": case["tokens"] * case["kv_heads"] * HD * 16}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _rows(g, *shape):
    """Rows as a cache meets them: unit normal, with a few dimensions that are three times as large."""
    x = torch.randn(*shape, HD, generator=g, device="cuda")
    x[..., 5::41] *= 3
    return x


def _pack(k, v):
    """``k``, ``v`` fp32 [tokens (a multiple of 8), heads, 128] as blocks [tokens / 8, heads, 1280] uint8."""
    n, h, _ = k.shape

    def parts(x):
        codes, scale, mid = _quantise(x)
        codes = codes.to(torch.uint8).view(n // 8, 8, h, 4, GROUP).permute(0, 2, 1, 3, 4)
        meta = torch.stack([scale, mid], -1).to(torch.bfloat16).view(n // 8, 8, h, 4, 2)
        return codes, meta.permute(0, 2, 1, 3, 4).contiguous().view(torch.uint8).view(n // 8, h, 128)

    def nibbles(c):
        return c[..., 0::2] | (c[..., 1::2] << 4)

    kc, km = parts(k)
    vc, vm = parts(v)
    kb = nibbles(kc.reshape(n // 8, h, 8, 4, 4, 8).transpose(3, 4)).reshape(n // 8, h, 512)
    vb = vc.reshape(n // 8, h, 4, 2, 4, 8, 4).permute(0, 1, 2, 5, 4, 3, 6)  # pair, unit, group, token, j
    vb = nibbles(vb).reshape(n // 8, h, 4, 8, 16).gather(3, _unit_order(k.device).expand(n // 8, h, 4, 8, 16))
    return torch.cat([kb, km, vb.reshape(n // 8, h, 512), vm], -1)


def _unit_order(device):
    pair, place = torch.arange(4, device=device)[:, None], torch.arange(8, device=device)[None, :]
    return (place ^ (2 * pair))[None, None, :, :, None]


def _filled(g, tokens, kv_heads, page, spare):
    """A cache with ``tokens`` rows of every head in ``ceil(tokens / page)`` pages in a random order, and
    the pages' order."""
    pages = -(-tokens // page)
    n = pages * page
    blocks = _pack(_rows(g, n, kv_heads), _rows(g, n, kv_heads))
    order = torch.randperm(pages + spare, generator=g, device="cuda")[:pages]
    cache = torch.zeros(pages + spare, kv_heads, 160 * page, dtype=torch.uint8, device="cuda")
    cache[order] = blocks.view(pages, page // 8, kv_heads, BLOCK_BYTES).transpose(1, 2).reshape(pages, kv_heads, -1)
    return cache, order


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    page, kv_heads = case["page"], case["kv_heads"]
    s = dict(case)
    if case["op"] == "attend":
        lengths = _lengths(case)
        counts = [-(-n // page) for n in lengths]
        cache, order = _filled(g, sum(counts) * page, kv_heads, page, 3)
        table = torch.zeros(len(lengths), max(counts), dtype=torch.int32)
        host, at = order.to("cpu", torch.int32), 0
        for b, c in enumerate(counts):
            table[b, :c] = host[at:at + c]
            at += c
        q = _rows(g, case["batch"], case["q_len"], case["heads"]).to(torch.bfloat16)
        s.update(q=q, out=torch.zeros_like(q), cache=cache, table=table.cuda(), most=max(lengths),
                 q_pos=torch.tensor([n - case["q_len"] for n in lengths], dtype=torch.int64, device="cuda"),
                 workspace=torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
        return s
    tokens = case["tokens"]
    if case["op"] == "append":
        heads, live = case["heads"], tokens - case["pad"]
        s["qkv"] = _rows(g, tokens, heads + 2 * kv_heads).to(torch.bfloat16).view(tokens, -1)
        s["weights"] = [(1 + 0.1 * torch.randn(HD, generator=g, device="cuda")).to(torch.bfloat16) for _ in "qk"]
        angle = torch.arange(case["context"], device="cuda", dtype=torch.float64)[:, None] / \
            THETA ** (torch.arange(0, HD, 2, device="cuda", dtype=torch.float64) / HD)
        angle = torch.cat([angle, angle], -1)
        s["cos"], s["sin"] = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
        if case["batch"] == 1:  # consecutive positions of one sequence
            positions = torch.arange(case["context"] - tokens, case["context"], device="cuda")
        else:  # one token of each sequence
            positions = torch.randint(0, case["context"], (tokens,), generator=g, device="cuda")
        s["positions"] = positions
        s["q_out"] = torch.zeros(tokens, heads, HD, dtype=torch.bfloat16, device="cuda")
        if case["batch"] == 1:
            slots, pages = _slots(g, int(positions[0]) % page, tokens, page)
        else:  # each sequence's own page
            pages = tokens + 2
            slots = torch.randperm(pages, generator=g, device="cuda")[:tokens] * page + positions % page
        slots[live:] = -1
        s["cache"] = torch.zeros(pages, kv_heads, 160 * page, dtype=torch.uint8, device="cuda")
    elif case["op"] == "store":
        s["key"], s["value"] = (_rows(g, tokens, kv_heads).to(torch.bfloat16) for _ in "kv")
        slots, pages = _slots(g, tokens % page, tokens, page)
        s["cache"] = torch.zeros(pages, kv_heads, 160 * page, dtype=torch.uint8, device="cuda")
    else:
        s["cache"], order = _filled(g, tokens, kv_heads, page, 3)
        at = torch.arange(tokens, device="cuda")
        slots = order[at // page] * page + at % page
    s["slots"] = slots
    s["back"] = [torch.zeros(tokens, kv_heads, HD, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    return s


def _slots(g, first, tokens, page):
    """Slots of ``tokens`` rows that begin at row ``first`` of a page, and the number of pages."""
    pages = -(-(first + tokens) // page) + 2
    at = torch.arange(first, first + tokens, device="cuda")
    return torch.randperm(pages, generator=g, device="cuda")[at // page] * page + at % page, pages


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "attend":
        return _attend(s)
    if s["op"] == "append":
        heads, kv_heads, n = s["heads"], s["kv_heads"], s["tokens"]
        live = (s["slots"] >= 0)[:, None, None]
        q, k, v = s["qkv"].float().view(n, -1, HD).split([heads, kv_heads, kv_heads], 1)
        cos, sin = (s[t][s["positions"]].float()[:, None] for t in ("cos", "sin"))
        q, k = (_rotate(_normed(x, w), cos, sin) for x, w in ((q, s["weights"][0]), (k, s["weights"][1])))
        return {"q": (q * live).to(torch.bfloat16), "k": (_held(k) * live).to(torch.bfloat16),
                "v": (_held(v) * live).to(torch.bfloat16)}
    if s["op"] == "store":
        return {"k": _held(s["key"].float()).to(torch.bfloat16), "v": _held(s["value"].float()).to(torch.bfloat16)}
    page, kv_heads = s["page"], s["kv_heads"]
    blocks = s["cache"].view(-1, kv_heads, page // 8, BLOCK_BYTES)
    k, v = _unpack(blocks[s["slots"] // page, :, s["slots"] % page // 8])
    at = (s["slots"] % 8)[:, None, None, None].expand(-1, kv_heads, 1, HD)
    return {"k": k.gather(2, at)[:, :, 0].to(torch.bfloat16), "v": v.gather(2, at)[:, :, 0].to(torch.bfloat16)}


def _run_own(s):
    from solort_b200 import ops

    if s["op"] == "attend":
        return ops.gqa_decode_paged_int4(s["q"], s["cache"], s["table"], s["q_pos"], max_kv_len=s["most"],
                                         out=s["out"], workspace=s["workspace"], stable_prefix=True)
    found = {}
    if s["op"] == "append":
        found["q"] = ops.qk_norm_rope_append_int4(
            s["qkv"], s["weights"][0], s["weights"][1], EPS, s["cos"], s["sin"], s["positions"], s["slots"],
            s["cache"], num_qo_heads=s["heads"], num_kv_heads=s["kv_heads"], q_out=s["q_out"])
    elif s["op"] == "store":
        ops.kv_store_int4(s["key"], s["value"], s["slots"], s["cache"])
    found["k"], found["v"] = ops.kv_load_int4(s["cache"], s["slots"], key=s["back"][0], value=s["back"][1])
    return found


def _quantise(x):
    """Codes [..., 4, 32], scales and mids [..., 4] of fp32 rows [..., 128]; the steps are the operators'
    own in 32 bits, so that values next to a border between two codes fall on the same side."""
    x = x.view(*x.shape[:-1], 4, GROUP)
    lo, hi = x.amin(-1), x.amax(-1)
    mid = (0.5 * lo + 0.5 * hi).to(torch.bfloat16).float()
    need = torch.maximum(hi - mid, mid - lo)
    scale = need / torch.full_like(need, 7.5)  # a quotient: by a number, torch takes a product with 1 / 7.5
    scale = ((scale.view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32)  # up to a bf16 value
    step = torch.where(scale > 0, scale, torch.ones_like(scale))
    codes = ((x - mid[..., None]) / step[..., None] + 7.5).round().clamp(0, 15)
    return codes, scale, mid


def _held(x):
    """What the cache holds for fp32 rows [..., 128]."""
    codes, scale, mid = _quantise(x)
    return (mid[..., None] + scale[..., None] * (codes - 7.5)).view(x.shape)


def _normed(x, w):
    """The norm of fp32 head rows; the mean of squares in 64 bits, for the sake of the borders again."""
    r = 1 / (x.double().square().mean(-1, keepdim=True) + float(torch.tensor(EPS))).sqrt()
    return x * r.float() * w.float()


def _rotate(x, cos, sin):
    return x * cos + torch.cat([-x[..., HD // 2:], x[..., :HD // 2]], -1) * sin


def _unpack(blocks):
    """fp32 keys and values [..., 8, 128] of blocks [..., 1280] uint8."""
    lead = blocks.shape[:-1]
    kb, km, vb, vm = blocks.split([512, 128, 512, 128], -1)

    def codes(b):  # nibbles in their order
        return torch.stack([b & 15, b >> 4], -1).flatten(-2)

    def values(c, meta):
        meta = meta.contiguous().view(torch.bfloat16).view(*lead, 8, 4, 2, 1).float()
        return (meta[..., 1, :] + meta[..., 0, :] * (c.float() - 7.5)).view(*lead, 8, HD)

    k = codes(kb).view(*lead, 8, 4, 4, 8).transpose(-3, -2).reshape(*lead, 8, 4, GROUP)
    v = vb.view(*lead, 4, 8, 16).gather(-2, _unit_order(blocks.device)[0, 0].expand(*lead, 4, 8, 16))
    v = codes(v).view(*lead, 4, 8, 4, 2, 4).movedim(-2, -4).transpose(-3, -2)  # pair, token, group, unit, j
    return values(k, km), values(v.reshape(*lead, 8, 4, GROUP), vm)


def _attend(s):
    q, kv_heads, page = s["q"], s["kv_heads"], s["page"]
    batch, t, heads, _ = q.shape
    blocks = s["cache"][s["table"]].view(batch, -1, kv_heads, page // 8, BLOCK_BYTES).transpose(1, 2)
    k, v = (x.reshape(batch, kv_heads, -1, HD) for x in _unpack(blocks))
    rows = q.float().view(batch, t, kv_heads, -1, HD).transpose(1, 2).reshape(batch, kv_heads, -1, HD)
    scores = (rows @ k.transpose(-1, -2) * HD ** -0.5).view(batch, kv_heads, t, -1, k.shape[2])
    last = s["q_pos"][:, None] + torch.arange(t, device=q.device)
    seen = torch.arange(k.shape[2], device=q.device) <= last[:, None, :, None, None]
    scores = torch.where(seen, scores, -torch.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    p = (p / p.sum(-1, keepdim=True)).view(batch, kv_heads, -1, k.shape[2])
    v = torch.where(seen.any(2).view(batch, 1, -1, 1), v, 0)  # rows behind a sequence's end hold anything
    out = (p @ v).view(batch, kv_heads, t, -1, HD).transpose(1, 2).reshape(q.shape)
    return out.to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits, one head or sequence at a time
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        group = case["heads"] // case["kv_heads"]
        for b, n in enumerate(_lengths(case)):
            at = torch.arange(n, device="cuda")
            slots = s["table"][b].long()[at // case["page"]] * case["page"] + at % case["page"]
            for h in range(case["kv_heads"]):
                k, v = _exact_rows(s["cache"], slots, h, case["page"])
                for t in range(case["q_len"]):
                    m = n - case["q_len"] + t + 1
                    q = s["q"][b, t, h * group:(h + 1) * group].double()
                    out[b, t, h * group:(h + 1) * group] = torch.softmax(q @ k[:m].T / HD ** 0.5, -1) @ v[:m]
        return out
    if case["op"] == "load":
        rows = [_exact_rows(s["cache"], s["slots"], h, case["page"]) for h in range(case["kv_heads"])]
        return {"k": torch.stack([r[0] for r in rows], 1), "v": torch.stack([r[1] for r in rows], 1)}
    if case["op"] == "store":
        return {"k": _exact_held(s["key"].double()), "v": _exact_held(s["value"].double())}
    heads, kv_heads = case["heads"], case["kv_heads"]
    x = s["qkv"].double().view(case["tokens"], -1, HD)
    cos, sin = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]
    done = []
    for h in range(heads + kv_heads):
        w = s["weights"][0 if h < heads else 1].double()
        y = x[:, h] * torch.rsqrt((x[:, h] ** 2).sum(-1, keepdim=True) / HD + EPS) * w
        a, b = y[:, :64], y[:, 64:]
        done.append(torch.cat([a * cos[:, :64] - b * sin[:, :64], b * cos[:, 64:] + a * sin[:, 64:]], -1))
    y = torch.stack(done, 1)
    y[s["slots"] < 0] = 0
    v = _exact_held(x[:, heads + kv_heads:])
    v[s["slots"] < 0] = 0
    return {"q": y[:, :heads], "k": _exact_held(y[:, heads:]), "v": v}


def _exact_held(x):
    found = torch.empty_like(x)
    for g in range(0, HD, GROUP):
        y = x[..., g:g + GROUP]
        lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
        mid = ((lo + hi) / 2).to(torch.bfloat16).double()
        need = torch.maximum(hi - mid, mid - lo) / 7.5
        near = need.to(torch.bfloat16)
        above = torch.nextafter(near, torch.full_like(near, float("inf")))
        scale = torch.where(near.double() >= need, near, above).double()
        steps = torch.where(scale > 0, (y - mid) / scale.clamp_min(1e-300), 0)
        found[..., g:g + GROUP] = mid + scale * ((steps - 0.5).round().clamp(-8, 7) + 0.5)
    return found


def _exact_rows(cache, slots, head, page):
    """Rows of one head in 64 bits, each value's byte found by its address in the cache."""
    d = torch.arange(HD, device="cuda")
    g, i, pair = d // 32, (slots % 8)[:, None], (slots % 8 // 2)[:, None]
    flat = cache.view(-1)
    base = ((slots // page * cache.shape[1] + head) * cache.shape[2] + slots % page // 8 * BLOCK_BYTES)[:, None]
    j = d % 8
    k = flat[base + 64 * i + 16 * (d % 32 // 8) + 4 * g + j // 2].long() >> (4 * (j % 2)) & 15
    u, j = d % 32 // 4, d % 4
    v = flat[base + 640 + 128 * pair + 16 * (u ^ (2 * pair)) + 4 * g + 2 * (i % 2) + j // 2]
    v = v.long() >> (4 * (j % 2)) & 15

    def real(at):  # the bf16 value at a byte address
        return ((flat[at].long() + 256 * flat[at + 1].long()) << 16).to(torch.int32).view(torch.float32).double()

    km, vm = base + 512 + 16 * i + 4 * g, base + 1152 + 16 * i + 4 * g
    return real(km + 2) + real(km) * (k - 7.5), real(vm + 2) + real(vm) * (v - 7.5)


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c, work(c))
