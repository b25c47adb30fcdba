"""The serving operators around a paged key/value cache, and the rotary embedding of training and serving, on one GPU.

``listed()`` are twelve fixed cases, ``draw(rng)`` gives more of the same ranges. Every case is a dict of plain
values with a ``kind``:

* ``pages``    a step's bookkeeping, from the lengths of the requests: pages of finished requests go back to the free list
               (``paged.release_pages``), new ones are assigned, and every new token gets its position and its slot in
               the cache (``paged.assign_pages``);
* ``rotary``   ``rotary``: queries and keys rotated by their positions, forward and backward;
* ``append``   ``paged.rotary_append``: queries rotated, keys rotated into the pages of the cache, values beside them;
* ``attend``   ``paged_attention``: the new tokens of a ragged batch of requests against their pages.

Lengths follow from the case (``len_seed``), values and the order of the pages from the seed of ``prepare``.
"""
from __future__ import annotations

import math
import random

import torch

own = False         # True: the framework's operators, False: their plain form

D = 128             # head dim of every configuration of this repository
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed() -> list:
    return [
        # one decoding step of a serving batch: every 64th request or so needs a new page (latency only)
        dict(name="pages_decode", kind="pages", requests=64, most_new=1, most_context=8192, page=64, finished=0, len_seed=1),
        # the step in which requests end and the prompts of new ones come in, small pages
        dict(name="pages_turnover", kind="pages", requests=200, most_new=777, most_context=4096, page=16, finished=40,
             len_seed=2),
        # training at an ordinary length, grouped-query heads, context stretched four times: forward and backward
        dict(name="rotary_train_8k", kind="rotary", batch=1, seq=8192, heads=32, kv_heads=8, dtype="bf16", rot=128,
             interleaved=False, scaling="yarn", start=0),
        # a batch in fp32 at odd sizes, half of the head rotated, adjacent pairs, far positions
        dict(name="rotary_partial_fp32", kind="rotary", batch=3, seq=1001, heads=12, kv_heads=12, dtype="fp32", rot=64,
             interleaved=True, scaling="linear", start=500_000),
        # the smallest call: one decoding step of a few requests
        dict(name="append_decode", kind="append", requests=24, most_new=1, most_context=4096, page=64, heads=32, kv_heads=8,
             rot=128, interleaved=False, len_seed=3),
        # prompts of several requests in one step, pages of 16, part of the head in adjacent pairs
        dict(name="append_prompts", kind="append", requests=11, most_new=2047, most_context=8192, page=16, heads=32,
             kv_heads=8, rot=96, interleaved=True, len_seed=4),
        # one user's decoding step: latency
        dict(name="decode_one", kind="attend", requests=1, most_new=1, most_context=1500, equal=True, page=64, heads=32,
             kv_heads=8, left=-1, sink=0, len_seed=5),
        # a serving batch of ragged lengths, one new token each
        dict(name="decode_ragged", kind="attend", requests=48, most_new=1, most_context=16000, equal=False, page=64,
             heads=32, kv_heads=8, left=-1, sink=0, len_seed=6),
        # the same with a head group that is no power of two, small pages, a window and sinks
        dict(name="decode_window", kind="attend", requests=33, most_new=1, most_context=20000, equal=False, page=16,
             heads=28, kv_heads=4, left=4095, sink=4, len_seed=7),
        # a chunk of one long prompt behind the keys of the chunks before it
        dict(name="chunk_32k", kind="attend", requests=1, most_new=512, most_context=32768, equal=True, page=128, heads=32,
             kv_heads=8, left=-1, sink=0, len_seed=8),
        # a mixed step: most requests decode, some bring a chunk of their prompt
        dict(name="mixed_step", kind="attend", requests=20, most_new=700, most_context=5000, equal=False, page=32, heads=32,
             kv_heads=8, left=-1, sink=0, len_seed=9),
        # a whole prompt at once, nothing cached before it (the largest case)
        dict(name="prompt_8k", kind="attend", requests=1, most_new=8192, most_context=8192, equal=True, page=64, heads=32,
             kv_heads=8, left=-1, sink=0, len_seed=10),
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    """One more case. Sizes are spread over their logarithm, most of them multiples of nothing."""
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        c = _draw(rng)
        if all(work(c)[k] <= most[k] for k in most) and _plain_bytes(c) <= 10e9:
            return c


def _draw(rng: random.Random) -> dict:
    kind = rng.choice(["pages", "rotary", "append", "attend", "attend", "attend", "attend"])
    seed = rng.randrange(1 << 20)
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "pages":
        n = _log(rng, 1, 1000)
        return dict(kind="pages", requests=n, most_new=rng.choice([1, _log(rng, 2, 2000)]), most_context=_log(rng, 2000, 20000),
                    page=page, finished=rng.choice([0, n // 4]), len_seed=seed)
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8) if kv * g >= 4])
    if kind == "rotary":
        return dict(kind="rotary", batch=rng.choice([1, 1, 2, 5]), seq=_log(rng, 1, 8000), heads=heads, kv_heads=kv,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), rot=rng.choice([128, 128, 64, 96, 32]),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]),
                    start=rng.choice([0, _log(rng, 1000, 1_000_000)]))
    if kind == "append":
        return dict(kind="append", requests=_log(rng, 1, 64), most_new=rng.choice([1, _log(rng, 2, 1500)]),
                    most_context=_log(rng, 2000, 8000), page=page, heads=heads, kv_heads=kv, rot=rng.choice([128, 128, 64, 96]),
                    interleaved=rng.random() < 0.5, len_seed=seed)
    left = rng.choice([-1, -1, _log(rng, 100, 8000)])
    form = rng.choice(["decode", "decode", "chunk", "mixed"])
    n = _log(rng, 1, 64) if form == "decode" else 1 if form == "chunk" else _log(rng, 2, 24)
    new = 1 if form == "decode" else _log(rng, 2, 4000)
    return dict(kind="attend", requests=n, most_new=new, most_context=new + _log(rng, 200, 32000), equal=form == "chunk",
                page=page, heads=heads, kv_heads=kv, left=left, sink=rng.choice([0, 4, 16]) if left >= 0 else 0, len_seed=seed)


# ------------------------------------------------------------------------------------------------
# lengths of a case
# ------------------------------------------------------------------------------------------------
def _lengths(c: dict) -> tuple:
    """(context, new) of every request: tokens with the new ones, and new tokens. Both are spread over their logarithm; of
    the requests of a mixed step most decode one token."""
    r = random.Random(c["len_seed"])
    n, most_new, most = c["requests"], c["most_new"], c["most_context"]
    if c.get("equal"):
        return [most] * n, [most_new] * n
    new = [most_new if i == 0 else 1 if most_new == 1 or r.random() < 0.7 else _log(r, 2, most_new) for i in range(n)]
    r.shuffle(new)
    context = [k + _log(r, min(20, most - k), most - k) if most > k else k for k in new]
    return context, new


def _page_counts(c: dict) -> tuple:
    """(pages held after the step, pages held before it) of every request."""
    context, new = _lengths(c)
    up = lambda x: -(-x // c["page"])
    return [up(x) for x in context], [up(x - k) for x, k in zip(context, new)]


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _inv_freq(rot: int, scaling: str) -> tuple:
    """(angle per position of every pair, factor of the rotated vector) in 64 bits: base 10000, stretched by 4 from 8192
    positions."""
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    base, factor, original = 10000.0, 4.0, 8192.0
    if scaling == "ntk":
        base *= factor ** (rot / (rot - 2))
    f = base ** (-i / rot)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        # pairs that turn more than 32 times within the original length keep their angle, those below one turn are stretched
        at = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if scaling == "bands":
        # the same idea by wavelength: between original / 4 and original a linear transition
        turns = original * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 1.0
    return f, 1.0


def prepare(case: dict, seed: int) -> dict:
    dev, c = torch.device("cuda"), case
    g = torch.Generator(device=dev).manual_seed(seed)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    # projections of normalised activations: standard normal
    rand = lambda *shape, dtype=torch.bfloat16: torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    s = dict(case=c)
    if c["kind"] == "rotary":
        f, s["magnitude"] = _inv_freq(c["rot"], c["scaling"])
        s["inv_freq"] = f.to(dev)
        s["pos"] = (torch.arange(c["seq"], device=dev) + c["start"]).to(torch.int32).repeat(c["batch"], 1)
        for name, h in (("q", c["heads"]), ("k", c["kv_heads"]), ("d_q", c["heads"]), ("d_k", c["kv_heads"])):
            s[name] = rand(c["batch"], c["seq"], h, D, dtype=DTYPES[c["dtype"]]).requires_grad_(name in "qk")
        return s
    context, new = _lengths(c)
    after, before = _page_counts(c)
    n, tokens, width = c["requests"], sum(new), max(after) + 1
    s.update(context=ints(context), new=ints(new), tokens=tokens)
    done = c.get("finished", 0)
    # the pages in a random order; the first of them belong to the requests
    pool = sum(before if c["kind"] == "pages" else after) + sum(after[:done]) + (sum(after) if c["kind"] == "pages" else 1)
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    held = before if c["kind"] == "pages" else after
    table = torch.full((n + done, width), -1, dtype=torch.int32, device=dev)
    at = torch.arange(width, device=dev)
    count = ints(held + after[:done])                       # (the last `done` rows: requests that have ended)
    first = torch.cumsum(count, 0, dtype=torch.int64) - count
    table = torch.where(at < count[:, None], order[(first[:, None] + at).clamp(max=pool - 1)], table)
    s["table"] = table
    if c["kind"] == "pages":
        s["context"], s["new"] = (torch.cat([x, x.new_zeros(done)]) for x in (s["context"], s["new"]))
        s["ended"] = torch.arange(n + done, device=dev) >= n
        s["ended_context"] = torch.cat([torch.zeros_like(ints(context)), ints(context[:done])])
        used = int(sum(held) + sum(after[:done]))
        s["free"] = torch.cat([order[used:], order.new_full((used,), -1)])      # a stack; what is above its top means nothing
        s["free_count"] = ints([pool - used])
        return s
    s["cu_new"] = torch.cat([ints([0]), torch.cumsum(s["new"], 0, dtype=torch.int32)])
    s["k_cache"], s["v_cache"] = (rand(pool, c["page"], c["kv_heads"], D) for _ in range(2))
    s["most_new"], s["most_context"] = max(new), max(context)
    if c["kind"] == "attend":
        s["q"] = rand(tokens, c["heads"], D)
        return s
    s["qkv"] = rand(tokens, (c["heads"] + 2 * c["kv_heads"]) * D)       # a projection's output, its parts are views of it
    f, s["magnitude"] = _inv_freq(c["rot"], "none")
    s["inv_freq"] = f.to(dev)
    s["pos"], s["slots"] = _positions(s, c["page"])
    return s


def _positions(s: dict, page: int) -> tuple:
    """Position and cache slot (page * page size + offset) of every new token, in token order."""
    t = torch.arange(s["tokens"], device=s["table"].device)
    cu = torch.cumsum(s["new"], 0, dtype=torch.int64)
    req = torch.searchsorted(cu, t, right=True)
    pos = s["context"][req] - cu[req] + t
    slots = s["table"][req, pos // page].long() * page + pos % page
    return pos.to(torch.int32), slots.to(torch.int32)


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _plain_pages(s: dict) -> dict:
    page, table, free, count = s["case"]["page"], s["table"], s["free"], s["free_count"].long()
    dev, n = table.device, free.shape[0]
    at = torch.arange(table.shape[1], device=dev)
    out = {}
    if s["case"]["finished"]:
        held = (s["ended_context"].long() + page - 1) // page * s["ended"]
        mine = at < held[:, None]
        place = torch.cumsum(mine.flatten(), 0).view_as(mine) - 1 + count
        free = torch.cat([free, free.new_zeros(1)]).index_put_((torch.where(mine, place, n),), table)[:n]
        count = count + held.sum()
        out["free"] = free
    after = (s["context"].long() + page - 1) // page
    before = ((s["context"] - s["new"]).clamp(min=0).long() + page - 1) // page
    need = after - before
    first = torch.cumsum(need, 0) - need
    place = count - 1 - first[:, None] - (at - before[:, None])
    fresh = (at >= before[:, None]) & (at < after[:, None])
    table = s["table"] = torch.where(fresh, free[place.clamp(0, n - 1)], table)
    pos, slots = _positions(s, page)
    cu = torch.cat([s["new"].new_zeros(1), torch.cumsum(s["new"], 0, dtype=torch.int32)])
    return out | {"table": table, "cu_new": cu, "pos": pos, "slots": slots, "free_count": (count - need.sum()).to(torch.int32)}


def _plain_rotate(x, pos, inv_freq, magnitude, interleaved, inverse=False):
    """x [..., heads, D] by pos [...]: angles in 64 bits, the rotation in 32."""
    ang = pos.double()[..., None] * inv_freq
    cos, sin = ((f(ang) * magnitude).float()[..., None, :] for f in (torch.cos, torch.sin))
    if inverse:
        sin = -sin
    half, xf = inv_freq.shape[0], x.float()
    a, b = (xf[..., 0:2 * half:2], xf[..., 1:2 * half:2]) if interleaved else (xf[..., :half], xf[..., half:2 * half])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([ra, rb], -1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    return torch.cat([turned, xf[..., 2 * half:]], -1).to(x.dtype)


def _plain_rotary(s: dict) -> dict:
    c = s["case"]
    turn = lambda x, inverse: _plain_rotate(x, s["pos"], s["inv_freq"], s["magnitude"], c["interleaved"], inverse)
    with torch.no_grad():
        return {"q": turn(s["q"], False), "k": turn(s["k"], False), "dq": turn(s["d_q"], True), "dk": turn(s["d_k"], True)}


def _split(s: dict) -> tuple:
    c = s["case"]
    return tuple(x.unflatten(1, (-1, D)) for x in s["qkv"].split([c["heads"] * D, c["kv_heads"] * D, c["kv_heads"] * D], 1))


def _plain_append(s: dict) -> dict:
    c = s["case"]
    q, k, v = _split(s)
    q, k = (_plain_rotate(x, s["pos"], s["inv_freq"], s["magnitude"], c["interleaved"]) for x in (q, k))
    at = s["slots"].long()
    s["k_cache"].view(-1, c["kv_heads"], D)[at] = k
    s["v_cache"].view(-1, c["kv_heads"], D)[at] = v
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s: dict) -> dict:
    """The requests side by side, padded to the longest: scores [requests, kv heads, group, new tokens, keys] in fp32."""
    c, q, dev = s["case"], s["q"], s["q"].device
    page, hk, group = c["page"], c["kv_heads"], c["heads"] // c["kv_heads"]
    key, row = torch.arange(s["most_context"], device=dev), torch.arange(s["most_new"], device=dev)
    slot = s["table"][:, key // page].clamp(min=0).long() * page + key % page
    k, v = (x.view(-1, hk, D)[slot].float() for x in (s["k_cache"], s["v_cache"]))
    at = (s["cu_new"][:-1, None] + row).clamp(max=s["tokens"] - 1)
    qs = q[at].float().unflatten(2, (hk, group))
    score = torch.einsum("bnhgd,blhd->bhgnl", qs, k).mul_(D ** -0.5)
    pos = (s["context"] - s["new"])[:, None] + row                              # [requests, new tokens]
    seen = key <= pos[..., None]
    if c["left"] >= 0:
        seen &= (key >= pos[..., None] - c["left"]) | (key < c["sink"])
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bhgnl,blhd->bnhgd", p, v) / total.permute(0, 3, 1, 2, 4)
    lse = (top + total.log()).squeeze(-1).flatten(1, 2)                          # [requests, heads, new tokens]
    t = torch.arange(s["tokens"], device=dev)
    req = torch.searchsorted(s["cu_new"][1:].contiguous(), t, right=True)
    i = t - s["cu_new"][req]
    return {"o": o.flatten(2, 3)[req, i].to(q.dtype), "lse": lse[req, :, i].t().contiguous()}


# ------------------------------------------------------------------------------------------------
def run(state: dict):
    kind, c = state["case"]["kind"], state["case"]
    if not own:
        return {"pages": _plain_pages, "rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend}[kind](state)
    import ultraattn_b200 as ua
    s = state
    if kind == "pages":
        out, count = {}, s["free_count"]
        if c["finished"]:
            count = ua.paged.release_pages(s["ended"], s["ended_context"], s["table"], s["free"], count, page_size=c["page"])
            out["free"] = s["free"]
        step = ua.paged.assign_pages(s["context"], s["new"], s["table"], s["free"], count, page_size=c["page"],
                                     tokens=s["tokens"])
        return out | {"table": s["table"], "cu_new": step.cu_new, "pos": step.pos, "slots": step.slots,
                      "free_count": step.free_count}
    if kind == "rotary":
        q, k = ua.rotary(s["q"], s["k"], s["pos"], s["inv_freq"], magnitude=s["magnitude"], interleaved=c["interleaved"])
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["d_q"], s["d_k"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    if kind == "append":
        q, k, v = _split(s)
        q = ua.paged.rotary_append(q, k, v, s["pos"], s["slots"], s["k_cache"], s["v_cache"], s["inv_freq"],
                                   magnitude=s["magnitude"], interleaved=c["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    o, lse = ua.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["context"], s["cu_new"],
                                most_new=s["most_new"], window_size=(c["left"], 0), sink_tokens=c["sink"])
    return {"o": o, "lse": lse}


# ------------------------------------------------------------------------------------------------
def _pairs(c: dict) -> float:
    """Visible (query, key) pairs of one head, over the batch."""
    tri, total = lambda n: n * (n + 1) / 2, 0.0
    for x, k in zip(*_lengths(c)):
        if c["left"] < 0:
            total += k * (x - k) + tri(k)
        else:
            w, s = c["left"] + 1, c["sink"]
            total += sum(min(p + 1, w) + max(0, min(s, p + 1 - w)) for p in range(x - k, x))
    return total


def _keys(c: dict) -> float:
    """Keys that some query of their request sees."""
    if c["left"] < 0:
        return float(sum(_lengths(c)[0]))
    return float(sum(min(x, k + c["left"]) + min(c["sink"], max(0, x - k - c["left"])) for x, k in zip(*_lengths(c))))


def _plain_bytes(c: dict) -> float:
    if c["kind"] != "attend":
        return 0.0
    context, new = _lengths(c)
    return 4.0 * len(new) * max(context) * (c["heads"] * max(new) + 4 * c["kv_heads"] * D)


def work(case: dict) -> dict:
    c = case
    if c["kind"] == "pages":
        context, new = _lengths(c)
        after, before = _page_counts(c)
        fresh, back = sum(after) - sum(before), sum(after[:c["finished"]])
        # lengths in; fresh pages from the free list into the table, released ones the other way; positions and slots out,
        # with the table entries of the pages they lie in
        return {"bytes": 4.0 * (2 * len(new) + len(new) + 1 + 2 * fresh + 2 * back + 2 * sum(new) + sum(
            -(-x // c["page"]) - (x - k) // c["page"] for x, k in zip(context, new))), "flops": 2.0 * sum(new)}
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[c.get("dtype", "bf16")]
    if c["kind"] == "rotary":
        # q and k in and out, and their gradients; three products and a sum for two values
        n = c["batch"] * c["seq"] * (c["heads"] + c["kv_heads"])
        return {"bytes": 4.0 * n * D * size + 8.0 * c["batch"] * c["seq"], "flops": 6.0 * n * c["rot"]}
    tokens = sum(_lengths(c)[1])
    if c["kind"] == "append":
        n = tokens * (c["heads"] + 2 * c["kv_heads"])
        return {"bytes": 2.0 * n * D * size + 8.0 * tokens, "flops": 3.0 * tokens * (c["heads"] + c["kv_heads"]) * c["rot"]}
    # q and the keys and values that are seen in, o and lse out, the pages' entries of the table
    keys = _keys(c)
    return {"bytes": 2.0 * tokens * c["heads"] * D * 2 + 4.0 * tokens * c["heads"] + 4.0 * keys * c["kv_heads"] * D +
            4.0 * keys / c["page"], "flops": 4.0 * _pairs(c) * c["heads"] * D}


# ------------------------------------------------------------------------------------------------
# the operators' definition in 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_turn(x, pos, inv_freq, magnitude, interleaved):
    """The pairs of a head as complex numbers, times magnitude * exp(i pos f)."""
    x = x.double()
    m = 2 * inv_freq.numel()
    pairs = torch.complex(x[..., :m:2], x[..., 1:m:2]) if interleaved else torch.complex(x[..., :m // 2], x[..., m // 2:m])
    phase = (pos.double().unsqueeze(-1) * inv_freq).unsqueeze(-2)
    z = pairs * torch.polar(torch.full_like(phase, magnitude), phase)
    y = x.clone()
    if interleaved:
        y[..., :m:2], y[..., 1:m:2] = z.real, z.imag
    else:
        y[..., :m // 2], y[..., m // 2:m] = z.real, z.imag
    return y


def exact(case: dict, seed: int):
    c = case
    if c["kind"] == "pages":
        return None                                     # whole numbers: they have to be equal
    s = prepare(case, seed)
    if c["kind"] == "rotary":
        f, m = s["inv_freq"], s["magnitude"]
        with torch.no_grad():
            # the transpose of a rotation is the rotation by the opposite angle
            return {"q": _exact_turn(s["q"], s["pos"], f, m, c["interleaved"]), "k": _exact_turn(s["k"], s["pos"], f, m, c["interleaved"]),
                    "dq": _exact_turn(s["d_q"], s["pos"], -f, m, c["interleaved"]),
                    "dk": _exact_turn(s["d_k"], s["pos"], -f, m, c["interleaved"])}
    if c["kind"] == "append":
        h, hk = c["heads"], c["kv_heads"]
        x = s["qkv"].view(s["tokens"], -1, D)
        turn = lambda y: _exact_turn(y, s["pos"], s["inv_freq"], s["magnitude"], c["interleaved"])
        kc, vc = s["k_cache"].double().flatten(0, 1), s["v_cache"].double().flatten(0, 1)
        kc.index_copy_(0, s["slots"].long(), turn(x[:, h:h + hk]))
        vc.index_copy_(0, s["slots"].long(), x[:, h + hk:].double())
        return {"q": turn(x[:, :h]), "k_cache": kc.view_as(s["k_cache"]), "v_cache": vc.view_as(s["v_cache"])}
    o = torch.empty(s["tokens"], c["heads"], D, dtype=torch.float64, device="cuda")
    lse = torch.empty(c["heads"], s["tokens"], dtype=torch.float64, device="cuda")
    group, first = c["heads"] // c["kv_heads"], 0
    for r, (x, k) in enumerate(zip(*_lengths(c))):
        pages = s["table"][r, :-(-x // c["page"])].long()
        for h in range(c["kv_heads"]):
            keys, values = (y[pages, :, h].reshape(-1, D)[:x].double() for y in (s["k_cache"], s["v_cache"]))
            q = s["q"][first:first + k, h * group:(h + 1) * group].double().transpose(0, 1)     # [group, new, D]
            score = q @ keys.t() / math.sqrt(D)
            i = torch.arange(x - k, x, device="cuda")[:, None]
            j = torch.arange(x, device="cuda")[None]
            hidden = j > i
            if c["left"] >= 0:
                hidden = hidden | ((j < i - c["left"]) & (j >= c["sink"]))
            score[:, hidden] = float("-inf")
            z = torch.logsumexp(score, -1)
            o[first:first + k, h * group:(h + 1) * group] = (torch.exp(score - z[..., None]) @ values).transpose(0, 1)
            lse[h * group:(h + 1) * group, first:first + k] = z
        first += k
    return {"o": o, "lse": lse}
