"""The operators of serving in few bits: products of weights in 8-bit integers with a scale for every
token and every output channel, the store that quantises keys and values into a paged cache of 4 bits, and
the attention over such a cache.

``kind`` of a case:

* ``linear``: ``x`` [rows, k] by a weight [n, k] in 8 bits. A token's row is divided by its largest magnitude over 127 and
  rounded to integers, multiplied with the weight's integers in whole numbers, and the sums multiplied by the token's
  and the channel's scale.
* ``gated``: the same by gate and up rows of a weight [2 n, k], ``silu(gate) * up`` of the results.
* ``store``: keys and values of ``tokens`` tokens into the pages of a 4-bit cache; every head's vector of a token gets a
  lowest value and a step in bfloat16, and its elements codes of 0 to 15. What the cache then holds for them comes back.
* ``attend``: ``q_len`` tokens of each of ``seqs`` sequences over such a cache, softmax in 32 bits, keys visible
  up to the token's own position (``window``: the last so many of them).

The cache as ``prepare`` lays it out: of every page and head, keys [offset, D / 2] bytes (element 2 i in the low
half of byte i, 2 i + 1 in the high one); values by fours of tokens [offset / 4, 16, D / 32, 4], where byte (c, w, j) of a four
has token j's elements 32 w + c (low) and 32 w + 16 + c (high); and [offset, 4] bfloat16: the keys' lowest value and step, the values'.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"


def listed():
    return [
        # one user's next word: q, k and v of the 4B size, one row
        _linear("8-bit product 1 row", 1, 6144, 2560, "bfloat16"),
        # a decoding batch on the 8B size's q, k and v
        _linear("8-bit product 24 rows", 24, 6144, 4096, "bfloat16"),
        # an ordinary prompt, the 4B size's down projection
        _linear("8-bit product 2048 rows", 2048, 2560, 9728, "bfloat16"),
        # the 32-bit mode with sizes that no tile divides
        _linear("8-bit product 37 rows float32", 37, 1001, 1100, "float32"),
        # the headline's batch of eight: the feed-forward's first half
        _gated("gated 8-bit product 8 rows", 8, 9728, 2560, "bfloat16"),
        # a prompt of 1,999 tokens through it
        _gated("gated 8-bit product 1999 rows", 1999, 9728, 2560, "bfloat16"),
        # eight requests store their next token
        _store("store 8 tokens", 8, 8, 128, 16, "bfloat16"),
        # a prompt's portion goes into the cache
        _store("store 2047 tokens", 2047, 8, 128, 16, "bfloat16"),
        # one user deep in a long document
        _attend("decode 1 over 32000", 1, 1, 32000, 32000, 32, 8, 128, 16, 0, "bfloat16"),
        # a busy server: contexts of very unequal lengths
        _attend("decode 48 ragged", 48, 1, 131, 2601, 32, 8, 128, 16, 0, "bfloat16"),
        # an ordinary prompt read in at once
        _attend("read 2048", 1, 2048, 2048, 2048, 32, 8, 128, 16, 0, "bfloat16"),
        # the 32-bit mode: short portions, a window, small pages
        _attend("portions of 7 in a window float32", 5, 7, 40, 700, 6, 2, 32, 8, 64, "float32"),
    ]


def _linear(name, rows, n, k, dtype):
    return {"name": name, "kind": "linear", "rows": rows, "n": n, "k": k, "dtype": dtype}


def _gated(name, rows, n, k, dtype):
    return {"name": name, "kind": "gated", "rows": rows, "n": n, "k": k, "dtype": dtype}


def _store(name, tokens, kv_heads, head_dim, page, dtype):
    return {"name": name, "kind": "store", "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype}


def _attend(name, seqs, q_len, shortest, longest, heads, kv_heads, head_dim, page, window, dtype):
    return {"name": name, "kind": "attend", "seqs": seqs, "q_len": q_len, "shortest": shortest, "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "window": window, "dtype": dtype}


def draw(rng):
    def spread(low, high):  # evenly over the logarithm
        return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.999))))))

    kind = rng.choice(["linear", "linear", "gated", "store", "attend", "attend", "attend"])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    if kind in ("linear", "gated"):
        rows, n, k = spread(1, 2048), spread(16, 9728), spread(64, 9728)
        if rng.random() < 0.5:  # half of them sizes as models have them
            n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
        rows = min(rows, max(1, 2048 * 9728 * 2560 // (n * k)))
        case = (_linear if kind == "linear" else _gated)("", rows, n, k, dtype)
    elif kind == "store":
        case = _store("", spread(1, 2048), rng.choice([1, 2, 4, 5, 8]), rng.choice([32, 64, 96, 128, 160, 256]), rng.choice([8, 16, 32, 24]), dtype)
    else:
        kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8])
        head_dim = rng.choice([32, 64, 96, 128, 128, 128, 256])
        longest = spread(1, 32000)
        # decoding for the most part; together no more than the largest listed ones
        q_len = 1 if rng.random() < 0.6 else spread(2, 1024)
        q_len = min(q_len, longest, max(1, 2048 * 1024 * 32 * 128 // (longest * kv_heads * group * head_dim)))
        seqs = max(1, min(spread(1, 48), 64000 // longest, 2048 * 1024 * 32 * 128 // (longest * q_len * kv_heads * group * head_dim)))
        shortest = rng.randint(q_len, longest)
        window = rng.choice([0, 0, 0, spread(1, 4096)])
        case = _attend("", seqs, q_len, shortest, longest, kv_heads * group, kv_heads, head_dim, rng.choice([8, 16, 16, 32, 24]), window, dtype)
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _lengths(case):
    """Keys of every sequence, its own tokens among them: from the shortest to the longest in equal ratios."""
    n, low, high = case["seqs"], case["shortest"], case["longest"]
    if n == 1:
        return [high]
    return [max(case["q_len"], min(high, round(low * (high / low) ** (i / (n - 1))))) for i in range(n)]


def _codes(x):
    """Codes 0 to 15, lowest value and step (bfloat16) of every vector of ``x`` [..., D], as the cache has them."""
    x = x.float()
    low = x.amin(-1, keepdim=True).to(torch.bfloat16)
    span = x.amax(-1, keepdim=True) - low.float()
    step = (span / torch.full_like(span, 15)).to(torch.bfloat16)  # by a tensor: by a number is a product with its reciprocal
    at = torch.where(step > 0, (x - low.float()) / step.float(), 0.0)
    return at.round().clamp(0, 15).to(torch.uint8), low[..., 0], step[..., 0]


def _pack_keys(codes):
    """[pages, heads, page, D] codes -> the pages' bytes."""
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _pack_values(codes):
    pages, heads, page, d = codes.shape
    c = codes.view(pages, heads, page // 4, 4, d // 32, 2, 16)   # four, token, w, half, c
    c = c[..., 0, :] | (c[..., 1, :] << 4)                       # four, token, w, c
    return c.permute(0, 1, 2, 5, 4, 3).reshape(pages, heads, page, d // 2).contiguous()


def prepare(case, seed):
    g = _generator(seed)
    dtype = getattr(torch, case["dtype"])

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    if case["kind"] in ("linear", "gated"):
        rows = case["n"] * (2 if case["kind"] == "gated" else 1)
        # activations as layers have them: a few channels are much larger than the others
        wide = torch.where(torch.rand(case["k"], generator=g, device=DEVICE) < 0.02, 8.0, 1.0)
        w = normal(rows, case["k"]) * (0.6 / math.sqrt(case["k"]))
        scale = w.abs().amax(-1) / 127
        state = {"case": case, "x": (normal(case["rows"], case["k"]) * wide).to(dtype), "scale": scale,
                 "values": (w / scale[:, None]).round().to(torch.int8)}
        if own:
            from qwen3_runtime_amd.ops import Int8Weight

            state["weight"] = Int8Weight(state["values"], scale)  # held as its kernels read it, as a loaded model's are
        return state

    page, heads, d = case["page"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "store":
        tokens = case["tokens"]
        pages = -(-tokens // page) + 2
        k, v = normal(tokens, heads, d).to(dtype), normal(tokens, heads, d).to(dtype)
        order = torch.randperm(pages, generator=g, device=DEVICE)
        at = torch.arange(tokens, device=DEVICE) + int(torch.randint(page, (1,), generator=g, device=DEVICE))
        slots = (order[at // page] * page + at % page).to(torch.int32)
        state = {"case": case, "k": k, "v": v, "slots": slots,
                 "k_pages": torch.zeros(pages, heads, page, d // 2, dtype=torch.uint8, device=DEVICE),
                 "v_pages": torch.zeros(pages, heads, page, d // 2, dtype=torch.uint8, device=DEVICE),
                 "steps": torch.zeros(pages, heads, page, 4, dtype=torch.bfloat16, device=DEVICE)}
    else:
        lens = _lengths(case)
        counts = [-(-n // page) for n in lens]
        pages = sum(counts) + 3
        order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
        table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32, device=DEVICE)
        for s, n in enumerate(counts):
            table[s, :n] = order[sum(counts[:s]): sum(counts[:s]) + n]
        k, k_low, k_step = _codes(normal(pages, heads, page, d))
        v, v_low, v_step = _codes(normal(pages, heads, page, d))
        q_len = case["q_len"]
        state = {"case": case, "q": normal(len(lens) * q_len, case["heads"] * d).to(dtype), "lens": lens, "table": table,
                 "kv_lens": torch.tensor(lens, dtype=torch.int32, device=DEVICE),
                 "k_pages": _pack_keys(k), "v_pages": _pack_values(v),
                 "steps": torch.stack([k_low, k_step, v_low, v_step], -1).contiguous()}
    if own:
        _as_a_step(state)
    return state


def _as_a_step(state):
    """The step's context and the cache's view, as the engine's step function has them for all its layers."""
    from qwen3_runtime_amd.parts.base import CacheView, GroupView, StepContext
    from qwen3_runtime_amd.parts.plan import CacheSpec

    case = state["case"]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    spec = CacheSpec("paged_kv", heads=case["kv_heads"], head_dim=case["head_dim"], bits=4)
    if case["kind"] == "store":
        group = GroupView(case["page"], None, i32([[0]]), state["slots"])
    else:
        lens, q_len = state["lens"], case["q_len"]
        group = GroupView(case["page"], case["window"] or None, state["table"], i32([0]))
        state["ctx"] = StepContext(
            ops=None, dtype=state["q"].dtype, device=torch.device(DEVICE), num_tokens=len(lens) * q_len, num_seqs=len(lens),
            positions=i32([n - q_len + i for n in lens for i in range(q_len)]), cu_q=i32([s * q_len for s in range(len(lens) + 1)]),
            kv_lens=state["kv_lens"], seq_of_token=i32([s for s in range(len(lens)) for _ in range(q_len)]), state_slots=i32([0] * len(lens)),
            first_span=i32([0] * len(lens)), q_lens_host=[q_len] * len(lens), kv_lens_host=list(lens), max_q_len=q_len, max_kv_len=max(lens),
            groups=[group])
    pages = {"k": state["k_pages"], "v": state["v_pages"], "steps": state["steps"]}
    state["cache"] = CacheView(spec, group=group, k=pages["k"], v=pages["v"], pages=pages)


# ---- one pass ------------------------------------------------------------------------------

_ops = []


def _framework():
    if not _ops:
        from qwen3_runtime_amd.ops.hip import HipOps

        _ops.append(HipOps())
    return _ops[0]


def run(state):
    case = state["case"]
    if case["kind"] == "linear":
        return _framework().linear(state["x"], state["weight"]) if own else _plain_linear(state["x"], state["values"], state["scale"]).to(state["x"].dtype)
    if case["kind"] == "gated":
        if own:
            return _framework().gated_linear(state["x"], state["weight"])
        gate, up = _plain_linear(state["x"], state["values"], state["scale"]).chunk(2, -1)
        return (gate / (1 + torch.exp(-gate)) * up).to(state["x"].dtype)
    if case["kind"] == "store":
        if own:
            _framework().kv_store(state["k"], state["v"], state["cache"])
        else:
            _plain_store(state)
        return _stored(state)
    if own:
        return _framework().paged_attention(state["q"], state["cache"], state["ctx"], case["heads"], case["kv_heads"], case["head_dim"],
                                            case["head_dim"] ** -0.5, case["window"] or None)
    return _plain_attend(state)


def _plain_linear(x, values, scale):
    x = x.float()
    most = x.abs().amax(-1, keepdim=True)
    top = torch.full_like(most, 127)  # a tensor: a quotient with a number is a product with a reciprocal
    by = torch.where(most < 2.0 ** -100, 0.0, top / most)  # the quotient stays in float32's range
    sums = (x * by).round().double() @ values.double().t()  # whole numbers beyond 2^24
    return sums.float() * (most / top) * scale


def _plain_store(state):
    page = state["case"]["page"]
    at, off = state["slots"].long() // page, state["slots"].long() % page
    k, k_low, k_step = _codes(state["k"])
    v, v_low, v_step = _codes(state["v"])
    state["k_pages"][at, :, off] = _pack_keys(k)
    tokens, heads, d = v.shape
    pages, fours = state["v_pages"].shape[0], page // 4
    v = v.view(tokens, heads, d // 32, 2, 16)
    v = (v[:, :, :, 0] | (v[:, :, :, 1] << 4)).transpose(2, 3)
    state["v_pages"].view(pages, heads, fours, 16, d // 32, 4)[at, :, off // 4, :, :, off % 4] = v
    state["steps"][at, :, off] = torch.stack([k_low, k_step, v_low, v_step], -1)


def _stored(state):
    """The stored tokens' keys and values as the cache holds them."""
    page, d = state["case"]["page"], state["case"]["head_dim"]
    at, off = state["slots"].long() // page, state["slots"].long() % page
    steps = state["steps"][at, :, off].float()
    keys = state["k_pages"][at, :, off]
    keys = torch.stack([keys & 15, keys >> 4], -1).flatten(-2)
    pages, heads = state["v_pages"].shape[:2]
    values = state["v_pages"].view(pages, heads, page // 4, 16, d // 32, 4)[at, :, off // 4, :, :, off % 4].transpose(2, 3)
    values = torch.stack([values & 15, values >> 4], -2).flatten(-3)
    return {"k": steps[..., 0:1] + steps[..., 1:2] * keys, "v": steps[..., 2:3] + steps[..., 3:4] * values}


def _plain_attend(state):
    case, table, q = state["case"], state["table"], state["q"]
    seqs, q_len, heads, kv_heads, d, page = case["seqs"], case["q_len"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    width = table.shape[1] * page
    pages = table.clamp(min=0).long()
    steps = state["steps"][pages].float()                                                    # [S, W, heads, page, 4]
    keys = state["k_pages"][pages]
    keys = steps[..., 0:1] + steps[..., 1:2] * torch.stack([keys & 15, keys >> 4], -1).flatten(-2)
    keys = keys.permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, width, d)
    values = state["v_pages"][pages].view(seqs, -1, kv_heads, page // 4, 16, d // 32, 4)
    values = torch.stack([values & 15, values >> 4], -2).permute(0, 1, 2, 3, 7, 5, 6, 4)     # [.., four, token, w, half, c]
    values = steps[..., 2:3] + steps[..., 3:4] * values.reshape(seqs, -1, kv_heads, page, d)
    values = values.permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, width, d)
    rows = q.float().view(seqs, q_len, kv_heads, heads // kv_heads, d).permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, -1, d)
    scores = torch.matmul(rows, keys.transpose(2, 3)) * d ** -0.5
    del keys
    key = torch.arange(width, device=DEVICE)
    position = state["kv_lens"].long()[:, None] - q_len + torch.arange(q_len, device=DEVICE)   # [S, q_len]
    seen = key <= position[..., None]
    if case["window"]:
        seen &= key > position[..., None] - case["window"]
    seen = seen[:, None, :, None].expand(seqs, 1, q_len, heads // kv_heads, width).reshape(seqs, 1, -1, width)
    scores = torch.where(seen, scores, -math.inf)
    scores = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(scores, values) / scores.sum(-1, keepdim=True)
    return out.view(seqs, kv_heads, q_len, -1, d).permute(0, 2, 1, 3, 4).reshape(seqs * q_len, heads * d).to(q.dtype)


# ---- what a pass cannot do without, and its results in 64 bits ---------------------------------


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] in ("linear", "gated"):
        rows, k, outs = case["rows"], case["k"], case["n"]
        n = outs * (2 if case["kind"] == "gated" else 1)
        return {"bytes": n * k + 4 * n + size * rows * (k + outs), "flops": 2 * rows * n * k}
    if case["kind"] == "store":
        vectors = case["tokens"] * case["kv_heads"] * 2
        return {"bytes": vectors * (case["head_dim"] * size + case["head_dim"] // 2 + 4), "flops": vectors * case["head_dim"] * 4}
    pairs = keys = 0
    for n in _lengths(case):
        span = case["window"] or n
        first = n - case["q_len"]
        pairs += sum(min(first + i + 1, span) for i in range(case["q_len"]))
        keys += min(n, span + case["q_len"] - 1)
    d = case["head_dim"]
    return {"bytes": keys * case["kv_heads"] * (d + 8) + 2 * size * case["seqs"] * case["q_len"] * case["heads"] * d,
            "flops": 4 * d * case["heads"] * pairs}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] in ("linear", "gated"):
        x = state["x"].double()
        most = x.abs().max(dim=1).values[:, None]
        # the codes are defined by two roundings to 32 bits: the factor's, and the product's in front of the rounding to whole numbers
        by = torch.where(most < 2.0 ** -100, 0.0, 127 / most).float().double()
        whole = torch.round((x * by).float().double())
        y = torch.matmul(whole, state["values"].double().t()) * (most / 127) * state["scale"].double()[None, :]
        if case["kind"] == "linear":
            return y
        gate, up = y[:, : case["n"]], y[:, case["n"]:]
        return gate * torch.sigmoid(gate) * up
    if case["kind"] == "store":
        held = {}
        for name in ("k", "v"):
            x = state[name].double()
            low = x.min(dim=-1, keepdim=True).values.to(torch.bfloat16).double()
            # the cache keeps these two in 16 bits; a difference and a quotient are rounded to 32 bits in front of the next step
            step = ((x.max(dim=-1, keepdim=True).values - low).float().double() / 15).float().to(torch.bfloat16).double()
            code = torch.round(((x - low).float().double() / torch.where(step > 0, step, 1.0)).float().double()).clamp(0, 15)
            held[name] = low + step * torch.where(step > 0, code, 0.0)
        return held
    d, group, page = case["head_dim"], case["heads"] // case["kv_heads"], case["page"]
    out = []
    for s, n in enumerate(state["lens"]):
        at = state["table"][s, torch.arange(n, device=DEVICE) // page].long()
        off = torch.arange(n, device=DEVICE) % page
        lows = state["steps"][at, :, off].double()                           # [n, heads, 4]
        byte = state["k_pages"][at, :, off].long()
        key = torch.empty(n, case["kv_heads"], d, dtype=torch.float64, device=DEVICE)
        key[..., 0::2], key[..., 1::2] = (byte % 16).double(), (byte // 16).double()
        fours = state["v_pages"].view(-1, case["kv_heads"], page // 4, 16, d // 32, 4)
        value = torch.empty_like(key)
        byte = fours[at, :, off // 4, :, :, off % 4].long()                 # [n, heads, 16, d / 32]
        for w in range(d // 32):
            value[..., 32 * w: 32 * w + 16] = (byte[..., w] % 16).double()
            value[..., 32 * w + 16: 32 * w + 32] = (byte[..., w] // 16).double()
        key = key * lows[..., 1:2] + lows[..., 0:1]
        value = value * lows[..., 3:4] + lows[..., 2:3]
        q = state["q"][s * case["q_len"]: (s + 1) * case["q_len"]].double().view(case["q_len"], case["heads"], d)
        position = torch.arange(n - case["q_len"], n, device=DEVICE)[:, None]
        hidden = torch.arange(n, device=DEVICE)[None, :] > position
        if case["window"]:
            hidden |= torch.arange(n, device=DEVICE)[None, :] <= position - case["window"]
        heads = []
        for h in range(case["heads"]):
            score = torch.matmul(q[:, h], key[:, h // group].t()) / math.sqrt(d)
            p = torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1)
            heads.append(torch.matmul(p, value[:, h // group]))
        out.append(torch.stack(heads, 1).reshape(case["q_len"], case["heads"] * d))
    return torch.cat(out)
