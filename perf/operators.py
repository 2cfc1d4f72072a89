"""The 4-bit key/value cache as timed cases: writing it, attending over it, thinning it out and reading it back.

Sizes are the attention shapes of the Llama-3.1-8B and 70B architectures (32 and 64 heads over 8 key/value heads of 128
channels), the batches, prompts and contexts of the decode harness and longer ones of the same kind, and small odd models.

A cache holds ``capacity`` entries for every sequence and key/value head:

* ``k_codes`` uint8 ``[B, KV, capacity, d/2]``: byte ``i`` holds channels ``2i`` (low half) and ``2i + 1``
* ``v_codes`` uint8 ``[B, KV, capacity/2, d]``: the rows of two neighbouring entries, in turns of two bytes
* ``params``  ``[B, KV, capacity, 4]`` in the model's type: scale and minimum of K, scale and minimum of V

and stands for ``minimum + scale * code``.  ``lengths[b]`` counts the entries of sequence ``b``, the call's own tokens among
them; a prompt shorter than the call's ``seq`` is padded on the left.
"""
import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
FLAGS = {"fp16": 1, "bf16": 1 | 2}
THETA = 500000.0
MOST_PAIRS = 32 * 2048 * 2048  # of queries and keys, over all heads
MOST_ENTRIES = 8 * 131072      # of a cache, over sequences and heads


def _append(name, batch, seq, heads, kv_heads, dim, capacity, fill, step, dtype):
    return {"name": name, "kind": "append", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "capacity": capacity, "fill": fill, "step": step, "dtype": dtype}


def _attend(name, batch, seq, heads, kv_heads, dim, capacity, fill, step, dtype, window=0, sinks=0, weights=False):
    return {"name": name, "kind": "attend", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "capacity": capacity, "fill": fill, "step": step, "dtype": dtype, "window": window, "sinks": sinks, "weights": weights}


def _evict(name, batch, kv_heads, dim, capacity, fill, step, keep, sinks, recent, dtype):
    return {"name": name, "kind": "evict", "batch": batch, "kv_heads": kv_heads, "dim": dim, "capacity": capacity, "fill": fill,
            "step": step, "keep": keep, "sinks": sinks, "recent": recent, "dtype": dtype}


def listed():
    return [
        # the new token of one user: the smallest write there is
        _append("append_step", 1, 1, 32, 8, 128, 4096, 700, 0, "fp16"),
        # eight prompts of 512 tokens
        _append("append_prompts", 8, 512, 32, 8, 128, 1024, 512, 0, "bf16"),
        # prompts of unequal lengths, padded on the left, in a small model of odd shape
        _append("append_ragged", 5, 37, 12, 3, 64, 64, 41, 9, "fp16"),
        # one user's token after a short prompt: latency
        _attend("step_short", 1, 1, 32, 8, 128, 256, 129, 0, "fp16"),
        # a serving batch, contexts of unequal lengths up to 4096
        _attend("step_batch", 32, 1, 32, 8, 128, 4096, 4096, 97, "bf16"),
        # one user with a long document, the larger model's heads
        _attend("step_long", 1, 1, 64, 8, 128, 131072, 131001, 0, "fp16"),
        # streaming: long contexts of which a window and the first tokens are visible
        _attend("step_window", 8, 1, 32, 8, 128, 32768, 32768, 3001, "bf16", window=1024, sinks=4),
        # a batch that thins its cache out: every step adds up what each entry was attended with
        _attend("step_weights", 8, 1, 32, 8, 128, 2048, 2048, 111, "fp16", weights=True),
        # one prompt of 2048 tokens
        _attend("prompt", 1, 2048, 32, 8, 128, 2048, 2048, 0, "bf16"),
        # later pieces of two prompts, window and first tokens, weights for the eviction behind them
        _attend("prompt_window", 2, 1000, 32, 8, 128, 5056, 5003, 1500, "fp16", window=1024, sinks=4, weights=True),
        # one user's cache cut back to its budget
        _evict("evict_one", 1, 8, 128, 1152, 1088, 0, 1024, 4, 256, "fp16"),
        # a batch of long caches cut by half, some short enough to stay as they are
        _evict("evict_batch", 4, 8, 128, 16384, 16001, 4500, 8192, 4, 1024, "bf16"),
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    kind = rng.choice(["append", "step", "step", "prompt", "evict"])
    dtype = rng.choice(["fp16", "bf16"])
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 8])
    up = lambda n: -(-n // 64) * 64  # noqa: E731
    if kind == "append":
        batch = _spread(rng, 1, 16)
        seq = _spread(rng, 1, 4096 // batch)
        fill = seq + rng.choice([0, _spread(rng, 1, 2000), -(seq // 3)])
        return _append("", batch, seq, heads, kv_heads, dim, up(max(fill, seq) + 1), fill, rng.choice([0, _spread(rng, 1, max(2, fill // 2))]),
                       dtype)
    if kind == "evict":
        batch = _spread(rng, 1, 8)
        fill = _spread(rng, 40, 65536 // (batch * kv_heads) * 2)
        keep = max(8, int(fill * rng.uniform(0.3, 0.99)))
        sinks, recent = rng.choice([0, 1, 4]), rng.randrange(0, keep - 4)
        return _evict("", batch, kv_heads, dim, up(fill + 7), fill, rng.choice([0, _spread(rng, 1, fill // 2)]), keep, sinks, recent, dtype)
    window, sinks = rng.choice([(0, 0), (_spread(rng, 1, 4096), rng.choice([0, 1, 4, 31]))])
    weights = rng.random() < 0.4
    if kind == "step":
        batch = _spread(rng, 1, 48)
        fill = _spread(rng, 1, MOST_ENTRIES // (batch * kv_heads) // 2)
        fill = min(fill, MOST_ENTRIES // 8)
        seq = rng.choice([1, 1, 1, 2, 5])
    else:
        batch = _spread(rng, 1, 4)
        seq = _spread(rng, 9, 2048)
        fill = min(8192, seq + rng.choice([0, _spread(rng, 1, 4096)]))
        most = MOST_PAIRS // (batch * heads * seq)
        fill = min(fill, max(64, most))
    return _attend("", batch, seq, heads, kv_heads, dim, up(fill + 1), fill, rng.choice([0, _spread(rng, 1, max(2, fill))]), dtype, window,
                   sinks, weights)


def _lengths(case):
    """Entries of each sequence: the first has ``fill``, each further one ``step`` fewer, none less than one."""
    return [max(1, case["fill"] - b * case["step"]) for b in range(case["batch"])]


# ---- the cache in plain operations ---------------------------------------------------------------------------------
def _nibbles(rows):
    """``[..., d/2]`` bytes -> ``[..., d]`` codes."""
    return torch.stack([rows & 15, rows >> 4], -1).flatten(-2)


def _bytes(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _v_rows(v_codes):
    """``[B, KV, capacity/2, d]`` -> rows ``[B, KV, capacity, d/2]`` of bytes, one for each entry."""
    b, h, pairs, d = v_codes.shape
    return v_codes.view(b, h, pairs, d // 4, 2, 2).transpose(3, 4).reshape(b, h, 2 * pairs, d // 2)


def _v_pairs(rows):
    """The inverse of ``_v_rows``."""
    b, h, capacity, half = rows.shape
    return rows.view(b, h, capacity // 2, 2, half // 2, 2).transpose(3, 4).reshape(b, h, capacity // 2, 2 * half)


def _quantise(x):
    """Rows of 16-bit numbers -> codes, scale, minimum."""
    low, high = x.float().amin(-1, keepdim=True), x.float().amax(-1, keepdim=True)
    scale = ((high - low) / 15).to(x.dtype)
    codes = torch.where(scale > 0, (x.float() - low) / scale.float(), 0).round().clamp(0, 15).to(torch.uint8)
    return codes, scale, low.to(x.dtype)


def _dense(state):
    """K and V of the whole cache in fp32."""
    p = state["params"].float()
    k = p[..., 1:2] + p[..., 0:1] * _nibbles(state["k_codes"]).float()
    v = p[..., 3:4] + p[..., 2:3] * _nibbles(_v_rows(state["v_codes"])).float()
    return k, v


def _last(k, v, lengths, count, dtype):
    """The last ``count`` entries of each sequence, zeros where it has fewer."""
    slot = (lengths[:, None] - count + torch.arange(count, device=k.device)).long()
    at = slot.clamp(min=0)[:, None, :, None].expand(-1, k.shape[1], -1, k.shape[3])
    there = (slot >= 0)[:, None, :, None]
    return torch.where(there, k.gather(2, at), 0).to(dtype), torch.where(there, v.gather(2, at), 0).to(dtype)


def _rotate(x, cos, sin):
    """Pairs ``(2i, 2i + 1)`` by their angle, in 64 bits: what lies next to a border between codes is decided here."""
    a, b = x[..., 0::2].double(), x[..., 1::2].double()
    return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2).to(x.dtype)


# ---- inputs ----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = TYPES[case["dtype"]]
    b, kv, d, capacity = case["batch"], case["kv_heads"], case["dim"], case["capacity"]
    randn = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    s = {"kind": case["kind"], "case": case, "flags": FLAGS[case["dtype"]],
         "lengths": torch.tensor(_lengths(case), dtype=torch.int32, device=dev)}
    # keys have channels that stand out, the same for all tokens of a head
    offset = randn(kv, d) * (torch.rand(kv, d, generator=gen, device=dev) < 0.05) * 4
    if case["kind"] == "append":
        h, seq = case["heads"], case["seq"]
        qkv = randn(b, seq, h + 2 * kv, d)
        qkv[:, :, h:h + kv] += offset
        s["qkv"] = qkv.to(dtype).view(b * seq, (h + 2 * kv) * d)
        s["positions"] = (s["lengths"][:, None].long() - seq + torch.arange(seq, device=dev)).clamp(min=0)
        inv = 1.0 / (THETA ** (torch.arange(0, d, 2, device=dev, dtype=torch.float32) / d))
        angle = torch.arange(capacity, device=dev, dtype=torch.float32)[:, None] * inv[None, :]
        s["cos"], s["sin"] = angle.cos(), angle.sin()
        s["k_codes"] = torch.zeros(b, kv, capacity, d // 2, dtype=torch.uint8, device=dev)
        s["v_codes"] = torch.zeros(b, kv, capacity // 2, d, dtype=torch.uint8, device=dev)
        s["params"] = torch.zeros(b, kv, capacity, 4, dtype=dtype, device=dev)
        return s
    s["k_codes"] = torch.empty(b, kv, capacity, d // 2, dtype=torch.uint8, device=dev)
    s["v_codes"] = torch.empty(b, kv, capacity // 2, d, dtype=torch.uint8, device=dev)
    s["params"] = torch.empty(b, kv, capacity, 4, dtype=dtype, device=dev)
    for i in range(b):  # a sequence at a time: the dense form of a whole cache is large
        k_codes, k_scale, k_min = _quantise((randn(kv, capacity, d) + offset[:, None]).to(dtype))
        v_codes, v_scale, v_min = _quantise(randn(kv, capacity, d).to(dtype))
        s["k_codes"][i], s["v_codes"][i] = _bytes(k_codes), _v_pairs(_bytes(v_codes)[None])[0]
        s["params"][i] = torch.cat([k_scale, k_min, v_scale, v_min], -1)
    if case["kind"] == "attend":
        s["q"] = (randn(b, case["seq"], case["heads"], d) * 1.5).to(dtype)
        # what the steps before have left there
        s["weights"] = torch.rand(b, kv, capacity, generator=gen, device=dev) if case["weights"] else None
    else:
        # few entries take most of the attention
        s["weights"] = (2.0 * randn(b, kv, capacity)).exp()
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[state["kind"]](state)


def _own(s):
    from matgptq_b200 import ops
    c, cache = s["case"], (s["k_codes"], s["v_codes"], s["params"])
    if c["kind"] == "append":
        q = ops.append_kv4(s["qkv"], s["positions"], s["cos"], s["sin"], s["lengths"], *cache, c["heads"], s["flags"])
        k, v = ops.dequantize_kv4(*cache, s["lengths"], c["seq"], s["flags"])
        return {"q": q, "k": k, "v": v}
    if c["kind"] == "attend":
        out = ops.attention_kv4(s["q"], *cache, s["lengths"], c["window"], c["sinks"], 1.0 / math.sqrt(c["dim"]), s["flags"], s["weights"])
        return {"out": out, "weights": s["weights"]}
    lengths, kept = ops.evict_kv4(*cache, s["weights"], s["lengths"], c["keep"], 0, c["sinks"], c["recent"], s["flags"])
    k, v = ops.dequantize_kv4(*cache, lengths, c["keep"], s["flags"])
    return {"lengths": lengths, "kept": kept, "k": k, "v": v, "weights": s["weights"]}


def _plain_append(s):
    c = s["case"]
    b, seq, h, kv, d = c["batch"], c["seq"], c["heads"], c["kv_heads"], c["dim"]
    qkv = s["qkv"].view(b, seq, h + 2 * kv, d)
    slot = s["lengths"][:, None].long() - seq + torch.arange(seq, device=qkv.device)
    cos, sin = (t[s["positions"]].double()[:, :, None] for t in (s["cos"], s["sin"]))
    turned = _rotate(qkv[:, :, :h + kv], cos, sin)
    q = torch.where((slot >= 0)[:, :, None, None], turned[:, :, :h], 0)
    # padding is written as the last token once more
    token = torch.where(slot >= 0, torch.arange(seq, device=qkv.device), seq - 1)
    row = torch.arange(b, device=qkv.device)[:, None]
    slot = slot.gather(1, token)
    k_codes, k_scale, k_min = _quantise(turned[:, :, h:][row, token])
    v_codes, v_scale, v_min = _quantise(qkv[:, :, h + kv:][row, token])
    s["k_codes"].transpose(1, 2)[row, slot] = _bytes(k_codes)
    units = s["v_codes"].view(b, kv, -1, d // 4, 2, 2).permute(0, 2, 4, 1, 3, 5)  # sequence, pair, which of it, head, unit, byte
    units[row, slot // 2, slot % 2] = _bytes(v_codes).view(b, seq, kv, d // 4, 2)
    s["params"].transpose(1, 2)[row, slot] = torch.cat([k_scale, k_min, v_scale, v_min], -1)
    # what the cache now holds of these tokens
    p = s["params"].transpose(1, 2)[row, slot].float()
    k = p[..., 1:2] + p[..., 0:1] * _nibbles(s["k_codes"].transpose(1, 2)[row, slot]).float()
    v = p[..., 3:4] + p[..., 2:3] * _nibbles(units[row, slot // 2, slot % 2].reshape(b, seq, kv, d // 2)).float()
    there = (token == torch.arange(seq, device=qkv.device))[:, :, None, None]
    k, v = (torch.where(there, t, 0).to(q.dtype).transpose(1, 2) for t in (k, v))
    return {"q": q, "k": k, "v": v}


def _visible(lengths, seq, capacity, window, sinks):
    """``[B, seq, capacity]``: which entries a query sees."""
    key = torch.arange(capacity, device=lengths.device)
    at = (lengths[:, None].long() - seq + torch.arange(seq, device=lengths.device))[:, :, None]
    seen = key <= at
    if window > 0:
        seen = seen & ((key > at - window) | (key < sinks))
    return seen


def _plain_attend(s):
    c, q = s["case"], s["q"]
    b, seq, h, d = q.shape
    kv = c["kv_heads"]
    k, v = _dense(s)
    rows = q.float().view(b, seq, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, h // kv * seq, d)
    seen = _visible(s["lengths"], seq, c["capacity"], c["window"], c["sinks"])[:, None].repeat(1, 1, h // kv, 1)
    score = (rows @ k.transpose(2, 3) / math.sqrt(d)).masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top > -math.inf, top, 0)).exp_()  # a row that sees nothing: zeros
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1))
    # entries behind the last one may hold anything
    v = torch.where(torch.arange(c["capacity"], device=q.device)[:, None] < s["lengths"][:, None, None, None], v, 0)
    out = (p @ v).view(b, kv, h // kv, seq, d).permute(0, 3, 1, 2, 4).reshape(b, seq, h, d).to(q.dtype)
    if s["weights"] is not None:
        s["weights"] += p.sum(2)
    return {"out": out, "weights": s["weights"]}


def _plain_evict(s):
    c, w = s["case"], s["weights"]
    b, kv, capacity = w.shape
    keep = c["keep"]
    lengths = s["lengths"][:, None, None]
    key = torch.arange(capacity, device=w.device)
    rank = torch.where((key < c["sinks"]) | (key >= lengths - c["recent"]), math.inf, w.double())
    rank = torch.where(key < lengths, rank, -math.inf)
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    cut = (lengths > keep).expand(b, kv, 1)
    at = torch.where(cut, torch.cat([kept, key[keep:].expand(b, kv, -1)], -1), key)  # where each slot's entry comes from
    rows = at[..., None].expand(-1, -1, -1, c["dim"] // 2)
    s["k_codes"].copy_(s["k_codes"].gather(2, rows))
    s["v_codes"].copy_(_v_pairs(_v_rows(s["v_codes"]).gather(2, rows)))
    s["params"].copy_(s["params"].gather(2, at[..., None].expand(-1, -1, -1, 4)))
    w.copy_(torch.where(cut & (key >= keep) & (key < lengths), 0, w.gather(2, at)))
    new = torch.where(s["lengths"] > keep, keep, s["lengths"])
    k, v = _last(*_dense(s), new, keep, s["params"].dtype)
    return {"lengths": new, "kept": torch.where(cut, kept, -1).int(), "k": k, "v": v, "weights": w}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    b, kv, d = case["batch"], case["kv_heads"], case["dim"]
    lengths = _lengths(case)
    entry = d + 8  # bytes of an entry of one head
    if case["kind"] == "append":
        h, seq = case["heads"], case["seq"]
        new = sum(min(n, seq) for n in lengths)
        angles = len(set().union(*(range(max(0, n - seq), n) for n in lengths)))
        read = new * (h + 2 * kv) * d * 2 + new * 8 + angles * d * 4
        return {"bytes": read + b * seq * h * d * 2 + new * kv * entry + b * seq * kv * d * 4, "flops": new * (h + 3 * kv) * d * 4}
    if case["kind"] == "evict":
        keep = case["keep"]
        cut, left = [n for n in lengths if n > keep], [n for n in lengths if n <= keep]
        moved = sum(cut) * kv * 8 + len(cut) * kv * keep * 2 * entry  # weights and kept entries, read and written
        return {"bytes": moved + sum(left) * kv * entry + b * kv * keep * (d * 4 + 4),
                "flops": sum(min(n, keep) for n in lengths) * kv * d * 4}
    h, seq, window, sinks = case["heads"], case["seq"], case["window"], case["sinks"]
    pairs = entries = 0
    for n in lengths:
        first = max(0, n - seq)  # position of the first query
        for at in range(first, n):
            pairs += at + 1 if not window or at + 1 <= window else window + min(sinks, at + 1 - window)
        start = max(0, first + 1 - window) if window else 0
        entries += n - start + min(sinks, start)
    moved = b * seq * h * d * 2 * 2 + entries * kv * entry + (entries * kv * 8 if case["weights"] else 0)
    return {"bytes": moved, "flops": pairs * h * 4 * d}


# ---- the definition, in 64 bits ------------------------------------------------------------------------------------
def _values(codes, scale, low):
    return low.double() + scale.double() * codes.double()


def _stored(x):
    """What a row of 16-bit numbers is kept as: sixteen levels from its minimum, in steps of a sixteenth-bit scale."""
    x64 = x.double()
    low, high = x64.min(-1, keepdim=True).values, x64.max(-1, keepdim=True).values
    scale = ((high - low) / 15).to(x.dtype).double()
    level = torch.round((x64 - low) / torch.where(scale == 0, torch.ones_like(scale), scale))
    return low + scale * torch.minimum(level, torch.full_like(level, 15)) * (scale != 0)


def exact(case, seed):
    s = prepare(case, seed)
    c, dev = case, s["lengths"].device
    if c["kind"] == "append":
        b, seq, h, kv, d = c["batch"], c["seq"], c["heads"], c["kv_heads"], c["dim"]
        x = s["qkv"].view(b, seq, h + 2 * kv, d).double().view(b, seq, h + 2 * kv, d // 2, 2)
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, :, None]
        turned = torch.view_as_real(torch.view_as_complex(x[:, :, :h + kv].contiguous()) * turn).flatten(-2)
        real = torch.arange(seq, device=dev)[None] >= seq - s["lengths"][:, None]
        real = real[:, :, None, None].double()
        k = _stored(turned[:, :, h:].to(TYPES[c["dtype"]]))
        v = _stored(s["qkv"].view(b, seq, h + 2 * kv, d)[:, :, h + kv:])
        return {"q": turned[:, :, :h] * real, "k": (k * real).transpose(1, 2), "v": (v * real).transpose(1, 2)}
    low, high = s["k_codes"] & 15, s["k_codes"] >> 4
    k_codes = torch.empty(*low.shape[:3], c["dim"], dtype=torch.uint8, device=dev)
    k_codes[..., 0::2], k_codes[..., 1::2] = low, high
    b, kv, pairs, d = s["v_codes"].shape
    v_bytes = s["v_codes"].view(b, kv, pairs, d // 4, 2, 2)
    v_codes = torch.empty(b, kv, pairs, 2, d // 4, 4, dtype=torch.uint8, device=dev)
    for which in range(2):
        for byte in range(2):
            v_codes[:, :, :, which, :, 2 * byte] = v_bytes[:, :, :, :, which, byte] & 15
            v_codes[:, :, :, which, :, 2 * byte + 1] = v_bytes[:, :, :, :, which, byte] >> 4
    v_codes = v_codes.view(b, kv, 2 * pairs, d)
    p = s["params"]
    if c["kind"] == "evict":
        new, kept_all, ks, vs, ws = [], [], [], [], []
        for i, n in enumerate(_lengths(c)):
            keep = c["keep"]
            k = _values(k_codes[i, :, :n], p[i, :, :n, 0:1], p[i, :, :n, 1:2])
            v = _values(v_codes[i, :, :n], p[i, :, :n, 2:3], p[i, :, :n, 3:4])
            w = s["weights"][i].double()
            pad = torch.zeros(kv, max(0, keep - n), d, dtype=torch.float64, device=dev)
            if n <= keep:
                kept = torch.full((kv, keep), -1, device=dev)
                k, v = torch.cat([pad, k], 1), torch.cat([pad, v], 1)
            else:
                middle = w[:, c["sinks"]:n - c["recent"]]
                order = torch.sort(-middle, dim=-1, stable=True).indices[:, :keep - c["sinks"] - c["recent"]] + c["sinks"]
                mark = torch.zeros(kv, n, dtype=torch.bool, device=dev)
                mark[:, :c["sinks"]] = True
                mark[:, n - c["recent"]:] = True
                mark.scatter_(1, order, True)
                kept = mark.nonzero()[:, 1].view(kv, keep)
                k, v = (t.gather(1, kept[..., None].expand(-1, -1, d)) for t in (k, v))
                w = torch.cat([w.gather(1, kept), torch.zeros(kv, n - keep, dtype=torch.float64, device=dev), w[:, n:]], 1)
            new.append(min(n, keep))
            kept_all.append(kept), ks.append(k), vs.append(v), ws.append(w)
        return {"lengths": torch.tensor(new, device=dev), "kept": torch.stack(kept_all), "k": torch.stack(ks), "v": torch.stack(vs),
                "weights": torch.stack(ws)}
    seq, h = c["seq"], c["heads"]
    out = torch.zeros(b, seq, h, d, dtype=torch.float64, device=dev)
    weights = s["weights"].double() if c["weights"] else None
    for i, n in enumerate(_lengths(c)):
        first = max(0, seq - n)  # queries before it are padding
        at = torch.arange(n - seq + first, n, device=dev)[:, None]
        key = torch.arange(n, device=dev)[None]
        hidden = key > at
        if c["window"]:
            hidden |= (at - key >= c["window"]) & (key >= c["sinks"])
        for j in range(kv):
            k = _values(k_codes[i, j, :n], p[i, j, :n, 0:1], p[i, j, :n, 1:2])
            v = _values(v_codes[i, j, :n], p[i, j, :n, 2:3], p[i, j, :n, 3:4])
            group = slice(j * (h // kv), (j + 1) * (h // kv))
            score = torch.einsum("qhd,kd->hqk", s["q"][i, first:, group].double(), k) / math.sqrt(d)
            prob = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            out[i, first:, group] = torch.einsum("hqk,kd->qhd", prob, v)
            if weights is not None:
                weights[i, j, :n] += prob.sum((0, 1))
    return {"out": out, "weights": weights}
