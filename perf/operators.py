"""Cases of the paged key/value store: writing new tokens into pages (16-bit elements, or 8- and
4-bit codes with one (scale, zero) per token and head), reading them back, and the causal attention
of a batch's newest tokens over their pages, with and without a sliding window and first tokens
that stay visible.

A store of ``pages`` pages holds, for every page and kv head, ``page`` token rows of ``dim``
elements: 16-bit rows as they are, codes of a row first-channel-in-low-bits.  Sequence b of a batch
owns the pages of row b of the block table, ``kv_lens[b]`` tokens including the newest
``cu[b + 1] - cu[b]``, which are rows cu[b] .. of the dense arrays.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _case(name, op, **kw):
    case = {"name": name, "op": op, "batch": 1, "tokens": 1, "context": 1, "ragged": False, "heads": 8, "group": 4, "dim": 128, "page": 16,
            "bits": 16, "type": "bf16", "window": 0, "sinks": 0}
    case.update(kw)
    return case


def listed():
    return [
        # a decode step's append: one token of each of 16 sequences into 8-bit pages, and its read-back
        _case("append_step_8bit", "append", batch=16, tokens=1, context=4096, bits=8),
        # a prompt chunk of 16 sequences entering 8-bit pages, and its read-back
        _case("append_prompt_8bit", "append", batch=16, tokens=2048, context=2048, page=64, bits=8),
        # ragged fp32 prompts of a small model entering 4-bit pages
        _case("append_ragged_4bit", "append", batch=7, tokens=1531, context=2750, ragged=True, heads=4, dim=64, page=32, bits=4, type="f32"),
        # whole ragged sequences read back from 8-bit pages, for a consumer of dense keys and values
        _case("read_back_8bit", "read", batch=8, tokens=8192, context=8192, ragged=True, page=32, bits=8),
        # one decode step of a single chat over 8-bit pages: latency counts
        _case("decode_short_8bit", "attend", batch=1, context=4096, bits=8),
        # decode of 16 long sequences over 16-bit pages: bandwidth counts
        _case("decode_long_bf16", "attend", batch=16, context=32768, page=64),
        # decode of ragged long sequences with eight query heads per kv head over 4-bit pages
        _case("decode_ragged_4bit", "attend", batch=8, context=65521, ragged=True, group=8, page=32, bits=4),
        # a draft of up to 7 tokens verified over ragged 8-bit pages
        _case("draft_ragged_8bit", "attend", batch=13, tokens=7, context=5003, ragged=True, page=32, bits=8),
        # a chunk of a long prompt over its history in 16-bit pages
        _case("chunk_bf16", "attend", batch=1, tokens=2048, context=10240, page=64),
        # ragged prompt chunks over 8-bit pages
        _case("chunk_ragged_8bit", "attend", batch=4, tokens=1024, context=7993, ragged=True, page=128, bits=8),
        # a decode step of 16 streaming sequences: four first tokens and a window stay visible
        _case("window_decode_bf16", "attend", batch=16, context=32768, page=64, window=4096, sinks=4),
        # a long prompt under the same mask, window within the prompt
        _case("window_prompt_bf16", "attend", batch=1, tokens=8192, context=8192, page=64, window=1024, sinks=4),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["append", "append", "read", "attend", "attend", "attend", "window", "window"])
    while True:
        bits = rng.choice([16, 8, 4])
        c = {"op": "attend" if op == "window" else op, "batch": log(1, 24), "ragged": rng.random() < 0.6, "heads": rng.choice([1, 2, 4, 8]),
             "group": rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), "dim": rng.choice([32, 64, 96, 128, 128]), "page": rng.choice([16, 32, 64, 128, 256]),
             "bits": bits, "type": rng.choice(["bf16", "bf16", "f16"]), "window": 0, "sinks": 0}
        if op in ("append", "read") and bits != 16 and rng.random() < 0.3:
            c["type"] = "f32"
        c["tokens"] = 1 if op in ("attend", "window") and rng.random() < 0.4 else log(1, 8192)
        c["context"] = c["tokens"] + log(1, 32768) - 1
        if op == "window":
            c["window"], c["sinks"] = log(1, 8192), rng.choice([0, 1, 4, 4, 21, 128])
        rows = c["batch"] * c["heads"] * c["context"]
        pairs = c["batch"] * c["heads"] * c["group"] * c["tokens"] * c["context"]
        if rows * c["dim"] <= 2**28 and pairs <= 2**30 and rows >= 64:
            return c


# ------------------------------------------------------------------ lengths and work


def _lengths(case):
    """(newest tokens, tokens with them) of each sequence, from the case alone."""
    n, t = case["tokens"], case["context"]
    if not case["ragged"]:
        return [n] * case["batch"], [t] * case["batch"]
    new = [max(1, n - (b * 7919) % (n // 2 + 1)) for b in range(case["batch"])]
    old = [max(0, (t - n) - (b * 104729) % ((t - n) * 3 // 4 + 1)) for b in range(case["batch"])]
    if case["op"] == "read":  # whole sequences
        return new, new
    return new, [x + y for x, y in zip(new, old)]


def _seen(new, kv, window, sinks):
    """(query, key) pairs of one sequence and head, and the keys that any query sees."""
    def upto(p):  # sum over positions 0 .. p of the visible tokens
        if p < 0:
            return 0
        if not window:
            return (p + 1) * (p + 2) // 2
        both = window + sinks
        full = min(p + 1, both)
        return full * (full + 1) // 2 + max(0, p + 1 - both) * both

    pairs = upto(kv - 1) - upto(kv - new - 1)
    if not window:
        return pairs, kv
    low = max(0, kv - new - window + 1)
    return pairs, kv - low + min(sinks, low)


def work(case):
    new, kv = _lengths(case)
    h, d, e = case["heads"], case["dim"], 4 if case["type"] == "f32" else 2
    row = d * case["bits"] // 8 + (8 if case["bits"] < 16 else 0)
    rows = sum(new) * h
    if case["op"] == "append":
        return {"bytes": 2 * rows * (2 * d * e + 2 * row), "flops": 0}
    if case["op"] == "read":
        return {"bytes": 2 * rows * (d * e + row), "flops": 0}
    seen = [_seen(n, t, case["window"], case["sinks"]) for n, t in zip(new, kv)]
    return {"bytes": 2 * sum(k for _, k in seen) * h * row + 2 * rows * case["group"] * d * e,
            "flops": 4 * d * h * case["group"] * sum(p for p, _ in seen)}


# ------------------------------------------------------------------ inputs


def _inputs(case, seed):
    """Everything a step has in hand: the pool with the sequences' history, the block table, the
    lengths, the new tokens and queries.  Keys have channels of unlike size, as trained ones do."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    new, kv = _lengths(case)
    h, d, page, bits = case["heads"], case["dim"], case["page"], case["bits"]
    dtype = _TYPES[case["type"]]
    per = -(-max(kv) // page)
    used = [-(-n // page) for n in kv]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((case["batch"], per), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s = {"case": case, "table": table, "cu": torch.tensor(cu, dtype=torch.int32, device=dev), "kv_lens": torch.tensor(kv, dtype=torch.int32, device=dev),
         "total": cu[-1], "most": max(new)}
    gain = torch.exp(0.5 * torch.randn(h, d, generator=g, device=dev))

    def rows(shape, keys):
        x = torch.randn(*shape, d, generator=g, device=dev)
        return x * gain[:, None] if keys and len(shape) == 3 else x * gain if keys else x

    for side in ("keys", "values"):
        if bits == 16:
            pool = torch.empty(pages, h, page, d, dtype=dtype, device=dev)
        else:
            pool = torch.empty(pages, h, page, d * bits // 8, dtype=torch.uint8, device=dev)
            s[side + "_params"] = torch.zeros(pages, h, page, 2, device=dev)
        for lo in range(0, pages, max(1, 2**26 // (h * page * d))):
            hi = min(pages, lo + max(1, 2**26 // (h * page * d)))
            x = rows((hi - lo, h, page), side == "keys")
            if bits == 16:
                pool[lo:hi] = x.to(dtype)
            else:
                pool[lo:hi], s[side + "_params"][lo:hi] = _codes(x, bits)
        s[side] = pool
    if case["op"] == "append":
        s["new_keys"], s["new_values"] = rows((cu[-1], h), True).to(dtype), rows((cu[-1], h), False).to(dtype)
    if case["op"] == "attend":
        s["query"] = torch.randn(cu[-1], h * case["group"], d, generator=g, device=dev).to(dtype)
        s["scale"] = 1.0 / math.sqrt(d)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # the handle over the pool and the step's batch, which every layer of a model shares
        K = _kivi()
        s["batch"] = K.PagesBatch(s["table"], s["cu"], s["kv_lens"], s["total"], s["most"])
        config = K.PagesConfig(bits=case["bits"], dtype=case["type"], num_pages=s["keys"].shape[0], page_size=case["page"],
                               num_kv_heads=case["heads"], head_dim=case["dim"])
        s["pages"] = K.KvPages(config, s["keys"], s["values"], s.get("keys_params"), s.get("values_params"))
    return s


def _kivi():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kivi-cache-rs_b200")
    if not os.path.isdir(package):
        package = os.path.join(os.getcwd(), "kivi-cache-rs_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import kivi_cache

    return kivi_cache


# ------------------------------------------------------------------ the framework's calls


def _run_own(s):
    case = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "attend":
        out = torch.empty_like(s["query"])
        s["pages"].attention_dev(s["batch"], s["query"], case["heads"] * case["group"], s["scale"], out, window=case["window"],
                                 sinks=case["sinks"], stream=stream)
        return out
    if case["op"] == "append":
        s["pages"].write_dev(s["batch"], s["new_keys"], s["new_values"], stream=stream)
    shape, dtype = (s["total"], case["heads"], case["dim"]), _TYPES[case["type"]]
    keys, values = torch.empty(shape, dtype=dtype, device="cuda"), torch.empty(shape, dtype=dtype, device="cuda")
    s["pages"].read_dev(s["batch"], keys, values, stream=stream)
    return keys, values


# ------------------------------------------------------------------ the plain form


def _codes(x, bits):
    """Codes (packed, first channel in the low bits) and (scale, zero) of the rows of x, in fp32."""
    top = 2**bits - 1
    zero = x.amin(-1, keepdim=True)
    scale = (x.amax(-1, keepdim=True) - zero) / torch.full((1,), float(top), device=x.device)
    c = torch.where(scale > 0, torch.round((x - zero) / scale), torch.zeros_like(x)).clamp_(0, top).to(torch.uint8)
    if bits == 4:
        c = c[..., 0::2] | (c[..., 1::2] << 4)
    return c, torch.cat((scale, zero), -1)


def _values(pool, params, bits, where):
    """The fp32 rows of a pool at ``where`` = (page, slot), any shape: [..., heads, dim]."""
    x = pool[where[0], :, where[1]]
    if bits == 16:
        return x.float()
    p = params[where[0], :, where[1]]
    if bits == 4:
        x = torch.stack((x & 15, x >> 4), -1).flatten(-2)
    return x.float() * p[..., :1] + p[..., 1:]


def _places(s):
    """(page, slot) of every one of the batch's newest tokens."""
    at = torch.arange(s["total"], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["cu"], at, right=True) - 1
    t = s["kv_lens"][b] - s["cu"][b + 1] + at
    page = s["case"]["page"]
    return s["table"][b, t // page].long(), (t % page).long()


def _run_plain(s):
    case = s["case"]
    bits, dtype = case["bits"], _TYPES[case["type"]]
    if case["op"] != "attend":
        where = _places(s)
        if case["op"] == "append":
            for side in ("keys", "values"):
                x = s["new_" + side]
                if bits == 16:
                    s[side][where[0], :, where[1]] = x
                else:
                    s[side][where[0], :, where[1]], s[side + "_params"][where[0], :, where[1]] = _codes(x.float(), bits)
        return tuple(_values(s[side], s.get(side + "_params"), bits, where).to(dtype) for side in ("keys", "values"))
    batch, page = case["batch"], case["page"]
    h, g, d, most = case["heads"], case["group"], case["dim"], s["most"]
    width = s["table"].shape[1] * page
    t = torch.arange(width, device="cuda")
    where = s["table"].clamp(min=0).long()[:, t // page], (t % page).expand(batch, width)
    new = (s["cu"][1:] - s["cu"][:-1])[:, None]
    i = torch.arange(most, device="cuda")[None]
    rows = (s["cu"][:-1, None] + i).clamp(max=s["total"] - 1).long()
    position = s["kv_lens"][:, None] - new + i                                  # [batch, most]
    seen = (t <= position[..., None]) & (t < s["kv_lens"][:, None, None])       # [batch, most, width]
    if case["window"]:
        seen &= (t > position[..., None] - case["window"]) | (t < case["sinks"])
    q = s["query"].float()[rows].view(batch, most, h, g, d).permute(0, 2, 3, 1, 4).reshape(batch, h, g * most, d)
    x = (q * s["scale"]) @ _values(s["keys"], s.get("keys_params"), bits, where).permute(0, 2, 3, 1)
    x = x.view(batch, h, g, most, width).masked_fill_(~seen[:, None, None], float("-inf"))
    x = (x - x.amax(-1, keepdim=True)).exp_().masked_fill_(~seen[:, None, None], 0.0)
    total = x.sum(-1, keepdim=True)
    v = _values(s["values"], s.get("values_params"), bits, where).permute(0, 2, 1, 3)
    o = (x.view(batch, h, g * most, width) @ v).view(batch, h, g, most, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, most, h * g, d)
    return o[(i < new).expand(batch, most)].to(dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s = _inputs(case, seed)
    new, kv = _lengths(case)
    h, g, d, page, bits = case["heads"], case["group"], case["dim"], case["page"], case["bits"]
    table = s["table"].long()

    def dense(side, b, lo, hi):
        """Tokens lo .. hi of sequence b as the pool holds them, [hi - lo, h, d] in 64 bits."""
        t = torch.arange(lo, hi, device="cuda")
        p, slot = table[b, torch.div(t, page, rounding_mode="floor")], t % page
        x = s[side][p, :, slot]
        if bits == 16:
            return x.double()
        q = s[side + "_params"][p, :, slot].double()
        if bits == 4:
            x = torch.stack((x.remainder(16), torch.div(x, 16, rounding_mode="floor")), -1).reshape(*x.shape[:-1], d)
        return q[..., 1:] + q[..., :1] * x.double()

    if case["op"] == "read":
        return tuple(torch.cat([dense(side, b, kv[b] - new[b], kv[b]) for b in range(len(kv))]) for side in ("keys", "values"))
    if case["op"] == "append":
        out = []
        for side in ("keys", "values"):
            x = s["new_" + side].double()
            if bits < 16:
                low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
                step = (high - low) / (2**bits - 1)
                x = low + step * torch.where(step > 0, torch.round((x - low) / step), torch.zeros_like(x))
            out.append(x)
        return tuple(out)
    out = torch.zeros(s["total"], h * g, d, dtype=torch.float64, device="cuda")
    start = 0
    for b, (n, length) in enumerate(zip(new, kv)):
        keys, values = dense("keys", b, 0, length), dense("values", b, 0, length)
        t = torch.arange(length, device="cuda")
        step = max(1, 2**27 // (g * length))
        for lo in range(0, n, step):
            hi = min(n, lo + step)
            p = torch.arange(length - n + lo, length - n + hi, device="cuda")[:, None]
            hidden = t > p
            if case["window"]:
                hidden |= (t <= p - case["window"]) & (t >= case["sinks"])
            for k in range(h):
                q = s["query"][start + lo:start + hi, k * g:(k + 1) * g].double()
                x = torch.einsum("igd,td->igt", q, keys[:, k]) * s["scale"]
                x.masked_fill_(hidden[:, None], float("-inf"))
                out[start + lo:start + hi, k * g:(k + 1) * g] = torch.softmax(x, -1) @ values[:, k]
        start += n
    return out
