"""The operators of a key/value cache held in 4 bits: storing tokens, reading them back, attention over the cache with
the weights that every cached token has received, and eviction by those weights.

    own                 False: plain forms of the operators; True: the calls that a program makes of litert_b200.ops
    listed()            the cases, by name
    draw(rng)           another one of the same ranges
    prepare(case, seed) what a program holds before the call, on the GPU
    run(state)          one pass, and its outputs
    work(case)          bytes and operations that a pass cannot do without
    exact(case, seed)   the outputs in 64 bits, from the operators' definitions

The cache, per tensor (keys, values): nibbles uint8 [b, s_max, nkv, h / 2], channel 2 i in the low half of byte i, and
float16 pairs (scale, least) [b, s_max, nkv, h / block, 2]; nibble u of a block stands for scale * u + least.

    append  k, v [b, t, nkv, h] -> slots positions[b] .. + counts[b]; then the written slots read back
    attend  q [b, t, n, h] over the first lengths[b] slots, query i of t over all but the last t - 1 - i of them;
            optionally scores[b, kvh, s] += the weights that slot s got from the KV head's queries
    evict   keeps `budget` slots of each KV head: the first `sinks`, the last `recent`, and those of the largest scores;
            in place, or into another cache; then the kept slots read back
"""
import math

import torch

own = False

#: (query heads, KV heads, head size) that decoder models have: one shared KV head, groups of 2 to 8, one each
HEADS = ((8, 1, 256), (4, 1, 256), (8, 1, 128), (8, 2, 128), (16, 2, 128), (8, 4, 64), (8, 8, 64))


def listed():
    return [
        # a decode step's new token of every sequence of a serving batch: a launch and little else
        dict(name="append f16 16 x 1", op="append", b=16, t=1, nkv=1, h=256, block=64, s_max=8192, f32=False, padded=False),
        # a padded batch of prompts in a graph's own float32, finer blocks
        dict(name="append f32 4 x 500 padded", op="append", b=4, t=500, nkv=2, h=128, block=32, s_max=2000, f32=True,
             padded=True),
        # whole prompts of a serving batch behind their prompt pass
        dict(name="append f16 16 x 8192", op="append", b=16, t=8192, nkv=1, h=256, block=64, s_max=8192, f32=False,
             padded=False),
        # an interactive request at its start: latency
        dict(name="attend f16 1 x 300", op="attend", b=1, t=1, n=8, nkv=8, h=64, block=64, s_max=300, f32=False, cap=0.0,
             mask=False, scores=False),
        # a serving batch of long, ragged sequences
        dict(name="attend f16 16 x 8192", op="attend", b=16, t=1, n=8, nkv=1, h=256, block=64, s_max=8192, f32=False,
             cap=0.0, mask=False, scores=False),
        # the composite as a graph holds it: float32 tensors, an additive mask over the whole cache, a logit cap
        dict(name="attend f32 mask 4 x 2000", op="attend", b=4, t=1, n=8, nkv=2, h=128, block=32, s_max=2000, f32=True,
             cap=50.0, mask=True, scores=False),
        # a serving batch whose cache will be evicted from: the weights are accumulated
        dict(name="attend f16 scores 16 x 8192", op="attend", b=16, t=1, n=16, nkv=2, h=128, block=64, s_max=8192, f32=False,
             cap=0.0, mask=False, scores=True),
        # four drafted tokens per sequence, checked in one pass
        dict(name="attend f16 drafts 8 x 4096", op="attend", b=8, t=4, n=8, nkv=1, h=256, block=64, s_max=4096, f32=False,
             cap=0.0, mask=False, scores=True),
        # the largest batch and the longest contexts
        dict(name="attend f16 64 x 32768", op="attend", b=64, t=1, n=8, nkv=1, h=256, block=64, s_max=32768, f32=False,
             cap=0.0, mask=False, scores=False),
        # a small cache, evicted to less than half
        dict(name="evict 4 x 600 to 256", op="evict", b=4, nkv=2, h=128, block=32, s_max=600, budget=256, sinks=4, recent=32,
             into=False),
        # a serving batch that has grown 256 tokens past its budget
        dict(name="evict 16 x 4352 to 4096", op="evict", b=16, nkv=1, h=256, block=64, s_max=4352, budget=4096, sinks=4,
             recent=256, into=False),
        # long prompts squeezed into the small cache that their replies are generated with
        dict(name="evict 8 x 32768 to 2048", op="evict", b=8, nkv=4, h=64, block=64, s_max=32768, budget=2048, sinks=4,
             recent=512, into=True),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "attend", "evict"))
    n, nkv, h = rng.choice(HEADS)
    block = rng.choice((32, 64))
    if op == "append":
        t = _log(rng, 1, 8192)
        b = _log(rng, 1, max(1, min(64, 16 * 8192 * 256 // (t * nkv * h * 2))))
        return dict(op=op, b=b, t=t, nkv=nkv, h=h, block=block, s_max=t + _log(rng, 1, 512), f32=rng.random() < 0.4,
                    padded=rng.random() < 0.5)
    if op == "attend":
        s_max = _log(rng, 16, 32768)
        b = _log(rng, 1, max(1, min(64, 16 * 32768 * 256 // (s_max * nkv * h))))
        f32 = rng.random() < 0.3
        return dict(op=op, b=b, t=rng.choice((1, 1, 1, 2, 4, 5)), n=n, nkv=nkv, h=h, block=block, s_max=s_max, f32=f32,
                    cap=rng.choice((0.0, 0.0, 50.0)), mask=f32 and rng.random() < 0.5, scores=rng.random() < 0.4)
    s_max = _log(rng, 64, 32768)
    budget = _log(rng, 16, s_max)
    b = _log(rng, 1, max(1, min(32, 4 * 8192 * 256 // (budget * nkv * h), 8 * 32768 * 256 // (s_max * nkv * h))))
    sinks = min(rng.choice((0, 1, 4)), budget)
    return dict(op=op, b=b, nkv=nkv, h=h, block=block, s_max=s_max, budget=budget, sinks=sinks,
                recent=rng.randint(0, (budget - sinks) // 2), into=rng.random() < 0.3)


# ---- inputs ----------------------------------------------------------------------------------------------


def _rng(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _rows(g, channels, b, t):
    """Keys or values: normal, some channels larger than others, as projections have them."""
    return _normal(g, b, t, *channels.shape) * channels


def _filled(g, c, s_max):
    """The four tensors of a cache whose slots all hold tokens."""
    b, nkv, h, block = c["b"], c["nkv"], c["h"], c["block"]
    cache = _empty(c, s_max)
    for at in (0, 1):
        channels = torch.exp(0.5 * _normal(g, nkv, h)) if at == 0 else torch.ones((nkv, h), device="cuda")
        for i in range(b):  # one sequence at a time: the work is in 64 bits
            cache[at][i], cache[2 + at][i] = _quantize(_rows(g, channels, 1, s_max)[0], block)
    return cache


def _empty(c, s_max):
    b, nkv, h, block = c["b"], c["nkv"], c["h"], c["block"]
    nibbles = [torch.zeros((b, s_max, nkv, h // 2), dtype=torch.uint8, device="cuda") for _ in range(2)]
    return nibbles + [torch.zeros((b, s_max, nkv, h // block, 2), dtype=torch.float16, device="cuda") for _ in range(2)]


def _integers(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=g, device="cuda").to(torch.int32)


def prepare(case, seed):
    g = _rng(seed)
    c = dict(case)
    st = {"case": c}
    b, nkv, h, s_max = c["b"], c["nkv"], c["h"], c["s_max"]
    if c["op"] == "append":
        t = c["t"]
        channels = torch.exp(0.5 * _normal(g, nkv, h))
        dtype = torch.float32 if c["f32"] else torch.float16
        st["k"], st["v"] = _rows(g, channels, b, t).to(dtype), _normal(g, b, t, nkv, h).to(dtype)
        st["cache"] = _empty(c, s_max)
        st["positions"] = _integers(g, 0, s_max - t, b)
        st["counts"] = _integers(g, (t + 1) // 2, t, b) if c["padded"] else None
        return st
    st["cache"] = _filled(g, c, s_max)
    if c["op"] == "attend":
        t, n = c["t"], c["n"]
        lengths = _integers(g, max(1, s_max // 64), s_max, b)
        q = 1.2 * _normal(g, b, t, n, h)
        st["q"] = q if c["f32"] else q.half()
        st["args"] = dict(scale=1.0 / math.sqrt(h), logit_cap=c["cap"], lengths=None, mask=None)
        if c["mask"]:
            # a graph's decode step: the cache's unwritten slots are masked out, no lengths
            limit = lengths[:, None] - torch.arange(t - 1, -1, -1, device="cuda")[None, :]
            past = torch.arange(s_max, device="cuda") >= limit[:, :, None]
            st["args"]["mask"] = torch.where(past, -1e30, 0.0).float()[:, None].contiguous()
        else:
            st["args"]["lengths"] = lengths
        st["scores"] = torch.exp(_normal(g, b, nkv, s_max)) if c["scores"] else None
        return st
    # sums of weights: most are small, some tokens have drawn none at all
    st["scores"] = torch.exp(2.0 * _normal(g, b, nkv, s_max))
    st["scores"][torch.rand((b, nkv, s_max), generator=g, device="cuda") < 0.1] = 0.0
    st["lengths"] = _integers(g, min(c["budget"] + 1, s_max), s_max, b)
    st["into"] = _empty(c, c["budget"]) if c["into"] else None
    return st


# ---- the plain forms -------------------------------------------------------------------------------------


def _quantize(x, block):
    """x [..., h] -> nibbles uint8 [..., h / 2] and (scale, least) float16 [..., h / block, 2]. The scale is the
    fifteenth of the range, difference and quotient rounded to float32 (the quotient by way of 64 bits: a division by a
    constant is a product in 32); which of the sixteen values an element is nearest to is decided in 64 bits."""
    x = x.unflatten(-1, (-1, block)).float()
    least = x.amin(-1).clamp(-65504, 65504).half()
    scale = ((x.amax(-1) - least.float()).double() / 15).float().clamp(0, 65504).half()
    s, m = scale.double()[..., None], least.double()[..., None]
    u = torch.where(s > 0, (x.double() - m) / torch.where(s > 0, s, 1.0), 0.0).round().clamp(0, 15).to(torch.uint8)
    u = u.flatten(-2)
    return u[..., 0::2] | (u[..., 1::2] << 4), torch.stack((scale, least), -1)


def _values(nibbles, scale):
    """float32 [..., h] that the nibbles stand for."""
    u = torch.stack((nibbles & 15, nibbles >> 4), -1).flatten(-2).float()
    block = u.shape[-1] // scale.shape[-2]
    s = scale.float()
    return (u.unflatten(-1, (-1, block)) * s[..., :1] + s[..., 1:]).flatten(-2)


def _read(cache, slots, valid, dtype):
    """Slots [b, t] of the keys and the values, zeros where they are not valid."""
    b = torch.arange(slots.shape[0], device="cuda")[:, None]
    slots = slots.clamp(0, cache[0].shape[1] - 1)
    return [torch.where(valid[..., None, None], _values(cache[i][b, slots], cache[2 + i][b, slots]), 0.0).to(dtype)
            for i in (0, 1)]


def _append(st):
    c, cache = st["case"], st["cache"]
    t, s_max = c["t"], c["s_max"]
    i = torch.arange(t, device="cuda")[None, :]
    slots = st["positions"].long()[:, None] + i
    limit = t if st["counts"] is None else st["counts"][:, None]
    valid = (i < limit) & (slots < s_max)
    rows = torch.nonzero(valid, as_tuple=True)
    at = (rows[0], slots[rows])
    for j, x in enumerate((st["k"], st["v"])):
        cache[j][at], cache[2 + j][at] = _quantize(x[rows], c["block"])
    return _read(cache, slots, valid, st["k"].dtype)


def _weights(st, k):
    """Softmax weights [b, nkv, t, group, s_max] of the keys k [b, s_max, nkv, h]."""
    c, a = st["case"], st["args"]
    b, t, n, nkv, h, s_max = (c[x] for x in ("b", "t", "n", "nkv", "h", "s_max"))
    q = st["q"].float().reshape(b, t, nkv, n // nkv, h).permute(0, 2, 1, 3, 4).reshape(b, nkv, t * (n // nkv), h)
    x = (torch.matmul(q, k.permute(0, 2, 3, 1)) * a["scale"]).reshape(b, nkv, t, n // nkv, s_max)
    if a["logit_cap"]:
        x = a["logit_cap"] * torch.tanh(x / a["logit_cap"])
    if a["mask"] is not None:
        x = x + a["mask"][:, :, :, None, :]
    lengths = a["lengths"] if a["lengths"] is not None else torch.full((b,), s_max, device="cuda")
    limit = lengths[:, None] - torch.arange(t - 1, -1, -1, device="cuda")[None, :]
    x = torch.where((torch.arange(s_max, device="cuda") < limit[..., None])[:, None, :, None, :], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, p / total, 0.0)


def _attend(st):
    c, cache = st["case"], st["cache"]
    b, t, n, nkv, h, s_max = (c[x] for x in ("b", "t", "n", "nkv", "h", "s_max"))
    w = _weights(st, _values(cache[0], cache[2]))
    v = _values(cache[1], cache[3])
    out = torch.matmul(w.reshape(b, nkv, t * (n // nkv), s_max), v.permute(0, 2, 1, 3))
    out = out.reshape(b, nkv, t, n // nkv, h).permute(0, 2, 1, 3, 4).reshape(b, t, n, h).to(st["q"].dtype)
    if st["scores"] is None:
        return out
    st["scores"] += w.sum((2, 3))
    return out, st["scores"]


def _evict(st):
    c, cache = st["case"], st["cache"]
    budget, s_max = c["budget"], c["s_max"]
    slot = torch.arange(s_max, device="cuda")
    length = st["lengths"].long()[:, None, None]
    key = torch.where((slot < c["sinks"]) | (slot >= length - c["recent"]), math.inf, st["scores"])
    key = torch.where(slot < length, key, -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    left = length.clamp(max=budget)
    j = torch.arange(budget, device="cuda")
    order = torch.where(j < left, order, s_max).sort(-1).values  # kept slots in their order, then nothing
    order = torch.where(length <= budget, torch.where(j < length, j, s_max), order)
    kept = torch.where(order < s_max, order, -1).to(torch.int32)
    at = order.clamp(max=s_max - 1)
    to = cache if st["into"] is None else st["into"]
    rows = torch.arange(c["b"], device="cuda")[:, None, None]
    heads = torch.arange(c["nkv"], device="cuda")[None, :, None]
    there = (kept >= 0).transpose(1, 2)
    for i in range(4):
        moved = cache[i][rows, at, heads].transpose(1, 2)
        to[i][:, :budget] = torch.where(there.reshape(there.shape + (1,) * (moved.dim() - 3)), moved, to[i][:, :budget])
    scores = torch.zeros((c["b"], c["nkv"], to[0].shape[1]), device="cuda")
    scores[..., :budget] = torch.where(kept >= 0, torch.gather(st["scores"], -1, at), 0.0)
    lengths = st["lengths"].clamp(max=budget)
    valid = j[None, :] < lengths[:, None]
    return [kept, scores, lengths] + _read(to, j.expand(c["b"], -1), valid, torch.float16)


# ---- the framework's calls -------------------------------------------------------------------------------


def _own(st):
    from litert_b200 import ops

    c, cache = st["case"], st["cache"]
    if "ws" not in st:
        st["ws"] = ops.Workspace("cuda")  # a program makes it once
    if c["op"] == "append":
        ops.kv_append_int4(st["k"], st["v"], st["positions"], *cache, counts=st["counts"])
        return ops.kv_read_int4(*cache, tokens=c["t"], positions=st["positions"], counts=st["counts"], dtype=st["k"].dtype)
    if c["op"] == "attend":
        out = ops.sdpa_decode_int4(st["q"], *cache, scores=st["scores"], ws=st["ws"], **st["args"])
        return out if st["scores"] is None else (out, st["scores"])
    kept, scores, lengths = ops.kv_evict_int4(*cache, st["scores"], st["lengths"], c["budget"], sinks=c["sinks"],
                                              recent=c["recent"], into=st["into"])
    to = cache if st["into"] is None else st["into"]
    return [kept, scores, lengths] + list(ops.kv_read_int4(*to, tokens=c["budget"], counts=lengths, dtype=torch.float16))


def run(st):
    if own:
        return _own(st)
    return {"append": _append, "attend": _attend, "evict": _evict}[st["case"]["op"]](st)


# ---- floors ----------------------------------------------------------------------------------------------


def work(case):
    c = dict(case)
    b, nkv, h, s_max = c["b"], c["nkv"], c["h"], c["s_max"]
    row = 2 * nkv * (h // 2 + 4 * (h // c["block"]))  # a token's keys and values in the cache
    if c["op"] == "append":
        tokens = b * c["t"] * (0.75 if c["padded"] else 1.0)
        elem = 4 if c["f32"] else 2
        # rows in, nibbles and pairs out, and the values read back
        return {"bytes": tokens * (2 * nkv * h * elem + row) + 2 * b * c["t"] * nkv * h * elem,
                "flops": 10 * tokens * nkv * h}
    if c["op"] == "attend":
        # lengths are uniform over the cache: half of it is read on average; a masked cache is read whole
        tokens = b * s_max if c["mask"] else b * (s_max + max(1, s_max // 64)) // 2
        qo = 2 * b * c["t"] * c["n"] * h * (4 if c["f32"] else 2)
        return {"bytes": tokens * row + qo + (4 * b * c["t"] * s_max if c["mask"] else 0) + (8 * tokens * nkv if c["scores"] else 0),
                "flops": 4 * tokens * c["t"] * c["n"] * h}
    budget = c["budget"]
    seen = b * nkv * (s_max + min(budget + 1, s_max)) // 2
    kept = b * budget
    # the scores in and out, the kept rows in and out, their slots, and the values read back
    s_out = budget if c["into"] else s_max
    return {"bytes": 4 * seen + 4 * b * nkv * s_out + 2 * kept * row + 4 * kept * nkv + 4 * kept * nkv * h, "flops": 4 * seen}


# ---- in 64 bits, from the definitions --------------------------------------------------------------------


def _exact_block_values(x, block):
    """What x [..., h] reads back as: blocks of sixteen equally spaced values."""
    y = x.double().reshape(*x.shape[:-1], -1, block)
    low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
    low = low.to(torch.float16).double()
    spread = (high - low).to(torch.float32).double()  # the definition rounds the range and its fifteenth to float32
    step = (spread / 15.0).to(torch.float32).to(torch.float16).double()
    n = torch.zeros_like(y)
    ok = (step > 0).expand_as(y)
    n[ok] = torch.clamp(torch.round(((y - low) / step.clamp(min=1e-300))[ok]), 0.0, 15.0)
    return (low + step * n).reshape(x.shape)


def _exact_cache(nibbles, pairs):
    h = 2 * nibbles.shape[-1]
    out = torch.empty(nibbles.shape[:-1] + (h,), dtype=torch.float64, device=nibbles.device)
    out[..., 0::2] = (nibbles % 16).double()
    out[..., 1::2] = torch.div(nibbles, 16, rounding_mode="floor").double()
    block = h // pairs.shape[-2]
    wide = pairs.double().repeat_interleave(block, dim=-2)
    return out * wide[..., 0] + wide[..., 1]


def _exact_attention(st, c, i):
    """Sequence i: outputs [t, n, h] and the slots' weights [nkv, s_max]."""
    t, n, nkv, s_max = c["t"], c["n"], c["nkv"], c["s_max"]
    a, group = st["args"], n // nkv
    k, v = (_exact_cache(st["cache"][j][i], st["cache"][2 + j][i]) for j in (0, 1))
    q = st["q"][i].double()
    out = torch.zeros_like(q)
    got = torch.zeros((nkv, s_max), dtype=torch.float64, device=q.device)
    length = s_max if a["lengths"] is None else int(a["lengths"][i])
    for j in range(t):
        seen = min(s_max, length - (t - 1 - j))
        if seen <= 0:
            continue
        for head in range(n):
            kvh = head // group
            x = torch.mv(k[:seen, kvh], q[j, head]) * a["scale"]
            if a["logit_cap"]:
                x = torch.tanh(x / a["logit_cap"]) * a["logit_cap"]
            if a["mask"] is not None:
                x = x + a["mask"][i, 0, j, :seen].double()
            w = torch.softmax(x, 0)
            out[j, head] = torch.mv(v[:seen, kvh].T, w)
            got[kvh, :seen] += w
    return out, got


def exact(case, seed):
    c = dict(case)
    st = prepare(case, seed)
    b, nkv, h = c["b"], c["nkv"], c["h"]
    if c["op"] == "append":
        outs = []
        for x in (st["k"], st["v"]):
            y = _exact_block_values(x, c["block"])
            if st["counts"] is not None:
                for i, n in enumerate(st["counts"].tolist()):
                    y[i, n:] = 0.0
            outs.append(y)
        return outs
    if c["op"] == "attend":
        outs, sums = [], []
        for i in range(b):
            out, got = _exact_attention(st, c, i)
            outs.append(out)
            sums.append(got)
        if st["scores"] is None:
            return torch.stack(outs)
        return torch.stack(outs), st["scores"].double() + torch.stack(sums)
    budget, s_out = c["budget"], c["budget"] if c["into"] else c["s_max"]
    scores = torch.zeros((b, nkv, s_out), dtype=torch.float64, device="cuda")
    values = [torch.zeros((b, budget, nkv, h), dtype=torch.float64, device="cuda") for _ in (0, 1)]
    for i, length in enumerate(st["lengths"].tolist()):
        for kvh in range(nkv):
            x = st["scores"][i, kvh, :length].double().cpu().tolist()
            ranked = sorted(range(length), key=lambda s: (not (s < c["sinks"] or s >= length - c["recent"]), -x[s], s))
            kept = torch.tensor(sorted(ranked[:budget]), device="cuda")
            scores[i, kvh, :len(kept)] = st["scores"][i, kvh, kept].double()
            for j in (0, 1):
                values[j][i, :len(kept), kvh] = _exact_cache(st["cache"][j][i, kept, kvh], st["cache"][2 + j][i, kept, kvh])
    return [None, scores, None] + values
