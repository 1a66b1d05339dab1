"""How near the attention over the 4-bit cache comes to its definition in 64 bits, by the size of its error, not by worst-case
sums: those of test_gpu_kv4.py are wider than an output of many slots is large.

What is allowed (`LIMIT`, relative to the root mean square of a row's outputs). A logit's error is absolute in its weight's
exponent: the fp32 sums behind it take at most 2 h / 16 + 32 < 64 steps for 256 channels, each off by 2^-23 (tensor cores may
truncate) of a partial sum of up to about 4 for the inputs below, in random directions once more per slot: 2^-23 * 4 * sqrt(64) /
2 = 2^-19. Exponential, weights as two fp16 numbers (2^-22) and the sums over slots add less than as much again: 2^-18. The
output's error is that, averaged by the weights as the output itself is, so their ratio is the same. The largest of N errors of
one size is below sqrt(2 ln N) < 5.3 sizes (N < 10^6), and slots are unlike: 8 x LIMIT for single elements.
One rounding of a weight or of a query to fp16 is 2^-11 / sqrt(12) or more, 2^-12.8 = 37 x LIMIT; it must not pass."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

LIMIT = 2.0 ** -18


@pytest.fixture(scope="module")
def ops():
    from litert_b200 import ops as o

    return o


@pytest.fixture(scope="module")
def ws(ops):
    return ops.Workspace("cuda")


def values64(nibbles, pairs):
    u = torch.stack((nibbles & 15, nibbles >> 4), -1).flatten(-2).double()
    wide = pairs.double().repeat_interleave(u.shape[-1] // pairs.shape[-2], dim=-2)
    return u * wide[..., 0] + wide[..., 1]


def attention64(q, cache, lengths=None, mask=None, cap=0.0, weigh=None):
    """float64 outputs [b, t, n, h] and weights summed per KV head [b, nkv, s]. weigh(p, values, i): other weights of the
    sequence's values (p [n, s] of one query token), for a restatement with a mistake."""
    b, t, n, h = q.shape
    s, nkv = cache[0].shape[1:3]
    group = n // nkv
    out = torch.zeros((b, t, n, h), dtype=torch.float64, device="cuda")
    got = torch.zeros((b, nkv, s), dtype=torch.float64, device="cuda")
    for i in range(b):
        k, v = (values64(cache[j][i], cache[2 + j][i]).transpose(0, 1) for j in (0, 1))  # [nkv, s, h]
        length = s if lengths is None else max(0, min(s, int(lengths[i])))
        for j in range(t):
            seen = length - (t - 1 - j)
            if seen <= 0:
                continue
            x = torch.einsum("gmh,gsh->gms", q[i, j].double().reshape(nkv, group, h), k[:, :seen]) / math.sqrt(h)
            if cap:
                x = cap * torch.tanh(x / cap)
            shown = torch.ones(seen, dtype=torch.bool, device="cuda")
            if mask is not None:
                m = mask[i, 0, j, :seen].double()
                shown = m > -math.inf
                x = torch.where(shown, x + m, -math.inf)
            if not shown.any():
                continue
            p = torch.softmax(x, -1)
            vv = torch.where(shown[:, None], v[:, :seen], 0.0)
            y = torch.einsum("gms,gsh->gmh", p, vv) if weigh is None else weigh(p, vv, i)
            out[i, j] = y.reshape(n, h)
            got[i, :, :seen] += p.sum(1)
    return out, got


def near(got, want, limit=LIMIT):
    """Whether got [..., h] is want (float64) up to errors of `limit` of a row's size, rounded to got's type; else why not.

    float32: its own rounding is below the limit. fp16: an element is the nearest fp16 number of want unless want lies within
    the error of the border between two; where borders lie is chance, so of N elements about sum(min(1, 2 limit size / step))
    may be others. Four standard deviations more are allowed."""
    size = want.square().mean(-1, keepdim=True).sqrt()
    size = torch.where(size > 0, size, 1.0)
    g = got.double()
    if not torch.isfinite(g).all():
        return "not finite"
    off = (g - want).abs()
    if got.dtype == torch.float32:
        off = off / size
        rms, most = float(off.square().mean().sqrt()), float(off.max())
        return None if rms <= limit and most <= 8 * limit else f"rms {rms:.2e}, largest {most:.2e} of the rows' size"
    step = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -14))) - 10)
    if bool((off > step / 2 + 8 * limit * size).any()):
        return f"an element is off by {float((off - step / 2).div(size).max()):.2e} of its row's size beyond its rounding"
    expected = float((2 * limit * size / step).clamp(max=1).sum())
    other = int((got != want.half()).sum())
    return None if other <= expected + 4 * math.sqrt(expected) + 1 else f"{other} of {got.numel()} are not the nearest, {expected:.0f} expected"


def quantized(x, block):
    y = x.unflatten(-1, (-1, block))
    least = y.amin(-1).half()
    scale = ((y.amax(-1) - least.float()) / 15).half()
    u = ((y - least.float()[..., None]) / scale.float()[..., None]).round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return u[..., 0::2] | (u[..., 1::2] << 4), torch.stack((scale, least), -1)


def filled(ops, seed, b, s, nkv, h, block):
    g = torch.Generator("cuda").manual_seed(seed)
    cache = ops.int4_kv_cache(b, s, nkv, h, block)
    for i in (0, 1):
        nibbles, pairs = quantized(torch.randn((b, s, nkv, h), generator=g, device="cuda"), block)
        cache[i].copy_(nibbles)
        cache[2 + i].copy_(pairs)
    return cache, g


def lengths_of(rng, b, s):
    return torch.from_numpy(rng.integers(max(1, s // 8), s + 1, b).astype(np.int32)).cuda()


#: (sequences, slots, query tokens, (query heads, KV heads, head size, block)): pairs of one CTA, of several, of many pieces;
#: every group size; windows of query tokens
CASES = [(1, 300, 1, (8, 8, 64, 64)), (5, 1000, 1, (8, 1, 256, 64)), (1, 5000, 1, (8, 1, 256, 32)), (3, 2100, 1, (8, 2, 128, 32)),
         (40, 700, 1, (12, 4, 64, 64)), (24, 9000, 1, (4, 1, 256, 64)), (2, 3000, 4, (8, 1, 256, 64)), (4, 1500, 5, (16, 2, 128, 64)),
         (3, 333, 1, (6, 1, 128, 64)), (2, 500, 2, (7, 1, 64, 32)), (2, 600, 1, (9, 3, 96, 32)), (1, 800, 3, (4, 2, 320, 64)),
         (2, 900, 17, (8, 1, 256, 64)), (1, 1300, 64, (8, 2, 128, 64)), (1, 257, 100, (4, 4, 64, 32)), (1, 150, 100, (2, 1, 96, 32))]


@pytest.mark.parametrize("b,s,t,layout", CASES)
@pytest.mark.parametrize("f32", [False, True])
def test_attention_is_as_exact_as_float32_sums(ops, ws, b, s, t, layout, f32):
    n, nkv, h, block = layout
    cache, g = filled(ops, s + t, b, s, nkv, h, block)
    lengths = lengths_of(np.random.default_rng(s), b, s)
    q = 1.2 * torch.randn((b, t, n, h), generator=g, device="cuda")
    q = q if f32 else q.half()
    want, weights = attention64(q, cache, lengths)
    wrong = near(ops.sdpa_decode_int4(q, *cache, lengths=lengths, ws=ws), want)
    assert wrong is None, wrong
    scores = torch.zeros((b, nkv, s), device="cuda")
    got = ops.sdpa_decode_int4(q, *cache, lengths=lengths, scores=scores, ws=ws)
    wrong = near(got, want)
    assert wrong is None, wrong
    # a weight is relative to its logit's error, and to that of the sum that divides it
    off = ((scores.double() - weights) / weights.clamp(min=1e-30))[weights > 0]
    assert float(off.square().mean().sqrt()) <= LIMIT and float(off.abs().max()) <= 8 * LIMIT
    assert not scores[weights == 0].any()


def test_the_measure_sees_one_rounding(ops):
    """Outputs of weights rounded once to fp16 (against a block's scale, as an operand would be), of queries so rounded, and of
    weights of neighbouring slots exchanged are refused; the definition's own are not."""
    b, s, n, nkv, h, block = 2, 1000, 8, 2, 128, 64
    cache, g = filled(ops, 1, b, s, nkv, h, block)
    q = 1.2 * torch.randn((b, 1, n, h), generator=g, device="cuda")
    want, _ = attention64(q, cache)

    def rounded(p, v, i):
        out = torch.zeros((nkv, n // nkv, h), dtype=torch.float64, device="cuda")
        for j in range(h // block):
            a = cache[3][i, :, :, j, 0].double().transpose(0, 1)[:, None]  # [nkv, 1, s]
            least = cache[3][i, :, :, j, 1].double().transpose(0, 1)[:, None]
            at = slice(j * block, (j + 1) * block)
            u = (v[..., at] - least.transpose(1, 2)) / a.transpose(1, 2) - 8
            out[..., at] = torch.einsum("gms,gsh->gmh", (p * a * 1024).half().double() / 1024, u) + ((8 * a + least) * p).sum(-1, keepdim=True)
        return out

    once, _ = attention64(q, cache, weigh=rounded)
    coarse, _ = attention64(q.half(), cache)
    mixed, _ = attention64(q, cache, weigh=lambda p, v, i: torch.einsum("gms,gsh->gmh", p.roll(1, -1), v))
    for dtype in (torch.float32, torch.float16):
        assert near(want.to(dtype), want) is None
        for wrong in (once, coarse, mixed, torch.zeros_like(want)):
            assert near(wrong.to(dtype), want) is not None


HEADS = [(8, 1, 256, 64), (8, 1, 256, 32), (8, 2, 128, 32), (4, 4, 64, 64), (6, 2, 64, 32), (6, 2, 96, 32)]


def dominated(q, cache, slot, above):
    """A slot's keys are those that every query of the first token has a logit of about `above` with."""
    b, t, n, h = q.shape
    nkv = cache[0].shape[2]
    mean = q[:, 0].float().reshape(b, nkv, n // nkv, h).mean(2)
    mean = mean * (above * math.sqrt(h) / mean.square().sum(-1, keepdim=True))
    cache[0][:, slot], cache[2][:, slot] = quantized(mean, h // cache[2].shape[3])


@pytest.mark.parametrize("layout", HEADS)
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("hidden", ["nan", "inf", "large"])
def test_hidden_slots_do_not_coarsen_the_others(ops, ws, layout, f32, hidden):
    """Slots behind -inf masks (a prefix; single ones; NaN, infinities, or the largest scales in them) beside small values and one
    slot of most of the weight: as exact as over a cache that has zeros there. So are slots that a mask of -1e30, the type's lowest
    value, or their own logits leave without weight, where what they hold is finite."""
    n, nkv, h, block = layout
    b, s, t = 4, 3000, 2
    cache, g = filled(ops, h, b, s, nkv, h, block)
    q = torch.randn((b, t, n, h), generator=g, device="cuda")
    q = q if f32 else q.half()
    cache[3].mul_(0.01)
    dominated(q, cache, 1500, 8.0)
    off = torch.zeros((b, s), dtype=torch.bool, device="cuda")
    off[0, :700] = True
    off[1, 5::16] = True
    off[2, 701:1400] = True
    off[3, :1400] = True
    off[3, 1700:] = True
    for i in (2, 3):
        clean = cache[i].clone()
        if hidden == "large":
            cache[i][off] = 65504.0
        else:
            cache[i][off] = float(hidden)
        cache[i][~off] = clean[~off]
    low = torch.finfo(torch.float32).min
    for value in (-math.inf,) if hidden != "large" else (-math.inf, -1e30, low):
        mask = torch.where(off, value, torch.zeros((b, s), device="cuda"))[:, None, None].expand(b, 1, t, s).contiguous()
        plain = [x.clone() for x in cache]
        for x in plain:
            x[off] = 0
        scores = torch.zeros((b, nkv, s), device="cuda")
        got = ops.sdpa_decode_int4(q, *cache, mask=mask, scores=scores, ws=ws)
        want, weights = attention64(q, plain, mask=torch.where(off, -math.inf, 0.0)[:, None, None].expand(b, 1, t, s))
        wrong = near(got, want, 2 * LIMIT)  # (logits up to twice as large as those that LIMIT is for)
        assert wrong is None, (value, wrong)
        off_by = ((scores.double() - weights) / weights.clamp(min=1e-30))[weights > 1e-20]
        assert float(off_by.square().mean().sqrt()) <= 2 * LIMIT


@pytest.mark.parametrize("layout", HEADS)
@pytest.mark.parametrize("f32", [False, True])
def test_slots_of_no_weight_and_later_drafts_do_not_coarsen_the_others(ops, ws, layout, f32):
    """Visible slots with the largest scales and a logit 60 below the others; a last draft's own slot with such scales, which
    earlier queries do not see; a first slot of zeros (scale 0) that has most of the weight."""
    n, nkv, h, block = layout
    b, s, t = 3, 1200, 3
    cache, g = filled(ops, h + 1, b, s, nkv, h, block)
    q = 0.5 * torch.randn((b, 1, n, h), generator=g, device="cuda").expand(b, t, n, h).contiguous()
    q[..., 0] = 6.0
    q = q if f32 else q.half()
    cache[3].mul_(0.01)
    far = torch.zeros((nkv, h), device="cuda")
    far[:, 0] = -10.0 * math.sqrt(h)  # its logit: -60
    for slot in (3, 17, 600, 900):
        cache[0][0, slot], cache[2][0, slot] = quantized(far, block)
        cache[3][0, slot, ..., 0] = 60000.0
    cache[3][1, s - 1, ..., 0] = 60000.0
    near_key = torch.zeros((nkv, h), device="cuda")
    near_key[:, 0] = 2.0 * math.sqrt(h)  # its logit: 12
    cache[0][2, 0], cache[2][2, 0] = quantized(near_key, block)
    cache[1][2, 0], cache[3][2, 0] = 0, 0
    want, _ = attention64(q, cache)
    got = ops.sdpa_decode_int4(q, *cache, ws=ws)
    # the logits' terms are up to 12 here, and what LIMIT counts steps of is 4
    for i, upto in ((0, t), (1, t - 1), (2, t)):
        wrong = near(got[i, :upto], want[i, :upto], 3 * LIMIT)
        assert wrong is None, (i, wrong)


@pytest.mark.parametrize("h,block", [(256, 64), (128, 32), (64, 32), (96, 32)])
@pytest.mark.parametrize("f32", [False, True])
def test_attention_is_exact_over_values_of_any_size(ops, ws, h, block, f32):
    """Value scales growing, shrinking and mixed by 2^18 along the cache, and by 2^9 between blocks: each block of a row by its own
    size."""
    rng = np.random.default_rng(h)
    b, s = 4, 700
    cache, g = filled(ops, h + 2, b, s, 1, h, block)
    size = 2.0 ** np.linspace(-9, 9, s)
    for i, z in enumerate((size, size[::-1], rng.permutation(size))):
        cache[3][i] = (cache[3][i].float() * torch.from_numpy(z.copy()).float().cuda()[:, None, None, None]).half()
    cache[3][3, :, :, 0] *= 2.0 ** -9
    q = torch.randn((b, 1, 8, h), generator=g, device="cuda")
    q = q if f32 else q.half()
    want, _ = attention64(q, cache)
    got = ops.sdpa_decode_int4(q, *cache, ws=ws)
    wrong = near(got.unflatten(-1, (-1, block)), want.unflatten(-1, (-1, block)))
    assert wrong is None, wrong


@pytest.mark.parametrize("n,nkv,h,block", [(8, 1, 256, 64), (4, 1, 256, 32), (8, 2, 128, 32), (8, 4, 64, 64)])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("kind", ["normal", "outlier", "halves"])
def test_sums_over_many_tiles_stay_exact(ops, ws, n, nkv, h, block, f32, kind):
    """A large batch, of which one warp walks through a hundred tiles of 16 slots and more: normal values; one large channel per
    block, beside which all others have small nibbles; a mask that hides the second half of every tile."""
    b, s = 300, 4096
    cache, g = filled(ops, 3, 2, s, nkv, h, block)
    if kind == "outlier":
        v = torch.randn((2, s, nkv, h), generator=g, device="cuda")
        v.unflatten(-1, (-1, block))[..., 3] = 20.0
        cache[1][:], cache[3][:] = quantized(v, block)
    mask = None
    if kind == "halves":
        mask = torch.zeros((2, 1, 1, s), device="cuda")
        mask[..., torch.arange(s, device="cuda") % 16 >= 8] = -math.inf
    q = 0.5 * torch.randn((2, 1, n, h), generator=g, device="cuda")
    q = q if f32 else q.half()
    want, _ = attention64(q, cache, mask=mask)
    many = lambda x: None if x is None else x.repeat(b // 2, *[1] * (x.dim() - 1))  # noqa: E731
    got = ops.sdpa_decode_int4(many(q), *[many(x) for x in cache], mask=many(mask), ws=ws)
    wrong = near(got, many(want))
    assert wrong is None, wrong
