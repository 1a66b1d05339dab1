"""The key/value cache in 4 bits against plain float64 restatements: storing, reading, attention, eviction, and a run of
them as a server strings them together."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

EPS32 = 2.0 ** -24  # half a step of float32, relative
EPS16 = 2.0 ** -11


@pytest.fixture(scope="module")
def ops():
    from litert_b200 import ops as o

    return o


@pytest.fixture(scope="module")
def ws(ops):
    return ops.Workspace("cuda")


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---- definitions -----------------------------------------------------------------------------------------
def quantize(x, block):
    """[..., h] -> (u [..., h], scale, least fp16 [..., h / block])."""
    y = x.reshape(*x.shape[:-1], -1, block)
    f = y.astype(np.float32)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        least = np.clip(f.min(-1), -65504, 65504).astype(np.float16)
        spread = f.max(-1) - least.astype(np.float32)
        scale = np.clip(spread / np.float32(15), 0, 65504).astype(np.float16)
        s, m = scale.astype(np.float64)[..., None], least.astype(np.float64)[..., None]
        u = np.where(s > 0, np.clip(np.rint((f.astype(np.float64) - m) / np.where(s > 0, s, 1.0)), 0, 15), 0)
    bad = ~np.isfinite(f).all(-1)
    scale[bad] = least[bad] = np.nan
    u[bad] = 0
    return u.reshape(x.shape).astype(np.uint8), scale, least


def pack(u):
    return u[..., 0::2] | (u[..., 1::2] << 4)


def values(cache, i):
    """float64 [b, s, nkv, h] of the keys (0) or values (1), and the same with every term's magnitude."""
    nib, pairs = cache[i].cpu().numpy(), cache[2 + i].cpu().numpy().astype(np.float64)
    u = np.stack((nib & 15, nib >> 4), -1).reshape(*nib.shape[:-1], -1).astype(np.float64)
    wide = np.repeat(pairs, u.shape[-1] // pairs.shape[-2], axis=-2)
    return u * wide[..., 0] + wide[..., 1], u * np.abs(wide[..., 0]) + np.abs(wide[..., 1])


def attention(q, k, v, k_mag, v_mag, limits, scale, cap, mask, v_half=None):
    """One sequence in float64: q [t, n, h], k / v [s, nkv, h]. Returns outputs, weights per KV head [nkv, s], and bounds
    of what float32 sums may be off by in either.

    A logit is a sum of at most 2 h + 32 rounded terms (products of a nibble and a query element are exact, one of the two
    fp32 halves of a query, the blocks' scales and least values), each step off by 2^-23 of the sum of the terms'
    magnitudes (tensor cores may truncate); the cap's tanh and division add four steps of the cap's value, scaling and
    mask four of the logit's. A weight is off by twice its logit's error (numerator and maximum's share) and by eight steps
    of (1 + |x - top| log2 e): exponent, exponential, division. Sums over s slots add s + 64 steps of the magnitudes; the
    weights' split into two fp16 numbers 2^-21. For fp16 queries a weight times its value
    scale a is one fp16 number, off by half a step, which counts (u - 8) times: v_half = 8 |a| bounds |u - 8| |a|."""
    t, n, h = q.shape
    s, nkv = k.shape[:2]
    step = 2 * EPS32
    out, weights = np.zeros((t, n, h)), np.zeros((nkv, s))
    out_off, weights_off = np.zeros((t, n, h)), np.zeros((nkv, s))
    for i in range(t):
        if limits[i] <= 0:
            continue
        for head in range(n):
            j = head // (n // nkv)
            x = k[:limits[i], j] @ q[i, head] * scale
            off = (2 * h + 32) * step * (k_mag[:limits[i], j] @ np.abs(q[i, head])) * scale
            if cap:
                x = cap * np.tanh(x / cap)
                off = off + 4 * step * np.abs(x)
            if mask is not None:
                m = mask[i, :limits[i]]
                x = np.where(np.isneginf(m), -np.inf, x + m)
            keep = ~np.isneginf(x)
            if not keep.any():
                continue
            top = x.max()
            x = np.where(keep, x, 0.0)
            off = off + 4 * step * np.abs(np.where(np.abs(x) < 1e20, x, 0.0))
            p = np.where(keep, np.exp(x - top), 0.0)
            w = p / p.sum()
            live = w > 1e-30
            rel = 2 * off[live].max() + 8 * step * (1 + 1.5 * (top - x[live]).max()) + (s + 64) * step
            vv = np.where(keep[:, None], v[:limits[i], j], 0.0)
            mag = np.where(keep[:, None], v_mag[:limits[i], j], 0.0)
            out[i, head] = w @ vv
            out_off[i, head] = (rel + (s + 64) * step + 2.0 ** -21) * (w @ mag)
            if v_half is not None:
                out_off[i, head] += EPS16 * (w @ np.where(keep[:, None], v_half[:limits[i], j], 0.0))
            weights[j, :limits[i]] += w
            weights_off[j, :limits[i]] += w * rel + 1e-30
    return out, weights, out_off, weights_off


def limits_of(length, s, t):
    length = min(max(int(length), 0), s)
    return [max(0, length - (t - 1 - i)) for i in range(t)]


def check_attention(ops, ws, q, cache, lengths=None, mask=None, scale=None, cap=0.0, with_scores=False):
    b, t, n, h = q.shape
    s, nkv = cache[0].shape[1:3]
    scores = torch.rand((b, nkv, s), device="cuda", generator=torch.Generator("cuda").manual_seed(5)) if with_scores else None
    before = scores.cpu().numpy() if with_scores else None
    got = ops.sdpa_decode_int4(q, *cache, lengths=None if lengths is None else dev(np.asarray(lengths, np.int32)),
                               mask=None if mask is None else dev(mask), scale=scale, logit_cap=cap, scores=scores, ws=ws)
    assert got.dtype == q.dtype and got.shape == q.shape
    got = got.cpu().numpy().astype(np.float64)
    (k, km), (v, vm) = values(cache, 0), values(cache, 1)
    half = 8 * np.repeat(np.abs(cache[3][..., 0].cpu().numpy().astype(np.float64)), h // cache[3].shape[3], axis=-1)
    qf = q.cpu().numpy().astype(np.float64)
    for i in range(b):
        lim = limits_of(s if lengths is None else lengths[i], s, t)
        with np.errstate(invalid="ignore"):
            want, w, off, w_off = attention(qf[i], k[i], v[i], km[i], vm[i], lim, scale or 1 / math.sqrt(h), cap,
                                            None if mask is None else mask[i, 0].astype(np.float64), half[i] if q.dtype == torch.float16 else None)
        bound = off + (EPS16 * np.abs(want) + 2.0 ** -25 if q.dtype == torch.float16 else EPS32 * np.abs(want))
        assert np.isfinite(got[i]).all(), i
        assert (np.abs(got[i] - want) <= bound).all(), (i, lim, np.max(np.abs(got[i] - want) - bound), np.max(np.abs(got[i] - want)))
        if with_scores:
            after = scores[i].cpu().numpy()
            assert (np.abs(after - (before[i] + w)) <= w_off + 2 * EPS32 * (before[i] + w)).all(), i
            assert np.array_equal(after[:, max(lim):], before[i][:, max(lim):])
    return got


def filled(ops, rng, b, s, nkv, h, block):
    """A cache whose slots all hold tokens, made without the package's kernels."""
    cache = ops.int4_kv_cache(b, s, nkv, h, block)
    for i in (0, 1):
        x = rng.standard_normal((b, s, nkv, h)) * np.exp(0.5 * rng.standard_normal((nkv, h)))
        u, scale, least = quantize(x.astype(np.float32), block)
        cache[i].copy_(torch.from_numpy(pack(u)))
        cache[2 + i].copy_(torch.from_numpy(np.stack((scale, least), -1)))
    return cache


def fill_nan(cache, where):
    """Pairs of the slots under the index `where` become NaN, their nibbles 15."""
    for i in (0, 1):
        cache[i][where] = 255
        cache[2 + i][where] = float("nan")


# ---- storing and reading ---------------------------------------------------------------------------------
SHAPES = [(64, 64), (64, 32), (96, 32), (128, 64), (128, 32), (256, 64), (256, 32), (512, 64), (32, 32), (320, 64)]


@pytest.mark.parametrize("h,block", SHAPES)
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_append_is_exact_and_touches_nothing_else(ops, h, block, dtype):
    rng = np.random.default_rng(h + block)
    b, t, nkv, s = 5, 7, 3, 20
    cache = ops.int4_kv_cache(b, s, nkv, h, block)
    for i in range(4):
        cache[i].view(torch.uint8).fill_(0xA5)
    before = [x.cpu().numpy().copy() for x in cache]
    rows = [(rng.standard_normal((b, t, nkv, h)) * 3).astype(dtype) for _ in (0, 1)]
    positions = np.asarray([0, 13, 17, -3, 100], np.int32)  # inside, to the end, past the end, before the start, outside
    counts = np.asarray([7, 3, 7, 7, 7], np.int32)
    ops.kv_append_int4(dev(rows[0]), dev(rows[1]), dev(positions), *cache, counts=dev(counts))
    for j in (0, 1):
        u, scale, least = quantize(rows[j], block)
        nib, pairs = before[j], before[2 + j]
        for i in range(b):
            for x in range(counts[i]):
                if 0 <= positions[i] + x < s:
                    nib[i, positions[i] + x] = pack(u[i, x])
                    pairs[i, positions[i] + x] = np.stack((scale[i, x], least[i, x]), -1)
        assert np.array_equal(cache[j].cpu().numpy(), nib)
        assert np.array_equal(cache[2 + j].cpu().numpy().view(np.uint16), pairs.view(np.uint16))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_read_gives_the_values_rounded_once(ops, dtype):
    rng = np.random.default_rng(3)
    cache = filled(ops, rng, 4, 33, 2, 96, 32)
    positions, counts = np.asarray([0, 30, -2, 40], np.int32), np.asarray([9, 5, 8, 9], np.int32)
    got = ops.kv_read_int4(*cache, tokens=9, positions=dev(positions), counts=dev(counts), dtype=dtype)
    for j in (0, 1):
        whole = values(cache, j)[0]
        want = np.zeros((4, 9, 2, 96))
        for i in range(4):
            for x in range(counts[i]):
                if 0 <= positions[i] + x < 33:
                    want[i, x] = whole[i, positions[i] + x]
        assert np.array_equal(got[j].cpu().numpy(), want.astype(np.float32).astype(got[j].cpu().numpy().dtype))
    k, v = ops.kv_read_int4(*cache, dtype=dtype)
    assert k.shape == (4, 33, 2, 96)
    assert np.array_equal(v.cpu().numpy(), values(cache, 1)[0].astype(np.float32).astype(v.cpu().numpy().dtype))


def test_append_reads_slices_of_a_fused_projection(ops):
    """Keys and values as views of one [b, t, (n + 2 nkv) h] tensor; views that start on odd elements; a broadcast token."""
    rng = np.random.default_rng(4)
    b, t, n, nkv, h = 2, 5, 4, 2, 64
    for pad in (0, 1):
        whole = torch.from_numpy(rng.standard_normal((b, t, pad + (n + 2 * nkv) * h)).astype(np.float16)).cuda()
        k = whole[..., pad + n * h:pad + (n + nkv) * h].view(b, t, nkv, h) if pad == 0 else \
            whole[..., pad + n * h:pad + (n + nkv) * h].unflatten(-1, (nkv, h))
        v = whole[..., pad + (n + nkv) * h:].unflatten(-1, (nkv, h))
        cache, want = ops.int4_kv_cache(b, 8, nkv, h), ops.int4_kv_cache(b, 8, nkv, h)
        at = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
        ops.kv_append_int4(k, v, at, *cache)
        ops.kv_append_int4(k.clone(), v.clone(), at, *want)
        assert all(torch.equal(x, y) for x, y in zip(cache, want)) and cache[0].any()
    one = k[:, :1].expand(b, 4, nkv, h)
    ops.kv_append_int4(one, one.transpose(2, 3).contiguous().transpose(2, 3), at, *cache)  # (heads and channels swapped)
    ops.kv_append_int4(one.contiguous(), one.contiguous(), at, *want)
    assert all(torch.equal(x, y) for x, y in zip(cache, want))


def test_append_at_the_borders_between_nibbles(ops):
    """Elements at, and a float32 step next to, every border; constant blocks; blocks of one huge and many tiny elements;
    subnormals; ranges beyond fp16; infinities and NaN."""
    rng = np.random.default_rng(5)
    rows = []
    for scale, least in ((0.25, -1.5), (0.3330078125, 0.10003662109375), (2.0 ** -14, 0.0), (1e-3, 5.0)):
        s, m = np.float64(np.float16(scale)), np.float64(np.float16(least))
        edge = (m + s * (np.arange(15) + 0.5)).astype(np.float32)
        x = np.full(64, np.float32(m), np.float32)
        x[1] = np.float32(m + 15 * s)
        x[2:17], x[17:32], x[32:47] = edge, np.nextafter(edge, np.float32(np.inf)), np.nextafter(edge, np.float32(-np.inf))
        rows.append(x)
    rows += [np.full(64, v, np.float32) for v in (0.0, -0.0, 1.0, 0.1, -7e4, 3e38)]
    rows.append(np.r_[np.float32(1e5), np.full(63, 1e-6, np.float32)])
    rows.append(np.r_[np.float32(-3e38), np.float32(3e38), np.zeros(62, np.float32)])
    rows.append((rng.standard_normal(64) * 1e-7).astype(np.float32))
    rows.append((rng.standard_normal(64) * 1e-40).astype(np.float32))
    for v in (np.inf, -np.inf, np.nan):
        x = rng.standard_normal(64).astype(np.float32)
        x[rng.integers(64)] = v
        rows.append(x)
    for base in rng.standard_normal(40):
        rows.append((base + rng.standard_normal(64) * 10.0 ** rng.uniform(-3, 3)).astype(np.float32))
    x = np.stack(rows)[None, :, None, :]
    cache = ops.int4_kv_cache(1, len(rows), 1, 64)
    ops.kv_append_int4(dev(x), dev(x[:, ::-1]), torch.zeros(1, dtype=torch.int32, device="cuda"), *cache)
    for j, y in ((0, x), (1, x[:, ::-1])):
        u, scale, least = quantize(y, 64)
        got = cache[2 + j].cpu().numpy()
        nan = np.isnan(scale)
        assert nan.sum() == 3 and np.isnan(got[..., 0][nan]).all() and np.isnan(got[..., 1][nan]).all()
        assert np.array_equal(got[..., 0][~nan], scale[~nan]) and np.array_equal(got[..., 1][~nan], least[~nan])
        assert np.array_equal(cache[j].cpu().numpy(), pack(u))
    k, _ = ops.kv_read_int4(*cache, dtype=torch.float32)
    assert np.isnan(k.cpu().numpy()[0, :, 0]).all(-1).sum() == 3


# ---- attention -------------------------------------------------------------------------------------------
#: (query heads, KV heads, head size, block): the tensor-core shapes in every grouping, and others
LAYOUTS = [(8, 1, 256, 64), (8, 1, 256, 32), (8, 2, 128, 64), (12, 4, 128, 32), (8, 8, 64, 64), (5, 1, 64, 32), (16, 1, 128, 64),
           (20, 2, 64, 64), (6, 2, 96, 32), (3, 1, 32, 32), (2, 1, 512, 64), (4, 2, 320, 64)]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("t", [1, 3])
def test_attention_over_ragged_lengths(ops, ws, layout, f32, t):
    """Lengths on and next to tiles (16 slots), none, one, the cache's last slot, negative and beyond; NaN behind every
    length."""
    n, nkv, h, block = layout
    rng = np.random.default_rng(n * 1000 + h + t)
    lengths = [0, 1, 2, 15, 16, 17, 31, 64, 129, 300, 301, -5, 400]
    b, s = len(lengths), 301
    cache = filled(ops, rng, b, s, nkv, h, block)
    for i, length in enumerate(lengths):
        if length < s:
            fill_nan([x[i] for x in cache], slice(max(0, length), None))
    q = torch.from_numpy(rng.standard_normal((b, t, n, h)).astype(np.float32)).cuda()
    got = check_attention(ops, ws, q if f32 else q.half(), cache, lengths, cap=20.0 if h == 128 else 0.0, with_scores=n % 3 != 0)
    assert not got[0].any() and not got[11].any()  # no cached token: zeros


@pytest.mark.parametrize("layout", [(8, 1, 256, 64), (8, 2, 128, 32), (4, 4, 64, 64), (6, 2, 96, 32)])
@pytest.mark.parametrize("t", [1, 4])
def test_attention_masks(ops, ws, layout, t):
    """Additive masks: ordinary values, the type's lowest value in places and over whole rows (equal weights then), -inf
    over slots that hold NaN and over whole rows (zeros)."""
    n, nkv, h, block = layout
    rng = np.random.default_rng(h + t)
    b, s = 6, 150
    low = np.finfo(np.float32).min
    mask = rng.standard_normal((b, 1, t, s)).astype(np.float32)
    mask[1, :, :, ::3] = low
    mask[2] = low
    mask[3, :, :, 40:90] = -np.inf
    mask[4] = -np.inf
    mask[5, :, :, 1:] = -1e30
    cache = filled(ops, rng, b, s, nkv, h, block)
    fill_nan([x[3] for x in cache], slice(40, 90))
    q = torch.from_numpy(rng.standard_normal((b, t, n, h)).astype(np.float32)).cuda()
    got = check_attention(ops, ws, q, cache, mask=mask, with_scores=True)
    assert not got[4].any() and got[2].any()
    check_attention(ops, ws, q.half(), cache, lengths=[150, 149, 130, 120, 5, 1], mask=mask, cap=15.0, with_scores=t == 4)


@pytest.mark.parametrize("h,block", [(256, 64), (128, 32), (64, 64), (96, 32)])
def test_later_drafts_do_not_reach_earlier_queries_and_nan_is_not_hidden(ops, ws, h, block):
    rng = np.random.default_rng(h)
    b, t, n, nkv, s, length = 2, 4, 4, 2, 64, 50
    cache = filled(ops, rng, b, s, nkv, h, block)
    fill_nan([x[0] for x in cache], slice(length - 2, length))  # the last two drafts' own slots
    fill_nan([x[1] for x in cache], slice(7, 8))                # a slot that everybody sees
    q = torch.from_numpy(rng.standard_normal((b, t, n, h)).astype(np.float32)).cuda()
    got = ops.sdpa_decode_int4(q, *cache, lengths=torch.full((b,), length, dtype=torch.int32, device="cuda"), ws=ws).cpu().numpy()
    assert np.isfinite(got[0, :2]).all() and np.isnan(got[0, 2:]).all() and np.isnan(got[1]).all()
    whole = filled(ops, np.random.default_rng(h), b, s, nkv, h, block)
    want = ops.sdpa_decode_int4(q, *whole, lengths=torch.full((b,), length, dtype=torch.int32, device="cuda"), ws=ws).cpu().numpy()
    assert np.array_equal(got[0, :2], want[0, :2])


@pytest.mark.parametrize("b,s,layout", [(1, 5000, (8, 1, 256, 64)), (3, 2100, (8, 2, 128, 64)), (40, 70, (8, 8, 64, 32)),
                                        (1, 17, (4, 1, 256, 32)), (2, 1500, (24, 2, 64, 64))])
@pytest.mark.parametrize("t", [1, 2])
def test_attention_over_many_pieces_and_many_sequences(ops, ws, b, s, layout, t):
    n, nkv, h, block = layout
    rng = np.random.default_rng(b + s)
    cache = filled(ops, rng, b, s, nkv, h, block)
    q = torch.from_numpy(rng.standard_normal((b, t, n, h)).astype(np.float16)).cuda()
    check_attention(ops, ws, q, cache, rng.integers(s // 2, s + 1, b), with_scores=True)
    check_attention(ops, ws, q.float(), cache, with_scores=t == 2)


@pytest.mark.parametrize("factor,scale", [(3e4, 1e-4), (1e-6, 1.0), (2.0 ** -20, 1e3), (6e4, 1e-7)])
def test_attention_queries_of_any_size(ops, ws, factor, scale):
    """Queries near fp16's ends; float32 queries far beyond them."""
    rng = np.random.default_rng(9)
    cache = filled(ops, rng, 2, 90, 1, 128, 64)
    q = torch.from_numpy(rng.uniform(-1, 1, (2, 1, 8, 128)).astype(np.float32)).cuda() * factor
    q[0, 0, 3] = 0.0
    check_attention(ops, ws, q.half(), cache, [90, 33], scale=scale)
    check_attention(ops, ws, q * (1e10 if factor > 1 else 1e-10), cache, [90, 33], scale=scale * (1e-10 if factor > 1 else 1e10))


@pytest.mark.parametrize("h,block", [(256, 64), (64, 32), (96, 32)])
def test_attention_over_values_of_any_size(ops, ws, h, block):
    """Value scales that differ by many orders of magnitude between tokens, growing and shrinking along the cache, and
    between blocks."""
    rng = np.random.default_rng(h)
    b, s, nkv = 4, 200, 1
    cache = filled(ops, rng, b, s, nkv, h, block)
    size = 2.0 ** np.linspace(-9, 9, s)
    for i, z in enumerate((size, size[::-1], rng.permutation(size))):
        cache[3][i] = (cache[3][i].float() * torch.from_numpy(z.copy()).float().cuda()[:, None, None, None]).half()
    cache[3][3, :, :, 0] *= 2.0 ** -9
    q = torch.from_numpy(rng.standard_normal((b, 1, 8, h)).astype(np.float32)).cuda()
    check_attention(ops, ws, q, cache, [200, 200, 200, 180], with_scores=True)


def test_attention_repeats_bit_for_bit_and_on_other_streams(ops):
    rng = np.random.default_rng(11)
    cache = filled(ops, rng, 5, 900, 2, 128, 64)
    q = torch.from_numpy(rng.standard_normal((5, 2, 8, 128)).astype(np.float16)).cuda()
    lengths = dev(np.asarray([900, 1, 456, 0, 777], np.int32))
    scores = torch.zeros((5, 2, 900), device="cuda")
    first = ops.sdpa_decode_int4(q, *cache, lengths=lengths, scores=scores)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in streams * 3:
        more = torch.zeros_like(scores)
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append((ops.sdpa_decode_int4(q, *cache, lengths=lengths, scores=more), more))
    torch.cuda.synchronize()
    for out, more in got:
        assert torch.equal(out, first) and torch.equal(more, scores)


def test_offsets_beyond_32_bits(ops, ws):
    """The third sequence of a cache of over 4 GB: nibbles, pairs and slots past 2^31 and 2^32 bytes."""
    b, s, nkv, h = 3, 65536, 64, 512
    cache = ops.int4_kv_cache(b, s, nkv, h)
    rng = np.random.default_rng(12)
    rows = rng.standard_normal((b, 3, nkv, h)).astype(np.float16)
    at = dev(np.asarray([0, 0, s - 3], np.int32))
    ops.kv_append_int4(dev(rows), dev(rows[:, ::-1]), at, *cache)
    k, v = ops.kv_read_int4(*cache, tokens=3, positions=at, dtype=torch.float32)
    for got, x in ((k, rows), (v, rows[:, ::-1])):
        u, scale, least = quantize(x, 64)
        want = u.reshape(*x.shape[:-1], -1, 64) * scale.astype(np.float32)[..., None] + least.astype(np.float32)[..., None]
        assert np.array_equal(got.cpu().numpy(), want.reshape(x.shape).astype(np.float32))
    del cache, k, v
    b, s, nkv, h = 3, 262144, 12, 256
    cache = ops.int4_kv_cache(b, s, nkv, h)
    rows = rng.standard_normal((b, 40, nkv, h)).astype(np.float16)
    at = dev(np.asarray([0, 0, s - 40], np.int32))
    ops.kv_append_int4(dev(rows), dev(rows[:, ::-1]), at, *cache)
    # everything else is hidden, so that the whole is a short cache's attention
    mask = torch.full((b, 1, 1, s), -math.inf, device="cuda")
    mask[:2, ..., :40] = 0
    mask[2, ..., s - 40:] = 0
    q = torch.from_numpy(rng.standard_normal((b, 1, 24, h)).astype(np.float16)).cuda()
    scores = torch.zeros((b, nkv, s), device="cuda")
    got = ops.sdpa_decode_int4(q, *cache, mask=mask, scores=scores, ws=ws).float()
    short = ops.int4_kv_cache(b, 40, nkv, h)
    ops.kv_append_int4(dev(rows), dev(rows[:, ::-1]), torch.zeros(b, dtype=torch.int32, device="cuda"), *short)
    few = torch.zeros((b, nkv, 40), device="cuda")
    want = ops.sdpa_decode_int4(q, *short, scores=few, ws=ws).float()
    # Two roundings of an output to fp16, and two of the weights: 40 of them, each at most half a step off, times |u - 8| <= 8
    # times a value scale, which is below (4.5 + 4.5) / 15 for normal numbers. (Sums in another order: below that.)
    assert torch.allclose(got, want, rtol=2 * EPS16, atol=2 * EPS16 * 8 * 0.6)
    assert torch.allclose(scores[2, :, s - 40:], few[2], rtol=1e-5, atol=1e-9) and not scores[2, :, :s - 40].any()
    kept, new, left = ops.kv_evict_int4(*cache, scores, torch.full((b,), s, dtype=torch.int32, device="cuda"), 16, recent=16)
    assert torch.equal(kept[2, 5].cpu(), torch.arange(s - 16, s, dtype=torch.int32)) and left.tolist() == [16] * 3
    for x, y in zip(cache, short):
        assert torch.equal(x[2, :16], y[2, 24:])


# ---- eviction --------------------------------------------------------------------------------------------
def evicted(scores, length, budget, sinks, recent):
    """Kept slots of one head."""
    if length <= budget:
        return list(range(length))
    rank = lambda x: -math.inf if x != x else x  # noqa: E731
    fixed = [s for s in range(length) if s < sinks or s >= length - recent]
    others = sorted(range(sinks, length - recent), key=lambda s: (scores[s] != scores[s], -rank(scores[s]), s))
    return sorted(fixed + others[:budget - len(fixed)])


def check_eviction(ops, cache, scores, lengths, budget, sinks, recent, into=None):
    b, s, nkv, _ = cache[0].shape
    before = [x.cpu().numpy().copy() for x in cache]
    to = cache if into is None else into
    there = [x.cpu().numpy().copy() for x in to]
    given = scores.clone()
    kept, new, left = ops.kv_evict_int4(*cache, scores, dev(np.asarray(lengths, np.int32)), budget, sinks=sinks, recent=recent, into=into)
    assert torch.equal(scores.view(torch.int32), given.view(torch.int32))
    sc = scores.cpu().numpy()
    assert left.tolist() == [min(budget, s, max(0, x)) for x in lengths]
    kept, new = kept.cpu().numpy(), new.cpu().numpy()
    for i in range(b):
        for j in range(nkv):
            want = evicted(sc[i, j].tolist(), min(s, max(0, lengths[i])), budget, sinks, recent)
            assert kept[i, j].tolist() == want + [-1] * (budget - len(want)), (i, j)
            assert np.array_equal(new[i, j, :len(want)].view(np.int32), sc[i, j, want].view(np.int32)) and not new[i, j, len(want):].any()
            for x in range(4):
                there[x][i, :len(want), j] = before[x][i, want, j]
    for x in range(4):
        assert np.array_equal(to[x].cpu().numpy().view(np.uint8), there[x].view(np.uint8)), x  # and nothing else was touched
    if into is not None:
        assert all(np.array_equal(x.cpu().numpy().view(np.uint8), y.view(np.uint8)) for x, y in zip(cache, before))


def random_cache(ops, seed, b, s, nkv, h, block):
    g = torch.Generator("cuda").manual_seed(seed)
    cache = ops.int4_kv_cache(b, s, nkv, h, block)
    for x in cache:
        x.view(torch.uint8).copy_(torch.randint(0, 256, x.view(torch.uint8).shape, generator=g, device="cuda").to(torch.uint8))
    return cache, g


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("budget,sinks,recent", [(40, 0, 0), (40, 4, 10), (40, 0, 40), (40, 40, 0), (40, 17, 23), (1, 0, 0), (1, 0, 1),
                                                 (199, 3, 3), (200, 0, 5)])
def test_eviction_keeps_the_right_slots(ops, into, budget, sinks, recent):
    """Ties (few distinct scores), both zeros, NaN, infinities, negative sums; lengths around the budget, none, beyond."""
    b, s, nkv, h, block = 9, 200, 2, 96, 32
    cache, g = random_cache(ops, budget + sinks, b, s, nkv, h, block)
    scores = torch.randn((b, nkv, s), generator=g, device="cuda")
    scores[1] = torch.randint(0, 3, (nkv, s), generator=g, device="cuda").float()
    scores[2] = 0.0
    scores[2, :, ::2] = -0.0
    scores[3, :, ::5] = float("nan")
    scores[4, :, 50:60], scores[4, :, 60:140] = float("inf"), -float("inf")
    scores[5] = float("nan")
    lengths = [200, 200, 200, 190, 200, 200, budget, 0, 4000]
    check_eviction(ops, cache, scores, lengths, budget, sinks, recent,
                   random_cache(ops, 1, b, max(budget, 60), nkv, h, block)[0] if into else None)


@pytest.mark.parametrize("b,s,nkv,h,block,budget", [(1, 9000, 1, 256, 64, 8000), (2, 3000, 1, 512, 32, 2500), (320, 700, 1, 64, 64, 650),
                                                    (100, 1300, 2, 256, 32, 1200), (1, 50000, 1, 64, 64, 1000)])
def test_eviction_of_more_rows_than_one_pass_moves(ops, b, s, nkv, h, block, budget):
    cache, g = random_cache(ops, s, b, s, nkv, h, block)
    scores = torch.rand((b, nkv, s), generator=g, device="cuda")
    scores = torch.where(torch.rand((b, nkv, s), generator=g, device="cuda") < 0.5, scores, torch.round(scores * 8) / 8)
    lengths = torch.randint(budget - 10, s + 1, (b,), generator=g, device="cuda").tolist()
    lengths[0] = s
    check_eviction(ops, cache, scores, lengths, budget, 4, 50)


# ---- together --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,nkv,h,block,f32", [(8, 1, 256, 64, False), (8, 4, 64, 32, True), (4, 2, 96, 32, True)])
def test_a_reply_with_evictions(ops, ws, n, nkv, h, block, f32):
    """A padded batch of prompts is stored and its last tokens attended to, replies grow, the cache is evicted from when it
    is full, and the replies go on: every step's outputs against float64 over the tokens that are still there, tracked by
    the kept slots."""
    rng = np.random.default_rng(h)
    dtype = np.float32 if f32 else np.float16
    b, s, budget, recent = 3, 48, 32, 8
    cache = ops.int4_kv_cache(b, s, nkv, h, block)
    scores = torch.zeros((b, nkv, s), device="cuda")
    counts = np.asarray([40, 25, 1], np.int32)
    token = lambda t: (rng.standard_normal((b, t, nkv, h)) * 1.5).astype(dtype)  # noqa: E731

    def stored(x):
        u, scale, least = quantize(x, block)
        wide = lambda y: np.repeat(y.astype(np.float64), block, -1)  # noqa: E731
        return u * wide(scale) + wide(least), u * np.abs(wide(scale)) + np.abs(wide(least)), 8 * np.abs(wide(scale))

    k, v = token(40), token(40)
    ops.kv_append_int4(dev(k), dev(v), torch.zeros(b, dtype=torch.int32, device="cuda"), *cache, counts=dev(counts))
    # per sequence and KV head: (key, its magnitudes, eight of its scales, value, ...) of the tokens still cached
    held = [[[tuple(z[i, x, j] for y in (k, v) for z in stored(y)) for x in range(counts[i])] for j in range(nkv)] for i in range(b)]
    lengths = dev(counts)
    evictions = 0
    for step in range(30):
        t = 3 if step % 7 == 3 else 1
        if int(lengths.max()) + t > s:
            ranked = scores.cpu().numpy()
            was = lengths.tolist()
            kept, scores, lengths = ops.kv_evict_int4(*cache, scores, lengths, budget, sinks=2, recent=recent)
            for i in range(b):
                for j in range(nkv):
                    want = evicted(ranked[i, j].tolist(), was[i], budget, 2, recent)
                    assert kept[i, j, :len(want)].tolist() == want
                    held[i][j] = [held[i][j][x] for x in want]
            evictions += 1
        k, v, q = token(t), token(t), rng.standard_normal((b, t, n, h)).astype(dtype)
        ops.kv_append_int4(dev(k), dev(v), lengths, *cache)
        lengths = lengths + t
        before = scores.cpu().numpy().copy()
        got = ops.sdpa_decode_int4(dev(q), *cache, lengths=lengths, scores=scores, ws=ws).cpu().numpy().astype(np.float64)
        now = stored(k) + stored(v)
        for i in range(b):
            for j in range(nkv):
                held[i][j] += [tuple(y[i, x, j] for y in now) for x in range(t)]
            rows = [np.stack([[y[c] for y in held[i][j]] for j in range(nkv)], 1) for c in range(6)]
            lim = limits_of(len(held[i][0]), s, t)
            assert lim[-1] == int(lengths[i])
            want, w, off, w_off = attention(q[i].astype(np.float64), rows[0], rows[3], rows[1], rows[4], lim, 1 / math.sqrt(h), 0.0, None,
                                             None if f32 else rows[5])
            bound = off + (EPS32 if f32 else EPS16) * np.abs(want) + 2.0 ** -25
            assert (np.abs(got[i] - want) <= bound).all(), (step, i)
            after = scores[i].cpu().numpy()
            assert (np.abs(after[:, :lim[-1]] - before[i][:, :lim[-1]] - w) <= w_off + 4 * EPS32 * (before[i][:, :lim[-1]] + w)).all()
    assert evictions >= 1


def test_a_captured_step_replays(ops):
    """Append, attention with scores and eviction into another cache as one CUDA graph, replayed over changed inputs; an
    eager call on another workspace in between."""
    rng = np.random.default_rng(21)
    b, s, nkv, n, h = 3, 200, 2, 8, 128
    cache, g = random_cache(ops, 2, b, s, nkv, h, 64)
    for i in (2, 3):
        cache[i].copy_(torch.randn(cache[i].shape, generator=g, device="cuda").half() * 0.2)
    into = ops.int4_kv_cache(b, 64, nkv, h)
    scores = torch.zeros((b, nkv, s), device="cuda")
    k, v, q = (torch.zeros((b, 1, m, h), dtype=torch.float16, device="cuda") for m in (nkv, nkv, n))
    at = dev(np.asarray([10, 100, 150], np.int32))
    lengths = at + 1
    ws = ops.Workspace("cuda")

    def step():
        ops.kv_append_int4(k, v, at, *cache)
        out = ops.sdpa_decode_int4(q, *cache, lengths=lengths, scores=scores, ws=ws)
        return [out] + list(ops.kv_evict_int4(*cache, scores, lengths, 64, recent=4, into=into))

    def fresh():
        for x in (k, v, q):
            x.copy_(torch.from_numpy(rng.standard_normal(x.shape).astype(np.float16)))

    fresh()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        fresh()
        scores.zero_()
        graph.replay()
        first = [x.clone() for x in outs + list(into) + list(cache) + [scores]]
        for x in into:
            x.zero_()
        ops.sdpa_decode_int4(q + 1, *cache, lengths=lengths)
        scores.zero_()
        again = step()
        for x, y in zip(first, again + list(into) + list(cache) + [scores]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_a_captured_call_keeps_its_workspace(ops):
    """A larger call later takes a larger workspace; the graph's stays its own."""
    cache, g = random_cache(ops, 3, 2, 9000, 2, 64, 32)  # (records of several CTAs, merged)
    for i in (2, 3):
        cache[i].copy_(torch.randn(cache[i].shape, generator=g, device="cuda").half() * 0.2)
    q = torch.randn((2, 1, 8, 64), generator=g, device="cuda")
    ws = ops.Workspace("cuda")
    want = ops.sdpa_decode_int4(q, *cache, ws=ws).clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sdpa_decode_int4(q, *cache, ws=ws)
    before, size = ws.sdpa.data_ptr(), ws.sdpa.numel()
    scores = torch.zeros((2, 2, 9000), device="cuda")
    ops.sdpa_decode_int4(q.expand(2, 1, 8, 64).repeat(1, 64, 1, 1), *cache, scores=scores, ws=ws)
    assert ws.sdpa.numel() > size and ws.sdpa.data_ptr() != before
    others = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(4)]  # (what would get its memory)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want) and all(bool((x == 255).all()) for x in others)


def test_rows_off_a_16_byte_boundary(ops, ws):
    """Queries, keys and values that begin anywhere, broadcast over the sequences, are those on a boundary."""
    rng = np.random.default_rng(31)
    for h, dtype in ((64, np.float16), (256, np.float32), (96, np.float16)):
        b, s, nkv, n = 2, 50, 2, 4
        def moved(shape):
            flat = dev(rng.standard_normal(1 + math.prod(shape)).astype(dtype))
            return flat[1:].view(shape)
        k, v, q = moved((1, 40, nkv, h)).expand(b, 40, nkv, h), moved((b, 40, nkv, h)), moved((b, 2, n, h))
        at, caches, outs = torch.zeros(b, dtype=torch.int32, device="cuda"), [], []
        for copy in (False, True):
            cache = ops.int4_kv_cache(b, s, nkv, h, 32)
            ops.kv_append_int4(k.clone() if copy else k, v.clone() if copy else v, at, *cache)
            caches.append(cache)
            outs.append(ops.sdpa_decode_int4(q.clone() if copy else q, *cache, lengths=at + 40, ws=ws))
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(*caches))
        assert torch.equal(*outs)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("h,block", [(256, 64), (96, 32)])
def test_both_host_paths_give_the_same(ops, monkeypatch, f32, h, block):
    """The calls through the extension, and again without it."""
    from litert_b200 import _lib

    native = ops._host
    assert native is not _lib._GeneralPath, "the extension is not built"
    b, s, nkv, n = 3, 70, 2, 6
    dtype = torch.float32 if f32 else torch.float16
    g = torch.Generator("cuda").manual_seed(7)
    k, v = (torch.randn((b, 20, nkv, h), generator=g, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn((b, 2, n, h), generator=g, device="cuda").to(dtype)
    mask = torch.randn((b, 1, 2, s), generator=g, device="cuda")
    at, counts = dev(np.asarray([0, 30, 45], np.int32)), dev(np.asarray([20, 7, 20], np.int32))
    results = []
    for path in (native, _lib._GeneralPath):
        monkeypatch.setattr(ops, "_host", path)
        ws = ops.Workspace("cuda")
        cache, scores = ops.int4_kv_cache(b, s, nkv, h, block), torch.zeros((b, nkv, s), device="cuda")
        ops.kv_append_int4(k, v, at, *cache, counts=counts)
        got = list(ops.kv_read_int4(*cache, tokens=25, positions=at, counts=counts, dtype=dtype))
        got += list(ops.kv_read_int4(*cache))
        for kw in (dict(), dict(scores=scores, lengths=at + counts, mask=mask, scale=0.1, logit_cap=4.0)):
            ops.sdpa_decode_int4(q, *cache, ws=ws)  # (the workspace is there)
            got.append(ops.sdpa_decode_int4(q, *cache, ws=ws, **kw))
        into = ops.int4_kv_cache(b, 30, nkv, h, block)
        got += list(ops.kv_evict_int4(*cache, scores, at + counts, 30, sinks=2, recent=5, into=into)) + list(into)
        got += list(ops.kv_evict_int4(*cache, scores, at + counts, 24)) + list(cache) + [scores]
        results.append(got)
    for x, y in zip(*results):
        assert x.dtype == y.dtype and x.shape == y.shape
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


def test_refusals(ops):
    cache = ops.int4_kv_cache(2, 16, 2, 64)
    x = torch.zeros((2, 1, 2, 64), device="cuda")
    at = torch.zeros(2, dtype=torch.int32, device="cuda")
    scores = torch.zeros((2, 2, 16), device="cuda")
    q = torch.zeros((2, 1, 4, 64), device="cuda")
    bad = [
        lambda: ops.kv_append_int4(x.bfloat16(), x.bfloat16(), at, *cache),
        lambda: ops.kv_append_int4(x, x.half(), at, *cache),
        lambda: ops.kv_append_int4(x[:1], x[:1], at, *cache),
        lambda: ops.kv_append_int4(x[..., :32], x[..., :32], at, *cache),
        lambda: ops.kv_append_int4(x, x.expand(2, 3, 2, 64), at, *cache),
        lambda: ops.kv_append_int4(x, x, at.long(), *cache),
        lambda: ops.kv_append_int4(x, x, at[:1], *cache),
        lambda: ops.kv_append_int4(x, x, None, *cache),
        lambda: ops.kv_append_int4(x, x, at, cache[0][:, ::2], cache[1][:, ::2], cache[2][:, ::2], cache[3][:, ::2]),
        lambda: ops.kv_append_int4(x, x, at, cache[0], cache[1][:, :8].contiguous(), cache[2], cache[3]),
        lambda: ops.kv_append_int4(x, x, at, cache[0], cache[1], cache[2].float(), cache[3]),
        lambda: ops.kv_append_int4(x.cpu(), x.cpu(), at, *cache),
        lambda: ops.kv_read_int4(*cache, dtype=torch.bfloat16),
        lambda: ops.kv_read_int4(*cache, tokens=-1),
        lambda: ops.kv_read_int4(*cache, counts=at.float()),
        lambda: ops.sdpa_decode_int4(q.bfloat16(), *cache),
        lambda: ops.sdpa_decode_int4(q[:, :, :3], *cache),
        lambda: ops.sdpa_decode_int4(q[:, :0], *cache),
        lambda: ops.sdpa_decode_int4(q[0], *cache),
        lambda: ops.sdpa_decode_int4(q, *cache, lengths=at[:1]),
        lambda: ops.sdpa_decode_int4(q, *cache, mask=torch.zeros((2, 1, 1, 15), device="cuda")),
        lambda: ops.sdpa_decode_int4(q, *cache, mask=torch.zeros((1, 1, 1, 16), device="cuda")),
        lambda: ops.sdpa_decode_int4(q, *cache, scores=scores[:, :1]),
        lambda: ops.sdpa_decode_int4(q, *cache, scores=scores.transpose(0, 1)),
        lambda: ops.sdpa_decode_int4(q, *cache, scores=scores.half()),
        lambda: ops.sdpa_decode_int4(q, *cache, scale=-1.0),
        lambda: ops.sdpa_decode_int4(q, *cache, logit_cap=float("nan")),
        lambda: ops.kv_evict_int4(*cache, scores, at, 0),
        lambda: ops.kv_evict_int4(*cache, scores, at, 17),
        lambda: ops.kv_evict_int4(*cache, scores, at, 4, sinks=3, recent=2),
        lambda: ops.kv_evict_int4(*cache, scores, at, 4, recent=-1),
        lambda: ops.kv_evict_int4(*cache, scores, None, 4),
        lambda: ops.kv_evict_int4(*cache, None, at, 4),
        lambda: ops.kv_evict_int4(*cache, scores[..., :8], at, 4),
        lambda: ops.kv_evict_int4(*cache, scores, at, 4, into=ops.int4_kv_cache(2, 16, 2, 64, 32)),
        lambda: ops.kv_evict_int4(*cache, scores, at, 9, into=ops.int4_kv_cache(2, 8, 2, 64)),
        lambda: ops.kv_evict_int4(*cache, scores, at, 4, into=cache[:3]),
        lambda: ops.kv_evict_int4(*cache, scores, at, 4, into=(cache[1], cache[0], cache[2], cache[3])),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ops.B200Error):
            call()
            pytest.fail(f"call {i} was taken")
    assert all(not t.any() for t in cache)
