"""Calls on the 4-bit cache at the edges of what is accepted: through the extension and through the general path."""
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops():
    from litert_b200 import ops as o

    return o


@pytest.fixture(params=["native", "general"])
def path(request, ops, monkeypatch):
    from litert_b200 import _lib

    if request.param == "general":
        monkeypatch.setattr(ops, "_host", _lib._GeneralPath)
    else:
        assert ops._host is not _lib._GeneralPath, "the extension is not built"
    return request.param


def test_a_cache_without_slots_heads_or_channels_is_not_made(ops):
    for shape in ((2, 0, 1, 64), (2, 8, 0, 64), (2, 8, 1, 0), (-1, 8, 1, 64)):
        with pytest.raises(ops.B200Error):
            ops.int4_kv_cache(*shape, device="cpu")
    assert ops.int4_kv_cache(0, 8, 1, 64, device="cpu")[0].shape == (0, 8, 1, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("s,nkv,half", [(16, 0, 32), (0, 2, 32), (16, 2, 0)])
def test_a_cache_without_slots_heads_or_channels_is_refused(ops, path, s, nkv, half):
    cache = [torch.zeros((2, s, nkv, half), dtype=torch.uint8, device="cuda") for _ in range(2)]
    cache += [torch.zeros((2, s, nkv, 1, 2), dtype=torch.float16, device="cuda") for _ in range(2)]
    ws = ops.Workspace("cuda")
    ws.sdpa_bytes(1 << 20)
    q, x = (torch.zeros((2, 1, m, 2 * half), device="cuda") for m in (4, nkv))
    at = torch.zeros(2, dtype=torch.int32, device="cuda")
    scores = torch.zeros((2, nkv, s), device="cuda")
    for call in (lambda: ops.sdpa_decode_int4(q, *cache, ws=ws), lambda: ops.sdpa_decode_int4(q, *cache),
                 lambda: ops.sdpa_decode_int4(q, *cache, scores=scores, ws=ws), lambda: ops.kv_append_int4(x, x, at, *cache),
                 lambda: ops.kv_read_int4(*cache), lambda: ops.kv_read_int4(*cache, tokens=1), lambda: ops.kv_evict_int4(*cache, scores, at, 1)):
        with pytest.raises(ops.B200Error):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("f32", [False, True])
def test_no_sequence_is_no_work(ops, path, f32):
    dtype = torch.float32 if f32 else torch.float16
    cache, into = ops.int4_kv_cache(0, 16, 2, 64), ops.int4_kv_cache(0, 8, 2, 64)
    at, scores = torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros((0, 2, 16), device="cuda")
    x, q = torch.zeros((0, 3, 2, 64), dtype=dtype, device="cuda"), torch.zeros((0, 1, 4, 64), dtype=dtype, device="cuda")
    ops.kv_append_int4(x, x, at, *cache, counts=at)
    assert [tuple(y.shape) for y in ops.kv_read_int4(*cache, tokens=5, dtype=dtype)] == [(0, 5, 2, 64)] * 2
    for ws in (None, ops.Workspace("cuda")):
        assert ops.sdpa_decode_int4(q, *cache, lengths=at, scores=scores, ws=ws).shape == q.shape
    for to, slots in ((None, 16), (into, 8)):
        kept, new, lengths = ops.kv_evict_int4(*cache, scores, at, 4, into=to)
        assert (kept.shape, new.shape, lengths.shape) == ((0, 2, 4), (0, 2, slots), (0,))


def test_no_sequence_needs_no_memory():
    """The C ABI, where an empty tensor has no address."""
    from litert_b200 import _lib, build

    build.build_kernels()
    lib = _lib.load()
    none = (None,) * 4
    assert lib.b200_kv4_append(None, None, 0, 0, 0, 0, 0, None, None, 0, 1, 2, 64, 32, 16, *none, None) == 0
    assert lib.b200_kv4_read(*none, 0, 16, 2, 64, 32, None, None, 1, 0, None, None, None) == 0
    assert lib.b200_kv4_sdpa(None, *none, None, None, None, None, 0, 1, 4, 2, 64, 32, 16, 0, 0.0, 0.0, None, 0, None) == 0
    assert lib.b200_kv4_evict(*none, 0, 16, 2, 64, 32, None, None, 4, 0, 0, *none, 16, None, None, None, None) == 0
    assert lib.b200_kv4_append(None, None, 0, 0, 0, 0, 0, None, None, 0, 1, 2, 80, 32, 16, *none, None) != 0  # (checked all the same)


def exact_nibbles(x, scale, least):
    """The integers nearest to (x - least) / scale in rational arithmetic, ties to even, clamped."""
    from fractions import Fraction

    s, m = Fraction(float(scale)), Fraction(float(least))
    return [max(0, min(15, round((Fraction(float(v)) - m) / s))) for v in x]


@pytest.mark.gpu
@pytest.mark.parametrize("block", [32, 64])
def test_the_nearest_nibble_is_exact_for_elements_of_any_size(ops, path, block):
    """float32 elements next to a border of which the difference to the least value does not fit 64 bits: tiny ones where a
    border is zero, and neighbours of every border."""
    import numpy as np

    rng = np.random.default_rng(block)
    rows = []
    for least, scale in ((-1.0, 2.0), (-3.0, 2.0), (-0.25, 0.5), (-29.0, 2.0), (-1000.0, 80.0), (-2.0 ** -10, 2.0 ** -9)):
        tiny = np.float32([0.0, 1e-30, -1e-30, 1e-45, -1e-45, 1e-38, -1e-38, 1e-20, -1e-20, 1e-12, -1e-12, 1e-9, -1e-9])
        edges = np.float32([least + scale * (k + 0.5) for k in range(15)])
        near = np.concatenate([edges, np.nextafter(edges, np.float32(np.inf)), np.nextafter(edges, np.float32(-np.inf))])
        for part in (np.resize(tiny, block - 2), rng.choice(near, block - 2), rng.choice(near, block - 2)):
            rows.append(np.concatenate([np.float32([least, least + 15 * scale]), part]))
    x = torch.from_numpy(np.stack(rows).astype(np.float32))[None, :, None].cuda()
    cache = ops.int4_kv_cache(1, len(rows), 1, block, block)
    ops.kv_append_int4(x, x, torch.zeros(1, dtype=torch.int32, device="cuda"), *cache)
    nibbles, pairs = cache[0][0, :, 0].cpu().numpy(), cache[2][0, :, 0, 0].cpu().numpy()
    got = np.stack((nibbles & 15, nibbles >> 4), -1).reshape(len(rows), block)
    for i, row in enumerate(rows):
        assert got[i].tolist() == exact_nibbles(row, pairs[i, 0], pairs[i, 1]), i


@pytest.mark.gpu
def test_a_budget_beyond_the_slots_is_refused_before_memory_is_taken(ops, path):
    cache = ops.int4_kv_cache(2, 16, 2, 64)
    scores, at = torch.zeros((2, 2, 16), device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for budget in (17, 1 << 28):
        with pytest.raises(ops.B200Error, match="budget"):
            ops.kv_evict_int4(*cache, scores, at, budget)
    assert torch.cuda.max_memory_allocated() == before


def test_caches_beyond_the_kernels_indexes_are_refused():
    """Slots are walked over in 32-bit integers, some hundreds at a time past the last. Refused on the host, on the CPU."""
    from litert_b200 import _lib, build

    build.build_kernels()
    lib = _lib.load()
    p = 1 << 20
    cache = (p, 2 * p, 3 * p, 4 * p)
    for s in (2 ** 31 - 1, 2 ** 30 + 1):
        calls = [
            lib.b200_kv4_append(p, p, 0, 0, 0, 0, 0, p, None, 1, 1, 1, 32, 32, s, *cache, None),
            lib.b200_kv4_read(*cache, 1, s, 1, 32, 32, None, None, 1, 0, p, p, None),
            lib.b200_kv4_sdpa(p, *cache, None, None, None, p, 1, 1, 1, 1, 32, 32, s, 0, 0.0, 0.0, p, 1 << 62, None),
            lib.b200_kv4_sdpa(p, *cache, None, None, None, p, 1, 1, 1, 1, 64, 32, s, 0, 0.0, 0.0, p, 1 << 62, None),
            lib.b200_kv4_evict(*cache, 1, s, 1, 32, 32, p << 10, p << 11, 4, 0, 0, *cache, s, p << 12, p << 13, p << 14, None),
            lib.b200_kv4_evict(*cache, 1, 64, 1, 32, 32, p << 10, p << 11, 4, 0, 0, p << 20, p << 22, p << 24, p << 26, s, p << 12, p << 30, p << 14, None),
        ]
        assert calls == [4] * 6, (s, calls)
        assert b"slots" in lib.b200_kv4_last_error()
