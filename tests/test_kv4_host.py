"""Refusals of the 4-bit cache's entry points. Nothing here reaches a GPU: every call is refused on the host."""
import ctypes

import pytest
import torch

P = 1 << 20  # stands for a device address; calls that carry it are refused before any use
MAX = ctypes.c_longlong(2 ** 31 - 1).value


@pytest.fixture(scope="module")
def lib():
    from litert_b200 import _lib, build

    build.build_kernels()
    return _lib.load()


CACHE = dict(b=2, s_max=64, nkv=2, h=64, block=32)


def _append(lib, k=P, v=P, dtype=0, positions=P, t=1, cache=(P, 2 * P, 3 * P, 4 * P), **c):
    c = {**CACHE, **c}
    return lib.b200_kv4_append(k, v, dtype, 0, 0, 0, 0, positions, None, c["b"], t, c["nkv"], c["h"], c["block"], c["s_max"], *cache,
                               None)


def _read(lib, dtype=0, t=1, k=P, v=P, cache=(P, 2 * P, 3 * P, 4 * P), **c):
    c = {**CACHE, **c}
    return lib.b200_kv4_read(*cache, c["b"], c["s_max"], c["nkv"], c["h"], c["block"], None, None, t, dtype, k, v, None)


def _sdpa(lib, q=P, out=P, t=1, n=4, dtype=0, scale=0.0, cap=0.0, ws=P, ws_bytes=None, cache=(P, 2 * P, 3 * P, 4 * P), **c):
    c = {**CACHE, **c}
    if ws_bytes is None:
        ws_bytes = lib.b200_kv4_sdpa_workspace_bytes(c["b"], t, n, c["nkv"], c["h"], c["block"], c["s_max"], 0)
    return lib.b200_kv4_sdpa(q, *cache, None, None, None, out, c["b"], t, n, c["nkv"], c["h"], c["block"], c["s_max"], dtype, scale, cap,
                             ws, ws_bytes, None)


def _evict(lib, budget=8, sinks=0, recent=0, to=None, s_to=None, scores=50 * P, lengths=51 * P, kept=52 * P, scores_out=53 * P,
           lengths_out=54 * P, cache=(P, 2 * P, 3 * P, 4 * P), **c):
    c = {**CACHE, **c}
    return lib.b200_kv4_evict(*cache, c["b"], c["s_max"], c["nkv"], c["h"], c["block"], scores, lengths, budget, sinks, recent,
                              *(to or cache), s_to or c["s_max"], kept, scores_out, lengths_out, None)


@pytest.mark.parametrize("call", [_append, _read, _sdpa, _evict])
@pytest.mark.parametrize("wrong", [dict(h=80), dict(block=16), dict(block=128, h=128), dict(h=1024), dict(h=0), dict(nkv=0),
                                   dict(s_max=0), dict(b=-1), dict(cache=(None, 2 * P, 3 * P, 4 * P)), dict(b=1 << 17),
                                   dict(cache=(P, 2 * P, 3 * P, None)), dict(cache=(P + 8, 2 * P, 3 * P, 4 * P)),
                                   dict(cache=(P, 2 * P, 3 * P + 2, 4 * P))])
def test_cache_that_is_none(lib, call, wrong):
    assert call(lib, **wrong) in (1, 4)
    assert lib.b200_kv4_last_error().startswith(b"b200_kv4_")


@pytest.mark.parametrize("wrong", [dict(k=None), dict(v=None), dict(positions=None), dict(dtype=1), dict(dtype=7), dict(t=-1),
                                   dict(k=P + 1), dict(dtype=2, v=P + 2), dict(t=2 ** 31 - 1, b=60000, nkv=60000)])
def test_append_refusals(lib, wrong):
    assert _append(lib, **wrong) in (1, 4)


@pytest.mark.parametrize("wrong", [dict(k=None), dict(v=None), dict(dtype=1), dict(t=-1), dict(k=P + 8),
                                   dict(t=2 ** 31 - 1, b=60000, nkv=60000)])
def test_read_refusals(lib, wrong):
    assert _read(lib, **wrong) in (1, 4)


@pytest.mark.parametrize("wrong", [dict(q=None), dict(out=None), dict(t=0), dict(t=1 << 20), dict(n=3), dict(n=0), dict(dtype=1),
                                   dict(scale=-1.0), dict(scale=float("nan")), dict(cap=-1.0), dict(cap=float("nan")),
                                   dict(ws=None), dict(ws_bytes=0), dict(ws=P + 4), dict(ws_bytes=64), dict(q=P + 8),
                                   dict(out=P + 1), dict(dtype=2, out=P + 2)])
def test_attention_refusals(lib, wrong):
    assert _sdpa(lib, **wrong) in (1, 4)


@pytest.mark.parametrize("wrong", [
    dict(budget=0), dict(budget=-4), dict(sinks=-1), dict(recent=-1), dict(sinks=5, recent=4), dict(budget=65),
    dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), dict(scores=None), dict(lengths=None), dict(kept=None), dict(scores_out=None),
    dict(lengths_out=None), dict(scores_out=50 * P), dict(lengths_out=51 * P), dict(scores_out=50 * P + 4),
    dict(to=(P, 2 * P, 3 * P, 5 * P)),                      # in place, but one tensor is another
    dict(s_to=32),                                          # in place, but of another length
    dict(to=(P + 64, 12 * P, 13 * P, 14 * P)),              # overlaps the source
    dict(to=(11 * P, 2 * P, 13 * P, 14 * P)),               # shares a tensor
    dict(to=(2 * P, 11 * P, 13 * P, 14 * P)),               # its keys are the source's values
    dict(to=(11 * P, 12 * P, 13 * P, 14 * P), s_to=7),      # too short for the budget
])
def test_eviction_refusals(lib, wrong):
    assert _evict(lib, **wrong) in (1, 4)


def test_the_workspace_does_not_grow_with_the_cache_where_no_logit_is_kept(lib):
    need = [lib.b200_kv4_sdpa_workspace_bytes(64, 1, 8, 1, 256, 64, s, 0) for s in (4096, 32768, 1 << 20)]
    assert need[0] == need[1] == need[2] < 32 << 20


def test_nothing_to_do_is_no_error(lib):
    assert _append(lib, b=0) == 0 and _append(lib, t=0) == 0
    assert _read(lib, b=0) == 0 and _read(lib, t=0) == 0
    assert _sdpa(lib, b=0) == 0 and _evict(lib, b=0) == 0
    assert lib.b200_kv4_sdpa_workspace_bytes(0, 1, 4, 2, 64, 32, 64, 0) == 0


def test_python_refusals():
    from litert_b200 import ops

    with pytest.raises(ops.B200Error, match="blocks"):
        ops.int4_kv_cache(1, 8, 1, 80, block=64, device="cpu")
    with pytest.raises(ops.B200Error, match="blocks"):
        ops.int4_kv_cache(1, 8, 1, 128, block=128, device="cpu")
    cache = ops.int4_kv_cache(1, 8, 1, 64, device="cpu")
    assert [tuple(t.shape) for t in cache] == [(1, 8, 1, 32)] * 2 + [(1, 8, 1, 1, 2)] * 2
    x = torch.zeros((1, 1, 1, 64))
    for call in (lambda: ops.kv_append_int4(x, x, torch.zeros(1, dtype=torch.int32), *cache), lambda: ops.kv_read_int4(*cache),
                 lambda: ops.sdpa_decode_int4(x, *cache),
                 lambda: ops.kv_evict_int4(*cache, torch.zeros((1, 1, 8)), torch.zeros(1, dtype=torch.int32), 4)):
        with pytest.raises(ops.B200Error, match="CUDA tensor"):
            call()
