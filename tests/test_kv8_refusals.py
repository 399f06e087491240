"""Host-side checks of the 8-bit cache operators: what is refused before anything reaches the device (no GPU needed)."""
import ctypes

import pytest
import torch


def _desc(cabi, **kw):
    d = dict(k=256, v=512, k_scale=1024, v_scale=2048, k_tail=4096, v_tail=8192, status=64, batch=1, heads=2, capacity=128, format=0)
    d.update(kw)
    return cabi.Kv8Desc(*[d[n] for n, _ in cabi.Kv8Desc._fields_])


@pytest.fixture()
def cabi(built_lib):
    from minference_b200 import _cabi

    return _cabi


@pytest.mark.parametrize("change, word", [
    ({"k": 0}, b"null"), ({"status": 0}, b"null"), ({"batch": 0}, b"sizes"), ({"heads": 0}, b"sizes"), ({"capacity": 0}, b"capacity"),
    ({"capacity": 100}, b"capacity"), ({"format": 7}, b"format"), ({"v": 520}, b"aligned"), ({"k_tail": 4104}, b"aligned")])
def test_descriptor_checks(cabi, change, word):
    lib = cabi.lib()
    d = ctypes.byref(_desc(cabi, **change))
    st = (ctypes.c_int64 * 3)(256, 128, 128)
    assert lib.minf_kv8_store(d, 256, 256, st, st, 1, None, 0, None, None) == -1 and word in lib.minf_last_error()
    assert lib.minf_kv8_load(d, None, 0, None, 0, 1, 256, 256, None) == -1 and word in lib.minf_last_error()
    assert lib.minf_kv8_attention(d, 256, st, 256, st, 2, 1, None, 0, 0, 1.0, None, None, None, None, None, 256, None) == -1
    assert word in lib.minf_last_error()


def test_store_checks(cabi):
    lib, d = cabi.lib(), ctypes.byref(_desc(cabi))
    ok = (ctypes.c_int64 * 3)(256, 128, 128)
    odd = (ctypes.c_int64 * 3)(256, 129, 128)
    for args, word in [((0, 256, ok, ok, 1, None, 0, None), b"null"), ((256, 264, ok, ok, 1, None, 0, None), b"aligned"),
                       ((256, 256, ok, odd, 1, None, 0, None), b"strides"), ((256, 256, ok, ok, -1, None, 0, None), b"n_tokens"),
                       ((256, 256, ok, ok, 1, None, 128, None), b"fit"), ((256, 256, ok, ok, 1, None, -1, None), b"outside"),
                       ((256, 256, ok, ok, 129, None, 0, None), b"fit")]:
        assert lib.minf_kv8_store(d, *args, None) == -1 and word in lib.minf_last_error(), args
    assert lib.minf_kv8_store(d, 256, 256, ok, ok, 0, None, 128, None, None) == 0        # nothing to store: no launch


def test_load_checks(cabi):
    lib, d = cabi.lib(), ctypes.byref(_desc(cabi))
    for args, word in [((None, 129, None, 0, 1, 256, 256), b"outside"), ((None, 1, None, 0, -1, 256, 256), b"count"),
                       ((None, 1, None, 0, 1, 0, 256), b"null"), ((None, 1, None, 0, 1, 256, 264), b"aligned")]:
        assert lib.minf_kv8_load(d, *args, None) == -1 and word in lib.minf_last_error(), args
    assert lib.minf_kv8_load(d, None, 1, None, 0, 0, None, None, None) == 0


def test_attention_checks(cabi):
    lib, d = cabi.lib(), ctypes.byref(_desc(cabi))
    st = (ctypes.c_int64 * 3)(512, 128, 128)
    bad = (ctypes.c_int64 * 3)(512, 130, 128)
    w = (ctypes.c_int64 * 3)(128, 128, 0)
    base = dict(q=256, qs=st, o=256, os=st, hq=4, n_q=1, lengths=None, n=100, longest=128, scale=1.0, lse=None, weights=None, ws=None,
                add=None, adds=None, scratch=256)
    for change, word in [({"q": 0}, b"null"), ({"o": 0}, b"null"), ({"hq": 3}, b"sizes"), ({"hq": 0}, b"sizes"), ({"n_q": 0}, b"sizes"),
                         ({"longest": 129}, b"max_length"), ({"longest": -1}, b"sizes"), ({"n": 129}, b"outside"), ({"n": -1}, b"outside"),
                         ({"scratch": 0}, b"scratch"), ({"scratch": 264}, b"aligned"), ({"os": bad}, b"strides"), ({"o": 260}, b"aligned"),
                         ({"weights": 256}, b"null"), ({"add": 256}, b"null"), ({"add": 256, "adds": w}, b"add_to")]:
        a = {**base, **change}
        if "scratch" in change and not change["scratch"]:
            a.update(weights=256, ws=w)              # weights always need scratch
        assert lib.minf_kv8_attention(d, *a.values(), None) == -1 and word in lib.minf_last_error(), (change, lib.minf_last_error())
    assert lib.minf_kv8_attention_scratch_bytes(1, 3, 2, 1, 128, 0) == 0
    assert lib.minf_kv8_attention_scratch_bytes(1, 4, 2, 1, 128, 1) >= 2 * 128 * 2 * 4


def test_evict_checks(cabi):
    lib = cabi.lib()
    other = dict(k=1 << 20, v=2 << 20, k_scale=5 << 20, v_scale=6 << 20, k_tail=3 << 20, v_tail=4 << 20)
    src = _desc(cabi, k=1 << 24, v=2 << 24, k_scale=5 << 24, v_scale=6 << 24, k_tail=3 << 24, v_tail=4 << 24)
    dst = _desc(cabi, capacity=64, **other)
    w = (ctypes.c_int64 * 3)(128, 128, 0)
    def call(s=src, d=dst, n=128, longest=128, weights=256, budget=32, recent=8, sink=4, kept=256):
        return lib.minf_kv8_evict(ctypes.byref(s), ctypes.byref(d), None, n, longest, weights, w, budget, recent, sink, kept, 256, 256, None)
    inside = dict(other, v=(1 << 24) + 32 * 128, capacity=64)      # its values in the middle of the source's keys
    for kw, word in [(dict(d=src), b"another"), (dict(d=_desc(cabi, **inside)), b"another"),
                     (dict(d=_desc(cabi, **dict(other, k_scale=(5 << 24) + 4))), b"another"), (dict(d=_desc(cabi, format=1, **other)), b"format"),
                     (dict(budget=0), b"budget"), (dict(recent=30), b"budget"), (dict(sink=-1), b"budget"), (dict(recent=-1), b"budget"),
                     (dict(budget=65), b"fit"), (dict(n=129), b"outside"), (dict(longest=129), b"max_length"), (dict(weights=0), b"null"),
                     (dict(kept=0), b"null")]:
        assert call(**kw) == -1 and word in lib.minf_last_error(), (kw, lib.minf_last_error())


def test_no_cpu_path(cabi):
    from minference_b200 import KV8Cache

    with pytest.raises(cabi.MInferB200Error):
        KV8Cache.empty(1, 1, 64, device="cpu")


def test_decode_layer_refusals(cabi):
    from minference_b200 import KV8HFCache, KV8Layer

    for kw in (dict(budget=0), dict(budget=8, recent=6, sink=4), dict(budget=8, sink=-1), dict(budget=8, slack=0)):
        with pytest.raises(cabi.MInferB200Error):
            KV8Layer(**kw)
        with pytest.raises(cabi.MInferB200Error):
            KV8HFCache(**kw)
    past = KV8HFCache()
    two = torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(cabi.MInferB200Error, match="one sequence"):
        past.update(two, two, 0)
    with pytest.raises(cabi.MInferB200Error):
        past.update(two[:1], two[:1], 0)                    # CPU tensors
    assert past.get_seq_length() == 0


def test_attention_refuses_misaligned_queries(cabi):
    lib, d = cabi.lib(), ctypes.byref(_desc(cabi))
    st, odd = (ctypes.c_int64 * 3)(512, 128, 128), (ctypes.c_int64 * 3)(512, 132, 128)
    for q, qs, word in [(264, st, b"aligned"), (256, odd, b"strides")]:
        rc = lib.minf_kv8_attention(d, q, qs, 256, st, 4, 1, None, 100, 128, 1.0, None, None, None, None, None, 256, None)
        assert rc == -1 and b"quer" in lib.minf_last_error() and word in lib.minf_last_error(), lib.minf_last_error()


def test_misaligned_tensors_are_copied(cabi):
    """A contiguous view at an odd address, and one whose stride along a dimension of size one is odd."""
    from types import SimpleNamespace

    from minference_b200.ops import kv8_cache

    cache = SimpleNamespace(batch=1, device=torch.device("cpu"))
    buf = torch.arange(2 * 128 + 8).to(torch.bfloat16)
    for t in (buf[1:257].view(1, 2, 1, 128), buf[:256].as_strided((1, 2, 1, 128), (129, 128, 3, 1))):
        r = kv8_cache._rows(t, "query", cache)
        assert torch.equal(r, t) and r.data_ptr() % 16 == 0 and not any(s % 8 for s in r.stride()[:3])


def test_load_to_the_end_wants_one_first_token(cabi, monkeypatch):
    """With a first token for each sequence there is no one number of tokens up to the capacity."""
    from types import SimpleNamespace

    from minference_b200.ops import kv8_cache

    calls = []
    monkeypatch.setattr(kv8_cache, "_launch", lambda entry, cache, *args: calls.append(args))
    cache = SimpleNamespace(batch=1, kv_heads=2, capacity=128, device=torch.device("cpu"), _ref=None)
    for batch in (1, 2):
        cache.batch = batch
        first = torch.zeros(batch, dtype=torch.int32)
        with pytest.raises(cabi.MInferB200Error, match="count"):
            kv8_cache.kv8_load(cache, 100, first=first)
        assert kv8_cache.kv8_load(cache, 100, first=first, count=5)[0].shape == (batch, 2, 5, 128)
    assert kv8_cache.kv8_load(cache, 100, first=28)[0].shape == (2, 2, 100, 128) and len(calls) == 3


@pytest.mark.parametrize("strides, taken", [
    ((200, 100, 1), True), ((100, 200, 1), True), ((1 << 20, 1 << 10, 1), True), ((150, 100, 1), False), ((150, 300, 1), True),
    ((100, 100, 1), False), ((100, 50, 1), False), ((99, 300, 1), False), ((100, 0, 1), False), ((0, 100, 1), False)])
def test_weights_of_two_heads_must_not_overlap(cabi, strides, taken):
    """Each element is written by one head of one sequence: [2, 2, >= 100] with 100 tokens of them written."""
    from minference_b200.ops import kv8_cache

    w = torch.zeros(1 << 21).as_strided((2, 2, 120), strides)
    if taken:
        kv8_cache._check_written(w, None, 100)
        kv8_cache._check_written(w, w, 100)
    else:
        with pytest.raises(cabi.MInferB200Error, match="written"):
            kv8_cache._check_written(w, None, 100)


def test_weights_that_interleave_without_overlapping_are_taken(cabi):
    """Three heads 100 elements apart and two sequences 150 apart: 50 tokens each, no two at the same place."""
    from minference_b200.ops import kv8_cache

    w = torch.zeros(1000).as_strided((2, 3, 50), (150, 100, 1))
    kv8_cache._check_written(w, None, 50)
    with pytest.raises(cabi.MInferB200Error):
        kv8_cache._check_written(w, None, 51)
    kv8_cache._check_written(torch.zeros(3, 1, 50).expand(3, 4, 50)[:, :1], None, 50)
    kv8_cache._check_written(torch.zeros(1, 1, 50).expand(4, 4, 50), None, 0)       # nothing is written
