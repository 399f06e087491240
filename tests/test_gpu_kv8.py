"""8-bit key/value cache operators on the GPU against their definition in 64 bits (tests/kv8_reference.py)."""
import math

import pytest
import torch

from tests import kv8_reference as R

pytestmark = pytest.mark.gpu
KINDS = [torch.float8_e4m3fn, torch.int8]
NAN = float("nan")


def _rows(gen, b, h, n, scale=1.0):
    """bf16 [b, h, n, 128] as a projection leaves them (heads inside), on the CPU and the GPU."""
    x = (torch.randn(b, n, h, 128, generator=gen) * scale).to(torch.bfloat16)
    return x.transpose(1, 2), x.cuda().transpose(1, 2)


def _poisoned(b, h, capacity, kind):
    """A cache full of what an earlier use could have left: NaN codes, scales and tails."""
    from minference_b200 import KV8Cache

    c = KV8Cache.empty(b, h, capacity, kind)
    for t in (c.k, c.v):
        t.view(torch.uint8).fill_(0x7f)
    for t in (c.k_scale, c.v_scale, c.k_tail, c.v_tail):
        t.fill_(NAN)
    return c


def _filled(gen, b, h, lengths, kind, capacity=None, v_scale=1.0):
    """(cache, reference) holding lengths[i] tokens of sequence i, stored in one padded call."""
    from minference_b200 import kv8_store

    n = max(max(lengths), 1)
    cache, ref = _poisoned(b, h, capacity or n, kind), R.RefCache(b, h, kind)
    k, dk = _rows(gen, b, h, n)
    v, dv = _rows(gen, b, h, n, v_scale)
    counts = torch.tensor(lengths, dtype=torch.int32)
    kv8_store(cache, dk, dv, 0, counts=counts.cuda())
    ref.append(k, v, counts)
    return cache, ref


def _check_values(cache, ref, lengths):
    """kv8_load gives the reference's values, rounded once to bf16, and zeros behind them; codes and scales are its own."""
    from minference_b200 import kv8_load

    k, v = kv8_load(cache, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    for name, got, codes, scales in (("k", k.cpu(), cache.k, cache.k_scale), ("v", v.cpu(), cache.v, cache.v_scale)):
        codes, scales = codes.cpu().double(), scales.cpu().double()
        for b, n in enumerate(lengths):
            for h in range(ref.heads):
                val, want_codes, want_scale = ref.values(name, b, h)
                assert torch.equal(got[b, h, n:], torch.zeros_like(got[b, h, n:]))
                full = n // 64 * 64
                torch.testing.assert_close(codes[b, h, :full], want_codes[:full], rtol=0, atol=0, equal_nan=True)
                assert torch.equal(scales[b, h, : full // 64], want_scale[:full:64])
                # the kernel's value is the fp32 product of code and scale
                want = (want_codes.float() * want_scale.float()[:, None]).to(torch.bfloat16)
                torch.testing.assert_close(got[b, h, :n], want, rtol=0, atol=0, equal_nan=True)


def _check_attention(cache, ref, lengths, s, hq, gen, as_int=False, weights=False, sm_scale=None, max_length=None, strided=True, finite=True):
    from minference_b200 import kv8_attention

    b, hkv = ref.batch, ref.heads
    q, dq = _rows(gen, b, hq, s)
    if not strided:
        dq = dq.contiguous()
    dev = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    kw = {}
    longest = max(lengths) if max_length is None else max_length
    if weights:
        before = torch.rand(b, hkv, cache.capacity, generator=gen)
        buf = before.cuda()
        kw = {"weights": buf, "add_to": buf}
    out, lse = kv8_attention(dq, cache, lengths[0] if as_int else dev, max_length=longest, sm_scale=sm_scale, return_lse=True, **kw)
    assert out.shape == (b, hq, s, 128) and out.dtype == torch.bfloat16 and lse.shape == (b, hq, s)
    out, lse = out.cpu().double(), lse.cpu().double()
    group = hq // hkv
    for i, n in enumerate(lengths):
        for h in range(hkv):
            total, tol_w = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
            for g in range(group):
                want, tol, want_lse, tol_lse, p, rel = R.attend(ref, q[i, h * group + g], i, h, sm_scale)
                got, got_lse = out[i, h * group + g], lse[i, h * group + g]
                if finite:
                    assert torch.isfinite(got).all()
                off = (got - want).abs() - tol
                assert not (off > 0).any(), (i, h, g, off.max().item(), tol.max().item())
                empty = want_lse == -math.inf
                assert torch.equal(got_lse[empty], want_lse[empty]) and torch.equal(got[empty], torch.zeros_like(got[empty]))
                assert ((got_lse[~empty] - want_lse[~empty]).abs() <= tol_lse[~empty]).all(), (got_lse, want_lse)
                total += p.sum(0)
                tol_w += (p * rel[:, None]).sum(0)
            if weights:
                got_w = buf[i, h].cpu().double()
                want_w = before[i, h, :n].double() + total
                # fp32: one rounding for each of the group * s sums, and the final one
                assert ((got_w[:n] - want_w).abs() <= tol_w + (group * s + 1) * 2.0 ** -24 * want_w).all()
                assert torch.equal(got_w[n:], before[i, h, n:].double())
    assert cache.status.tolist() == [0, 0, 0, 0]


# ------------------------------------------------------------------------------------------------- store and load


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("steps", [[1], [63], [64], [65], [1, 1, 1], [5, 58, 1, 1], [63, 2], [64, 64], [100, 1000, 27], [1, 200], [130, 0, 62, 65]])
def test_store_in_steps(kind, steps):
    from minference_b200 import kv8_store

    gen = torch.Generator().manual_seed(sum(steps))
    total = sum(steps)
    cache, ref = _poisoned(2, 3, total, kind), R.RefCache(2, 3, kind)
    at = 0
    for n in steps:
        k, dk = _rows(gen, 2, 3, n)
        v, dv = _rows(gen, 2, 3, n, 7.0)
        kv8_store(cache, dk, dv, at)
        ref.append(k, v)
        at += n
    _check_values(cache, ref, [total, total])
    assert cache.status.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("kind", KINDS)
def test_store_padded_batch_of_different_lengths(kind):
    from minference_b200 import kv8_store

    gen = torch.Generator().manual_seed(1)
    first = [0, 1, 63, 64, 130, 200]
    cache, ref = _filled(gen, 6, 2, first, kind, capacity=448)
    k, dk = _rows(gen, 6, 2, 190)
    v, dv = _rows(gen, 6, 2, 190)
    counts = torch.tensor([190, 63, 1, 0, 61, 190], dtype=torch.int32)
    kv8_store(cache, dk, dv, torch.tensor(first, dtype=torch.int32, device="cuda"), counts=counts.cuda())
    ref.append(k, v, counts)
    _check_values(cache, ref, [a + int(c) for a, c in zip(first, counts)])
    assert cache.status.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("kind", KINDS)
def test_store_touches_only_its_blocks(kind):
    from minference_b200 import KV8Cache, kv8_store

    gen = torch.Generator().manual_seed(2)
    cache = _poisoned(1, 2, 512, kind)
    names = ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail")
    before = {n: getattr(cache, n).view(torch.uint8).clone() for n in names}
    _, dk = _rows(gen, 1, 2, 100)
    kv8_store(cache, dk, dk, 150)                # tokens 150..249: completes block 2, leaves block 3 in the tail (rows 0..57)
    for n in names:
        now, was = getattr(cache, n).view(torch.uint8), before[n]
        if n in ("k", "v"):
            now, was = now.view(1, 2, 8, -1), was.view(1, 2, 8, -1)
            rest = [0, 1, 3, 4, 5, 6, 7]
            assert torch.equal(now[:, :, rest], was[:, :, rest]) and not torch.equal(now, was)
        elif n.endswith("scale"):
            now, was = now.view(1, 2, 8, 4), was.view(1, 2, 8, 4)
            assert torch.equal(now[:, :, [0, 1, 3, 4, 5, 6, 7]], was[:, :, [0, 1, 3, 4, 5, 6, 7]])
        else:
            now, was = now.view(1, 2, 64, -1), was.view(1, 2, 64, -1)
            assert torch.equal(now[:, :, 58:], was[:, :, 58:])
    assert isinstance(cache, KV8Cache)


@pytest.mark.parametrize("kind", KINDS)
def test_quantisation_at_its_edges(kind):
    """Blocks of zeros, of one value, of powers of two next to the largest code, of tiny and huge values, halves between two
    codes, infinities and NaN."""
    from minference_b200 import kv8_store

    blocks = []
    for fill in (0.0, -0.0, 1.0, 448.0, 450.0, 2.0 ** -126, 2.0 ** -133, 3e38, -127.0, 127.0 / 2 ** 20):
        blocks.append(torch.full((64, 128), fill))
    ramp = torch.linspace(-130, 130, 64 * 128).reshape(64, 128)
    halves = (torch.arange(64 * 128).reshape(64, 128) % 253 - 126) / 2.0
    halves[0, 0] = 127.0
    bad = torch.randn(64, 128, generator=torch.Generator().manual_seed(3))
    bad[3, 5], bad[7, 9], bad[60, 127] = NAN, math.inf, -math.inf
    only_bad = torch.full((64, 128), NAN)
    x = torch.stack(blocks + [ramp, halves, bad, only_bad]).reshape(1, 1, -1, 128).to(torch.bfloat16)
    n = x.shape[2]
    cache, ref = _poisoned(1, 1, n, kind), R.RefCache(1, 1, kind)
    kv8_store(cache, x.cuda(), x.flip(2).cuda(), 0)
    ref.append(x, x.flip(2))
    _check_values(cache, ref, [n])


def test_store_refuses_what_does_not_fit_on_the_device():
    from minference_b200 import KV8Cache, _cabi, kv8_load, kv8_store

    gen = torch.Generator().manual_seed(4)
    cache = KV8Cache.empty(5, 1, 128)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).zero_()
    cache.k_tail.zero_(), cache.v_tail.zero_(), cache.k_scale.fill_(1), cache.v_scale.fill_(1)
    _, dk = _rows(gen, 5, 1, 70)
    start = torch.tensor([60, 58, -1, 0, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    counts = torch.tensor([70, 70, 3, -4, 1], dtype=torch.int32, device="cuda")
    kv8_store(cache, dk, dk, start, counts=counts)
    k, _ = kv8_load(cache, 128)
    assert [bool(k[i].any()) for i in range(5)] == [False, True, False, False, False]
    with pytest.raises(_cabi.MInferB200Error, match="0x10"):
        cache.check()
    cache.check()                                # reported once
    with pytest.raises(_cabi.MInferB200Error):
        kv8_store(cache, dk, dk, 59)
    with pytest.raises(_cabi.MInferB200Error):
        kv8_store(cache, dk.float(), dk, 0)
    with pytest.raises(_cabi.MInferB200Error):
        kv8_store(cache, dk[:4], dk[:4], 0)
    with pytest.raises(_cabi.MInferB200Error):
        kv8_store(cache, dk, dk, start.long())
    assert torch.equal(kv8_load(cache, 128)[0], k)


@pytest.mark.parametrize("kind", KINDS)
def test_load_windows(kind):
    from minference_b200 import kv8_load

    gen = torch.Generator().manual_seed(5)
    lengths = [0, 1, 64, 150, 333]
    cache, _ = _filled(gen, 5, 2, lengths, kind, capacity=384)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    whole = torch.nn.functional.pad(kv8_load(cache, n)[0], (0, 0, 100, 100))
    first = torch.tensor([-100, 0, 17, 128, 320], dtype=torch.int32, device="cuda")
    part, _ = kv8_load(cache, n, first=first, count=101)
    for i, f in enumerate(first.tolist()):
        w = whole[i, :, f + 100: f + 201]
        assert torch.equal(part[i, :, : w.shape[1]], w) and not part[i, :, w.shape[1]:].any()
    assert kv8_load(cache, n, count=0)[0].shape == (5, 2, 0, 128)


# ------------------------------------------------------------------------------------------------------ attention


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 320, 1000, 4133])
def test_one_token_lengths(kind, n):
    gen = torch.Generator().manual_seed(n)
    cache, ref = _filled(gen, 1, 2, [n], kind, capacity=max(n, 64) + 128)
    _check_attention(cache, ref, [n], 1, 8, gen, as_int=True, weights=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq, hkv", [(1, 1), (3, 3), (8, 1), (6, 2), (7, 1), (16, 1), (18, 2), (40, 1)])
def test_head_layouts(kind, hq, hkv):
    gen = torch.Generator().manual_seed(hq)
    lengths = [300, 777, 64]
    cache, ref = _filled(gen, 3, hkv, lengths, kind)
    _check_attention(cache, ref, lengths, 1, hq, gen, weights=True, strided=hq % 2 == 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("s, hq, hkv", [(2, 4, 1), (5, 8, 2), (3, 2, 2), (16, 4, 2), (33, 2, 1), (64, 4, 1), (130, 2, 2)])
def test_several_tokens_are_causal(kind, s, hq, hkv):
    gen = torch.Generator().manual_seed(s)
    lengths = [s, s + 1, 700, max(s - 1, 0), 0, 64 + s // 2]
    cache, ref = _filled(gen, 6, hkv, lengths, kind)
    _check_attention(cache, ref, lengths, s, hq, gen, weights=True)


@pytest.mark.parametrize("kind", KINDS)
def test_ragged_batch_with_a_loose_bound(kind):
    gen = torch.Generator().manual_seed(6)
    lengths = [0, 1, 64, 1999, 2048, 77, 640, 1025]
    cache, ref = _filled(gen, 8, 2, lengths, kind, capacity=4096)
    for bound in (2048, 4096):
        _check_attention(cache, ref, lengths, 1, 8, gen, weights=True, max_length=bound)


@pytest.mark.parametrize("sm_scale", [0.0, 1.0, -0.3, 0.011])
def test_logit_scale(sm_scale):
    gen = torch.Generator().manual_seed(7)
    cache, ref = _filled(gen, 1, 1, [500], torch.int8)
    _check_attention(cache, ref, [500], 2, 4, gen, sm_scale=sm_scale)


@pytest.mark.parametrize("kind", KINDS)
def test_scales_that_differ_by_many_orders(kind):
    """Blocks whose values differ by 2^60, and the tokens with the largest weights in the blocks with the smallest values."""
    from minference_b200 import kv8_store

    gen = torch.Generator().manual_seed(8)
    n = 64 * 7 + 20
    cache, ref = _poisoned(1, 1, n, kind), R.RefCache(1, 1, kind)
    k, v = torch.randn(1, 1, n, 128, generator=gen), torch.randn(1, 1, n, 128, generator=gen)
    for i in range(8):
        v[:, :, 64 * i: 64 * i + 64] *= 2.0 ** (20 * ((i * 3) % 4) - 30)
        k[:, :, 64 * i: 64 * i + 64] *= 2.0 ** (-(i % 3))
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    kv8_store(cache, k.cuda(), v.cuda(), 0)
    ref.append(k, v)
    _check_attention(cache, ref, [n], 1, 8, gen, weights=True)


@pytest.mark.parametrize("kind", KINDS)
def test_queries_of_any_magnitude(kind):
    from minference_b200 import kv8_attention

    gen = torch.Generator().manual_seed(9)
    cache, ref = _filled(gen, 1, 1, [200], kind)
    mags = [0.0, 2.0 ** -60, 2.0 ** -20, 1.0, 2.0 ** 6, 2.0 ** 30, 2.0 ** -126, 3.0]
    q = (torch.randn(1, 8, 1, 128, generator=gen) * torch.tensor(mags)[None, :, None, None]).to(torch.bfloat16)
    scale = [0.05 / m if 2.0 ** -100 < m else 0.05 for m in mags]
    for i in range(8):
        out, lse = kv8_attention(q.cuda(), cache, 200, sm_scale=scale[i], return_lse=True)
        want, tol, want_lse, tol_lse, _, _ = R.attend(ref, q[0, i], 0, 0, scale[i])
        assert ((out[0, i].cpu().double() - want).abs() <= tol).all()
        assert ((lse[0, i].cpu().double() - want_lse).abs() <= tol_lse).all()


@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [128, 150])
def test_unseen_tokens_may_hold_anything(bad, kind, n):
    """The last of five new tokens has NaN or infinite keys and values: the queries before it do not notice."""
    from minference_b200 import kv8_attention, kv8_store

    gen = torch.Generator().manual_seed(10)
    k, _ = _rows(gen, 1, 2, n)
    v, _ = _rows(gen, 1, 2, n)
    clean = R.RefCache(1, 2, kind)
    if n % 64:                                   # in the tail: the clean sequence is what the earlier queries see
        clean.append(k, v)
        kb, vb = k.clone(), v.clone()
    else:                                        # in a complete block: its scale goes by the finite values
        kb, vb = k.clone(), v.clone()
        k, v = k.clone(), v.clone()
        k[:, :, -1], v[:, :, -1] = 0, 0
        clean.append(k, v)
    kb[:, :, -1], vb[:, :, -1] = bad, bad
    cache = _poisoned(1, 2, n, kind)
    kv8_store(cache, kb.cuda(), vb.cuda(), 0)
    q, dq = _rows(gen, 1, 8, 5)
    out = kv8_attention(dq, cache, n).cpu().double()
    for h in range(8):
        want, tol, *_ = R.attend(clean, q[0, h], 0, h // 4)
        assert ((out[0, h, :4] - want[:4]).abs() <= tol[:4]).all(), h


def test_non_finite_values_that_are_seen_show():
    from minference_b200 import kv8_attention, kv8_store

    gen = torch.Generator().manual_seed(11)
    k, dk = _rows(gen, 1, 1, 100)
    v, dv = _rows(gen, 1, 1, 100)
    dv = dv.clone()
    dv[:, :, 70, 3] = NAN
    cache = _poisoned(1, 1, 128, torch.float8_e4m3fn)
    kv8_store(cache, dk, dv, 0)
    out = kv8_attention(_rows(gen, 1, 4, 1)[1], cache, 100)
    assert out[..., 3].isnan().all() and torch.isfinite(out[..., :3]).all() and torch.isfinite(out[..., 4:]).all()
    q = torch.full((1, 4, 1, 128), NAN, dtype=torch.bfloat16, device="cuda")
    out, lse = kv8_attention(q, cache, 100, return_lse=True)
    assert out.isnan().all() and lse.isnan().all()


def test_weights_views_and_separate_sum():
    from minference_b200 import kv8_attention

    gen = torch.Generator().manual_seed(12)
    cache, _ = _filled(gen, 2, 2, [130, 90], torch.float8_e4m3fn)
    _, dq = _rows(gen, 2, 4, 1)
    n = torch.tensor([130, 90], dtype=torch.int32, device="cuda")
    plain = torch.zeros(2, 2, 192, device="cuda")
    kv8_attention(dq, cache, n, max_length=130, weights=plain)
    base = torch.rand(2, 2, 192, device="cuda")
    wide = torch.full((2, 4, 400), -5.0, device="cuda")
    view = wide[:, ::2, 7:199]
    kv8_attention(dq, cache, n, max_length=130, weights=view, add_to=base)
    for i, m in enumerate((130, 90)):
        assert torch.equal(view[i, :, :m], (plain + base)[i, :, :m]) and (view[i, :, m:] == -5.0).all()
    assert (wide[:, 1::2] == -5.0).all()
    assert torch.allclose(plain.sum(-1), torch.full((2, 2), 2.0, device="cuda"), atol=1e-5)      # two query heads a head


def test_attention_is_the_same_every_time():
    from minference_b200 import kv8_attention

    gen = torch.Generator().manual_seed(13)
    cache, _ = _filled(gen, 2, 2, [5000, 3333], torch.int8)
    _, dq = _rows(gen, 2, 8, 1)
    n = torch.tensor([5000, 3333], dtype=torch.int32, device="cuda")
    w = [torch.zeros(2, 2, cache.capacity, device="cuda") for _ in range(2)]
    outs = [kv8_attention(dq, cache, n, weights=x, return_lse=True) for x in w]
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1]) and torch.equal(w[0], w[1])


def test_attention_clips_lengths_on_the_device():
    from minference_b200 import _cabi, kv8_attention

    gen = torch.Generator().manual_seed(14)
    cache, ref = _filled(gen, 3, 1, [192, 192, 192], torch.float8_e4m3fn)
    _, dq = _rows(gen, 3, 2, 1)
    n = torch.tensor([1 << 30, -7, 192], dtype=torch.int32, device="cuda")
    out = kv8_attention(dq, cache, n)
    full = kv8_attention(dq, cache, 192)
    assert torch.equal(out[0], full[0]) and torch.equal(out[2], full[2]) and not out[1].any()
    with pytest.raises(_cabi.MInferB200Error, match="0x10"):
        cache.check()


def test_python_refusals():
    from minference_b200 import KV8Cache, _cabi, kv8_attention, kv8_evict, kv8_load

    cache = KV8Cache.empty(2, 2, 128)
    q = torch.zeros(2, 4, 1, 128, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(2, 2, 128, device="cuda")
    bad = [lambda: kv8_attention(q[:1], cache, 1), lambda: kv8_attention(q.half(), cache, 1), lambda: kv8_attention(q[:, :3], cache, 1),
           lambda: kv8_attention(q[..., :64], cache, 1), lambda: kv8_attention(q, cache, 129), lambda: kv8_attention(q, cache, -1),
           lambda: kv8_attention(q, cache, 5, max_length=4), lambda: kv8_attention(q, cache, 5, max_length=200),
           lambda: kv8_attention(q, cache, 5, add_to=w), lambda: kv8_attention(q, cache, 100, weights=w[..., :99]),
           lambda: kv8_attention(q, cache, 5, weights=w.double()), lambda: kv8_attention(q, cache, 5, weights=w.transpose(1, 2)),
           lambda: kv8_attention(q, cache, 5, weights=w[:1].expand(2, 2, 128)), lambda: kv8_attention(q, cache, 5, weights=w[:, :1].expand(2, 2, 128)),
           lambda: kv8_attention(q, cache, 5, max_length=100, weights=w[..., :100], add_to=w[..., 10:110]),
           lambda: kv8_attention(q.cpu(), cache, 1), lambda: kv8_attention(q[:, :, :0], cache, 1),
           lambda: kv8_attention(q, cache, torch.tensor([1, 1], dtype=torch.int32)), lambda: kv8_load(cache, 129), lambda: kv8_load(cache, 1, count=-1),
           lambda: kv8_evict(cache, 128, w, 0, recent=0), lambda: kv8_evict(cache, 128, w, 8, recent=6, sink=3),
           lambda: kv8_evict(cache, 128, w, 8, recent=2, out=cache), lambda: kv8_evict(cache, 128, w[..., :100], 8, recent=2),
           lambda: kv8_evict(cache, 128, w, 100, recent=2, out=KV8Cache.empty(2, 2, 64)),
           lambda: kv8_evict(cache, 128, w, 8, recent=2, out=KV8Cache.empty(2, 2, 64, torch.int8)),
           lambda: KV8Cache.empty(1, 1, 64, torch.float16), lambda: KV8Cache.empty(1, 0, 64), lambda: KV8Cache.empty(1, 1, 0),
           lambda: KV8Cache(cache.k[:, :, :100], cache.v, cache.k_scale, cache.v_scale, cache.k_tail, cache.v_tail),
           lambda: KV8Cache(cache.k, cache.v, cache.k_scale[..., :1], cache.v_scale, cache.k_tail, cache.v_tail),
           lambda: KV8Cache(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_tail.half(), cache.v_tail)]
    for i, call in enumerate(bad):
        with pytest.raises(_cabi.MInferB200Error):
            call()
            pytest.fail(f"call {i} was taken")
    cache.check()


def test_offsets_beyond_32_bits():
    """A cache whose codes pass 2^31 bytes, filled at its end only: the last head's last tokens."""
    from minference_b200 import KV8Cache, kv8_attention, kv8_load, kv8_store

    gen = torch.Generator().manual_seed(15)
    heads, cap = 9, 2 * 1024 * 1024                          # 9 * 2M * 128 = 2.4e9 bytes of keys
    cache = KV8Cache.empty(1, heads, cap)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).zero_()
    cache.k_scale.fill_(1), cache.v_scale.fill_(1)
    cache.k_tail.zero_(), cache.v_tail.zero_()               # the 56 tokens before the new ones, in the block they complete
    k, dk = _rows(gen, 1, heads, 200)
    v, dv = _rows(gen, 1, heads, 200)
    kv8_store(cache, dk * 4, dv, cap - 200)
    ref = R.RefCache(1, heads, torch.float8_e4m3fn)
    ref.append((k * 4)[:, :, 8:], v[:, :, 8:])               # three whole blocks; the 8 tokens before them pass unchecked
    lk, lv = kv8_load(cache, cap, first=cap - 192, count=192)
    assert torch.equal(lk.cpu()[0, 8].double(), ref.values("k", 0, 8)[0]) and torch.equal(lv.cpu()[0, 8].double(), ref.values("v", 0, 8)[0])
    # keys of zeros elsewhere: their logits are 0, the last tokens' far above once the query points at one of them
    q = (lk[:, :, -1:] * 8).contiguous()
    w = torch.zeros(1, heads, cap, device="cuda")
    out = kv8_attention(q, cache, cap, weights=w)
    for h in range(heads):
        assert torch.equal(out[0, h, 0], lv[0, h, -1]) and abs(w[0, h, -1].item() - 1) < 1e-6, h


# ------------------------------------------------------------------------------------------------------- eviction


def _check_evict(cache, ref, weights, lengths, budget, recent, sink, **kw):
    from minference_b200 import kv8_evict

    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    small, new_lengths, new_weights, kept = kv8_evict(cache, n, weights.cuda(), budget, recent=recent, sink=sink, **kw)
    want = ref.evict(weights, budget, recent, sink)
    held = [min(m, budget) for m in lengths]
    assert new_lengths.tolist() == held and kept.shape == (ref.batch, ref.heads, budget) and new_weights.shape[2] == small.capacity
    for b in range(ref.batch):
        for h in range(ref.heads):
            got = kept[b, h].tolist()
            assert got[: held[b]] == want[b][h] and all(x == -1 for x in got[held[b]:]), (b, h)
            w = new_weights[b, h].cpu()
            torch.testing.assert_close(w[: held[b]], weights[b, h][want[b][h]].float(), rtol=0, atol=0, equal_nan=True)
            assert not w[held[b]:].any()
    _check_values(small, ref, held)
    assert cache.status.tolist() == [0, 0, 0, 0] and small.status.tolist() == [0, 0, 0, 0]
    return small, held


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lengths, budget, recent, sink", [
    ([300], 100, 30, 4), ([300], 128, 128, 0), ([300], 64, 0, 64), ([300], 70, 60, 10), ([65], 64, 1, 0), ([1], 1, 0, 0), ([2], 1, 0, 0),
    ([0, 1, 99, 100, 101, 500], 100, 25, 4), ([3000, 2049], 1001, 250, 4), ([5000], 4999, 10, 10), ([1025, 1024], 1, 0, 0)])
def test_evict(kind, lengths, budget, recent, sink):
    gen = torch.Generator().manual_seed(budget)
    cache, ref = _filled(gen, len(lengths), 2, lengths, kind, capacity=max(max(lengths), budget))
    weights = torch.exp(2 * torch.randn(len(lengths), 2, cache.capacity, generator=gen))
    _check_evict(cache, ref, weights, lengths, budget, recent, sink)


@pytest.mark.parametrize("case", ["all equal", "few values", "zeros", "negative", "signed zeros", "nan and inf", "subnormal", "one bit apart"])
def test_evict_ties_and_odd_weights(case):
    gen = torch.Generator().manual_seed(20)
    n = 2500
    w = {"all equal": torch.full((n,), 0.25), "few values": torch.randint(0, 3, (n,), generator=gen).float(),
         "zeros": (torch.rand(n, generator=gen) < 0.02).float(), "negative": -torch.rand(n, generator=gen),
         "signed zeros": torch.zeros(n) * (torch.randint(0, 2, (n,), generator=gen) * 2 - 1),
         "nan and inf": torch.randn(n, generator=gen), "subnormal": torch.randint(0, 500, (n,), generator=gen).float() * 2.0 ** -149,
         "one bit apart": 1 + torch.randint(0, 300, (n,), generator=gen).float() * 2.0 ** -23}[case]
    if case == "nan and inf":
        w[torch.randperm(n, generator=gen)[:300]] = NAN
        w[torch.randperm(n, generator=gen)[:900]] = math.inf
        w[torch.randperm(n, generator=gen)[:300]] = -math.inf
    cache, ref = _filled(gen, 1, 2, [n], torch.float8_e4m3fn)
    weights = torch.stack((w, w.flip(0)))[None].expand(1, 2, n)
    weights = torch.nn.functional.pad(weights, (0, cache.capacity - n), value=1e30)       # behind the last token: not looked at
    for budget in (777, 640):
        _check_evict(cache, R_copy(ref), weights, [n], budget, 100, 3)


@pytest.mark.parametrize("kind", KINDS)
def test_evict_values_at_their_edges(kind):
    """Requantising blocks that mix zeros, the tiniest and the largest values (e4m3's largest code overflows fp32 there), halves
    between two codes, infinities and NaN."""
    from minference_b200 import kv8_store

    gen = torch.Generator().manual_seed(22)
    parts = [torch.full((64, 128), f) for f in (0.0, 448.0, 2.0 ** -133, 3e38, 3.3895e38, -127.0)]
    halves = (torch.arange(64 * 128).reshape(64, 128) % 253 - 126) / 2.0
    bad = torch.randn(64, 128, generator=gen)
    bad[3, 5], bad[7, 9], bad[60, 127] = NAN, math.inf, -math.inf
    x = torch.stack(parts + [halves, bad, torch.full((64, 128), NAN), torch.randn(64, 128, generator=gen)]).reshape(1, 1, -1, 128).to(torch.bfloat16)
    x = torch.cat((x, x[:, :, 300:333]), 2)
    n = x.shape[2]
    cache, ref = _poisoned(1, 1, n, kind), R.RefCache(1, 1, kind)
    kv8_store(cache, x.cuda(), x.flip(2).cuda(), 0)
    ref.append(x, x.flip(2))
    for budget in (n, 513, 200):
        weights = torch.rand(1, 1, cache.capacity, generator=gen)
        _check_evict(cache, R_copy(ref), weights, [n], budget, 20, 3)


def R_copy(ref):
    new = R.RefCache(ref.batch, ref.heads, ref.kind)
    new.raw = {n: [list(x) for x in t] for n, t in ref.raw.items()}
    return new


def test_evict_with_a_bound_a_view_and_a_larger_cache():
    from minference_b200 import KV8Cache

    gen = torch.Generator().manual_seed(21)
    lengths = [400, 333]
    cache, ref = _filled(gen, 2, 2, lengths, torch.int8, capacity=1024)
    wide = torch.rand(2, 5, 900, generator=gen)
    weights = wide[:, 1:5:2, 100:]
    out = _poisoned(2, 2, 512, torch.int8)
    small, held = _check_evict(cache, ref, weights, lengths, 150, 20, 4, max_length=400, out=out)
    assert small is out and isinstance(out, KV8Cache) and out.capacity == 512


# ------------------------------------------------------------------------------------------------- used together


@pytest.mark.parametrize("kind", KINDS)
def test_prompt_decode_evict_decode(kind):
    """A prompt is stored, tokens are decoded with their weights summed up, the cache is cut down, decoding goes on."""
    from minference_b200 import KV8Cache, kv8_attention, kv8_store

    gen = torch.Generator().manual_seed(30)
    b, hkv, hq = 2, 2, 8
    lengths = [500, 413]
    cache, ref = _filled(gen, b, hkv, lengths, kind, capacity=640)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    sums = torch.zeros(b, hkv, cache.capacity, device="cuda")
    want_sums = torch.zeros(b, hkv, cache.capacity, dtype=torch.float64)

    def step(cache, ref, n, lengths, sums, want_sums):
        k, dk = _rows(gen, b, hkv, 1)
        v, dv = _rows(gen, b, hkv, 1)
        q, dq = _rows(gen, b, hq, 1)
        kv8_store(cache, dk, dv, n)
        ref.append(k, v)
        n += 1
        out = kv8_attention(dq, cache, n, weights=sums, add_to=sums)
        lengths = [x + 1 for x in lengths]
        for i in range(b):
            for h in range(hq):
                want, tol, _, _, p, _ = R.attend(ref, q[i, h], i, h // 4)
                assert ((out[i, h].cpu().double() - want).abs() <= tol).all()
                want_sums[i, h // 4, : lengths[i]] += p.sum(0)
        return lengths

    for _ in range(70):                          # across a block's end
        lengths = step(cache, ref, n, lengths, sums, want_sums)
    assert torch.allclose(sums.cpu().double(), want_sums, rtol=1e-4, atol=1e-6)
    small, lengths = _check_evict(cache, ref, sums.cpu(), lengths, 200, 64, 4, out=KV8Cache.empty(b, hkv, 320, kind))
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    sums, want_sums = torch.zeros(b, hkv, 320, device="cuda"), torch.zeros(b, hkv, 320, dtype=torch.float64)
    for _ in range(60):
        lengths = step(small, ref, n, lengths, sums, want_sums)
    cache.check(), small.check()


def test_decoding_step_in_a_cuda_graph():
    """One captured step (store, attention with weights) replayed for growing lengths equals the eager steps; two graphs over
    one cache do not disturb each other."""
    from minference_b200 import kv8_attention, kv8_store

    gen = torch.Generator().manual_seed(31)
    steps = [[_rows(gen, 2, h, 1)[1].contiguous() for h in (2, 2, 8)] for _ in range(6)]

    def fresh():
        g = torch.Generator().manual_seed(32)
        cache, _ = _filled(g, 2, 2, [125, 60], torch.float8_e4m3fn, capacity=256)
        return cache, torch.tensor([125, 60], dtype=torch.int32, device="cuda"), torch.zeros(2, 2, 256, device="cuda")

    cache, n, sums = fresh()
    eager = []
    for k, v, q in steps:
        kv8_store(cache, k, v, n)
        n += 1
        eager.append(kv8_attention(q, cache, n, weights=sums, add_to=sums).clone())
    want_sums = sums
    cache, n, sums = fresh()
    k, v, q = [torch.empty_like(t) for t in steps[0]]
    graphs = []
    for _ in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            kv8_store(cache, k, v, n)
            n += 1
            out = kv8_attention(q, cache, n, weights=sums, add_to=sums)
        graphs.append((g, out))
    for i, (sk, sv, sq) in enumerate(steps):
        k.copy_(sk), v.copy_(sv), q.copy_(sq)
        g, out = graphs[i % 2]
        g.replay()
        assert torch.equal(out, eager[i]), i
    assert torch.equal(sums, want_sums) and n.tolist() == [131, 66]
    cache.check()


def test_on_another_stream():
    from minference_b200 import kv8_attention, kv8_evict, kv8_load, kv8_store

    gen = torch.Generator().manual_seed(33)
    _, dk = _rows(gen, 1, 2, 1000)
    _, dq = _rows(gen, 1, 8, 1)
    results = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            cache = _poisoned(1, 2, 1024, torch.int8)
            kv8_store(cache, dk, dk, 0)
            w = torch.zeros(1, 2, 1024, device="cuda")
            out = kv8_attention(dq, cache, 1000, weights=w)
            small, n, w2, kept = kv8_evict(cache, 1000, w, 333, recent=50)
            results.append((out, w[..., :1000], w2, kept, *kv8_load(small, n, count=333)))
        stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("kind", KINDS)
def test_many_sequences(kind):
    """More sequences than a warp has lanes, lengths of every sort among them, in the narrow and the wide kernel."""
    gen = torch.Generator().manual_seed(41)
    lengths = [(37 * i * i) % 500 for i in range(70)]
    lengths[3] = lengths[32] = lengths[33] = lengths[69] = 0
    lengths[31], lengths[64] = 6000, 4999
    cache, ref = _filled(gen, 70, 1, lengths, kind)
    _check_attention(cache, ref, lengths, 1, 4, gen, weights=True)
    _check_attention(cache, ref, lengths, 5, 4, gen)
    _check_attention(cache, ref, lengths, 33, 1, gen, weights=True)
    same = [1000] * 40
    cache, ref = _filled(gen, 40, 2, same, kind)
    _check_attention(cache, ref, same, 1, 4, gen)
    _check_attention(cache, ref, same, 1, 4, gen, as_int=True, weights=True)


@pytest.mark.parametrize("s, hq", [(1, 4), (5, 8), (40, 2)])
def test_one_length_for_a_batch(s, hq):
    gen = torch.Generator().manual_seed(42)
    cache, ref = _filled(gen, 3, 2, [3011] * 3, torch.float8_e4m3fn)
    _check_attention(cache, ref, [3011] * 3, s, hq, gen, as_int=True, weights=True)
    _check_attention(cache, ref, [3011] * 3, s, hq, gen, as_int=True, max_length=3050)


def test_only_empty_sequences():
    from minference_b200 import kv8_attention, kv8_evict

    gen = torch.Generator().manual_seed(43)
    cache = _poisoned(2, 2, 2048, torch.float8_e4m3fn)
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    for s in (1, 5, 64):
        _, dq = _rows(gen, 2, 4, s)
        w = torch.full((2, 2, 2048), -3.0, device="cuda")
        for lengths in (n, 0):
            out, lse = kv8_attention(dq, cache, lengths, max_length=2048, weights=w, return_lse=True)
            assert not out.any() and (lse == -math.inf).all() and (w == -3.0).all()
    small, m, w2, kept = kv8_evict(cache, n, torch.full((2, 2, 2048), NAN, device="cuda"), 100, recent=10)
    assert m.tolist() == [0, 0] and not w2.any() and (kept == -1).all()
    cache.check()


def test_misaligned_inputs():
    from minference_b200 import KV8Cache, kv8_attention, kv8_load, kv8_store

    gen = torch.Generator().manual_seed(44)
    raw = torch.randn(2 * 300 * 128 + 1, generator=gen).to(torch.bfloat16).cuda()
    k = raw[1:].view(1, 2, 300, 128)
    q = raw[1:1 + 8 * 128].view(1, 8, 1, 128)
    assert k.is_contiguous() and k.data_ptr() % 16 and q.data_ptr() % 16
    outs = []
    for kk, qq in ((k, q), (k.clone(), q.clone())):
        cache = KV8Cache.empty(1, 2, 300)
        kv8_store(cache, kk, kk, 0)
        outs.append((*kv8_load(cache, 300), kv8_attention(qq, cache, 300)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("s, hq", [(1, 8), (40, 8)])
def test_attention_and_eviction_in_a_cuda_graph(s, hq):
    """Captured attention of either kernel with weights, and the eviction behind it, replayed for other lengths."""
    from minference_b200 import KV8Cache, kv8_attention, kv8_evict, kv8_load

    gen = torch.Generator().manual_seed(45)
    cache, _ = _filled(gen, 2, 2, [4096, 4096], torch.int8)
    _, dq = _rows(gen, 2, hq, s)
    n = torch.tensor([4096, 4096], dtype=torch.int32, device="cuda")
    out_cache = KV8Cache.empty(2, 2, 700, torch.int8)

    def step():
        w = torch.zeros(2, 2, 4096, device="cuda")
        out = kv8_attention(dq, cache, n, max_length=4096, weights=w)
        small, m, w2, kept = kv8_evict(cache, n, w, 700, recent=64, sink=4, max_length=4096, out=out_cache)
        return out, w, m, w2, kept, *kv8_load(small, m)

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        got = step()
    # lengths inside a block read a tail that holds another block's tokens, here NaN: the same numbers all the same
    for lengths in ([4096, 4096], [2944, 704], [0, 64], [3001, 701], [777, 2222]):
        n.copy_(torch.tensor(lengths, dtype=torch.int32))
        want = [t.clone() for t in step()]
        for t in got[:2]:
            t.zero_()
        out_cache.k.view(torch.uint8).zero_(), out_cache.v_tail.zero_()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            torch.testing.assert_close(a, b, rtol=0, atol=0, equal_nan=True)
    cache.check()


@pytest.mark.parametrize("s", [1, 40])
def test_two_streams_read_one_cache(s):
    """Calls that overlap in time share no scratch memory."""
    from minference_b200 import kv8_attention

    gen = torch.Generator().manual_seed(46)
    cache, _ = _filled(gen, 2, 4, [9000, 7000], torch.float8_e4m3fn)
    n = torch.tensor([9000, 7000], dtype=torch.int32, device="cuda")
    qs = [_rows(gen, 2, 8, s)[1] for _ in range(2)]
    new = lambda: torch.zeros(2, 4, cache.capacity, device="cuda")
    want = []
    for q in qs:
        w = new()
        want.append((kv8_attention(q, cache, n, weights=w), w))
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                w = new()
                got[i].append((kv8_attention(qs[i], cache, n, weights=w), w))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for pair in got[i] for a, b in zip(pair, want[i]))


@pytest.mark.parametrize("s, hq, hkv, n", [(1, 4, 2, 700), (3, 4, 2, 9000), (40, 4, 2, 300)])
def test_query_and_output_layouts(s, hq, hkv, n):
    """Queries sliced out of a joint projection, head-major, with gaps, and expanded over the batch give the same numbers."""
    from minference_b200 import kv8_attention

    gen = torch.Generator().manual_seed(47)
    cache, _ = _filled(gen, 2, hkv, [n, n], torch.float8_e4m3fn)
    joint = torch.randn(2, s, hq + 2 * hkv, 128, generator=gen).to(torch.bfloat16).cuda()
    q = joint[:, :, :hq].transpose(1, 2)
    plain = q.contiguous()
    want = kv8_attention(plain, cache, n)
    assert want.is_contiguous() and want.shape == (2, hq, s, 128)
    gaps = torch.zeros(2, hq, 2 * s, 136, dtype=torch.bfloat16, device="cuda")[:, :, ::2, :128]
    gaps.copy_(plain)
    for x in (q, gaps, plain.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(kv8_attention(x, cache, n), want)
    one = plain[:1].expand(2, hq, s, 128)
    assert torch.equal(kv8_attention(one, cache, n), kv8_attention(one.contiguous(), cache, n))
