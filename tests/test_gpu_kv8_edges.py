"""Attention over the 8-bit cache and the layer around it where a wrong rounding, padding or unit of weights would show, against
the definition in 64 bits (tests/kv8_reference.py)."""
import math

import pytest
import torch

from tests import kv8_reference as R
from tests.test_gpu_kv8 import KINDS, _check_attention, _filled, _poisoned, _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gap", [20, 24, 26])
@pytest.mark.parametrize("s, hq", [(1, 4), (1, 12), (1, 24), (1, 25), (40, 2)])
def test_many_weak_tokens_behind_a_strong_one_of_no_value(kind, gap, s, hq):
    """One token of 32 has a logit ``gap`` bits above the others and a value of zero: the output is the weak tokens' alone.
    Their numerators are rounded to f16 relative to the largest, which is 2^7 at least: half a step is 2^-11 of a normal
    number and 2^-25 of the smallest ones, 2^-32 of the largest numerator -- 2^(gap - 32) of a weak one, however many there are."""
    from minference_b200 import kv8_attention, kv8_store

    gen = torch.Generator().manual_seed(gap + s)
    n = 2048
    k, v = torch.zeros(1, 1, n, 128), 1 + 0.1 * torch.rand(1, 1, n, 128, generator=gen)
    k[..., 0] = torch.randn(n, generator=gen)
    k[:, :, ::32, 0] = gap
    v[:, :, ::32] = 0
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    cache, ref = _poisoned(1, 1, n, kind), R.RefCache(1, 1, kind)
    kv8_store(cache, k.cuda(), v.cuda(), 0)
    ref.append(k, v)
    q = torch.zeros(1, hq, s, 128, dtype=torch.bfloat16)
    q[..., 0] = 1
    scale = math.log(2)                          # logits of k[..., 0] bits
    out = kv8_attention(q.cuda(), cache, n, sm_scale=scale).cpu().double()
    _, codes, sv = ref.values("v", 0, 0)
    for h in range(hq):
        want, _, _, _, p, rel = R.attend(ref, q[0, h], 0, 0, scale)
        half_steps = 2.0 ** -32 * (p * sv).amax(-1)[:, None] * codes.abs().sum(0)
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + rel[:, None]) * want.abs() + half_steps        # (no value is negative)
        assert (half_steps <= 2.0 ** (gap - 30) * want).all()
        off = (out[0, h] - want).abs()
        assert (off <= tol).all(), (h, (off / want).max().item(), (tol / want).max().item())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [100, 1000, 20001])
@pytest.mark.parametrize("hq", [1, 2, 3, 5, 6, 7, 11, 23, 25, 30])
def test_weights_next_to_an_infinite_key(kind, n, hq):
    """A key of -inf that every head's logit goes to -inf with: its weight is zero, whatever the padding columns of the heads
    (zero times that key) hold."""
    from minference_b200 import kv8_attention, kv8_store

    gen = torch.Generator().manual_seed(n + hq)
    k, _ = _rows(gen, 1, 1, n)
    v, dv = _rows(gen, 1, 1, n)
    q, _ = _rows(gen, 1, hq, 1)
    k[:, :, -2], q[..., 0] = 0, 1
    k[:, :, -2, 0] = -math.inf                   # in the tail: those blocks keep infinities
    cache = _poisoned(1, 1, n, kind)
    kv8_store(cache, k.cuda(), dv, 0)
    w = torch.zeros(1, 1, cache.capacity, device="cuda")
    out, lse = kv8_attention(q.cuda(), cache, n, weights=w, return_lse=True)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    w = w[0, 0].cpu().double()
    assert torch.isfinite(w).all() and w[n - 2] == 0 and not w[n:].any()
    assert abs(w.sum().item() - hq) <= 1e-5 * hq


def _layer_with(gen, n, hq, hkv, kind, **options):
    """(KV8Layer holding n tokens, queries, keys on the GPU; queries on the CPU, its definition)."""
    from minference_b200 import KV8Layer

    kv, ref = KV8Layer(kind, **options), R.RefCache(1, hkv, kind)
    k, dk = _rows(gen, 1, hkv, n)
    v, dv = _rows(gen, 1, hkv, n)
    q, dq = _rows(gen, 1, hq, n)
    kv.append(dk, dv)
    ref.append(k, v)
    return kv, dq, dk, dv, q, ref


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 50, 64, 300])
@pytest.mark.parametrize("scaling", [1 / 128, 0.25, None])
def test_a_prompts_weights_are_those_of_the_models_scaling(kind, n, scaling):
    """The patched attention function hands a prompt's weights on with the scale the model uses: the probabilities of its last
    64 queries."""
    from types import SimpleNamespace

    from minference_b200 import MInferenceConfig
    from minference_b200.patch import _make_attention_function

    gen = torch.Generator().manual_seed(n)
    hq, hkv = 4, 2
    kv, dq, dk, dv, q, ref = _layer_with(gen, n, hq, hkv, kind, budget=400, slack=50)
    key = dk.view(dk.shape)
    key.minf_kv8 = kv
    module = SimpleNamespace(layer_idx=0, config=SimpleNamespace(num_hidden_layers=1), num_key_value_groups=hq // hkv, is_causal=True, training=False)
    _make_attention_function(MInferenceConfig(attn_type="dense"))(module, dq, key, dv, scaling=scaling)
    assert kv.held == n
    for h in range(hkv):
        want, tol = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
        for g in range(hq // hkv):
            _, _, _, _, p, rel = R.attend(ref, q[0, h * (hq // hkv) + g, -64:], 0, h, scaling)
            want += p.sum(0)
            tol += (p * rel[:, None]).sum(0)
        got = kv.sums[0, h, :n].cpu().double()
        if scaling is None:
            # the estimator's scores, of keys in bf16 and logits rounded to bf16 twice, stay as they were: no more than their sum here
            assert abs(got.sum() - want.sum()) <= 2.0 ** -7 * want.sum()
        else:
            assert ((got - want).abs() <= tol + (hq // hkv * 64 + 1) * 2.0 ** -24 * want).all(), (got - want).abs().max()
    assert not kv.sums[..., n:].any()


def test_eviction_of_a_prompt_goes_by_the_models_scaling():
    """A scale of zero makes all tokens a query sees alike: the earliest are kept, whatever the keys are."""
    gen = torch.Generator().manual_seed(8)
    kv, dq, dk, _, _, _ = _layer_with(gen, 500, 4, 2, torch.int8, budget=128, recent=16, sink=4)
    kv.after_prompt(dq, dk, 0.0)
    assert kv.held == 128
    w = kv.sums[0, :, :112]                      # the sink and the earliest: each of 2 x 64 queries sees them among 437 to 500 tokens
    want = 2 * (1 / torch.arange(437.0, 501.0).double()).sum().item()
    assert ((w.double() - want).abs() <= 2.0 ** -15 * want).all()


@pytest.mark.parametrize("new", [64, 65, 700])
def test_a_long_follow_up_adds_the_weights_of_its_last_queries(new):
    """As a prompt does, and in memory that does not grow with the new tokens times those held."""
    from minference_b200 import KV8Layer, kv8_attention

    gen = torch.Generator().manual_seed(new)
    kv = KV8Layer(torch.int8, budget=256, slack=4096)
    kv.append(_rows(gen, 1, 2, 300)[1], _rows(gen, 1, 2, 300)[1])
    kv.sums[..., :300] = torch.rand(1, 2, 300, generator=gen).cuda()
    before = kv.sums.clone()
    kv.append(_rows(gen, 1, 2, new)[1], _rows(gen, 1, 2, new)[1])
    _, dq = _rows(gen, 1, 8, new)
    out = kv.attend(dq)
    n = 300 + new
    assert kv.held == n and torch.equal(out, kv8_attention(dq, kv.cache, n))
    want = torch.zeros_like(kv.sums)
    want[..., :300] = before[..., :300]
    kv8_attention(dq[:, :, -64:], kv.cache, n, weights=want, add_to=want)
    assert torch.equal(kv.sums[..., :n], want[..., :n]) and not kv.sums[..., n:].any()


def test_a_long_follow_up_under_a_budget_needs_little_memory():
    from minference_b200 import KV8Layer

    kv = KV8Layer(budget=512, slack=64)
    rows = lambda h, n: torch.randn(1, h, n, 128, dtype=torch.bfloat16, device="cuda")
    kv.append(rows(8, 500), rows(8, 500))
    k, v, q = rows(8, 4096), rows(8, 4096), rows(32, 4096)
    kv.append(k, v)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    out = kv.attend(q)
    torch.cuda.synchronize()
    # 33.5 MB of output; logits of 64 queries of 32 heads over 4596 tokens, 38 MB; parts of 64 x 32 rows and of all rows where
    # they are split (of 148 CTAs with 128 rows of 512 bytes at most): 10 MB each.  All rows' logits would be 2.4 GB
    assert torch.cuda.max_memory_allocated() - base <= 128 << 20
    assert kv.held == 512 and torch.isfinite(out).all()


@pytest.mark.parametrize("how", ["evict", "grow"])
def test_what_the_device_reported_outlives_the_layers_cache(how):
    """A layer that cuts its cache down, or moves to a larger one, goes on reporting what happened before."""
    from minference_b200 import KV8Layer, _cabi
    from minference_b200._cabi import MInferB200Error

    gen = torch.Generator().manual_seed(10)
    kv = KV8Layer(budget=100, slack=10)
    kv.append(_rows(gen, 1, 2, 105)[1], _rows(gen, 1, 2, 105)[1])
    kv.cache.status[_cabi.ST_ERROR] = 1          # as an abandoned wait leaves it
    old = kv.cache
    if how == "evict":
        kv.evict()
    else:
        kv.append(_rows(gen, 1, 2, 5000)[1], _rows(gen, 1, 2, 5000)[1])
    assert kv.cache is not old
    with pytest.raises(MInferB200Error, match="0x1 "):
        kv.cache.check()
    kv.cache.check()


def test_every_exponent_of_an_e4m3_scale():
    """Blocks whose largest value is 448 * 2^p or next to it, for every p that a scale may take: scales are 2^p to the bit."""
    from minference_b200 import kv8_store

    cache = _poisoned(1, 1, 64 * 440, torch.float8_e4m3fn)
    p = torch.arange(-100, 120, dtype=torch.float64)
    tops = torch.stack((448 * torch.exp2(p), 450 * torch.exp2(p - 1)), 1).flatten()      # (450 = 448 + one bf16 step)
    x = torch.zeros(1, 1, 440, 64, 128)
    x[0, 0, :, 5, 7] = -tops.float()
    x = x.view(1, 1, -1, 128).to(torch.bfloat16).cuda()
    kv8_store(cache, x, x, 0)
    want = torch.exp2(p).repeat_interleave(2).float().clone()
    assert torch.equal(cache.k_scale.cpu().flatten(), want) and torch.equal(cache.v_scale.cpu().flatten(), want)


@pytest.mark.parametrize("s, hq", [(1, 4), (40, 2)])
def test_a_backward_pass_is_refused(s, hq):
    """The operator is forward only: a gradient that would have to pass through it is an error, not a zero."""
    from minference_b200 import kv8_attention
    from minference_b200._cabi import MInferB200Error

    gen = torch.Generator().manual_seed(5)
    cache, _ = _filled(gen, 1, 1, [100], torch.int8)
    _, q = _rows(gen, 1, hq, s)
    want, want_lse = kv8_attention(q, cache, 100, return_lse=True)
    leaf = q.detach().clone().requires_grad_()
    out, lse = kv8_attention(leaf, cache, 100, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse) and out.requires_grad and out.stride() == torch.empty_like(leaf).stride()
    with pytest.raises(MInferB200Error, match="forward only"):
        (out.float() * 2).sum().backward()
    with pytest.raises(MInferB200Error, match="forward only"):
        kv8_attention(leaf, cache, 100, return_lse=True)[1].sum().backward()
    out, _ = kv8_attention(leaf, cache, 100, return_lse=True)
    assert torch.equal(out.mul_(2), want * 2)    # an output of its own, not a view
    with torch.no_grad():
        assert not kv8_attention(leaf, cache, 100).requires_grad
    assert not kv8_attention(q, cache, 100).requires_grad and leaf.grad is None


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("s, hq", [(1, 24), (1, 25), (6, 4), (5, 5), (24, 1), (25, 1), (3, 8), (8, 3), (1, 8), (1, 9), (1, 16), (1, 17)])
def test_rows_around_the_kernels_borders(kind, s, hq):
    """24 rows are the narrow kernel's last, 25 the wide one's first; 8 and 16 fill groups of columns."""
    gen = torch.Generator().manual_seed(100 * s + hq)
    lengths = [700, 65, max(s - 1, 0)]
    cache, ref = _filled(gen, 3, 1, lengths, kind)
    _check_attention(cache, ref, lengths, s, hq, gen, weights=True)


@pytest.mark.parametrize("kind", KINDS)
def test_going_back_into_a_complete_block(kind):
    """Proposed tokens fill a block and are then dropped: its tokens go back into the tail by the documented lines."""
    from minference_b200 import kv8_load, kv8_store

    gen = torch.Generator().manual_seed(12)
    cache, ref = _filled(gen, 1, 2, [190], kind, capacity=320)
    k, dk = _rows(gen, 1, 2, 5)
    v, dv = _rows(gen, 1, 2, 5)
    kv8_store(cache, dk, dv, 190)                # 195 tokens: block 2 is complete, the tail holds 192 to 194
    ref.append(k, v)
    kept = 191
    block = kept // 64 * 64
    cache.k_tail[:], cache.v_tail[:] = kv8_load(cache, 195, first=block, count=64)
    back = R.RefCache(1, 2, kind)
    for name in ("k", "v"):
        for h in range(2):
            x = ref.values(name, 0, h)[0]        # of the block that was complete: values of codes, rounded to bf16
            x[block:] = x[block:].to(torch.bfloat16).double()
            back.raw[name][0][h] = torch.cat((ref.raw[name][0][h][:block], x[block:kept]))
    _check_attention(cache, back, [kept], 1, 8, gen, weights=True)
    k, dk = _rows(gen, 1, 2, 70)
    v, dv = _rows(gen, 1, 2, 70)
    kv8_store(cache, dk, dv, kept)
    back.append(k, v)
    _check_attention(cache, back, [kept + 70], 3, 8, gen)


@pytest.mark.parametrize("s", [1, 40])
def test_the_first_call_of_a_process_may_be_captured(s):
    import subprocess
    import sys

    from tests.conftest import ROOT

    code = f"""
import torch
from minference_b200 import KV8Cache, kv8_attention, kv8_evict, kv8_store
gen = torch.Generator("cuda").manual_seed(1)
rows = lambda h, n: torch.randn(1, h, n, 128, generator=gen, device="cuda").to(torch.bfloat16)
cache, out = KV8Cache.empty(1, 2, 512), KV8Cache.empty(1, 2, 64)
k, v, q = rows(2, 300), rows(2, 300), rows(8, {s})
def step():
    kv8_store(cache, k, v, 0)
    w = torch.zeros(1, 2, 512, device="cuda")
    return kv8_attention(q, cache, 300, weights=w), w, kv8_evict(cache, 300, w, 64, recent=8, out=out)[3]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_a_long_prompt_of_another_scaling_needs_little_memory():
    from minference_b200 import KV8Layer

    n = 65536
    rows = lambda h: torch.randn(1, h, n, 128, dtype=torch.bfloat16, device="cuda")
    kv, k, q = KV8Layer(budget=4096), rows(8), rows(32)
    kv.append(k, k)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    kv.after_prompt(q, k, 0.05)
    torch.cuda.synchronize()
    # logits of 64 queries of a query head for each of 8 heads, 134 MB; their parts, at most 148 CTAs' 128 rows of 512 bytes;
    # the smaller cache, 11 MB.  All query heads' logits would be 537 MB
    assert torch.cuda.max_memory_allocated() - base <= 192 << 20
    assert kv.held == 4096 and abs(kv.sums.sum().item() / 2048) <= 1 + 1e-5


def test_going_back_by_a_smaller_length():
    """To a multiple of 64, and inside the block that was incomplete, a smaller length is all it takes."""
    from minference_b200 import kv8_store

    gen = torch.Generator().manual_seed(13)
    cache, ref = _filled(gen, 1, 2, [170], torch.float8_e4m3fn, capacity=320)
    for kept in (169, 129, 128, 64):
        cut = R.RefCache(1, 2, torch.float8_e4m3fn)
        for name in ("k", "v"):
            for h in range(2):
                cut.raw[name][0][h] = ref.raw[name][0][h][:kept]
        _check_attention(cache, cut, [kept], 1, 8, gen)
    k, dk = _rows(gen, 1, 2, 80)
    v, dv = _rows(gen, 1, 2, 80)
    kv8_store(cache, dk, dv, 64)
    cut.append(k, v)
    _check_attention(cache, cut, [144], 1, 8, gen)
