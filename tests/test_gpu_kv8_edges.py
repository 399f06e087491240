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
