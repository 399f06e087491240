"""Decoding over 8-bit caches after the sparse prefill: the runner and a patched Hugging Face model, against the same steps
with plain fp32 attention over the values read back from the cache (``kv8_load``)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DENSE = {"starting_layer": 1 << 30, "best_pattern": []}


def _plain_attend(self, query, sm_scale=None):
    """KV8Layer.attend with elementary torch operations over what kv8_load gives back."""
    from minference_b200 import kv8_load

    b, h, s, d = query.shape
    n, hkv = self.held, self.cache.kv_heads
    k, v = (t.float() for t in kv8_load(self.cache, n, count=n))
    q = query.float().reshape(b, hkv, h // hkv * s, d)
    seen = torch.arange(n, device=q.device)[None, :] < (n - s + 1 + torch.arange(s, device=q.device))[:, None]
    logits = (q @ k.transpose(2, 3)) * (d ** -0.5 if sm_scale is None else sm_scale)
    p = torch.softmax(logits.masked_fill(~seen.repeat(h // hkv, 1), -math.inf), -1)
    if self.budget is not None:
        self.sums[..., :n] += p.sum(2)
        self.plain_weights = True
    out = (p @ v).view(b, h, s, d).to(query.dtype)
    if self.budget is not None and self.held >= self.budget + self.slack:
        self.evict()
    return out


def _close(a, b):
    # the bound of the whole-model prefill test: bf16 activations through two layers
    scale = b.abs().max().item()
    assert torch.isfinite(a).all()
    assert (a - b).abs().max().item() <= 3e-2 * scale + 1e-3, ((a - b).abs().max().item(), scale)


@pytest.fixture(scope="module")
def tiny():
    from minference_b200.prefill_runner import LlamaPrefill, LlamaShape

    shape = LlamaShape(layers=2, hidden=512, q_heads=8, kv_heads=2, head_dim=128, ffn=1024, vocab=1000)
    model = LlamaPrefill(shape, "cuda", seed=1, init_std=0.05)
    ids = torch.randint(0, shape.vocab, (900,), generator=torch.Generator().manual_seed(2))
    return shape, model, ids


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_decoding_steps_match_plain_attention(tiny, dtype, monkeypatch):
    from minference_b200 import KV8Layer

    shape, model, ids = tiny
    runs = []
    for plain in (False, True):
        if plain:
            monkeypatch.setattr(KV8Layer, "attend", _plain_attend)
        kv = model.new_kv(dtype=dtype)
        logits = [model.prefill(ids, DENSE, chunk=256, kv=kv)[None]]
        for step in ([7], [9], [3, 1, 4, 1, 5], list(range(100, 170)), [2]):        # single tokens, five, a follow-up of 70
            logits.append(model.decode(torch.tensor(step), kv))
        assert [x.held for x in kv] == [x.seen for x in kv] == [978, 978]
        for x in kv:
            x.cache.check()
        runs.append(torch.cat(logits))
    _close(*runs)


def test_decoding_follows_the_whole_network(tiny):
    """int8 keys and values move the next logits by less than the prefill test's bound: the cache holds the right tokens at
    the right positions."""
    from minference_b200.prefill_runner import dense_reference_logits

    shape, model, ids = tiny
    kv = model.new_kv(dtype=torch.int8)
    model.prefill(ids, DENSE, kv=kv)
    more = torch.tensor([5, 6, 7])
    for i in range(3):
        logits = model.decode(more[i:i + 1], kv)[-1]
        _close(logits, dense_reference_logits(model, torch.cat((ids, more[: i + 1]))))


def test_eviction_during_decoding(tiny, monkeypatch):
    """A budget cuts the prompt and the growing cache down; every step equals plain attention over what the cache then holds."""
    from minference_b200 import KV8Layer, kv8_attention, kv8_load

    shape, model, ids = tiny
    kv = model.new_kv(dtype=torch.float8_e4m3fn, budget=200, recent=40, sink=4, slack=20)
    model.prefill(ids, DENSE, kv=kv)
    assert all(x.held == 200 and x.seen == 900 for x in kv)
    seen_both = []

    def both(self, query, sm_scale=None):
        before = self.sums.clone()
        n = self.held
        want = _plain_attend(self, query, sm_scale) if n < self.budget + self.slack else None
        if want is not None:
            sums = before.clone()
            got = kv8_attention(query, self.cache, n, sm_scale=sm_scale, weights=sums, add_to=sums)
            assert (got.float() - want.float()).abs().max() <= 2.0 ** -6 * want.float().abs().max()     # bf16 both, one rounding each and P's
            assert torch.allclose(sums[..., :n], self.sums[..., :n], rtol=1e-4, atol=1e-5)
            seen_both.append(n)
            return got
        return real(self, query, sm_scale)

    real = KV8Layer.attend
    monkeypatch.setattr(KV8Layer, "attend", both)
    for t in range(45):
        model.decode(torch.tensor([t]), kv)
    assert all(x.seen == 945 and 200 <= x.held < 220 for x in kv) and min(seen_both) == 201 and max(seen_both) == 219
    k, _ = kv8_load(kv[0].cache, kv[0].held, count=kv[0].held)
    assert torch.isfinite(k.float()).all()


def test_generate_and_growth(tiny):
    shape, model, ids = tiny
    kv = model.new_kv(capacity=64)
    out = model.generate(ids[:30], 6, DENSE, kv=kv)
    assert out.shape == (6,) and kv[0].held == 35
    start = kv[0].cache.capacity
    model.decode(torch.arange(start), kv)                   # more than there is room for: the cache grows and keeps its tokens
    assert kv[0].cache.capacity > start and kv[0].held == 35 + start
    again = model.new_kv(capacity=8 * start)
    model.generate(ids[:30], 6, DENSE, kv=again)
    model.decode(torch.arange(start), again)
    from minference_b200 import kv8_load

    n = kv[0].held
    for a, b in zip(kv, again):
        for x, y in zip(kv8_load(a.cache, n, count=n), kv8_load(b.cache, n, count=n)):
            assert torch.equal(x, y)


def test_prompt_weights_are_the_estimators_scores():
    from minference_b200.modules.kv8_decode import prompt_weights
    from minference_b200.synthetic import make_qkv

    q, k, _ = make_qkv(300, 4, 2, seed=3, dtype=torch.bfloat16)
    w = prompt_weights(q.cuda(), k.cuda())
    assert w.shape == (1, 2, 300)
    p = torch.softmax((q[:, :, -64:].double() @ k.double().repeat_interleave(2, 1).transpose(2, 3) / 128 ** 0.5).masked_fill(
        torch.arange(300)[None, :] > torch.arange(236, 300)[:, None], -math.inf), -1)
    want = p.sum(2).view(1, 2, 2, 300).sum(2)
    # the estimator rounds its logits to bf16 twice (product and division): 2 * 2^-8 of logits up to their largest magnitude
    top = (q[:, :, -64:].double() @ k.double().repeat_interleave(2, 1).transpose(2, 3) / 128 ** 0.5).abs().max().item()
    rel = 2 * (math.exp(2 * 2.0 ** -8 * top) - 1)
    assert ((w.cpu().double() - want).abs() <= rel * want + 1e-6).all()


def test_hugging_face_model(tmp_path, monkeypatch):
    from transformers import DynamicCache, LlamaConfig, LlamaForCausalLM

    from minference_b200 import KV8HFCache, KV8Layer, MInference

    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=128, max_position_embeddings=4096, rope_theta=5e5, attn_implementation="sdpa")
    model = LlamaForCausalLM(cfg).to(torch.bfloat16).cuda().eval()
    ids = torch.randint(0, 1000, (1, 700), device="cuda")
    more = torch.randint(0, 1000, (1, 8), device="cuda")

    def steps(past):
        with torch.no_grad():
            out = [model(ids, past_key_values=past, use_cache=True).logits[:, -1:]]
            for a, b in ((0, 1), (1, 2), (2, 7), (7, 8)):        # one token, one, five at once, one
                out.append(model(more[:, a:b], past_key_values=past, use_cache=True).logits)
        return torch.cat(out, 1).float()

    stock = steps(DynamicCache())                                # the model as it came
    model = MInference("dense")(model)
    past = KV8HFCache(dtype=torch.int8)
    got = steps(past)
    assert past.get_seq_length() == 708 and past.layers[0].kv.held == 708
    with monkeypatch.context() as m:
        m.setattr(KV8Layer, "attend", _plain_attend)
        _close(got, steps(KV8HFCache(dtype=torch.int8)))
    _close(got, stock)                                           # and the tokens are where the stock cache has them
    with torch.no_grad():
        out = model.generate(ids, past_key_values=KV8HFCache(budget=256, slack=4), max_new_tokens=12, do_sample=False)
    assert out.shape == (1, 712)
    import minference_b200._cabi as cabi

    with pytest.raises(cabi.MInferB200Error):
        past.crop(5)


@pytest.mark.parametrize("n", [1, 2, 40, 64, 65, 130])
def test_short_prompts_with_a_budget(tiny, n):
    """Prompts shorter than the estimator's 64 queries and around the budget, then decoding past it."""
    shape, model, ids = tiny
    kv = model.new_kv(budget=64, recent=16, slack=8, dtype=torch.int8)
    model.prefill(ids[:n], DENSE, kv=kv)
    assert all(x.seen == n and x.held == min(n, 64) for x in kv)
    for x in kv:                # four heads' 64 queries at most, each with probabilities that sum to one (2^-7: should they be bf16)
        held = x.sums[..., : x.held].sum(-1)
        assert (held <= 4 * min(n, 64) * (1 + 2.0 ** -7)).all() and (n > 64 or (held >= 4 * n * (1 - 2.0 ** -7)).all())
    for t in range(80):
        assert torch.isfinite(model.decode(torch.tensor([t]), kv)).all()
    assert all(x.seen == n + 80 and x.held < 64 + 8 for x in kv)
