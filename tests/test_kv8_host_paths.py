"""Host paths around the 8-bit cache that must not go wrong without a word (no GPU needed: the storage is stubbed)."""
from types import SimpleNamespace

import pytest
import torch


@pytest.fixture()
def cabi(built_lib):
    from minference_b200 import _cabi

    return _cabi


@pytest.fixture()
def counted(monkeypatch):
    """KV8Layer that only counts its tokens and answers with zeros."""
    from minference_b200 import KV8Layer

    def append(self, key, value):
        self.held += key.shape[2]
        self.seen += key.shape[2]

    monkeypatch.setattr(KV8Layer, "append", append)
    monkeypatch.setattr(KV8Layer, "attend", lambda self, query, sm_scale=None: torch.zeros_like(query))


def _model(layers, implementation="sdpa"):
    from transformers import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=50, hidden_size=256, intermediate_size=64, num_hidden_layers=layers, num_attention_heads=2,
                      num_key_value_heads=1, head_dim=128, max_position_embeddings=256, attn_implementation=implementation)
    return LlamaForCausalLM(cfg).eval()


IDS = torch.arange(6)[None]


@torch.no_grad()
def _steps(model, past, steps=3):
    model(IDS, past_key_values=past, use_cache=True)
    for _ in range(steps):
        model(IDS[:, :1], past_key_values=past, use_cache=True)


@pytest.mark.parametrize("layers", [1, 2])
def test_a_model_that_is_not_patched_is_refused(cabi, counted, layers):
    """Its attention would see the new tokens alone.  Two layers show it in the first call, one layer in the second."""
    from minference_b200 import KV8HFCache

    past = KV8HFCache()
    with pytest.raises(cabi.MInferB200Error, match="patched"):
        _steps(_model(layers), past, 1)
    past.reset()
    assert past.get_seq_length() == 0


def test_a_copy_of_the_keys_is_refused(cabi, counted):
    """A step between the cache and the attention function that makes another tensor of the keys loses their mark."""
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS

    from minference_b200 import KV8HFCache, MInference

    model = MInference("dense")(_model(2))
    name = model.config._attn_implementation
    real = ALL_ATTENTION_FUNCTIONS[name]
    ALL_ATTENTION_FUNCTIONS[name] = lambda module, q, k, v, mask, **kw: real(module, q, k.clone(), v, mask, **kw)
    try:
        with pytest.raises(cabi.MInferB200Error, match="patched"):
            _steps(model, KV8HFCache())
    finally:
        ALL_ATTENTION_FUNCTIONS[name] = real


@pytest.mark.parametrize("layers", [1, 2])
@pytest.mark.filterwarnings("ignore:minference_b200. this prefill")
def test_a_patched_model_is_taken(cabi, counted, layers):
    from minference_b200 import KV8HFCache, MInference

    model, past = MInference("dense")(_model(layers)), KV8HFCache()
    _steps(model, past)
    assert past.get_seq_length() == 9
    past.reset()
    _steps(model, past)
    assert past.get_seq_length() == 9


@pytest.fixture(scope="module")
def runner():
    from minference_b200.prefill_runner import LlamaPrefill, LlamaShape

    return LlamaPrefill(LlamaShape(layers=2, hidden=64, q_heads=2, kv_heads=1, head_dim=128, ffn=64, vocab=50), "cpu")


@pytest.mark.parametrize("option", [{"positions": torch.arange(6)}, {"attention": lambda q, k, v, layer: q},
                                    {"positions": torch.arange(6), "attention": lambda q, k, v, layer: q}])
def test_a_sharded_prompt_is_not_kept(cabi, counted, runner, option):
    """Under the ring a rank has a part of the prompt: it must not become the cache that decoding goes on from."""
    kv = runner.new_kv()
    with pytest.raises(cabi.MInferB200Error, match="whole prompt"):
        runner.prefill(IDS[0], {}, kv=kv, **option)
    assert all(x.seen == 0 for x in kv)


def test_a_decoding_step_with_a_mask_is_refused(cabi, counted):
    """The attention over the cache takes no mask: one that the model hands on must not be left out without a word."""
    from minference_b200 import KV8Layer, MInferenceConfig
    from minference_b200.patch import _make_attention_function

    attention = _make_attention_function(MInferenceConfig(attn_type="dense"))
    kv, q, key = KV8Layer(), torch.zeros(1, 2, 1, 128), torch.zeros(1, 1, 1, 128)
    kv.append(torch.zeros(1, 1, 9, 128), None)
    key.minf_kv8 = kv
    assert attention(None, q, key, key, None)[0].shape == (1, 1, 2, 128)
    with pytest.raises(cabi.MInferB200Error, match="mask"):
        attention(None, q, key, key, torch.zeros(1, 1, 1, 9))


def test_the_runner_wants_a_cache_for_every_layer(cabi, counted, runner):
    """Fewer would leave layers out of a decoding step without a word."""
    for kv in (runner.new_kv()[:1], runner.new_kv() + runner.new_kv(), []):
        with pytest.raises(cabi.MInferB200Error, match="2 layers"):
            runner.decode(IDS[0, :1], kv)
        with pytest.raises(cabi.MInferB200Error, match="2 layers"):
            runner.prefill(IDS[0], {}, kv=kv)
    assert runner.decode(IDS[0, :1], runner.new_kv()).shape == (1, 50)


def test_generate_refuses_what_it_would_leave_out(cabi, counted, runner, monkeypatch):
    monkeypatch.setattr(type(runner), "prefill", lambda self, ids, cfg, kv=None: torch.arange(50.0))
    assert runner.generate(IDS[0], 1, {}).tolist() == [49]
    for n in (0, -1):
        with pytest.raises(cabi.MInferB200Error, match="new_tokens"):
            runner.generate(IDS[0], n, {})
    with pytest.raises(cabi.MInferB200Error, match="options"):
        runner.generate(IDS[0], 1, {}, kv=runner.new_kv(), budget=100)


def test_a_layer_that_holds_nothing_is_refused(cabi):
    from minference_b200 import KV8Layer

    for kv in (KV8Layer(), KV8Layer(budget=100)):
        with pytest.raises(cabi.MInferB200Error, match="no tokens"):
            kv.attend(torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16))
        with pytest.raises(cabi.MInferB200Error, match="no tokens|no budget"):
            kv.evict()
    kv = KV8Layer()
    kv.cache = "something"
    with pytest.raises(cabi.MInferB200Error, match="no budget"):
        kv.evict()
    with pytest.raises(cabi.MInferB200Error, match="float8_e4m3fn or int8"):
        KV8Layer(torch.float16)
