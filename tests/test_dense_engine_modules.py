"""DenseEngine takes the modules' weights: it notices modules that change afterwards (no GPU: no kernel runs)."""

import pytest
import torch

from flashloop_amd import DenseEngine, PagedKVCache
from flashloop_amd.model import OuroConfig, OuroForCausalLM, RMSNorm, RotaryEmbedding

TINY = OuroConfig(vocab_size=64, hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1)
IDS = torch.zeros(1, 3, dtype=torch.long)


def _engine():
    """An engine between two calls of a sequence of 3 tokens, whose model's passes are left out."""
    engine = DenseEngine(OuroForCausalLM.random_init(TINY, seed=1))

    def feed(ids, counts, rows):
        for r, n in zip(rows, counts):
            engine._lens[r] += n
        engine._lengths_to_device()
        return torch.zeros(len(rows), TINY.vocab_size)

    engine._feed = feed

    def advance(ids):
        engine.cache.lens.add_(1)
        return torch.zeros(len(engine._lens), TINY.vocab_size)

    engine._advance = advance
    engine.prefill(IDS)
    return engine


def _hook(model):
    model.model.layers[1].mlp.up_proj.register_forward_hook(lambda *a: None)


def _pre_hook(model):
    model.lm_head.register_forward_pre_hook(lambda *a: None)


def _forward(model):
    model.model.norm.forward = lambda x: x


def _parameter(model):
    m = model.model.layers[0].self_attn.o_proj
    m.weight = torch.nn.Parameter(m.weight.detach().clone())


def _data(model):
    m = model.model.embed_tokens
    m.weight.data = m.weight.data.clone()


def _bias(model):
    m = model.model.layers[1].self_attn.q_proj
    m.bias = torch.nn.Parameter(torch.zeros(m.weight.shape[0], dtype=torch.bfloat16))


def _module(model):
    model.model.layers[0].input_layernorm_2 = RMSNorm(TINY.hidden_size, TINY.rms_norm_eps).to(torch.bfloat16)


def _layer(model):
    model.model.layers[0], model.model.layers[1] = model.model.layers[1], model.model.layers[0]


def _rotary(model):
    model.model.rotary_emb = RotaryEmbedding(128, 5e5)


def _frequencies(model):
    model.model.rotary_emb.inv_freq = model.model.rotary_emb.inv_freq * 2


def _eps(model):
    model.model.layers[0].input_layernorm.eps = 1e-3


def _embedding_norm(model):
    model.model.embed_tokens.max_norm = 1.0


PLAIN = [_parameter, _data, _module, _layer, _rotary, _frequencies]  # what a new prompt can take
OTHER = [_hook, _pre_hook, _forward, _bias, _eps, _embedding_norm]  # what it refuses


@pytest.mark.parametrize("change", PLAIN + OTHER)
def test_changed_modules(change):
    engine = _engine()
    engine.extend(IDS)
    engine.decode(IDS[:, :1])
    assert engine.positions == (7,)
    change(engine.model)
    for call in (lambda: engine.extend(IDS), lambda: engine.decode(IDS[:, :1])):
        with pytest.raises(RuntimeError, match="replaced or hooked"):
            call()
        assert engine.positions == (7,) and engine.cache.lens.tolist() == [7]
    engine.reset()
    if change in OTHER:
        with pytest.raises(ValueError, match="DenseEngine needs"):
            engine.prefill(IDS)
        with pytest.raises(ValueError, match="DenseEngine needs"):
            engine.generate(IDS, max_new_tokens=2)
        assert engine.cache is None
        return
    engine.prefill(IDS)
    engine.decode(IDS[:, :1])
    layers = engine.model.model.layers
    for i, (got, layer) in enumerate(zip(engine._weights[0], layers)):
        for w, m in zip(got, (layer.self_attn.q_proj, layer.self_attn.k_proj, layer.self_attn.v_proj, layer.self_attn.o_proj, layer.mlp.gate_proj,
                              layer.mlp.up_proj, layer.mlp.down_proj, layer.input_layernorm, layer.input_layernorm_2,
                              layer.post_attention_layernorm, layer.post_attention_layernorm_2)):
            assert w.data_ptr() == m.weight.data_ptr(), i


def test_weights_changed_in_place():
    """The same storage: the next call computes with the new values, and none is refused."""
    engine = _engine()
    with torch.no_grad():
        engine.model.model.layers[0].mlp.down_proj.weight.zero_()
    engine.model.load_state_dict(OuroForCausalLM.random_init(TINY, seed=2).state_dict())
    engine.extend(IDS)
    engine.decode(IDS[:, :1])
    engine.model.model.layers[0].register_forward_hook(lambda *a: None)  # (a layer is never called)
    engine.decode(IDS[:, :1])
    assert engine.positions == (8,)


def test_calls_run_on_the_models_device(monkeypatch):
    """With another device current, the model's is made the current one for a call; prompts on another device are refused."""
    entered = []

    class Current:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            entered.append(self.device)

        def __exit__(self, *exc):
            entered.append(None)

    engine = _engine()
    for call in (lambda: engine.extend(IDS), lambda: engine.decode(IDS[:, :1])):
        call()
    assert entered == []  # (a model on the CPU)
    far = torch.device("cuda", 1)
    monkeypatch.setattr(torch.cuda, "device", Current)
    monkeypatch.setattr(DenseEngine, "device", far)
    engine.decode(IDS[:, :1])
    assert entered == [far, None]
    held = engine.cache
    for cache, call in ((held, lambda: engine.extend(IDS)), (None, lambda: engine.prefill(IDS)), (None, lambda: engine.generate(IDS, max_new_tokens=1)),
                        (None, lambda: engine.generate(IDS, max_new_tokens=1, num_beams=2))):
        engine.cache = cache
        entered.clear()
        with pytest.raises(ValueError, match="input_ids lie on cpu, the model on cuda:1"):
            call()
        assert entered[0] == far and entered[-1] is None


def test_cache_refusals():
    """Sizes that hold nothing, and shared pages of rows that come later or are not there (a row before the first is the last one
    of a list)."""
    for sizes in ((0, 2, 1, 20), (1, 0, 1, 20), (1, 2, 0, 20), (1, 2, 1, 0), (1, 2, 1, -5)):
        with pytest.raises(ValueError, match="positive"):
            PagedKVCache(*sizes, "cpu", page_size=16)
    for shared in ([(0, 0)], [(0, 0), (-1, 1)], [(1, 1), (1, 1)], [(0, 0), (0, -1)], [(0, 0), (2, 1)]):
        with pytest.raises(ValueError, match="shared"):
            PagedKVCache(1, 2, 1, 40, "cpu", page_size=16, shared=shared)
    assert PagedKVCache(1, 2, 1, 40, "cpu", page_size=16, shared=[]).table.tolist() == [[0, 1, 2], [3, 4, 5]]
    cache = PagedKVCache(1, 2, 1, 40, "cpu", page_size=16, shared=[(0, 5), (0, 1)])
    assert cache.table.tolist() == [[0, 1, 2], [0, 3, 4]] and cache.k_pages.shape[1] == 5
