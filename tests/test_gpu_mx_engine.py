"""Engines on 4-bit weights (``FlashLoopConfig(weight_bits=4)``) against bf16 engines whose weights
hold the 4-bit values: what is left between them is the rounding of a prompt's rows to 8 bits.

That rounding is 2^-4 of a value at most, about 2^-4 / sqrt(12) = 0.018 in relative norm; the 2 layers
and 4 loops take four such products each, so 32 independent ones add up to sqrt(32) * 0.018 = 0.1 of
the hidden rows' norm, and with the same for the cached keys and values to 0.15.  Every row is kept and
every key selected, so that no selection near a border tells the engines apart."""

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

from flashloop_amd import FlashLoopBatchEngine, FlashLoopConfig, FlashLoopEngine, flashloop, kernels  # noqa: E402
from flashloop_amd.model import OuroConfig, OuroForCausalLM  # noqa: E402

DEV = "cuda"
APART = 0.15
MODEL = OuroConfig(vocab_size=520, hidden_size=256, intermediate_size=520, num_hidden_layers=2, num_attention_heads=2,
                   num_key_value_heads=2, init_std=0.06)
ALL = dict(prefill_fraction_loop3=1.0, prefill_fraction_loop4=1.0, enable_sparse_decode=False)


def _say(*what):
    print("case:", *what, flush=True)


@pytest.fixture(scope="module")
def models():
    """(model, the same with its Linear weights rounded to 4 bits)."""
    model = OuroForCausalLM.random_init(MODEL, seed=3, device=DEV)
    rounded = copy.deepcopy(model)
    for m in rounded.modules():
        if isinstance(m, torch.nn.Linear):
            m.weight.data.copy_(kernels.mx_dequantize(kernels.mx_quantize(m.weight.data, 4)))
    return model, rounded


def _ids(n, seed=0):
    return torch.randint(0, MODEL.vocab_size, (1, n), generator=torch.Generator().manual_seed(seed)).to(DEV)


def _near(got, want):
    got, want = got.double(), want.double()
    apart = ((got - want).norm(dim=-1) / want.norm(dim=-1)).max().item()
    assert apart < APART, apart


@pytest.mark.parametrize("tokens", [1, 70, 300])
def test_engine_follows_the_rounded_weights(models, tokens):
    _say("engine", tokens)
    model, rounded = models
    before = {n: p.clone() for n, p in model.named_parameters()}
    four = FlashLoopEngine(model, config=FlashLoopConfig(weight_bits=4, **ALL))
    sixteen = FlashLoopEngine(rounded, config=FlashLoopConfig(**ALL))
    ids = _ids(tokens)
    a, b = (e.prefill(ids, all_logits=True).logits for e in (four, sixteen))
    assert a.shape == (1, tokens, MODEL.vocab_size) and a.dtype == torch.float32
    _near(a, b)
    for step in range(4):
        tok = _ids(1, seed=50 + step)
        _near(four.decode(tok).logits, sixteen.decode(tok).logits)
    assert all(torch.equal(p, before[n]) for n, p in model.named_parameters())


def test_graph_steps_equal_eager_steps(models):
    _say("graph steps")
    model, _ = models
    cfg = FlashLoopConfig(weight_bits=4)
    graph, eager = FlashLoopEngine(model, config=cfg), FlashLoopEngine(model, config=cfg, use_graphs=False)
    ids = _ids(200, seed=1)
    assert torch.equal(graph.prefill(ids).logits, eager.prefill(ids).logits)
    for step in range(6):
        tok = _ids(1, seed=80 + step)
        assert torch.equal(graph.decode(tok).logits, eager.decode(tok).logits)


@pytest.mark.parametrize("batch", [3, 9])
def test_batch_follows_single_sequences(models, batch):
    """Up to 8 sequences decode through the GEMVs, more through the products of 8-bit rows."""
    _say("batch", batch)
    model, _ = models
    cfg = FlashLoopConfig(weight_bits=4, **ALL)
    lengths = [20 + 13 * b for b in range(batch)]
    ids = torch.zeros(batch, max(lengths), dtype=torch.long, device=DEV)
    mask = torch.zeros_like(ids)
    for b, n in enumerate(lengths):
        ids[b, :n], mask[b, :n] = _ids(n, seed=b)[0], 1
    for graphs in (False, True):
        eng = FlashLoopBatchEngine(model, config=cfg, use_graphs=graphs)
        out = eng.prefill(ids, mask)
        steps = [torch.cat([_ids(1, seed=100 * s + b) for b in range(batch)]) for s in range(3)]
        got = [out.logits] + [eng.decode(t).logits.clone() for t in steps]
        for b in (0, batch - 1):
            one = FlashLoopEngine(model, config=cfg)
            want = [one.prefill(ids[b:b + 1, :lengths[b]]).logits] + [one.decode(t[b:b + 1]).logits.clone() for t in steps]
            for g, w in zip(got, want):
                _near(g[b:b + 1], w)


def test_unchained_steps_and_wide_rows(models):
    """Separate norm launches (as rows wider than the chained GEMV's take) give the chained step's logits."""
    _say("unchained")
    model, _ = models
    cfg = FlashLoopConfig(weight_bits=4, **ALL)
    chained, apart = (FlashLoopEngine(model, config=cfg, use_graphs=False) for _ in range(2))
    apart.fused_chain = False
    ids = _ids(64, seed=5)
    chained.prefill(ids), apart.prefill(ids)
    for step in range(3):
        tok = _ids(1, seed=30 + step)
        _near(chained.decode(tok).logits, apart.decode(tok).logits)


def test_hook_context_generates(models):
    _say("hooks")
    model, _ = models
    ids = _ids(40, seed=7)
    with flashloop(model, weight_bits=4):
        got = model.generate(ids, max_new_tokens=6)
    eng = FlashLoopEngine(model, config=FlashLoopConfig(weight_bits=4))
    assert torch.equal(got, eng.generate(ids, max_new_tokens=6)) and got.shape == (1, 46)


def test_changed_weights_are_quantized_again(models):
    _say("changed weights")
    model = copy.deepcopy(models[0])
    eng = FlashLoopEngine(model, config=FlashLoopConfig(weight_bits=4))
    ids = _ids(30, seed=9)
    first = eng.prefill(ids).logits
    with torch.no_grad():
        model.lm_head.weight.mul_(2)
    eng.reset()
    assert torch.equal(eng.prefill(ids).logits, first)
    eng.reset()
    eng.quantize_weights()
    assert torch.equal(eng.prefill(ids).logits, 2 * first)
    batch = FlashLoopBatchEngine(model, config=FlashLoopConfig(weight_bits=4))
    assert torch.equal(batch.prefill(ids).logits, 2 * first)
    tok = _ids(1)
    before = batch.decode(tok).logits.clone()
    with torch.no_grad():
        model.lm_head.weight.mul_(2)
    batch.quantize_weights()
    batch.reset()
    batch.prefill(ids)
    assert torch.equal(batch.decode(tok).logits, 2 * before)  # (a new graph, not the old copies')


def test_replaced_modules_are_refused(models):
    _say("refusals")
    model = copy.deepcopy(models[0])
    with pytest.raises(ValueError, match="weight_bits=4"):
        FlashLoopEngine(model).quantize_weights()
    eng = FlashLoopEngine(model, config=FlashLoopConfig(weight_bits=4))
    handle = model.model.layers[0].self_attn.q_proj.register_forward_hook(lambda *a: None)
    with pytest.raises(RuntimeError, match="weight_bits=4"):
        eng.prefill(_ids(10))
    with pytest.raises(ValueError, match="plain Linear"):
        FlashLoopEngine(model, config=FlashLoopConfig(weight_bits=4))
    handle.remove()
    eng.prefill(_ids(10))
    eng.fused_decode, eng.use_graphs = False, False
    with pytest.raises(RuntimeError, match="weight_bits=4"):
        eng.decode(_ids(1))
    model.lm_head.bias = torch.nn.Parameter(torch.zeros(MODEL.vocab_size, device=DEV))
    with pytest.raises(ValueError, match="plain Linear"):
        FlashLoopEngine(model, config=FlashLoopConfig(weight_bits=4))
