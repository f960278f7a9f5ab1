"""Engines on 4-bit weights in the forms that real models run -- sparse decoding, more than 8 sequences, the
widths of a real layer, rows wider than the chained products take -- and what they refuse.

A step of up to 8 sequences on the same cache differs from the bf16 engine's on the 4-bit values by bf16
roundings alone: about 14 of each engine in each of a layer's four passes, each 2^-8 / sqrt(3) = 0.00226 in
relative norm at most, so with two layers sqrt(2 * 8 * 14) * 0.00226 = 0.034, and half as much again for what
SwiGLU and softmax make of them.  More sequences go through 8-bit rows: 0.018 for each of four
products a pass, 0.1 for two layers and 0.15 together with the cached rows of their prompts."""

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

from flashloop_amd import FlashLoopBatchEngine, FlashLoopConfig, FlashLoopEngine, kernels  # noqa: E402
from flashloop_amd.model import MLP, OuroConfig, OuroForCausalLM, RMSNorm  # noqa: E402

DEV = "cuda"
ROUNDINGS, ROWS = 0.05, 0.15
SMALL = OuroConfig(vocab_size=520, hidden_size=256, intermediate_size=520, num_hidden_layers=2, num_attention_heads=2,
                   num_key_value_heads=2, init_std=0.06)
LAYER = OuroConfig(vocab_size=49152, num_hidden_layers=1)  # a real model's widths
WIDE = OuroConfig(vocab_size=520, hidden_size=4224, intermediate_size=520, num_hidden_layers=1, num_attention_heads=33,
                  num_key_value_heads=33)
KEPT = dict(prefill_fraction_loop3=1.0, prefill_fraction_loop4=1.0, decode_key_fraction=1.0)  # (nothing to choose: no border)


def _say(*what):
    print("case:", *what, flush=True)


_MODELS = {}


def _models(name):
    """(model, the same with its Linear weights rounded to 4 bits)."""
    if name not in _MODELS:
        model = OuroForCausalLM.random_init({"small": SMALL, "layer": LAYER, "wide": WIDE}[name], seed=3, device=DEV)
        rounded = copy.deepcopy(model)
        for m in rounded.modules():
            if isinstance(m, torch.nn.Linear):
                m.weight.data.copy_(kernels.mx_dequantize(kernels.mx_quantize(m.weight.data, 4)))
        _MODELS[name] = model, rounded
    return _MODELS[name]


def _ids(n, seed=0):
    return torch.randint(0, 520, (1, n), generator=torch.Generator().manual_seed(seed)).to(DEV)


def _near(got, want, most):
    got, want = got.double(), want.double()
    apart = ((got - want).norm(dim=-1) / want.norm(dim=-1)).max().item()
    print(f"apart {apart:.4f} of {most}", flush=True)
    assert apart < most, apart


def _prompts(batch):
    lengths = [20 + 13 * b for b in range(batch)]
    ids = torch.zeros(batch, max(lengths), dtype=torch.long, device=DEV)
    mask = torch.zeros_like(ids)
    for b, n in enumerate(lengths):
        ids[b, :n], mask[b, :n] = _ids(n, seed=b)[0], 1
    return ids, mask, lengths


@pytest.mark.parametrize("sparse", [True, False])
@pytest.mark.parametrize("name", ["small", "layer", "wide"])
@pytest.mark.parametrize("graphs", [False, True])
def test_decode_of_one_sequence_on_the_same_cache(name, sparse, graphs):
    _say("decode on the same cache", name, sparse, graphs)
    model, rounded = _models(name)
    cfg = dict(KEPT, enable_sparse_decode=sparse)
    four, twin = (FlashLoopEngine(model, config=FlashLoopConfig(weight_bits=4, **cfg), use_graphs=graphs) for _ in range(2))
    sixteen = FlashLoopEngine(rounded, config=FlashLoopConfig(**cfg), use_graphs=False)
    sixteen.fused_chain = name != "wide"  # (the chained products take rows of up to 4096 values)
    ids = _ids(90, seed=2)
    assert torch.equal(four.prefill(ids).logits, twin.prefill(ids).logits)
    sixteen._state, twin._state = twin._state, None
    for step in range(3):
        tok = _ids(1, seed=60 + step)
        _near(four.decode(tok).logits, sixteen.decode(tok).logits, ROUNDINGS)


@pytest.mark.parametrize("sparse", [True, False])
@pytest.mark.parametrize("name,batch", [("small", 2), ("small", 8), ("small", 9), ("small", 17), ("layer", 5), ("layer", 8), ("layer", 12),
                                        ("wide", 3), ("wide", 9)])
def test_decode_of_a_batch_on_the_same_cache(name, batch, sparse):
    """The batch's caches come from its own prompts in both engines' case; sequences of the bf16 batch engine
    past 8 decode through the modules."""
    _say("batch on the same cache", name, batch, sparse)
    model, rounded = _models(name)
    cfg = dict(KEPT, enable_sparse_decode=sparse)
    ids, mask, _ = _prompts(batch)
    four, twin = (FlashLoopBatchEngine(model, config=FlashLoopConfig(weight_bits=4, **cfg), use_graphs=False) for _ in range(2))
    sixteen = FlashLoopBatchEngine(rounded, config=FlashLoopConfig(**cfg), use_graphs=False)
    sixteen._one.fused_chain = name != "wide"
    assert torch.equal(four.prefill(ids, mask).logits, twin.prefill(ids, mask).logits)
    sixteen._state, twin._state = twin._state, None
    for step in range(3):
        tok = torch.cat([_ids(1, seed=100 * step + b) for b in range(batch)])
        _near(four.decode(tok).logits, sixteen.decode(tok).logits, ROUNDINGS if batch <= 8 else ROWS)


@pytest.mark.parametrize("batch", [9, 16])
def test_sparse_decode_of_many_sequences(batch):
    """More than 8 sequences with the default selections: graph steps equal eager ones, and a sequence that keeps
    every key follows itself decoded alone."""
    _say("sparse decode of many", batch)
    model, _ = _models("small")
    ids, mask, lengths = _prompts(batch)
    graph, eager = (FlashLoopBatchEngine(model, config=FlashLoopConfig(weight_bits=4), use_graphs=g) for g in (True, False))
    assert torch.equal(graph.prefill(ids, mask).logits, eager.prefill(ids, mask).logits)
    for step in range(4):
        tok = torch.cat([_ids(1, seed=100 * step + b) for b in range(batch)])
        assert torch.equal(graph.decode(tok).logits, eager.decode(tok).logits)
    many = FlashLoopBatchEngine(model, config=FlashLoopConfig(weight_bits=4, **KEPT), use_graphs=False)
    many.prefill(ids, mask)
    toks = [torch.cat([_ids(1, seed=100 * s + b) for b in range(batch)]) for s in range(2)]
    got = [many.decode(t).logits.clone() for t in toks]
    for b in (0, batch - 1):
        one = FlashLoopEngine(model, config=FlashLoopConfig(weight_bits=4, **KEPT), use_graphs=False)
        one.prefill(ids[b:b + 1, :lengths[b]])
        for t, g in zip(toks, got):
            _near(g[b:b + 1], one.decode(t[b:b + 1]).logits, ROWS)


def _swap(owner, name, new):
    setattr(owner, name, new)


def _hook(m):
    m.register_forward_hook(lambda *a: None)


def _linear_like(m):
    return torch.nn.Linear(m.in_features, m.out_features, bias=False, device=DEV, dtype=torch.bfloat16)


@pytest.mark.parametrize("change", [
    lambda m: _hook(m.lm_head),
    lambda m: m.lm_head.register_forward_pre_hook(lambda *a: None),
    lambda m: _swap(m, "lm_head", _linear_like(m.lm_head)),
    lambda m: _swap(m.lm_head, "weight", torch.nn.Parameter(m.lm_head.weight.detach().clone())),
    lambda m: _swap(m.lm_head, "bias", torch.nn.Parameter(torch.zeros(520, device=DEV, dtype=torch.bfloat16))),
    lambda m: _swap(m.lm_head, "forward", lambda x: x),
    lambda m: _hook(m.model.layers[1].mlp.down_proj),
    lambda m: _swap(m.model.layers[0].self_attn, "q_proj", _linear_like(m.model.layers[0].self_attn.q_proj)),
    lambda m: _swap(m.model.layers[0].mlp.up_proj, "weight", torch.nn.Parameter(m.model.layers[0].mlp.up_proj.weight.detach() * 2)),
    lambda m: _swap(m.model.layers[1], "mlp", MLP(SMALL).to(DEV, torch.bfloat16)),
    lambda m: _swap(m.model.layers[1], "input_layernorm", RMSNorm(256, 1e-6).to(DEV, torch.bfloat16)),
    lambda m: _swap(m.model, "norm", RMSNorm(256, 1e-6).to(DEV, torch.bfloat16)),
    lambda m: m.model.layers.__setitem__(0, copy.deepcopy(m.model.layers[0])),
])
def test_changed_modules_are_refused(change):
    """Whatever the 4-bit copies would not follow: in a prompt, in a step, and until they are made anew."""
    _say("changed modules")
    model = copy.deepcopy(_models("small")[0])
    eng = FlashLoopEngine(model, config=FlashLoopConfig(weight_bits=4), use_graphs=False)
    batch = FlashLoopBatchEngine(model, config=FlashLoopConfig(weight_bits=4), use_graphs=False)
    ids, mask, _ = _prompts(9)
    eng.prefill(_ids(20))
    batch.prefill(ids, mask)
    change(model)
    with pytest.raises(RuntimeError, match="weight_bits=4"):
        eng.decode(_ids(1))
    with pytest.raises(RuntimeError, match="weight_bits=4"):
        batch.decode(ids[:, :1])
    eng.reset()
    with pytest.raises(RuntimeError, match="weight_bits=4"):
        eng.prefill(_ids(20))
    batch.reset()
    with pytest.raises(RuntimeError, match="weight_bits=4"):
        batch.prefill(ids, mask)


def test_new_modules_are_taken_anew():
    _say("new modules")
    model = copy.deepcopy(_models("small")[0])
    eng = FlashLoopEngine(model, config=FlashLoopConfig(weight_bits=4))
    first = eng.prefill(_ids(20)).logits.clone()
    head = _linear_like(model.lm_head)
    with torch.no_grad():
        head.weight.copy_(2 * model.lm_head.weight)
    model.lm_head = head
    eng.reset()
    eng.quantize_weights()
    assert torch.equal(eng.prefill(_ids(20)).logits, 2 * first)
    eng.decode(_ids(1))


@pytest.mark.parametrize("name", ["small", "layer"])
@pytest.mark.parametrize("batch", [1, 8])
def test_separate_norms_follow_the_chained_ones(name, batch):
    """Separate launches round the norms and the sum on their own: roundings apart, no more."""
    _say("separate norms", name, batch)
    model, _ = _models(name)
    cfg = FlashLoopConfig(weight_bits=4, **KEPT)
    ids, mask, _ = _prompts(batch)
    chained, apart = (FlashLoopBatchEngine(model, config=cfg, use_graphs=False) for _ in range(2))
    apart._one.fused_chain = False
    assert torch.equal(chained.prefill(ids, mask).logits, apart.prefill(ids, mask).logits)
    for step in range(3):
        tok = torch.cat([_ids(1, seed=100 * step + b) for b in range(batch)])
        _near(apart.decode(tok).logits, chained.decode(tok).logits, ROUNDINGS)
