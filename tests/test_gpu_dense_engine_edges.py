"""DenseEngine on models of unusual sizes and after calls that failed."""

import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu

from flashloop_amd import DenseEngine  # noqa: E402
from flashloop_amd.model import OuroConfig, OuroForCausalLM  # noqa: E402

TINY = OuroConfig(vocab_size=1024, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=2,
                  num_key_value_heads=2, init_std=0.06)


def _ids(rows, t, vocab, seed=3):
    return torch.randint(0, vocab, (rows, t), generator=torch.Generator().manual_seed(seed)).cuda()


def _near(got, want, what):
    """Both run the model in bf16 with different roundings in between."""
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all()
    assert (got - want).norm() < 3e-2 * want.norm(), (what, ((got - want).norm() / want.norm()).item())


@pytest.mark.parametrize("vocab", [1021, 1022, 1023])
@pytest.mark.parametrize("rows", [1, 3, 8, 9])
def test_vocabularies_of_any_size(vocab, rows):
    """Steps of up to 8 sequences (fused) and of more: the fused product takes multiples of 4 outputs only."""
    print(f"case: dense engine vocabulary {vocab} rows {rows}", flush=True)
    model = OuroForCausalLM.random_init(dataclasses.replace(TINY, vocab_size=vocab), seed=11, device="cuda")
    ids = _ids(rows, 12, vocab)
    for graphs in (True, False):
        engine = DenseEngine(model, use_graphs=graphs)
        engine.prefill(ids[:, :9], decode_capacity=8)
        for t in range(9, 12):
            out = engine.decode(ids[:, t: t + 1])
            assert out.logits.shape == (rows, vocab) and out.logits.dtype == torch.float32
            for b in range(rows):
                _near(out.logits[b], model.dense_forward(ids[b: b + 1, : t + 1])[0], (graphs, t, b))
    engine.reset()
    assert [len(o) for o in engine.generate(ids, max_new_tokens=4, num_beams=2)] == [16] * rows
