"""DenseEngine's beam search against a plain one, on logits from tables and a plain selection (no GPU)."""

import pytest
import torch

from beam_util import CASES, plain_search, table_engine, tables_of
from flashloop_amd import DenseEngine, kernels
from flashloop_amd.model import OuroConfig, OuroForCausalLM
from paged_util import plain_select

TINY = OuroConfig(vocab_size=24, hidden_size=128, intermediate_size=256, num_hidden_layers=1, num_attention_heads=1, num_key_value_heads=1)


@pytest.mark.parametrize("beams,new,eos,penalty,kind", CASES)
def test_search(monkeypatch, beams, new, eos, penalty, kind):
    """Every sequence of a batch gets the completion that it gets alone."""
    monkeypatch.setattr(kernels, "beam_select", lambda x, s, n: (lambda t, b, k: (t.float(), b, k))(*plain_select(x, s, n)))
    model = OuroForCausalLM.random_init(TINY, seed=1)
    prompts = torch.randint(0, 24, (4, 3), generator=torch.Generator().manual_seed(5))
    for seed in range(6):
        first, tables = tables_of(kind, 4, new, eos, 24, seed)
        got = table_engine(model, first, tables, "cpu").generate(prompts, max_new_tokens=new, eos_token_id=eos, num_beams=beams, length_penalty=penalty)
        for b in range(4):
            want = plain_search(first[b], tables[b], beams, new, eos, penalty)
            assert got[b].tolist() == prompts[b].tolist() + want[1], (seed, b, want)


def test_plain_search():
    """The definition on a case worked out by hand: the EOS (token 0) ends a likely beginning at once, or a longer completion
    with a better mean."""
    log = lambda *p: torch.log(torch.tensor(p))
    first = log(0.4, 0.6, 1e-9)
    table = torch.stack([torch.stack([log(1 / 3, 1 / 3, 1 / 3), log(0.5, 0.1, 0.4), log(1 / 3, 1 / 3, 1 / 3)])] * 2)
    table[1, 2] = log(0.9, 0.05, 0.05)
    # ends at once: 0.4; 1 0: 0.3; 1 2 0: 0.6 * 0.4 * 0.9 = 0.216
    for penalty, tokens in ((0.0, [0]), (1.0, [1, 2, 0]), (4.0, [1, 2, 0])):
        score, got = plain_search(first, table, 2, 3, 0, penalty)
        assert got == tokens
        p = {1: 0.4, 3: 0.216}[len(tokens)]
        assert abs(score - float(torch.log(torch.tensor(p, dtype=torch.float64))) / len(tokens) ** penalty) < 1e-6


def test_penalties_out_of_range():
    """Quotients that fp32 cannot hold apart are refused before anything runs; the largest that is taken still tells
    completions apart."""
    model = OuroForCausalLM.random_init(TINY, seed=1)
    engine, ids = DenseEngine(model), torch.zeros(1, 3, dtype=torch.long)
    for penalty, new in ((-0.1, 4), (float("nan"), 4), (float("inf"), 4), (float("inf"), 1), (60.0, 4), (400.0, 12), (20.0, 100)):
        with pytest.raises(ValueError, match="length_penalty"):
            engine.generate(ids, max_new_tokens=new, num_beams=2, length_penalty=penalty)
    assert engine.cache is None


@pytest.mark.parametrize("penalty", [30.0, 57.0])
def test_large_penalties(monkeypatch, penalty):
    monkeypatch.setattr(kernels, "beam_select", lambda x, s, n: (lambda t, b, k: (t.float(), b, k))(*plain_select(x, s, n)))
    model = OuroForCausalLM.random_init(TINY, seed=1)
    first, tables = tables_of("ends", 2, 4, 3, 24, 1)
    got = table_engine(model, first, tables, "cpu").generate(torch.zeros(2, 1, dtype=torch.long), max_new_tokens=4, eos_token_id=3, num_beams=3,
                                                             length_penalty=penalty)
    for b in range(2):
        assert got[b].tolist()[1:] == plain_search(first[b], tables[b], 3, 4, 3, penalty)[1]
