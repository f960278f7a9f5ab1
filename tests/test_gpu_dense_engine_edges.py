"""DenseEngine on models of unusual sizes and after calls that failed."""

import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu

from beam_util import CASES, plain_search, table_engine, tables_of  # noqa: E402
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


class _Stop(Exception):
    pass


def _stops_at(monkeypatch, name, calls):
    """kernels.<name> raises at its ``calls``-th call from now on, once."""
    from flashloop_amd import kernels

    plain, left = getattr(kernels, name), [calls]

    def call(*a, **kw):
        left[0] -= 1
        if left[0] == 0:
            raise _Stop(name)
        return plain(*a, **kw)

    monkeypatch.setattr(kernels, name, call)


@pytest.mark.parametrize("rows", [2, 9])
@pytest.mark.parametrize("graphs,calls", [(False, 3), (True, 3), (True, 11)])
def test_steps_that_fail_leave_the_sequences_as_they_were(monkeypatch, rows, graphs, calls):
    """A step that raises half-way, in its warm-up and in its capture (8 layers and loops): positions, lengths on the
    device and the cache are those before it, and the next steps are the same as without it."""
    print(f"case: dense engine failing step rows {rows} graphs {graphs} calls {calls}", flush=True)
    model = OuroForCausalLM.random_init(TINY, seed=12, device="cuda")
    ids = _ids(rows, 20, TINY.vocab_size)
    engine, plain = (DenseEngine(model, use_graphs=graphs, page_size=16) for _ in range(2))
    for e in (engine, plain):
        e.prefill(ids[:, :14], decode_capacity=8)
    with monkeypatch.context() as m:
        _stops_at(m, "paged_attention", calls)
        with pytest.raises(_Stop):
            engine.decode(ids[:, 14:15])
    assert engine.positions == (14,) * rows and engine.cache.lens.tolist() == [14] * rows
    for t in range(14, 17):
        assert torch.equal(engine.decode(ids[:, t: t + 1]).logits, plain.decode(ids[:, t: t + 1]).logits), t
    # more tokens that stop in their second chunk
    engine.chunk = 2 * rows - 1
    with monkeypatch.context() as m:
        _stops_at(m, "paged_attention", 8 + 3)
        with pytest.raises(_Stop):
            engine.extend(ids[:, 17:19])
    assert engine.positions == (17,) * rows and engine.cache.lens.tolist() == [17] * rows
    engine.chunk = plain.chunk
    assert torch.equal(engine.extend(ids[:, 17:19]).logits, plain.extend(ids[:, 17:19]).logits)
    assert torch.equal(engine.decode(ids[:, 19:20]).logits, plain.decode(ids[:, 19:20]).logits)


def test_prompts_that_fail_leave_no_cache(monkeypatch):
    print("case: dense engine failing prompt", flush=True)
    model = OuroForCausalLM.random_init(TINY, seed=13, device="cuda")
    ids = _ids(2, 9, TINY.vocab_size)
    engine = DenseEngine(model)
    for call in (lambda: engine.prefill(ids), lambda: engine.generate(ids, max_new_tokens=3),
                 lambda: engine.generate(ids, max_new_tokens=3, num_beams=2)):
        with monkeypatch.context() as m:
            _stops_at(m, "paged_attention", 5)
            with pytest.raises(_Stop):
                call()
        assert engine.cache is None and engine.positions == ()
    assert torch.equal(engine.prefill(ids).logits, DenseEngine(model).prefill(ids).logits)


def test_generation_that_fails_can_begin_again(monkeypatch):
    """A step or a rearrangement that raises on the way: no cache is left, and the same call then gives what it gives without."""
    print("case: dense engine failing generation", flush=True)
    model = OuroForCausalLM.random_init(TINY, seed=14, device="cuda")
    ids = _ids(2, 20, TINY.vocab_size)
    engine = DenseEngine(model, page_size=16)
    for beams, name, calls in ((1, "paged_attention", 8 + 3), (3, "paged_attention", 8 + 8 + 5), (3, "paged_reorder", 2), (3, "beam_select", 3)):
        want = DenseEngine(model, page_size=16).generate(ids, max_new_tokens=6, num_beams=beams)
        with monkeypatch.context() as m:
            _stops_at(m, name, calls)
            with pytest.raises(_Stop):
                engine.generate(ids, max_new_tokens=6, num_beams=beams)
        assert engine.cache is None and engine.positions == ()
        got = engine.generate(ids, max_new_tokens=6, num_beams=beams)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        engine.reset()


@pytest.mark.parametrize("beams,new,eos,penalty,kind", CASES)
def test_beam_search_on_tables(beams, new, eos, penalty, kind):
    """The search with the selection's kernel against a plain one, on logits from tables."""
    print(f"case: beams on tables {beams} {new} {eos} {penalty} {kind}", flush=True)
    model = OuroForCausalLM.random_init(dataclasses.replace(TINY, vocab_size=24, num_hidden_layers=1), seed=1, device="cuda")
    prompts = _ids(5, 3, 24)
    for seed in range(3):
        first, tables = tables_of(kind, 5, new, eos, 24, 10 + seed)
        got = table_engine(model, first, tables, "cuda").generate(prompts, max_new_tokens=new, eos_token_id=eos, num_beams=beams,
                                                                   length_penalty=penalty)
        for b in range(5):
            want = plain_search(first[b], tables[b], beams, new, eos, penalty)
            assert got[b].tolist() == prompts[b].tolist() + want[1], (seed, b, want)
