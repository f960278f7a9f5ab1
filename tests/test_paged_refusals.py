"""What the operators on K/V pages, the beam selection and DenseEngine refuse, without a GPU: malformed tensors
in the front end, and in the C ABI every argument that is checked before a launch."""

import dataclasses

import pytest
import torch

from flashloop_amd import DenseEngine, PagedKVCache, _lib, kernels
from flashloop_amd.model import OuroConfig, OuroForCausalLM
from paged_util import plain_reorder, plain_select

needs_library = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="library not built")
BF = torch.bfloat16


def _pages(n=4, kv=2, page=16):
    return torch.zeros(n, kv, page, 128, dtype=BF), torch.zeros(n, kv, page, 128, dtype=BF)


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@needs_library
def test_paged_operands():
    k, v = _pages()
    q = torch.zeros(3, 512, dtype=BF)
    kv = torch.zeros(3, 256, dtype=BF)
    rope = torch.zeros(9, 128, dtype=BF), torch.zeros(9, 128, dtype=BF)
    table, lens = _i32(3, 2), _i32(3)
    attend = lambda *a, **kw: kernels.paged_attention(*a, **kw)
    with pytest.raises(RuntimeError, match="device"):
        attend(q, k, v, table, lens, 0.1)
    with pytest.raises(RuntimeError, match="device"):
        kernels.paged_append(q, kv, kv, rope, k, v, table, lens)
    for bad in ((k[..., :64], v[..., :64]), (k, v[:3]), (k[0], v[0]), (k.float(), v.float()), (k, v.float()),
                (k.transpose(0, 1), v.transpose(0, 1))):
        with pytest.raises(ValueError, match="pages"):
            attend(q, *bad, table, lens, 0.1)
        with pytest.raises(ValueError):
            kernels.paged_append(q, kv, kv, rope, *bad, table, lens)
    for t, l, s in ((table[0], lens, None), (table, lens[:2], None), (table.long(), lens, None), (table, lens.long(), None),
                    (table, lens, _i32(4).long()), (table.t().contiguous().t(), lens, None)):
        with pytest.raises(ValueError, match="page_table|kv_lens|q_starts"):
            attend(q, k, v, t, l, 0.1, s)
    with pytest.raises(ValueError, match="one row a sequence"):
        attend(q[:2], k, v, table, lens, 0.1)
    with pytest.raises(ValueError, match="q_starts"):
        attend(q, k, v, table, lens, 0.1, _i32(3))
    for bad in (q.float(), q[:, :100], q[0], q[:, :0]):
        with pytest.raises(ValueError, match="q must be"):
            attend(bad, k, v, table, lens, 0.1)
    with pytest.raises(ValueError, match="share"):
        attend(q[:, :384], k, v, table, lens, 0.1)
    with pytest.raises(ValueError, match="k and v"):
        kernels.paged_append(q, kv[:, :128], kv[:, :128], rope, k, v, table, lens)
    with pytest.raises(ValueError, match="k and v"):
        kernels.paged_append(q, kv, kv[:2], rope, k, v, table, lens)
    with pytest.raises(ValueError, match="without q"):
        kernels.paged_append(None, kv, kv, rope, k, v, table, lens)
    with pytest.raises(ValueError, match="no out"):
        kernels.paged_append(q, kv, kv, None, k, v, table, lens, out=q)
    with pytest.raises(ValueError, match="rows, k"):
        kernels.paged_append(q[:2], kv, kv, rope, k, v, table, lens)
    for bad in ((rope[0][:, :64], rope[1][:, :64]), (rope[0], rope[1].float()), (rope[0].half(), rope[1].half()), (rope[0], rope[1][:5])):
        with pytest.raises(ValueError, match="rope"):
            kernels.paged_append(q, kv, kv, bad, k, v, table, lens)
    for bad in (q.float(), q[:2], torch.zeros(3, 514, dtype=BF)[:, ::1][:, :512].t().contiguous().t()):
        with pytest.raises(ValueError, match="out"):
            kernels.paged_append(q, kv, kv, rope, k, v, table, lens, out=bad)


@needs_library
def test_beam_operands():
    x, s = torch.zeros(6, 50), torch.zeros(2, 3)
    with pytest.raises(RuntimeError, match="device"):
        kernels.beam_select(x, s)
    for bad in (s[0], s.double()):
        with pytest.raises(ValueError, match="scores"):
            kernels.beam_select(x, bad)
    for bad in (x[:5], x[0], x[None]):
        with pytest.raises(ValueError, match="logits"):
            kernels.beam_select(bad, s)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        kernels.beam_select(x.half(), s)
    for count in (0, 65, 200):
        with pytest.raises(ValueError, match="count"):
            kernels.beam_select(x, s, count)
    with pytest.raises(ValueError, match="count"):
        kernels.beam_select(x[:, :1], s, 4)
    with pytest.raises(ValueError, match="beams"):
        kernels.beam_select(torch.zeros(65, 9), torch.zeros(1, 65), 3)
    k, v = _pages()
    table, lens, parents = _i32(4, 2), _i32(4), _i32(2, 2)
    with pytest.raises(RuntimeError, match="device"):
        kernels.paged_reorder(k, v, table, lens, parents)
    with pytest.raises(ValueError, match="pages"):
        kernels.paged_reorder(k, v[:2], table, lens, parents)
    with pytest.raises(ValueError, match="pages"):
        kernels.paged_reorder(k.float(), v.float(), table, lens, parents)
    for t, l, p in ((table[:3], lens, parents), (table, lens[:3], parents), (table, lens, parents[0]), (table.long(), lens, parents),
                    (table, lens, parents.long())):
        with pytest.raises(ValueError):
            kernels.paged_reorder(k, v, t, l, p)


@needs_library
def test_c_abi_refusals():
    lib = _lib.load()
    p = 0x10000

    def says(rc, text):
        assert rc == _lib.FL_E_INVALID and text in lib.fl_last_error(), (rc, lib.fl_last_error())

    def attend(q=p, stride=512, k=p, table=p, starts=None, rows=3, seqs=3, heads=4, kv=2, width=2, pages=4, page=16, max_q=1, max_kv=32,
               scaling=0.1):
        return lib.fl_paged_attention(q, stride, k, p, p, table, p, starts, rows, seqs, heads, kv, width, pages, page, max_q, max_kv,
                                      scaling, None, 0, None)

    says(attend(q=None), b"null")
    says(attend(table=None), b"null")
    says(attend(rows=-1), b"sizes")
    says(attend(pages=0), b"sizes")
    says(attend(heads=3), b"multiple")
    for page in (8, 24, 2048):
        says(attend(page=page), b"page size")
    says(attend(stride=504), b"stride")
    says(attend(stride=516), b"stride")
    says(attend(seqs=2), b"one row")
    says(attend(max_q=0), b"max_q")
    says(attend(scaling=0.0), b"scaling")
    says(attend(scaling=float("nan")), b"scaling")
    says(attend(scaling=float("inf")), b"scaling")
    says(attend(width=1 << 28), b"too many tokens")
    says(attend(k=p + 8), b"aligned")
    says(attend(starts=p, seqs=0), b"without a sequence")
    says(attend(starts=p, rows=1 << 30, seqs=1, heads=8, kv=1, stride=1024), b"too many rows")
    assert attend(rows=0, seqs=0) == _lib.FL_OK
    assert lib.fl_paged_attention_workspace(0, 1, 1, 1, 1, 1) == 0 == lib.fl_paged_attention_workspace(1, 1, 3, 2, 1, 1)

    def append(q=p, qs=512, k=p, ks=256, out=p, cos=p, sin=p, positions=9, rows=3, seqs=3, heads=4, kv=2, width=2, pages=4, page=16,
               starts=None):
        return lib.fl_paged_append(q, qs, k, ks, p, 256, out, 512, cos, sin, 0, positions, p, p, p, p, starts, rows, seqs, heads, kv,
                                   width, pages, page, None)

    says(append(k=None), b"null")
    says(append(sin=None), b"one rope table")
    says(append(q=None), b"null q")
    says(append(positions=0), b"rope")
    says(append(kv=0), b"head")
    says(append(page=12), b"page size")
    says(append(rows=2), b"one row")
    says(append(ks=248), b"stride")
    says(append(qs=504), b"stride")
    says(append(q=p + 2), b"aligned")
    says(append(starts=p, seqs=0), b"without a sequence")
    assert append(rows=0, seqs=0) == _lib.FL_OK

    def select(x=p, stride=50, seqs=2, beams=3, vocab=50, count=6, ws=p, size=1 << 20):
        return lib.fl_beam_select(x, 1, stride, p, seqs, beams, vocab, count, p, p, p, ws, size, None)

    says(select(x=None), b"null")
    says(select(beams=0), b"beams")
    says(select(beams=65), b"beams")
    says(select(vocab=0), b"tokens")
    says(select(count=65), b"candidates")
    says(select(vocab=1, count=4, stride=1), b"candidates")
    says(select(stride=49), b"overlap")
    says(select(x=p + 2), b"aligned")
    says(select(ws=None), b"workspace")
    says(select(size=8), b"workspace")
    assert select(seqs=0) == _lib.FL_OK

    def reorder(k=p, table=p, out=2 * p, seqs=2, beams=2, layers=1, width=2, pages=4, kv=2, page=16):
        return lib.fl_paged_reorder(k, p, table, out, p, p, seqs, beams, layers, width, pages, kv, page, None)

    says(reorder(k=None), b"null")
    says(reorder(out=p), b"old one")
    says(reorder(layers=0), b"sizes")
    says(reorder(beams=65), b"beams")
    says(reorder(page=20), b"page size")
    says(reorder(k=p + 8), b"aligned")
    says(reorder(seqs=40000), b"too many beams")
    assert reorder(seqs=0) == _lib.FL_OK


TINY = OuroConfig(vocab_size=64, hidden_size=128, intermediate_size=256, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1)


def test_dense_engine_refusals():
    model = OuroForCausalLM.random_init(TINY, seed=1)
    engine = DenseEngine(model)  # (weights are looked at, nothing is run)
    ids = torch.zeros(2, 4, dtype=torch.long)
    with pytest.raises(RuntimeError, match="prefill"):
        engine.decode(ids[:, :1])
    with pytest.raises(RuntimeError, match="prefill"):
        engine.extend(ids)
    with pytest.raises(ValueError, match="right-padded"):
        engine.prefill(ids, torch.tensor([[0, 1, 1, 1], [1, 1, 1, 1]]))
    with pytest.raises(ValueError, match="no tokens"):
        engine.prefill(ids, torch.tensor([[0, 0, 0, 0], [1, 1, 1, 1]]))
    with pytest.raises(ValueError, match="shape"):
        engine.prefill(ids, torch.ones(2, 3))
    with pytest.raises(ValueError, match="decode_capacity"):
        engine.prefill(ids, decode_capacity=-1)
    with pytest.raises(ValueError, match="B, T"):
        engine.prefill(ids[0])
    for kw, match in (({"max_new_tokens": 0}, "max_new_tokens"), ({"max_new_tokens": 1, "num_beams": 0}, "num_beams"),
                      ({"max_new_tokens": 1, "num_beams": 33}, "num_beams"), ({"max_new_tokens": 1, "num_beams": 2, "length_penalty": -1.0}, "length")):
        with pytest.raises(ValueError, match=match):
            engine.generate(ids, **kw)
    with pytest.raises(ValueError, match="chunk"):
        DenseEngine(model, chunk=0)
    with pytest.raises(ValueError, match="page_size"):
        PagedKVCache(1, 1, 1, 10, "cpu", page_size=24)
    with pytest.raises(ValueError, match="channels"):
        DenseEngine(OuroForCausalLM.random_init(dataclasses.replace(TINY, head_dim=64), seed=1))
    with pytest.raises(ValueError, match="multiple"):
        DenseEngine(OuroForCausalLM.random_init(dataclasses.replace(TINY, num_attention_heads=3, num_key_value_heads=2), seed=1))
    with pytest.raises(ValueError, match="bf16"):
        DenseEngine(OuroForCausalLM.random_init(TINY, seed=1, dtype=torch.float32))
    hooked = OuroForCausalLM.random_init(TINY, seed=1)
    hooked.model.layers[0].self_attn.q_proj.register_forward_hook(lambda *a: None)
    with pytest.raises(ValueError, match="plain"):
        DenseEngine(hooked)


def test_shared_tables():
    cache = PagedKVCache(2, 6, 1, 50, "cpu", page_size=16, shared=[(0, 2)] * 3 + [(3, 0)] * 3)
    table = cache.table.tolist()
    assert cache.capacity == 64 and cache.k_pages.shape == (2, 4 + 2 * 2 + 3 * 4, 1, 16, 128)
    assert table[1][:2] == table[0][:2] == table[2][:2] and cache.storage_bytes == 4 * cache.k_pages.numel()
    own = [p for r in table[:1] for p in r] + [p for r in table[1:3] for p in r[2:]] + [p for r in table[3:] for p in r]
    assert sorted(own) == list(range(20))


def test_plain_forms():
    """The definitions that the GPU tests compare with, on cases worked out by hand."""
    x = torch.log(torch.tensor([[0.5, 0.25, 0.25], [0.1, 0.8, 0.1]]))
    best, beams, tokens = plain_select(x, torch.log(torch.tensor([[0.5, 0.25]])), 4)
    assert beams.tolist() == [[0, 1, 0, 0]] and tokens.tolist() == [[0, 1, 1, 2]]
    assert torch.allclose(best, torch.log(torch.tensor([[0.25, 0.2, 0.125, 0.125]], dtype=torch.float64)), atol=1e-6)
    best, beams, tokens = plain_select(x, torch.tensor([[-torch.inf, 0.0]]), 5)
    assert beams.tolist() == [[1, 1, 1, 0, 0]] and tokens.tolist() == [[1, 0, 2, 0, 1]]
    new, copies = plain_reorder([[0, 1, 2], [0, 3, 4], [0, 5, 6]], 20, [[1, 1, 0]], 16)
    assert new == [[0, 3, 2], [0, 5, 4], [0, 1, 6]] and copies == [(0, 3, 5)]
