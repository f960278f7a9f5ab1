"""The looped model with every loop dense, decoding from a bf16 cache in pages.

``FlashLoopEngine`` runs the reference's lazy updates; ``OuroForCausalLM.generate`` runs the model without them
and without a cache.  ``DenseEngine`` is the model without them and with one: what a FlashLoop run is compared
with at any length, and what serves models that the packed cache does not hold (grouped KV heads, another
number of loops).  Every loop of every layer has its own keys and values
(flashloop/engine.py:396-537), in pages that a table names per sequence:

* prompts of different lengths are fed together, in chunks of rows (``prefill``), and more tokens may follow
  on cached ones (``extend``): ``paged_append`` rotates q and k and places k and v, ``paged_attention`` reads;
* ``decode`` advances every sequence by a token, replaying a captured HIP graph;
* ``generate(num_beams=K)`` is beam search: ``beam_select`` takes the continuations, and ``paged_reorder`` lets
  beams share their full pages (the prompt's above all) and copies only the page that is being filled.
"""

from __future__ import annotations

import contextlib
import functools
import gc
import math
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import kernels
from ._lib import HEAD_DIM, MAX_BEAMS
from .engine import _calls_are_plain, _is_plain
from .model import MLP, OuroConfig, OuroForCausalLM, RMSNorm, RotaryEmbedding


class PagedKVCache:
    """Keys and values of ``slots`` (loop, layer) pairs for ``rows`` sequences in pages: ``k_pages`` / ``v_pages``
    bf16 [slots, pages, KV heads, page, 128], ``table`` i32 [rows, pages of a row], ``lens`` i32 [rows].

    ``shared[r]``: (row, pages): row r begins with that many pages of an earlier row."""

    def __init__(self, slots: int, rows: int, kv_heads: int, capacity: int, device, *, page_size: int = 64,
                 shared: list[tuple[int, int]] | None = None) -> None:
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if slots < 1 or rows < 1 or kv_heads < 1 or capacity < 1:
            raise ValueError(f"slots, rows, KV heads and capacity must be positive, got {slots}, {rows}, {kv_heads} and {capacity}")
        if shared and (len(shared) != rows or any(not 0 <= src <= r or pages < 0 for r, (src, pages) in enumerate(shared))):
            raise ValueError("shared must name, for every row, that row or an earlier one and how many of its pages it shares")
        width = -(-capacity // page_size)
        table, used = [], 0
        for r in range(rows):
            src, common = shared[r] if shared else (r, 0)
            common = 0 if src == r else min(common, width)
            table.append((table[src][:common] if common else []) + list(range(used, used + width - common)))
            used += width - common
        self.page_size, self.capacity = page_size, width * page_size
        self.k_pages, self.v_pages = (torch.empty(slots, used, kv_heads, page_size, HEAD_DIM, dtype=torch.bfloat16, device=device)
                                      for _ in range(2))
        self.table = torch.tensor(table, dtype=torch.int32, device=device)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=device)

    @property
    def storage_bytes(self) -> int:
        return 2 * (self.k_pages.numel() + self.v_pages.numel())

    def reorder(self, parents: torch.Tensor) -> None:
        """Row s * K + k takes over the state of row s * K + parents[s, k] (i32 [S, K])."""
        self.table.copy_(kernels.paged_reorder(self.k_pages, self.v_pages, self.table, self.lens, parents))


def _on_its_device(method):
    """A method of an engine with its model's device as the current one (kernels and captures take the current device's
    streams)."""

    @functools.wraps(method)
    def call(self, *args, **kw):
        device = self.device
        with torch.cuda.device(device) if device.type == "cuda" else contextlib.nullcontext():
            return method(self, *args, **kw)

    return call


@dataclass(frozen=True)
class DenseOutput:
    logits: torch.Tensor  # [B, vocab] f32, at each sequence's last token
    positions: tuple[int, ...]  # tokens of every sequence


class DenseEngine:
    """Prefill, decode and generate of a ragged batch (right-padded prompts) with every loop dense.

    The kernels take the modules' weights.  A prompt takes the modules as they are then (in-place changes of a weight
    are seen at any time); where a module was replaced or hooked or has another weight since, ``extend`` and ``decode``
    raise."""

    def __init__(self, model: OuroForCausalLM, *, page_size: int = 64, chunk: int = 2048, use_graphs: bool = True) -> None:
        cfg = model.config
        if int(cfg.head_dim) != HEAD_DIM:
            raise ValueError(f"head_dim={cfg.head_dim}: the HIP kernels are built for {HEAD_DIM} channels per head")
        if cfg.num_attention_heads % cfg.num_key_value_heads:
            raise ValueError("the query heads must be a multiple of the KV heads")
        if chunk < 1:
            raise ValueError(f"chunk must be positive, got {chunk}")
        self.model = model.eval()
        self.config = cfg
        self.page_size, self.chunk, self.use_graphs = page_size, int(chunk), bool(use_graphs)
        self._weights = self._plain_weights()
        self.reset()

    @classmethod
    def from_random_init(cls, model_config: OuroConfig, *, seed: int = 0, device="cuda", **kw) -> "DenseEngine":
        return cls(OuroForCausalLM.random_init(model_config, seed=seed, device=device), **kw)

    def _plain_weights(self):
        """(per layer: q, k, v, o, gate, up, down, four norms; final norm; lm_head; eps).  The kernels take the
        weights, not the modules, so modules that do more than multiply by them are refused."""
        bb = self.model.model
        eps = {float(bb.norm.eps)}
        seen = []  # (the table that a module is in, its name there, the module, its class, its tensor's name and address)

        def child(owner, name, kind, tensor=None):
            m = getattr(owner, name)
            seen.append((owner._modules, name, m, kind, tensor, getattr(m, tensor).data_ptr() if tensor and _is_plain(m, kind) else None))
            return m

        def weight(owner, name, kind=torch.nn.Linear):
            m = child(owner, name, kind, "weight")
            w = m.weight if _is_plain(m, kind) else None
            if w is None or w.dtype != torch.bfloat16 or not w.is_contiguous() or w.data_ptr() % 16 or getattr(m, "bias", None) is not None:
                raise ValueError("DenseEngine needs plain bf16 Linear and RMSNorm layers without a bias")
            if kind is RMSNorm:
                eps.add(float(m.eps))
            return w.detach()

        hidden = bb.norm.weight.numel()
        if hidden % 8 or hidden > 8192 or any(l.mlp.up_proj.weight.shape[0] % 8 for l in bb.layers):
            raise ValueError("DenseEngine needs a hidden width (up to 8192) and an MLP width that are multiples of 8")
        emb, rot = child(bb, "embed_tokens", torch.nn.Embedding, "weight"), child(bb, "rotary_emb", RotaryEmbedding, "inv_freq")
        if (not _is_plain(emb, torch.nn.Embedding) or not _is_plain(rot, RotaryEmbedding) or emb.max_norm is not None
                or emb.weight.dtype != torch.bfloat16 or not emb.weight.is_contiguous() or emb.weight.data_ptr() % 16
                or rot.inv_freq.dtype not in (torch.float32, torch.bfloat16)):
            raise ValueError("DenseEngine needs plain embedding (bf16) and rotary modules")
        layers = []
        for i, layer in enumerate(bb.layers):
            seen.append((bb.layers._modules, str(i), layer, None, None, None))
            a, m = child(layer, "self_attn", None), child(layer, "mlp", MLP)
            if not _is_plain(m, MLP):
                raise ValueError("DenseEngine needs plain MLP modules")
            layers.append((*(weight(a, n) for n in ("q_proj", "k_proj", "v_proj", "o_proj")),
                           *(weight(m, n) for n in ("gate_proj", "up_proj", "down_proj")),
                           *(weight(layer, n, RMSNorm) for n in ("input_layernorm", "input_layernorm_2", "post_attention_layernorm",
                                                                 "post_attention_layernorm_2"))))
        final, head = weight(bb, "norm", RMSNorm), weight(self.model, "lm_head")
        if len(eps) != 1:
            raise ValueError("DenseEngine needs RMSNorm layers of one eps")
        self._seen, self._held = seen, (emb.weight.detach(), rot.inv_freq)  # (held: no other tensor gets these addresses)
        return layers, final, head, eps.pop()

    def _same_modules(self) -> bool:
        """Whether the modules are those, plain and with the tensors, that ``_weights`` were taken from."""
        bb, eps = self.model.model, self._weights[3]
        if not _calls_are_plain() or len(bb.layers) != len(self._weights[0]) or bb.embed_tokens.max_norm is not None:
            return False
        for table, name, m, kind, tensor, at in self._seen:  # (340 modules of 24 layers in 0.1 ms)
            if table.get(name) is not m:
                return False
            if kind is None:
                continue
            own = m.__dict__
            if type(m) is not kind or own["_forward_hooks"] or own["_forward_pre_hooks"] or "forward" in own:
                return False
            if at is not None:
                t = own["_buffers" if kind is RotaryEmbedding else "_parameters"].get(tensor)
                if t is None or t.data_ptr() != at or own["_parameters"].get("bias") is not None or "bias" in own:
                    return False
                if kind is RMSNorm and m.eps != eps:
                    return False
        return True

    def _check_modules(self) -> None:
        if not self._same_modules():
            raise RuntimeError("a module of the model was replaced or hooked, or has another weight, since these sequences' prompts; call "
                               "reset(): the next prompt takes the modules as they are then")

    def reset(self) -> None:
        """Drop the cache and the captured step."""
        self._release()
        self.cache: PagedKVCache | None = None
        self._lens: list[int] = []  # host mirror of the cache's lengths
        self._rope = None

    def _release(self) -> None:
        if getattr(self, "_graph", None) is not None:
            self._graph.reset()
        self._graph = self._tok = self._pos = self._out = None

    @property
    def device(self) -> torch.device:
        return next(self.model.parameters()).device

    @property
    def positions(self) -> tuple[int, ...]:
        return tuple(self._lens)

    # ------------------------------------------------------------------ the layers
    def _layers(self):
        """(loop, layer, slot) in order, with each step's weights, the next input norm and the final norm."""
        layers, final, _, _ = self._weights
        loops, nl = self.config.total_ut_steps, len(layers)
        for loop in range(loops):
            for li, w in enumerate(layers):
                last = li == nl - 1
                nxt = None if last and loop == loops - 1 else layers[(li + 1) % nl][7]
                yield loop * nl + li, w, nxt, final if last else None

    def _rows(self, hid: torch.Tensor, table, lens, starts, max_q: int, max_kv: int) -> torch.Tensor:
        """The model over rows [n, hidden]; the rows after the last loop's final norm."""
        c, eps = self.cache, self._weights[3]
        _, z = kernels.norm_chain(hid, w_b=self._weights[0][0][7], eps=eps, want_h=False)
        for slot, w, nxt, final in self._layers():
            k_pages, v_pages = c.k_pages[slot], c.v_pages[slot]
            q, k, v = F.linear(z, w[0]), F.linear(z, w[1]), F.linear(z, w[2])
            kernels.paged_append(q, k, v, self._rope, k_pages, v_pages, table, lens, starts, out=q)
            o = kernels.paged_attention(q, k_pages, v_pages, table, lens, HEAD_DIM**-0.5, starts, max_q=max_q, max_kv=max_kv)
            hid, z = kernels.norm_chain(hid, x=F.linear(o, w[3]), w_a=w[8], w_b=w[9], eps=eps)
            y = F.linear(kernels.swiglu(F.linear(z, w[4]), F.linear(z, w[5])), w[6])
            hid, z = kernels.norm_chain(hid, x=y, w_a=w[10], w_f=final, w_b=nxt, eps=eps)
        return hid

    def _step(self, out: torch.Tensor) -> torch.Tensor:
        """One token a sequence, at its next position: logits into ``out``.  Up to 8 sequences of one KV head a query head
        run on the fused GEMVs (norms, rotation and SwiGLU within them), as ``FlashLoopEngine``'s steps do."""
        c, (layers, _, head, eps) = self.cache, self._weights
        c.lens.add_(1)
        self._pos.add_(1)
        bb = self.model.model
        h, cos, sin = kernels.decode_inputs(self._tok, self._pos, bb.embed_tokens.weight, bb.rotary_emb.inv_freq)
        rows = h.shape[0]
        hid, rope = h.view(rows, -1), (cos.view(rows, -1), sin.view(rows, -1))
        cfg = self.config
        if rows > 8 or cfg.num_attention_heads != cfg.num_key_value_heads or hid.shape[1] > 4096:
            h = self._rows(hid, c.table, c.lens, None, 1, c.capacity)
            return out.copy_(F.linear(h, head))
        pending = dict(w_b=layers[0][7], want_h=False)
        for slot, w, nxt, final in self._layers():
            h, (q, k, v) = kernels.gemv_chain(hid, list(w[:3]), eps=eps, epilogue=kernels.EPI_ROPE, rope=rope, **pending)
            hid = hid if h is None else h
            kernels.paged_append(None, k, v, None, c.k_pages[slot], c.v_pages[slot], c.table, c.lens)
            o = kernels.paged_attention(q, c.k_pages[slot], c.v_pages[slot], c.table, c.lens, HEAD_DIM**-0.5, max_kv=c.capacity)
            hid, act = kernels.gemv_chain(hid, list(w[4:6]), x=kernels.gemv(o, [w[3]]), w_a=w[8], w_b=w[9], eps=eps,
                                          epilogue=kernels.EPI_SWIGLU)
            pending = dict(x=kernels.gemv(act, [w[6]]), w_a=w[10], w_f=final, w_b=nxt)
        if head.shape[0] % 4:  # (the fused product takes multiples of 4 outputs)
            return out.copy_(F.linear(kernels.norm_chain(hid, eps=eps, **pending)[0], head))
        _, logits = kernels.gemv_chain(hid, [head], eps=eps, epilogue=kernels.EPI_F32, out=out, **pending)
        return logits

    # ------------------------------------------------------------------ prompts
    def _lengths(self, input_ids: torch.Tensor, attention_mask: torch.Tensor | None) -> list[int]:
        if input_ids.ndim != 2 or input_ids.shape[0] < 1 or input_ids.shape[1] < 1:
            raise ValueError("input_ids must be [B, T] with B, T >= 1")
        if input_ids.device != self.device:
            raise ValueError(f"input_ids lie on {input_ids.device}, the model on {self.device}")
        if attention_mask is None:
            return [input_ids.shape[1]] * input_ids.shape[0]
        if tuple(attention_mask.shape) != tuple(input_ids.shape):
            raise ValueError("attention_mask must have the shape of input_ids")
        m = attention_mask.to(torch.bool).cpu()
        lengths = [int(x) for x in m.sum(dim=1).tolist()]
        for b, n in enumerate(lengths):
            if not bool(m[b, :n].all()):
                raise ValueError("prompts must be right-padded (attention_mask 1...1 0...0)")
        return lengths

    def _feed(self, input_ids: torch.Tensor, counts: list[int], rows: list[int]) -> torch.Tensor:
        """The first counts[i] tokens of input_ids[i] onto cache row rows[i], at most ``chunk`` rows of all of them
        at a time; the logits [len(rows), vocab] of each one's last token."""
        c, dev = self.cache, input_ids.device
        at = torch.tensor(rows, device=dev)
        table = c.table.index_select(0, at)
        done = [0] * len(rows)
        last = torch.empty(len(rows), self.config.hidden_size, dtype=torch.bfloat16, device=dev)
        while any(d < n for d, n in zip(done, counts)):
            room, step = self.chunk, []
            for d, n in zip(done, counts):
                step.append(min(n - d, room))
                room -= step[-1]
            starts = [0]
            for r in step:
                starts.append(starts[-1] + r)
            for i, r in enumerate(step):
                self._lens[rows[i]] += r
            lens = [self._lens[r] for r in rows]
            meta = torch.tensor(starts + lens, dtype=torch.int32).to(dev)
            ids = torch.cat([input_ids[i, d: d + r] for i, (d, r) in enumerate(zip(done, step)) if r])
            h = self._rows(self.model.model.embed_tokens(ids), table, meta[len(starts):].contiguous(), meta[: len(starts)].contiguous(),
                           max(step), max(lens))
            ends = [i for i, (d, r, n) in enumerate(zip(done, step, counts)) if r and d + r == n]
            if ends:
                last[ends] = h[[starts[i + 1] - 1 for i in ends]]
            done = [d + r for d, r in zip(done, step)]
        self._lengths_to_device()
        return F.linear(last, self._weights[2]).float()

    def _lengths_to_device(self) -> None:
        self.cache.lens.copy_(torch.tensor(self._lens, dtype=torch.int32))
        if self._pos is not None:
            self._pos.copy_(torch.tensor(self._lens)[:, None] - 1)

    def _begin(self, input_ids: torch.Tensor, counts: list[int], extra: int, beams: int) -> None:
        if not self._same_modules():
            self._weights = self._plain_weights()
        capacity = max(counts) + int(extra)
        cfg, dev = self.config, input_ids.device
        shared = None
        if beams > 1:  # the beams of a sequence begin with the full pages of its prompt
            shared = [(b * beams, n // self.page_size) for b, n in enumerate(counts) for _ in range(beams)]
        self.cache = PagedKVCache(cfg.total_ut_steps * len(self._weights[0]), len(counts) * beams, cfg.num_key_value_heads, capacity, dev,
                                  page_size=self.page_size, shared=shared)
        self._lens = [0] * (len(counts) * beams)
        probe = torch.empty(0, dtype=torch.bfloat16, device=dev)
        self._rope = tuple(t[0].contiguous() for t in
                           self.model.model.rotary_emb(probe, torch.arange(self.cache.capacity, device=dev)[None]))

    @_on_its_device
    @torch.inference_mode()
    def prefill(self, input_ids: torch.Tensor, attention_mask: torch.Tensor | None = None, *,
                decode_capacity: int = 4096) -> DenseOutput:
        """Feed ``input_ids`` [B, T] (right-padded; ``attention_mask`` marks the real tokens) into a new cache with room for
        ``decode_capacity`` more tokens a sequence."""
        if self.cache is not None:
            raise RuntimeError("engine cache is already initialized; call reset()")
        counts = self._lengths(input_ids, attention_mask)
        if min(counts) < 1:
            raise ValueError(f"sequence {counts.index(min(counts))} has no tokens")
        if decode_capacity < 0:
            raise ValueError(f"decode_capacity={decode_capacity} is negative")
        logits = self._first(input_ids, counts, decode_capacity, 1)
        return DenseOutput(logits, self.positions)

    def _first(self, input_ids: torch.Tensor, counts: list[int], extra: int, beams: int) -> torch.Tensor:
        """Prompts into a new cache, each on the first of its beams' rows; no cache is left if that fails."""
        try:
            self._begin(input_ids, counts, extra, beams)
            return self._feed(input_ids, counts, list(range(0, len(counts) * beams, beams)))
        except BaseException:
            self.reset()
            raise

    @_on_its_device
    @torch.inference_mode()
    def extend(self, input_ids: torch.Tensor, attention_mask: torch.Tensor | None = None) -> DenseOutput:
        """More tokens [B, T] (right-padded, at least one a sequence) onto the cached sequences: the logits of the last."""
        self._need()
        counts = self._lengths(input_ids, attention_mask)
        if len(counts) != len(self._lens):
            raise ValueError(f"extend takes tokens for {len(self._lens)} sequences, got {len(counts)}")
        if min(counts) < 1:
            raise ValueError(f"sequence {counts.index(min(counts))} has no tokens")
        self._room(counts)
        self._check_modules()
        before = list(self._lens)
        try:
            logits = self._feed(input_ids, counts, list(range(len(counts))))
        except BaseException:  # (what was fed lies behind the sequences' ends, where the next call writes)
            self._lens = before
            self._lengths_to_device()
            raise
        return DenseOutput(logits, self.positions)

    def _need(self) -> None:
        if self.cache is None:
            raise RuntimeError("engine cache has not been initialized; call prefill() first")

    def _room(self, counts) -> None:
        for b, (t, n) in enumerate(zip(self._lens, counts)):
            if t + n > self.cache.capacity:
                raise ValueError(f"sequence {b} has {t} tokens: the cache has room for {self.cache.capacity} (decode_capacity)")

    # ------------------------------------------------------------------ decode
    @_on_its_device
    @torch.inference_mode()
    def decode(self, token_ids: torch.Tensor) -> DenseOutput:
        """One token for every sequence: ``token_ids`` [B, 1].  With graphs on, the returned logits live in the graph's
        output buffer until the next step.  A token outside the vocabulary gives its sequence NaN logits and rows
        (``FlashLoopEngine.decode``)."""
        self._need()
        rows = len(self._lens)
        if tuple(token_ids.shape) != (rows, 1):
            raise ValueError(f"decode requires token_ids of shape ({rows}, 1)")
        self._room([1] * rows)
        try:
            logits = self._advance(token_ids)
            self._check_modules()  # (while the GPU runs the step)
        except BaseException:  # (a step counts its token before it runs)
            self._release()
            self._lengths_to_device()
            raise
        self._lens = [t + 1 for t in self._lens]
        return DenseOutput(logits, self.positions)

    def _advance(self, token_ids: torch.Tensor) -> torch.Tensor:
        rows, dev = len(self._lens), self.cache.lens.device
        if self._out is None:
            self._out = torch.empty(rows, self.config.vocab_size, dtype=torch.float32, device=dev)
            self._tok = torch.zeros(rows, 1, dtype=torch.long, device=dev)
            self._pos = (self.cache.lens - 1).long()[:, None]  # (of the last token: a step writes the next)
        self._tok.copy_(token_ids)
        if not self.use_graphs:
            return self._step(torch.empty_like(self._out))
        if self._graph is None:
            self._capture()
        self._graph.replay()
        return self._out

    def _capture(self) -> None:
        """Capture a step (lengths live on the device).  A warm-up on a side stream sizes workspaces and library
        handles; it writes the rows that the replay writes again."""
        side = torch.cuda.Stream()  # default priority
        side.wait_stream(torch.cuda.current_stream())
        try:
            with torch.cuda.stream(side):
                self._step(self._out)
                self.cache.lens.sub_(1)
                self._pos.sub_(1)
        finally:
            torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        was_enabled = gc.isenabled()
        gc.disable()  # (a graph destroyed by a collection during a capture aborts the process)
        try:
            with torch.cuda.graph(graph):
                self._step(self._out)
        except BaseException:
            graph.reset()
            raise
        finally:
            if was_enabled:
                gc.enable()
        self._graph = graph

    # ------------------------------------------------------------------ generate
    @_on_its_device
    @torch.inference_mode()
    def generate(self, input_ids: torch.Tensor, attention_mask: torch.Tensor | None = None, *, max_new_tokens: int,
                 eos_token_id: int | None = None, num_beams: int = 1, length_penalty: float = 1.0) -> list[torch.Tensor]:
        """Greedy generation, or beam search with ``num_beams`` > 1: each sequence's prompt and completion (1-D).

        Beam search returns the completion with the largest sum of log-probabilities divided by
        length ** ``length_penalty`` (tokens of the completion, the EOS among them) of those that ended and those still running
        at the end.  Of a step's 2 * ``num_beams`` best continuations an EOS ends those among the first ``num_beams``; the best others go
        on.  A sequence's search ends when none of its running beams can pass the best one that ended."""
        if int(max_new_tokens) <= 0:
            raise ValueError("max_new_tokens must be positive")
        if not 1 <= num_beams <= MAX_BEAMS // 2:
            raise ValueError(f"num_beams must be 1..{MAX_BEAMS // 2}, got {num_beams}")
        if not length_penalty >= 0:
            raise ValueError(f"length_penalty={length_penalty} is negative")
        # (sums of log-probabilities are fp32, and so are their quotients)
        if num_beams > 1 and not length_penalty * math.log(int(max_new_tokens)) < 80:
            raise ValueError(f"length_penalty={length_penalty}: {max_new_tokens} ** length_penalty is past fp32's range")
        if 2 * num_beams > self.config.vocab_size:
            raise ValueError(f"num_beams={num_beams} needs a vocabulary of {2 * num_beams}")
        if self.cache is not None:
            raise RuntimeError("engine cache is already initialized; call reset()")
        if eos_token_id is None:
            eos_token_id = getattr(self.config, "eos_token_id", None)
        try:
            if num_beams == 1:
                return self._greedy(input_ids, attention_mask, int(max_new_tokens), eos_token_id)
            return self._beams(input_ids, attention_mask, int(max_new_tokens), eos_token_id, num_beams, float(length_penalty))
        except BaseException:
            self.reset()
            raise

    def _greedy(self, input_ids, attention_mask, new, eos) -> list[torch.Tensor]:
        counts = self._lengths(input_ids, attention_mask)
        logits = self.prefill(input_ids, attention_mask, decode_capacity=new).logits
        done = torch.zeros(len(counts), dtype=torch.bool, device=input_ids.device)
        steps = []
        for step in range(new):
            nxt = torch.argmax(logits, dim=-1, keepdim=True)
            steps.append((nxt[:, 0].clone(), done.clone()))
            if eos is not None:
                done = done | (nxt[:, 0] == int(eos))
                if bool(done.all()):
                    break
            if step + 1 < new:
                logits = self.decode(nxt).logits
        tokens, ended = torch.stack([s[0] for s in steps], 1), torch.stack([s[1] for s in steps], 1)
        return [torch.cat([input_ids[b, :n], tokens[b][~ended[b]]]) for b, n in enumerate(counts)]

    def _beams(self, input_ids, attention_mask, new, eos, k, penalty) -> list[torch.Tensor]:
        counts = self._lengths(input_ids, attention_mask)
        if min(counts) < 1:
            raise ValueError(f"sequence {counts.index(min(counts))} has no tokens")
        bsz, dev = len(counts), input_ids.device
        logits = self._first(input_ids, counts, new, k).repeat_interleave(k, dim=0)
        self._lens = [n for n in counts for _ in range(k)]
        self._lengths_to_device()
        scores = torch.full((bsz, k), -torch.inf, device=dev)  # (the beams are one until they part)
        scores[:, 0] = 0.0
        history = torch.zeros(bsz, k, new, dtype=torch.long, device=dev)
        best = torch.full((bsz,), -torch.inf, device=dev)
        best_tokens = torch.zeros(bsz, new, dtype=torch.long, device=dev)
        best_len = torch.zeros(bsz, dtype=torch.long, device=dev)

        def keep(value, tokens, length):
            """Take completions [B] that pass the best so far."""
            nonlocal best, best_tokens, best_len
            better = value > best
            best = torch.where(better, value, best)
            best_tokens = torch.where(better[:, None], tokens, best_tokens)
            best_len = torch.where(better, length, best_len)

        for step in range(new):
            top, parents, tokens = kernels.beam_select(logits, scores, 2 * k)
            past = torch.gather(history, 1, parents.long()[..., None].expand(-1, -1, new))
            past[:, :, step] = tokens
            if eos is None:
                order = torch.arange(k, device=dev).expand(bsz, k)
            else:
                ends = tokens == int(eos)
                value = torch.where(ends, top, -torch.inf)[:, :k] / (step + 1) ** penalty
                value, at = value.max(1)
                keep(value, torch.gather(past, 1, at[:, None, None].expand(-1, 1, new))[:, 0], torch.full_like(best_len, step + 1))
                order = torch.sort(ends.int(), dim=1, stable=True).indices[:, :k]  # those that go on, the best first
            scores = torch.gather(top, 1, order)
            history = torch.gather(past, 1, order[..., None].expand(-1, -1, new))
            if step + 1 == new:
                break
            # a sum only falls and a completion is at most `new` long: no running beam ends above this
            if eos is not None and bool((scores[:, 0] / new**penalty <= best).all()):
                break
            self.cache.reorder(torch.gather(parents, 1, order).contiguous())
            logits = self.decode(torch.gather(tokens, 1, order).view(-1, 1)).logits
        if step + 1 == new:
            keep(scores[:, 0] / new**penalty, history[:, 0], torch.full_like(best_len, new))
        return [torch.cat([input_ids[b, :n], best_tokens[b, : int(l)]]) for b, (n, l) in enumerate(zip(counts, best_len.tolist()))]
