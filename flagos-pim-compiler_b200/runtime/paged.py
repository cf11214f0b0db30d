"""LLaMA decoding over a paged KV cache: batches, beam search, caches of bounded size.

``PagedLlama`` runs the weights of a compiled program (one rank) with a cache of pages beside the program's static one:

    runner = LlamaRunner(prog, hal); runner.load_checkpoint("<hf dir>")
    gen = PagedLlama(runner, rows=4, max_slots=512)
    out = gen.greedy(prompts, steps=64)                 # [rows, prompt_len] ids -> [rows, steps]
    best = gen.beam_search(prompt, steps=64, eos=2)     # rows beams of one prompt
    gen = PagedLlama(runner, rows=4, max_slots=512, budget=256, recent=64, sink=4)   # evicts to 256 slots a head

A prompt goes through the program's prefill plan (which overwrites the program's static cache), whose KV blocks are then
copied into the row's pages, with accumulated weights of 0 where the cache is bounded; from there on a step is the decode
plan's projections around ``PagedAppend`` / ``PagedAttention`` (and ``PagedEvict``) for all rows at once, captured into one
CUDA graph after its first run.  Everything runs on the rank's stream.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import numpy as np

from backend import _native as nat
from backend.cuda_paged import BeamReorder, BeamSelect, PagedAppend, PagedAttention, PagedEvict, complaints, forget
from memory.paged_kv import PagedKVCache, PagedKVSpec
from runtime.executor import execute_plan


@dataclass
class BeamResult:
    tokens: np.ndarray  # [beams, steps], best beam first
    scores: np.ndarray  # [beams] sum of log-probabilities
    done: np.ndarray    # [beams] whether the beam met `eos`


class PagedLlama:
    def __init__(self, runner, rows: int, max_slots: int, *, page_size: int = 16, budget: int | None = None,
                 recent: int = 0, sink: int = 0, num_pages: int | None = None) -> None:
        import torch

        prog, hal = runner.prog, runner.hal
        if prog.tp != 1 or prog.batch != 1 or "prefill" not in prog.plans:
            raise ValueError("PagedLlama takes a program of one rank and one sequence with a prefill plan")
        self.torch, self.prog, self.hal, self.cfg = torch, prog, hal, prog.cfg
        cfg = prog.cfg
        if max_slots < max(prog.prompt_len, budget or 0) + 1:
            raise ValueError(f"max_slots={max_slots} leaves no room to decode after a {prog.prompt_len}-token prompt, or "
                             f"for a token over the budget")
        if budget is not None and not (0 < budget and recent >= 0 and sink >= 0 and recent + sink <= budget):
            raise ValueError("budget must be positive and at least recent + sink")
        self.rows, self.budget = rows, budget
        self.stream = hal.stream(0)
        self.device = torch.device("cuda", hal.device_of(0))
        max_pages = -(-max_slots // page_size)
        self.spec = PagedKVSpec(cfg.num_layers, cfg.num_kv_heads, cfg.head_dim, cfg.dtype, page_size,
                                num_pages or rows * max_pages, rows, max_pages)
        dt = {"float32": torch.float32, "bfloat16": torch.bfloat16}[cfg.dtype]
        with torch.cuda.device(self.device), torch.cuda.stream(self.stream):
            self.cache = PagedKVCache(self.spec, self.device, track=budget is not None)

            def buf(*shape, dtype=dt):
                return torch.zeros(*shape, dtype=dtype, device=self.device)

            hd, hq, hkv = cfg.head_dim, cfg.num_heads, cfg.num_kv_heads
            self.ids = buf(rows, dtype=torch.int32)
            self.lengths, self.next_lengths, self.cut_lengths = (buf(rows, dtype=torch.int32) for _ in range(3))
            self.positions, self.next_positions = (buf(rows, dtype=torch.int32) for _ in range(2))
            self.x, self.h = buf(rows, cfg.hidden_size), buf(rows, cfg.hidden_size)
            self.qkv = buf(rows, (hq + 2 * hkv) * hd)
            self.q_rot, self.attn = buf(rows, hq, hd), buf(rows, hq, hd)
            self.act, self.logits = buf(rows, cfg.intermediate_size), buf(rows, cfg.vocab_size)
            self.next_ids = buf(rows, dtype=torch.int32)
            self.err = buf(2, dtype=torch.int32)  # embedding, projections
            self._build(recent, sink)
        self._imports: dict[int, list] = {}    # row -> the operators that take its prompt in
        self.graph, self._warm = None, False
        self.slots = np.zeros(rows, np.int64)  # slots in use after the steps enqueued so far
        self.pos_host = 0                      # position of the rows' next token
        self._beam_tables = False              # the device has the only true table (beam search)
        self._beam_slots = 0                   # slots that each beam has pages for

    # -- one step ---------------------------------------------------------------------------------------------
    def _weight(self, name: str) -> int:
        return self.hal.arena_ptr(0) + self.prog.dpu_plans[0].weight[name]

    def _projection(self, x, weight, out, k, ncols, mode=nat.PROJ_PLAIN, norm=None, residual=None, inter=0):
        a = nat.ProjectionArgs(x=x.data_ptr(), norm_weight=self._weight(norm) if norm else None,
                               weight=self._weight(weight), out=out.data_ptr(), rows=self.rows, k=k, ncols=ncols,
                               eps=self.cfg.rms_eps, inter=inter, err_flag=self.err.data_ptr() + 4,
                               residual=residual.data_ptr() if residual is not None else None)
        return a, mode

    def _build(self, recent: int, sink: int) -> None:
        """The operators and projections of a step, bound to its buffers."""
        torch, cfg, c = self.torch, self.cfg, self.cache
        hd, hq, hkv, h, i = cfg.head_dim, cfg.num_heads, cfg.num_kv_heads, cfg.hidden_size, cfg.intermediate_size
        self.code = nat.DTYPE_CODE[cfg.dtype]
        arena = self.hal.arena(0)

        def rotary(name):
            at = self.prog.dpu_plans[0].weight[f"model.rotary.{name}"]
            return arena[at:at + cfg.max_seq * hd // 2 * 4].view(torch.float32).view(cfg.max_seq, hd // 2)

        q, k, v = (t.view(self.rows, -1, hd) for t in self.qkv.split([hq * hd, hkv * hd, hkv * hd], dim=1))
        self.layers, self.ops, need = [], [], 0
        for l in range(cfg.num_layers):
            p = f"model.layers.{l}."
            track = {} if self.budget is None else dict(slot_positions=c.slot_positions[l], weights=c.weights[l])
            append = PagedAppend(k, v, c.k(l), c.v(l), c.table, self.lengths, self.next_lengths, q=q, q_out=self.q_rot,
                                 cos=rotary("cos"), sin=rotary("sin"), positions=self.positions,
                                 positions_out=self.next_positions, pair_order=True, **track)
            attend = PagedAttention(self.q_rot, c.k(l), c.v(l), c.table, self.next_lengths, self.attn,
                                    weights=track.get("weights"))
            evict = None
            if self.budget is not None:
                evict = PagedEvict(c.k(l), c.v(l), c.table, self.next_lengths, c.weights[l], c.slot_positions[l],
                                   self.next_positions, c.weights[l], c.slot_positions[l], self.cut_lengths,
                                   budget=self.budget, recent=recent, sink=sink)
            self.ops += [o for o in (append, attend, evict) if o is not None]
            self.layers.append((
                self._projection(self.x, p + "self_attn.qkv_proj.weight", self.qkv, h, (hq + 2 * hkv) * hd,
                                 norm=p + "input_layernorm.weight"),
                append, attend,
                self._projection(self.attn, p + "self_attn.o_proj.weight", self.h, hq * hd, h, residual=self.x),
                self._projection(self.h, p + "mlp.gate_up_proj.weight", self.act, h, 2 * i, nat.PROJ_SILU_MUL,
                                 norm=p + "post_attention_layernorm.weight", inter=i),
                self._projection(self.act, p + "mlp.down_proj.weight", self.x, i, h, residual=self.h),
                evict))
        self.head = self._projection(self.x, "lm_head.weight", self.logits, h, cfg.vocab_size, norm="model.norm.weight")
        projections = [x for layer in self.layers for x in layer if isinstance(x, tuple)] + [self.head]
        need = max(nat.lib.pim_projection_scratch_bytes(ctypes.byref(a), self.code, mode) for a, mode in projections)
        # (decode rows: the work counter of the dynamic kernel, which must read zero)
        self.scratch = torch.zeros(max(need, 256), dtype=torch.uint8, device=self.device)

    def _project(self, projection) -> None:
        a, mode = projection
        nat.check(nat.lib.pim_projection(ctypes.byref(a), self.code, mode, self.scratch.data_ptr(), self.scratch.numel(),
                                         self.stream.cuda_stream), "projection")

    def _enqueue(self) -> None:
        """A step for the tokens in ``ids``: K and V into the pages, ``logits``, lengths and positions advanced."""
        cfg = self.cfg
        nat.check(nat.lib.pim_embedding(self.ids.data_ptr(), self._weight("model.embed_tokens.weight"), self.x.data_ptr(),
                                        self.rows, cfg.hidden_size, cfg.vocab_size, self.code, self.err.data_ptr(),
                                        self.stream.cuda_stream), "embedding")
        for qkv, append, attend, o_proj, mlp_in, down, evict in self.layers:
            self._project(qkv)
            append()
            attend()
            if evict is not None:
                evict()
            self._project(o_proj)
            self._project(mlp_in)
            self._project(down)
        self._project(self.head)
        self.lengths.copy_(self.next_lengths if self.budget is None else self.cut_lengths)
        self.positions.copy_(self.next_positions)

    def step(self) -> None:
        """Enqueues one step for the tokens in ``ids`` (a graph replay from the second one on)."""
        torch = self.torch
        if self._beam_tables and (self.slots + 1 > self._beam_slots).any():  # (no page behind them)
            raise ValueError(f"the search took pages for {self._beam_slots} slots a beam, and all are in use")
        if (self.slots + 1 > self.spec.slots).any() or int(self.pos_host) >= self.cfg.max_seq:
            raise ValueError(f"no room: {int(self.slots.max())} of {self.spec.slots} slots, position {self.pos_host} of "
                             f"{self.cfg.max_seq}")
        with torch.cuda.device(self.device), torch.cuda.stream(self.stream):
            if not self._beam_tables and self.cache.reserve(self.slots + 1):
                self.cache.upload()
            if self.graph is None and self._warm:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=self.stream):
                    self._enqueue()
                self.graph = graph
            if self.graph is None:
                self._enqueue()
                self._warm = True
            else:
                self.graph.replay()
        self.slots += 1
        self.pos_host += 1
        if self.budget is not None:
            self.slots = np.minimum(self.slots, self.budget)
            self.cache.trim(self.slots)  # (what takes these pages next is enqueued behind this step)

    # -- prompts ------------------------------------------------------------------------------------------------
    def reset(self) -> None:
        """Gives every page back and empties the rows; errors that nobody asked for are forgotten."""
        with self.torch.cuda.device(self.device), self.torch.cuda.stream(self.stream):
            for row in range(self.rows):
                self.cache.release(row)
            self.lengths.zero_()
            self.positions.zero_()
            self.err.zero_()
            forget(self._bound())
        self.slots[:] = 0
        self.pos_host = 0
        self._beam_tables = False

    def _prompt(self, prompt) -> "object":
        """The prefill plan on one prompt; its last position's logits (a view of the plan's output)."""
        ids = np.asarray(prompt, np.int32).reshape(1, -1)
        if ids.shape[1] != self.prog.prompt_len:
            raise ValueError(f"the prefill plan takes {self.prog.prompt_len} tokens, got {ids.shape[1]}")
        plan = self.prog.plans["prefill"]
        execute_plan(plan, self.hal, tokens=ids, pos=np.zeros(1, np.int32))
        ref = plan.meta["outputs"]["logits"]
        n = self.cfg.vocab_size * self.logits.element_size()
        return self.hal.host_tensor(plan)[ref.offset:ref.offset + n].view(self.logits.dtype)

    def _blocks(self, layer: int):
        """K and V of the prefill's static cache, [max_seq, kv_heads, head_dim] views of the arena."""
        spec = self.prog.kv_specs[0]
        item = self.logits.element_size()
        arena = self.hal.arena(0).view(self.logits.dtype)
        out = []
        for which in "kv":
            at = [spec.kv_off[(layer, h, which)] // item for h in spec.kv_heads]
            pitch = at[1] - at[0] if len(at) > 1 else spec.max_seq * spec.head_dim
            out.append(arena.as_strided((spec.max_seq, len(at), spec.head_dim), (spec.head_dim, pitch, 1), at[0]))
        return out

    def _import(self, row: int) -> None:
        """The prompt's K and V from the static cache into the row's pages."""
        if row not in self._imports:
            self._imports[row] = self._bind_import(row)
        for op in self._imports[row]:
            op()

    def _bind_import(self, row: int) -> list:
        """A row's operators for that, one a layer; kept, as those of a step are."""
        torch, c, n = self.torch, self.cache, self.prog.prompt_len
        starts = torch.tensor([0, n], dtype=torch.int32, device=self.device)
        zero = torch.zeros(1, dtype=torch.int32, device=self.device)
        ops = []
        for l in range(self.cfg.num_layers):
            k, v = (t[:n] for t in self._blocks(l))
            track = {} if self.budget is None else dict(slot_positions=c.slot_positions[l, row:row + 1],
                                                        weights=c.weights[l, row:row + 1])
            ops.append(PagedAppend(k, v, c.k(l), c.v(l), c.table[row:row + 1], zero, self.lengths[row:row + 1],
                                   positions_out=self.positions[row:row + 1], positions=torch.zeros_like(zero),
                                   starts=starts, **track))
        return ops

    def _start(self, prompts) -> None:
        """Every row's prompt into its pages and its last logits into ``logits``."""
        torch, n = self.torch, self.prog.prompt_len
        self.reset()
        with torch.cuda.device(self.device), torch.cuda.stream(self.stream):
            self.cache.reserve([n] * len(prompts))
            self.cache.upload()
            for row, prompt in enumerate(prompts):
                self.logits[row].copy_(self._prompt(prompt))
                self._import(row)
        self.slots[:len(prompts)] = n
        self.pos_host = n

    def _bound(self) -> list:
        return [*self.ops, *(op for ops in self._imports.values() for op in ops)]

    # -- generation -------------------------------------------------------------------------------------------------
    def check(self, *more) -> None:
        """Raises if a step (or a call of the operators ``more``) met a bad id, length, position, page or logit.  Waits for
        the device; every flag is cleared, so what follows is judged by itself."""
        said = complaints([*self._bound(), *more])
        if bool(self.err.any()):
            self.err.zero_()
            self.torch.cuda.synchronize(self.device)
            said.append("a token id was outside the vocabulary, or a projection's wait ran out")
        if said:
            raise ValueError("; ".join(said))

    def greedy(self, prompts, steps: int, keep_logits: list | None = None) -> np.ndarray:
        """[rows, steps] tokens; ``keep_logits`` (a list) receives each step's [rows, vocab] logits."""
        torch = self.torch
        prompts = np.asarray(prompts, np.int32)
        if steps < 1:
            raise ValueError(f"steps must be positive, got {steps}")
        if prompts.shape != (self.rows, self.prog.prompt_len):
            raise ValueError(f"expected prompts of shape {(self.rows, self.prog.prompt_len)}, got {prompts.shape}")
        self._start(prompts)
        got = []
        with torch.cuda.device(self.device), torch.cuda.stream(self.stream):
            for i in range(steps):
                if i:
                    self.ids.copy_(self.next_ids)
                    self.step()
                if keep_logits is not None:
                    keep_logits.append(self.logits.float().cpu().numpy())
                nat.check(nat.lib.pim_argmax(self.logits.data_ptr(), self.next_ids.data_ptr(), self.rows,
                                             self.cfg.vocab_size, self.code, self.stream.cuda_stream), "argmax")
                got.append(self.next_ids.clone())
            out = torch.stack(got, dim=1).cpu().numpy()
        self.check()
        return out

    def beam_search(self, prompt, steps: int, eos: int = -1, pad: int = 0) -> BeamResult:
        """The ``rows`` best continuations of one prompt found by beam search, ``steps`` tokens each (``pad`` behind
        ``eos``).  Needs a cache without eviction: beams share pages."""
        if self.budget is not None:
            raise ValueError("beam search shares pages between beams: it takes a cache without a budget")
        torch, w, n = self.torch, self.rows, self.prog.prompt_len
        if steps < 1:
            raise ValueError(f"steps must be positive, got {steps}")
        if n + steps - 1 > self.spec.slots:
            raise ValueError(f"{n} + {steps - 1} slots, the table holds {self.spec.slots}")
        self._start([prompt])
        with torch.cuda.device(self.device), torch.cuda.stream(self.stream):
            c = self.cache
            c.share_prompt(n)
            try:  # a tail for each beam: its partly filled page and what the search will fill
                c.reserve([n + steps - 1] * w)
            except MemoryError:
                self.reset()  # (rows that hold the prompt's pages and no tail must not take a step)
                raise
            c.upload()
            self._beam_tables = True  # from here on the table is the device's
            self._beam_slots = n + steps - 1
            scores, next_scores = (torch.zeros(1, w, device=self.device) for _ in range(2))
            done, next_done, parents, tokens = (torch.zeros(1, w, dtype=torch.int32, device=self.device) for _ in range(4))
            table_out = torch.zeros_like(c.table)
            length = torch.zeros(1, dtype=torch.int32, device=self.device)
            first = BeamSelect(self.logits[:1].view(1, 1, -1), scores[:, :1], next_scores, parents, tokens,
                               done_out=next_done, eos=eos, pad=pad)
            select = BeamSelect(self.logits.view(1, w, -1), scores, next_scores, parents, tokens, done=done,
                                done_out=next_done, eos=eos, pad=pad)
            reorder = BeamReorder(c.pages, c.table, length, parents, table_out)
            history = []
            for i in range(steps):
                if i:
                    self.step()
                (select if i else first)()
                length.copy_(self.lengths[:1])
                reorder()
                c.table.copy_(table_out)
                scores.copy_(next_scores)
                done.copy_(next_done)
                self.ids.copy_(tokens[0])
                if not i:
                    self.lengths.copy_(self.lengths[:1].expand(w).clone())
                    self.positions.copy_(self.positions[:1].expand(w).clone())
                    self.slots[:] = n
                history.append((parents.clone(), tokens.clone()))
            par = torch.cat([p for p, _ in history]).cpu().numpy()
            tok = torch.cat([t for _, t in history]).cpu().numpy()
            result = BeamResult(np.zeros((w, steps), np.int32), scores[0].cpu().numpy(), done[0].cpu().numpy().astype(bool))
        for j in range(w):
            at = j
            for i in range(steps - 1, -1, -1):
                result.tokens[j, i] = tok[i, at]
                at = par[i, at]
        self.check(first, select, reorder)
        return result
