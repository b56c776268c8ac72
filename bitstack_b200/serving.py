"""Serving many requests of different lengths with one decoder: prompts come and go, every step makes one token for
each request that is running.

`BitStackLlamaDecoder` (decode.py) keeps a dense cache with one position for the whole batch and takes the largest
logit.  `PagedDecoder` runs the same layers over a paged cache: the requests' lengths, their block tables and the stack
of free pages live on the device (`glue.page_tables` / `glue.release_pages`), a prompt's keys and values go into pages
(`glue.rope_paged_cache`), a step attends over them (`glue.paged_decode_attention`), and every request has its own
temperature, top-k, top-p and min-p (`glue.sample_step`).  A step touches the host nowhere, so it can be captured in a
CUDA graph; requests are admitted and released between steps.  The reference has no generation loop at all (its model
calls are whole-sequence evaluations, bitstack/utils/model_utils.py:116-133).
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch
import torch.nn.functional as F

from . import _lib, glue
from .decode import BitStackLlamaDecoder
from .linear import forward_grouped, own_workspace


class OutOfPages(RuntimeError):
    """The pool has too few free pages (or the request's table row is too narrow) for what was asked."""


class PagedDecoder:
    """`rows` request slots over `model`'s weights and a pool of `num_pages` pages of `page_size` positions."""

    def __init__(self, model: BitStackLlamaDecoder, rows: int, num_pages: int, page_size: int = 16):
        if model.world != 1:
            raise ValueError("PagedDecoder runs on one device; the tensor-parallel decoder keeps the dense cache")
        if model.shape.head_dim not in (64, 128):
            raise ValueError(f"paged attention is built for head_dim 64 and 128 (the model has {model.shape.head_dim})")
        if rows < 1 or num_pages < 1 or page_size < 1:
            raise ValueError("rows, num_pages and page_size must be at least 1")
        self.model, self.rows, self.page_size, self.device = model, rows, page_size, model.device
        s, dev = model.shape, model.device
        zeros = lambda *n, t: torch.zeros(*n, dtype=t, device=dev)  # noqa: E731
        width = -(-model.max_len // page_size)
        self.lens, self.active = zeros(rows, t=torch.int32), zeros(rows, t=torch.int32)
        self.max_positions = width * page_size                 # of a request: whole pages
        self.cos, self.sin = (model.cos, model.sin) if self.max_positions <= model.max_len else self._rotary(self.max_positions)
        self.block_table = torch.full((rows, width), -1, dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=dev)     # the lowest page is on top
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=dev)
        pool = (num_pages, model.kv_local, page_size, s.head_dim)
        self.k_pages = [zeros(pool, t=torch.float16) for _ in range(s.n_layers)]
        self.v_pages = [zeros(pool, t=torch.float16) for _ in range(s.n_layers)]
        self.tokens = zeros(rows, t=torch.int64)              # what every row feeds to the next step
        self.positions = torch.full((rows,), -1, dtype=torch.int64, device=dev)   # of the last step; -1: the row made no step
        self.uniforms, self.logprobs = zeros(rows, t=torch.float32), zeros(rows, t=torch.float32)
        self.temperature, self.top_k = zeros(rows, t=torch.float32), zeros(rows, t=torch.int32)
        self.top_p, self.min_p = torch.ones(rows, dtype=torch.float32, device=dev), zeros(rows, t=torch.float32)
        self.logits: Optional[torch.Tensor] = None             # of the last step (of the captured one: the graph's own buffer)
        self._running = [False] * rows                         # the host's view of which rows are taken
        self._graph = None

    def _rotary(self, n):
        s = self.model.shape
        inv_freq = 1.0 / (s.rope_theta ** (torch.arange(0, s.head_dim, 2, device=self.device, dtype=torch.float32) / s.head_dim))
        freqs = torch.outer(torch.arange(n, device=self.device, dtype=torch.float32), inv_freq)
        return tuple(torch.cat([f, f], dim=-1).half() for f in (freqs.cos(), freqs.sin()))

    # ------------------------------------------------------------------ requests
    def free_rows(self) -> List[int]:
        return [i for i, busy in enumerate(self._running) if not busy]

    @torch.no_grad()
    def submit(self, prompts: Sequence[torch.Tensor], temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0,
               uniforms: Optional[torch.Tensor] = None) -> List[int]:
        """Admits prompts (1-D token tensors, at least one token each) to free rows, runs them in one ragged batch and
        draws the first token of each (`tokens[row]`).  Returns their rows.  Raises OutOfPages, with nothing changed, when
        they do not fit.  `uniforms`: one number per prompt (default: drawn from the device's generator)."""
        lengths = [int(p.numel()) for p in prompts]
        if not lengths or min(lengths) < 1:
            raise ValueError("a prompt must have at least one token")
        if max(lengths) > self.max_positions:
            raise ValueError(f"a prompt of {max(lengths)} tokens is longer than a request's {self.max_positions} positions")
        ids = torch.cat([p.reshape(-1) for p in prompts]).to(self.device)
        if ids.dtype not in (torch.int32, torch.int64) or bool(((ids < 0) | (ids >= self.model.shape.vocab)).any()):
            raise ValueError(f"prompts must be integer tokens in [0, {self.model.shape.vocab})")
        free = self.free_rows()
        if len(free) < len(prompts):
            raise OutOfPages(f"{len(prompts)} prompts, {len(free)} free rows")
        rows = sorted(free[:len(prompts)])                    # the token list goes row after row
        dev, total = self.device, sum(lengths)
        if sum(-(-n // self.page_size) for n in lengths) > int(self.free_count):
            raise OutOfPages(f"{sum(-(-n // self.page_size) for n in lengths)} pages needed, {int(self.free_count)} free")
        at = torch.tensor(rows, device=dev)
        new = torch.zeros(self.rows, dtype=torch.int32, device=dev)
        new[at] = torch.tensor(lengths, dtype=torch.int32, device=dev)
        self.temperature[at], self.top_k[at], self.top_p[at], self.min_p[at] = float(temperature), int(top_k), float(top_p), float(min_p)
        slots, positions, _, _ = glue.page_tables(self.lens, new, self.block_table, self.free_pages, self.free_count, self.page_size, total)
        try:
            hidden = self._prompt(ids, slots, positions, lengths)
            logits = hidden @ self.model.lm_head.t()
            u = torch.rand(len(rows), device=dev) if uniforms is None else uniforms.to(dev, torch.float32)
            drawn = torch.empty(len(rows), dtype=torch.int64, device=dev)
            logprobs = torch.empty(len(rows), dtype=torch.float32, device=dev)
            glue.sample_step(logits, u, drawn, self.temperature[at], self.top_k[at], self.top_p[at], self.min_p[at], logprobs=logprobs)
        except BaseException:                                  # the prompts' pages go back
            done = new > 0
            glue.release_pages(done, self.lens, self.block_table, self.free_pages, self.free_count, self.page_size)
            raise
        self.tokens[at], self.logprobs[at], self.active[at] = drawn, logprobs, 1
        for r in rows:
            self._running[r] = True
        return rows

    @torch.no_grad()
    def release(self, rows: Sequence[int]) -> None:
        """Ends requests: their pages are free for others, their rows idle."""
        for r in rows:
            if not self._running[r]:
                raise ValueError(f"row {r} runs no request")
        done = torch.zeros(self.rows, dtype=torch.bool, device=self.device)
        done[torch.tensor(list(rows), dtype=torch.int64, device=self.device)] = True
        glue.release_pages(done, self.lens, self.block_table, self.free_pages, self.free_count, self.page_size)
        self.active.masked_fill_(done, 0)
        for r in rows:
            self._running[r] = False

    # ------------------------------------------------------------------ the model
    def _prompt(self, ids, slots, positions, lengths):
        """Hidden states (normalised) of the last token of every prompt of a ragged batch, K and V written into pages."""
        m, s = self.model, self.model.shape
        hd, hq, hkv = s.head_dim, m.q_local, m.kv_local
        h = m.embed.index_select(0, ids)
        page, row = torch.div(slots, self.page_size, rounding_mode="floor"), torch.remainder(slots, self.page_size)
        for i, lay in enumerate(m.layers):
            x = F.rms_norm(h, (s.hidden,), lay["in_norm"], s.rms_eps)
            q, k, v = forward_grouped([lay["self_attn.q_proj"], lay["self_attn.k_proj"], lay["self_attn.v_proj"]], x)
            q = glue.rope_paged_cache(q, k, v, self.cos, self.sin, positions, slots, self.k_pages[i], self.v_pages[i], hq, hkv, hd)
            keys, values = self.k_pages[i][page, :, row], self.v_pages[i][page, :, row]       # [tokens, kv heads, head_dim]
            att, lo = torch.empty_like(q), 0
            for n in lengths:
                qs, ks, vs = (t[lo:lo + n].view(1, n, -1, hd).transpose(1, 2) for t in (q, keys, values))
                att[lo:lo + n] = F.scaled_dot_product_attention(qs, ks, vs, is_causal=True, enable_gqa=True).transpose(1, 2).reshape(n, hq * hd)
                lo += n
            h = h + lay["self_attn.o_proj"](att)
            x = F.rms_norm(h, (s.hidden,), lay["post_norm"], s.rms_eps)
            g, u = forward_grouped([lay["mlp.gate_proj"], lay["mlp.up_proj"]], x)
            h = h + lay["mlp.down_proj"](F.silu(g) * u)
        last = torch.tensor(lengths, device=self.device).cumsum(0) - 1
        return F.rms_norm(h.index_select(0, last), (s.hidden,), m.final_norm, s.rms_eps)

    def _step(self):
        m, s, n = self.model, self.model.shape, self.rows
        _, _, _, last = glue.page_tables(self.lens, self.active, self.block_table, self.free_pages, self.free_count, self.page_size)
        h = m.embed.index_select(0, self.tokens)
        am = torch.empty(n, dtype=torch.float32, device=self.device) if n <= 6 else None
        delta = None
        for i, lay in enumerate(m.layers):
            x = glue.add_rmsnorm(h, delta, lay["in_norm"], s.rms_eps, absmax=am)
            q, k, v = forward_grouped([lay["self_attn.q_proj"], lay["self_attn.k_proj"], lay["self_attn.v_proj"]], x, x_absmax=am)
            att = glue.paged_decode_attention(q, k, v, self.cos, self.sin, last, self.block_table, self.k_pages[i], self.v_pages[i],
                                              m.q_local, m.kv_local, s.head_dim)
            x = glue.add_rmsnorm(h, lay["self_attn.o_proj"](att), lay["post_norm"], s.rms_eps, absmax=am)
            g, u = forward_grouped([lay["mlp.gate_proj"], lay["mlp.up_proj"]], x, x_absmax=am)
            a = glue.silu_mul(g, u, absmax=am)
            delta = forward_grouped([lay["mlp.down_proj"]], a, x_absmax=am)[0] if am is not None else lay["mlp.down_proj"](a)
        logits = glue.add_rmsnorm(h, delta, m.final_norm, s.rms_eps) @ m.lm_head.t()
        drawn, logprobs = torch.empty_like(self.tokens), torch.empty_like(self.logprobs)
        glue.sample_step(logits, self.uniforms, drawn, self.temperature, self.top_k, self.top_p, self.min_p, logprobs=logprobs)
        made = last >= 0                                      # idle rows, and rows that the pool had no page for, keep their token
        self.tokens.copy_(torch.where(made, drawn, self.tokens))
        self.logprobs.copy_(torch.where(made, logprobs, self.logprobs))
        self.positions.copy_(last)
        self.logits = logits

    @torch.no_grad()
    def step(self, uniforms: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One token for every running row: `tokens` (returned), `logprobs` and `positions` hold the result on the device.
        A running row whose `positions` entry is -1 made no step (no free page, or its table row is full) and does so again
        once pages are free.  `uniforms` (one per row): the numbers to draw with, default from the device's generator."""
        if uniforms is None:
            self.uniforms.uniform_()
        else:
            self.uniforms.copy_(uniforms)
        if self._graph is not None:
            self._graph.replay()
        else:
            self._step()
        return self.tokens

    @torch.no_grad()
    def capture(self):
        """Captures the step in a CUDA graph, which `step` replays from then on.  No row makes a step by it: the rows are
        idle in the runs that warm it up, and running again afterwards, also where this raises (an earlier graph then stays)."""
        kept = self.active.clone(), self.tokens.clone(), self.logprobs.clone(), self.positions.clone()
        here, stream, logits = torch.cuda.current_stream(self.device), torch.cuda.Stream(self.device), self.logits
        self.active.zero_()
        stream.wait_stream(here)
        try:
            with own_workspace(stream) as scratch:
                with torch.cuda.stream(stream):
                    for _ in range(2):
                        self._step()
                here.wait_stream(stream)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    self._step()
            graph.scratch = scratch                            # of the projections: the graph's alone, and there as long as it is
            self._graph, logits = graph, self.logits
        finally:
            self.logits = logits
            here.wait_stream(stream)
            for t, old in zip((self.active, self.tokens, self.logprobs, self.positions), kept):
                t.copy_(old)
        return graph

    @torch.no_grad()
    def generate(self, prompts: Sequence[torch.Tensor], steps: int, **sampling) -> List[List[int]]:
        """Host-facing: admits the prompts, makes `steps` tokens (at least one) for each (the first of them from the prompt) and
        releases them.  Raises OutOfPages when the pool runs out on the way."""
        if steps < 1:
            raise ValueError(f"steps must be at least 1, got {steps}: a prompt gives its first token when it is admitted")
        rows = self.submit(prompts, **sampling)
        try:
            out = [self.tokens[rows].tolist()]
            for _ in range(steps - 1):
                self.step()
                if bool((self.positions[rows] < 0).any()):
                    raise OutOfPages("the pool ran out of pages, or a request reached the decoder's length")
                out.append(self.tokens[rows].tolist())
        finally:
            self.release(rows)
        with torch.cuda.device(self.device):
            _lib.check_device_status()
        return [list(t) for t in zip(*out)]
