"""Greedy generation on one GPU: one compiled prefill that seeds the explicit KV state, then one
compiled decode call per token -- picked on the host (``__call__``) or, with no host work per
token at all, picked on the device inside a replayed CUDA graph (``on_device``).

The counterpart of the reference's ``examples/single_gpu_generate.py`` -- which has to feed the
prompt through its decode step token by token because its prefill cannot seed the decode state
(``examples/single_gpu_generate.py:3-4``).  Here ``StatefulPrefill`` writes the prompt's keys and
values into the caches that ``StatefulDecoder`` appends to.
"""

from __future__ import annotations

import torch

from . import runtime as rt
from .engine import graphed
from .frontend import make_backend
from .hf import PagedDecoder, StatefulDecoder, StatefulPrefill


class GreedyGenerator:
    """Compiles the two wrappers once for a (batch, prompt length, capacity) and reuses them."""

    def __init__(self, model: torch.nn.Module, batch: int, prompt_tokens: int, capacity: int,
                 per_row_lengths: bool = False):
        """``per_row_lengths``: every row keeps its own valid length, so that one batch can hold
        prompts of different lengths (``prompt_lengths`` of ``__call__``); ``prompt_tokens`` is
        then the padded prompt length the prefill is compiled for."""
        if capacity <= prompt_tokens:
            raise ValueError("capacity must exceed the prompt length")
        self.batch, self.prompt_tokens, self.capacity = batch, prompt_tokens, capacity
        self.per_row_lengths = per_row_lengths
        self.device = next(model.parameters()).device
        prefill = StatefulPrefill(model, capacity).eval()
        decode = StatefulDecoder(model, capacity).eval()
        self.state = prefill.make_state(batch, device=self.device, per_row_lengths=per_row_lengths)
        self.prefill_backend = make_backend(mode="prefill")
        self.decode_backend = make_backend(mode="decode")
        self._prefill = torch.compile(prefill, backend=self.prefill_backend, fullgraph=True,
                                      dynamic=False)
        self._decode = torch.compile(decode, backend=self.decode_backend, fullgraph=True,
                                     dynamic=False)

    @torch.no_grad()
    def __call__(self, input_ids: torch.Tensor, new_tokens: int,
                 prompt_lengths: torch.Tensor | None = None) -> torch.Tensor:
        """``input_ids`` ``[batch, prompt_tokens]`` -> generated ids ``[batch, new_tokens]``.

        ``prompt_lengths`` (int ``[batch]``, needs ``per_row_lengths``): the real length of every
        row's prompt; rows are padded at the end up to ``prompt_tokens`` with any valid id.  The
        causal prefill cannot see the padding from a real position; after it the valid lengths
        are set to the real lengths, so decode overwrites the padded rows of the caches and
        never attends to them."""
        if tuple(input_ids.shape) != (self.batch, self.prompt_tokens):
            raise ValueError("this generator was compiled for another prompt shape")
        if self.prompt_tokens + new_tokens > self.capacity:
            raise ValueError("the KV capacity cannot hold the prompt plus the new tokens")
        if prompt_lengths is not None and not self.per_row_lengths:
            raise ValueError("prompt_lengths needs a generator built with per_row_lengths=True")
        logits = self._prefill(input_ids.to(self.device), *self.state)
        if prompt_lengths is None:
            token = logits[:, -1].float().argmax(-1, keepdim=True)
            position = torch.full((self.batch, 1), self.prompt_tokens, dtype=torch.int64,
                                  device=self.device)
        else:
            lengths = prompt_lengths.to(self.device, torch.int64)
            if lengths.shape != (self.batch,) or int(lengths.min()) < 1 or \
                    int(lengths.max()) > self.prompt_tokens:
                raise ValueError("prompt_lengths must hold one length in 1..prompt_tokens per row")
            rows = torch.arange(self.batch, device=self.device)
            token = logits[rows, lengths - 1].float().argmax(-1, keepdim=True)
            position = lengths[:, None].clone()
            for index in range(2, len(self.state), 3):
                self.state[index].copy_(lengths.to(torch.int32))
        produced = [token]
        for _ in range(new_tokens - 1):
            logits = self._decode(token, position, *self.state)
            token = logits[:, -1].float().argmax(-1, keepdim=True)
            produced.append(token)
            position = position + 1
        for backend in (self.prefill_backend, self.decode_backend):
            if backend.megabake_last_callable is not None:
                backend.megabake_last_callable.check()
        return torch.cat(produced, dim=1)

    # -- the multi-step loop with the pick on the device ------------------------------------
    def _build_loop(self, steps_per_graph: int):
        """Capture ``steps_per_graph`` x (decode launch, greedy pick) in one CUDA graph.  The
        pick writes the next id into the very tensor the next decode launch reads and advances
        the positions, so a replay needs nothing from the host (the reference lists this loop
        as future work, ``docs/roadmap.md:180``)."""
        if 2 * steps_per_graph + 1 > self.capacity:
            raise ValueError("the KV capacity is too small to warm this many steps up")
        self._token = torch.zeros(self.batch, 1, dtype=torch.int64, device=self.device)
        self._position = torch.zeros(self.batch, 1, dtype=torch.int64, device=self.device)
        self._picked = torch.zeros(self.batch, self.capacity, dtype=torch.int64, device=self.device)
        self._cursor = torch.zeros(self.batch, dtype=torch.int32, device=self.device)
        for index in range(2, len(self.state), 3):
            self.state[index].zero_()  # the warm-up runs of the capture start from an empty cache

        def loop(token, position, *state):
            for _ in range(steps_per_graph):
                logits = self._decode(token, position, *state)
                rt.greedy_advance(logits, token, position, self._picked, self._cursor)
            return self._picked

        self._loop = graphed(loop, self._token, self._position, *self.state)
        self._loop_steps = steps_per_graph

    @torch.no_grad()
    def on_device(self, input_ids: torch.Tensor, new_tokens: int,
                  steps_per_graph: int = 1) -> torch.Tensor:
        """Same result as ``__call__``, but every token after the prompt is picked by
        ``mb_greedy_advance`` on the device and the decode steps run as replays of one CUDA
        graph holding ``steps_per_graph`` steps; the host reads the ids once, at the end.
        ``new_tokens - 1`` must be a multiple of ``steps_per_graph``."""
        if tuple(input_ids.shape) != (self.batch, self.prompt_tokens):
            raise ValueError("this generator was compiled for another prompt shape")
        if self.prompt_tokens + new_tokens > self.capacity:
            raise ValueError("the KV capacity cannot hold the prompt plus the new tokens")
        if steps_per_graph < 1 or (new_tokens - 1) % steps_per_graph:
            raise ValueError("new_tokens - 1 must be a multiple of steps_per_graph")
        if getattr(self, "_loop_steps", None) != steps_per_graph:
            self._build_loop(steps_per_graph)
        logits = self._prefill(input_ids.to(self.device), *self.state)
        self._cursor.zero_()
        self._position.fill_(self.prompt_tokens)
        # the first pick comes from the prompt's last position; positions stay where they are
        rt.greedy_advance(logits[:, -1].contiguous(), self._token, None, self._picked,
                          self._cursor)
        for _ in range((new_tokens - 1) // steps_per_graph):
            self._loop(self._token, self._position, *self.state)
        for backend in (self.prefill_backend, self.decode_backend):
            if backend.megabake_last_callable is not None:
                backend.megabake_last_callable.check()
        if int(self._cursor.max()) != new_tokens or int(self._cursor.min()) != new_tokens:
            raise RuntimeError("the device-side loop produced an unexpected number of tokens")
        return self._picked[:, :new_tokens].clone()


class PagedGenerator:
    """Greedy generation of many prompts of any lengths over one paged cache: requests take a row of the table as one
    becomes free and pages of the pool as they grow, and give both back when they end.

    ``requests`` rows run at once; ``pages`` pages of ``page_size`` tokens are shared by them (default: enough for all
    of them to grow to ``capacity``).  A prompt is admitted when its row and the pages for all of its tokens are there, so
    no request is refused later.  Prompts admitted together go through the model in one pass, of ``prompt_tokens`` tokens at
    most where there are several: its activations do not grow with how many prompts wait.  Decode steps are one CUDA graph:
    pages, attention, projections and the greedy pick, without the host; at the end it is checked once that no wait inside
    a kernel ran out (``CompilerError``)."""

    def __init__(self, model: torch.nn.Module, requests: int, capacity: int, *, page_size: int = 64,
                 pages: int | None = None, prompt_tokens: int = 8192):
        self.decoder = PagedDecoder(model).eval()
        self.prompt_tokens = prompt_tokens
        self.state = self.decoder.make_paged_state(requests, capacity, page_size=page_size, pages=pages)
        self.requests, self.pages = requests, self.state.free_pages.numel()
        self.device = self.state.lengths.device
        int32 = torch.int32
        # the row behind the last one takes what belongs to no request
        self._picked = torch.zeros(requests + 1, dtype=torch.int64, device=self.device)
        self._produced = torch.zeros(requests + 1, dtype=torch.int64, device=self.device)
        self._log = torch.zeros(requests + 1, self.state.capacity, dtype=torch.int64, device=self.device)
        self._counts = torch.zeros(requests, dtype=int32, device=self.device)
        self._graph = None

    def _pages_of(self, tokens: int) -> int:
        return -(-tokens // self.state.page_size)

    def _pick(self, logits: torch.Tensor, rows: torch.Tensor) -> None:
        """The greedy pick of every row of ``logits`` becomes the next id of request ``rows`` and is logged."""
        picked = torch.empty(logits.shape[0], dtype=torch.int64, device=self.device)
        rt.greedy_advance(logits, picked)
        rows = torch.where(rows < 0, self.requests, rows).long()
        self._picked.index_copy_(0, rows, picked)
        self._log.index_put_((rows, self._produced[rows]), picked)
        self._produced.index_add_(0, rows, (rows < self.requests).long())

    def _decode(self) -> None:
        batch = self.state.reserve(self._counts, self.requests)
        rows = torch.where(batch.rows < 0, self.requests, batch.rows).long()
        logits = self.decoder(self._picked[rows], batch, self.state, one_token=True)
        self._pick(logits, batch.rows)

    def _decode_step(self) -> None:
        if self._graph is None:
            self._decode()          # once without a graph: what is set up lazily is set up here
            torch.cuda.synchronize(self.device)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                self._decode()
            self._graph = graph
        else:
            self._graph.replay()

    def _prefill(self, prompts: dict[int, torch.Tensor]) -> None:
        """Admit ``prompts`` (by row) and pick their first new ids."""
        total = sum(p.numel() for p in prompts.values())
        counts = torch.zeros(self.requests, dtype=torch.int32)
        last, rows, at = [], sorted(prompts), 0
        for row in rows:
            counts[row] = prompts[row].numel()
            at += prompts[row].numel()
            last.append(at - 1)
        batch = self.state.reserve(counts.to(self.device), total)
        ids = torch.cat([prompts[row].flatten() for row in rows]).to(self.device, torch.int64)
        logits = self.decoder(ids, batch, self.state, tokens=torch.tensor(last, device=self.device))
        self._pick(logits, torch.tensor(rows, device=self.device))

    @torch.no_grad()
    def __call__(self, prompts: list[torch.Tensor], new_tokens: int | list[int]) -> list[torch.Tensor]:
        """``new_tokens`` ids (one number, or one per prompt) after each of ``prompts`` (1-d, any lengths)."""
        wanted = [new_tokens] * len(prompts) if isinstance(new_tokens, int) else list(new_tokens)
        if len(wanted) != len(prompts):
            raise ValueError("new_tokens must be one number, or one per prompt")
        for prompt, count in zip(prompts, wanted):
            # the last id is picked and never fed back
            if prompt.numel() < 1 or count < 1 or prompt.numel() + count - 1 > self.state.capacity or \
                    self._pages_of(prompt.numel() + count - 1) > self.pages:
                raise ValueError("every prompt needs a token, a new one, and room for them in a row and in the pool")
        with torch.cuda.device(self.device):
            return self._run(prompts, wanted)

    def _run(self, prompts: list[torch.Tensor], wanted: list[int]) -> list[torch.Tensor]:
        self.state.reset()
        self._produced.zero_()
        waiting, running, done = list(range(len(prompts))), {}, {}   # running: row -> [prompt, ids produced]
        free_pages, active = self.pages, None
        while waiting or running:
            admitted, tokens = {}, 0
            for row in range(self.requests):
                if not waiting or row in running:
                    continue
                length = prompts[waiting[0]].numel()
                need = self._pages_of(length + wanted[waiting[0]] - 1)
                if need > free_pages or (admitted and tokens + length > self.prompt_tokens):
                    break
                free_pages -= need
                tokens += length
                index = waiting.pop(0)
                running[row] = [index, 1]
                admitted[row] = prompts[index]
            if admitted:
                self._prefill(admitted)
            else:
                now = sorted(running)
                if now != active:
                    counts = torch.zeros(self.requests, dtype=torch.int32)
                    counts[now] = 1
                    self._counts.copy_(counts)
                    active = now
                self._decode_step()
                for entry in running.values():
                    entry[1] += 1
            ended = [row for row, (index, count) in running.items() if count == wanted[index]]
            if ended:
                counts = torch.zeros(self.requests, dtype=torch.int32)
                counts[ended] = -self.state.capacity
                for row in ended:
                    index, count = running.pop(row)
                    done[index] = self._log[row, :count].clone()
                    free_pages += self._pages_of(prompts[index].numel() + count - 1)
                    self._produced[row] = 0
                self.state.reserve(counts.to(self.device), 0)
        self.state.check()
        return [done[index] for index in range(len(prompts))]
