"""Beam search over paged caches, on the device.

The reference samples one sequence greedily (src/spark_vllm_ascend/integration/
head.py:12-31).  Here a step of logits becomes the next step's rows without the host:
``torch_ops.beam_select`` takes each sequence's best continuations, ``DeviceBlockTables.fork``
the pages that they share and ``torch_ops.copy_pages`` the last pages that they write to.

    search = BeamSearch(tables, torch_ops.PageSet(cache.planes()), beams, eos_id)
    t = tables.step(lens)           # the prompts, in each sequence's first row
    ... logits [rows, vocab] of the prompts' last tokens ...
    for _ in range(n):
        search.step(logits)
        t = tables.step(search.query_lens())
        ... packed [rows, vocab] of packed_tokens(), at t's positions and slots ...
        logits = packed[search.last_rows(t)]
    search.sequences()
"""
from __future__ import annotations

import torch

from ..native import torch_ops
from .block_table import DeviceBlockTables


class BeamSearch:
    """The beams of several sequences: row s * beams + b of `tables` is sequence s's beam b,
    the best first; `pages` are the caches that the tables' pages are of.  A sequence
    starts with one beam, its prompt in row s * beams.  A beam ends with eos_id (-1: none
    does) and keeps its score and place among the others; it takes no more tokens, and its
    pages are given up.

    Nothing is read back, so that a step is not refused where the pool has no page left for
    a beam: one whose tokens the cache does not hold all (there was no page for its copy of
    a last page or for its new token, or the tables' max_tokens are fewer than the rows)
    offers nothing in the next step.  A sequence none of whose beams had room has scores
    of -inf alone.  (Whether the tables held the prompts is for the caller to see:
    tables.lens before the first step.)"""

    def __init__(self, tables: DeviceBlockTables, pages: torch_ops.PageSet, beams: int,
                 eos_id: int = -1, pad_id: int = 0):
        rows = tables.lens.numel()
        if not 1 <= beams <= 64 or rows % beams:
            raise ValueError("the tables must have `beams` rows, 1 to 64, for each sequence")
        if not isinstance(pages, torch_ops.PageSet):
            raise ValueError("pages must be a PageSet")
        if pages.num_blocks != tables.free_pages.numel():
            raise ValueError("the caches must have as many pages as the tables")
        self.tables, self.pages, self.beams = tables, pages, beams
        self.eos_id, self.pad_id = eos_id, pad_id
        dev = tables.lens.device
        self.scores = torch.zeros((rows // beams, beams), dtype=torch.float32, device=dev)
        self.scores[:, 1:] = float("-inf")
        self.done = torch.zeros(rows, dtype=torch.bool, device=dev)
        self._history: list = []
        self._held = None  # the tokens that each row of the tables must hold

    def step(self, logits: torch.Tensor) -> torch.Tensor:
        """Goes on from the rows' logits [rows, vocab] (those of a row without a score, or
        done, are not looked at): the rows' next tokens, int64 [rows], pad_id where a beam is
        done or there is none.  The tables' rows are those of the new beams, and
        tables.step(query_lens()) takes their tokens before the next step.  Not in a graph's
        capture: a step's scores and tokens are buffers of their own, that a replay would
        not go on from (beam_select, tables.fork and copy_pages can be captured)."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a step of BeamSearch cannot be captured: replays would start from "
                               "the same scores")
        lens = self.tables.lens
        if self._held is None:
            self._held = lens.clone()
        scores = torch.where(lens < self._held, float("-inf"), self.scores.view(-1))
        best = torch_ops.beam_select(logits, scores, self.beams, self.beams, done=self.done,
                                     pad_id=self.pad_id)
        parents, tokens = best.parents.view(-1), best.tokens.view(-1)
        at = parents.clamp(min=0).long()
        self.scores = best.scores
        self.done = (tokens == self.eos_id) | self.done[at] | (parents < 0)
        self._held = torch.where(self.done, 0, self._held[at] + 1)
        going_on = torch.where(self.done, -1, parents)
        torch_ops.copy_pages(self.pages, self.tables.fork(going_on))
        self._history.append((parents, torch.where(parents < 0, self.pad_id, tokens)))
        return self._history[-1][1]

    def query_lens(self) -> torch.Tensor:
        """The tokens a row takes in the next step, 1 or 0: tables.step's argument.  What the
        model is given for them is packed_tokens(), not step's tokens, once a beam is done."""
        return (~self.done).to(torch.int32)

    def packed_tokens(self) -> torch.Tensor:
        """The rows' next tokens as tables.step(query_lens()) packs them, int64 [rows]: row
        after row those of the beams that go on, pad_id behind them (of no sequence: their
        slots are -1)."""
        if not self._history:
            raise RuntimeError("there is no token before the first step")
        rows, tokens = self.done.numel(), self._history[-1][1]
        out = tokens.new_full((rows + 1,), self.pad_id)
        out[torch.where(self.done, rows, torch.cumsum(~self.done, 0) - 1)] = tokens
        return out[:rows]

    def last_rows(self, tables: torch_ops.RequestTables) -> torch.Tensor:
        """Where the rows' last tokens stand in the packed tokens of a tables.step, int64
        [rows]: step's logits are those there.  (Any of a row that takes no tokens, whose
        logits are not looked at.)"""
        return (tables.query_start_loc[1:].long() - 1).clamp(min=0)

    def sequences(self) -> torch.Tensor:
        """The beams' tokens so far, int64 [seqs, beams, steps], the best first (`scores`;
        rows of -inf are no beams), pad_id behind the end of one that is done."""
        rows = self.done.numel()
        at = torch.arange(rows, device=self.done.device)
        out = []
        for parents, tokens in reversed(self._history):
            out.append(tokens[at])
            at = parents[at].clamp(min=0).long()
        if not out:
            return at.new_zeros((rows // self.beams, self.beams, 0))
        return torch.stack(out[::-1], 1).view(rows // self.beams, self.beams, -1)
