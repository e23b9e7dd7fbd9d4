"""Ragged requests decoding over a paged KV cache, with verified drafts.

The counterpart of ``graph_decode.DecodeStep`` for requests of different
lengths: prompts are packed without padding, every request has its own
position, and a step may give a request several drafted tokens and keep only
those that the target accepts.

    step = PagedDecode.new(mgr, batch, max_len)
    first = step.prefill(mgr, prompts, names)        # a list of 1-D id tensors
    step.input_ids.copy_(first)
    mgr._setup_forward_batch(names, seq_lens=[1] * batch)
    graph, out = capture_graph(mgr, step)            # then graph.replay() per token

    mgr._setup_forward_batch(names, seq_lens=[k + 1] * batch)
    accepted, tokens = step.verify(mgr, drafts, draft_probs, accept, last)

Lengths, pages and positions live on the device (``kernels.page_tables``); no
step synchronises with the host.  Pages that rejected drafts took go back to
the pool with the next step's tables.  GPU, float16 or bfloat16 models.

A token that finds no place (the pool is short of pages, or the request is at
its table's end) is not cached and does not count: ``placed`` says how many of
each request's tokens the last step had room for.  A request with none keeps
its length and has to be given the same token again once others have left:

    graph.replay()
    nxt = out.logits.argmax(-1, keepdim=True)
    step.input_ids.copy_(torch.where(step.placed[:, None] > 0, nxt, step.input_ids))
"""

from __future__ import annotations

from typing import Dict, Optional, Sequence, Tuple

import torch

from .decoder import PagedKV
from .kernels.paged import PagedStep, verify_drafts


class PagedDecode:
    """Resident state of ``batch`` requests; the pool holds ``num_pages`` pages of ``page`` positions."""

    def __init__(self, mgr, batch: int, max_len: int, *, page: int = 16, num_pages: Optional[int] = None) -> None:
        device, dtype = mgr.pool.device, mgr.pool.dtype
        self.batch, self.max_len, self.start = batch, max_len, 0
        self.kv = PagedKV(mgr.model.config, batch, max_len, device, dtype, page=page, num_pages=num_pages)
        i32 = dict(dtype=torch.int32, device=device)
        self.input_ids = torch.zeros((batch, 1), dtype=torch.long, device=device)
        self.lens = torch.zeros(batch, **i32)         # cached positions of each request
        self.start_lens = torch.zeros(batch, **i32)   # its prompt's length, for rewind
        self.placed = torch.zeros(batch, **i32)       # tokens of each that the last step had room for
        self.one = torch.ones(batch, **i32)
        self.none = torch.zeros(batch, **i32)
        self.step = self.kv.new_step(batch, 1)
        self._chunks: Dict[int, Tuple[PagedStep, torch.Tensor]] = {}

    @classmethod
    def new(cls, mgr, batch: int, max_len: int, **kwargs) -> "PagedDecode":
        return cls(mgr, batch, max_len, **kwargs)

    @property
    def kv_pos(self) -> torch.Tensor:
        return self.lens

    def rewind(self) -> None:
        """Every request back to the end of its prompt; the pages after it go
        back to the pool.  One that is not that far (it has left) stays."""
        torch.minimum(self.lens, self.start_lens, out=self.lens)
        self.kv.tables(self.lens, self.none, self.kv.new_step(0, 0))

    def prefill(self, mgr, prompts: Sequence[torch.Tensor], lora_names) -> torch.Tensor:
        """Run the prompts, packed, each with its adapter, into an empty cache;
        the greedy next token of every request, ``(batch, 1)``."""
        counts = [int(p.numel()) for p in prompts]
        if len(counts) != self.batch or min(counts) < 1 or max(counts) >= self.max_len:
            raise ValueError(f"{self.batch} prompts of 1 to {self.max_len - 1} tokens expected, got {counts}")
        need, pages = sum(-(-c // self.kv.page) for c in counts), self.kv.state.free.numel()
        if need > pages:
            raise ValueError(f"the prompts need {need} pages of {self.kv.page} positions, the pool has {pages}")
        device = self.lens.device
        ends = torch.tensor(counts, dtype=torch.int32).cumsum(0) - 1
        self.start = max(counts)
        self.start_lens.copy_(torch.tensor(counts, dtype=torch.int32))
        self.lens.zero_()  # and so it stays if the prompts do not get through
        self.kv.tables(self.none, self.none, self.kv.new_step(0, 0))
        step = self.kv.tables(self.none, self.start_lens, self.kv.new_step(sum(counts), max(counts)))
        out = mgr.forward_with_lora(input_ids=torch.cat([p.reshape(-1) for p in prompts]).to(device), lora_names=lora_names,
                                    seq_lens=counts, past_key_values=self.kv, paged_step=step,
                                    logit_rows=ends.to(device))
        self.lens.copy_(self.start_lens)
        self.placed.copy_(self.start_lens)
        return out.logits.argmax(dim=-1, keepdim=True)

    def run(self, mgr):
        """One token of every request: ``input_ids`` at its position, which then
        advances.  Logits of a request whose token has no place are NaN."""
        self.kv.tables(self.lens, self.one, self.step)
        out = mgr.model(input_ids=self.input_ids, past_key_values=self.kv, paged_step=self.step)
        torch.ge(self.step.slots, 0, out=self.placed)
        self.lens.add_(self.placed)
        return out

    def verify(self, mgr, drafts: torch.Tensor, draft_probs: Optional[torch.Tensor], accept: torch.Tensor,
               last: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """``input_ids`` and the ``k`` drafted tokens ``drafts [batch, k]`` of
        every request in one step; ``kernels.verify_drafts``' accepted counts and
        tokens for the numbers ``accept [batch, k]`` and ``last [batch]``.  Every
        request keeps its accepted drafts, and ``input_ids`` becomes the token
        after them (0 where the probabilities had no mass).  Drafts without a
        place are not looked at; a request without any keeps its ``input_ids``,
        and its tokens are -1."""
        k = int(drafts.shape[1])
        if k not in self._chunks:
            if self.lens.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"the step of {k} drafts does not exist yet: its lengths would only be written when the "
                                   "graph runs; verify as many drafts once before capturing")
            self._chunks[k] = (self.kv.new_step(self.batch * (k + 1), k + 1), torch.full_like(self.one, k + 1))
        step, new = self._chunks[k]
        self.kv.tables(self.lens, new, step)
        ids = torch.cat((self.input_ids, drafts), dim=1)
        # A request's first rows are the ones with a place: they come first among the target's rows.
        outside = (step.slots < 0).view(self.batch, k + 1)
        torch.sum(~outside, 1, dtype=torch.int32, out=self.placed)
        rows = torch.argsort(outside.view(-1), stable=True)
        indptr = torch.cat((self.none[:1], self.placed.cumsum(0, dtype=torch.int32)))
        logits = mgr.model(input_ids=ids, past_key_values=self.kv, paged_step=step, logit_rows=rows).logits
        probs = torch.softmax(logits.float(), dim=-1)
        accepted, tokens = verify_drafts(probs, draft_probs, drafts, indptr, accept, last)
        some = self.placed > 0
        self.lens.add_(accepted).add_(some)
        after = tokens.gather(1, accepted.long()[:, None]).clamp_(min=0)
        self.input_ids.copy_(torch.where(some[:, None], after, self.input_ids))
        return accepted, tokens
