"""Sessions that grow token by token, in pages of a shared pool.

`SessionSlab` gives every session a ring of the same length and overwrites its
oldest frame.  `PagedSlab` keeps one layer's caches of sessions whose lengths
differ: a session holds pages of a pool, takes more as it grows and gives them
back when it ends.  A session that has a budget instead stops growing there: a
new token takes the place of the held one that attention has looked at least
(per kv head, by the softmax weight each token was given so far), so its pages
never change and its steps can be captured in a CUDA graph.

    slab = PagedSlab(64, H=16, Dh=128, dtype=torch.bfloat16, page=64, n_pages=4096, max_tokens=8192)
    slab.reserve(i, 4096)                       # pages for session i, once
    y = slab.append_and_attend(q, k, v)         # one decoding step of all sessions

The host never reads the device: pages are handed out by `reserve`, which the
caller asks for what a session is going to hold.  A token for which its session
has no page is dropped, with those behind it, and reported by `ops.check_status`:
`lens` counts what is held, so a session can go on after a later `reserve`.
"""
from __future__ import annotations

from typing import List, Optional

import torch
from torch import Tensor

from . import ops


class PagedSlab:
    """One layer's paged K/V caches of `n_sessions` sessions (state as described in include/we_b200.h).

    A budget (`keep`) also sets the width of the table, and with it the workspaces of a step: it can be lowered later, not
    raised."""

    def __init__(self, n_sessions: int, H: int, Dh: int, dtype: torch.dtype, page: int, n_pages: int,
                 max_tokens: int, keep: Optional[int] = None, sink: int = 0, recent: int = 0, device="cuda"):
        if page not in (16, 32, 64, 128, 256):
            raise ValueError("page must be 16, 32, 64, 128 or 256 tokens")
        if min(n_sessions, H, n_pages, max_tokens) < 1:
            raise ValueError("sessions, heads, pages and tokens must be at least 1")
        if keep is not None and not (0 <= sink and 0 <= recent and 1 <= keep and sink + recent <= keep <= max_tokens):
            raise ValueError("a budget needs 0 <= sink + recent <= keep <= max_tokens")
        self.n_sessions, self.page = n_sessions, page
        self.keep, self.sink, self.recent = keep, sink, recent
        # (what a session can come to hold: workspaces are sized by the width of the table)
        self.max_tokens = max_tokens
        self.max_pages = -(-(max_tokens if keep is None else keep) // page)
        self.kv = torch.zeros(2, n_pages, H, page, Dh, dtype=dtype, device=device)
        self.weights = torch.zeros(n_pages, H, page, dtype=torch.float32, device=device)
        self.positions = torch.zeros(n_pages, H, page, dtype=torch.int32, device=device)
        self.table = torch.full((n_sessions, self.max_pages), -1, dtype=torch.int32, device=device)  # -1: no page
        self.lens = torch.zeros(n_sessions, H, dtype=torch.int32, device=device)
        self.next_pos = torch.zeros(n_sessions, H, dtype=torch.int32, device=device)
        if self.kv.is_cuda:
            # made here, not within the first captured step: a graph that holds its making clears it at every replay
            ops.status_word(self.kv.device)
        self._free: List[int] = list(range(n_pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(n_sessions)]

    # -- pages (host bookkeeping) --------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def room(self, i: int) -> int:
        """Tokens session i has pages for."""
        return len(self._pages[i]) * self.page

    def reserve(self, i: int, tokens: int) -> None:
        """Pages for `tokens` tokens of session i, under a budget for no more than that (what it has already counts;
        none are given back)."""
        have, want = self._pages[i], -(-tokens // self.page)
        if want > -(-self.max_tokens // self.page):
            raise ValueError(f"a session holds at most {-(-self.max_tokens // self.page) * self.page} tokens")
        want = min(want, self.max_pages)
        if want - len(have) > len(self._free):
            raise RuntimeError(f"the pool has {len(self._free)} free pages, session {i} needs {want - len(have)} more")
        if want <= len(have):
            return
        new = [self._free.pop() for _ in range(want - len(have))]
        self.table[i, len(have):want] = torch.tensor(new, dtype=torch.int32)
        have += new

    def release(self, i: int) -> None:
        """Ends session i: its pages go back to the pool and it holds nothing."""
        self._free += reversed(self._pages[i])
        self._pages[i] = []
        self.table[i].fill_(-1)
        self.lens[i].zero_()
        self.next_pos[i].zero_()

    # -- the layer-step ------------------------------------------------------
    def append(self, k: Tensor, v: Tensor, n_new: Optional[Tensor] = None, w_new: Optional[Tensor] = None) -> None:
        """k / v [S, H, T, Dh]: T new tokens of every session, or the first `n_new[s]` of them (int32 [S], on the
        device); `w_new` float32 [S, H, T] the weights they come with.  Under a budget the least attended tokens
        are evicted.  Every session must have pages for what it holds afterwards (`reserve`)."""
        if self.keep is not None:
            a = (self.kv, self.table, self.lens, self.next_pos, k, v, self.weights, self.positions, self.keep,
                 self.sink, self.recent, n_new, w_new)
            (ops.paged_append_evict_op if torch.compiler.is_compiling() else ops.paged_append_evict_)(*a)
        else:
            a = (self.kv, self.table, self.lens, self.next_pos, k, v, n_new, self.weights, self.positions, w_new)
            (ops.paged_append_op if torch.compiler.is_compiling() else ops.paged_append_)(*a)

    def attend(self, q: Tensor, scale: float = 0.0, n_new: Optional[Tensor] = None) -> Tensor:
        """q [S, Hq, 1, Dh] over what every session holds; under a budget the weights are added up.  Sessions with
        `n_new[s] == 0` sit out: their rows of the output are 0 and their weights stay as they are."""
        weights = self.weights if self.keep is not None else None
        if torch.compiler.is_compiling():
            return ops.paged_attn_op(q, self.kv, self.table, self.lens, float(scale), weights, n_new)
        return ops.paged_attn(q, self.kv, self.table, self.lens, float(scale), weights, n_new=n_new)

    def append_and_attend(self, q: Tensor, k: Tensor, v: Tensor, n_new: Optional[Tensor] = None,
                          scale: float = 0.0) -> Tensor:
        """One decoding step: append k / v [S, H, 1, Dh], then attend with q [S, Hq, 1, Dh].  Sessions with
        `n_new[s] == 0` sit the step out (their rows of q, k and v are not read): nothing of theirs changes, and their
        rows of the output are 0."""
        self.append(k, v, n_new)
        return self.attend(q, scale, n_new)
