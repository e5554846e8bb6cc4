"""Paged key/value history on B200: rotary embedding, page writes, attention.

The history of the streaming stack is one ring per stream (`rope_kv`,
`history_attention`; the reference keeps one bounded buffer per stream,
fast_moss/streaming.py:68-79).  Here sequences of very different length
share one pool of pages, a batch may hold any number of new tokens of each
sequence (a prompt beside single tokens), key heads may be shared by groups
of query heads, and heads are 64 or 128 wide.

  k_pages, v_pages  contiguous bf16 [pages, kv_heads, page_size, head_dim],
                    page_size 16, 32, 64, 128 or 256
  page_table        int32 [sequences, columns]: position p of sequence s
                    lies in page page_table[s, p // page_size], row
                    p % page_size
  q_start           int64 [sequences + 1], not decreasing: sequence s owns
                    the packed rows q_start[s] .. q_start[s + 1] - 1
  kv_len            int64 [sequences]: positions with the new tokens, which
                    are the last ones

The index tensors stay on the device, so a captured call can be replayed
with other lengths, tables and row counts in them.
What they say wrongly (a page outside the pool, a position outside the table,
for `rope_paged_kv` a row beyond the packed ones) is left out and reported
through the device error word.
"""

import torch

from . import _lib


def rope_paged_kv(q, k, v, q_start, kv_len, page_table, max_period, k_pages, v_pages, *,
                  q_weight=None, k_weight=None, eps=1e-6, interleaved=True):
    """Rotary embedding of a ragged batch of new tokens, the rotated keys and
    the values written into their pages (`rope_kv` for a paged history).

    q [N, Hq, D], k and v [N, Hkv, D] (BF16 or FP32, any strides, D 64 or
    128), packed rows of all sequences; the rest as in the module's
    description.  q_weight, k_weight: FP32 [D] RMS norm weights applied
    before the rotation (None: no norm), as in `qk_norm_rope`.  Returns the
    rotated queries as contiguous bf16 [N, Hq, D]; rows of no sequence are
    not written.  Positions outside the table and pages outside the pool are
    skipped and reported through the device error word.
    """
    return _lib.binding().rope_paged_kv(q, k_pages, v_pages, q_start, kv_len, page_table, k, v,
                                        q_weight, k_weight, max_period, eps, interleaved)


def paged_attention(q, k_pages, v_pages, q_start, kv_len, page_table, *, context=None, scale=None,
                    max_tokens=None, out=None):
    """Causal attention of a ragged batch of new tokens over their paged
    history (`history_attention` for a paged history).

    q: bf16 [N, Hq, D], packed rows of all sequences (Hq a multiple of the
    pages' Hkv, D 64 or 128); the new tokens' keys and values are already in
    their pages (`rope_paged_kv`).  The token at position p attends to
    positions (p - context, p] (context None: all), with scale 1/sqrt(D) by
    default.  max_tokens: an upper bound of the new tokens of any sequence,
    if the caller knows one without reading the device; it only chooses
    between kernels.  Returns bf16 [N, Hq, D] (or fills `out`); rows of no
    sequence are not written, rows that attend to nothing are zero.
    """
    if context is not None and context < 1:
        raise ValueError("context must be at least 1")
    if max_tokens is not None and max_tokens < 1:
        raise ValueError("max_tokens must be at least 1")
    return _lib.binding().paged_attention(q, k_pages, v_pages, q_start, kv_len, page_table,
                                          context or 0, scale, max_tokens or 0, out)


class PagedHistory:
    """Paged attention history of many sequences over every layer of a stack.

    All sequences share `pages` pages of `page_size` positions (the same page
    numbers in every layer), taken as they grow and given back when they are
    reset or, with a window of `context` positions, once every position of a
    page lies before it.  Pages are accounted for on the host; the tensors that
    the kernels read are updated in place, on the current stream:

      k_pages[i], v_pages[i]  [pages, heads, page_size, head_dim] bf16 of layer i
      page_table              int32 [sequences, columns], -1 where there is no page
      q_start                 int64 [sequences + 1], rows of the step in progress
      kv_len                  int64 [sequences], positions with that step

    A sequence holds at most `max_positions` positions.  `lengths` and `rows` are
    kv_len and q_start[-1] as the host knows them.
    """

    def __init__(self, layers, sequences, heads, head_dim, device, *, pages, max_positions,
                 page_size=16, context=None):
        if min(layers, sequences, heads, pages, max_positions) < 1:
            raise ValueError("layers, sequences, heads, pages and max_positions must be positive")
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError("page_size must be 16, 32, 64, 128 or 256")
        if context is not None and context < 1:
            raise ValueError("context must be at least 1")
        self.sequences = sequences
        self.page_size = page_size
        self.context = context
        self.max_positions = max_positions
        columns = -(-max_positions // page_size)
        shape = (pages, heads, page_size, head_dim)
        self.k_pages = [torch.zeros(shape, device=device, dtype=torch.bfloat16)
                        for _ in range(layers)]
        self.v_pages = [torch.zeros(shape, device=device, dtype=torch.bfloat16)
                        for _ in range(layers)]
        self.page_table = torch.full((sequences, columns), -1, device=device, dtype=torch.int32)
        self.q_start = torch.zeros(sequences + 1, device=device, dtype=torch.int64)
        self.kv_len = torch.zeros(sequences, device=device, dtype=torch.int64)
        self.lengths = [0] * sequences
        self.rows = 0
        self._free = list(range(pages - 1, -1, -1))
        self._pages = [{} for _ in range(sequences)]  # column -> page
        self._changed = {}  # entries of page_table (flat) that the device lacks

    @property
    def free_pages(self):
        return len(self._free)

    def _needed(self, new):
        """Columns that each sequence's next `new` positions need and lack."""
        size = self.page_size
        return [[c for c in range(have // size, -(-(have + n) // size)) if c not in held]
                for have, n, held in zip(self.lengths, new, self._pages)]

    def advance(self, new):
        """Makes room for new[s] tokens of every sequence s (0 for those that
        pause) and points the index tensors at them.  Returns the number of
        packed rows.  Raises, with nothing changed, ValueError where a sequence
        would pass `max_positions` and RuntimeError where the pages do not
        suffice (reset a sequence, or advance fewer)."""
        new = [int(n) for n in new]
        if len(new) != self.sequences or min(new) < 0:
            raise ValueError("expected a token count, 0 or more, for every sequence")
        if any(have + n > self.max_positions for have, n in zip(self.lengths, new)):
            raise ValueError(f"a sequence holds at most {self.max_positions} positions")
        gone = self._behind_window()
        needed = self._needed(new)
        if sum(map(len, needed)) > len(self._free) + sum(map(len, gone)):
            raise RuntimeError("out of history pages")
        for s, columns in enumerate(gone):
            self._give_back(s, columns)
        start = [0]
        for s, n in enumerate(new):
            for c in needed[s]:
                page = self._free.pop()
                self._pages[s][c] = page
                self._changed[s * self.page_table.shape[1] + c] = page
            self.lengths[s] += n
            start.append(start[-1] + n)
        self.rows = start[-1]
        with torch.inference_mode():
            if self._changed:
                device = self.page_table.device
                at = torch.tensor(list(self._changed)).to(device)
                page = torch.tensor(list(self._changed.values()), dtype=torch.int32).to(device)
                self.page_table.view(-1).index_copy_(0, at, page)
                self._changed.clear()
            self.q_start.copy_(torch.tensor(start))
            self.kv_len.copy_(torch.tensor(self.lengths))
        return self.rows

    def _behind_window(self):
        """Columns of every sequence whose positions no later token attends to."""
        if self.context is None:
            return [[] for _ in range(self.sequences)]
        return [[c for c in held if (c + 1) * self.page_size <= have - self.context + 1]
                for have, held in zip(self.lengths, self._pages)]

    def _give_back(self, s, columns):
        for c in columns:
            self._free.append(self._pages[s].pop(c))
            self._changed[s * self.page_table.shape[1] + c] = -1

    def reset(self, sequences=None):
        """Starts the given sequences (all by default) afresh; their pages go
        back to the pool.  Raises ValueError, with nothing changed, where one does
        not exist."""
        sequences = list(range(self.sequences) if sequences is None else sequences)
        for s in sequences:
            if not 0 <= s < self.sequences:
                raise ValueError(f"no sequence {s}")
        for s in sequences:
            self._give_back(s, list(self._pages[s]))
            self.lengths[s] = 0
