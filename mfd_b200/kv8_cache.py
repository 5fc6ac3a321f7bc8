"""An 8-bit paged K/V cache of one attention layer for a batch of requests: the pages, their owners and the four operators
on them (ops.kv8_append, kv8_attention, kv8_page_weights, kv8_evict) with the bookkeeping between.

A page holds page_size consecutive tokens of one request for every KV head, K and V in int8 or float8 e4m3 with one
float32 scale per page, KV head and tensor.  A verify step reads the cache and the tree's own bf16 keys (attention), counts
the attention weight of the accepted nodes per page (weigh), quantises their keys and values into the open pages
(append), and drops the least used pages of requests that have grown past their budget (evict).

Which request owns which page is decided on the host: reserve() and evict() read a few integers back (they
synchronise); attention(), weigh() and append() only launch.

What it does not do:
- Pages come back through evict() alone.  A request that has finished keeps its pages, and reserve() makes room for as many
  tokens in every request: a server that admits and retires requests keeps its own tables and calls the operators.
- append() and evict() bind seq_lens (and evict() page_table and mass) to new tensors, so a CUDA graph of a whole step is built
  from the operators, with tensors that stay.
- After an eviction seq_lens counts the tokens that are held, not those that were seen.  The position of the next token, for
  rotary embeddings, is the caller's to keep.
- Pages enter with mass 0, a prompt's too, and the attention among a step's own nodes is credited to no page: mass is what later
  steps gave a page through weigh().
"""

from __future__ import annotations

import torch

from . import ops


class KV8Cache:
    def __init__(self, batch: int, num_pages: int, num_kv_heads: int, max_pages: int, page_size: int = 64,
                 head_dim: int = 128, dtype: torch.dtype = torch.int8, device="cuda"):
        """num_pages in the pool, at most max_pages a request.  dtype: torch.int8 or torch.float8_e4m3fn."""
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        self.page_size = page_size
        self.k = torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)
        self.v = torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)
        self.k_scale = torch.ones(num_pages, num_kv_heads, device=device)
        self.v_scale = torch.ones(num_pages, num_kv_heads, device=device)
        self.page_table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.mass = torch.zeros(batch, max_pages, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self._free = list(range(num_pages))
        self._pages = [0] * batch  # pages a request owns

    def reserve(self, tokens: int) -> None:
        """Give every request pages for `tokens` more tokens.  Reads the lengths back.  All or nothing: where it raises,
        no request has got a page."""
        self._check_status()
        need = [-(-(t + tokens) // self.page_size) for t in self.seq_lens.tolist()]
        for b, n in enumerate(need):
            if n > self.page_table.shape[1]:
                raise RuntimeError(f"KV8Cache: request {b} needs {n} pages, its table holds {self.page_table.shape[1]}")
        places = [(b, i) for b, n in enumerate(need) for i in range(self._pages[b], n)]
        if len(places) > len(self._free):
            raise RuntimeError(f"KV8Cache: no free page for {len(places) - len(self._free)} of the {len(places)} wanted")
        if places:
            ids = self._free[-len(places):]
            at = torch.tensor(places, device=self.page_table.device).t()
            self.page_table[at[0], at[1]] = torch.tensor(ids, dtype=torch.int32, device=self.page_table.device)
            del self._free[-len(places):]
            self._pages = [max(p, n) for p, n in zip(self._pages, need)]

    def _check_status(self) -> None:
        if int(self.status):
            raise RuntimeError("KV8Cache: an append found no page for some of its rows, which the lengths count (set seq_lens to "
                               "what the pages hold and status to 0 to go on)")

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor, path: torch.Tensor | None = None,
               counts: torch.Tensor | None = None) -> None:
        """Quantise rows of k_new, v_new [bs, n, Hkv, D] into the cache: a prompt (counts rows each), or the accepted
        path of a tree.  The pages must be there (reserve).  Where one was not, its rows are lost, though the length counts
        them, self.status becomes nonzero, and reserve() and evict() raise."""
        self.seq_lens = ops.kv8_append(self.k, self.v, self.k_scale, self.v_scale, k_new, v_new, self.page_table,
                                       self.seq_lens, path=path, counts=counts, status=self.status)

    def attention(self, q: torch.Tensor, scale: float, k_new: torch.Tensor | None = None,
                  v_new: torch.Tensor | None = None, anc: torch.Tensor | None = None, return_lse: bool = False):
        """q [bs, n, H, D] over the cached tokens and the nodes' own keys (ops.kv8_attention)."""
        return ops.kv8_attention(q, self.k, self.v, self.k_scale, self.v_scale, self.page_table, self.seq_lens, scale,
                                 k_new=k_new, v_new=v_new, anc=anc, return_lse=return_lse)

    def weigh(self, q: torch.Tensor, lse: torch.Tensor, scale: float, path: torch.Tensor | None = None,
              counts: torch.Tensor | None = None, decay: float = 1.0) -> None:
        """Add the accepted nodes' attention weights to the pages' mass (before their rows are appended)."""
        ops.kv8_page_weights(q, lse, self.k, self.k_scale, self.page_table, self.seq_lens, scale, self.mass, path=path,
                             counts=counts, decay=decay, out=self.mass)

    def evict(self, keep_pages: int, sink_pages: int = 1, recent_pages: int = 2) -> list[list[int]]:
        """Drop the pages of least mass of every request that fills more than keep_pages; they return to the pool.
        Returns the dropped page ids per request.  Pages that are reserved but still empty stay with their request."""
        self._check_status()
        table, mass, lens, freed, counts = ops.kv8_evict(self.page_table, self.mass, self.seq_lens, self.page_size,
                                                         keep_pages, sink_pages, recent_pages)
        n = counts.tolist()
        gone = [row[:c] for row, c in zip(freed.tolist(), n)] if any(n) else [[] for _ in n]
        if any(n):
            old, used = self.page_table.tolist(), self.seq_lens.tolist()
            rows, cols, ids = [], [], []
            for b, t in enumerate(used):
                filled = -(-t // self.page_size)
                for i, page in enumerate(old[b][filled:self._pages[b]]):  # reserved ahead: behind the pages that stay
                    rows.append(b)
                    cols.append(filled - n[b] + i)
                    ids.append(page)
                self._pages[b] -= n[b]
                self._free.extend(gone[b])
            if ids:
                at = torch.tensor([rows, cols, ids], device=table.device)
                table[at[0], at[1]] = at[2].to(torch.int32)
            self.page_table, self.mass, self.seq_lens = table, mass, lens
        return gone
