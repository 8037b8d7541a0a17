"""Paged KV cache of the gated full-attention layers, on the device.

The reference verifies its tree over SGLang's paged cache: SGLang keeps the
page tables (req_to_token), hands out the slots of new tokens and moves the
accepted ones (fc1_branch64.py:31-34, :44).  A host without SGLang keeps them
here: page tables, free stack and caches live on the GPU, and every step is
four operators on the current stream with no host read-back --

    plan    tables and maps from the requests' lengths   dft_page_plan
    append  a layer's new K / V rows into their slots    dft_kv_append
    attend  causal attention of the new tokens           dft_chunk_attn
            (a tree's nodes: tree(), dft_tree_attn)
    commit  the accepted path's rows compacted           dft_kv_commit

so prompts, single tokens and tree steps can be captured and replayed at any
lengths.  Steps of one cache run in stream order: its tables are shared.
"""
from __future__ import annotations

import torch

from . import _lib as L
from . import kernels as K


class PagedKV:
    """rows: requests that may hold pages at a time; max_len: longest request
    in tokens; n_pages: pages of the pool (default: every row at max_len)."""

    def __init__(self, rows, max_len, layers, Hkv, D, page_size=16, n_pages=None, dtype=torch.bfloat16, device=None):
        if rows <= 0 or max_len <= 0 or layers <= 0 or page_size <= 0:
            raise L.DFTError("PagedKV: rows, max_len, layers and page_size must be positive")
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.device, self.page_size, self.max_len = dev, int(page_size), int(max_len)
        max_pages = -(-self.max_len // self.page_size)
        self.n_pages = rows * max_pages if n_pages is None else int(n_pages)
        self.block_table = torch.full((rows, max_pages), -1, dtype=torch.int32, device=dev)
        self.held = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(self.n_pages - 1, -1, -1, dtype=torch.int32, device=dev)
        self.n_free = torch.full((1,), self.n_pages, dtype=torch.int32, device=dev)
        slots = self.n_pages * self.page_size
        self.k_cache = torch.zeros(layers, slots, Hkv, D, dtype=dtype, device=dev)
        self.v_cache = torch.zeros_like(self.k_cache)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.maps = None

    def outputs(self, B, tokens):
        """Map buffers for plans of B requests and at most `tokens` new tokens,
        to be kept across steps (a captured step needs them to stay)."""
        keys = min(self.k_cache.shape[1], B * self.block_table.shape[1] * self.page_size)
        return K.page_plan_outputs(B, tokens, keys, self.device)

    def plan(self, cached, fresh, tokens=None, rows=None, out=None):
        """Bring request b (table row rows[b], or b) to cached[b] + fresh[b]
        tokens and make the step's maps; `tokens` bounds sum(fresh) when out is
        not given.  cached = fresh = 0 gives a request's pages back."""
        if out is None:
            if tokens is None:
                raise L.DFTError("PagedKV.plan: pass tokens (a bound on the new tokens) or out")
            out = self.outputs(cached.numel(), int(tokens))
        self.maps = K.page_plan(cached, fresh, self.block_table, self.held, self.free_pages, self.n_free,
                                self.page_size, rows=rows, out=out, status=self.status)
        return self.maps

    def _planned(self):
        if self.maps is None:
            raise L.DFTError("PagedKV: plan first")
        return self.maps

    def append(self, layer, k, v):
        """k, v [tokens, Hkv, D] of the planned new tokens into layer's cache."""
        m = self._planned()
        K.kv_append(k, v, self.k_cache[layer], self.v_cache[layer], m["slot_map"], status=self.status)

    def attend(self, layer, q, sm_scale=None, o=None):
        """Causal attention of the planned new tokens, q [tokens, Hq, D]."""
        m = self._planned()
        return K.chunk_attention(q, self.k_cache[layer], self.v_cache[layer], m["qo_indptr"], m["kv_indptr"],
                                 m["kv_indices"], sm_scale=sm_scale, o=o, status=self.status)

    def tree(self, anc, Hq, sm_scale=None):
        """The tree-masked verify over the planned keys, whose last N per
        request are the tree's nodes: a planned TreeAttentionWrapper that reads
        anc [B, N, N] (float32, or converted at every run) and the buffers of the
        last plan at every run (plan later steps into them: out=maps).  How a
        request's keys are split follows the table's width, max_len, since the
        host knows no lengths."""
        from .tree_attn import TreeAttentionWrapper
        m = self._planned()
        B = m["qo_indptr"].numel() - 1
        if anc.dim() != 3 or anc.shape[0] != B or anc.shape[1] != anc.shape[2]:
            raise L.DFTError("PagedKV.tree: anc is [B, N, N] for the planned B requests")
        if anc.device != m["qo_indptr"].device:
            raise L.DFTError(f"PagedKV.tree: anc is read at every run and must be on {m['qo_indptr'].device}")
        N = anc.shape[1]
        Hkv, D = self.k_cache.shape[2:]
        longest = self.block_table.shape[1] * self.page_size
        t = TreeAttentionWrapper(self.device).plan(m["kv_indptr"], m["kv_indices"], Hq, Hkv, D, n=N, anc=anc,
                                                   kv_lens_host=[max(longest, N)] * B, sm_scale=sm_scale,
                                                   live_anc=True)
        t.status = self.status
        return t

    def commit(self, path, accept_len, N):
        """Compact the accepted path's rows of every layer (path, accept_len as
        accept_greedy returns them); the caller then counts min(accept_len, P)
        of the N planned tokens as cached."""
        m = self._planned()
        K.kv_commit(self.k_cache, self.v_cache, m["kv_indptr"], m["kv_indices"], path, accept_len, N,
                    status=self.status)

    def device_status(self) -> int:
        """Bits raised so far (DFT_DEV_*); reads the device (syncs)."""
        return int(self.status.item())
