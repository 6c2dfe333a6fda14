"""Paged KV cache resident on the GPU of a stage owner.

Pages hold 64 tokens of one layer's K (and V) for every local KV head:
``k[layer] : [num_pages, Hkv, 64, 128]``, bf16 or (``kv_dtype="fp8"``) e4m3 with
one scale byte per token, head and side (:mod:`..ops.kv_fp8`; 258 bytes a token
and head instead of 512).  A sequence owns an ordered list of pages (its block-table row); pages are reference counted so a forked
sequence can share a prefix copy-on-write.

The reference keeps a static ``[B, Hkv, Smax, D]`` tensor per layer with
prepare/commit append, snapshot/restore/fork/rollback
(si/model/qwen3_cache.py:25-360); paging replaces the static slab so that
sequences of different lengths share one pool without fragmentation.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch

PAGE = 64


class OutOfPages(RuntimeError):
    pass


class PageAllocator:
    """Free-list page allocator with reference counts (host side)."""

    def __init__(self, num_pages: int):
        self.num_pages = num_pages
        self._free = list(range(num_pages - 1, -1, -1))
        self._ref = [0] * num_pages

    @property
    def free(self) -> int:
        return len(self._free)

    def alloc(self, n: int) -> list[int]:
        if n > len(self._free):
            raise OutOfPages(f"need {n} pages, {len(self._free)} free")
        out = [self._free.pop() for _ in range(n)]
        for p in out:
            self._ref[p] = 1
        return out

    def retain(self, pages: list[int]) -> None:
        for p in pages:
            self._ref[p] += 1

    def release(self, pages: list[int]) -> None:
        for p in pages:
            self._ref[p] -= 1
            if self._ref[p] == 0:
                self._free.append(p)
            elif self._ref[p] < 0:
                raise RuntimeError(f"page {p} released twice")

    def refcount(self, p: int) -> int:
        return self._ref[p]


@dataclass
class SeqPages:
    pages: list[int] = field(default_factory=list)
    length: int = 0  # tokens stored


class PagedKVCache:
    def __init__(self, num_layers: int, num_kv_heads: int, num_pages: int, device,
                 head_dim: int = 128, dtype=torch.bfloat16, latent_dim: int | None = None,
                 kv_dtype: str = "bf16"):
        """``latent_dim`` set: one MLA latent row per token, ``k[layer] : [num_pages, 64,
        latent_dim]`` and no separate V (the latent cache holds both).  ``kv_dtype`` "fp8": e4m3
        pages, whose scales are ``scales[layer] : [num_pages, Hkv, 2, 64]``."""
        if kv_dtype not in ("bf16", "fp8"):
            raise ValueError(f"kv_dtype must be 'bf16' or 'fp8', not {kv_dtype!r}")
        if kv_dtype == "fp8" and (latent_dim is not None or head_dim != 128):
            raise ValueError("the e4m3 KV cache holds K and V heads of 128 (no MLA latent rows)")
        self.kv_dtype = kv_dtype
        self.scales = None
        self.num_layers = num_layers
        self.num_kv_heads = num_kv_heads
        self.num_pages = num_pages
        self.head_dim = head_dim
        self.latent_dim = latent_dim
        self.device = torch.device(device)
        if latent_dim is not None:
            self.k = torch.zeros((num_layers, num_pages, PAGE, latent_dim), dtype=dtype,
                                 device=self.device)
            self.v = None
        else:
            shape = (num_layers, num_pages, num_kv_heads, PAGE, head_dim)
            if kv_dtype == "fp8":
                dtype = torch.float8_e4m3fn
                self.scales = torch.zeros((num_layers, num_pages, num_kv_heads, 2, PAGE),
                                          dtype=torch.uint8, device=self.device)
            self.k = torch.zeros(shape, dtype=dtype, device=self.device)
            self.v = torch.zeros(shape, dtype=dtype, device=self.device)
        self.alloc = PageAllocator(num_pages)
        self.seqs: dict[str, SeqPages] = {}

    @staticmethod
    def pages_for(tokens: int) -> int:
        return (tokens + PAGE - 1) // PAGE

    @classmethod
    def bytes_per_page(cls, num_layers: int, num_kv_heads: int, head_dim: int = 128,
                       elem: int = 2, kv_dtype: str = "bf16") -> int:
        token = head_dim + 1 if kv_dtype == "fp8" else head_dim * elem
        return 2 * num_layers * num_kv_heads * PAGE * token

    def layer(self, i: int):
        return self.k[i], (self.v[i] if self.v is not None else None)

    def layer_scales(self, i: int):
        """Scale bytes of layer ``i``, or None for a bf16 cache."""
        return self.scales[i] if self.scales is not None else None

    def rows(self, i: int, seq_id: str, start: int, count: int):
        """K and V of layer ``i`` for tokens ``start .. start + count - 1`` of a sequence as bf16
        [count, Hkv, 128], whatever the cache holds (MLA latent caches have no K and V rows)."""
        if self.latent_dim is not None:
            raise ValueError("an MLA latent cache has no K and V rows")
        if start < 0 or count < 0 or start + count > len(self.seqs[seq_id].pages) * PAGE:
            raise ValueError(f"tokens {start} .. {start + count} are not in the pages of {seq_id}")
        slots = torch.tensor(self.slots(seq_id, start, count), dtype=torch.int32, device=self.device)
        if self.scales is not None:
            from ..ops.attention import read_kv_fp8
            return read_kv_fp8(self.k[i], self.v[i], self.scales[i], slots)
        page, off = slots.long() // PAGE, slots.long() % PAGE
        return self.k[i][page, :, off], self.v[i][page, :, off]

    # ------------------------------------------------------------ sequences
    def open(self, seq_id: str) -> SeqPages:
        if seq_id in self.seqs:
            raise KeyError(f"sequence {seq_id} already open")
        s = SeqPages()
        self.seqs[seq_id] = s
        return s

    def reserve(self, seq_id: str, total_tokens: int) -> SeqPages:
        """Make sure the sequence owns pages for ``total_tokens`` tokens."""
        s = self.seqs[seq_id]
        need = self.pages_for(total_tokens) - len(s.pages)
        if need > 0:
            s.pages.extend(self.alloc.alloc(need))
        return s

    def slots(self, seq_id: str, start: int, count: int) -> list[int]:
        s = self.seqs[seq_id]
        return [s.pages[p // PAGE] * PAGE + p % PAGE for p in range(start, start + count)]

    def close(self, seq_id: str) -> None:
        s = self.seqs.pop(seq_id, None)
        if s is not None:
            self.alloc.release(s.pages)

    def fork(self, src: str, dst: str) -> None:
        """Share all of ``src``'s pages with a new sequence ``dst`` (prefix reuse)."""
        s = self.seqs[src]
        self.alloc.retain(s.pages)
        self.seqs[dst] = SeqPages(pages=list(s.pages), length=s.length)

    def fork_prefix(self, src: str, dst: str, tokens: int) -> SeqPages:
        """Open ``dst`` on the whole pages of the first ``tokens`` tokens of ``src``, shared, not
        copied: appending never writes a full page again, so both sequences may go on
        (:meth:`truncate` copies the page that it makes writable)."""
        s = self.seqs[src]
        if dst in self.seqs:
            raise KeyError(f"sequence {dst} already open")
        if not 0 <= tokens <= s.length:
            raise ValueError(f"{src} holds {s.length} tokens, not {tokens}")
        pages = s.pages[:tokens // PAGE]
        self.alloc.retain(pages)
        self.seqs[dst] = SeqPages(pages=list(pages), length=len(pages) * PAGE)
        return self.seqs[dst]

    def truncate(self, seq_id: str, length: int) -> None:
        """Roll a sequence back to ``length`` tokens, releasing unused whole pages.  A page that is
        kept in part, and that other sequences share, is copied first: the sequence writes its rest
        again (:class:`OutOfPages` if there is none for the copy; nothing has changed then)."""
        s = self.seqs[seq_id]
        keep = self.pages_for(length)
        if length < s.length and length % PAGE and self.alloc.refcount(s.pages[keep - 1]) > 1:
            old, (new,) = s.pages[keep - 1], self.alloc.alloc(1)
            for t in (self.k, self.v, self.scales):
                if t is not None:
                    raw = t.view(torch.uint8)   # (indexing is not defined for every cache type)
                    raw[:, new] = raw[:, old]
            s.pages[keep - 1] = new
            self.alloc.release([old])
        if keep < len(s.pages):
            self.alloc.release(s.pages[keep:])
            del s.pages[keep:]
        s.length = min(s.length, length)

    def snapshot(self, seq_id: str) -> dict:
        """Host copy of the sequence's KV (checkpoint / migration payload)."""
        s = self.seqs[seq_id]
        idx = torch.tensor(s.pages, dtype=torch.long, device=self.device)
        take = ((lambda t: t.view(torch.uint8)[:, idx].view(t.dtype).cpu())
                if self.scales is not None else (lambda t: t[:, idx].cpu()))
        snap = {"length": s.length, "k": take(self.k),
                "v": take(self.v) if self.v is not None else None}
        if self.scales is not None:
            snap["scales"] = self.scales[:, idx].cpu()
        return snap

    def restore(self, seq_id: str, snap: dict) -> None:
        if ("scales" in snap) != (self.scales is not None):
            raise ValueError(f"the snapshot is not of a {self.kv_dtype} cache")
        if seq_id not in self.seqs:
            self.open(seq_id)
        s = self.reserve(seq_id, max(1, int(snap["length"])))
        n = snap["k"].shape[1]
        idx = torch.tensor(s.pages[:n], dtype=torch.long, device=self.device)
        raw = (lambda t: t.view(torch.uint8)) if self.scales is not None else (lambda t: t)
        raw(self.k)[:, idx] = raw(snap["k"]).to(self.device)
        if self.v is not None:
            raw(self.v)[:, idx] = raw(snap["v"]).to(self.device)
        if self.scales is not None:
            self.scales[:, idx] = snap["scales"].to(self.device)
        s.length = int(snap["length"])
