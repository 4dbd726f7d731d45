"""Paged KV arena: device K/V pools plus host-side page accounting.

Layout on the device: one tensor [layers, 2, pages, page_tokens, kv_heads,
head_dim] bf16, so a layer's K or V pool is a contiguous view
[pages, page_tokens, kv_heads, head_dim] (the layout the K4 KV-write and K6
attention kernels take). A B200 holds 180 GB of HBM3e; the arena is sized by
the planner's `arena_pages` from what is left after weights and activations.

Accounting (`PagePool`, pure Python, CPU-testable): a free stack, page lists
per key, and a hold count per page. A key owns the pages it writes. Another
key may read a resident key's first `tokens` tokens as one of its segments
(borrowing: a question reads its document's pages, every row reads the one
copy of the shared instruction prefix); a borrow holds the parent's pages so
they are not freed under the reader. Retained keys stay resident after use
until evicted (KV reuse across operators).

An 8-bit arena (dtype int8 or float8_e4m3fn) holds codes [layers, 2, pages,
kv_heads, page_tokens, head_dim] and, beside them, exponent bytes [layers, 2,
pages, kv_heads, page_tokens / 16]; a layer's K or V is then a `Pages8`
(ops/kv8.py). Twice the tokens fit.

Forking and compacting. `fork` starts a key as a copy of another one's first
tokens: whole pages are shared (each owner holds them), only the page the
tokens end in is copied, so several continuations of one prompt cost a page
each. A key that goes back into shared pages takes its own first (`unshare`).
In an 8-bit arena a token shares its exponent with the 16-token block it is
in: a key forked from, or rewound to, the middle of a block keeps the exponent
that the tokens dropped there had grown (and the mark, if one was not finite).
Where that matters, fork at the parent's end or at a multiple of 16, and give
tokens that will be dropped a key of their own, as the engine's regions do.
`compact` moves the held pages to the lowest page numbers. The accounting is
PagePool's; KVArena's methods of the same names also copy the pages, in every
layer with one launch (ops.kv_copy_pages), ordered on the current stream
behind the passes that read the old places. They are called between passes.

Reference behavior: quail/backends/quail/executor/pages.py (PageArena:
free list, owned/borrowed pages, holds, retention) and arena.py (KVArena).
"""

from __future__ import annotations

from collections import OrderedDict

import numpy as np
import torch


class ArenaFullError(RuntimeError):
    """The arena cannot hold a request even when empty."""


class PagePool:
    """Page accounting; with `state_slots`, also one recurrent-state slot per key.

    Hybrid models (Gated DeltaNet layers) keep a fixed-size state per key
    instead of per-token KV: the state after the key's tokens. A reader of a
    key starts its own state from it, so borrowing holds the parent's slot
    as it holds the parent's pages.
    """

    def __init__(self, num_pages: int, page_tokens: int, state_slots: int = 0):
        self.num_pages = num_pages
        self.page_tokens = page_tokens
        self.state_slots = state_slots
        self.slot_free = list(range(state_slots - 1, -1, -1))
        self.slot_of: dict = {}          # key -> its state slot
        self.slot_holds = np.zeros(max(state_slots, 1), dtype=np.int32)
        self.slot_borrows: dict = {}     # key -> slots of the keys it reads
        self.free = list(range(num_pages - 1, -1, -1))  # stack: pop() gives the lowest id first
        self.owned: dict = {}          # key -> page ids it writes
        self.tokens: dict = {}         # key -> tokens resident
        self.holds = np.zeros(num_pages, dtype=np.int32)
        self.borrows: dict = {}        # key -> page lists it holds of the keys it reads
        self.owners = np.zeros(num_pages, dtype=np.int32)   # keys that own each page (over 1: shared by forks)
        self.retained: OrderedDict = OrderedDict()  # key -> None, oldest first

    # ------------------------------------------------------------ queries
    def pages_needed(self, tokens: int) -> int:
        return -(-tokens // self.page_tokens)

    @property
    def free_pages(self) -> int:
        return len(self.free)

    def resident(self, key) -> bool:
        return key in self.owned

    def pages_of(self, key) -> list[int]:
        return self.owned[key]

    # ------------------------------------------------------------ alloc / grow
    def alloc(self, key, tokens: int, capacity: int = 0):
        """Pages for `tokens` new tokens of a new key (at least `capacity` tokens
        of room, so later growth up to it needs no new pages), or None if the
        pool is short."""
        if key in self.owned:
            raise KeyError(f"{key!r} already resident")
        need = self.pages_needed(max(tokens, capacity))
        if need > len(self.free) or (self.state_slots and not self.slot_free):
            return None
        pages = [self.free.pop() for _ in range(need)]
        if self.state_slots:
            slot = self.slot_free.pop()
            self.slot_of[key] = slot
            self.slot_holds[slot] += 1
            self.slot_borrows[key] = []
        self.owned[key] = pages
        self.tokens[key] = tokens
        self.holds[pages] += 1
        self.owners[pages] += 1
        self.borrows[key] = []
        return pages

    def grow(self, key, tokens: int):
        """Extend a resident key to `tokens` tokens; returns the new pages or None."""
        have = self.owned[key]
        need = -(-tokens // self.page_tokens) - len(have)
        if need <= 0:
            if tokens > self.tokens[key]:
                self.tokens[key] = tokens
            return []
        if need > len(self.free):
            return None
        new = [self.free.pop() for _ in range(max(need, 0))]
        have.extend(new)
        if new:
            self.holds[new] += 1
            self.owners[new] += 1
        self.tokens[key] = max(self.tokens[key], tokens)
        return new

    def borrow(self, reader, parent) -> None:
        """`reader` reads `parent`'s pages: hold them until the reader is freed."""
        if parent not in self.owned:
            raise KeyError(f"borrow parent {parent!r} is not resident")
        pages = list(self.owned[parent])
        self.holds[pages] += 1
        self.borrows.setdefault(reader, []).append(pages)
        if self.state_slots:
            slot = self.slot_of[parent]
            self.slot_holds[slot] += 1
            self.slot_borrows.setdefault(reader, []).append(slot)

    # ------------------------------------------------------------ release
    def _drop(self, pages) -> None:
        if not pages:
            return
        self.holds[pages] -= 1
        for p in pages:
            if self.holds[p] == 0:
                self.free.append(p)

    def _drop_slot(self, slot: int) -> None:
        self.slot_holds[slot] -= 1
        if self.slot_holds[slot] == 0:
            self.slot_free.append(slot)

    def free_key(self, key) -> None:
        """Release a key's own pages and the holds it took on borrowed parents."""
        for pages in self.borrows.pop(key, []):
            self._drop(pages)
        for slot in self.slot_borrows.pop(key, []):
            self._drop_slot(slot)
        if key in self.slot_of:
            self._drop_slot(self.slot_of.pop(key))
        pages = self.owned.pop(key, None)
        self.tokens.pop(key, None)
        self.retained.pop(key, None)
        if pages:
            self.owners[pages] -= 1
            self._drop(pages)

    def rewind(self, key, tokens: int) -> None:
        """Trim a resident key back to its first `tokens` tokens and release the pages past them
        (pages a reader still holds stay held until it is freed)."""
        have = self.owned[key]
        keep = self.pages_needed(tokens)
        if tokens < self.tokens[key] and tokens % self.page_tokens and self.owners[have[keep - 1]] > 1:
            raise ValueError(f"{key!r} shares the page of token {tokens} with a fork: unshare it first")
        if keep < len(have):
            self.owners[have[keep:]] -= 1
            self._drop(have[keep:])
            del have[keep:]
        self.tokens[key] = min(self.tokens[key], tokens)

    def adopt(self, old, new) -> None:
        """Give a resident key's pages, holds and state slot to a new key (no longer retained)."""
        if new in self.owned:
            raise KeyError(f"{new!r} already resident")
        self.owned[new] = self.owned.pop(old)
        self.tokens[new] = self.tokens.pop(old)
        self.borrows[new] = self.borrows.pop(old, [])
        if old in self.slot_of:
            self.slot_of[new] = self.slot_of.pop(old)
            self.slot_borrows[new] = self.slot_borrows.pop(old, [])
        self.retained.pop(old, None)

    # ------------------------------------------------------------ fork / compact
    def fork(self, parent, child, tokens: int | None = None):
        """Make `child` a key whose first `tokens` tokens (default: all) are `parent`'s: whole pages are
        shared, and the page they end in, if partly filled, is a new one. The child also holds what the
        parent borrows. Returns the [(source page, copy)] to copy, or None if the pool is short."""
        if child in self.owned:
            raise KeyError(f"{child!r} already resident")
        tokens = self.tokens[parent] if tokens is None else tokens
        if not 0 <= tokens <= self.tokens[parent]:
            raise ValueError(f"{parent!r} holds {self.tokens[parent]} tokens, not {tokens}")
        if self.state_slots and tokens != self.tokens[parent]:
            raise ValueError("a recurrent state stands at its key's last token: fork there")
        full, part = divmod(tokens, self.page_tokens)
        if (part and not self.free) or (self.state_slots and not self.slot_free):
            return None
        have = self.owned[parent]
        pages = list(have[:full])
        moves = []
        if part:
            pages.append(self.free.pop())
            moves.append((have[full], pages[-1]))
        self.owned[child] = pages
        self.tokens[child] = tokens
        if pages:
            self.holds[pages] += 1
            self.owners[pages] += 1
        self.borrows[child] = [list(b) for b in self.borrows.get(parent, [])]
        for b in self.borrows[child]:
            self.holds[b] += 1
        if self.state_slots:
            slot = self.slot_free.pop()
            self.slot_of[child] = slot
            self.slot_holds[slot] += 1
            self.slot_borrows[child] = list(self.slot_borrows.get(parent, []))
            for held in self.slot_borrows[child]:
                self.slot_holds[held] += 1
        return moves

    def unshare(self, key, tokens: int):
        """Give `key` its own page of token `tokens` and own pages after it, where forks share them, so that
        it may be rewound to `tokens` and written. Returns the [(source page, copy)] to copy, or None if
        the pool is short (nothing is changed then)."""
        if not 0 <= tokens <= self.tokens[key]:
            raise ValueError(f"{key!r} holds {self.tokens[key]} tokens, not {tokens}")
        have = self.owned[key]
        at = tokens // self.page_tokens
        shared = [i for i in range(at, len(have)) if self.owners[have[i]] > 1]
        if len(shared) > len(self.free):
            return None
        moves = []
        for i in shared:
            old, new = have[i], self.free.pop()
            have[i] = new
            self.holds[new] += 1
            self.owners[new] += 1
            self.owners[old] -= 1
            moves.append((old, new))
            self._drop([old])
        return moves

    def compact(self) -> list:
        """Move the held pages to the lowest page numbers: the [(old page, new page)] moves, none of whose
        new pages was held. Every table here names the new pages; pages past the held ones are free."""
        held = np.flatnonzero(self.holds)
        n = held.size
        src = held[held >= n]
        dst = np.flatnonzero(self.holds[:n] == 0)
        if src.size:
            place = np.arange(self.num_pages)
            place[src] = dst
            for pages in self.owned.values():
                pages[:] = place[pages].tolist()
            for lists in self.borrows.values():
                for pages in lists:
                    pages[:] = place[pages].tolist()
            for count in (self.holds, self.owners):
                count[dst] = count[src]
                count[src] = 0
        self.free = list(range(self.num_pages - 1, n - 1, -1))
        return list(zip(src.tolist(), dst.tolist()))

    def retain(self, key) -> None:
        self.retained[key] = None
        self.retained.move_to_end(key)

    def evict_retained(self, pages_needed: int) -> list:
        """Free retained keys, oldest first, until `pages_needed` pages are free."""
        evicted = []
        while self.free_pages < pages_needed and self.retained:
            key, _ = self.retained.popitem(last=False)
            self.free_key(key)
            evicted.append(key)
        return evicted

    def check(self) -> None:
        """Invariant: every page is free xor held; holds match owners and borrows."""
        expect = np.zeros(self.num_pages, dtype=np.int32)
        for pages in self.owned.values():
            expect[pages] += 1
        for held in self.borrows.values():
            for pages in held:
                expect[pages] += 1
        assert np.array_equal(expect, self.holds), "hold counts drifted"
        mine = np.zeros(self.num_pages, dtype=np.int32)
        for pages in self.owned.values():
            mine[pages] += 1
        assert np.array_equal(mine, self.owners), "owner counts drifted"
        free = set(self.free)
        assert len(free) == len(self.free), "page freed twice"
        for p in range(self.num_pages):
            assert (p in free) == (self.holds[p] == 0), f"page {p} free/held mismatch"
        if self.state_slots:
            want = np.zeros(self.state_slots, dtype=np.int32)
            for slot in self.slot_of.values():
                want[slot] += 1
            for slots in self.slot_borrows.values():
                for slot in slots:
                    want[slot] += 1
            assert np.array_equal(want, self.slot_holds[:self.state_slots]), "state slot holds drifted"
            sf = set(self.slot_free)
            assert len(sf) == len(self.slot_free), "state slot freed twice"
            for q in range(self.state_slots):
                assert (q in sf) == (want[q] == 0), f"state slot {q} free/held mismatch"


class KVArena:
    """Device K/V pools with a PagePool."""

    def __init__(self, num_layers: int, num_pages: int, page_tokens: int, kv_heads: int, head_dim: int,
                 device="cuda", dtype=torch.bfloat16, state_slots: int = 0, state_shapes: dict | None = None,
                 layer_geoms: list | None = None):
        self.num_layers = num_layers
        self.page_tokens = page_tokens
        self.kv_heads = kv_heads
        self.head_dim = head_dim
        self.device = torch.device(device)
        # layers of another (KV heads, head_dim) (Gemma 4's global layers) get a pool tensor of
        # their own, addressed by the same page ids
        geoms = list(layer_geoms) if layer_geoms else [(kv_heads, head_dim)] * num_layers
        assert len(geoms) == num_layers
        self._where = []
        count: dict = {}
        for g in geoms:
            self._where.append((g, count.get(g, 0)))
            count[g] = count.get(g, 0) + 1
        self.kv8 = dtype in (torch.int8, torch.float8_e4m3fn)
        self.bytes: dict = {}            # 8-bit arenas: the exponent bytes of each group
        if self.kv8:
            from quail_b200.ops.kv8 import KV8_BLOCK, check_kv8
            for g in count:
                check_kv8(dtype, page_tokens, g[1])
            self.groups = {g: torch.zeros(n, 2, num_pages, g[0], page_tokens, g[1], device=device, dtype=dtype)
                           for g, n in count.items()}
            self.bytes = {g: torch.zeros(n, 2, num_pages, g[0], page_tokens // KV8_BLOCK, device=device,
                                         dtype=torch.uint8) for g, n in count.items()}
        else:
            self.groups = {g: torch.zeros(n, 2, num_pages, page_tokens, g[0], g[1], device=device, dtype=dtype)
                           for g, n in count.items()}
        self.kv = self.groups.get((kv_heads, head_dim), next(iter(self.groups.values())))
        self.pool = PagePool(num_pages, page_tokens, state_slots)
        # recurrent states of hybrid models: name -> [slots, *shape] fp32 (e.g. conv window, delta-rule state)
        self.states = {name: torch.zeros(state_slots, *shape, device=device, dtype=torch.float32)
                       for name, shape in (state_shapes or {}).items()}

    @classmethod
    def for_model(cls, cfg, num_pages: int, page_tokens: int, device="cuda", dtype=torch.bfloat16,
                  state_slots: int = 0) -> "KVArena":
        """KV pages for the model's attention layers; state slots for its Gated DeltaNet layers."""
        shapes = None
        if cfg.is_hybrid:
            shapes = {}
            G = len(cfg.gdn_layers)
            if G:
                shapes["conv"] = (G, cfg.conv_width - 1, cfg.gdn_conv_dim)
                shapes["ssm"] = (G, cfg.gdn_value_heads, cfg.gdn_key_dim, cfg.gdn_value_dim)
            if cfg.conv_layers:
                shapes["sconv"] = (len(cfg.conv_layers), cfg.conv_width - 1, cfg.hidden)
            state_slots = state_slots or 64
        geoms = [cfg.attn_geometry(i) for i in cfg.attn_layers] if getattr(cfg, "gemma4", False) else None
        return cls(len(cfg.attn_layers), num_pages, page_tokens, cfg.num_kv_heads, cfg.head_dim, device=device,
                   dtype=dtype, state_slots=state_slots if cfg.is_hybrid else 0, state_shapes=shapes,
                   layer_geoms=geoms)

    @property
    def num_pages(self) -> int:
        return self.pool.num_pages

    def layer(self, i: int):
        g, j = self._where[i]
        t = self.groups[g]
        if self.kv8:
            from quail_b200.ops.kv8 import Pages8
            b = self.bytes[g]
            return Pages8(t[j, 0], b[j, 0]), Pages8(t[j, 1], b[j, 1])
        return t[j, 0], t[j, 1]

    # ------------------------------------------------------------ fork / compact
    def copy_pages(self, moves) -> None:
        """Copy page contents in every layer: [(from, to)], no page in both columns, none twice in `to`."""
        if not moves:
            return
        src, dst = zip(*moves)
        if len(set(dst)) != len(dst) or set(src) & set(dst):
            raise ValueError("pages are copied to distinct pages that are not themselves copied")
        pools = [*self.groups.values(), *self.bytes.values()]
        ids = torch.tensor([src, dst], dtype=torch.int32, device=self.device)
        if self.device.type == "cuda":
            from quail_b200 import ops
            for i in range(0, len(pools), 8):
                ops.kv_copy_pages(pools[i:i + 8], ids[0], ids[1])
        else:
            for pool in pools:
                raw = pool.view(torch.uint8)
                raw[:, :, ids[1].long()] = raw[:, :, ids[0].long()]

    def fork(self, parent, child, tokens: int | None = None) -> bool:
        """PagePool.fork with its copies made; False if the arena is short of pages or state slots."""
        moves = self.pool.fork(parent, child, tokens)
        if moves is None:
            return False
        self.copy_pages(moves)
        if self.pool.state_slots:
            for t in self.states.values():
                t[self.pool.slot_of[child]] = t[self.pool.slot_of[parent]]
        return True

    def unshare(self, key, tokens: int) -> bool:
        """PagePool.unshare with its copies made; False if the arena is short of pages."""
        moves = self.pool.unshare(key, tokens)
        if moves is None:
            return False
        self.copy_pages(moves)
        return True

    def compact(self) -> int:
        """PagePool.compact with the pages moved; returns how many moved."""
        moves = self.pool.compact()
        self.copy_pages(moves)
        return len(moves)

    @staticmethod
    def bytes_per_page(num_layers, page_tokens, kv_heads, head_dim, elem_bytes=2) -> int:
        return num_layers * 2 * page_tokens * kv_heads * head_dim * elem_bytes
