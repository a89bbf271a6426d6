"""Paged KV arena on the GPU: per-layer K and V pools in 16-token pages.

The surface the packer and the attention path use, as the reference KVArena
(quail/backends/quail/executor/arena.py:1-24, 35-147, 347-437, 522-563,
644-648, 839-887) defines it for full-attention models: alloc / activate /
alloc_temporary / free_key / pin / retain, residency queries, capacity_rows,
layer_kv / paged_kv and block tables. Sliding-window pools and recurrent
state slots (other model families) are not part of this engine.

HBM layout: one allocation split [k0, v0, k1, v1, ...]; each pool is
(num_pages * page_tokens, num_kv_heads, head_dim) bf16, so page p holds pool
rows p*T .. p*T + T - 1 and a KV row is num_kv_heads * head_dim contiguous
bf16 (2 KiB for Qwen3-4B). At 16 tokens a page is 32 KiB per layer and pool.

With dtype=torch.float8_e4m3fn K and V are kept in 8 bits instead (half the
bytes a token takes and a reader moves): each pool holds e4m3 codes, and
`scales` one E8M0 byte b (2^(b - 127)) for K and one for V per (layer, page,
KV head), (num_layers, num_pages, num_kv_heads, 2).
"""

import warnings
from array import array
from dataclasses import dataclass, replace

import numpy as np
import torch

from quail_amd import _lib
from quail_amd.pages import PageArena

FP8 = torch.float8_e4m3fn


class _Claim:
    """What keeps a key's pages in the arena: queued borrowers that will
    read them (holds), admissions reading them now (reads), and whether a
    free was asked for meanwhile (done when the last claim goes)."""

    __slots__ = ("holds", "reads", "free_asked")

    def __init__(self):
        self.holds = 0
        self.reads = 0
        self.free_asked = False


@dataclass(frozen=True)
class _Thinned:
    """A key whose rows are no longer its first tokens: its id in the accounting
    (a key of the same name that comes later has another), the rows it held
    after the last thinning, the tokens dropped until then, and the number of
    the token that each of those rows holds, int32 (layers, KV heads, rows) or
    None where they were not kept."""

    ident: int
    held: int
    dropped: int
    numbers: torch.Tensor | None


class KVArena:
    def __init__(self, num_layers: int, num_pages: int, page_tokens: int, num_kv_heads: int,
                 d_head: int, dtype=torch.bfloat16, device="cuda", v_dtype=None):
        if v_dtype is None:
            v_dtype = FP8 if dtype == FP8 else torch.float16
        if dtype == FP8:
            if v_dtype != FP8:
                raise ValueError("8-bit pages hold K and V in e4m3")
            if page_tokens != 16 or d_head not in (64, 128):
                raise ValueError(f"8-bit pages have 16 rows of head_dim 64 or 128, not "
                                 f"{page_tokens} of {d_head}")
        elif dtype != torch.bfloat16 or v_dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("K pages are bf16; V pages bf16 or fp16")
        self.torch = torch
        self.dtype = dtype
        # whether K and V are e4m3 codes with a scale per (page, KV head)
        self.eight_bit = dtype == FP8
        self.v_dtype = v_dtype
        self.device = device
        self.num_layers = num_layers
        self.kv_shape = (num_kv_heads, d_head)
        self.sliding_layers = frozenset()
        self.has_sliding = False
        self.num_state_slots = 0
        self._build(num_pages, page_tokens)
        self.evicted_keys = 0
        self.evicted_pages = 0
        self.evicted_prefix_tokens = 0

    def _build(self, num_pages, page_tokens):
        heads, dim = self.kv_shape
        self.accounting = PageArena(num_pages, page_tokens)
        rows = num_pages * page_tokens
        size = rows * heads * dim
        storage = torch.empty(2 * self.num_layers * size, dtype=self.dtype, device=self.device)
        parts = storage.split([size] * (2 * self.num_layers))
        self.k = [p.view(rows, heads, dim) for p in parts[0::2]]
        # V pages: bf16 as the reference's arena holds them, or fp16 (the
        # default here: the same 16-bit slots; bf16 V rows are converted once,
        # when written, and the PV product then keeps 11 bits of each
        # probability instead of 8)
        self.v = [p.view(self.v_dtype).view(rows, heads, dim) for p in parts[1::2]]
        self.storage = storage
        self.scales = None
        if self.eight_bit:
            self.scales = torch.full((self.num_layers, num_pages, heads, 2), 127,
                                     dtype=torch.uint8, device=self.device)
            self._layer_scales = list(self.scales.unbind(0))
            self._pointers = [(k.data_ptr(), v.data_ptr(), s.data_ptr())
                              for k, v, s in zip(self.k, self.v, self._layer_scales)]
        self._claims = {}
        self._thinned = {}      # key -> _Thinned

    # ---- sizes -------------------------------------------------------------

    @property
    def page_tokens(self) -> int:
        return self.accounting.page_tokens

    @property
    def num_pages(self) -> int:
        return self.accounting.num_pages

    @property
    def free_pages(self) -> int:
        return self.accounting.free_pages

    @property
    def retained_pages(self) -> int:
        return self.accounting.retained_pages

    def pages_needed(self, tokens: int) -> int:
        return self.accounting.pages_needed(tokens)

    def page_cost(self, tokens: int, sliding_tokens: int = 0) -> int:
        return self.accounting.pages_needed(tokens)

    # ---- residency ---------------------------------------------------------

    def is_resident(self, key) -> bool:
        return self.accounting.is_resident(key)

    def resident_keys(self):
        return self.accounting.resident_keys()

    def owned_pages(self, key) -> list:
        """The page ids the key's block table reads: borrowed, then its own."""
        return self.accounting.table_pages(key)

    def tokens(self, key) -> int:
        return self.accounting.key_tokens(key)

    def capacity_rows(self, key) -> np.ndarray:
        """Pool row of every row in the key's pages, in logical order (host int64)."""
        pages = np.asarray(self.accounting.table_pages(key), dtype=np.int64)
        t = self.page_tokens
        return (pages[:, None] * t + np.arange(t, dtype=np.int64)).reshape(-1)

    # ---- allocation ----------------------------------------------------------

    def _borrow_plan(self, borrow):
        if borrow is None:
            return []
        parent, shared = borrow
        self.check_whole(parent)
        return self.accounting.shared_pages(parent, shared)

    def can_borrow(self, parent, shared: int) -> bool:
        acct = self.accounting
        return (acct.is_resident(parent) and not self.is_thinned(parent)
                and shared <= acct.key_tokens(parent))

    def alloc(self, key, tokens: int, capacity_tokens=None, base_tokens=None, borrow=None):
        """Pages for a fresh key, or None when the free list is short.
        borrow = (parent key, shared tokens): the key reads the parent's
        first pages as its own leading pages."""
        return self.accounting.alloc(key, tokens, capacity_tokens,
                                     borrowed=self._borrow_plan(borrow))

    def _evict_until(self, satisfied) -> tuple:
        """Free retained keys in the accounting's victim order until
        satisfied() holds (arena.py:478-492); a key a queued borrower will
        read (held) or that an admission is reading is never a victim.
        Returns the evicted keys."""
        acct = self.accounting
        keep = frozenset(self._claims)
        keys = []
        while not satisfied():
            victim = acct.pop_retained_victim(keep=keep)
            if victim is None:
                break
            key, _, tokens = victim
            self.evicted_keys += 1
            self.evicted_prefix_tokens += tokens
            self.evicted_pages += self.free_key(key)
            keys.append(key)
        return tuple(keys)

    def _evict_for_pages(self, need: int) -> None:
        self._evict_until(lambda: self.accounting.free_pages >= need)

    def evict_retained(self, pages_needed: int) -> tuple:
        """Free retained keys until pages_needed pages have come free
        (arena.py:468-476). Returns the evicted keys."""
        start = self.accounting.free_pages
        return self._evict_until(lambda: self.accounting.free_pages - start >= pages_needed)

    def reserve(self, key, tokens: int, *, capacity_tokens: int, borrow=None,
                extension=False, share_points=()) -> bool:
        """Pages for an admitted document (arena.py:584-642): retained KV is
        evicted until its capacity fits, never the document's own pages or
        the parent it borrows from; then it is activated (pinned). False
        leaves it as it was (evictions may have happened)."""
        acct = self.accounting
        self.check_whole(key)
        if acct.is_resident(key):
            held = len(acct.table_pages(key))
        else:
            held = len(self._borrow_plan(borrow))
        need = max(0, acct.pages_needed(capacity_tokens) - held)
        protected = (key,) if borrow is None else (key, borrow[0])
        self.read_state(protected)
        try:
            self._evict_until(lambda: acct.free_pages >= need)
            if acct.free_pages < need:
                return False
            return self.activate(key, tokens, capacity_tokens=capacity_tokens,
                                 borrow=borrow) is not None
        finally:
            self.done_reading(protected)

    def activate(self, key, tokens: int, capacity_tokens=None, base_tokens=None, borrow=None):
        """Make a prefix active (pinned), evicting retained KV when needed."""
        acct = self.accounting
        self.check_whole(key)
        capacity = tokens if capacity_tokens is None else capacity_tokens
        if acct.is_resident(key):
            acct.pin(key)
            need = max(0, acct.pages_needed(capacity) - len(acct.table_pages(key)))
            self._evict_for_pages(need)
            if need > acct.free_pages:
                return None
            acct.grow(key, capacity)
            acct.set_tokens(key, tokens)
            return acct.owned_pages(key)
        borrowed = self._borrow_plan(borrow)
        self._evict_for_pages(acct.pages_needed(capacity) - len(borrowed))
        pages = self.alloc(key, tokens, capacity, base_tokens, borrow=borrow)
        if pages is not None:
            acct.pin(key)
        return pages

    def alloc_temporary(self, tokens: int, sliding_tokens=None):
        key = object()
        pages = self.alloc(key, tokens, base_tokens=0)
        return None if pages is None else (key, pages)

    # ---- copies, forks and compaction ----------------------------------------------

    def copy_pages(self, src, dst) -> None:
        """Pages src[i] -> dst[i] in every layer, K and V (and their scales),
        on the current stream. Page ids are host values; each destination is
        named once and is no source (ValueError otherwise)."""
        src, dst = list(src), list(dst)
        if len(src) != len(dst):
            raise ValueError(f"{len(src)} source pages for {len(dst)} destinations")
        if not self.storage.is_cuda:
            raise ValueError("page copies run on the GPU; this arena is on the CPU")
        try:
            src, dst = array("i", src), array("i", dst)
        except OverflowError as err:
            raise ValueError(f"page ids of {self.num_pages} pages: {err}") from err
        device = self.storage.device.index
        if device != torch.cuda.current_device():
            with torch.cuda.device(device):
                self._copy_pages(src, dst)
        else:
            self._copy_pages(src, dst)

    def _copy_pages(self, src, dst):
        from quail_amd.engine import _stream
        heads, dim = self.kv_shape
        page = self.page_tokens * heads * dim * self.storage.element_size()
        scales = (None, 0, 0, 0)
        if self.eight_bit:
            scales = (self.scales.data_ptr(), self.num_layers, 2 * heads * self.num_pages, 2 * heads)
        try:
            _lib.call("qx_copy_pages", self.storage.data_ptr(), 2 * self.num_layers,
                      self.num_pages * page, page, *scales, src.buffer_info()[0],
                      dst.buffer_info()[0], len(src), self.num_pages, _stream())
        except _lib.QxError as err:
            if "hipError" in str(err):
                raise
            raise ValueError(str(err)) from err

    def fork(self, key, children, tokens=None, capacity_tokens=None):
        """New keys that continue the first `tokens` tokens of a resident key
        (all of them by default), each in pages of its own from there: they
        read the key's full pages as borrowed ones, and its partial last page
        is copied (current stream) into the first page of each. Returns the
        children's own pages, or None with nothing changed when the free list
        is short (evict retained keys first)."""
        acct = self.accounting
        children = list(children)
        if len(set(children)) != len(children):
            raise ValueError("a fork names each child once")
        held = acct.key_tokens(key)
        tokens = held if tokens is None else tokens
        capacity = tokens if capacity_tokens is None else capacity_tokens
        if not 0 <= tokens <= held:
            raise ValueError(f"fork of {tokens} tokens from a key that holds {held}")
        if tokens != held:
            self.check_whole(key)
        if capacity < tokens:
            raise ValueError(f"capacity of {capacity} tokens for a fork of {tokens}")
        for child in children:
            if acct.is_resident(child):
                raise KeyError(f"{child!r} already resident")
        full, rest = divmod(tokens, self.page_tokens)
        shared = acct.shared_pages(key, full * self.page_tokens)
        table = acct.table_pages(key)
        if len(shared) != full or len(table) < acct.pages_needed(tokens):
            raise ValueError("the key's leading pages were dropped")
        if rest and children and not self.storage.is_cuda:
            raise ValueError("page copies run on the GPU; this arena is on the CPU")
        need = acct.pages_needed(capacity) - full
        if need * len(children) > acct.free_pages:
            return None
        pages = [acct.alloc(child, tokens, capacity, borrowed=shared) for child in children]
        if rest and children:
            self.copy_pages([table[full]] * len(children), [own[0] for own in pages])
        if self.is_thinned(key):
            self._thinned.update((child, replace(self._thinned[key], ident=acct.key_id(child)))
                                 for child in children)
        return pages

    def compact(self) -> int:
        """Move the resident keys' pages to the lowest ids (current stream),
        so that the pages past them are free in one run; returns the pages
        moved. Between stages only: ValueError while a key is pinned, held or
        being read, or a pack's temporary pages live."""
        if self._claims:
            raise ValueError("keys are held for borrowers or being read")
        if not self.storage.is_cuda:
            raise ValueError("page copies run on the GPU; this arena is on the CPU")
        src, dst = self.accounting.compact()
        if src:
            self.copy_pages(src, dst)
        return len(src)

    def free_key(self, key) -> int:
        """Free a key's pages, or once its holds and reads are over (a key
        queued borrowers will read, or that an admission reads, waits for
        them). Returns the pages that went free now."""
        claim = self._claims.get(key)
        if claim is not None:
            claim.free_asked = True
            return 0
        return self._free(key)

    def _free(self, key) -> int:
        freed = self.accounting.free_key(key)
        self._thinned.pop(key, None)
        return freed

    def pin(self, key) -> None:
        self.accounting.pin(key)

    def retain(self, key, tokens=None, priority=None) -> None:
        """Keep a key's first `tokens` (all of them by default) for a later
        operator; it becomes evictable."""
        if tokens is not None:
            if tokens != self.accounting.key_tokens(key):
                self.check_whole(key)
            self.accounting.rewind(key, tokens)
        self.accounting.retain(key, priority)

    # ---- thinning ------------------------------------------------------------------

    def thin_rows(self, tables, weights, keep, *, sinks=0, recent=0, newest=None, tokens=None):
        """Keep the heaviest rows of sequences that a caller lays out: of every
        (layer, sequence, KV head) the first `sinks` rows, the last `recent`
        and the heaviest of the others by `weights`, min(used, keep) in all
        (ties: the first; a NaN is heavier than every number). Kept rows below
        `keep` stay where they are, the j-th dropped place takes the j-th kept
        row past them (current stream), and rows from `keep` on stay as they
        were: the caller reads min(used, keep) rows afterwards. Keys keep the
        rotation they were written with.

        `sinks` and `recent` count places. A kept row that moves leaves the
        tokens' order, so of a sequence that was thinned before the last
        `recent` rows are its newest tokens only if it grew by as many since.
        Sequences that are thinned over and over take `newest` and `tokens`
        instead of `recent`: then the tokens numbered below `sinks` and the
        last `newest` ones stay, as far as they are held, wherever their rows
        lie. tokens: int32 in the shape of `weights`, the number of the token
        that each row holds (from 0, no two rows of a head alike), negative for
        rows appended since the last call, which hold the last tokens in order
        (at first every row is one); tables["tokens"], int32, one per sequence:
        the tokens it has had so far, dropped ones among them.

        tables: used (int32, one per sequence), table (int32 rows of pages) and
        max_used, a bound of used, as a plan or read_pages' tables have them;
        no page is in two sequences. weights: fp32 (layers, sequences, KV heads,
        columns), as Engine.key_weights gathers them. 8-bit pages are kept whole:
        `keep` is then a multiple of their 16 rows.

        Returns (kept, weights): int32 (layers, sequences, KV heads, min(keep,
        columns)), the row that each slot holds as it was numbered before, -1
        past min(used, keep); and the slots' weights in the shape of `weights`,
        0 past them. With `tokens` also the slots' numbers in that shape, -1
        past them: the next call's `tokens`."""
        from quail_amd.engine import _launch
        used, table = tables["used"], tables["table"]
        heads, dim = self.kv_shape
        for name, t, dims in (("used", used, 1), ("table", table, 2)):
            if t.dtype != torch.int32 or t.dim() != dims or t.stride(-1) != 1:
                raise ValueError(f"{name}: int32 of {dims} dimension(s), rows contiguous")
        seqs, max_used = used.shape[0], int(tables["max_used"])
        if weights.dtype != torch.float32 or weights.dim() != 4 or \
                weights.shape[:3] != (self.num_layers, seqs, heads) or \
                (weights.shape[3] > 1 and weights.stride(3) != 1):
            raise ValueError(f"weights: fp32 ({self.num_layers} layers, {seqs} sequences, {heads} heads, "
                             f"columns), columns contiguous, not {tuple(weights.shape)} "
                             f"{weights.dtype}")
        cols = weights.shape[3]
        if table.shape[0] < seqs or max_used > table.shape[1] * self.page_tokens:
            raise ValueError(f"{seqs} sequences of up to {max_used} rows in a table of "
                             f"{table.shape[0]} times {table.shape[1]} pages")
        if max_used > cols:
            raise ValueError(f"{cols} columns of weights for up to {max_used} rows")
        if tables.get("pages", 0) > self.num_pages:
            raise ValueError(f"page {tables['pages'] - 1} in the plan's table, {self.num_pages} in the "
                             "arena")
        by_token = newest is not None
        if by_token != (tokens is not None) or (by_token and recent):
            raise ValueError("newest goes with the rows' tokens, and not with recent")
        last = newest if by_token else recent
        if keep < 0 or sinks < 0 or last < 0 or sinks + last > keep:
            raise ValueError(f"{sinks} first and {last} last rows of {keep} that stay")
        if by_token:
            if tokens.dtype != torch.int32 or tokens.shape != weights.shape or (cols > 1 and tokens.stride(3) != 1):
                raise ValueError(f"tokens: int32 {tuple(weights.shape)}, columns contiguous, not "
                                 f"{tuple(tokens.shape)} {tokens.dtype}")
            total = tables.get("tokens")
            if not torch.is_tensor(total) or total.dtype != torch.int32 or total.shape != (seqs,) or \
                    (seqs > 1 and total.stride(0) != 1):
                raise ValueError(f"the tables' tokens: int32, one for each of {seqs} sequences")
        if self.eight_bit and keep % self.page_tokens:
            raise ValueError(f"8-bit pages are kept whole: {keep} rows are not a multiple of "
                             f"{self.page_tokens}")
        device = self.storage.get_device()
        if device < 0:
            raise ValueError("rows are thinned on the GPU; this arena is on the CPU")
        if not used.get_device() == table.get_device() == weights.get_device() == device or \
                by_token and not tokens.get_device() == total.get_device() == device:
            raise ValueError(f"tables and weights on the arena's GPU {device}")
        shape = (self.num_layers, seqs, heads)
        kept = torch.empty(*shape, min(keep, cols), dtype=torch.int32, device=weights.device)
        out = torch.empty_like(weights, memory_format=torch.contiguous_format)
        scales = (None, 0) if self.scales is None else (self.scales.data_ptr(), self.scales.stride(0))
        pool = self.num_pages * self.page_tokens * heads * dim * self.storage.element_size()
        pages = (self.storage.data_ptr(), pool, self.storage.element_size(), *scales,
                 weights.data_ptr(), *weights.stride()[:3])
        rows = (used.data_ptr(), table.data_ptr(), table.stride(0), *shape, dim, self.page_tokens,
                max_used, cols, keep, sinks, last, kept.data_ptr(), out.data_ptr())
        try:
            if by_token:
                left = torch.empty_like(out, dtype=torch.int32)
                _launch(device, "qx_thin_rows_by_token", *pages, tokens.data_ptr(), *tokens.stride()[:3],
                        total.data_ptr(), *rows, left.data_ptr())
                return kept, out, left
            _launch(device, "qx_thin_rows", *pages, *rows)
        except _lib.QxError as err:
            if "hipError" in str(err):
                raise
            raise ValueError(str(err)) from err
        return kept, out

    def thin(self, keys, weights, keep, *, sinks=0, recent=0, newest=None):
        """thin_rows of resident keys, whose pages past `keep` rows go free.
        `weights` has a row per key, in the keys' order. A thinned key's rows
        are no longer its first tokens: it is read and continued by a caller
        (read_pages, append_rows, fork of all it holds), not lent, packed or
        activated again. ValueError where a key lends or borrows pages, is held
        or is being read, is retained (pin it first: an eviction may take it, and
        fewer tokens would be retained with another priority) or is named twice.

        A key that is thinned again as it grows takes `newest`, from the first
        time on: its first `sinks` and last `newest` tokens stay wherever their
        rows lie (the arena keeps the tokens' numbers). `recent` protects the
        last places, whose rows are its newest tokens only where it grew by as
        many since it was thinned: RuntimeWarning where it did not. ValueError
        for `newest` of a key that was thinned without.

        Returns (kept, weights) as thin_rows does."""
        acct = self.accounting
        keys = list(keys)
        if len(set(keys)) != len(keys):
            raise ValueError("a key is thinned once")
        pages = set()
        for key in keys:
            if key in self._claims:
                raise ValueError(f"{key!r} is held for borrowers or being read")
            if acct.is_retained(key):
                raise ValueError(f"{key!r} is retained, so that an eviction may take it: pin it first")
            if acct.borrowed_pages(key):
                raise ValueError(f"{key!r} borrows pages")
            pages.update(acct.owned_pages(key))
        for other in acct.resident_keys():
            if not pages.isdisjoint(acct.borrowed_pages(other)):
                raise ValueError(f"{other!r} borrows pages of the keys")
        found = [self._thinned[key] if self.is_thinned(key) else None for key in keys]
        if newest is not None and any(f is not None and f.numbers is None for f in found):
            raise ValueError("a key was thinned without newest: the tokens that its rows hold are not known")
        if keys:
            table, used = self.block_table(keys)
        else:
            table, used = np.zeros((0, 0), dtype=np.int32), np.zeros(0, dtype=np.int32)
        if any(len(acct.table_pages(key)) < acct.pages_needed(n) for key, n in zip(keys, used.tolist())):
            raise ValueError("a key's leading pages were dropped")
        device = self.storage.device if keys else weights.device
        tables = dict(used=torch.from_numpy(used).to(device), table=torch.from_numpy(table).to(device),
                      max_used=max([0, *used.tolist()]))
        by_token = {}
        if newest is None:
            for key, n, f in zip(keys, used.tolist(), found):
                if f is not None and keep < n < f.held + recent:
                    warnings.warn(f"{key!r} grew by {n - f.held} rows since it was thinned: its last {recent} "
                                  "places are not its newest tokens (newest protects those)",
                                  RuntimeWarning, stacklevel=2)
        else:
            total = [n + (0 if f is None else f.dropped) for n, f in zip(used.tolist(), found)]
            tables["tokens"] = torch.tensor(total, dtype=torch.int32).to(device)
            cols = max([*weights.shape[-1:], tables["max_used"]])
            tokens = torch.full((self.num_layers, len(keys), self.kv_shape[0], cols), -1, dtype=torch.int32,
                                device=device)
            for s, f in enumerate(found):
                if f is not None:
                    tokens[:, s, :, :f.held] = f.numbers
                    if f.numbers.is_cuda:      # made on the stream of the thinning before
                        f.numbers.record_stream(torch.cuda.current_stream(f.numbers.device))
            by_token = dict(newest=newest, tokens=tokens)
        result = self.thin_rows(tables, weights, keep, sinks=sinks, recent=recent, **by_token)
        for s, (key, n, f) in enumerate(zip(keys, used.tolist(), found)):
            if n > keep:
                acct.rewind(key, keep)
                numbers = None if newest is None else result[2][:, s, :, :keep].clone()
                self._thinned[key] = _Thinned(acct.key_id(key), keep, n - keep + (0 if f is None else f.dropped),
                                              numbers)
        return result if newest is None else result[:2]

    def append_rows(self, key, count: int):
        """Room for `count` more rows of a resident key: their pool rows (host
        int64), or None with nothing changed when the free list is short.
        ValueError where one of them lies in a page that another key reads (a
        key that was rewound into a page it had lent, or holds fewer tokens
        than it borrows): a fork of it has that page of its own. ValueError for
        a retained key, which an eviction may take with the rows just handed
        out: pin it first."""
        acct = self.accounting
        tokens = acct.key_tokens(key)
        if count < 0:
            raise ValueError(f"{count} more rows")
        if len(acct.table_pages(key)) < acct.pages_needed(tokens):
            raise ValueError(f"{key!r}: leading pages were dropped")
        if acct.is_retained(key):
            raise ValueError(f"{key!r} is retained, so that an eviction may take it: pin it first")
        if count and acct.holders(key, tokens // self.page_tokens, acct.pages_needed(tokens + count)) > 1:
            raise ValueError(f"{key!r}: another key reads the page of row {tokens} or one after it")
        if acct.grow(key, tokens + count) is None:
            return None
        acct.set_tokens(key, tokens + count)
        return self.capacity_rows(key)[tokens:tokens + count]

    def is_thinned(self, key) -> bool:
        """Whether a resident key's rows are no longer its first tokens."""
        found = self._thinned.get(key)
        return found is not None and self.is_resident(key) and self.accounting.key_id(key) == found.ident

    def check_whole(self, key) -> None:
        """ValueError for a thinned key."""
        if self._thinned and self.is_thinned(key):
            raise ValueError(f"{key!r} was thinned: its rows are not its first tokens")

    # ---- holds and reads: keys that admitted or queued readers need -------------

    def _claim(self, key) -> "_Claim":
        claim = self._claims.get(key)
        if claim is None:
            claim = self._claims[key] = _Claim()
        return claim

    def _settle(self, key) -> None:
        """Forget a key's claim once nothing keeps it; free its pages then
        if a free was asked for while it was kept."""
        claim = self._claims[key]
        if claim.holds or claim.reads:
            return
        del self._claims[key]
        if claim.free_asked:
            self._free(key)

    def hold(self, key, borrowers: int) -> None:
        """Keep a key for `borrowers` documents that will read its pages."""
        if borrowers:
            self._claim(key).holds += borrowers

    def release(self, key) -> None:
        """One borrower of the key was admitted, or will not come."""
        claim = self._claims.get(key)
        if claim is not None and claim.holds:
            claim.holds -= 1
            self._settle(key)

    def drop_holds(self, keys=None) -> bool:
        """Release every hold on the keys (all by default): freed keys go
        free, retained ones become evictable. True when any hold went."""
        pool = self._claims if keys is None else keys
        held = [k for k in pool if k in self._claims and self._claims[k].holds]
        for key in held:
            self._claims[key].holds = 0
            self._settle(key)
        return bool(held)

    def read_state(self, keys) -> None:
        """Keep each key's pages until done_reading for the same keys."""
        for key in keys:
            self._claim(key).reads += 1

    def done_reading(self, keys) -> None:
        for key in keys:
            self._claims[key].reads -= 1
            self._settle(key)

    def origin(self, tokens: int) -> int:
        """The first row a key's pages must hold for a borrower of `tokens`
        rows: 0 (every layer keeps every row; no sliding window)."""
        return 0

    def keep_window(self, key, shared: int) -> None:
        """No sliding window: every row a borrower reads stays."""

    # ---- tensors read by attention ---------------------------------------------

    def layer_kv(self, layer: int):
        """Flat K and V pools of one layer: (rows, num_kv_heads, head_dim)."""
        return self.k[layer], self.v[layer]

    def layer_scales(self, layer: int):
        """The E8M0 bytes of one layer of an 8-bit arena: (num_pages,
        num_kv_heads, 2), K's and V's."""
        return self._layer_scales[layer]

    def layer_pointers(self, layer: int):
        """The addresses of a layer's K codes, V codes and scales (8 bits)."""
        return self._pointers[layer]

    def paged_kv(self, layer: int):
        heads, dim = self.kv_shape
        shape = (-1, self.page_tokens, heads, dim)
        return self.k[layer].view(shape), self.v[layer].view(shape)

    def block_table_rows(self, pages, pad_to=None) -> np.ndarray:
        """(len(pages), width) int32 table, each row zero-padded on the right."""
        width = max(len(p) for p in pages)
        if pad_to:
            width = max(width, pad_to)
        table = np.zeros((len(pages), width), dtype=np.int32)
        for row, p in enumerate(pages):
            table[row, :len(p)] = p
        return table

    def block_table(self, keys, pad_to=None):
        table = self.block_table_rows([self.owned_pages(k) for k in keys], pad_to)
        used = np.asarray([self.accounting.key_tokens(k) for k in keys], dtype=np.int32)
        return table, used
