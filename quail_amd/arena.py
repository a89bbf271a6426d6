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

from array import array

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
        return self.accounting.shared_pages(parent, shared)

    def can_borrow(self, parent, shared: int) -> bool:
        acct = self.accounting
        return acct.is_resident(parent) and shared <= acct.key_tokens(parent)

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
        return self.accounting.free_key(key)

    def pin(self, key) -> None:
        self.accounting.pin(key)

    def retain(self, key, tokens=None, priority=None) -> None:
        """Keep a key's first `tokens` (all of them by default) for a later
        operator; it becomes evictable."""
        if tokens is not None:
            self.accounting.rewind(key, tokens)
        self.accounting.retain(key, priority)

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
            self.accounting.free_key(key)

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
