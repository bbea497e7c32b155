"""Pages shared between sequences: fork, reserve (copy on write), release and compact.

FlashAttnTile's caches give every sequence its own pages (``paging.py:133-169``).
:class:`PagePool` lets rows of one page table hold the same pages -- the samples
of one prompt, beams, conversations behind one system prompt:

    pool = PagePool.allocate(num_pages, batch, max_seq_len, kv_heads, head_dim, page_size)
    pool.reserve(prompt_len, rows=row0)               # pages for the prompt; prefill fills them
    pool.fork(src, dst)                               # rows dst become copies of rows src: no K/V moves
    pool.reserve(1)                                   # every row may append a token: shared tails are copied
    pool.append(new_k, new_v)                         # one token per row
    pool.release(rows)                                # pages that nobody holds any more are free again
    pool.compact()                                    # live pages move to the lowest ids

State beside the cache, all on the device: ``refs`` (table entries that hold
each page; 0: free), ``owned`` (leading entries of each row that hold pages; later
ones are never read, and 0 where a row has given pages back) and ``released`` (1 for a
row from its release until it is forked to or reserved by name: a step over all rows
can leave it out).  Every operation runs on the current stream without host
synchronisation (with value checks on, the checks read the arguments and the
outcome back), so a whole serving step can be captured in a CUDA graph.  Results
are whole numbers that follow from the arguments alone: the lowest free page
ids are taken first, rows are served in the order given.
"""

from __future__ import annotations

import torch

from . import _config, _lib
from .kernels.append import _QUANT
from .kernels.pages import check_rows, check_storage, launch, pool_call, scales_of
from .paging import PagedKVCache, _assert, validate_metadata


def _whole_table(cache: PagedKVCache) -> torch.Tensor:
    """Leading table entries that the lengths reach, as a mask."""
    need = torch.div(cache.seq_lens + (cache.page_size - 1), cache.page_size, rounding_mode="floor")
    cols = torch.arange(cache.max_pages_per_seq, device=cache.page_table.device)
    return cols[None, :] < need[:, None]


class PagePool:
    """A paged cache whose rows may share pages."""

    def __init__(self, cache: PagedKVCache, scales=None, refs: torch.Tensor | None = None,
                 owned: torch.Tensor | None = None):
        """Take over ``cache`` (and the ``scales`` of an 8-bit one).  Without ``refs``
        and ``owned`` the rows own the pages that their lengths reach, and the table
        entries past them are set to 0."""
        validate_metadata(cache)
        k_scale, v_scale = scales_of(scales)
        check_storage("PagePool", cache.k_cache, cache.v_cache, k_scale, v_scale)
        table, lens = cache.page_table, cache.seq_lens
        dev = cache.k_cache.device
        _assert(cache.batch_size > 0 and cache.max_pages_per_seq > 0 and cache.num_pages > 0, "PagePool: empty cache")
        if table.device != dev or lens.device != dev:
            raise ValueError("PagePool: page_table and seq_lens must be on the cache's device")
        if table.stride(1) != 1 or not lens.is_contiguous():
            raise ValueError("PagePool: page_table rows and seq_lens must be contiguous (they are updated in place)")
        if (refs is None) != (owned is None):
            raise ValueError("PagePool: give refs and owned together")
        if refs is None:
            held = _whole_table(cache)
            owned = held.sum(dim=1, dtype=torch.int32)
            table.masked_fill_(~held, 0)
            counted = torch.where(held, table, cache.num_pages).long().clamp_(0, cache.num_pages)
            refs = torch.zeros(cache.num_pages + 1, dtype=torch.int32, device=dev)
            refs.index_add_(0, counted.reshape(-1), torch.ones(counted.numel(), dtype=torch.int32, device=dev))
            refs = refs[:-1].clone()
        for name, t, n in (("refs", refs, cache.num_pages), ("owned", owned, cache.batch_size)):
            if t.dtype != torch.int32 or tuple(t.shape) != (n,) or not t.is_contiguous() or t.device != dev:
                raise ValueError(f"PagePool: {name} must be a contiguous int32 [{n}] tensor on the cache's device")
        self.cache = cache
        self.scales = scales
        self.refs = refs
        self.owned = owned
        self.released = torch.zeros(cache.batch_size, dtype=torch.int32, device=dev)
        self.live: torch.Tensor | None = None
        lib = _lib.load()
        self._scratch = torch.zeros(lib.fat_page_scratch_size(cache.num_pages, cache.batch_size), dtype=torch.uint8,
                                    device=dev)
        self._call = pool_call(cache.k_cache, cache.v_cache, cache.page_size, k_scale, v_scale)
        c = self._call
        c.page_table, c.page_table_stride, c.max_pages = table.data_ptr(), table.stride(0), table.shape[1]
        c.seq_lens, c.owned, c.refs = lens.data_ptr(), owned.data_ptr(), refs.data_ptr()
        c.released = self.released.data_ptr()
        c.scratch, c.scratch_bytes, c.batch = self._scratch.data_ptr(), self._scratch.numel(), cache.batch_size

    @classmethod
    def allocate(cls, num_pages: int, batch: int, max_seq_len: int, num_kv_heads: int, head_dim: int, page_size: int,
                 dtype: torch.dtype = torch.float16, device: torch.device | str = "cuda") -> "PagePool":
        """A pool of ``num_pages`` free pages and ``batch`` empty rows (zeroed storage; unit scales for 8-bit types)."""
        for name, n in (("num_pages", num_pages), ("batch", batch), ("max_seq_len", max_seq_len),
                        ("num_kv_heads", num_kv_heads), ("head_dim", head_dim), ("page_size", page_size)):
            _assert(n > 0, f"{name} must be positive")
        k = torch.zeros((num_pages, page_size, num_kv_heads, head_dim), dtype=dtype, device=device)
        table = torch.zeros((batch, -(-max_seq_len // page_size)), dtype=torch.int32, device=device)
        cache = PagedKVCache(k, torch.zeros_like(k), table, torch.zeros(batch, dtype=torch.int32, device=device),
                             page_size)
        scales = None
        if dtype in _QUANT:
            scales = {n: torch.ones((num_pages, num_kv_heads), dtype=torch.float32, device=device) for n in ("k", "v")}
        return cls(cache, scales=scales)

    # ------------------------------------------------------------------ value checks
    def _check_row_values(self, what: str, *named, distinct: str | None = None) -> None:
        if not _config.validate_values():
            return
        for name, rows in named:
            if rows.numel() == 0:
                continue
            lo, hi = (int(x) for x in torch.stack(torch.aminmax(rows)).tolist())
            _assert(lo >= 0 and hi < self.cache.batch_size,
                    f"{what}: {name} holds a row outside [0, {self.cache.batch_size})")
            if name == distinct:
                _assert(rows.unique().numel() == rows.numel(), f"{what}: {name} holds a row twice")

    def _check_outcome(self, what: str) -> None:
        """With value checks on: read the error word back and raise what the call recorded."""
        if not _config.validate_values():
            return
        bits = _lib.read_device_error(self.cache.k_cache.device)
        if bits & _lib.FAT_DEVERR_NO_PAGE:
            raise RuntimeError(f"{what}: not enough free pages" if what == "reserve"
                               else f"{what}: a page is not held by its row alone (reserve it first)")
        if bits & _lib.FAT_DEVERR_BAD_LENGTH:
            raise RuntimeError(f"{what}: a row exceeds page-table capacity {self.cache.capacity}")
        if bits:
            raise RuntimeError(f"{what}: device error {bits}")

    # ------------------------------------------------------------------ operations
    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Row ``dst[i]`` becomes a copy of row ``src[i]``: its length and the pages
        that length reaches, each held once more.  What ``dst[i]`` held is released.
        All sources are read first, so rows may be both (beams).  ``dst`` is distinct."""
        dev = self.cache.k_cache.device
        src, dst = check_rows("fork", src, dev, "src"), check_rows("fork", dst, dev, "dst")
        if src.numel() != dst.numel():
            raise ValueError(f"fork: src has {src.numel()} rows, dst {dst.numel()}")
        self._check_row_values("fork", ("src", src), ("dst", dst), distinct="dst")
        launch("fat_fork_sequences", self._call, dev, src.data_ptr(), dst.data_ptr(), src.numel())
        self._check_outcome("fork")

    def reserve(self, tokens: int = 1, rows: torch.Tensor | None = None, skip_released: bool = False) -> None:
        """Make room for ``tokens`` more tokens in each row of ``rows`` (all rows by
        default): shared, partly filled tail pages are copied, missing pages taken.

        ``skip_released``, for all rows: those that were released and neither forked to
        nor reserved by name since take nothing."""
        if not isinstance(tokens, int) or tokens < 0:
            raise ValueError(f"reserve: tokens must be a non-negative integer, got {tokens}")
        dev = self.cache.k_cache.device
        n = self.cache.batch_size
        if rows is not None:
            rows = check_rows("reserve", rows, dev, "rows")
            n = rows.numel()
            self._check_row_values("reserve", ("rows", rows), distinct="rows")
        launch("fat_reserve_tokens", self._call, dev, _lib.ptr(rows), n, tokens, skip_released=bool(skip_released))
        self._check_outcome("reserve")

    def release(self, rows: torch.Tensor) -> None:
        """Give the pages of ``rows`` back and empty the rows (marked in ``released``)."""
        dev = self.cache.k_cache.device
        rows = check_rows("release", rows, dev, "rows")
        self._check_row_values("release", ("rows", rows), distinct="rows")
        launch("fat_release_sequences", self._call, dev, rows.data_ptr(), rows.numel())
        self._check_outcome("release")

    def append(self, new_k: torch.Tensor, new_v: torch.Tensor, skip_released: bool = False) -> None:
        """Append one token per row (``paging.append_tokens``; quantised on write for an
        8-bit cache), to pages that a row holds alone: ``reserve`` comes first.
        ``skip_released`` leaves out the rows that ``reserve`` does."""
        c = self.cache
        shape = (c.batch_size, c.num_kv_heads, c.head_dim)
        quant = c.k_cache.dtype in _QUANT
        allowed = (torch.float16, torch.bfloat16, torch.float32) if quant else (c.k_cache.dtype,)
        for name, t in (("new_k", new_k), ("new_v", new_v)):
            _assert(tuple(t.shape) == shape, f"{name} must be [{shape[0]}, {shape[1]}, {shape[2]}], got {tuple(t.shape)}")
            _assert(t.dtype in allowed and t.dtype == new_k.dtype,
                    f"{name} dtype {t.dtype} does not fit a {c.k_cache.dtype} cache")
            _assert(t.device == c.k_cache.device, f"{name} must be on the cache device")
        if new_k.stride() != new_v.stride() or new_k.stride(2) != 1:
            new_k, new_v = new_k.contiguous(), new_v.contiguous()
        launch("fat_append_to_pool", self._call, c.k_cache.device, new_k.data_ptr(), new_v.data_ptr(),
               new_k.stride(0), new_k.stride(1), _lib.DTYPE_CODE[c.k_cache.dtype], _lib.DTYPE_CODE[new_k.dtype],
               skip_released=bool(skip_released))
        self._check_outcome("append")

    def compact(self, in_place: bool = True) -> "PagePool":
        """Move the live pages to ids ``[0, L)``; ``live`` of the result is ``L`` (int32 ``[1]`` on the device).

        In place, table and counts are renamed where they are.  Otherwise the
        result is a new pool with its own table and counts and the same storage,
        lengths and owned counts: this pool's table stays readable (for a step in
        flight) until one of the pages moved from is reused, and is then stale."""
        dev = self.cache.k_cache.device
        new = self
        if not in_place:
            old = self.cache
            new = object.__new__(type(self))
            new.__dict__.update(self.__dict__)
            table = torch.empty(old.page_table.shape, dtype=torch.int32, device=dev)
            new.cache = PagedKVCache(old.k_cache, old.v_cache, table, old.seq_lens, old.page_size)
            new.refs = torch.empty_like(self.refs)
            new._call = type(self._call).from_buffer_copy(self._call)
            new._call.page_table, new._call.refs = table.data_ptr(), new.refs.data_ptr()
            new._call.page_table_stride = table.shape[1]
        live = torch.empty(1, dtype=torch.int32, device=dev) if new.live is None or not in_place else new.live
        launch("fat_compact_pages", self._call, dev, new._call.page_table, new._call.page_table_stride,
               new._call.refs, live.data_ptr())
        new.live = live
        self._check_outcome("compact")
        return new

    def free_pages(self) -> int:
        """Pages that no row holds (reads the counts back)."""
        return int((self.refs <= 0).sum())


__all__ = ["PagePool"]
