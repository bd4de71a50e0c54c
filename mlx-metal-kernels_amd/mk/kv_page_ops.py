"""Pages of a paged KV cache as sequences come, branch and go: copied, forked,
freed and compacted, for all layers at once.  The reference has no
counterpart: its block tables are fixed (ops/paged_kv_ops.py:99-115).

``pages`` is a list of page arrays that share page ids: K and V pages
[NUM_PAGES, PAGE_SIZE, ...] of every layer, fp16 / bf16 values or the codes
and scales of a quantized cache.  They are changed in place; tables, lengths
and counts come back as new tensors.

``ref_counts`` int32 [NUM_PAGES] counts the references to each page: those of
the block table (``count_page_refs``) and of whoever else holds pages (another
table, a cache of prefixes).  A page whose count is 0 is free.  Everything
stays on the device, and pages are taken by ascending id for rows in order, so
a step whose parents a device computes (beams, samples) needs no host, and
equal inputs give equal tables.
"""

from __future__ import annotations

from array import array

import torch

from . import _lib
from ._common import ci_safe_mode_enabled, narrow_i32
from .kv_cache_ops import host_checks_enabled

MAX_ROWS = 4096  # rows of a forked table
_SHAPE, _NBYTES = torch.Tensor.shape.__get__, torch.Tensor.nbytes.__get__  # (as functions of a tensor)


def _backend(backend: str) -> bool:
    """Whether the tensor-op path is asked for."""
    name = backend.lower()
    if name not in ("auto", "reference", "metal"):
        raise ValueError("backend must be one of 'reference', 'metal', 'auto'")
    return ci_safe_mode_enabled() or name == "reference"


def _check_pages(pages, num_pages, device):
    """Dense arrays of ``num_pages`` pages (None: those of the first), of one page size, on one device."""
    size = None
    # the shapes that there are, once each: a cache of many layers has one or two
    for shape in set(map(_SHAPE, pages)):
        if len(shape) < 2:
            raise ValueError(f"page arrays must be [NUM_PAGES,PAGE_SIZE,...], got {tuple(shape)}")
        if num_pages is None:
            num_pages = shape[0]
        if size is None:
            size = shape[1]
        if shape[0] != num_pages or shape[1] != size:
            raise ValueError(f"page arrays must share NUM_PAGES={num_pages} and PAGE_SIZE={size}, got {tuple(shape)}")
    if not all(map(torch.Tensor.is_contiguous, pages)):
        raise ValueError("page arrays must be contiguous for the in-place move")
    for d in set(map(torch.Tensor.get_device, pages)):  # -1: the host
        if d != (-1 if device.type == "cpu" else device.index):
            raise ValueError(f"tensors are on different devices: {device} and others")
    return num_pages, size


def _addresses(pages, num_pages):
    """Host arrays of the addresses and of the bytes a page, as the library takes them."""
    return (array("Q", map(torch.Tensor.data_ptr, pages)),
            array("q", [n // num_pages for n in map(_NBYTES, pages)]))


def _ids(t, device, name):
    if not isinstance(t, torch.Tensor):
        t = torch.as_tensor(t, dtype=torch.int32)
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
    return narrow_i32(t, device)


def count_page_refs(block_table, num_pages: int):
    """int32 [num_pages]: how often the table names each page (entries outside of the pages count nowhere)."""
    t = block_table.reshape(-1).long()
    ok = (t >= 0) & (t < num_pages)
    counts = torch.zeros(num_pages, dtype=torch.int32, device=block_table.device)
    return counts.index_add_(0, torch.where(ok, t, 0), ok.to(torch.int32)) if num_pages else counts


# ----------------------------------------------------------------- copy


def copy_kv_pages(pages, src, dst, *, backend: str = "auto"):
    """Page src[i] onto page dst[i] in every array of ``pages``, in place;
    returns ``pages``.  src, dst int32 [n] (device, host or a list).  No
    page may be the destination of two pairs, or the source of one and the
    destination of another.  Entries are checked on the host unless that is off
    (``host_checks_enabled``); then pairs with an entry outside of the pages are
    skipped."""
    reference = _backend(backend)
    if len(pages) == 0:
        raise ValueError("no page arrays given")
    dev = pages[0].device
    num_pages, _ = _check_pages(pages, None, dev)
    src, dst = _ids(src, dev, "src"), _ids(dst, dev, "dst")
    if src.dim() != 1 or src.shape != dst.shape:
        raise ValueError(f"src and dst must be [n], got {tuple(src.shape)}, {tuple(dst.shape)}")
    n = src.shape[0]
    if n and host_checks_enabled(src):
        s, d = src.cpu(), dst.cpu()
        both = torch.cat([s, d])
        if int(both.min()) < 0 or int(both.max()) >= num_pages:
            raise ValueError(f"src and dst must be in [0, {num_pages}), got {int(both.min())} to {int(both.max())}")
        if d.unique().numel() != n:
            raise ValueError("a page is the destination of two copies")
        if torch.isin(s, d).any():
            raise ValueError("a page is the source of one copy and the destination of another")
    if reference:
        for i, (a, b) in enumerate(zip(src.tolist(), dst.tolist())):
            if 0 <= a < num_pages and 0 <= b < num_pages:
                for t in pages:
                    t[b] = t[a]
        return pages
    _lib.require_device(pages[0])
    if n and num_pages:
        at, size = _addresses(pages, num_pages)
        _lib.launch("mk_copy_kv_pages", dev, at.buffer_info()[0], size.buffer_info()[0], len(pages), src.data_ptr(),
                    dst.data_ptr(), n, num_pages)
    return pages


# ----------------------------------------------------------------- fork


def _check_table(block_table, ref_counts):
    if block_table.dim() != 2 or block_table.shape[1] == 0:
        raise ValueError(f"block_table must be 2-D [B,MAX_BLOCKS], got {tuple(block_table.shape)}")
    if ref_counts.dim() != 1 or ref_counts.shape[0] == 0:
        raise ValueError(f"ref_counts must be [NUM_PAGES], got {tuple(ref_counts.shape)}")
    for name, t in (("block_table", block_table), ("ref_counts", ref_counts)):
        if t.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
        if t.device != block_table.device:
            raise ValueError(f"tensors are on different devices: {block_table.device} and {t.device}")


def _check_counts(block_table, ref_counts):
    """The host's check that no page has fewer references than the table holds."""
    table, refs = block_table.cpu(), ref_counts.cpu()
    if table.numel() and (int(table.min()) < -1 or int(table.max()) >= refs.shape[0]):
        raise ValueError(f"block_table entries must be in [-1, {refs.shape[0]}), got {int(table.min())} to "
                         f"{int(table.max())}")
    if (refs < count_page_refs(table, refs.shape[0])).any():
        raise ValueError("ref_counts are below the block table's own references")


def fork_kv_sequences(pages, block_table, lengths, ref_counts, parents, *, reserve: int = 1, page_size=None,
                      backend: str = "auto"):
    """The rows of the next step: row r continues row ``parents[r]`` of
    ``block_table`` [B, MAX_BLOCKS] with its ``lengths[parents[r]]`` positions
    (-1: an empty row).  A parent named by several rows is forked, one named by
    none is freed.

    Rows share the pages of their parent.  With ``reserve`` > 0 every row can
    take so many more positions afterwards: it gets the pages for them, and a
    copy of its partly filled last page, in every array of ``pages``, where
    somebody else holds that page too (of the rows that share it the longest,
    then the first, keeps it, if nobody else does).  ``reserve=0`` only shares.
    Table entries behind a row's positions are dropped and handed out anew.

    Returns (block_table [n, MAX_BLOCKS], lengths [n], ref_counts, ready bool
    [n]); the given ones stay as they are, but pages that only dropped rows held
    are free and may have been given away.  ``ready`` is false for a row whose
    pages did not suffice or whose table row is full: it got none, still shares
    its last page, reads as its parent did, and must not be appended to before
    another call says it is ready.  A row that needs no pages is ready also
    behind one whose pages did not suffice.  An empty row has no pages and may
    stay in a batch at position 0: a decode step writes and reads nothing for
    it.  n = len(parents) <= 4096.

    ``page_size`` is needed only without page arrays (``pages=[]``: the tables
    alone).  Entries, counts and parents are checked on the host unless that is
    off (``host_checks_enabled``); then entries outside of the pages are empty
    ones, and parents outside of [0, B) empty rows."""
    reference = _backend(backend)
    _check_table(block_table, ref_counts)
    dev = block_table.device
    num_pages = ref_counts.shape[0]
    _, size = _check_pages(pages, num_pages, dev)
    if size is None:
        size = page_size
    if size is None or size <= 0 or (page_size is not None and page_size != size):
        raise ValueError(f"page_size must be that of the page arrays and positive, got {page_size} for {size}")
    if reserve < 0:
        raise ValueError(f"reserve must be non-negative, got {reserve}")
    B, blocks = block_table.shape
    lengths = _ids(lengths, dev, "lengths")
    if tuple(lengths.shape) != (B,):
        raise ValueError(f"lengths must have shape [B]={(B,)}, got {tuple(lengths.shape)}")
    parents = _ids(parents, dev, "parents")
    if parents.dim() != 1 or parents.shape[0] > MAX_ROWS:
        raise ValueError(f"parents must be [n] with n <= {MAX_ROWS}, got {tuple(parents.shape)}")
    n = parents.shape[0]
    if (blocks + 1) * size >= 2 ** 31 or n * (blocks + 1) >= 2 ** 31:
        raise ValueError(f"a row's positions and a table's entries must fit 31 bits, got {n} rows of {blocks} x {size}")
    if host_checks_enabled(block_table):
        _check_counts(block_table, ref_counts)
        if B and (int(lengths.min()) < 0 or int(lengths.max()) > blocks * size):
            raise ValueError(f"lengths must be in [0, {blocks * size}], got {int(lengths.min())} to {int(lengths.max())}")
        if n and (int(parents.min()) < -1 or int(parents.max()) >= B):
            raise ValueError(f"parents must be in [-1, {B}), got {int(parents.min())} to {int(parents.max())}")
    if reference:
        return _reference_fork(pages, block_table, lengths, ref_counts, parents, reserve, size)
    _lib.require_device(block_table)
    table, refs = narrow_i32(block_table, dev), narrow_i32(ref_counts, dev)
    new_table = torch.empty((n, blocks), dtype=torch.int32, device=dev)
    new_refs = torch.empty_like(refs)
    ready = torch.empty(n, dtype=torch.bool, device=dev)
    ints = 2 * n + 1 + min(num_pages, n * (1 + -(-reserve // size))) if reserve else 0
    buf = torch.empty(n + ints, dtype=torch.int32, device=dev)  # the new lengths, then the workspace
    at, sizes = _addresses(pages, num_pages)
    base = buf.data_ptr()
    _lib.launch("mk_fork_kv_sequences", dev, at.buffer_info()[0], sizes.buffer_info()[0], len(pages),
                table.data_ptr() or None, lengths.data_ptr() or None, refs.data_ptr(), parents.data_ptr() or None,
                new_table.data_ptr() or None, base or None, new_refs.data_ptr(), ready.data_ptr() or None,
                base + 4 * n if ints else None, ints, B, n, blocks, size, num_pages, reserve)
    return new_table, buf[:n], new_refs, ready


def _reference_fork(pages, block_table, lengths, ref_counts, parents, reserve, P):
    dev, num_pages = block_table.device, ref_counts.shape[0]
    B, blocks = block_table.shape
    old, lens, refs = block_table.tolist(), lengths.tolist(), ref_counts.tolist()
    rows, taken = [], {}
    for row in old:
        for p in row:
            if 0 <= p < num_pages:
                refs[p] -= 1
    for parent in parents.tolist():
        live = 0 <= parent < B
        L = min(max(lens[parent], 0), blocks * P) if live else 0
        used = -(-L // P)
        entries = [p if 0 <= p < num_pages else -1 for p in old[parent][:used]] if live else []
        for p in entries:
            if p >= 0:
                refs[p] += 1
        last = entries[-1] if L % P else -1
        rows.append([live, L, entries, last])
        if last >= 0:
            taken.setdefault(last, []).append(len(rows) - 1)
    keeper = {p: max(own, key=lambda r: (rows[r][1] % P, -r)) for p, own in taken.items() if refs[p] == len(own)}
    free = [p for p in range(num_pages) if refs[p] == 0]
    ready, used = [], 0
    for r, (live, L, entries, last) in enumerate(rows):
        fits = not live or reserve == 0 or L + reserve <= blocks * P
        need = -(-(L + reserve) // P) - len(entries) if live and fits and reserve else 0
        copy = bool(live and fits and reserve and last >= 0 and keeper.get(last) != r)
        got = free[used:used + need + copy]
        used += need + copy
        ready.append(fits and used <= len(free) if need + copy else fits)
        if not ready[-1] or not got:
            continue
        for p in got:
            refs[p] += 1
        if copy:
            refs[last] -= 1
            entries[-1] = got.pop(0)
            for t in pages:
                t[entries[-1]] = t[last]
        entries += got
    table = torch.full((len(rows), blocks), -1, dtype=torch.int32)
    for r, (_, _, entries, _) in enumerate(rows):
        table[r, :len(entries)] = torch.tensor(entries, dtype=torch.int32)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    return table.to(dev), ints([r[1] for r in rows]), ints(refs), torch.tensor(ready, dtype=torch.bool, device=dev)


# ----------------------------------------------------------------- compact


def compact_kv_pages(pages, block_table, ref_counts, *, backend: str = "auto"):
    """The live pages (count above 0) of a pool to ids [0, live): of those past
    it, the i-th moves onto the i-th free page below it, in every array of
    ``pages``, in place; the tail of the pool is then free to be given back.

    Returns (block_table through the map, ref_counts, page_map int32
    [NUM_PAGES]: where each page is now, -1 for a free one, with which other
    holders rename theirs, live int32 [1]); the given ones stay as they are."""
    reference = _backend(backend)
    _check_table(block_table, ref_counts)
    dev = block_table.device
    num_pages = ref_counts.shape[0]
    _check_pages(pages, num_pages, dev)
    if host_checks_enabled(block_table):
        _check_counts(block_table, ref_counts)
    if reference:
        held = ref_counts > 0
        live = held.sum().to(torch.int32).reshape(1)
        ids = torch.arange(num_pages, device=dev)
        src, dst = ids[held & (ids >= live)], ids[~held & (ids < live)]
        page_map = torch.where(held, ids, -1).index_put((src,), dst)
        refs = torch.zeros_like(ref_counts).index_put((page_map[held],), ref_counts[held])
        ok = (block_table >= 0) & (block_table < num_pages)
        table = torch.where(ok, page_map[torch.where(ok, block_table, 0).long()], -1)
        for t in pages:
            t[dst] = t[src]
        return table.to(torch.int32), refs.to(torch.int32), page_map.to(torch.int32), live
    _lib.require_device(block_table)
    table, refs = narrow_i32(block_table, dev), narrow_i32(ref_counts, dev)
    new_table = torch.empty_like(table)
    new_refs, page_map = torch.empty_like(refs), torch.empty_like(refs)
    ints = num_pages + -(-num_pages // 8192)
    buf = torch.empty(2 + ints, dtype=torch.int32, device=dev)  # live and moved pages, then the workspace
    at, sizes = _addresses(pages, num_pages)
    base = buf.data_ptr()
    _lib.launch("mk_compact_kv_pages", dev, at.buffer_info()[0], sizes.buffer_info()[0], len(pages),
                table.data_ptr() or None, refs.data_ptr(), new_table.data_ptr() or None, new_refs.data_ptr(),
                page_map.data_ptr(), base, base + 8, ints, table.numel(), num_pages)
    return new_table, new_refs, page_map, buf[:1]
