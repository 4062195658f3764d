"""Pages of a cache pool: accepted paths, forked and freed rows, compaction.

No counterpart in the reference, whose engine moves pages on the host.  These
operators keep the block tables and reference counts of a pool on the device,
beside the caches that PreparedCacheWrite fills and PreparedAttention and
PreparedTreeAttention read, so a speculative or branching decode loop needs no
host round trip and can be captured in a graph.

`caches` is a tensor or a list of tensors that share page numbers (the layers
of a pool, or the compact planner's whole backing as [blocks, stride bytes]);
page p of a cache is cache[p].  All operators move whole 16-byte units and
never touch bytes outside the pages' payload.

Entries of a block table are page numbers; -1 (anything outside the pool) is no
page.  refs INT32 [pages] counts the owners of each page: the table rows that
name it and whatever else holds it; 0 is a free page.
"""
import ctypes

import torch

from .runtime import PageCompactArgs, PageForkArgs, PathCommitArgs, library, native_launcher

UNIT = 16
MAX_PAGES = 2 ** 22


def _ints(tensor, shape, device, what):
    """A contiguous INT32 tensor of `shape` (None: any extent) on `device`."""
    if (not isinstance(tensor, torch.Tensor) or tensor.dtype != torch.int32 or tensor.ndim != len(shape)
            or any(want is not None and want != got for want, got in zip(shape, tensor.shape))
            or tensor.device != device or not tensor.is_contiguous()):
        sizes = ",".join("*" if n is None else str(n) for n in shape)
        raise ValueError(f"Expected contiguous INT32 {what}[{sizes}] on the caches' GPU")


def _extent(x):
    """Bytes from a tensor's first to its last."""
    if x.is_contiguous():
        return x.nbytes
    return (1 + sum((n - 1) * step for n, step in zip(x.shape, x.stride()))) * x.element_size() if x.numel() else 0


def _overlaps(tensor, others):
    first, end = tensor.data_ptr(), tensor.data_ptr() + _extent(tensor)
    for x in others:
        at = x.data_ptr()
        if at < end and first < at + _extent(x):
            return True
    return False


def _overlap(a, b):
    return _overlaps(a, (b,))


def _inner(cache, first):
    """Bytes of the dimensions from `first` on, which have to be one run."""
    run = 1
    for size, stride in zip(reversed(cache.shape[first:]), reversed(cache.stride()[first:])):
        if size != 1 and stride != run:
            return 0
        run *= size
    return run * cache.element_size()


def _runs(c, dims):
    """(start, strides of the first `dims` dimensions, bytes from the first to
    the last of the dimensions from each on), all in bytes."""
    size = c.element_size()
    steps = tuple(s * size for s in c.stride()[:dims])
    spans = [_inner(c, dims)]
    for n, step in zip(reversed(c.shape[:dims]), reversed(steps)):
        spans.append(spans[-1] + (n - 1) * step)
    return c.data_ptr(), steps, spans[::-1]


def _apart(a, b):
    """Whether two caches (as _runs) share no byte: separate memory, or runs
    that lie side by side in the same strides (layers interleaved in a pool's
    pages, parts of its rows)."""
    (at_a, steps, spans_a), (at_b, steps_b, spans_b) = a, b
    ahead = at_b - at_a
    if ahead >= spans_a[0] or -ahead >= spans_b[0]:
        return True
    if steps != steps_b:
        return False
    # In steps of one stride that every run of both keeps to.
    return any(step and not any(s % step for s in steps[:level])
               and spans_a[level + 1] <= ahead % step <= step - spans_b[level + 1]
               for level, step in enumerate(steps))


def _all_apart(caches, dims):
    runs = sorted(_runs(c, dims) for c in caches)
    if all(a[0] + a[2][0] <= b[0] for a, b in zip(runs, runs[1:])):
        return True                                     # memory of their own
    step = runs[0][1][0]
    if step and all(r[1] == runs[0][1] for r in runs):
        # Pages interleaved in one backing: neighbours within a stride, and the last to the next stride's first.
        places = sorted((r[0] % step, r[2][1]) for r in runs)
        if all(at + size <= after for (at, size), (after, _) in zip(places, places[1:] + [(places[0][0] + step, 0)])):
            return True
    return all(_apart(a, b) for i, a in enumerate(runs) for b in runs[:i])


def _check_caches(caches, dims):
    """The caches as a list, after the checks all operators share: on one GPU,
    the same number of pages, each page (dims = 1) or row of a page (2) one run
    of bytes, everything in 16-byte units, no two pages overlapping."""
    caches = list(caches) if isinstance(caches, (list, tuple)) else [caches]
    if not caches or any(not isinstance(c, torch.Tensor) or c.device.type != "cuda" or c.ndim <= dims for c in caches):
        raise ValueError("Expected one or more GPU caches [pages, rows, ...]" if dims == 2 else
                         "Expected one or more GPU caches [pages, ...]")
    device, leading = caches[0].device, tuple(caches[0].shape[:dims])
    for c in caches:
        size = c.element_size()
        inner = _inner(c, dims)
        span = inner if dims == 1 else (c.shape[1] - 1) * c.stride(1) * size + inner
        if c.device != device or tuple(c.shape[:dims]) != leading:
            raise ValueError("Caches must have the same pages on the same GPU")
        if not inner or inner % UNIT or c.data_ptr() % UNIT or any(s * size % UNIT for s in c.stride()[:dims]):
            raise ValueError(f"Cache pages and rows must be contiguous in whole {UNIT}-byte units")
        if (c.shape[0] > 1 and c.stride(0) * size < span) or (dims == 2 and c.shape[1] > 1 and c.stride(1) * size < inner):
            raise ValueError("Cache pages and rows must not overlap")
    if not _all_apart(caches, dims):
        raise ValueError("Caches must not overlap")
    if not 1 <= leading[0] <= MAX_PAGES:
        raise ValueError(f"Expected 1..{MAX_PAGES} pages")
    return caches


def _spans(caches, dims):
    """Device array of CacheSpan (include/sharedkv_hip.h)."""
    rows = [[c.data_ptr(), c.stride(0) * c.element_size(), c.stride(1) * c.element_size() if dims == 2 else 0,
             _inner(c, dims)] for c in caches]
    return torch.tensor(rows, dtype=torch.int64, device=caches[0].device), [row[3] for row in rows]


class _Prepared:
    """Shared end of the constructors, and run()."""

    def _finish(self, name, device):
        self._name = name
        self.native = native_launcher()
        self.argument_address = ctypes.addressof(self.args)
        self.device_index = device.index if device.index is not None else torch.cuda.current_device()

    def _launch(self):
        self.native.launch(self._name, self.argument_address, self.device_index)


class PreparedPathCommit(_Prepared):
    """Keeps the accepted path of each request's drafted tokens.

    cu_q INT32 [batch + 1] and seq_lens INT32 [batch] are those of the tree
    launch: T = cu_q[b + 1] - cu_q[b] drafted rows behind C = seq_lens[b] - T
    committed ones.  paths INT32 [batch, depth] names the accepted tokens by
    their index in the request, rising (root first); path_lens INT32 [batch]
    says how many.  A path ends before its first entry that does not rise or is
    none of the request's tokens.  run() moves row C + paths[b][k] to row C + k
    in every cache [pages, rows, ...] of `caches` and returns .seq_lens INT32
    [batch] = C + accepted (0 for padding requests, seq_lens 0).  Rows on no
    page of the pool stay.  The pages behind belong to the request alone
    (PreparedPageFork sees to that).  No allocations or host reads in run().
    """

    def __init__(self, caches, block_table, cu_q, seq_lens, paths, path_lens, *, output=None):
        self.caches = caches = _check_caches(caches, 2)
        device = caches[0].device
        if not isinstance(seq_lens, torch.Tensor) or not isinstance(paths, torch.Tensor) or paths.ndim != 2:
            raise ValueError("Expected INT32 seq_lens[batch] and paths[batch, depth]")
        batch = seq_lens.numel()
        _ints(seq_lens, (batch,), device, "seq_lens")
        _ints(cu_q, (batch + 1,), device, "cu_q")
        _ints(block_table, (batch, None), device, "block_table")
        _ints(paths, (batch, None), device, "paths")
        _ints(path_lens, (batch,), device, "path_lens")
        if not batch or not paths.shape[1] or not block_table.shape[1]:
            raise ValueError("Expected one request, path entry and table entry or more")
        self.seq_lens = output if output is not None else torch.empty_like(seq_lens)
        _ints(self.seq_lens, (batch,), device, "output")
        if _overlaps(self.seq_lens, (seq_lens, cu_q, block_table, paths, path_lens, *caches)):
            raise ValueError("The new lengths need a buffer of their own")
        self.block_table, self.inputs = block_table, (cu_q, seq_lens, paths, path_lens)
        self.spans, sizes = _spans(caches, 2)
        self.args = PathCommitArgs(
            caches=self.spans.data_ptr(), table=block_table.data_ptr(), cuQ=cu_q.data_ptr(),
            seqLens=seq_lens.data_ptr(), paths=paths.data_ptr(), pathLens=path_lens.data_ptr(),
            lengths=self.seq_lens.data_ptr(), cacheCount=len(caches), batch=batch, depth=paths.shape[1],
            tokens=2 ** 31 - 1, tableWidth=block_table.shape[1], pages=caches[0].shape[0],
            pageRows=caches[0].shape[1], rowBytes=max(sizes))
        self._finish("path_commit", device)

    def run(self):
        """Launch on the current stream of the caches' device; returns .seq_lens."""
        self._launch()
        return self.seq_lens


def _table_outputs(block_table, shape, refs, outputs, device):
    table, counts = outputs
    table = torch.empty(shape, dtype=torch.int32, device=device) if table is None else table
    counts = torch.empty_like(refs) if counts is None else counts
    _ints(table, shape, device, "new block table")
    _ints(counts, tuple(refs.shape), device, "new refs")
    return table, counts


def _check_aliases(pairs, others):
    """An output may be the input that it replaces, whole; no other overlap."""
    outputs = [out for out, _ in pairs]
    for out, source in pairs:
        same = source is not None and out.data_ptr() == source.data_ptr() and out.numel() == source.numel()
        rest = [x for x in others + [o for o in outputs if o is not out] + [s for _, s in pairs if s is not None]
                if not (same and x is source)]
        if any(x.numel() and out.numel() and _overlap(out, x) for x in rest):
            raise ValueError("Outputs may be the inputs they replace, and must not overlap anything else")


class PreparedPageFork(_Prepared):
    """Rows of a block table that go on as other rows: forked, reordered, grown
    and ended requests.

    Every row of block_table INT32 [rows, width], with seq_lens INT32 [rows]
    tokens in pages of `page_size`, is given up; row i of the new table
    continues row parents[i] (INT32 [children]; outside [0, rows): an empty row
    of length 0) and has pages for length + room tokens (at most `width`).  The
    parent's whole pages are shared.  Of its other pages the first of its
    children keeps those that no one else owns (refs 1); all others come from
    the lowest pages that are free (refs 0) when the call begins, by row, then
    entry, and a partly filled page is copied in every cache [pages, ...] of
    `caches`.  Pages given up are free for the next call.  Where free pages run
    out, an entry is -1, a row without its partly filled page is cut back to
    its whole pages, and .missing (INT32 [1]) counts the entries.

    run() returns (.block_table [children, width], .seq_lens [children],
    .refs [pages]); `output` gives their buffers, which may be the inputs they
    replace.  No allocations or host reads in run(); launches of one operator
    that may overlap need an operator each (they share its workspace).
    """

    def __init__(self, caches, block_table, seq_lens, refs, parents, *, room=0, page_size=32, output=None):
        self.caches = caches = _check_caches(caches, 1)
        device, pages = caches[0].device, caches[0].shape[0]
        if not isinstance(block_table, torch.Tensor) or block_table.ndim != 2 or not isinstance(parents, torch.Tensor):
            raise ValueError("Expected INT32 block_table[rows, width] and parents[children]")
        rows, width = block_table.shape
        children = parents.numel()
        _ints(block_table, (rows, width), device, "block_table")
        _ints(seq_lens, (rows,), device, "seq_lens")
        _ints(refs, (pages,), device, "refs")
        _ints(parents, (children,), device, "parents")
        if not rows or not width or not children:
            raise ValueError("Expected one row, entry and child or more")
        if not isinstance(room, int) or not 0 <= room < 2 ** 30 or not isinstance(page_size, int) \
                or not 1 <= page_size < 2 ** 24:
            raise ValueError("Expected room for 0 .. 2**30 - 1 tokens and pages of 1 .. 2**24 - 1")
        new_table, new_lens, new_refs = output if output is not None else (None, None, None)
        self.block_table, self.refs = _table_outputs(block_table, (children, width), refs, (new_table, new_refs), device)
        self.seq_lens = new_lens if new_lens is not None else torch.empty(children, dtype=torch.int32, device=device)
        _ints(self.seq_lens, (children,), device, "new seq_lens")
        _check_aliases([(self.block_table, block_table), (self.seq_lens, seq_lens), (self.refs, refs)],
                       [parents, *caches])
        self.missing = torch.zeros(1, dtype=torch.int32, device=device)
        self.inputs = block_table, seq_lens, refs, parents
        self.spans, sizes = _spans(caches, 1)
        # The counts' changes in it are zero between launches.
        self.workspace = torch.zeros(int(library().sharedkv_page_fork_workspace(children, width, pages)),
                                     dtype=torch.uint8, device=device)
        torch.cuda.current_stream(device).synchronize()      # run() may come on another stream
        self.args = PageForkArgs(
            caches=self.spans.data_ptr(), table=block_table.data_ptr(), seqLens=seq_lens.data_ptr(),
            refs=refs.data_ptr(), parents=parents.data_ptr(), newTable=self.block_table.data_ptr(),
            newLens=self.seq_lens.data_ptr(), newRefs=self.refs.data_ptr(), missing=self.missing.data_ptr(),
            workspace=self.workspace.data_ptr(), cacheCount=len(caches), rows=rows, children=children, width=width,
            pages=pages, pageRows=page_size, room=room, pageBytes=sum(sizes))
        self._finish("page_fork", device)

    def run(self):
        """Launch on the current stream of the caches' device; returns
        (.block_table, .seq_lens, .refs)."""
        self._launch()
        return self.block_table, self.seq_lens, self.refs


class PreparedPageCompact(_Prepared):
    """Moves the pages in use to the front of the pool.

    With L pages in use (refs > 0), those from L on move, in order, to the free
    pages below L, in order, in every cache [pages, ...] of `caches`; the
    entries of block_table INT32 [rows, width] and the refs INT32 [pages]
    follow, and pages [L, pages) are free.  .moved INT32 [pages] gives each
    page's new number (-1 for free ones), for whatever else names pages; .live
    INT32 [1] is L.  Entries outside the pool or on free pages become -1.

    run() returns (.block_table, .refs, .moved); `output` gives the buffers of
    the first two, which may be the inputs they replace.  No allocations or
    host reads in run(); launches of one operator that may overlap need an
    operator each (they share its workspace).
    """

    def __init__(self, caches, block_table, refs, *, output=None):
        self.caches = caches = _check_caches(caches, 1)
        device, pages = caches[0].device, caches[0].shape[0]
        _ints(block_table, (None, None), device, "block_table")
        _ints(refs, (pages,), device, "refs")
        if not block_table.numel():
            raise ValueError("Expected one row and entry or more")
        self.block_table, self.refs = _table_outputs(block_table, tuple(block_table.shape), refs,
                                                     output if output is not None else (None, None), device)
        _check_aliases([(self.block_table, block_table), (self.refs, refs)], caches)
        self.moved = torch.empty_like(refs)
        self.live = torch.zeros(1, dtype=torch.int32, device=device)
        self.inputs = block_table, refs
        self.spans, sizes = _spans(caches, 1)
        self.workspace = torch.empty(int(library().sharedkv_page_compact_workspace(pages)), dtype=torch.uint8,
                                     device=device)
        self.args = PageCompactArgs(
            caches=self.spans.data_ptr(), table=block_table.data_ptr(), refs=refs.data_ptr(),
            newTable=self.block_table.data_ptr(), newRefs=self.refs.data_ptr(), moved=self.moved.data_ptr(),
            live=self.live.data_ptr(), workspace=self.workspace.data_ptr(), cacheCount=len(caches),
            rows=block_table.shape[0], width=block_table.shape[1], pages=pages, pageBytes=sum(sizes))
        self._finish("page_compact", device)

    def run(self):
        """Launch on the current stream of the caches' device; returns
        (.block_table, .refs, .moved)."""
        self._launch()
        return self.block_table, self.refs, self.moved
