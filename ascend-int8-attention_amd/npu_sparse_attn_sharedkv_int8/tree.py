"""PreparedTreeAttention: attention of drafted-token trees over the INT8 caches.

No counterpart in the reference, whose draft path lists each token's physical
slots (SharedKVCase.ori_indices) and reads every token's rows for itself.
Here the drafted tokens of a request form a tree and share what they read.

Request b has the query tokens cu_q[b] .. cu_q[b + 1] - 1, its drafted tokens,
and seq_lens[b] rows, the drafted ones included: C = seq_lens[b] - T committed
rows, and the row of drafted token i is logical row C + i of the original
cache (written before the launch, by PreparedCacheWrite).  parents[i] is the
index in the request of token i's parent; an index that is not below the
token's own (-1, by convention) makes it a root, a child of the last committed
token.  A token of depth d (0 for a root) stands at position C + d and sees
  * the original rows j < C with j > C + d - window,
  * its ancestors and itself, those fewer than `window` steps above it,
  * with ratio 128, the compressed rows r < C // 128, those that the committed
    tokens completed, or with causal_compressed=True r < (C + d + 1) // 128,
    those completed up to its own position.
PreparedAttention sees the compressed rows up to a token's position.  A chain is
PreparedAttention over the same rows with ratio 1 and, with ratio 128, with
causal_compressed: its drafted tokens' compressed rows are then written before
the launch, like their rows of the original cache.  Without it a token whose
path passes a multiple of 128 rows misses the row that ends there, and the
original rows of it that have left the window.  With it, row C // 128 + k is one
row for the request: every token from the depth that completes it on sees it, so
where several nodes of a tree stand at that depth (and their paths complete
different rows) the branches have to be requests of their own.  Top-k layers
(ratio 4) have a list of their own for every token, so nothing is shared:
PreparedAttention takes them, with the ancestors' slots in ori_indices.

  out = sum_j e^{s_j} v_j / (e^{sink} + sum_j e^{s_j}),  lse = log of the denominator
"""
import ctypes

import torch

from .attention import _check_cache
from .c8_attention import BLOCK, MAX_HEADS
from .pages import _overlaps
from .runtime import TreeAttentionArgs, library, native_launcher

RATIOS = (1, 128)
MAX_WINDOW = 2 ** 31 - 1


def _check_query(q):
    if q.device.type != "cuda" or q.dtype != torch.bfloat16 or q.ndim != 3 or q.shape[-1] != 512:
        raise ValueError("Expected BF16 Q[T,H,512] on a GPU")
    if not 1 <= q.shape[1] <= MAX_HEADS or not q.is_contiguous() or q.data_ptr() % 16:
        raise ValueError(f"Expected 1..{MAX_HEADS} heads and contiguous, 16-byte aligned Q")


def _check_inputs(case, parents, ori_scale, cmp_scale):
    """Refuses what the kernel cannot take; returns the launch's geometry, (device, the argument block's sizes)."""
    q = case.q
    _check_query(q)
    tokens, heads, _ = q.shape
    if case.ratio not in RATIOS or case.cmp_indices is not None or case.ori_indices is not None:
        raise ValueError("Trees attend a window (ratio 1) or a window and every compressed row (ratio 128); "
                         "layers with lists per token (ratio 4, explicit slots) go through PreparedAttention")
    if not 1 <= case.window <= MAX_WINDOW:
        raise ValueError("Expected a positive window")
    device, batch = q.device, case.seq_lens.numel()
    caches = [(case.ori, case.ori_block_table, ori_scale)]
    if case.ratio != 1:
        caches.append((case.cmp, case.cmp_block_table, cmp_scale))
    for cache, table, scale in caches:
        _check_cache(cache, table, scale, batch, device)
        if (cache.shape[1] != BLOCK or cache.stride(0) % 16 or cache.data_ptr() % 16 or scale.data_ptr() % 16
                or not table.shape[1]):
            raise ValueError(f"Expected pages of {BLOCK} rows, 16-byte aligned, and a block table of one page or more")
    if not batch or tuple(case.cu_q.shape) != (batch + 1,) or case.seq_lens.ndim != 1 \
            or tuple(case.sink.shape) != (heads,):
        raise ValueError("Invalid sequence metadata or sink shape")
    if not isinstance(parents, torch.Tensor) or tuple(parents.shape) != (tokens,):
        raise ValueError("Expected INT32 parents[T]")
    for x, dtype in ((case.cu_q, torch.int32), (case.seq_lens, torch.int32), (case.sink, torch.float32),
                     (parents, torch.int32)):
        if x.dtype != dtype or x.device != device or not x.is_contiguous():
            raise ValueError("Invalid metadata dtype, device or contiguity")
    sizes = dict(tokens=tokens, heads=heads, batch=batch, oriPages=case.ori.shape[0], oriStride=case.ori.stride(0),
                 oriTableWidth=case.ori_block_table.shape[1], ratio=case.ratio, window=case.window,
                 softmaxScale=case.softmax_scale)
    if case.ratio != 1:
        sizes.update(cmpPages=case.cmp.shape[0], cmpStride=case.cmp.stride(0),
                     cmpTableWidth=case.cmp_block_table.shape[1])
    return device, sizes


def _layout(case, parents):
    """What _check_inputs judges but for alignment: inputs laid out alike pass alike, and this is quicker to compare."""
    cmp = (case.cmp, case.cmp_block_table) if case.ratio != 1 else ()
    return (case.ratio, case.window, case.softmax_scale, case.cmp_indices is None, case.ori_indices is None,
            *[(x.shape, x.stride(), x.dtype, x.device) if isinstance(x, torch.Tensor) else None for x in (
                case.q, case.ori, case.ori_block_table, case.cu_q, case.seq_lens, case.sink, parents, *cmp)])


def _check_outputs(out, lse, case, parents, scales):
    q = case.q
    if (out is None or tuple(out.shape) != tuple(q.shape) or out.device != q.device or out.dtype != torch.bfloat16
            or not out.is_contiguous() or out.data_ptr() % 16):
        raise ValueError("Invalid output buffer")
    if lse is not None and (tuple(lse.shape) != tuple(q.shape[:2]) or lse.dtype != torch.float32
                            or lse.device != q.device or not lse.is_contiguous()):
        raise ValueError("Invalid FP32 LSE[T,H] output buffer")
    # A work-group may end, and write, before another reads.
    inputs = [q, parents, case.cu_q, case.seq_lens, case.sink, case.ori, case.ori_block_table, scales[0]]
    if case.ratio != 1:
        inputs += [case.cmp, case.cmp_block_table, scales[1]]
    if _overlaps(out, inputs) or lse is not None and _overlaps(lse, inputs + [out]):
        raise ValueError("Outputs must not overlap inputs or each other")


class PreparedTreeAttention:
    """run() launches on the current stream of the inputs' device, allocates
    nothing and reads nothing back.  Its scratch comes from
    scratch_allocator(name, shape, dtype, device), by default a new tensor, and
    is cleared by the first run (a new tensor of its own before that); launches
    that may overlap must not share it (an operator each, or an allocator by
    stream).

    Protocol: BF16 q[T, H, 512], 1..128 heads; INT8 caches [P, 32, 1, 512] with
    any page stride that is a multiple of 16 bytes; frozen FP32[512] scales;
    ratio 1 (window only) or 128 (and every compressed row of the committed
    tokens, or with causal_compressed of a token's own position); any window >= 1
    (2**30 attends the whole context); cu_q rises from 0.  Rows on pages outside the pool or past
    the block table are masked.  Tokens past cu_q[batch], and those of requests
    with seq_lens 0, are graph padding: their outputs are zero.
    """

    def __init__(self, case, parents, ori_scale, cmp_scale=None, *, output=None, return_lse=False, lse_output=None,
                 scratch_allocator=None, causal_compressed=False):
        self.geometry = _check_inputs(case, parents, ori_scale, cmp_scale)
        self.layout = _layout(case, parents)
        q, device = case.q, case.q.device
        self.case, self.parents, self.scales = case, parents, (ori_scale, cmp_scale)
        self.out = output if output is not None else torch.empty_like(q)
        self.lse = lse_output
        if lse_output is None and return_lse:
            self.lse = torch.empty(q.shape[:2], dtype=torch.float32, device=device)
        _check_outputs(self.out, self.lse, case, parents, self.scales)
        _, sizes = self.geometry
        self.args = TreeAttentionArgs(**sizes, oriScale=ori_scale.data_ptr(),
                                      cmpScale=cmp_scale.data_ptr() if case.ratio != 1 else 0,
                                      causalCompressed=int(bool(causal_compressed)))
        self._bind()
        self._take_scratch(scratch_allocator, device)
        self.native = native_launcher()
        self.argument_address = ctypes.addressof(self.args)
        self.device_index = device.index if device.index is not None else torch.cuda.current_device()

    def _take_scratch(self, allocator, device):
        sizes = ctypes.c_uint64(), ctypes.c_uint64()
        if self.args.tokens and library().sharedkv_tree_scratch(ctypes.addressof(self.args), *map(ctypes.byref, sizes)):
            raise ValueError("This launch is outside the tree kernel's limits (some 2^30 query rows, 2^24 requests)")
        allocate = allocator or (lambda name, shape, dtype, dev: torch.empty(shape, dtype=dtype, device=dev))
        tickets, states = (size.value // 4 for size in sizes)
        self.workspace = self.partial = None
        self._unclear = False
        if states:
            # Merge tickets, which every launch leaves zero, and partition states.
            self.workspace = allocate("tree_workspace", (tickets,), torch.int32, device)
            self.partial = allocate("tree_partial", (states,), torch.float32, device)
            # A caller's scratch is cleared by the first run, in its stream's order, so that making an operator in a
            # serving loop waits for nothing.  Under capture a clear only becomes part of that graph: run() clears too,
            # until it has done so eagerly.
            self._unclear = allocator is not None or torch.cuda.is_current_stream_capturing()
            if not self._unclear:
                self.workspace.zero_()
                torch.cuda.current_stream(device).synchronize()  # run() may come on another stream
            self.args.workspace, self.args.partial = self.workspace.data_ptr(), self.partial.data_ptr()

    def _bind(self):
        case, args = self.case, self.args
        cmp = case.ratio != 1
        for name, tensor in (("q", case.q), ("ori", case.ori), ("oriTable", case.ori_block_table),
                             ("cmp", case.cmp if cmp else None), ("cmpTable", case.cmp_block_table if cmp else None),
                             ("cuQ", case.cu_q), ("seqLens", case.seq_lens), ("sinks", case.sink),
                             ("parents", self.parents), ("out", self.out), ("lse", self.lse)):
            setattr(args, name, tensor.data_ptr() if tensor is not None else 0)

    def _rebind_same_geometry(self, case, parents, *, output=None, lse_output=None):
        """Serving fast path: same geometry, new tensors, under the constructor's checks (the kernel reads them by it)."""
        if _layout(case, parents) != self.layout or (case.q.data_ptr() | case.ori.data_ptr()) % 16 \
                or case.ratio != 1 and case.cmp.data_ptr() % 16:
            if _check_inputs(case, parents, *self.scales) != self.geometry:
                raise ValueError("Rebinding keeps the device and every size of the launch")
        out, lse = (output, lse_output) if output is not None else (self.out, self.lse)
        _check_outputs(out, lse, case, parents, self.scales)
        self.case, self.parents, self.out, self.lse = case, parents, out, lse
        self._bind()

    def run(self):
        """Launch on the current stream of the case's device; returns .out."""
        if self._unclear:
            with torch.cuda.device(self.device_index):
                self.workspace.zero_()
                self._unclear = torch.cuda.is_current_stream_capturing()
        if self.args.tokens:
            self.native.launch("tree_attention", self.argument_address, self.device_index)
        return self.out
