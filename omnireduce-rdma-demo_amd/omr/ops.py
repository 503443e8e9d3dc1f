"""Device-tensor front end of the C ABI (include/omr.h).

Every function here is a thin call through libomr.so on torch-allocated HBM buffers and the current HIP
stream; torch provides memory and streams only.  Names follow the reference: the worker scan
(client.cc:19-31), the aggregator sum (server.cc:83-99), the generator (client.cc:396-421).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib
from .layout import MESSAGE_SIZE, NUM_SLOTS, Layout


def _stream(stream: Optional[torch.cuda.Stream] = None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("expected a device (HIP) tensor")
    if not t.is_contiguous():
        raise ValueError("expected a contiguous tensor")
    return t.data_ptr()


def _ptr_array(ts: Sequence[torch.Tensor]):
    arr = (ctypes.c_void_p * len(ts))()
    for i, t in enumerate(ts):
        arr[i] = _ptr(t)
    return arr


def _check_f32(t: torch.Tensor, n: int, name: str) -> None:
    if t.dtype != torch.float32 or t.numel() != n:
        raise ValueError(f"{name}: expected float32[{n}], got {t.dtype}[{t.numel()}]")


# ------------------------------------------------------------------ generator (client.cc:396-421)

def gen_bitmap(worker_id: int, density_ratio: float, num_blocks: int) -> np.ndarray:
    """The reference bitmap of worker `worker_id` (srand(myId+1); rand()%100/(double)101 < r)."""
    lib = _lib.load()
    bm = np.empty(num_blocks, dtype=np.int32)
    cnt = ctypes.c_uint64(0)
    _lib.check(lib.omr_gen_bitmap(worker_id, float(density_ratio), num_blocks,
                                  bm.ctypes.data_as(ctypes.c_void_p), ctypes.byref(cnt)), "omr_gen_bitmap")
    return bm


def fill_blocks(bitmap: torch.Tensor, layout: Layout, mode: int = 0, seed: int = 0,
                out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Device fill from a device int32 bitmap: mode 0 = 0.01f (client.cc:415-419), 1 = hashed [-1,1)."""
    if bitmap.dtype != torch.int32 or bitmap.numel() != layout.nb:
        raise ValueError("bitmap must be int32[nb]")
    if out is None:
        out = torch.empty(layout.n, dtype=torch.float32, device=bitmap.device)
    _check_f32(out, layout.n, "out")
    _lib.check(_lib.load().omr_fill_blocks_f32(_ptr(bitmap), layout.nb, layout.block_size, mode, seed,
                                               _ptr(out), _stream(stream)), "omr_fill_blocks_f32")
    return out


def make_worker_buffer(worker_id: int, density_ratio: float, layout: Layout, device="cuda", mode: int = 0,
                       seed: Optional[int] = None) -> torch.Tensor:
    bm = torch.from_numpy(gen_bitmap(worker_id, density_ratio, layout.nb)).to(device)
    return fill_blocks(bm, layout, mode=mode, seed=worker_id + 1 if seed is None else seed)


# ------------------------------------------------------------------ scan + sum

@dataclass
class ScanResult:
    flags: Optional[torch.Tensor]  # int32 [m][nb]
    masks: torch.Tensor  # uint64-as-int64 [m(+1)][rows]
    next_offsets: Optional[torch.Tensor]  # uint32-as-int32 [m(+1)][nb]
    out: Optional[torch.Tensor]


class ScanSumPlan:
    """Preallocated outputs for repeated fused scan+sum launches (no allocation per call, capturable).

    flags        int32  [m, nb]             per-worker block flags (the reference's int *bitmap)
    masks        int64  [m(+1), rows]       per-worker row masks (+ the union row at index m when m > 1)
    next_offsets int32  [m(+1), nb]         per-worker next-offset chains (+ the aggregator chain), uint32 bits
    """

    def __init__(self, layout: Layout, m: int = 1, with_flags: bool = True, with_next: bool = True,
                 device="cuda", fused: bool = False, row_masks: bool = False):
        """fused=True (m = 1 only): one single-pass launch (omr_scan_sum_fused_f32) producing flags, next
        offsets and the aggregated blocks; with row_masks=True it is the multi-rank round's worker scan
        (omr_worker_scan_f32), which also ORs the row masks into `masks` (zeroed before each run)."""
        if not 1 <= m <= _lib.OMR_MAX_WORKERS:
            raise ValueError(f"m={m} out of range")
        lib = _lib.load()
        _lib.check(lib.omr_layout_check(layout.n, layout.block_size, layout.num_lanes, layout.num_threads),
                   "omr_layout_check")
        if fused and (m != 1 or not with_next):
            raise ValueError("the fused single-pass kernel is the m = 1 step with next offsets")
        self.layout, self.m, self.fused = layout, m, fused
        arrays = m if m == 1 else m + 1
        self.flags = torch.empty((m, layout.nb), dtype=torch.int32, device=device) if with_flags else None
        self.row_masks = bool(fused and row_masks)
        self.masks = (None if fused and not row_masks else
                      torch.zeros((arrays, layout.rows), dtype=torch.int64, device=device))
        self.next_offsets = (torch.empty((arrays, layout.nb), dtype=torch.int32, device=device)
                             if with_next else None)
        ws = lib.omr_scan_workspace_bytes(layout.n, layout.block_size, layout.num_lanes, layout.num_threads)
        self.workspace = torch.zeros(max(ws, 16), dtype=torch.uint8, device=device) if fused else None

    def bind(self, buf: torch.Tensor, out: Optional[torch.Tensor] = None, stream=None):
        """The fused m = 1 launch with its arguments checked and converted once: returns a zero-argument callable
        that issues omr_scan_sum_fused_f32 (one C call per step, for a host-light loop; raises on error)."""
        if not self.fused or self.row_masks or self.m != 1:
            raise ValueError("bind(): the fused m = 1 scan + sum only")
        L = self.layout
        _check_f32(buf, L.n, "buf")
        if out is not None:
            _check_f32(out, L.n, "out")
        fn = _lib.load().omr_scan_sum_fused_f32
        args = (_ptr(buf), L.n, L.block_size, L.num_lanes, L.num_threads, _ptr(self.flags), _ptr(self.next_offsets),
                _ptr(out), _ptr(self.workspace), self.workspace.numel(), _stream(stream))

        def launch():
            rc = fn(*args)
            if rc:
                _lib.check(rc, "omr_scan_sum_fused_f32")
        return launch

    def run(self, bufs: Sequence[torch.Tensor], out: Optional[torch.Tensor] = None, stream=None,
            with_next: bool = True, zero_masks: bool = True) -> ScanResult:
        """Fused scan (+ sum into `out`) and, unless with_next=False, the next-offset chains."""
        L = self.layout
        if len(bufs) != self.m:
            raise ValueError(f"expected {self.m} worker buffers, got {len(bufs)}")
        for i, b in enumerate(bufs):
            _check_f32(b, L.n, f"bufs[{i}]")
        if out is not None:
            _check_f32(out, L.n, "out")
        if self.fused and self.row_masks:
            if zero_masks:
                self.masks.zero_()
            _lib.check(_lib.load().omr_worker_scan_f32(
                _ptr(bufs[0]), L.n, L.block_size, L.num_lanes, L.num_threads, _ptr(self.flags),
                _ptr(self.next_offsets), _ptr(self.masks), _ptr(out), _ptr(self.workspace), self.workspace.numel(),
                _stream(stream)), "omr_worker_scan_f32")
            return ScanResult(self.flags, self.masks, self.next_offsets, out)
        if self.fused:
            _lib.check(_lib.load().omr_scan_sum_fused_f32(
                _ptr(bufs[0]), L.n, L.block_size, L.num_lanes, L.num_threads, _ptr(self.flags),
                _ptr(self.next_offsets), _ptr(out), _ptr(self.workspace), self.workspace.numel(), _stream(stream)),
                "omr_scan_sum_fused_f32")
            return ScanResult(self.flags, self.masks, self.next_offsets, out)
        arr = _ptr_array(bufs)
        nxt = self.next_offsets if with_next else None
        _lib.check(_lib.load().omr_scan_sum_f32(arr, self.m, L.n, L.block_size, L.num_lanes, L.num_threads,
                                                _ptr(self.flags), _ptr(self.masks), _ptr(nxt),
                                                _ptr(out), _stream(stream)), "omr_scan_sum_f32")
        return ScanResult(self.flags, self.masks, self.next_offsets, out)

    def resolve_next(self, stream=None) -> torch.Tensor:
        """Next-offset chains from the masks of the last run (the second kernel of run())."""
        L = self.layout
        if self.next_offsets is None:
            raise ValueError("plan built with with_next=False")
        _lib.check(_lib.load().omr_next_offsets(_ptr(self.masks), self.masks.shape[0], L.n, L.block_size,
                                                L.num_lanes, L.num_threads, _ptr(self.next_offsets),
                                                _stream(stream)), "omr_next_offsets")
        return self.next_offsets


def scan_workspace(layout: Layout, device="cuda") -> torch.Tensor:
    """Zeroed workspace for the single-pass kernels (omr_scan_workspace_bytes; one per concurrently running whole-
    tensor call, or ONE shared by concurrent per-partition calls)."""
    ws = _lib.load().omr_scan_workspace_bytes(layout.n, layout.block_size, layout.num_lanes, layout.num_threads)
    return torch.zeros(max(ws, 16), dtype=torch.uint8, device=device)


def scan_partition(buf: torch.Tensor, layout: Layout, part: int, flags: Optional[torch.Tensor],
                   next_offsets: torch.Tensor, out: Optional[torch.Tensor], workspace: torch.Tensor,
                   stream=None) -> None:
    """The single-pass worker step for partition `part` only (omr_scan_partition_f32): the reference's per-thread
    seam, worker thread res->threadId walking its own DATA_SIZE_PER_THREAD slice (client.cc:19-31, :168-223).
    flags / next_offsets / out are whole-tensor arrays (global indexing); only the partition's entries are written.
    Safe to call from several host threads at once, one partition and one stream each (ctypes drops the GIL)."""
    _check_f32(buf, layout.n, "buf")
    if out is not None:
        _check_f32(out, layout.n, "out")
    lib = _lib.load()
    rc = lib.omr_scan_partition_f32(_ptr(buf), layout.n, layout.block_size, layout.num_lanes, layout.num_threads,
                                    part, _ptr(flags), _ptr(next_offsets), _ptr(out), _ptr(workspace),
                                    workspace.numel(), _stream(stream))
    _lib.check(rc, "omr_scan_partition_f32")


def scan(buf: torch.Tensor, layout: Layout, stream=None) -> ScanResult:
    """Worker-side scan (client.cc:19-31): flags, row masks and next offsets of one gradient buffer."""
    return ScanSumPlan(layout, 1, device=buf.device).run([buf], None, stream)


def scan_sum(bufs: Sequence[torch.Tensor], layout: Layout, out: Optional[torch.Tensor] = None,
             stream=None) -> ScanResult:
    """m worker scans + aggregator sum (server.cc:83-99) in one HBM pass."""
    if out is None:
        out = torch.zeros(layout.n, dtype=torch.float32, device=bufs[0].device)
    return ScanSumPlan(layout, len(bufs), device=bufs[0].device).run(bufs, out, stream)


def next_offsets(masks: torch.Tensor, layout: Layout, stream=None) -> torch.Tensor:
    """Next-offset chains from row masks [count, rows] (client.cc:19-31; server.cc:86-96 on a union)."""
    if masks.dim() == 1:
        masks = masks.view(1, -1)
    if masks.dtype != torch.int64 or masks.shape[1] != layout.rows:
        raise ValueError("masks must be int64[count, rows]")
    count = masks.shape[0]
    nxt = torch.empty((count, layout.nb), dtype=torch.int32, device=masks.device)
    _lib.check(_lib.load().omr_next_offsets(_ptr(masks.contiguous()), count, layout.n, layout.block_size,
                                            layout.num_lanes, layout.num_threads, _ptr(nxt), _stream(stream)),
               "omr_next_offsets")
    return nxt


# ------------------------------------------------------------------ compaction and block movement

class CompactPlan:
    def __init__(self, rows: int, num_lanes: int, device="cuda"):
        self.rows, self.num_lanes = rows, num_lanes
        ws = _lib.load().omr_compact_workspace_bytes(rows)
        self.workspace = torch.empty(ws, dtype=torch.uint8, device=device)
        self.count = torch.zeros(1, dtype=torch.int32, device=device)
        self.block_list = torch.empty(rows * num_lanes, dtype=torch.int32, device=device)

    def run(self, masks: torch.Tensor, row_begin: int = 0, row_end: Optional[int] = None, stream=None):
        row_end = self.rows if row_end is None else row_end
        _lib.check(_lib.load().omr_compact(_ptr(masks), row_begin, row_end, self.num_lanes,
                                           _ptr(self.block_list), _ptr(self.count), _ptr(self.workspace),
                                           self.workspace.numel(), _stream(stream)), "omr_compact")
        return self.block_list, self.count


def compact(masks: torch.Tensor, layout: Layout, row_begin: int = 0, row_end: Optional[int] = None,
            stream=None) -> torch.Tensor:
    """Global indices of the non-zero blocks of rows [row_begin, row_end), increasing (synchronises)."""
    plan = CompactPlan(layout.rows, layout.num_lanes, device=masks.device)
    lst, cnt = plan.run(masks.contiguous(), row_begin, row_end, stream)
    return lst[: int(cnt.item())].clone()


def gather_blocks(src: torch.Tensor, block_list: torch.Tensor, num: int, block_size: int,
                  packed: torch.Tensor, stream=None) -> torch.Tensor:
    """Pack listed blocks contiguously (worker gather, common.cc:405-407)."""
    if num:
        _lib.check(_lib.load().omr_gather_blocks_f32(_ptr(src), _ptr(block_list), num, block_size,
                                                     _ptr(packed), _stream(stream)), "omr_gather_blocks_f32")
    return packed


def scatter_blocks(packed: torch.Tensor, block_list: torch.Tensor, num: int, block_size: int,
                   dst: torch.Tensor, stream=None) -> torch.Tensor:
    """Write packed blocks back in place (worker result copy, client.cc:89)."""
    if num:
        _lib.check(_lib.load().omr_scatter_blocks_f32(_ptr(packed), _ptr(block_list), num, block_size,
                                                      _ptr(dst), _stream(stream)), "omr_scatter_blocks_f32")
    return dst


def block_sum(inputs: Sequence[torch.Tensor], block_list: torch.Tensor, num: int, block_size: int,
              out: torch.Tensor, stream=None) -> torch.Tensor:
    """out[b] = ((0 + in_0[b]) + in_1[b]) + ... for listed blocks b (server.cc:97-98, rank order)."""
    if num:
        arr = _ptr_array(inputs)
        _lib.check(_lib.load().omr_block_sum_f32(arr, len(inputs), _ptr(block_list), num, block_size,
                                                 _ptr(out), _stream(stream)), "omr_block_sum_f32")
    return out


# ------------------------------------------------------------------ operators that make the gradient

# The two ends of a language model: their parameter gradients are the fp32 tensors the all-reduce sums.  Every output may
# be given (a view of the flat gradient, say); what is not given is allocated on the call's stream.  Nothing here records
# autograd nodes: inputs that require a gradient give outputs that do not, and the backward passes are calls of their own.
# Work runs on `stream`, or on the current stream of the tensors' device.  A plan's workspace serves one call at a time:
# calls that may overlap (two streams, two captured graphs replayed side by side) need a plan each, and a captured graph
# needs its plan and its tensors for as long as it is replayed.

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# (torch.cuda.current_stream(i).cuda_stream and torch.cuda.current_device(), without the objects they make)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_MAX_DIM = 1 << 24  # OMR_MAX_DIM
_F32 = torch.float32


def _sizes(count: int, rows: int, dim: int, least: int = 0):
    """A plan's sizes are in range (the C calls take unsigned integers)."""
    if not (0 <= count < 1 << 40 and least <= rows < 1 << 31 and 0 < dim <= _MAX_DIM):
        raise ValueError(f"no such sizes: {count} tokens (rows), a table of {rows}, rows of {dim}")


class _Call:
    """The device and stream of one call; every tensor must be on that device.  (Short calls are bound by what is done
    here: a look at a tensor costs 50 to 80 ns, and is made once.)"""

    __slots__ = ("index", "stream", "ptr")

    def __init__(self, t: torch.Tensor, stream: Optional[torch.cuda.Stream]):
        self.index = index = t.get_device()
        if index < 0:
            raise ValueError("expected a device (HIP) tensor")
        self.stream = stream
        if stream is None:
            self.ptr = _raw_stream(index)
        elif stream.device.index != index:
            raise ValueError(f"the stream is on {stream.device}, the tensors on {self.device}")
        else:
            self.ptr = stream.cuda_stream

    @property
    def device(self) -> torch.device:
        return torch.device("cuda", self.index)

    def launch(self, what: str, fn, *args) -> None:
        """fn(*args, stream) with the tensors' device as the current one."""
        if _current_device() == self.index:
            rc = fn(*args, self.ptr)
        else:
            with torch.cuda.device(self.index):
                rc = fn(*args, self.ptr)
        if rc != 0:
            _lib.check(rc, what)

    def empty(self, shape, dtype) -> torch.Tensor:
        if self.stream is None:
            return torch.empty(shape, dtype=dtype, device=self.device)
        with torch.cuda.stream(self.stream):
            return torch.empty(shape, dtype=dtype, device=self.device)

    def on(self, t: torch.Tensor, name: str) -> int:
        if t.get_device() != self.index:  # (-1: not on a device)
            raise ValueError(f"{name} is on {t.device}, expected {self.device}")
        return t.data_ptr()

    def rows(self, t: torch.Tensor, name: str, dim: Optional[int] = None, rows: Optional[int] = None,
             dtype: Optional[torch.dtype] = None, out: bool = False):
        """(pointer, rows, dim, row stride) of a tensor taken as rows of its last dimension."""
        if t.dtype not in _DTYPES if dtype is None else t.dtype is not dtype:
            raise ValueError(f"{name}: element type {t.dtype}" + (f", expected {dtype}" if dtype is not None else ""))
        shape = t.shape
        strides = t.stride()
        dims = len(shape)
        if dims == 2:
            n, d = shape
            stride, one = strides
        else:
            d = shape[-1] if dims else 0
            n, stride, one = t.numel() // max(d, 1), d, strides[-1] if dims else 1
            if not t.is_contiguous() and dims > 1:
                raise ValueError(f"{name}: more than two dimensions must be contiguous (stride {strides})")
        if not 0 < d <= _MAX_DIM or (dim is not None and d != dim):
            raise ValueError(f"{name}: rows of {dim if dim is not None else f'1 to {_MAX_DIM}'} elements expected, got "
                             f"shape {tuple(shape)}")
        if rows is not None and n != rows:
            raise ValueError(f"{name}: {rows} rows expected, got shape {tuple(shape)}")
        if one != 1 and d > 1:
            raise ValueError(f"{name}: the elements of a row must be consecutive (stride {strides})")
        if n <= 1:
            stride = d
        elif out and stride < d:
            raise ValueError(f"{name}: an output's rows must not overlap (stride {strides})")
        if t.get_device() != self.index:
            self.on(t, name)
        return t.data_ptr(), n, d, stride

    def vector(self, t: Optional[torch.Tensor], name: str, n: int, dtype: torch.dtype = _F32) -> Optional[int]:
        if t is None:
            return None
        if t.dtype is not dtype or t.numel() != n or not t.is_contiguous():
            raise ValueError(f"{name}: expected contiguous {dtype}[{n}], got {t.dtype}{tuple(t.shape)}")
        if t.get_device() != self.index:
            return self.on(t, name)  # (says so)
        return t.data_ptr()

    def ids(self, t: torch.Tensor, name: str):
        wide = t.dtype is torch.int64
        if not (wide or t.dtype is torch.int32) or not t.is_contiguous():
            raise ValueError(f"{name}: expected contiguous int32 or int64, got {t.dtype} (stride {t.stride()})")
        return self.on(t, name), int(wide), t.numel()


class _Workspace:
    """Device memory of a plan: allocated once, lent to one call at a time."""

    def __init__(self, nbytes: int, device):
        if nbytes == 0:
            raise ValueError("no call takes such sizes: too many tokens or rows, or rows too long")
        self.bytes = nbytes
        self.tensor = torch.empty(nbytes, dtype=torch.uint8, device=device)
        self.device = self.tensor.device
        self.ptr = self.tensor.data_ptr()
        self._home = torch.cuda.current_stream(self.device).cuda_stream

    def lend(self, call: _Call) -> int:
        if call.index != self.device.index:
            raise ValueError(f"the plan is on {self.device}, the tensors on {call.device}")
        if call.ptr != self._home:  # used away from the stream it was allocated on: not reused before that work is done
            self.tensor.record_stream(call.stream if call.stream is not None
                                      else torch.cuda.current_stream(call.index))
        return self.ptr


def embed(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, out: Optional[torch.Tensor] = None,
          out_dtype: Optional[torch.dtype] = None, stream=None) -> torch.Tensor:
    """Embedding lookup: out[..., :] = scale * table[ids, :], rounded once to out's type (default: the table's).  An id
    outside [0, rows) names no row (padding): a row of zeros."""
    call = _Call(table, stream)
    if table.dim() != 2:
        raise ValueError(f"table: expected [rows, dim], got shape {tuple(table.shape)}")
    tp, rows, dim, tstride = call.rows(table, "table")
    ip, ids64, n = call.ids(ids, "ids")
    if out_dtype is not None and out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype: element type {out_dtype}")
    if out is None:
        out = call.empty((*ids.shape, dim), out_dtype if out_dtype is not None else table.dtype)
    op, _, _, ostride = call.rows(out, "out", dim, n, out_dtype, out=True)
    call.launch("omr_embed", _lib.load().omr_embed, tp, _DTYPES[table.dtype], rows, dim, tstride, ip, ids64, n, scale, op,
                _DTYPES[out.dtype], ostride)
    return out


class EmbedGradPlan:
    """The embedding table's fp32 gradient by sorted tokens, for at most max_tokens tokens a call."""

    def __init__(self, max_tokens: int, num_rows: int, dim: int, device="cuda"):
        _sizes(max_tokens, num_rows, dim)
        self.max_tokens, self.num_rows, self.dim = max_tokens, num_rows, dim
        self.workspace = _Workspace(_lib.load().omr_embed_grad_workspace_bytes(max_tokens, num_rows, dim), device)

    def run(self, grad_out: torch.Tensor, ids: torch.Tensor, grad_table: Optional[torch.Tensor] = None,
            scale: float = 1.0, accumulate: bool = False, stream=None) -> torch.Tensor:
        """grad_table[v, :] = scale * (sum of grad_out's rows whose id is v, in token order), every row of it, or added
        to the rows that tokens name (accumulate).  Ids outside [0, rows) contribute nothing."""
        call = _Call(grad_out, stream)
        ip, ids64, n = call.ids(ids, "ids")
        if n > self.max_tokens:
            raise ValueError(f"{n} tokens, the plan is for {self.max_tokens}")
        gp, _, _, gstride = call.rows(grad_out, "grad_out", self.dim, n)
        if grad_table is None:
            if accumulate:
                raise ValueError("accumulate needs a grad_table")
            grad_table = call.empty((self.num_rows, self.dim), torch.float32)
        tp, _, _, tstride = call.rows(grad_table, "grad_table", self.dim, self.num_rows, torch.float32, out=True)
        call.launch("omr_embed_grad_f32", _lib.load().omr_embed_grad_f32, gp, _DTYPES[grad_out.dtype], gstride, ip, ids64,
                    n, self.num_rows, self.dim, scale, tp, tstride, int(accumulate), self.workspace.lend(call),
                    self.workspace.bytes)
        return grad_table


@dataclass
class LayerNormResult:
    out: torch.Tensor
    mean: torch.Tensor  # fp32, one a row
    rstd: torch.Tensor


@dataclass
class LayerNormGrads:
    grad_x: torch.Tensor
    grad_weight: Optional[torch.Tensor]  # fp32 [dim]
    grad_bias: Optional[torch.Tensor]


def _param(call: _Call, t: Optional[torch.Tensor], name: str, x: torch.Tensor, dim: int):
    if t is None:
        return None
    dtype = t.dtype
    if dtype is not _F32 and dtype is not x.dtype:
        raise ValueError(f"{name}: expected fp32 or {x.dtype}, got {dtype}")
    return call.vector(t, name, dim, dtype)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, out: Optional[torch.Tensor] = None, mean: Optional[torch.Tensor] = None,
               rstd: Optional[torch.Tensor] = None, stream=None) -> LayerNormResult:
    """Layer norm over the last dimension; out may be x.  mean and rstd (fp32, one a row) are what the gradient takes."""
    call = _Call(x, stream)
    xp, n, dim, xstride = call.rows(x, "x")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("weight and bias must have one element type")
    wp, bp = _param(call, weight, "weight", x, dim), _param(call, bias, "bias", x, dim)
    pdt = weight.dtype if weight is not None else bias.dtype if bias is not None else torch.float32
    if out is None:
        out = call.empty(x.shape, x.dtype)
    op, _, _, ostride = call.rows(out, "out", dim, n, x.dtype, out=True)
    if mean is None:
        mean = call.empty(x.shape[:-1], torch.float32)
    if rstd is None:
        rstd = call.empty(x.shape[:-1], torch.float32)
    call.launch("omr_layer_norm", _lib.load().omr_layer_norm, xp, _DTYPES[x.dtype], n, dim, xstride, wp, bp, _DTYPES[pdt],
                eps, op, ostride, call.vector(mean, "mean", n), call.vector(rstd, "rstd", n))
    return LayerNormResult(out, mean, rstd)


class LayerNormGradPlan:
    """The layer norm's backward pass, with the reduction of the weight's and bias's gradients, for at most max_rows
    rows a call."""

    def __init__(self, max_rows: int, dim: int, device="cuda"):
        _sizes(max_rows, 0, dim)
        self.max_rows, self.dim = max_rows, dim
        self.workspace = _Workspace(_lib.load().omr_layer_norm_grad_workspace_bytes(max_rows, dim), device)

    def run(self, grad_out: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
            weight: Optional[torch.Tensor] = None, grad_x: Optional[torch.Tensor] = None,
            grad_weight: Optional[torch.Tensor] = None, grad_bias: Optional[torch.Tensor] = None,
            accumulate: bool = False, params: bool = True, stream=None) -> LayerNormGrads:
        """grad_x (may be grad_out or x), and the fp32 gradients of weight and bias, written or added to what is there
        (accumulate).  params=False: grad_x alone."""
        call = _Call(x, stream)
        xp, n, dim, xstride = call.rows(x, "x", self.dim)
        if n > self.max_rows:
            raise ValueError(f"{n} rows, the plan is for {self.max_rows}")
        gp, _, _, gstride = call.rows(grad_out, "grad_out", dim, n, x.dtype)
        wp = _param(call, weight, "weight", x, dim)
        pdt = weight.dtype if weight is not None else torch.float32
        if grad_x is None:
            grad_x = call.empty(x.shape, x.dtype)
        op, _, _, ostride = call.rows(grad_x, "grad_x", dim, n, x.dtype, out=True)
        if not params:
            if grad_weight is not None or grad_bias is not None:
                raise ValueError("params=False takes no grad_weight or grad_bias")
        elif accumulate:
            if grad_weight is None and grad_bias is None:
                raise ValueError("accumulate needs a grad_weight or a grad_bias")
        else:
            grad_weight = grad_weight if grad_weight is not None else call.empty((dim,), torch.float32)
            grad_bias = grad_bias if grad_bias is not None else call.empty((dim,), torch.float32)
        call.launch("omr_layer_norm_grad", _lib.load().omr_layer_norm_grad, gp, gstride, xp, _DTYPES[x.dtype], n, dim,
                    xstride, call.vector(mean, "mean", n), call.vector(rstd, "rstd", n), wp, _DTYPES[pdt], op, ostride,
                    call.vector(grad_weight, "grad_weight", dim), call.vector(grad_bias, "grad_bias", dim),
                    int(accumulate), self.workspace.lend(call), self.workspace.bytes)
        return LayerNormGrads(grad_x, grad_weight, grad_bias)


class VocabLossPlan:
    """Softmax cross entropy of hidden [tokens, dim] against the output layer's weight [vocab, dim] (bf16 or fp16),
    forward and backward, without keeping the logits, for at most max_tokens tokens a call.  The backward pass holds the
    logits' gradients in `dtype`, whatever grad_weight's type is.

    pack: room to lay rows out again that are not whole 16-byte pieces (implied by a dim that is no multiple of 8).
    grads=False: forward only."""

    def __init__(self, max_tokens: int, vocab: int, dim: int, dtype: torch.dtype = torch.bfloat16, device="cuda",
                 grads: bool = True, pack: bool = False):
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype: bfloat16 or float16, got {dtype}")
        _sizes(max_tokens, vocab, dim, least=1)
        self.max_tokens, self.vocab, self.dim, self.dtype, self.grads = max_tokens, vocab, dim, dtype, grads
        self.workspace = _Workspace(_lib.load().omr_vocab_loss_workspace_bytes(max_tokens, vocab, dim, int(pack),
                                                                               int(grads)), device)

    def _inputs(self, call: _Call, hidden, weight, targets):
        hp, n, _, hstride = call.rows(hidden, "hidden", self.dim, None, self.dtype)
        wp, _, _, wstride = call.rows(weight, "weight", self.dim, self.vocab, self.dtype)
        tp, t64, nt = call.ids(targets, "targets")
        if nt != n:
            raise ValueError(f"targets: {n} expected, got shape {tuple(targets.shape)}")
        if n > self.max_tokens:
            raise ValueError(f"{n} tokens, the plan is for {self.max_tokens}")
        return (hp, hstride, wp, wstride, _DTYPES[self.dtype], n, self.vocab, self.dim, tp, t64), n

    def forward(self, hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                loss: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None, stream=None):
        """(loss, lse), fp32, one a token: loss = lse - logit of the target; 0 where the target names no row."""
        call = _Call(hidden, stream)
        args, n = self._inputs(call, hidden, weight, targets)
        if loss is None:
            loss = call.empty(targets.shape, torch.float32)
        if lse is None:
            lse = call.empty(targets.shape, torch.float32)
        call.launch("omr_vocab_loss", _lib.load().omr_vocab_loss, *args, call.vector(loss, "loss", n),
                    call.vector(lse, "lse", n), self.workspace.lend(call), self.workspace.bytes)
        return loss, lse

    def backward(self, hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor,
                 grad_loss: torch.Tensor, grad_hidden: Optional[torch.Tensor] = None,
                 grad_weight: Optional[torch.Tensor] = None, accumulate: bool = False, need_hidden: bool = True,
                 need_weight: bool = True, stream=None):
        """(grad_hidden, grad_weight) for grad_loss (fp32, one a token, or one for all, which in fp16 saves a pass over
        hidden).  grad_weight is fp32 or of the weight's type (default), written or added to (accumulate); need_hidden /
        need_weight=False leave one out."""
        if not self.grads:
            raise ValueError("the plan was made with grads=False")
        call = _Call(hidden, stream)
        args, n = self._inputs(call, hidden, weight, targets)
        if grad_loss.dtype != torch.float32 or grad_loss.numel() not in (n, 1):
            raise ValueError(f"grad_loss: fp32, {n} or one, got {grad_loss.dtype}{tuple(grad_loss.shape)}")
        if grad_loss.numel() == 1 or all(s == 0 for s in grad_loss.stride()):
            gstride = 0  # (also the gradient of a sum: one value, expanded)
        elif grad_loss.is_contiguous():
            gstride = 1
        else:
            raise ValueError(f"grad_loss must be contiguous or one value (stride {grad_loss.stride()})")
        hp = wp = None
        hstride = wstride = self.dim
        if need_hidden:
            if grad_hidden is None:
                grad_hidden = call.empty(hidden.shape, self.dtype)
            hp, _, _, hstride = call.rows(grad_hidden, "grad_hidden", self.dim, n, self.dtype, out=True)
        elif grad_hidden is not None:
            raise ValueError("need_hidden=False takes no grad_hidden")
        if need_weight:
            if grad_weight is None:
                if accumulate:
                    raise ValueError("accumulate needs a grad_weight")
                grad_weight = call.empty(weight.shape, self.dtype)
            if grad_weight.dtype not in (torch.float32, self.dtype):
                raise ValueError(f"grad_weight: fp32 or {self.dtype}, got {grad_weight.dtype}")
            wp, _, _, wstride = call.rows(grad_weight, "grad_weight", self.dim, self.vocab, out=True)
        elif grad_weight is not None or accumulate:
            raise ValueError("need_weight=False takes no grad_weight")
        call.launch("omr_vocab_loss_grad", _lib.load().omr_vocab_loss_grad, *args, call.vector(lse, "lse", n),
                    call.on(grad_loss, "grad_loss"), gstride, hp, hstride, wp,
                    _DTYPES[grad_weight.dtype] if wp is not None else 0, wstride, int(accumulate),
                    self.workspace.lend(call), self.workspace.bytes)
        return grad_hidden, grad_weight


# ------------------------------------------------------------------ host-resident end-to-end path

class HostPlan:
    """omr_host_plan: H2D -> in-place scan + aggregate -> D2H over row chunks on three HIP streams, for a
    gradient that starts and ends in pinned host memory (the reference's registered region)."""

    def __init__(self, layout: Layout, chunk_rows: int = 512):
        self.layout = layout
        self._p = ctypes.c_void_p()
        rc = _lib.load().omr_host_plan_create(layout.n, layout.block_size, layout.num_lanes, layout.num_threads,
                                              chunk_rows, ctypes.byref(self._p))
        if rc != 0:
            raise _lib.OmrError(f"omr_host_plan_create rc={rc}: {_lib.load().omr_host_last_error().decode()}")

    def run(self, host_buf: torch.Tensor, flags: Optional[torch.Tensor] = None,
            next_offsets: Optional[torch.Tensor] = None, zero_copy: bool = False) -> float:
        """zero_copy: the single-pass kernel reads and writes the pinned buffer in place over PCIe instead of
        staging it through HBM (omr_host_scan_sum_zero_copy_f32)."""
        L = self.layout
        for t, n, dt in ((host_buf, L.n, torch.float32), (flags, L.nb, torch.int32),
                         (next_offsets, L.nb, torch.int32)):
            if t is not None and (t.is_cuda or t.dtype != dt or t.numel() != n or not t.is_contiguous()):
                raise ValueError("host tensors must be contiguous CPU tensors of the layout's size")
        secs = ctypes.c_double()
        lib = _lib.load()
        fn = lib.omr_host_scan_sum_zero_copy_f32 if zero_copy else lib.omr_host_scan_sum_f32
        rc = fn(self._p, host_buf.data_ptr(), flags.data_ptr() if flags is not None else None,
                next_offsets.data_ptr() if next_offsets is not None else None, ctypes.byref(secs))
        if rc != 0:
            raise _lib.OmrError(f"omr_host_scan_sum{'_zero_copy' if zero_copy else ''}_f32 rc={rc}: "
                                f"{lib.omr_host_last_error().decode()}")
        return secs.value

    def close(self):
        if self._p:
            _lib.load().omr_host_plan_destroy(self._p)
            self._p = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ------------------------------------------------------------------ message-level round (wire format)

class _DeviceView:
    """A device buffer owned by the library, exposed to torch through __cuda_array_interface__ (no copy)."""

    def __init__(self, ptr: int, shape, typestr: str):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (ptr, False),
                                         "version": 3, "strides": None}


class MessageRound:
    """The round as the reference's messages (include/omr.h omr_msg_*): m workers on one device, every worker
    message and aggregator reply in the wire format of common.cc:399-443, results written in place."""

    def __init__(self, layout: Layout, m: int, device="cuda"):
        lib = _lib.load()
        self.layout, self.m, self.device = layout, m, torch.device(device)
        self._p = ctypes.c_void_p()
        _lib.check(lib.omr_msg_plan_create(layout.n, layout.block_size, layout.num_lanes, layout.num_threads, m,
                                           ctypes.byref(self._p)), "omr_msg_plan_create")

    def run(self, bufs: Sequence[torch.Tensor], outs: Optional[Sequence[torch.Tensor]] = None, stream=None) -> int:
        L = self.layout
        outs = list(bufs) if outs is None else list(outs)
        if len(bufs) != self.m or len(outs) != self.m:
            raise ValueError(f"expected {self.m} worker buffers")
        for i, (b, o) in enumerate(zip(bufs, outs)):
            _check_f32(b, L.n, f"bufs[{i}]")
            _check_f32(o, L.n, f"outs[{i}]")
        maxr = ctypes.c_uint32()
        _lib.check(_lib.load().omr_msg_round_f32(self._p, _ptr_array(bufs), _ptr_array(outs), ctypes.byref(maxr),
                                                 _stream(stream)), "omr_msg_round_f32")
        return maxr.value

    def logs(self, worker: int) -> dict:
        """Copies of the wire logs: messages / replies [G, cap, 2*MESSAGE_SIZE] f32, imm / reply_imm [G, cap]
        (uint32 bits in int32), rounds [G]."""
        msg, imm, rep, rimm, rnd = (ctypes.c_void_p() for _ in range(5))
        cap = ctypes.c_uint32()
        _lib.check(_lib.load().omr_msg_logs(self._p, worker, ctypes.byref(msg), ctypes.byref(imm), ctypes.byref(rep),
                                            ctypes.byref(rimm), ctypes.byref(rnd), ctypes.byref(cap)), "omr_msg_logs")
        G, c, W = self.layout.num_threads * NUM_SLOTS, cap.value, 2 * MESSAGE_SIZE
        torch.cuda.synchronize(self.device)
        view = (lambda p, shape, t: torch.as_tensor(_DeviceView(p.value, shape, t), device=self.device).clone())
        return {"messages": view(msg, (G, c, W), "<f4"), "imm": view(imm, (G, c), "<i4"),
                "replies": view(rep, (G, c, W), "<f4"), "reply_imm": view(rimm, (G, c), "<i4"),
                "rounds": view(rnd, (G,), "<i4"), "cap": c}

    def close(self):
        if self._p:
            _lib.load().omr_msg_plan_destroy(self._p)
            self._p = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 (interpreter shutdown)
            pass
