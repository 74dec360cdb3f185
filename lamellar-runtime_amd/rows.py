"""RowArray: a distributed table whose batched ops move whole rows.

The element arrays (array.py) gather, add and store single elements; a table that a model looks up
by token or a serving process keeps per cached position is used a row at a time. A RowArray has
`rows` rows of `row_len` elements, its rows distributed over the PEs by the layouts of the element
arrays (Block or Cyclic), each row whole on its owner's GPU. The element types are f32, f16 and
bf16, and two 8-bit codes (i8, e4m3) with one f32 scale per `group` elements of a row.

  batch_load_rows(index, scale)        scale * row, as f32 / f16 / bf16: an embedding lookup, or an
                                       8-bit cache read back
  batch_add_rows(index, vals, scale)   row += scale * the sum of the batch's values of that row: the
                                       lookup's gradient (or, with scale = -rate, its update)
  batch_store_rows(index, vals)        row = vals, quantised when the array holds codes

Sums and scaling are in f32 and round once to the array's (or the result's) type. The outcome of a
batch depends on its arguments alone: the records of a row are added in an order fixed by the
indices, and of several records stored to one row the last one of the batch stands, on the highest
PE that names the row when several do.

Indices are integers of any shape: torch tensors (int32 and int64 are read as they are), numpy arrays,
lists, one number. Values are torch tensors of f32, f16 or bf16; host sequences are taken as f32. A
batch has at most 2^25 records and 2^36 elements, at a PE that sends them and at one that gets them.

A lookup is not recorded by autograd: its gradient is the caller's batch_add_rows. Batches write a tensor
that the caller gave (from_tensor, out) in place and raise its version, as torch's in-place operations do.

Handles are lazy, as the element arrays': spawn() enqueues the batch on torch's current stream,
value() gives its result for work ordered after it on that stream, block() waits and raises what the
batch found wrong. A spawned batch reads its inputs in stream order, so later work on the stream may
change them; batches that write one array are ordered by the caller if they use several streams. At one
PE a batch may be captured into a graph; each graph has its own workspace. With several PEs every batch is collective: all PEs issue the same sequence of
batches (an empty one where a PE has nothing to send).
"""
from __future__ import annotations

import ctypes
import numbers

import numpy as np
import torch
import torch.distributed as dist

from . import _capi
from .array import _Handle
from .engine import _FORCE_EXCHANGE, Owned, index_input
from .kernels import LamellarError, check
from .types import DTYPES, Distribution, LmrStatus


class RowType:
    """One element type of a row: lmr_row_type_t code, torch dtype, whether it is an 8-bit code."""

    def __init__(self, name, code, torch_dtype, largest=None):
        self.name, self.code, self.torch, self.largest = name, code, torch_dtype, largest
        self.is_code = largest is not None

    def __repr__(self):
        return f"RowType({self.name})"


ROW_TYPES = {t.name: t for t in (
    RowType("f32", 0, torch.float32), RowType("f16", 1, torch.float16), RowType("bf16", 2, torch.bfloat16),
    RowType("i8", 3, torch.int8, 127.0), RowType("e4m3", 4, torch.float8_e4m3fn, 448.0))}
_BY_TORCH = {t.torch: t for t in ROW_TYPES.values()}
_VALUES = {k: t for t in ROW_TYPES.values() if not t.is_code for k in (t.name, t.torch)}
MAX_ROW_LEN = 1 << 18                     # LMR_ROW_MAX_LEN
MAX_ROWS = 0xFFFFFFF0                     # LMR_ROWS_MAX, of one PE
MAX_BATCH = 1 << 25                       # LMR_ROW_MAX_BATCH, records that one PE sends or gets
MAX_VALUES = 1 << 36                      # LMR_ROW_MAX_VALUES, their elements
SCAN = 1024                               # LMR_ROW_SCAN: stores of more records use claims
_INT = (torch.int64, torch.int32)


def row_type_of(t) -> RowType:
    r = t if isinstance(t, RowType) else ROW_TYPES.get(t) if isinstance(t, str) else _BY_TORCH.get(t)
    if r is None:
        raise LamellarError(LmrStatus.UNSUPPORTED, f"no row element type {t!r} ({', '.join(ROW_TYPES)})")
    return r


def _value_type(t) -> RowType:
    r = _VALUES.get(t) if isinstance(t, (str, torch.dtype)) else row_type_of(t)
    if r is None or r.is_code:
        raise LamellarError(LmrStatus.UNSUPPORTED, f"values are f32, f16 or bf16, not {t}")
    return r


def _again(e):
    """The same exception without its traceback, which would hold the batch's tensors."""
    c = type(e).__new__(type(e), *e.args)
    c.__dict__.update(e.__dict__)
    return c


class RowsHandle(_Handle):
    """A batch of rows: spawn() enqueues it, value() its result without waiting, block() the result
    once the device has finished (raising its errors)."""

    def __init__(self, array, launch):
        self._array, self._launch = array, launch
        self._res = self._error = None
        self._launched = False

    def spawn(self):
        if not self._launched:
            self._launched = True
            launch, self._launch = self._launch, None      # its tensors live as long as the stream needs them
            try:
                self._res = launch()
            except BaseException as e:
                self._error = _again(e)
                raise
        elif self._error is not None:                      # it has no result, however often it is asked
            raise _again(self._error)
        return self

    def value(self):
        return self.spawn()._res

    _value = value


class _Table:
    """lmr_rows_t over tensors that the caller keeps alive."""

    def __init__(self, data, scales, claims, rows, row_len, rtype, group):
        self.data, self.scales, self.claims = data, scales, claims
        self.rows, self.row_len, self.rtype, self.group = rows, row_len, rtype, group
        self.c = _capi.lmr_rows_t(data.data_ptr(), scales.data_ptr() if scales is not None else None,
                                  claims.data_ptr() if claims is not None else None, rows, row_len, rtype.code,
                                  group or 0)
        self.ptr = ctypes.addressof(self.c)
        self.lo = data.data_ptr()
        self.hi = self.lo + data.numel() * data.element_size()
        self.scales_lo = scales.data_ptr() if scales is not None else 0
        self.scales_hi = self.scales_lo + scales.numel() * 4 if scales is not None else 0

    def overlaps(self, t, n):
        """Whether t (n rows of row_len) reaches into the table's rows or scales."""
        if n == 0:
            return False
        lo = t.data_ptr()
        hi = lo + ((n - 1) * t.stride(0) + self.row_len) * t.element_size()
        return lo < self.hi and self.lo < hi or lo < self.scales_hi and self.scales_lo < hi


class RowArray:
    """A table of `rows` x `row_len` elements distributed by rows; zero-filled when made."""

    def __init__(self, team, rows, row_len, distribution=Distribution.Block, dtype="f32", group=None):
        self._set_up(team, int(rows), int(row_len), distribution, row_type_of(dtype), group)
        n, dev = self.num_rows_local(), team.kernels.device
        data = torch.zeros(n, self.row_len, dtype=torch.uint8 if self.rtype.is_code else self.rtype.torch, device=dev)
        scales = torch.zeros(n, self.row_len // self.group, device=dev) if self.rtype.is_code else None
        self._adopt(data, scales)

    @classmethod
    def new(cls, team, rows, row_len, distribution=Distribution.Block, dtype="f32", group=None):
        """As the element arrays' `new`: a handle whose block() gives the array."""
        class _New:
            def block(_self):
                return cls(team, rows, row_len, distribution, dtype, group)
        return _New()

    @classmethod
    def from_tensor(cls, team, data, scales=None, dtype=None, rows=None, distribution=Distribution.Block):
        """An array over memory that the caller already has: `data`, this PE's rows (2-D, contiguous,
        on the team's device), shared, not copied. 8-bit codes come as int8, float8_e4m3fn, or uint8
        with `dtype`, and with `scales` (rows x groups, f32). `rows`: the rows of all PEs (the default:
        this PE's, at one PE)."""
        if not isinstance(data, torch.Tensor) or data.dim() != 2 or not data.is_contiguous() or data.is_neg():
            raise LamellarError(LmrStatus.INVALID, "from_tensor takes a contiguous 2-D tensor of rows")
        rt = row_type_of(data.dtype if dtype is None else dtype)
        if data.dtype != rt.torch and not (rt.is_code and data.dtype == torch.uint8):
            raise LamellarError(LmrStatus.INVALID, f"{data.dtype} holds no {rt.name}")
        if _device_of(data) != _device_of(team.kernels):
            raise LamellarError(LmrStatus.INVALID, f"the rows are on {data.device}, the team on {team.kernels.device}")
        group = None
        if rt.is_code:
            if not isinstance(scales, torch.Tensor) or scales.dim() != 2 or scales.dtype != torch.float32 or \
                    not scales.is_contiguous() or scales.device != data.device or scales.shape[0] != data.shape[0] or \
                    scales.shape[1] == 0 or data.shape[1] % scales.shape[1]:
                raise LamellarError(LmrStatus.INVALID, "8-bit rows need contiguous f32 scales, rows x groups, beside them")
            group = data.shape[1] // scales.shape[1]
        elif scales is not None:
            raise LamellarError(LmrStatus.INVALID, f"{rt.name} rows have no scales")
        if rows is None:
            if team.num_pes() > 1:
                raise LamellarError(LmrStatus.INVALID, "with several PEs from_tensor needs the rows of all of them")
            rows = data.shape[0]
        a = object.__new__(cls)
        a._set_up(team, int(rows), int(data.shape[1]), distribution, rt, group)
        if a.num_rows_local() != data.shape[0]:
            raise LamellarError(LmrStatus.LENGTH, f"{data.shape[0]} rows here, {a.num_rows_local()} by the layout")
        a._adopt(data, scales)
        return a

    def _set_up(self, team, rows, row_len, distribution, rt, group):
        if rows < 1 or row_len < 1 or row_len > MAX_ROW_LEN:
            raise LamellarError(LmrStatus.INVALID, f"a row array of {rows} x {row_len} (row_len: 1 to {MAX_ROW_LEN})")
        if rt.is_code:
            group = row_len if group is None else int(group)
            if group < 1 or row_len % group:
                raise LamellarError(LmrStatus.INVALID, f"groups of {group} do not divide rows of {row_len}")
        elif group is not None:
            raise LamellarError(LmrStatus.INVALID, f"{rt.name} rows have no groups")
        self.team, self.rtype, self.row_len, self.group = team, rt, row_len, group
        self._out_type = ROW_TYPES["bf16"] if rt.is_code else rt
        self._distributed = team.num_pes() > 1 or _FORCE_EXCHANGE
        self.layout = _capi.lmr_layout_t()
        check(_capi.lib().lmr_layout_new(ctypes.byref(self.layout), rows, team.num_pes(), team.my_pe(),
                                         int(distribution)), "lmr_layout_new")
        if self.num_rows_local() > MAX_ROWS:
            raise LamellarError(LmrStatus.INVALID, f"{self.num_rows_local()} rows on one PE (at most {MAX_ROWS})")

    def _adopt(self, data, scales):
        self._table = _Table(data.detach(), scales, None, self.num_rows_local(), self.row_len, self.rtype, self.group)
        self._streams = set()             # streams whose work may still use the tensors when the array is dropped
        self.team.barrier()

    # ---- layout ----
    def num_rows(self):
        return int(self.layout.size)

    def __len__(self):
        return self.num_rows()

    @property
    def dtype(self):
        return self.rtype.name

    def num_pes(self):
        return self.team.num_pes()

    def my_pe(self):
        return self.team.my_pe()

    def num_rows_local(self):
        return int(_capi.lib().lmr_num_elems_pe(ctypes.byref(self.layout), self.team.my_pe()))

    def local_rows(self):
        """This PE's rows, a tensor over the array's own memory (8-bit rows: their codes)."""
        return self._table.data.view(self.rtype.torch)

    def local_scales(self):
        """This PE's scales (rows x groups), a tensor over the array's own memory; None without codes."""
        return self._table.scales

    def barrier(self):
        self.team.barrier()

    def wait_all(self):
        self.team.kernels.synchronize()
        self.team.kernels.check_errors()

    # ---- batched ops ----
    def batch_load_rows(self, index, scale=1.0, out_dtype=None, pad=None, out=None):
        """scale * row for every index, in input order: index.shape + (row_len,). Type: `out_dtype`
        (the array's own by default; bf16 for 8-bit rows). An index equal to `pad` gives zeros. `out`:
        a tensor to write instead of a new one; its rows may be strided."""
        scale, pad = _scale(scale), _pad(pad)
        if out is not None:
            if not isinstance(out, torch.Tensor):
                raise LamellarError(LmrStatus.INVALID, f"out is a tensor, not {type(out).__name__}")
            rt = _value_type(out.dtype)
            if out_dtype is not None and _value_type(out_dtype) is not rt:
                raise LamellarError(LmrStatus.INVALID, f"out is {rt.name}, not {out_dtype}")
        else:
            rt = self._out_type if out_dtype is None else _value_type(out_dtype)
        return RowsHandle(self, lambda: self._load(index, scale, rt, pad, out))

    def batch_add_rows(self, index, vals, scale=1.0, pad=None):
        """row += scale * (sum of the values that name it). vals: index.shape + (row_len,), or one row
        for every index. 8-bit rows refuse it: a sum of codes has no code."""
        if self.rtype.is_code:
            raise LamellarError(LmrStatus.UNSUPPORTED, f"batch_add_rows on {self.rtype.name} rows")
        scale, pad = _scale(scale), _pad(pad)
        return RowsHandle(self, lambda: self._write(index, vals, scale, pad, True))

    def batch_store_rows(self, index, vals, pad=None):
        """row = vals, rounded (f16, bf16) or quantised by groups (i8, e4m3) as it is stored."""
        pad = _pad(pad)
        return RowsHandle(self, lambda: self._write(index, vals, 1.0, pad, False))

    # ---- one PE's part, and the exchange ----
    def _on_stream(self, k):
        """The current stream, which will use the array's memory: its reuse waits for that stream."""
        s = k.stream_id()
        if s not in self._streams:
            self._streams.add(s)
            k.keep_for_stream([t for t in (self._table.data, self._table.scales, self._table.claims) if t is not None])
        return s

    def _claims(self, k, stream):
        """The table with the words that stores of many records need: made once. Inside a capture the graph
        gets its own (a replay clears them first, and may come when the array is gone)."""
        t = self._table
        capturing = k.capturing()
        if t.claims is not None and not capturing:
            return t
        claims = torch.zeros(t.rows, dtype=torch.int32, device=k.device)
        if capturing:
            return _Table(t.data, t.scales, claims, t.rows, t.row_len, t.rtype, t.group)
        t.claims, t.c.claims = claims, claims.data_ptr()
        self._streams = {stream}          # other streams are told of it when they next use the array
        return t

    def _index(self, k, index, pad):
        """(1-D index tensor of 4 or 8 bytes, the shape it had)."""
        if isinstance(index, Owned):
            index = index.value
        if isinstance(index, torch.Tensor):
            shape = index.shape
            if index.dtype in _INT and index.device == k.device:
                if len(shape) != 1 or not index.is_contiguous():
                    index = index.reshape(-1).contiguous()
                return index, shape
            if index.dtype.is_floating_point or index.dtype.is_complex or index.dtype == torch.bool:
                raise LamellarError(LmrStatus.INVALID, f"row indices are integers, not {index.dtype}")
            unsigned = index.dtype == torch.uint64
            index = index_input(k, index)[1]
            return _no_wrap(index, pad) if unsigned else index, shape
        if isinstance(index, numbers.Integral) and type(index) is not bool:
            i = int(index)
            return torch.tensor([i if _fits(i) else _nowhere(pad)], dtype=torch.int64, device=k.device), torch.Size([])
        a = np.asarray(index)
        if a.size and a.dtype.kind not in "iu":
            raise LamellarError(LmrStatus.INVALID, f"row indices are integers below 2^63, not {a.dtype}")
        i = index_input(k, a.reshape(-1))[1]
        return _no_wrap(i, pad) if a.dtype == np.uint64 else i, torch.Size(a.shape)

    def _values(self, k, vals, n):
        """(n x row_len tensor whose rows are contiguous, their type)."""
        if isinstance(vals, Owned):
            vals = vals.value
        if not isinstance(vals, torch.Tensor):
            vals = torch.from_numpy(np.ascontiguousarray(np.asarray(vals), dtype=np.float32))
        rt = _value_type(vals.dtype)
        if vals.is_neg():
            vals = vals.resolve_neg()
        if vals.shape == (n, self.row_len) and vals.device == k.device and vals.stride(1) == 1 and \
                vals.stride(0) >= self.row_len:
            if self._table.overlaps(vals, n):
                raise LamellarError(LmrStatus.INVALID, "the values lie in the array's own memory")
            return vals, rt
        if vals.dim() == 0 or vals.shape[-1] != self.row_len:
            raise LamellarError(LmrStatus.LENGTH, f"values of {tuple(vals.shape)} for rows of {self.row_len}")
        if vals.device != k.device:
            vals = vals.to(k.device)
        vals = vals.detach().reshape(-1, self.row_len)
        if vals.shape[0] != n:
            if vals.shape[0] != 1:
                raise LamellarError(LmrStatus.LENGTH, f"{n} indices vs {vals.shape[0]} rows of values")
            vals = vals.expand(n, self.row_len)
        if (self.row_len > 1 and vals.stride(1) != 1) or (n > 1 and 0 < vals.stride(0) < self.row_len):
            vals = vals.contiguous()
        if self._table.overlaps(vals, n):
            raise LamellarError(LmrStatus.INVALID, "the values lie in the array's own memory")
        return vals, rt

    def _load(self, index, scale, rt, pad, out):
        k = self.team.kernels
        idx, shape = self._index(k, index, pad)
        n, shape = idx.numel(), (*shape, self.row_len)
        alone = not self._distributed
        stride = self.row_len
        fresh = out is None
        if fresh:
            rows = out = torch.empty(shape, dtype=rt.torch, device=k.device)
            if len(shape) != 2:
                rows = out.view(n, self.row_len)
        else:
            rows = self._out_rows(k, out, shape, n)
            if n > 1:
                stride = rows.stride(0)
        stream = self._on_stream(k)
        if not alone:
            self._exchange_load(k, idx, scale, rt, pad, rows, n, stride)
        elif n:
            k.rows_load(self._table, idx, n, pad, scale, rows, rt.code, stride, stream)
        if not fresh:
            _written(out)
        return out

    def _out_rows(self, k, out, shape, n):
        if out.shape != shape:
            raise LamellarError(LmrStatus.LENGTH, f"out is {tuple(out.shape)}, the batch {shape}")
        if out.device != k.device:
            raise LamellarError(LmrStatus.INVALID, f"out is on {out.device}, the team on {k.device}")
        if n == 0:
            return out
        try:
            rows = out.detach().view(n, self.row_len)
        except RuntimeError:
            rows = None
        if rows is None or rows.is_neg() or (self.row_len > 1 and rows.stride(1) != 1) or (n > 1 and rows.stride(0) < self.row_len):
            raise LamellarError(LmrStatus.INVALID, "out's rows are not contiguous, evenly spaced and plain: strides "
                                                   f"{out.stride()}{', negated' if out.is_neg() else ''}")
        if self._table.overlaps(rows, n):
            raise LamellarError(LmrStatus.INVALID, "out lies in the array's own memory")
        return rows

    def _write(self, index, vals, scale, pad, add):
        k = self.team.kernels
        idx, _ = self._index(k, index, pad)
        n = idx.numel()
        vals, rt = self._values(k, vals, n)
        stream = self._on_stream(k)
        if self._distributed:
            idx, vals, pad = self._exchange_values(k, idx, vals, pad)
            n = idx.numel()
        if n == 0:
            return None
        stride = vals.stride(0) if n > 1 else self.row_len
        if add:
            table = self._table
            k.rows_add(table, idx, n, pad, scale, vals, rt.code, stride, stream)
        else:
            table = self._table if n <= SCAN else self._claims(k, stream)
            k.rows_store(table, idx, n, pad, vals, rt.code, stride, stream)
        _written(table.data)
        if table.scales is not None:
            _written(table.scales)
        return None

    # Records travel to their rows' owner in input order (the stable pack), sources one after the
    # other: the owner sees one batch in an order that every run repeats. The counts are read on the
    # host, so a batch over several PEs waits for its pack. Every PE gets the counts of all, so that a
    # batch too large for one of them is turned down by all of them, before its records travel.
    def _pack(self, k, idx, pad):
        gidx = idx.to(torch.int64)
        kept = None
        if pad is not None:
            kept = (gidx != pad).nonzero().reshape(-1)
            gidx = gidx[kept]
        n = int(gidx.numel())
        loc, _, pos, counts = k.pack(self.layout, gidx, n, None, DTYPES["u8"], 8)
        sent = [int(c) for c in counts.cpu().tolist()]
        every = _all_gather(self.team, [idx.numel(), *sent])
        for p in range(len(sent)):
            most = max(every[p][0], sum(e[1 + p] for e in every))
            if most > MAX_BATCH or most * self.row_len > MAX_VALUES:
                raise LamellarError(LmrStatus.INVALID, f"PE {p} would send or get {most} rows of {self.row_len} (at most "
                                                       f"{MAX_BATCH}, of {MAX_VALUES} elements)")
        got = [e[1 + self.team.my_pe()] for e in every]
        m = sum(sent)                                   # an index out of bounds is dropped there
        pos = pos[:m]
        loc = loc.view(torch.int64)[:m].view(-1, 1) if m else gidx[:0].view(0, 1)
        return _all_to_all(self.team, loc, sent, got).view(-1), (pos if kept is None else kept[pos]), sent, got

    def _exchange_load(self, k, idx, scale, rt, pad, rows, n, stride):
        mine, pos, sent, got = self._pack(k, idx, pad)
        reply = torch.empty(mine.numel(), self.row_len, dtype=rt.torch, device=k.device)
        if mine.numel():
            k.rows_load(self._table, mine, mine.numel(), None, scale, reply, rt.code, self.row_len, k.stream_id())
        reply = _all_to_all(self.team, reply, got, sent)
        if n == 0:
            return
        m = pos.numel()
        if stride == self.row_len:
            if m < n:
                rows.zero_()                            # pads, and what was out of bounds
            whole = _Table(rows, None, None, n, self.row_len, rt, None)
            if m:
                k.rows_store(whole, pos, m, None, reply, rt.code, self.row_len, k.stream_id())
            return
        # strided rows: a lookup in what came back, -1 for those that get zeros
        where = torch.empty(n, dtype=torch.int64, device=k.device) if m == n else torch.full((n,), -1, dtype=torch.int64, device=k.device)
        if m:
            k.scatter_results(torch.arange(m, device=k.device), pos if pos.dtype == torch.int32 else pos.to(torch.int32), m, 8, where)
        back = _Table(reply, None, None, m, self.row_len, rt, None)
        k.rows_load(back, where, n, -1, 1.0, rows, rt.code, stride, k.stream_id())

    def _exchange_values(self, k, idx, vals, pad):
        mine, pos, sent, got = self._pack(k, idx, pad)
        return mine, _all_to_all(self.team, vals.index_select(0, pos), sent, got), None


def _written(t):
    """Tells autograd that t's memory was changed: what a backward pass has saved of it is no longer good."""
    torch.autograd.graph.increment_version(t)


def _device_of(x):
    d = x.device
    return (d.type, d.index or 0)


def _scale(x):
    if type(x) is float:
        return x
    if not isinstance(x, numbers.Real) or type(x) is bool:
        raise LamellarError(LmrStatus.INVALID, f"scale is a number, not {type(x).__name__}")
    return float(x)


def _fits(i):
    return -(1 << 63) <= i < 1 << 63


def _pad(x):
    if x is None or type(x) is int and _fits(x):
        return x
    if not isinstance(x, numbers.Integral) or type(x) is bool or not _fits(int(x)):
        raise LamellarError(LmrStatus.INVALID, f"pad is an index, not {x!r}")
    return int(x)


def _nowhere(pad):
    """A number of 64 bits that is neither a row nor the pad."""
    return -(1 << 63) if pad != -(1 << 63) else 1 - (1 << 63)


def _no_wrap(i, pad):
    """Unsigned indices read as signed ones: those of 2^63 and more name no row, whatever they look like."""
    return torch.where(i < 0, _nowhere(pad), i)


def _all_gather(team, numbers_of_this):
    """Every PE's list of whole numbers, equally many from each, in PE order."""
    dev = team.kernels.device if dist.get_backend(team.group) == "nccl" else torch.device("cpu")
    mine = torch.tensor(numbers_of_this, dtype=torch.int64).to(dev)
    every = torch.empty(team.num_pes() * mine.numel(), dtype=torch.int64, device=dev)
    dist.all_gather_into_tensor(every, mine, group=team.group)
    return every.cpu().view(team.num_pes(), -1).tolist()


def _all_to_all(team, rows, sent, got):
    """rows (2-D, contiguous): sent[p] of them to PE p, got[p] from PE p, in PE order. On the device
    over RCCL; a host process group gets host tensors."""
    width = rows.shape[1]
    flat = rows.contiguous().view(torch.uint8) if rows.numel() else rows.new_empty(rows.shape[0], width * rows.element_size(), dtype=torch.uint8)
    if flat.shape[1] % 4 == 0:
        flat = flat.view(torch.int32) if flat.numel() else flat.new_empty(flat.shape[0], flat.shape[1] // 4, dtype=torch.int32)
    back = torch.empty(sum(got), flat.shape[1], dtype=flat.dtype, device=flat.device)
    if flat.is_cuda and dist.get_backend(team.group) != "nccl":
        host = torch.empty(back.shape, dtype=flat.dtype)
        dist.all_to_all_single(host, flat.cpu(), output_split_sizes=got, input_split_sizes=sent, group=team.group)
        back.copy_(host)
    else:
        dist.all_to_all_single(back, flat, output_split_sizes=got, input_split_sizes=sent, group=team.group)
    if back.numel():
        return back.view(rows.dtype)
    return back.new_empty(sum(got), width, dtype=rows.dtype)


__all__ = ["RowArray", "RowsHandle", "RowType", "ROW_TYPES", "row_type_of"]
