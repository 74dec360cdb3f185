"""RowArray without a GPU: what it refuses (Python and C entry points), and its exchange over two and
three PEs (gloo, CPU test double of the device kernels) against the plain forms of rowref.py."""
import ctypes
import os
import sys
import tempfile
import time
import warnings

import numpy as np
import pytest
import torch
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

from test_dist_gloo import CpuTestKernels  # noqa: E402


class CpuRowKernels(CpuTestKernels):
    """The row operators of one PE in plain torch, records one after the other."""

    def stream_id(self):
        return 0

    def keep_for_stream(self, tensors):
        pass

    def capturing(self):
        return False

    def pack(self, layout, gidx, n, vals, dt, iw, stable=True, want_pos=True):
        ok = (gidx >= 0) & (gidx < layout.size)          # out of bounds: reported and dropped
        if not bool(ok.all()):
            self.err |= 1
        kept = ok.nonzero().reshape(-1)
        loc, v, pos, counts = super().pack(layout, gidx[kept].contiguous(), int(kept.numel()), vals, dt, iw)
        return loc, v, kept.to(torch.int32)[pos.long()], counts

    def _live(self, table, idx, pad):
        out = []
        for t, i in enumerate(idx.tolist()):
            if i == pad:
                continue
            if not 0 <= i < table.rows:
                self.err |= 1
                continue
            out.append((t, i))
        return out

    def rows_load(self, table, idx, n, pad, scale, out, out_type, stride, stream):
        import rowref as ref
        out.zero_()
        for t, i in self._live(table, idx, pad):
            v = table.data[i]
            if table.rtype.is_code:
                v = ref.codes_f64(v, table.rtype.name).float() * table.scales[i].repeat_interleave(table.group)
            out[t] = (v.float() * scale).to(out.dtype)

    def rows_add(self, table, idx, n, pad, scale, vals, val_type, stride, stream):
        for t, i in self._live(table, idx, pad):
            table.data[i] = (table.data[i].float() + scale * vals[t].float()).to(table.data.dtype)

    def rows_store(self, table, idx, n, pad, vals, val_type, stride, stream):
        import rowref as ref
        for t, i in self._live(table, idx, pad):
            if table.rtype.is_code:
                table.data[i], table.scales[i] = (x[0] for x in ref.quantise(vals[t:t + 1], table.rtype.name, table.group))
            else:
                table.data[i] = vals[t].to(table.data.dtype)


@pytest.fixture(scope="module")
def team(lam):
    return lam.LamellarWorldBuilder().with_kernels(CpuRowKernels).build().team()


def refused(lam, status, f, *a, **k):
    with pytest.raises(lam.LamellarError) as e:
        f(*a, **k)
    assert e.value.status == status, e.value


INVALID, OOB, UNSUPPORTED, LENGTH = 1, 2, 5, 8


def test_refused_arrays(lam, team):
    R = lam.RowArray
    for rows, width in [(0, 4), (4, 0), (-1, 4), (4, (1 << 18) + 1)]:
        refused(lam, INVALID, R, team, rows, width)
    refused(lam, UNSUPPORTED, R, team, 4, 4, dtype="f64")
    refused(lam, UNSUPPORTED, R, team, 4, 4, dtype="u8")
    refused(lam, INVALID, R, team, 4, 10, dtype="i8", group=4)
    refused(lam, INVALID, R, team, 4, 10, dtype="e4m3", group=0)
    refused(lam, INVALID, R, team, 4, 10, dtype="bf16", group=5)
    F = R.from_tensor
    refused(lam, INVALID, F, team, torch.zeros(4))
    refused(lam, INVALID, F, team, torch.zeros(4, 6)[:, :3])
    refused(lam, INVALID, F, team, np.zeros((4, 6)))
    refused(lam, UNSUPPORTED, F, team, torch.zeros(4, 6, dtype=torch.float64))
    refused(lam, UNSUPPORTED, F, team, torch.zeros(4, 6, dtype=torch.uint8))          # codes of which type?
    refused(lam, INVALID, F, team, torch.zeros(4, 6), dtype="bf16")
    refused(lam, INVALID, F, team, torch.zeros(4, 6), scales=torch.ones(4, 1))
    codes = torch.zeros(4, 6, dtype=torch.int8)
    for s in (None, torch.ones(4), torch.ones(3, 2), torch.ones(4, 4), torch.ones(4, 2, dtype=torch.float64),
              torch.ones(4, 0), torch.ones(2, 4).t()):
        refused(lam, INVALID, F, team, codes, scales=s)
    refused(lam, LENGTH, F, team, torch.zeros(4, 6), rows=5)
    a = F(team, codes, scales=torch.ones(4, 2))
    assert (a.dtype, a.group, len(a), a.row_len) == ("i8", 3, 4, 6) and a.local_rows().data_ptr() == codes.data_ptr()
    assert R.new(team, 3, 5, dtype="e4m3").block().group == 5
    e = F(team, torch.ones(4, 6).to(torch.float8_e4m3fn), scales=torch.ones(4, 1))
    assert e.dtype == "e4m3" and e.batch_load_rows([1]).block().dtype == torch.bfloat16
    refused(lam, INVALID, R._set_up, object.__new__(R), team, 0xFFFFFFF1, 1, lam.Distribution.Block, lam.ROW_TYPES["i8"], 1)


def test_refused_batches(lam, team):
    a = lam.RowArray(team, 10, 6)
    c = lam.RowArray(team, 10, 6, dtype="i8", group=3)
    v = torch.ones(3, 6)
    for h in (lambda i, **k: a.batch_load_rows(i, **k).block(), lambda i, **k: a.batch_add_rows(i, v, **k).block(),
              lambda i, **k: c.batch_store_rows(i, v, **k).block()):
        refused(lam, INVALID, h, torch.ones(3))
        refused(lam, INVALID, h, [0.5, 1.0, 2.0])
        refused(lam, INVALID, h, torch.ones(3, dtype=torch.bool))
        refused(lam, INVALID, h, [0, 1, 2], pad=0.5)
        refused(lam, INVALID, h, [0, 1, 2], pad=1 << 63)
        refused(lam, OOB, h, [0, 10, 2])
        refused(lam, OOB, h, [0, -1, 2])
    a.local_rows().zero_()                               # (records within bounds beside those were applied)
    refused(lam, UNSUPPORTED, c.batch_add_rows, [0, 1, 2], v)
    refused(lam, INVALID, a.batch_load_rows, [0], scale="2")
    refused(lam, INVALID, a.batch_add_rows, [0], v, scale=torch.ones(1))
    refused(lam, UNSUPPORTED, a.batch_load_rows, [0], out_dtype="f64")
    refused(lam, UNSUPPORTED, a.batch_load_rows, [0], out_dtype="i8")
    refused(lam, UNSUPPORTED, a.batch_load_rows, [0], out=torch.empty(1, 6, dtype=torch.int32))
    refused(lam, INVALID, a.batch_load_rows, [0], out=torch.empty(1, 6), out_dtype="bf16")
    refused(lam, INVALID, a.batch_load_rows, [0], out=np.empty((1, 6)))
    mem = torch.empty(100)
    for out, status in [(torch.empty(2, 6), LENGTH), (torch.empty(18), LENGTH), (torch.empty(6, 3).t(), INVALID),
                        (mem.as_strided((3, 6), (4, 1)), INVALID), (mem.as_strided((3, 6), (0, 1)), INVALID),
                        (a.local_rows()[:3], INVALID)]:
        refused(lam, status, a.batch_load_rows([0, 1, 2], out=out).spawn)
    for vals, status in [(torch.ones(2, 6), LENGTH), (torch.ones(3, 5), LENGTH), (torch.tensor(1.0), LENGTH),
                         (torch.ones(3, 6, dtype=torch.float64), UNSUPPORTED), (torch.ones(3, 6, dtype=torch.int8), UNSUPPORTED),
                         (torch.ones(3, 6, dtype=torch.int64), UNSUPPORTED), (a.local_rows()[:3], INVALID)]:
        refused(lam, status, a.batch_add_rows([0, 1, 2], vals).spawn)
        refused(lam, status, a.batch_store_rows([0, 1, 2], vals).spawn)
    assert not a.local_rows().any()                      # nothing of the refused was applied
    with pytest.warns(RuntimeWarning):
        h = a.batch_load_rows([1])
        del h


def test_one_pe_batches(lam, team):
    """The calls that are not refused, on the test double."""
    a = lam.RowArray(team, 10, 4, dtype="bf16")
    a.batch_store_rows([1, 2, 1], torch.arange(12.0).view(3, 4)).block()
    assert a.batch_load_rows(1, out_dtype="f32").block().tolist() == [8, 9, 10, 11]
    a.batch_add_rows([[1], [1]], torch.ones(4), scale=0.5).block()
    assert a.batch_load_rows([[1, -1]], pad=-1).block().tolist() == [[[9, 10, 11, 12], [0, 0, 0, 0]]]
    a.batch_store_rows(lam.Owned(torch.tensor([4])), lam.Owned(torch.ones(1, 4))).block()
    assert a.batch_load_rows(lam.Owned([4])).block().tolist() == [[1, 1, 1, 1]]
    h = a.batch_load_rows([2])
    assert h.value() is h.spawn().value() is h.block()
    assert a.batch_add_rows([], torch.ones(0, 4)).block() is None
    assert a.batch_add_rows([], torch.ones(4)).block() is None
    assert a.batch_load_rows(np.int64(2)).block().shape == (4,)
    weight = torch.nn.Parameter(torch.ones(3, 4))        # a parameter's memory, its gradient left alone
    p = lam.RowArray.from_tensor(team, weight)
    p.batch_add_rows([2], torch.ones(4, requires_grad=True), scale=2).block()
    assert weight[2].tolist() == [3, 3, 3, 3] and not p.local_rows().requires_grad


def test_c_entry_refusals(capi, lam):
    """Argument checks of the C entry points: each call here is turned down before it looks at the
    context or the device (the context pointer stands for one; nothing reads it)."""
    from lamellar_runtime_amd._capi import lmr_rows_t
    ctx = ctypes.c_void_p(64)
    p = 1 << 20                                          # stands for device memory

    def table(**k):
        d = dict(data=p, scales=p, claims=p, rows=10, row_len=8, type=0, group=4)
        d.update(k)
        return ctypes.byref(lmr_rows_t(**d))

    def load(t, ctx=ctx, idx=p, iw=8, n=3, out=p, ty=0, stride=8):
        return capi.lmr_rows_load(ctx, t, idx, iw, n, 0, 0, 1.0, out, ty, stride, None)

    def add(t, ctx=ctx, idx=p, iw=8, n=3, out=p, ty=0, stride=8, work=None, nbytes=0):
        return capi.lmr_rows_add(ctx, t, idx, iw, n, 0, 0, 1.0, out, ty, stride, work, nbytes, None)

    def store(t, ctx=ctx, idx=p, iw=8, n=3, out=p, ty=0, stride=8):
        return capi.lmr_rows_store(ctx, t, idx, iw, n, 0, 0, out, ty, stride, None)

    for f in (load, add, store):
        assert f(None) == 1 and f(table(), ctx=None) == 1
        for bad in (dict(type=5), dict(row_len=0), dict(row_len=(1 << 18) + 1), dict(rows=1 << 32), dict(data=None), dict(data=p + 2),
                    dict(type=1, data=p + 1), dict(type=3, group=0), dict(type=4, group=3), dict(type=3, scales=None),
                    dict(type=4, scales=p + 2), dict(claims=p + 2)):
            assert f(table(**bad)) == 1, (f, bad)
        for bad in (dict(idx=None), dict(idx=p + 4), dict(iw=2), dict(iw=1), dict(out=None), dict(out=p + 2), dict(ty=1, out=p + 1),
                    dict(ty=3), dict(stride=7), dict(n=(1 << 25) + 1), dict(stride=1 << 32)):
            assert f(table(), **bad) == 1, (f, bad)
        if f is not add:
            assert f(table(), n=0) == 0 and f(table(type=4), n=0, idx=None, out=None) == 0
    assert load(table(), stride=0) == 1                  # every record's output in one place
    assert add(table(), n=0) == 0 and add(table(type=3)) == 5 and add(table(type=4), n=0) == 5
    big = 1 << 16
    need = capi.lmr_rows_add_workspace(table(), big)
    if need:
        assert add(table(), n=big, work=p, nbytes=need - 1) == 7 and add(table(), n=big, work=None, nbytes=need) == 7
        assert add(table(), n=big, work=p + 4, nbytes=need) == 7


def test_captured_store_has_its_own_claims(lam):
    """A store of many records that is captured into a graph takes claim words of its own, also where an
    eager store has made the array's: a replay may come when the array is gone."""
    seen = []

    class Kernels(CpuRowKernels):
        graph = False

        def capturing(self):
            return self.graph

        def rows_store(self, table, *a):
            seen.append(table.claims)
            super().rows_store(table, *a)

    team = lam.LamellarWorldBuilder().with_kernels(Kernels).build().team()
    a = lam.RowArray(team, 7, 2)
    i, v = torch.arange(1025) % 7, torch.ones(1025, 2)
    a.batch_store_rows(i, v).block()
    for graph in (True, True, False):
        team.kernels.graph = graph
        a.batch_store_rows(i, v).spawn()
    team.kernels.graph = False
    own = seen[0]
    assert a._table.claims is own and own.numel() == 7 and seen[3] is own
    assert all(c is not own and c.numel() == 7 and not c.any() for c in seen[1:3]) and seen[1] is not seen[2]


def test_refused_handles_stay_refused(lam, team):
    """A handle whose batch was turned down raises every time it is asked, and gives no result."""
    a = lam.RowArray(team, 10, 6)
    for h in (a.batch_add_rows([0, 1, 2], torch.ones(2, 6)), a.batch_store_rows([0, 1, 2], torch.ones(2, 6)),
              a.batch_load_rows([0, 1, 2], out=torch.empty(2, 6))):
        for call in (h.spawn, h.value, h.block, h.spawn):
            refused(lam, LENGTH, call)
        with warnings.catch_warnings():
            warnings.simplefilter("error")               # it was spawned: nothing to warn of
            del h, call
    bad = a.batch_load_rows(torch.ones(3))
    refused(lam, INVALID, bad.value)
    refused(lam, INVALID, bad.block)
    assert not a.local_rows().any()


def test_writes_are_seen_by_autograd(lam):
    """A batch that writes raises the version of what it wrote, so that a backward pass over a tensor saved
    before it is refused, as after torch's own in-place operations; a lookup leaves the table's version."""

    class Kernels(CpuRowKernels):                        # writes past torch, as the device does
        def rows_load(self, table, idx, n, pad, scale, out, *a):
            out.numpy()[:] = scale

        def rows_add(self, table, *a):
            table.data.numpy()[0] += 1

        def rows_store(self, table, *a):
            table.data.numpy()[0] = 5

    team = lam.LamellarWorldBuilder().with_kernels(Kernels).build().team()
    for write in ("batch_add_rows", "batch_store_rows"):
        weight = torch.nn.Parameter(torch.ones(4, 3))
        a = lam.RowArray.from_tensor(team, weight)
        loss = (weight * weight).sum()
        a.batch_load_rows([1, 2]).block()
        loss.backward(retain_graph=True)
        getattr(a, write)([0], torch.ones(1, 3)).block()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    codes, scales = torch.zeros(4, 6, dtype=torch.uint8), torch.ones(4, 2, requires_grad=True)
    c = lam.RowArray.from_tensor(team, codes, scales=scales, dtype="i8")
    loss, was = (scales * scales).sum(), codes._version
    c.batch_store_rows([0], torch.ones(1, 6)).block()
    assert codes._version > was
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    out, w = torch.zeros(2, 3), torch.ones(2, 3, requires_grad=True)
    loss = (w * out).sum()
    a.batch_load_rows([1, 2], out=out).block()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        d = lam.RowArray(team, 4, 3)
        d.batch_store_rows([0], torch.ones(1, 3)).block()
        d.batch_load_rows([0], out=torch.empty(1, 3)).block()


def test_refused_numbers(lam, team):
    """Truth values are no indices, pads or scales, alone or in a list; integers past 63 bits name no row, and
    none of them is taken for another number (2^64 - 1 is not the pad -1)."""
    a = lam.RowArray(team, 10, 6)
    v = torch.ones(6)
    for h in (a.batch_load_rows, lambda i, **k: a.batch_add_rows(i, v, **k), lambda i, **k: a.batch_store_rows(i, v, **k)):
        for i in (True, np.bool_(True), [True], np.ones(1, dtype=bool), torch.tensor(True)):
            refused(lam, INVALID, lambda: h(i).block())
        for pad in (True, np.bool_(False), torch.tensor(1)):
            refused(lam, INVALID, lambda: h([1], pad=pad).block())
        top = (1 << 64) - 1
        for i in (np.array([top], dtype=np.uint64), np.uint64(top), top, [top], -(1 << 63) - 1,
                  torch.tensor([-1]).view(torch.uint64)):
            for pad in (-1, -(1 << 63), None):
                refused(lam, OOB, lambda: h(i, pad=pad).block())
        a.local_rows().zero_()
        for i in ([1 << 70], [1, 1 << 63]):              # lists that have no integer type
            refused(lam, INVALID, lambda: h(i).block())
    assert not a.local_rows().any()
    for scale in (True, np.bool_(True), np.str_("2"), np.complex64(2), 1j):
        refused(lam, INVALID, lambda: a.batch_load_rows([1], scale=scale).block())
        refused(lam, INVALID, lambda: a.batch_add_rows([1], v, scale=scale).block())
    a.batch_add_rows(np.uint64(3), v, scale=np.float16(0.5)).block()
    a.batch_add_rows(np.array([3], dtype=np.uint64), v, scale=2).block()
    a.batch_add_rows([3, np.int8(3), -1], v, pad=np.int64(-1)).block()
    a.batch_add_rows(torch.tensor([3], dtype=torch.uint16), v).block()
    assert (a.local_rows()[3] == 5.5).all() and int((a.local_rows() != 0).sum()) == 6


def test_exchange_places_rows_by_the_row_kernels(lam, monkeypatch):
    """What comes back from the owners is put into `out`, whole or strided, pads and indices out of bounds as
    zeros, by the row operators."""
    from lamellar_runtime_amd import rows as rows_module
    calls = []

    class Kernels(CpuRowKernels):
        def rows_load(self, table, idx, n, pad, scale, out, out_type, stride, stream):
            calls.append(out.data_ptr())
            super().rows_load(table, idx, n, pad, scale, out, out_type, stride, stream)

        def rows_store(self, table, *a):
            calls.append(table.data.data_ptr())
            super().rows_store(table, *a)

    monkeypatch.setattr(rows_module, "_all_gather", lambda team, mine: [mine])
    monkeypatch.setattr(rows_module, "_all_to_all", lambda team, rows, sent, got: rows)
    team = lam.LamellarWorldBuilder().with_kernels(Kernels).build().team()
    a = lam.RowArray.from_tensor(team, torch.arange(24.0).view(6, 4))
    a._distributed = True
    i = torch.tensor([5, -1, 0, 9, 5])
    exp = torch.where(((i >= 0) & (i < 6))[:, None], a.local_rows()[i.clamp(0, 5)], 0.0)
    wide = torch.full((5, 9), 7.0)
    for out in (wide[:, 2:6], torch.full((5, 4), 7.0)):
        calls.clear()
        h = a.batch_load_rows(i, pad=-1, out=out)
        refused(lam, OOB, h.block)
        assert torch.equal(h.value(), exp) and calls[-1] == out.data_ptr()
    assert (wide[:, :2] == 7).all() and (wide[:, 6:] == 7).all()
    got = a.batch_load_rows([[1], [4]], scale=2).block()
    assert torch.equal(got[:, 0], a.local_rows()[[1, 4]] * 2)
    assert not a.batch_load_rows([-1, -1], pad=-1).block().any()


def test_refused_memory(lam, team):
    """Values and outputs that lie in the array's scales, as in its rows, are turned down: the batch would read
    what it writes. Neighbours of either in one allocation are taken."""
    mem = torch.zeros(100)
    scales = mem[10:50].view(10, 4)
    a = lam.RowArray.from_tensor(team, torch.zeros(10, 4, dtype=torch.int8), scales=scales)
    for part in (scales, scales[2:5], mem[7:19].view(3, 4), mem[49:61].view(3, 4), mem[46:66].view(4, 5)[:, 1:], a.local_scales()[9:]):
        i = list(range(len(part)))
        refused(lam, INVALID, a.batch_store_rows(i, part).spawn)
        refused(lam, INVALID, a.batch_load_rows(i, out=part).spawn)
    refused(lam, INVALID, a.batch_store_rows([1, 2], scales[3]).spawn)
    for part in (mem[2:10].view(2, 4), mem[50:58].view(2, 4)):
        a.batch_store_rows([1, 2], part).block()
        a.batch_load_rows([1, 2], out=part).block()
    b = lam.RowArray.from_tensor(team, mem[60:80].view(5, 4))
    refused(lam, INVALID, b.batch_add_rows([0], mem[76:80]).spawn)
    refused(lam, INVALID, b.batch_load_rows([0], out=mem[57:61].view(1, 4)).spawn)
    b.batch_add_rows([0], mem[80:84]).block()


def test_negated_views(lam):
    """Values that are a view whose sign torch keeps beside the memory (the imaginary part of a conjugate) are
    taken with their sign; such an output is turned down."""

    def raw(t):                                          # what the memory holds, as the device sees it
        return torch._neg_view(t) if t.is_neg() else t

    class Kernels(CpuRowKernels):
        def rows_add(self, table, idx, n, pad, scale, vals, *a):
            super().rows_add(table, idx, n, pad, scale, raw(vals), *a)

        def rows_store(self, table, idx, n, pad, vals, *a):
            super().rows_store(table, idx, n, pad, raw(vals), *a)

    team = lam.LamellarWorldBuilder().with_kernels(Kernels).build().team()
    for width in (1, 4):
        a = lam.RowArray(team, 5, width)
        v = torch.complex(torch.zeros(3, width), torch.ones(3, width)).conj().imag
        assert v.is_neg() and (v == -1).all()
        for vals in (v, torch._neg_view(torch.ones(3, width)), v[:1]):
            a.local_rows().zero_()
            i = list(range(len(vals)))
            a.batch_add_rows(i, vals, scale=2).block()
            assert (a.local_rows()[i] == -2).all()
            a.batch_store_rows(i, vals).block()
            assert (a.local_rows()[i] == -1).all()
        for out in (torch._neg_view(torch.ones(3, width)),):
            refused(lam, INVALID, a.batch_load_rows([0, 1, 2], out=out).spawn)
    refused(lam, INVALID, lam.RowArray.from_tensor, team, torch._neg_view(torch.ones(3, 4)))


# ------------------------------------------------------------------ several PEs
def _inputs(rank, n, rows, width, seed):
    g = torch.Generator().manual_seed(seed * 10 + rank)
    i = torch.randint(rows, (n,), generator=g)
    return i, torch.randint(-8, 9, (n, width), generator=g).float() / 8


def _worker(rank, ws, port, outdir, dist_kind):
    sys.path.insert(0, ROOT)
    sys.path.insert(0, os.path.join(ROOT, "tests"))
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(ws), LOCAL_RANK=str(rank))
    from _lamellar_bootstrap import load_package
    lam = load_package()
    from test_batch_rows import CpuRowKernels, _inputs
    world = lam.LamellarWorldBuilder().with_kernels(CpuRowKernels).build()
    team, res = world.team(), {}
    rows, width = 23, 6
    n = [40, 0, 7][rank]                                 # a PE with nothing to send takes part
    a = lam.RowArray(team, rows, width, dist_kind)
    i, v = _inputs(rank, n, rows, width, 1)
    a.batch_add_rows(i, v, scale=0.5).block()
    team.barrier()
    res["after_add"] = a.batch_load_rows(torch.arange(rows)).block().numpy()
    i, _ = _inputs(rank, n, rows, width, 2)
    i[::3] = -1                                          # places of no row
    wide = torch.full((n, width + 3), 7.0)
    out = a.batch_load_rows(i, scale=2.0, pad=-1, out=wide[:, 1:width + 1]).block()
    res["load_index"], res["loaded"], res["wide"] = i.numpy(), out.numpy(), wide.numpy()
    team.barrier()
    i, v = _inputs(rank, n, rows, width, 3)
    a.batch_store_rows(i, v).block()
    team.barrier()
    res["after_store"] = a.batch_load_rows(torch.arange(rows)).block().numpy()
    c = lam.RowArray(team, 2, width, dist_kind, dtype="e4m3", group=3)     # fewer rows than PEs
    i, v = _inputs(rank, n, 2, width, 4)
    c.batch_store_rows(i, v.to(torch.float16)).block()
    team.barrier()
    res["codes"] = c.batch_load_rows([[0], [1]], out_dtype="f32").block().numpy()
    h = a.batch_load_rows([rows if rank == 0 else 1])
    try:
        h.block()
        res["oob"] = np.array(0)
    except lam.LamellarError as e:
        res["oob"] = np.array(int(e.status))
    res["oob_rows"] = h.value().numpy()
    shard = torch.zeros(a.num_rows_local(), width)
    b = lam.RowArray.from_tensor(team, shard, rows=rows, distribution=dist_kind)
    b.batch_add_rows([5], torch.ones(width)).block()
    team.barrier()
    res["five"] = b.batch_load_rows([5]).block().numpy()
    np.savez(os.path.join(outdir, f"pe{rank}.npz"), **res)
    import torch.distributed as dist
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("ws,dist_kind", [(2, 0), (2, 1), (3, 0), (3, 1)])
def test_exchange_gloo(ws, dist_kind):
    import rowref as ref
    rows, width = 23, 6
    port = 29900 + ws * 11 + dist_kind * 5 + (os.getpid() % 200)
    with tempfile.TemporaryDirectory() as d:
        mp.spawn(_worker, args=(ws, port, d, dist_kind), nprocs=ws, join=True)
        pe = [{k: torch.from_numpy(v) for k, v in np.load(os.path.join(d, f"pe{r}.npz")).items()} for r in range(ws)]
    ins = {s: [_inputs(r, [40, 0, 7][r], rows if s < 4 else 2, width, s) for r in range(ws)] for s in (1, 3, 4)}
    cat = {s: (torch.cat([x[0] for x in ins[s]]), torch.cat([x[1] for x in ins[s]])) for s in ins}
    exact, _ = ref.add(torch.zeros(rows, width), *cat[1], 0.5)           # eighths: every sum is exact
    stored = exact.float()
    for r, t in ref.last_records(cat[3][0], rows).items():
        stored[r] = cat[3][1][t]
    codes, scales = ref.quantise(cat[4][1].half(), "e4m3", 3)
    last = ref.last_records(cat[4][0], 2)
    for p, r in enumerate(pe):
        assert torch.equal(r["after_add"].double(), exact)
        assert torch.equal(r["loaded"].double(), ref.load(exact.float(), r["load_index"], 2.0, pad=-1))
        assert (r["wide"][:, 0] == 7).all() and (r["wide"][:, width + 1:] == 7).all()
        assert torch.equal(r["after_store"], stored)
        for row in (0, 1):
            exp = ref.load(ref.codes_f64(codes, "e4m3"), torch.tensor([last[row]]), 1.0, scales, 3)
            assert torch.equal(r["codes"][row, 0].double(), exp[0].float().double())
        assert int(r["oob"]) == (2 if p == 0 else 0)
        assert torch.equal(r["oob_rows"][0], torch.zeros(width) if p == 0 else stored[1])
        assert (r["five"] == ws).all()


def _limit_worker(rank, ws, port, outdir):
    sys.path.insert(0, ROOT)
    sys.path.insert(0, os.path.join(ROOT, "tests"))
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(ws), LOCAL_RANK=str(rank))
    from _lamellar_bootstrap import load_package
    lam = load_package()
    from lamellar_runtime_amd import rows as rows_module
    from test_batch_rows import CpuRowKernels

    class Kernels(CpuRowKernels):                        # the device's limits, lowered
        def _check(self, table, n):
            if n > 20 or n * table.row_len > 100:
                raise lam.LamellarError(1, "too many")

        def rows_load(self, table, idx, n, *a):
            self._check(table, n)
            super().rows_load(table, idx, n, *a)

        def rows_add(self, table, idx, n, *a):
            self._check(table, n)
            super().rows_add(table, idx, n, *a)

        def rows_store(self, table, idx, n, *a):
            self._check(table, n)
            super().rows_store(table, idx, n, *a)

    rows_module.MAX_BATCH, rows_module.MAX_VALUES = 20, 100
    team, res = lam.LamellarWorldBuilder().with_kernels(Kernels).build().team(), []
    for width, n in ((2, [11, 11]), (8, [7, 6]), (2, [21, 0]), (2, [11, 9])):
        a = lam.RowArray(team, 10, width)
        i = torch.full((n[rank],), 2)                    # all of PE 0's
        spread = i.clone() if n[1] else torch.arange(n[rank]) % 10
        for h in (a.batch_load_rows(spread), a.batch_add_rows(spread, torch.ones(width)), a.batch_store_rows(spread, torch.ones(width))):
            try:
                h.block()
                res.append(0)
            except lam.LamellarError as e:
                res.append(int(e.status))
        team.barrier()
    np.savez(os.path.join(outdir, f"pe{rank}.npz"), res=np.array(res))
    torch.distributed.barrier()
    torch.distributed.destroy_process_group()


def test_exchange_limits():
    """A batch that would be too large for one PE is turned down by every PE, none waits for another."""
    with tempfile.TemporaryDirectory() as d:
        ctx = mp.spawn(_limit_worker, args=(2, 30350 + os.getpid() % 200, d), nprocs=2, join=False)
        try:
            until = time.monotonic() + 60
            while not ctx.join(timeout=1):
                assert time.monotonic() < until, "a PE waits"
        finally:
            for p in ctx.processes:
                if p.is_alive():
                    p.kill()
        for r in range(2):
            assert np.load(os.path.join(d, f"pe{r}.npz"))["res"].tolist() == [1] * 9 + [0] * 3
