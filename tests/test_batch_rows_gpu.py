"""RowArray on the device against plain 64-bit forms (rowref.py): lookups, their gradient, 8-bit
rows written and read back, at the sizes, types, layouts and masks where each can go wrong."""
import numpy as np
import pytest
import torch

import rowref as ref

pytestmark = pytest.mark.gpu

FLOATS = ["f32", "f16", "bf16"]
CODES = ["i8", "e4m3"]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def indices(g, n, rows, how, dtype=torch.int64):
    if how == "same":
        i = torch.full((n,), int(torch.randint(rows, (1,), generator=g)))
    elif how == "distinct":
        i = torch.randperm(rows, generator=g)[:n]
    elif how == "few":                                   # a handful of rows, runs of any length
        i = torch.randint(min(rows, 5), (n,), generator=g) * max(1, (rows - 1) // 5)
    elif how == "skewed":                                # one row has a third of the records, the others few
        i = torch.randint(rows, (n,), generator=g)
        i[torch.rand(n, generator=g) < 0.34] = rows - 1
    else:
        i = torch.randint(rows, (n,), generator=g)
    return i.to(dtype)


def float_array(lam, world, g, rows, width, kind):
    t = torch.randn(rows, width, generator=g).to(ref.TORCH[kind])
    return lam.RowArray.from_tensor(world.team(), t.cuda()), t


def code_array(lam, world, g, rows, width, group, kind):
    """An 8-bit array filled by hand: (array, f64 codes, scales)"""
    if kind == "i8":
        c = torch.randint(-127, 128, (rows, width), generator=g).to(torch.int8)
    else:
        c = (torch.randn(rows, width, generator=g) * 120).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.rand(rows, width // group, generator=g) + 0.01
    c = c.view(torch.uint8)
    a = lam.RowArray.from_tensor(world.team(), c.cuda(), scales=s.cuda(), dtype=kind)
    return a, ref.codes_f64(c, kind), s


def check_close(got, exact, bound):
    d = (got.cpu().double() - exact).abs()
    bad = ~(d <= bound)
    assert not bad.any(), (int(bad.sum()), tuple(bad.nonzero()[0].tolist()), float((d / bound.clamp(min=1e-300)).max()))


# ------------------------------------------------------------------ load
@pytest.mark.parametrize("out", FLOATS)
@pytest.mark.parametrize("kind", FLOATS)
@pytest.mark.parametrize("n,rows,width", [(1, 1, 1), (3, 5, 7), (17, 100, 64), (300, 41, 1001), (5, 9, 8192),
                                          (2500, 1000, 72), (70000, 3000, 33), (20000, 50, 520)])
def test_load(lam, world, kind, out, n, rows, width):
    g = gen(n + width)
    a, t = float_array(lam, world, g, rows, width, kind)
    i = indices(g, n, rows, "any", torch.int32 if n % 2 else torch.int64)
    got = a.batch_load_rows(i.cuda(), scale=1.7, out_dtype=out).block()
    assert got.shape == (n, width) and got.dtype == ref.TORCH[out]
    exact = ref.load(t, i, 1.7)
    check_close(got, exact, ref.load_bound(exact, out, 1))


@pytest.mark.parametrize("out", FLOATS)
@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("n,rows,width,group", [(1, 1, 1, 1), (5, 9, 30, 3), (33, 50, 128, 128), (70, 64, 640, 80), (9, 20, 1000, 100),
                                                (3000, 500, 1024, 128), (300, 40, 1152, 576), (40, 7, 4096, 4096), (60000, 100, 36, 12),
                                                (4000, 200, 56, 56)])
def test_load_codes(lam, world, kind, out, n, rows, width, group):
    g = gen(n + width)
    a, c, s = code_array(lam, world, g, rows, width, group, kind)
    i = indices(g, n, rows, "any", torch.int64 if n % 2 else torch.int32)
    got = a.batch_load_rows(i.cuda(), scale=0.3, out_dtype=out).block()
    exact = ref.load(c, i, 0.3, s, group)
    check_close(got, exact, ref.load_bound(exact, out, 2))


def test_load_every_code(lam, world):
    """All 256 codes of both types, NaN codes of e4m3 included."""
    for kind in CODES:
        c = torch.arange(256, dtype=torch.uint8).view(1, 256)
        a = lam.RowArray.from_tensor(world.team(), c.cuda(), scales=torch.ones(1, 1).cuda(), dtype=kind)
        got = a.batch_load_rows([0], out_dtype="f32").block().cpu().double()
        exp = ref.codes_f64(c, kind)
        assert torch.equal(torch.isnan(got), torch.isnan(exp))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(exp))


@pytest.mark.parametrize("kind,out,scale", [("f32", "f32", 1.0), ("f32", "f16", 1.0), ("f32", "bf16", 3.0), ("f16", "f32", 1.0),
                                            ("bf16", "f16", 1.0)])
def test_load_specials(lam, world, kind, out, scale):
    """Infinities, NaN, subnormals, halfway values and values that overflow the output's type."""
    v = [0.0, -0.0, float("inf"), -float("inf"), float("nan"), 65504.0, 65519.0, 65520.0, 3.0e38, 1e-40, 6e-8, 3e-8, 2.98e-8,
         1.00390625, 1.01171875, 1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 1e-45]
    t = torch.tensor([v]).to(ref.TORCH[kind])
    a = lam.RowArray.from_tensor(world.team(), t.cuda())
    got = a.batch_load_rows([0, 0], scale=scale, out_dtype=out).block().cpu()
    exp = (t.float() * scale).to(ref.TORCH[out]).expand(2, -1)
    assert torch.equal(torch.isnan(got), torch.isnan(exp))
    assert torch.equal(torch.nan_to_num(got.float(), nan=7.0), torch.nan_to_num(exp.float(), nan=7.0))


def test_load_pads_and_out_of_bounds(lam, world):
    g = gen(4)
    a, t = float_array(lam, world, g, 50, 200, "bf16")
    i = torch.tensor([3, -1, 49, -1, 0])
    got = a.batch_load_rows(i.cuda(), pad=-1, out_dtype="f32").block()
    exact = ref.load(t, i, pad=-1)
    assert torch.equal(got.cpu().double(), exact)
    # a pad that is a row's index masks that row
    got = a.batch_load_rows(i.to(torch.int32).cuda(), pad=49, out_dtype="f32").spawn()
    assert torch.equal(got.value().cpu()[2], torch.zeros(200))
    with pytest.raises(lam.LamellarError) as e:
        got.block()                                      # -1 is no pad there
    assert e.value.status == 2
    for bad in (50, -2, 1 << 40, -(1 << 62)):
        h = a.batch_load_rows(torch.tensor([1, bad, 2]).cuda(), out_dtype="f32")
        with pytest.raises(lam.LamellarError) as e:
            h.block()
        assert e.value.status == 2
        assert torch.equal(h.value().cpu(), torch.stack([t[1], torch.zeros(200), t[2]]).float())
    c, codes, s = code_array(lam, world, g, 20, 64, 32, "e4m3")
    got = c.batch_load_rows(torch.tensor([-7, 3, -7]).cuda(), pad=-7, out_dtype="f32").block().cpu().double()
    exact = ref.load(codes, torch.tensor([-7, 3, -7]), 1.0, s, 32, -7)
    check_close(got, exact, ref.load_bound(exact, "f32", 2))
    assert not a.batch_load_rows(torch.full((9,), -1).cuda(), pad=-1).block().any()


def test_load_shapes_strides_and_inputs(lam, world):
    g = gen(5)
    a, t = float_array(lam, world, g, 60, 48, "f16")
    i = torch.randint(60, (3, 4), generator=g)
    exp = t[i]
    assert torch.equal(a.batch_load_rows(i.cuda()).block().cpu(), exp)
    assert torch.equal(a.batch_load_rows(i.numpy()).block().cpu(), exp)
    assert torch.equal(a.batch_load_rows(i.tolist()).block().cpu(), exp)
    assert torch.equal(a.batch_load_rows(i.t().cuda()).block().cpu(), exp.transpose(0, 1))
    assert torch.equal(a.batch_load_rows(i.to(torch.uint8).cuda()).block().cpu(), exp)
    assert torch.equal(a.batch_load_rows(7).block().cpu(), t[7])
    assert a.batch_load_rows(torch.empty(0, dtype=torch.int64).cuda()).block().shape == (0, 48)
    assert a.batch_load_rows([]).block().shape == (0, 48)
    # rows of a wider output, at an odd place; what lies between them stays
    wide = torch.full((12, 101), 5.0, dtype=torch.float16).cuda()
    out = wide[:, 3:51]
    assert a.batch_load_rows(i.reshape(-1).cuda(), out=out).block() is out
    w = wide.cpu()
    assert torch.equal(w[:, 3:51], exp.reshape(12, 48)) and (w[:, :3] == 5).all() and (w[:, 51:] == 5).all()
    # a table that begins at an odd element of its memory
    mem = torch.randn(61 * 47 + 1, generator=g).to(torch.bfloat16).cuda()
    b = lam.RowArray.from_tensor(world.team(), mem[1:].view(61, 47))
    got = b.batch_load_rows(torch.arange(61).cuda()).block()
    assert torch.equal(got, mem[1:].view(61, 47))


# ------------------------------------------------------------------ add
@pytest.mark.parametrize("kind,vals", [("f32", "bf16"), ("f32", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "bf16"),
                                       ("f32", "f16")])
@pytest.mark.parametrize("n,rows,width,how", [
    (1, 1, 1, "same"), (2, 1, 3, "same"), (5, 9, 64, "any"), (63, 700, 1001, "distinct"), (300, 7, 520, "any"),
    (511, 600, 33, "skewed"), (512, 600, 8, "any"), (513, 600, 40, "skewed"), (1024, 900, 1024, "skewed"), (1025, 70, 1024, "skewed"),
    (700, 9, 1500, "few"), (513, 400, 2600, "skewed"), (257, 100, 8200, "skewed"), (1500, 1, 72, "same"),
    (4096, 5000, 130, "few"), (4099, 4099, 264, "distinct"), (9000, 100000, 96, "any"), (20000, 1 << 19, 24, "skewed")])
def test_add(lam, world, kind, vals, n, rows, width, how):
    g = gen(n + width)
    a, t = float_array(lam, world, g, rows, width, kind)
    i = indices(g, n, rows, how, torch.int32 if n % 2 else torch.int64)
    v = torch.randn(n, width, generator=g).to(ref.TORCH[vals])
    a.batch_add_rows(i.cuda(), v.cuda(), scale=0.37).block()
    exact, bound = ref.add(t, i, v, 0.37)
    check_close(a.local_rows(), exact, bound)


@pytest.mark.parametrize("n,rows,width,how", [(70000, 3000, 264, "skewed"), (140001, 2, 64, "any"), (33000, 20000, 1000, "same"),
                                              (66000, 40, 16, "any")])
def test_add_large(lam, world, n, rows, width, how):
    """Runs far longer than one workgroup's share, and many of them."""
    g = gen(n)
    a, t = float_array(lam, world, g, rows, width, "f32")
    i = indices(g, n, rows, how)
    v = torch.randn(n, width, generator=g).to(torch.bfloat16)
    a.batch_add_rows(i.cuda(), v.cuda()).block()
    exact, bound = ref.add(t, i, v)
    check_close(a.local_rows(), exact, bound)


@pytest.mark.parametrize("n", [1025, 4097, 6143, 6144, 6145, 7169, 32767, 32768, 32769, 65536, 65537, 262143, 262145, 1 << 20, (1 << 20) + 1, 3000001])
@pytest.mark.parametrize("rows", [700, 3000017])
def test_add_many_records(lam, world, n, rows):
    """Sorted by each means, tiles of each size, few and many of them. Whole numbers: the sums are exact (below 2^24: a row
    has at most 16 n / rows + 2^16 records of at most 8)."""
    g = gen(n)
    a = lam.RowArray(world.team(), rows, 2)
    i = torch.where(torch.rand(n, generator=g) < 0.5, torch.randint(rows, (n,), generator=g),
                    torch.randint(rows // 16 + 1, (n,), generator=g))
    i[-1], i[0] = rows - 1, 0
    v = torch.randint(-8, 9, (n, 2), generator=g)
    a.batch_add_rows(i.cuda(), v.float().cuda()).block()
    exp = torch.zeros(rows, 2, dtype=torch.float64).index_add_(0, i, v.double())
    assert torch.equal(a.local_rows().double().cpu(), exp)


@pytest.mark.parametrize("n", [700, 6144, 6145, 20000])
@pytest.mark.parametrize("rows", [3, 511, 512, (1 << 18) - 1, 1 << 18, (1 << 20) + 7, (1 << 27) + 3])
def test_add_key_widths(lam, world, n, rows):
    """Tables of few to many rows: one to four sort passes, indices at both ends."""
    g = gen(n)
    a = lam.RowArray(world.team(), rows, 1, dtype="f16")
    i = torch.randint(rows, (n,), generator=g)
    i[: n // 4] = rows - 1 - torch.randint(min(rows, 40), (n // 4,), generator=g)
    i[-3:] = 0
    v = torch.randint(-4, 5, (n, 1), generator=g).to(torch.float16)       # every sum exact, below 2^11
    a.batch_add_rows(i.cuda(), v.cuda()).block()
    at, back = torch.unique(i, return_inverse=True)
    exact = torch.zeros(len(at), 1, dtype=torch.float64).index_add_(0, back, v.double())
    fits = exact.abs() <= 2048                                            # (3 rows: some sums are larger and round)
    got = a.batch_load_rows(at.cuda(), out_dtype="f32").block().cpu().double()
    assert torch.equal(got[fits], exact[fits])
    assert ((got - exact).abs() <= exact.abs() * ref.u("f16")).all()
    assert int((a.local_rows() != 0).sum()) == int((exact != 0).sum())


def test_add_very_many(lam, world):
    """More tiles than one launch adds up by itself (the sort's prefix launch)."""
    n, rows, width = 1200007, 5000, 8
    g = gen(n)
    a, t = float_array(lam, world, g, rows, width, "f32")
    i = indices(g, n, rows, "skewed")
    v = torch.randn(n, width, generator=g).to(torch.bfloat16)
    a.batch_add_rows(i.cuda(), v.cuda(), scale=0.5).block()
    exact, bound = ref.add(t, i, v, 0.5)
    check_close(a.local_rows(), exact, bound)


@pytest.mark.parametrize("width", [24, 520, 1001])
@pytest.mark.parametrize("shift", [0, 1, 5])
def test_add_runs_at_borders(lam, world, width, shift):
    """Runs of every length around the powers of two, so that they begin and end before, on and behind
    any border of 8 to 64 records, runs of several borders among them."""
    g = gen(shift)
    lengths = [1] * shift
    for k in (8, 16, 32, 64, 128):
        for d in (-2, -1, 0, 1, 2):
            lengths += [k + d, 3, 1, 2 * k + d, k]
    rows = len(lengths)
    i = torch.repeat_interleave(torch.arange(rows), torch.tensor(lengths))[torch.randperm(sum(lengths), generator=g)]
    a, t = float_array(lam, world, g, rows, width, "f32")
    v = torch.randn(i.numel(), width, generator=g).to(torch.bfloat16)
    a.batch_add_rows(i.cuda(), v.cuda()).block()
    exact, bound = ref.add(t, i, v)
    check_close(a.local_rows(), exact, bound)


@pytest.mark.parametrize("n,how", [(400, "skewed"), (30000, "skewed"), (30000, "same"), (5000, "any")])
def test_add_repeats_its_bits(lam, world, n, how):
    g = gen(n)
    t = torch.randn(900, 520, generator=g).cuda()
    i = indices(g, n, 900, how).cuda()
    v = torch.randn(n, 520, generator=g).to(torch.bfloat16).cuda()
    seen = []
    for _ in range(4):
        a = lam.RowArray.from_tensor(world.team(), t.clone())
        a.batch_add_rows(i, v).block()
        seen.append(a.local_rows())
    assert all(torch.equal(seen[0], x) for x in seen[1:])


@pytest.mark.parametrize("n", [40, 3000])
def test_add_pads_and_out_of_bounds(lam, world, n):
    g = gen(n)
    rows, width = 90, 72
    a, t = float_array(lam, world, g, rows, width, "f32")
    i = indices(g, n, rows, "any")
    i[::3] = -1
    v = torch.randn(n, width, generator=g)
    a.batch_add_rows(i.cuda(), v.cuda(), pad=-1).block()
    exact, bound = ref.add(t, i, v, pad=-1)
    check_close(a.local_rows(), exact, bound)
    # nothing but pads
    before = a.local_rows().clone()
    a.batch_add_rows(torch.full((n,), 5).cuda(), v.cuda(), pad=5).block()
    assert torch.equal(before, a.local_rows())
    # an index out of bounds is skipped and reported; NaN values of it reach nothing
    i = indices(g, n, rows, "any")
    i[1], i[7], i[20] = rows, -1, 1 << 33
    w = v.clone()
    w[1], w[7], w[20] = float("nan"), float("inf"), float("nan")
    with pytest.raises(lam.LamellarError) as e:
        a.batch_add_rows(i.cuda(), w.cuda()).block()
    assert e.value.status == 2
    exact, bound = ref.add(before.cpu(), i, torch.nan_to_num(w, nan=0.0, posinf=0.0))
    check_close(a.local_rows(), exact, bound)


@pytest.mark.parametrize("n", [6, 700])
def test_add_strided_broadcast_and_shapes(lam, world, n):
    g = gen(n)
    rows, width = 30, 40
    a, t = float_array(lam, world, g, rows, width, "f32")
    i = indices(g, n, rows, "any")
    whole = torch.randn(n, 3 * width + 1, generator=g).to(torch.bfloat16)
    v = whole[:, width + 1:2 * width + 1]                # rows of a wider tensor, at an odd place
    a.batch_add_rows(i.cuda(), whole.cuda()[:, width + 1:2 * width + 1]).block()
    exact, bound = ref.add(t, i, v)
    check_close(a.local_rows(), exact, bound)
    now = a.local_rows().cpu().clone()
    one = torch.randn(width, generator=g)
    a.batch_add_rows(i.cuda(), one.cuda(), scale=2.0).block()            # one row for every record
    exact, bound = ref.add(now, i, one[None], 2.0)
    check_close(a.local_rows(), exact, bound)
    now = a.local_rows().cpu().clone()
    a.batch_add_rows(i.view(2, -1).cuda(), one.cuda().expand(2, n // 2, width)).block()
    exact, bound = ref.add(now, i, one[None])
    check_close(a.local_rows(), exact, bound)
    now = a.local_rows().cpu().clone()
    cols = torch.randn(width, n, generator=g)
    a.batch_add_rows(i.cuda(), cols.cuda().t()).block()                  # columns: copied by the call
    exact, bound = ref.add(now, i, cols.t())
    check_close(a.local_rows(), exact, bound)
    now = a.local_rows().cpu().clone()
    a.batch_add_rows(i.numpy(), cols.t().numpy()).block()
    exact, bound = ref.add(now, i, cols.t())
    check_close(a.local_rows(), exact, bound)


def test_add_specials(lam, world):
    """An infinity or NaN reaches its own row's element and no other."""
    for n in (8, 2000):
        a = lam.RowArray(world.team(), 10, 16)
        i = torch.arange(n) % 5
        v = torch.ones(n, 16)
        v[0, 3], v[1, 4], v[6, 4] = float("inf"), float("nan"), -float("inf")
        a.batch_add_rows(i.cuda(), v.cuda()).block()
        got = a.local_rows().cpu()
        exp = torch.zeros(10, 16).index_add_(0, i, v)
        assert torch.equal(torch.isnan(got), torch.isnan(exp))
        assert torch.equal(torch.nan_to_num(got, nan=9.0), torch.nan_to_num(exp, nan=9.0))


def test_gradient_by_differences(lam, world):
    """loss = sum(w * lookup(table)): what batch_add_rows makes of w, against (loss(T + hE) - loss(T - hE)) / 2h.
    The loss is linear and every number a multiple of 2^-6 below 2^6, so that the lookups and h = 1 are exact;
    the sums of both sides are then exact too (below 2^24 steps) and equal."""
    g = gen(1)
    rows, width, n, scale = 37, 24, 500, 0.5
    t = torch.randint(-64, 64, (rows, width), generator=g) / 64.0
    i = indices(g, n, rows, "skewed")
    w = torch.randint(-64, 64, (n, width), generator=g) / 64.0

    def loss(tab):
        a = lam.RowArray.from_tensor(world.team(), tab.cuda())
        return float((a.batch_load_rows(i.cuda(), scale=scale).block().double() * w.double().cuda()).sum())

    grad = lam.RowArray(world.team(), rows, width)
    grad.batch_add_rows(i.cuda(), w.cuda(), scale=scale).block()
    got = grad.local_rows().cpu().double()
    for _ in range(6):
        e = torch.randint(-2, 3, (rows, width), generator=g).float()
        assert (loss(t + e) - loss(t - e)) / 2 == float((got * e).sum())


# ------------------------------------------------------------------ store
@pytest.mark.parametrize("vals", FLOATS)
@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("n,rows,width,group", [(1, 1, 1, 1), (4, 9, 30, 3), (64, 100, 1024, 128), (65, 300, 640, 80), (200, 4000, 96, 32),
                                                (3000, 5000, 256, 64), (5, 6, 4097, 4097), (37, 50, 1200, 600), (2000, 2000, 1000, 100),
                                                (10, 30, 8192, 512), (1030, 2048, 192, 192), (2600, 2600, 16, 8), (999, 1000, 7, 7),
                                                (2049, 2100, 130, 26), (3, 3, 1500, 500), (2050, 2100, 1100, 1100)])
def test_store_codes(lam, world, kind, vals, n, rows, width, group):
    g = gen(n + width)
    a = lam.RowArray(world.team(), rows, width, dtype=kind, group=group)
    i = indices(g, n, rows, "distinct", torch.int32 if n % 2 else torch.int64)
    v = (torch.randn(n, width, generator=g) * torch.exp(torch.randn(n, 1, generator=g) * 2)).to(ref.TORCH[vals])
    a.batch_store_rows(i.cuda(), v.cuda()).block()
    codes, scales = ref.quantise(v, kind, group)
    got_c, got_s = a.local_rows().cpu().view(torch.uint8), a.local_scales().cpu()
    assert torch.equal(got_s[i.long()], scales)
    c, e = ref.codes_f64(got_c[i.long()], kind), ref.codes_f64(codes, kind)
    assert torch.equal(c, e), (int((c != e).sum()), c.numel())
    # and within half a step of the values: i8 half a scale; e4m3 half a step of a 4-bit significand,
    # at least half of 2^-9 scales; 3 roundings in f32 before the code's
    s = scales.double().repeat_interleave(group, dim=1)
    x = v.double()
    step = s if kind == "i8" else torch.maximum(x.abs() * 2.0 ** -3, s * 2.0 ** -9)
    assert ((c * s - x).abs() <= step * 0.5 * (1 + 2.0 ** -10) + x.abs() * 4 * ref.U32).all()
    rest = torch.ones(rows, dtype=torch.bool)
    rest[i.long()] = False
    assert not got_c[rest].any() and not got_s[rest].any()               # the other rows stay as they were


@pytest.mark.parametrize("kind", CODES)
def test_store_codes_specials(lam, world, kind):
    group, width = 8, 32
    v = torch.randn(9, width, generator=gen(2))
    v[1] = 0.0
    v[2, 9] = float("nan")
    v[3, 16] = -float("inf")
    v[4] = 1e-45
    v[5, 0:8] = 2.0 ** -130
    v[6] = 3.0e38
    v[7, 8:16] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -126.5])      # halves go to the even code
    v[8, 24:32] = torch.tensor([448.0, 17.0, 18.0, 19.0, -17.0, 2.0 ** -10, 2.0 ** -9 * 1.5, 1.0625])
    a = lam.RowArray(world.team(), 9, width, dtype=kind, group=group)
    a.batch_store_rows(torch.arange(9).cuda(), v.cuda()).block()
    codes, scales = ref.quantise(v, kind, group)
    s = a.local_scales().cpu()
    assert torch.equal(torch.isnan(s), torch.isnan(scales)) and torch.equal(torch.nan_to_num(s), torch.nan_to_num(scales))
    assert torch.equal(ref.codes_f64(a.local_rows().cpu().view(torch.uint8), kind), ref.codes_f64(codes, kind))
    back = a.batch_load_rows(torch.arange(9).cuda(), out_dtype="f32").block().cpu()
    assert torch.isnan(back[2, 8:16]).all() and torch.isnan(back[3, 16:24]).all() and int(torch.isnan(back).sum()) == 16
    assert not back[1].any()


@pytest.mark.parametrize("n,rows,width,how", [(2, 1, 3, "same"), (40, 6, 100, "any"), (700, 3, 1024, "any"), (5000, 50, 72, "skewed"),
                                              (30000, 20000, 40, "any")])
@pytest.mark.parametrize("kind", ["bf16", "i8", "e4m3"])
def test_store_last_record_wins(lam, world, kind, n, rows, width, how):
    g = gen(n)
    group = None if kind == "bf16" else width // (4 if width % 4 == 0 else 1)
    a = lam.RowArray(world.team(), rows, width, dtype=kind, group=group)
    i = indices(g, n, rows, how)
    v = torch.randn(n, width, generator=g).to(torch.bfloat16)
    for _ in range(2):                                   # the second call finds what the first one left
        a.batch_store_rows(i.cuda(), v.cuda()).block()
        last = ref.last_records(i, rows)
        at, t = torch.tensor(list(last)), torch.tensor([last[r] for r in last])
        if kind == "bf16":
            assert torch.equal(a.local_rows().cpu()[at], v[t])
        else:
            codes, scales = ref.quantise(v[t], kind, group)
            assert torch.equal(a.local_scales().cpu()[at], scales)
            assert torch.equal(ref.codes_f64(a.local_rows().cpu()[at].view(torch.uint8), kind), ref.codes_f64(codes, kind))
        i, v = i.flip(0), v * 2


@pytest.mark.parametrize("kind", FLOATS)
@pytest.mark.parametrize("vals", FLOATS)
def test_store_floats(lam, world, kind, vals):
    g = gen(8)
    for n, rows, width in [(1, 1, 1), (30, 90, 33), (1000, 3000, 520)]:
        a, t = float_array(lam, world, g, rows, width, kind)
        i = indices(g, n, rows, "distinct")
        v = torch.randn(n, width, generator=g).to(ref.TORCH[vals])
        a.batch_store_rows(i.cuda(), v.cuda()).block()
        exp = t.clone()
        exp[i] = v.to(ref.TORCH[kind])
        assert torch.equal(a.local_rows().cpu(), exp)


@pytest.mark.parametrize("n", [50, 4000])
def test_store_pads_strides_and_out_of_bounds(lam, world, n):
    g = gen(n)
    rows, width, group = 6000, 96, 32
    a = lam.RowArray(world.team(), rows, width, dtype="e4m3", group=group)
    i = indices(g, n, rows, "distinct", torch.int32)
    i[::4] = -1
    whole = torch.randn(n, 3 * width + 1, generator=g).to(torch.float16)
    v = whole[:, 2 * width + 1:]
    a.batch_store_rows(i.cuda(), whole.cuda()[:, 2 * width + 1:], pad=-1).block()
    live = i >= 0
    codes, scales = ref.quantise(v[live], "e4m3", group)
    at = i[live].long()
    assert torch.equal(ref.codes_f64(a.local_rows().cpu()[at].view(torch.uint8), "e4m3"), ref.codes_f64(codes, "e4m3"))
    assert torch.equal(a.local_scales().cpu()[at], scales)
    assert int((a.local_scales().cpu() != 0).any(1).sum()) == int(live.sum())
    before = a.local_rows().clone()
    with pytest.raises(lam.LamellarError) as e:
        a.batch_store_rows(torch.tensor([rows, -1, 1 << 35]).cuda(), torch.ones(3, width).cuda()).block()
    assert e.value.status == 2
    assert torch.equal(before.view(torch.uint8), a.local_rows().view(torch.uint8))
    a.batch_store_rows([7, 3, 7], torch.ones(width).cuda()).block()       # one row for every record
    assert (a.batch_load_rows([3, 7], out_dtype="f32").block() == 1).all()


def test_rows_past_32_bits(lam, world):
    """Rows whose elements start past 2^32: offsets in 64 bits in every operator."""
    width = 32768
    rows = (1 << 17) + 9
    i = torch.tensor([0, rows - 1, 1 << 17, 5])
    v = torch.randn(4, width, generator=gen(3)).to(torch.bfloat16)
    a = lam.RowArray(world.team(), rows, width, dtype="e4m3", group=128)
    a.batch_store_rows(i.cuda(), v.cuda()).block()
    codes, scales = ref.quantise(v, "e4m3", 128)
    got = a.batch_load_rows(i.cuda(), out_dtype="f32").block()
    exact = ref.load(ref.codes_f64(codes, "e4m3"), torch.arange(4), 1.0, scales, 128)
    check_close(got, exact, ref.load_bound(exact, "f32", 2))
    assert int((a.local_scales() != 0).any(1).sum()) == 4
    del a
    b = lam.RowArray(world.team(), rows, width, dtype="bf16")
    b.batch_add_rows(i.cuda(), v.cuda()).block()
    assert torch.equal(b.batch_load_rows(i.cuda()).block().cpu(), v)
    many = i.repeat(1000)                                # the sorted path
    b.batch_add_rows(many.cuda(), torch.ones(width, device="cuda"), scale=0.001).block()
    exact, bound = ref.add(v, torch.arange(4).repeat(1000), torch.ones(1, width), 0.001)
    check_close(b.batch_load_rows(i.cuda()).block(), exact, bound)


# ------------------------------------------------------------------ streams, graphs, together
def test_other_streams_and_open_session(lam, world):
    """A batch on a side stream, its array dropped before the stream has run; and one between deferred
    element batches, which stay deferred."""
    g = gen(6)
    t = torch.randn(4000, 1024, generator=g)
    i = torch.randint(4000, (9000,), generator=g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = lam.RowArray.from_tensor(world.team(), t.cuda())
        v = torch.ones(9000, 1024, device="cuda")
        a.batch_add_rows(i.cuda(), v).spawn()
        got = a.batch_load_rows(i.cuda()).spawn().value()
    del a
    torch.cuda.current_stream().wait_stream(side)
    count = torch.bincount(i, minlength=4000)
    exact, bound = ref.add(t, i, torch.ones(1, 1024))
    check_close(got, exact[i], bound[i] + 1e-300)
    assert int(count.sum()) == 9000
    e = lam.AtomicArray(world.team(), 1000, lam.Distribution.Block, "u64")
    idx = torch.randint(1000, (70000,), generator=g).cuda()
    e.batch_add(idx, 1).spawn()
    b = lam.RowArray.from_tensor(world.team(), t.cuda())
    row = b.batch_load_rows([5]).spawn().value()
    e.batch_add(idx, 1).block()
    assert torch.equal(row.cpu()[0], t[5]) and int(e.sum().block()) == 140000


@pytest.mark.parametrize("n,rows,width", [(48, 64, 256), (2500, 3000, 264)])
def test_captured_and_replayed(lam, world, n, rows, width):
    """Lookup, its gradient, a cache write and its read in one graph; every replay on new inputs equals
    the eager calls, with eager batches of the same arrays' context between the replays."""
    g = gen(n)
    t = torch.randn(rows, width, generator=g)
    mine, plain = (lam.RowArray.from_tensor(world.team(), t.cuda()) for _ in range(2))
    cache, pcache = (lam.RowArray(world.team(), rows, width, dtype="e4m3", group=width // 2) for _ in range(2))
    idx, vals = torch.zeros(n, dtype=torch.int64, device="cuda"), torch.zeros(n, width, device="cuda")

    def step(tab, c, i, v):
        x = tab.batch_load_rows(i, scale=2.0).spawn().value()
        tab.batch_add_rows(i, v, scale=-0.1).spawn()
        c.batch_store_rows(i, x).spawn()
        return x, c.batch_load_rows(i, out_dtype="f32").spawn().value()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = [lam.RowArray.from_tensor(world.team(), t.cuda()), lam.RowArray(world.team(), rows, width, dtype="e4m3", group=width // 2)]
        step(*warm, idx, vals)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x, back = step(mine, cache, idx, vals)
    for r in range(4):
        i = indices(g, n, rows, "skewed" if r % 2 else "any").cuda()
        v = torch.randn(n, width, generator=g).cuda()
        idx.copy_(i)
        vals.copy_(v)
        graph.replay()
        ex, eback = step(plain, pcache, i, v)
        torch.cuda.synchronize()
        assert torch.equal(x, ex) and torch.equal(back, eback), r
        assert torch.equal(mine.local_rows(), plain.local_rows()), r
        assert torch.equal(cache.local_rows().view(torch.uint8), pcache.local_rows().view(torch.uint8)), r
        assert torch.equal(cache.local_scales(), pcache.local_scales()), r
    world.wait_all()


def test_training_steps(lam, world):
    """Steps of a model that is a table and a vector: lookup, a loss, its gradient back into the table,
    against the same steps in torch in 64 bits."""
    g = gen(12)
    rows, width, n, rate = 300, 64, 800, 0.05
    t = torch.randn(rows, width, generator=g)
    w = torch.randn(width, generator=g)
    table = lam.RowArray.from_tensor(world.team(), t.cuda())
    exact = t.double()
    for _ in range(5):
        i = indices(g, n, rows, "skewed")
        y = torch.randn(n, generator=g)
        x = table.batch_load_rows(i.cuda(), scale=0.5).spawn().value()
        d = (x @ w.cuda() - y.cuda()) / n
        table.batch_add_rows(i.cuda(), d[:, None] * w.cuda(), scale=-rate * 0.5).block()
        dx = (exact[i] * 0.5 @ w.double() - y.double()) / n
        exact = exact.index_add(0, i, dx[:, None] * w.double() * (-rate * 0.5))
    # 5 steps of f32 work on numbers of size ~1 with at most 800 terms a row: 5 * 800 half steps of
    # terms below 2^-2 in size, and the matrix product's 64 terms of at most 2^6
    assert float((table.local_rows().cpu().double() - exact).abs().max()) < 5 * 800 * ref.U32 * 2.0 ** -2 + 64 * 2.0 ** 6 * ref.U32


def test_decode_steps(lam, world):
    """A cache that grows by a row per sequence and step, its pages in any order, read back ragged."""
    g = gen(13)
    page, width, seqs, group = 16, 128, 3, 64
    cache = lam.RowArray(world.team(), 40 * page, width, dtype="i8", group=group)
    pages = torch.randperm(40, generator=g)
    book = [[] for _ in range(seqs)]
    kept = [[] for _ in range(seqs)]
    for step in range(20):
        slots, vals = [], torch.randn(seqs, width, generator=g).to(torch.bfloat16)
        for q in range(seqs):
            if step % (q + 1):                           # not every sequence goes on at every step
                slots.append(-1)
                continue
            at = len(book[q])
            slots.append(int(pages[q * 10 + at // page]) * page + at % page)
            book[q].append(slots[-1])
            kept[q].append(vals[q])
        cache.batch_store_rows(torch.tensor(slots, dtype=torch.int32).cuda(), vals.cuda(), pad=-1).spawn()
        flat = torch.tensor(sum(book, []), dtype=torch.int32)
        got = cache.batch_load_rows(flat.cuda(), out_dtype="f32").spawn().value()
        v = torch.stack(sum(kept, []))
        codes, scales = ref.quantise(v, "i8", group)
        exact = ref.load(ref.codes_f64(codes, "i8"), torch.arange(len(v)), 1.0, scales, group)
        check_close(got, exact, ref.load_bound(exact, "f32", 2))
    cache.wait_all()


def test_captured_sums_of_every_size(lam, world):
    """Sums of few to many records, one after the other in one graph; whole numbers, so that they are exact."""
    g = gen(77)
    sizes = [300, 900, 5003, 7001, 32768, 40000, 300001]
    tab = lam.RowArray(world.team(), 4099, 24)
    idx = [torch.zeros(n, dtype=torch.int64, device="cuda") for n in sizes]
    val = [torch.zeros(n, 24, device="cuda") for n in sizes]
    tab.batch_add_rows(idx[0], val[0]).block()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i, v in zip(idx, val):
            tab.batch_add_rows(i, v).spawn()
    exp = torch.zeros(4099, 24, dtype=torch.float64)
    for r in range(3):
        for i, v in zip(idx, val):
            i.copy_(indices(g, i.numel(), 4099, "skewed" if r % 2 else "any"))
            v.copy_(torch.randint(-8, 9, v.shape, generator=g).float())
            exp.index_add_(0, i.cpu(), v.double().cpu())
        graph.replay()
        other = lam.RowArray(world.team(), 4099, 24)                # eager work between the replays
        other.batch_add_rows(idx[3], val[3]).block()
        torch.cuda.synchronize()
        assert torch.equal(tab.local_rows().double().cpu(), exp), r


def test_two_graphs_at_once(lam, world):
    """Two captured gradients and cache writes, each with its own workspace, replayed on two streams."""
    g = gen(21)
    n, rows, width = 3000, 2000, 136
    streams, graphs, sets = [torch.cuda.Stream() for _ in range(2)], [], []
    for q in range(2):
        t = torch.randn(rows, width, generator=g)
        i, v = indices(g, n, rows, "skewed"), torch.randn(n, width, generator=g)
        a, c = lam.RowArray.from_tensor(world.team(), t.cuda()), lam.RowArray(world.team(), rows, width, dtype="i8", group=17)
        sets.append((t, i, v, a, c, i.cuda(), v.cuda()))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[q]):
            a.batch_add_rows(sets[q][5], sets[q][6], scale=0.25).spawn()
            c.batch_store_rows(sets[q][5], sets[q][6]).spawn()           # its first store is the captured one
        graphs.append(graph)
    for _ in range(3):
        for q in range(2):
            with torch.cuda.stream(streams[q]):
                graphs[q].replay()
    torch.cuda.synchronize()
    for t, i, v, a, c, _, _ in sets:
        now, total = t, 0.0                               # three calls' bounds, and this side's rounding between
        for _ in range(3):
            exact, bound = ref.add(now, i, v, 0.25)
            now, total = exact.float(), total + bound + exact.abs() * ref.U32
        check_close(a.local_rows(), exact, total)
        last = ref.last_records(i, rows)
        at, rec = torch.tensor(list(last)), torch.tensor([last[r] for r in last])
        codes, scales = ref.quantise(v[rec], "i8", 17)
        assert torch.equal(c.local_scales().cpu()[at], scales)
        assert torch.equal(c.local_rows().cpu()[at].view(torch.uint8), codes)
    world.wait_all()


def test_captured_on_a_warmed_array(lam, world):
    """Stores of many records, eager first, then captured, on the same array; replays on new inputs with
    eager stores between them, and one when the array is gone and its memory used otherwise."""
    g = gen(31)
    n, rows, width, group = 1500, 600, 40, 8
    mem, scales = torch.zeros(rows, width, dtype=torch.uint8).cuda(), torch.zeros(rows, width // group).cuda()
    a = lam.RowArray.from_tensor(world.team(), mem, scales=scales, dtype="i8")
    idx, vals = indices(g, n, rows, "any").cuda(), torch.randn(n, width, generator=g).cuda()
    a.batch_store_rows(idx, vals).block()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.batch_store_rows(idx, vals).spawn()

    def check(i, v):
        last = ref.last_records(i, rows)
        at, t = torch.tensor(list(last)), torch.tensor([last[r] for r in last])
        codes, exp = ref.quantise(v[t], "i8", group)
        assert torch.equal(scales.cpu()[at], exp) and torch.equal(mem.cpu()[at], codes)

    for r in range(4):
        if r == 3:
            torch.cuda.synchronize()
            del a
            other = [torch.full((rows,), 1 << 30, dtype=torch.int32, device="cuda") for _ in range(8)]
        i, v = indices(g, n, rows, "skewed" if r % 2 else "any"), torch.randn(n, width, generator=g)
        idx.copy_(i)
        vals.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        check(i, v)
        if r < 3:
            i, v = indices(g, 2000, rows, "any"), torch.randn(2000, width, generator=g)
            a.batch_store_rows(i.cuda(), v.cuda()).block()
            check(i, v)
    assert all((o == 1 << 30).all() for o in other)


@pytest.mark.parametrize("width", [1 << 18, (1 << 18) - 1, (1 << 18) - 8])
def test_longest_rows(lam, world, width):
    g = gen(width)
    for n in (5, 700):
        rows = 6
        a, t = float_array(lam, world, g, rows, width, "bf16")
        i = indices(g, n, rows, "any")
        got = a.batch_load_rows(i.cuda(), out_dtype="f32").block()
        assert torch.equal(got.cpu()[[0, n - 1]], t[i[[0, n - 1]]].float())
        s = lam.RowArray(world.team(), rows, width)
        s.batch_add_rows(i.cuda(), torch.ones(width, device="cuda")).block()
        assert torch.equal(s.local_rows().cpu(), torch.bincount(i, minlength=rows).float()[:, None].expand(rows, width))
    for group in (width, 4 if width % 4 == 0 else 3):
        if width % group:
            continue
        q = lam.RowArray(world.team(), rows, width, dtype="i8", group=group)
        q.batch_store_rows([3, 0], t[:2].cuda()).block()
        codes, scales = ref.quantise(t[:2], "i8", group)
        assert torch.equal(q.local_scales().cpu()[[3, 0]], scales)
        assert torch.equal(q.local_rows().cpu()[[3, 0]].view(torch.uint8), codes)
        exact = ref.load(ref.codes_f64(codes, "i8"), torch.tensor([1, 0]), 1.0, scales, group)
        check_close(q.batch_load_rows([0, 3], out_dtype="f32").block(), exact, ref.load_bound(exact, "f32", 2))


def test_batches_past_32_bits(lam, world):
    """Values and results of more than 2^32 elements."""
    n, width, rows = 70000, 65536, 10
    t = torch.arange(rows * 4).view(rows, 4).float().repeat(1, width // 4).to(torch.bfloat16)
    a = lam.RowArray.from_tensor(world.team(), t.cuda())
    i = torch.arange(n, device="cuda") % rows
    got = a.batch_load_rows(i).spawn().value()
    for k in (0, 65535, 65536, n - 11, n - 1):
        assert torch.equal(got[k].cpu(), t[k % rows]), k
    s = lam.RowArray(world.team(), rows, width)
    s.batch_add_rows(i, got).block()
    assert torch.equal(s.local_rows().cpu(), t.float() * (n // rows))     # whole numbers below 2^24
    q = lam.RowArray(world.team(), rows, width, dtype="i8", group=64)
    got[-1].fill_(1.0)
    q.batch_store_rows(i, got).block()
    assert torch.equal(q.batch_load_rows([rows - 1], out_dtype="f32").block().cpu(), torch.ones(1, width))


@pytest.mark.parametrize("kind", CODES)
def test_load_codes_far_scales(lam, world, kind):
    """scale * (code * s) where scale * s would leave f32's range (or its normal numbers) although the result
    does not, zero codes among them: the same bits for groups that are a multiple of 8 and others."""
    codes = torch.tensor([0.0, 1.0, -2.0, 3.0, 120.0, 0.0, -0.0, 96.0] * 3)
    c = codes.to(torch.int8 if kind == "i8" else torch.float8_e4m3fn).view(torch.uint8).expand(4, -1).contiguous()
    s = torch.tensor([1e30, 1e-30, 2.0 ** -126, 3.0])
    for scale in (1e10, 1e-10, 2.0 ** -120, 1.0):
        got = []
        for group in (24, 8, 12, 1):
            a = lam.RowArray.from_tensor(world.team(), c.cuda(), scales=s[:, None].expand(4, 24 // group).contiguous().cuda(), dtype=kind)
            got.append(a.batch_load_rows([0, 1, 2, 3], scale=scale, out_dtype="f32").block().cpu())
        exp = codes * s[:, None] * scale                 # two f32 roundings, in this order
        assert all(torch.equal(x, exp) for x in got), (scale, [(x != exp).nonzero().tolist() for x in got])
        assert not exp[:, 0].any() and torch.isfinite(exp[1:]).all()


def test_earlier_errors_are_left(lam, world):
    """An error that an earlier call left in the runtime is no row batch's: the batch runs, and the error is still
    there afterwards for whoever asks."""
    import ctypes
    path = next(x.split()[-1] for x in open("/proc/self/maps") if "libamdhip64" in x)
    hip = ctypes.CDLL(path)                              # the library that is loaded already
    k = world.team().kernels
    a = lam.RowArray(world.team(), 3000, 16)
    c = lam.RowArray(world.team(), 3000, 16, dtype="i8")
    idx = {n: torch.arange(n, dtype=torch.int64, device="cuda") for n in (5, 2000)}
    val = {n: torch.ones(n, 16, device="cuda") for n in idx}
    c.batch_store_rows(idx[2000], val[2000]).block()     # its claims exist
    work = torch.empty(k.lib.lmr_rows_add_workspace(a._table.ptr, 2000), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    hip.hipGetLastError()
    assert hip.hipSetDevice(1 << 20) == 101              # refused on the host
    kept = hip.hipGetDevice(ctypes.byref(ctypes.c_int())) == 0 and hip.hipPeekAtLastError() == 101
    left = []
    for n in (5, 2000):
        i, v, s = idx[n].data_ptr(), val[n].data_ptr(), k.stream_id()
        left.append(k.lib.lmr_rows_add(k.ctx, a._table.ptr, i, 8, n, 0, 0, 2.0, v, 0, 16, work.data_ptr(), work.numel(), s))
        left.append(hip.hipPeekAtLastError())
        left.append(k.lib.lmr_rows_store(k.ctx, c._table.ptr, i, 8, n, 0, 0, v, 0, 16, s))
        left.append(hip.hipPeekAtLastError())
        left.append(k.lib.lmr_rows_load(k.ctx, a._table.ptr, i, 8, n, 0, 0, 1.0, v, 0, 16, s))
        left.append(hip.hipPeekAtLastError())
    hip.hipGetLastError()
    torch.cuda.synchronize()
    assert kept and left == [0, 101] * 6, (kept, left)
    assert (a.local_rows()[:5] == 4).all() and (a.local_rows()[5:2000] == 2).all()
    assert (val[5] == 2).all() and (val[2000][:5] == 4).all() and (val[2000][5:] == 2).all()
    assert (c.local_rows()[:2000] == 127).all()
    world.wait_all()


def check_training_steps(got, steps, start, w, scale, rate, drop=None):
    """Whether the f32 rows `got` are within f32 arithmetic of the steps (indices, targets) in 64 bits; `drop`: a
    record that the plain form leaves out of every step. The bound, with U half an f32 step, follows the steps:
    a lookup is exact (scale is a power of two); a product of K terms, any order, is off by K U sum |x w|, the
    subtraction and the division by one U of their results each, a value d w by the error of d and one U; a row's
    sum, its scaling and the addition to the row as in ref.add; and the table's error so far goes through the
    lookup."""
    U = ref.U32 * (1 + 2.0 ** -10)
    s, (n, k) = abs(ref.f32_of(-rate * scale)), (len(steps[0][0]), len(w))
    exact, err, w = start.double(), torch.zeros(start.shape, dtype=torch.float64), w.double()
    for i, y in steps:
        y = y.double()
        x = exact[i] * scale
        z = x @ w - y
        d = z / n
        off = scale * err[i] @ w.abs() + U * (k * (x.abs() @ w.abs()) + z.abs())
        off = off / n + U * d.abs()
        v, voff = d[:, None] * w, off[:, None] * w.abs() + U * (d[:, None] * w).abs()
        if drop is not None:
            v[drop] = 0.0
        total, size, far = (torch.zeros_like(exact).index_add_(0, i, t) for t in (v, v.abs(), voff))
        count = torch.bincount(i, minlength=len(exact)).double()[:, None]
        new = exact - s * total
        err = err + s * far + U * (s * size * (count + 1) + (new.abs() + exact.abs()) * (count > 0))
        exact = new
    return bool(((got.cpu().double() - exact).abs() <= err).all())


def test_training_steps_to_the_last_record(lam, world):
    """Steps of a model that is a table and a vector, within the steps' own f32 bound: close enough to tell a
    single missing record."""
    g = gen(12)
    rows, width, n, rate, scale = 300, 64, 800, 0.05, 0.5
    t, w = torch.randn(rows, width, generator=g), torch.randn(width, generator=g)
    table, steps = lam.RowArray.from_tensor(world.team(), t.cuda()), []
    for _ in range(5):
        i, y = indices(g, n, rows, "skewed"), torch.randn(n, generator=g)
        x = table.batch_load_rows(i.cuda(), scale=scale).spawn().value()
        d = (x @ w.cuda() - y.cuda()) / n
        table.batch_add_rows(i.cuda(), d[:, None] * w.cuda(), scale=-rate * scale).block()
        steps.append((i, y))
    assert check_training_steps(table.local_rows(), steps, t, w, scale, rate)
    for drop in (0, 17, n - 1):
        assert not check_training_steps(table.local_rows(), steps, t, w, scale, rate, drop)


@pytest.mark.parametrize("kind", FLOATS)
@pytest.mark.parametrize("vals", FLOATS)
@pytest.mark.parametrize("n,rows,width,how", [(1025, 300, 33, "any"), (2050, 4000, 520, "skewed"), (5000, 6000, 7, "distinct"),
                                              (3000, 40, 1032, "few")])
def test_store_floats_by_claims(lam, world, kind, vals, n, rows, width, how):
    """More records than the scan of the list takes, of repeated rows, pads among them."""
    g = gen(n)
    a, t = float_array(lam, world, g, rows, width, kind)
    for _ in range(2):                                   # the second call finds the claims that the first one left
        i = indices(g, n, rows, how)
        i[::7] = -1
        v = torch.randn(n, width, generator=g).to(ref.TORCH[vals])
        a.batch_store_rows(i.cuda(), v.cuda(), pad=-1).block()
        last = ref.last_records(i, rows, -1)
        at, rec = torch.tensor(list(last)), torch.tensor([last[r] for r in last])
        t[at] = v[rec].to(ref.TORCH[kind])
        assert torch.equal(a.local_rows().cpu(), t)
