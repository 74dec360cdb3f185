"""Plain 64-bit forms of the row operators, and how far f32 arithmetic may be from them (test-only).

Bounds count half a step per rounding: u(t) = finfo(t).eps / 2 relative, or half the least subnormal
step where a result is below the normal range."""
import torch

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LARGEST = {"i8": 127.0, "e4m3": 448.0}
U32 = 2.0 ** -24
LEAST_STEP = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}


def u(t):
    return torch.finfo(TORCH[t]).eps / 2


def live_rows(idx, rows, pad=None):
    """(mask of the records that name a row, whether some other one is out of bounds)"""
    i = idx.to(torch.int64)
    inside = (i >= 0) & (i < rows)
    padded = (i == pad) if pad is not None else torch.zeros_like(inside)
    return inside & ~padded, bool((~inside & ~padded).any())


def f32_of(x):
    """A Python float as the f32 it is passed as, in 64 bits."""
    return float(torch.tensor(x, dtype=torch.float32))


def codes_f64(codes, kind):
    return codes.view(torch.int8 if kind == "i8" else torch.float8_e4m3fn).to(torch.float32).double()


def load(table, idx, scale=1.0, scales=None, group=None, pad=None):
    """table: values (any float type) or f64 codes with their scales"""
    live, _ = live_rows(idx, table.shape[0], pad)
    at = torch.where(live, idx.to(torch.int64), 0)
    v = table[at].double()
    if scales is not None:
        v = v * scales[at].double().repeat_interleave(group, dim=1)
    return torch.where(live[:, None], v * f32_of(scale), 0.0)


def load_bound(exact, out, roundings):
    """`roundings` in f32 (products), then one to the output's type."""
    return exact.abs() * (u(out) + roundings * U32) * (1 + 2.0 ** -10) + LEAST_STEP[out]


def add(table, idx, vals, scale=1.0, pad=None):
    """(the rows after, how far f32 sums and one rounding to the table's type may be off)"""
    rows = table.shape[0]
    live, _ = live_rows(idx, rows, pad)
    at = idx.to(torch.int64)[live]
    v = vals.double().expand(idx.numel(), table.shape[1])[live]
    s = f32_of(scale)
    total = torch.zeros(table.shape, dtype=torch.float64).index_add_(0, at, v)
    size = torch.zeros(table.shape, dtype=torch.float64).index_add_(0, at, v.abs())
    count = torch.zeros(rows, dtype=torch.float64).index_add_(0, at, torch.ones(at.numel(), dtype=torch.float64))
    exact = table.double() + s * total
    kind = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}[table.dtype]
    # m - 1 additions of the sum, each at most half a step of a partial sum (<= size), the product
    # with the scale and the addition to the row, then the rounding to the row's type
    bound = U32 * (abs(s) * size * (count[:, None] + 1) + exact.abs() + table.double().abs())
    bound = bound * (1 + 2.0 ** -10) + exact.abs() * u(kind) * (1 + 2.0 ** -10) + LEAST_STEP[kind]
    bound[count == 0] = 0.0                            # rows that no record names keep their bits
    return exact, bound


def quantise(vals, kind, group):
    """The stored codes and scales, rounding by rounding in f32: (uint8 codes, f32 scales)."""
    x = vals.to(torch.float32).reshape(vals.shape[0], -1, group)
    top = x.abs().amax(-1)
    fine = torch.isfinite(top)
    inv_q = torch.tensor(1.0 / LARGEST[kind], dtype=torch.float32)
    scale = (torch.where(fine, top, 0.0) * inv_q).clamp(min=2.0 ** -126)
    y = torch.where(fine[:, :, None], x, 0.0) * (1.0 / scale)[:, :, None]
    codes = torch.round(y).to(torch.int8) if kind == "i8" else y.to(torch.float8_e4m3fn)
    scale = torch.where(fine, scale, float("nan"))
    return codes.view(torch.uint8).reshape(vals.shape), scale


def last_records(idx, rows, pad=None):
    """{row: the last record that names it}"""
    live, _ = live_rows(idx, rows, pad)
    return {int(r): t for t, (r, ok) in enumerate(zip(idx.tolist(), live.tolist())) if ok}
