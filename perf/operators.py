"""What the row operators are measured on: lookup, its gradient, the 8-bit cache's write and read.

A case names one operator and its sizes. `run` is one pass as a user's program makes it; with `own` false
the same arithmetic in elementary torch operations.

  lookup    out[t] = scale * table[index[t]], rounded to the output's type
  gradient  table[r] += scale * sum of grads[t] over the t with index[t] = r, in 32 bits, rounded once
  write     rows quantised to 8 bits with a scale per group as they are stored, then read back
  read      rows of the 8-bit cache by index, as values of 16 or 32 bits
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "e4m3": 1}
LARGEST = {"i8": 127.0, "e4m3": 448.0}     # the largest code
LEAST = 2.0 ** -126                        # the least scale of a group
PAGE = 16                                  # cache rows a page holds
ZIPF = 2.7                                 # tokens are drawn with weight 1 / (rank + ZIPF)

_world = []


def team():
    """The one-PE world that a user's program builds once."""
    if not _world:
        from _lamellar_bootstrap import load_package
        _world.append(load_package().LamellarWorldBuilder().build())
    return _world[0].team()


def listed():
    return [
        # the next token of 16 sequences being served
        dict(name="lookup 16 bf16", op="lookup", n=16, rows=32768, width=4096, kind="bf16", out="bf16", scale=1.0),
        # a training batch, 32-bit weights read as bf16 activations, scaled by sqrt(width)
        dict(name="lookup 8191 f32", op="lookup", n=8191, rows=50257, width=2048, kind="f32", out="bf16", scale=2048 ** 0.5),
        # a long batch over a large vocabulary
        dict(name="lookup 65536 bf16", op="lookup", n=65536, rows=131072, width=4096, kind="bf16", out="bf16", scale=1.0),
        # a small fine-tuning batch, gradients in 32 bits
        dict(name="gradient 500 f32", op="gradient", n=500, rows=32000, width=1024, kind="f32", vals="f32", scale=1.0),
        # a training batch: bf16 gradients into a 32-bit accumulator
        dict(name="gradient 16384 bf16", op="gradient", n=16384, rows=50257, width=2048, kind="f32", vals="bf16", scale=2048 ** 0.5),
        # the same of a large model and batch
        dict(name="gradient 131072 bf16", op="gradient", n=131072, rows=131072, width=4096, kind="f32", vals="bf16", scale=1.0),
        # 16-bit weights and an odd width
        dict(name="gradient 5003 f16", op="gradient", n=5003, rows=20011, width=1001, kind="f16", vals="f16", scale=0.5),
        # one new row for each of 64 sequences being served, some of the batch's places empty
        dict(name="write 64 e4m3", op="write", n=64, rows=65536, width=1024, group=128, kind="e4m3", vals="bf16", packed=3, empty=5),
        # a prompt, the rows a third of a fused projection's
        dict(name="write 16384 i8", op="write", n=16384, rows=131072, width=2048, group=128, kind="i8", vals="bf16", packed=3, empty=0),
        # heads of 80 values in f16
        dict(name="write 4099 e4m3", op="write", n=4099, rows=16384, width=640, group=80, kind="e4m3", vals="f16", packed=1, empty=0),
        # the context of one sequence
        dict(name="read 2000 i8", op="read", n=2000, rows=65536, width=1024, group=128, kind="i8", out="f16", scale=1.0),
        # the contexts of many sequences
        dict(name="read 262144 e4m3", op="read", n=262144, rows=524288, width=1024, group=128, kind="e4m3", out="bf16", scale=1.0),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["lookup", "gradient", "write", "read"])
    case = dict(op=op)
    if op in ("lookup", "gradient"):
        n = _between(rng, 1, 131072)
        width = _between(rng, 64, 8192)
        if rng.random() < 0.7:
            width = -(-width // 64) * 64
        width = max(64, min(width, (1 << 28) // n))
        rows = max(1000, min(_between(rng, 1000, 262144), (1 << 29) // width))
        case.update(n=n, rows=rows, width=width, kind=rng.choice(["f32", "f16", "bf16"]),
                    scale=rng.choice([1.0, round(math.sqrt(width), 3), 0.125]))
        case["out" if op == "lookup" else "vals"] = rng.choice(["f32", "f16", "bf16"])
        return case
    n = _between(rng, 1, 262144 if op == "read" else 65536)
    group = rng.choice([32, 64, 64, 80, 96, 100, 128, 128, 128, 192, 256, 576])
    width = group * min(_between(rng, 1, 32), 4096 // group)
    width = max(group, min(width, (1 << 28) // n // group * group))
    rows = max(256, -(-n * rng.choice([1, 2, 3]) // PAGE) * PAGE + 256)
    case.update(n=n, rows=rows, width=width, group=group, kind=rng.choice(["i8", "e4m3"]))
    if op == "write":
        case.update(vals=rng.choice(["f32", "f16", "bf16"]), packed=rng.choice([1, 2, 3]), empty=rng.choice([0, 0, n // 8]))
    else:
        case.update(out=rng.choice(["f32", "f16", "bf16"]), scale=rng.choice([1.0, 0.5]))
    return case


def _tokens(g, n, rows):
    """Token ids as text has them: few frequent ones, many rare ones, in no order of the table."""
    weight = 1.0 / (torch.arange(rows, device="cuda", dtype=torch.float64) + ZIPF)
    upto = torch.cumsum(weight, 0)
    rank = torch.searchsorted(upto, torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * upto[-1])
    place = torch.randperm(rows, generator=g, device="cuda")
    return place[rank.clamp_(max=rows - 1)]


def _slots(g, n, rows):
    """n cache rows: pages in any order, the last page used in part."""
    page = torch.randperm(rows // PAGE, generator=g, device="cuda")[: -(-n // PAGE)]
    slot = page[:, None] * PAGE + torch.arange(PAGE, device="cuda")
    return slot.reshape(-1)[:n].to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, n, rows, width = case, case["n"], case["rows"], case["width"]
    s = dict(case=case)
    if c["op"] in ("lookup", "gradient"):
        s["table"] = torch.randn(rows, width, generator=g, device="cuda").mul_(0.02).to(TYPES[c["kind"]])
        s["index"] = _tokens(g, n, rows)
        if c["op"] == "gradient":
            s["vals"] = torch.randn(n, width, generator=g, device="cuda").mul_(0.01).to(TYPES[c["vals"]])
        if own:
            s["array"] = _package().RowArray.from_tensor(team(), s["table"])
        return s
    s["index"] = _slots(g, n, rows)
    loud = torch.exp(torch.randn(rows, width // c["group"], generator=g, device="cuda"))   # groups differ in size
    if c["op"] == "write":
        whole = torch.randn(n, c["packed"] * width, generator=g, device="cuda")
        whole.view(n, -1, c["group"]).mul_(loud[:n].repeat(1, c["packed"])[:, :, None])
        s["vals"] = whole.to(TYPES[c["vals"]])[:, width * (c["packed"] - 1):]
        if c["empty"]:
            s["index"][torch.randperm(n, generator=g, device="cuda")[: c["empty"]]] = -1
        s["codes"] = torch.zeros(rows, width, dtype=torch.uint8, device="cuda")
        s["scales"] = torch.zeros(rows, width // c["group"], device="cuda")
    else:
        x = torch.randn(rows, width, generator=g, device="cuda")
        if c["kind"] == "i8":
            s["codes"] = x.mul_(40.0).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
        else:
            s["codes"] = x.mul_(140.0).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        s["scales"] = loud / LARGEST[c["kind"]]
    if own:
        s["array"] = _package().RowArray.from_tensor(team(), s["codes"], scales=s["scales"], dtype=c["kind"])
    return s


def _package():
    from _lamellar_bootstrap import load_package
    return load_package()


def _values(codes, kind):
    return codes.view(torch.int8 if kind == "i8" else torch.float8_e4m3fn).to(torch.float32)


def _quantise(vals, kind, group):
    x = vals.to(torch.float32).reshape(vals.shape[0], -1, group)
    scale = (x.abs().amax(-1) * (1.0 / LARGEST[kind])).clamp(min=LEAST)
    y = x * torch.reciprocal(scale)[:, :, None]
    codes = torch.round(y).to(torch.int8) if kind == "i8" else y.to(torch.float8_e4m3fn)
    return codes.view(torch.uint8).reshape(vals.shape), scale


def _read(s, index, kind, group, scale, out):
    """The rows as `out`, those of index -1 empty."""
    at = index.clamp(min=0).long()
    v = _values(s["codes"][at], kind).view(index.numel(), -1, group) * s["scales"][at][:, :, None] * scale
    return torch.where((index >= 0)[:, None], v.view(index.numel(), -1), 0.0).to(out)


def run(s):
    c = s["case"]
    if own:
        a = s["array"]
        if c["op"] == "lookup":
            return a.batch_load_rows(s["index"], scale=c["scale"], out_dtype=c["out"]).spawn().value()
        if c["op"] == "gradient":
            a.batch_add_rows(s["index"], s["vals"], scale=c["scale"]).spawn()
            return s["table"]
        if c["op"] == "write":
            a.batch_store_rows(s["index"], s["vals"], pad=-1).spawn()
            return a.batch_load_rows(s["index"], out_dtype=c["vals"], pad=-1).spawn().value()
        return a.batch_load_rows(s["index"], scale=c["scale"], out_dtype=c["out"]).spawn().value()
    if c["op"] == "lookup":
        return (s["table"][s["index"]].to(torch.float32) * c["scale"]).to(TYPES[c["out"]])
    if c["op"] == "gradient":
        named, place = torch.unique(s["index"], return_inverse=True)
        acc = torch.zeros(named.numel(), c["width"], device="cuda")
        acc.index_add_(0, place, s["vals"].to(torch.float32))
        s["table"][named] = (s["table"][named].to(torch.float32) + acc * c["scale"]).to(s["table"].dtype)
        return s["table"]
    if c["op"] == "write":
        codes, scale = _quantise(s["vals"], c["kind"], c["group"])
        if c["empty"]:
            used = s["index"] >= 0
            at, codes, scale = s["index"][used].long(), codes[used], scale[used]
        else:
            at = s["index"].long()
        s["codes"][at] = codes
        s["scales"][at] = scale
        return _read(s, s["index"], c["kind"], c["group"], 1.0, TYPES[c["vals"]])
    return _read(s, s["index"], c["kind"], c["group"], c["scale"], TYPES[c["out"]])


def work(case):
    c, n, width = case, case["n"], case["width"]
    if c["op"] in ("lookup", "gradient"):
        # rows that n tokens name, in the mean
        weight = 1.0 / (torch.arange(c["rows"], dtype=torch.float64) + ZIPF)
        named = float((-torch.expm1(n * torch.log1p(-weight / weight.sum()))).sum())
        if c["op"] == "lookup":
            return {"bytes": named * width * BYTES[c["kind"]] + n * width * BYTES[c["out"]] + 8 * n, "flops": n * width}
        return {"bytes": n * width * BYTES[c["vals"]] + 2 * named * width * BYTES[c["kind"]] + 8 * n,
                "flops": n * width + 2 * named * width}
    groups = width // c["group"]
    if c["op"] == "write":      # values in, codes and scales out; read back: codes and scales in, values out
        used = n - c["empty"]
        return {"bytes": used * width * BYTES[c["vals"]] + 2 * used * (width + 4 * groups) + n * width * BYTES[c["vals"]] + 8 * n, "flops": 4 * n * width}
    return {"bytes": n * (width + 4 * groups) + n * width * BYTES[c["out"]] + 4 * n, "flops": 2 * n * width}


def exact(case, seed):
    s = prepare(case, seed)
    c, n = case, case["n"]
    if c["op"] == "lookup":
        out = torch.empty(n, c["width"], dtype=torch.float64, device="cuda")
        for a in range(0, n, 8192):
            torch.mul(torch.index_select(s["table"], 0, s["index"][a:a + 8192]).double(), c["scale"], out=out[a:a + 8192])
        return out
    if c["op"] == "gradient":
        total = s["table"].double()
        for a in range(0, n, 8192):
            total.index_put_((s["index"][a:a + 8192],), s["vals"][a:a + 8192].double() * c["scale"], accumulate=True)
        return total
    out = torch.zeros(n, c["width"], dtype=torch.float64, device="cuda")
    for a in range(0, n, 8192):
        at = s["index"][a:a + 8192]
        live = at >= 0
        if c["op"] == "write":
            x = s["vals"][a:a + 8192].double().reshape(at.numel(), -1, c["group"])
            step = x.abs().amax(-1, keepdim=True) / LARGEST[c["kind"]]
            y = torch.where(step > 0, x / step.clamp(min=1e-300), 0.0)
            if c["kind"] == "i8":
                y = torch.round(y)
            else:          # 3 bits behind the leading one, 2^-9 the least step; halves go to the even code
                unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                y = torch.round(y / unit) * unit
            v = (y * step).reshape(at.numel(), -1)
        else:
            code = s["codes"][at.clamp(min=0).long()]
            code = code.view(torch.int8).double() if c["kind"] == "i8" else code.view(torch.float8_e4m3fn).double()
            v = code * s["scales"][at.clamp(min=0).long()].double().repeat_interleave(c["group"], dim=1) * c["scale"]
        out[a:a + 8192] = torch.where(live[:, None], v, 0.0)
    return out
