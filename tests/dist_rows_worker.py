"""One PE of the row batches over several PEs (test_batch_rows_pes.py): every PE shares the box's GPU.

Runs lookups, adds and stores whose rows collide across PEs through RowArray's exchange and the HIP
kernels of every owner, and saves this PE's records and results."""
import os
import sys

import numpy as np

sys.path.insert(0, os.environ["LMR_ROOT"])
sys.path.insert(0, os.path.join(os.environ["LMR_ROOT"], "tests"))

import torch  # noqa: E402
import torch.distributed as dist  # noqa: E402

from _lamellar_bootstrap import load_package  # noqa: E402

lam = load_package()

ROWS, WIDTH, GROUP = 5003, 72, 24


def inputs(rank, case):
    """This PE's records of a case: (indices, values)."""
    n = {"add": [4000, 0, 300], "load": [700, 2500, 1], "store": [1500, 900, 0]}[case][rank]
    g = torch.Generator().manual_seed(rank * 100 + len(case))
    i = (ROWS ** torch.rand(n, generator=g)).long().clamp(max=ROWS - 1)
    return i, torch.randn(n, WIDTH, generator=g)


def start():
    return torch.randn(ROWS, WIDTH, generator=torch.Generator().manual_seed(99))


def main():
    rank, ws = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    kind = lam.Distribution(int(os.environ["LMR_DIST"]))
    world = lam.LamellarWorldBuilder().build()
    team, res = world.team(), {}
    everything = torch.arange(ROWS).cuda()
    a = lam.RowArray(team, ROWS, WIDTH, kind)
    if rank == 0:
        a.batch_store_rows(everything, start().cuda()).block()
    else:
        a.batch_store_rows([], torch.empty(0, WIDTH)).block()
    team.barrier()
    i, v = inputs(rank, "add")
    a.batch_add_rows(i.cuda(), v.to(torch.bfloat16).cuda(), scale=0.5).block()
    team.barrier()
    res["added"] = a.batch_load_rows(everything).block().cpu().numpy()
    i, _ = inputs(rank, "load")
    i[::5] = -1
    wide = torch.full((len(i), WIDTH + 5), 3.0, dtype=torch.float16).cuda()
    a.batch_load_rows(i.to(torch.int32).cuda(), scale=2.0, pad=-1, out=wide[:, 1:WIDTH + 1]).block()
    res["index"], res["wide"] = i.numpy(), wide.cpu().numpy()
    c = lam.RowArray(team, ROWS, WIDTH, kind, dtype="e4m3", group=GROUP)
    i, v = inputs(rank, "store")
    c.batch_store_rows(i.cuda(), v.to(torch.bfloat16).cuda()).block()
    team.barrier()
    res["stored"] = c.batch_load_rows(everything, out_dtype="f32").block().cpu().numpy()
    h = c.batch_load_rows(torch.tensor([3, ROWS + rank]).cuda(), out_dtype="f32")
    try:
        h.block()
        res["oob"] = np.array(0)
    except lam.LamellarError as e:
        res["oob"] = np.array(int(e.status))
    res["oob_rows"] = h.value().cpu().numpy()
    team.barrier()
    np.savez(os.path.join(os.environ["LMR_OUT"], f"pe{rank}.npz"), **res)
    dist.barrier()
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
