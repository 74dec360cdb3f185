"""Row batches over 1 (RCCL to itself), 2 and 3 PEs that share the box's GPU, against the plain forms
of rowref.py over every PE's records, sources in PE order."""
import os
import subprocess
import sys
import tempfile

import numpy as np
import pytest
import torch

import rowref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WORKER = os.path.join(ROOT, "tests", "dist_rows_worker.py")
pytestmark = pytest.mark.gpu


def run_pes(ws, dist_kind, env_extra, outdir, port):
    env = dict(os.environ, LMR_ROOT=ROOT, LMR_OUT=outdir, LMR_DIST=str(dist_kind), MASTER_ADDR="127.0.0.1",
               MASTER_PORT=str(port), WORLD_SIZE=str(ws), **env_extra)
    procs = [subprocess.Popen([sys.executable, "-u", WORKER], env=dict(env, RANK=str(r), LOCAL_RANK=str(r)))
             for r in range(ws)]
    try:
        rcs = [p.wait(timeout=100) for p in procs]
    finally:
        for p in procs:
            if p.poll() is None:
                p.kill()
    assert rcs == [0] * ws, rcs
    return [{k: torch.from_numpy(v) for k, v in np.load(os.path.join(outdir, f"pe{r}.npz")).items()} for r in range(ws)]


@pytest.mark.parametrize("ws,dist_kind,env", [(1, 0, {"LAMELLAR_FORCE_EXCHANGE": "1"}), (2, 0, {"LAMELLAR_COMM_BACKEND": "gloo"}),
                                              (2, 1, {"LAMELLAR_COMM_BACKEND": "gloo"}), (3, 1, {"LAMELLAR_COMM_BACKEND": "gloo"})],
                         ids=["rccl-1", "gloo-2-block", "gloo-2-cyclic", "gloo-3-cyclic"])
def test_rows_over_pes(ws, dist_kind, env):
    os.environ.setdefault("LMR_ROOT", ROOT)
    from dist_rows_worker import GROUP, ROWS, WIDTH, inputs, start
    port = 30100 + ws * 13 + dist_kind * 7 + (os.getpid() % 200)
    with tempfile.TemporaryDirectory() as d:
        pe = run_pes(ws, dist_kind, env, d, port)
    both = {c: [torch.cat(x) for x in zip(*(inputs(r, c) for r in range(ws)))] for c in ("add", "store")}
    exact, bound = ref.add(start(), both["add"][0], both["add"][1].to(torch.bfloat16), 0.5)
    codes, scales = ref.quantise(both["store"][1].to(torch.bfloat16), "e4m3", GROUP)
    last = ref.last_records(both["store"][0], ROWS)
    stored = torch.zeros(ROWS, WIDTH, dtype=torch.float64)
    at, t = torch.tensor(list(last)), torch.tensor([last[r] for r in last])
    stored[at] = ref.load(ref.codes_f64(codes, "e4m3"), t, 1.0, scales, GROUP)
    for p, r in enumerate(pe):
        assert (((r["added"].double() - exact).abs()) <= bound).all()
        assert torch.equal(r["added"], pe[0]["added"])
        got = ref.load(r["added"], r["index"], 2.0, pad=-1)
        w = r["wide"]
        assert ((w[:, 1:WIDTH + 1].double() - got).abs() <= ref.load_bound(got, "f16", 1)).all()
        assert (w[:, 0] == 3).all() and (w[:, WIDTH + 1:] == 3).all()
        assert ((r["stored"].double() - stored).abs() <= ref.load_bound(stored, "f32", 2)).all()
        assert int(r["oob"]) == 2
        assert torch.equal(r["oob_rows"], torch.stack([r["stored"][3], torch.zeros(WIDTH)]))
