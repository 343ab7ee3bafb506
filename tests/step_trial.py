"""tests/step_trial.py -- eight steps of the B = 6 training loop with look-ahead in a process of its own, on the default schedule.

    python tests/step_trial.py <streams used before the Trainer exists>

Child process of tests/test_step_gpu.py: where the step's streams sit among the streams of a process depends on what used streams before
it.  SCP_FORCE_COLLECTIVES=1 adds the multi-GPU schedule's communication stream (one-rank RCCL group).  Every host wait is bounded
(SCP_DEVICE_TIMEOUT_S).  Prints one line: OK, or the DeviceStall."""
import os
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "self-corr-pose_amd"), os.path.join(ROOT, "tests")):
    sys.path.insert(0, p)
os.environ.setdefault("SCP_DEVICE_TIMEOUT_S", "45")

import numpy as np  # noqa: E402
import torch  # noqa: E402

n_pre, t0 = int(sys.argv[1]), time.time()
pre = [torch.cuda.Stream() for _ in range(n_pre)]
for s in pre:
    with torch.cuda.stream(s):
        torch.zeros(8, device="cuda").add_(1.0)
torch.cuda.synchronize()

import scp_amd.dino as dino  # noqa: E402
from scp_amd import streams, synthetic  # noqa: E402
from scp_amd.flags import Options  # noqa: E402
from scp_amd.trainer import Trainer  # noqa: E402

dino.ALLOW_RANDOM_INIT = True
if os.environ.get("SCP_FORCE_COLLECTIVES") == "1":
    import socket
    import torch.distributed as dist
    with socket.socket() as _s:
        _s.bind(("127.0.0.1", 0))
        _port = _s.getsockname()[1]
    os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
    os.environ.setdefault("MASTER_PORT", str(_port))
    dist.init_process_group("nccl", rank=0, world_size=1)
try:
    opts = Options("laptop_wild6d", batch_size=2, repeat=3, train=True, total_iters=100, img_size=256, ngpu=1, local_rank=-1)
    torch.manual_seed(0)
    tr = Trainer(opts, prior=synthetic.bottle_like(3), device="cuda")
    batches = [synthetic.make_batch(2, 3, 256, seed=10 + k, device="cuda") for k in range(8)]
    hist, pending = [], []
    for i, data in enumerate(batches):
        total, aux, grad = tr.step(data, next_data=batches[i + 1] if i + 1 < len(batches) else None)
        pending.append(total.detach())
        if (i + 1) % 2 == 0:
            hist += tr._read_back(pending, "steps %d..%d" % (i, i + 1))
            pending = []
    assert np.isfinite(hist).all(), hist
    print("OK   pre=%d  %.1f s" % (n_pre, time.time() - t0), flush=True)
    os._exit(0)
except streams.DeviceStall as e:
    print("HANG pre=%d  %.1f s  %s" % (n_pre, time.time() - t0, e), flush=True)
    os._exit(3)
