"""A rank that is done ends its process group and the group's threads."""
import os
import socket

import pytest
import torch
import torch.multiprocessing as mp

pytestmark = pytest.mark.timeout(300)


def _threads():
    return len(os.listdir("/proc/self/task"))


def _rank(rank, port, out):
    os.environ.update(RANK=str(rank), LOCAL_RANK=str(rank), WORLD_SIZE="2",
                      MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    import torch.distributed as dist
    from pytorch_distributed_train_amd.flags import DistEnv
    from pytorch_distributed_train_amd.parallel.comm import (TorchDistComm,
                                                             shutdown)
    shutdown()  # nothing to end yet
    torch.set_num_threads(1)
    before = _threads()
    comm = TorchDistComm(DistEnv.from_env())
    t = torch.ones(1000) * (rank + 1)
    comm.allreduce_sum(t).wait()
    assert bool((t == 3).all())
    during = _threads()
    shutdown()
    assert not dist.is_initialized()
    shutdown()
    torch.save((before, during, _threads()), f"{out}/{rank}.pt")


def test_shutdown_joins_the_groups_threads(tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_rank, args=(port, str(tmp_path)), nprocs=2)
    for r in range(2):
        before, during, after = torch.load(tmp_path / f"{r}.pt")
        assert during > before  # the group's threads
        assert after < during, (before, during, after)
