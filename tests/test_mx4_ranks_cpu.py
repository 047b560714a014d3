"""Data in 4 bits over several ranks: 32 neighbouring variables share a scale, so shards begin at multiples of 32 - the rounded matrix is the same
for any number of ranks, the columns come back in order, and boundaries that cut a block are refused on every rank."""
import os
import subprocess
import sys

import numpy as np
import pytest

from linearcorex_amd.comm import Comm, SingleComm
from tests import mx4_reference as R
from tests.test_distributed_cpu import free_port

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def comm(world, rank, bounds=None):
    c = Comm.__new__(Comm)
    c.world, c.rank, c.bounds = world, rank, bounds
    return c


@pytest.mark.parametrize("nv,world", [(100, 1), (100, 2), (100, 3), (100, 4), (256, 8), (257, 8), (5000, 8), (20000, 7), (33, 2), (32, 1)])
def test_shards_keep_blocks_of_32_together(nv, world):
    x = np.random.RandomState(nv).randn(3, nv)
    whole = R.round4(x)
    end = 0
    for r in range(world):
        c0, c1 = comm(world, r).shard(nv, unit=32)
        assert c0 == end and c0 % 32 == 0 and c1 > c0
        assert np.array_equal(R.round4(x[:, c0:c1]), whole[:, c0:c1])
        assert c1 - c0 <= 32 * -(-(-(-nv // 32)) // world)               # balanced to a block
        assert comm(world, 0).shard(nv, r, 32) == (c0, c1)
        end = c1
    assert end == nv and SingleComm().shard(nv, unit=32) == (0, nv)
    # the balanced split of a fit in the working precision is what it was
    assert comm(world, world - 1).shard(nv) == (nv * (world - 1) // world, nv)


def test_what_would_cut_a_block_is_refused():
    with pytest.raises(ValueError, match="blocks of 32"):
        comm(4, 0).shard(96, unit=32)
    with pytest.raises(ValueError, match="must stay together"):
        comm(2, 0, [0, 40, 100]).shard(100, unit=32)
    c = comm(2, 1, [0, 64, 100])
    assert c.shard(100, unit=32) == (64, 100) and comm(2, 0, [0, 40, 100]).shard(100) == (0, 40)


def test_two_ranks_cut_and_gather_whole_blocks():
    code = r'''
import os, sys
sys.path.insert(0, %r)
import numpy as np
import torch
import torch.distributed as dist
rank = int(sys.argv[1])
dist.init_process_group("gloo", rank=rank, world_size=2, init_method="tcp://127.0.0.1:%d")
from linearcorex_amd import Corex
from linearcorex_amd.comm import Comm
model = Corex(n_hidden=3, x_storage="mx4", comm=Comm())
model.nv, model._ex = 100, (None, torch.zeros(1))
c0, c1 = model._shard()
assert (c0, c1) == ((0, 64) if rank == 0 else (64, 100)), (c0, c1)
full = np.arange(300, dtype=np.float32).reshape(3, 100)
assert np.array_equal(model._gather(full[:, c0:c1]), full)
assert np.array_equal(model._gather(np.ascontiguousarray(full[:, c0:c1].T), "X_i Z_j"), full.T)
dense = Corex(n_hidden=3, comm=Comm())
dense.nv, dense._ex = 100, model._ex
assert dense._shard() == ((0, 50) if rank == 0 else (50, 100))
assert np.array_equal(dense._gather(full[:, 50 * rank:50 * rank + 50]), full)
cut = Corex(n_hidden=3, x_storage="mx4", comm=Comm(bounds=[0, 40, 100]))
try:
    cut.fit(np.random.RandomState(0).randn(10, 100))
    raise SystemExit("a cut block was accepted")
except ValueError as e:
    assert "must stay together" in str(e), e
dist.barrier()
dist.destroy_process_group()
print("RANKS_OK")
''' % (ROOT, free_port())
    procs = [subprocess.Popen([sys.executable, "-c", code, str(r)], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True) for r in range(2)]
    for p in procs:
        out, err = p.communicate(timeout=180)
        assert p.returncode == 0 and "RANKS_OK" in out, (out[-500:], err[-2000:])
