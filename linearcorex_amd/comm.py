"""Sharding of the n_variables axis across ranks (one process per GPU) and the exchange steps.

torch.distributed is used as plumbing only: backend "nccl" is RCCL over xGMI on the GPU box, "gloo"
in the CPU tests.  The algorithm needs, per moment evaluation:
    L1  all-reduce(sum) of  [ Y_partial (n_samples x m) | W_p.W_p^T (m x m) ]   -> `allreduce_y`
    L2  all-reduce(sum) of 2 scalars                                             -> `allreduce_s(2)`
and per update: H (m x m), [Y_g | Bj], and the tangent scalar.  With one rank every call is a no-op.
"""
from __future__ import annotations

import numpy as np


class _FirstContactWatchdog:
    """Bounds first contact with a transport (LCX_FIRST_CONTACT_TIMEOUT_S, default 600 s, 0 = unbounded).  A rank that blocks inside
    ncclCommInitRank - or in the group collectives around it because ANOTHER rank blocks there - cannot be rescued in-process (RCCL's own
    contract), and waiting forever turns one bad link into a job that never reports: after the limit the rank says which step it was in,
    dumps the stacks of all its threads and exits with code 3.  Whoever started the ranks sees a non-zero exit and may start a FRESH set
    on another transport (benchkit/launch.py does); nothing is retried inside this process."""

    def __init__(self, rank):
        import os
        try:
            self.seconds = float(os.environ.get("LCX_FIRST_CONTACT_TIMEOUT_S", "600"))
        except ValueError:
            self.seconds = 600.0
        self.rank, self.what, self.timer, self.t0 = rank, "start", None, 0.0

    def step(self, what):
        self.what = what

    def _fire(self):
        import faulthandler
        import os
        import sys
        import time
        sys.stderr.write("linearcorex_amd: rank %d: first contact with the exchange transport did not finish within %.0f s "
                         "(LCX_FIRST_CONTACT_TIMEOUT_S); step in progress for this rank: %s (%.0f s since bind_engine began).  "
                         "Stacks of all threads follow; exiting with code 3 - start a fresh set of ranks, e.g. with LCX_EXCHANGE=hook\n"
                         % (self.rank, self.seconds, self.what, time.time() - self.t0))
        try:
            faulthandler.dump_traceback(file=sys.stderr, all_threads=True)
            sys.stderr.flush()
        finally:
            os._exit(3)

    def __enter__(self):
        import threading
        import time
        self.t0 = time.time()
        if self.seconds > 0:
            self.timer = threading.Timer(self.seconds, self._fire)
            self.timer.daemon = True
            self.timer.start()
        return self

    def __exit__(self, *exc):
        if self.timer is not None:
            self.timer.cancel()
        return False


class Comm:
    def __init__(self, group=None, always_exchange=False, bounds=None):
        """always_exchange: issue every exchange step even in a group of one rank (the all-reduces are then
        identities).  Used to run the multi-rank device path - the world>1 kernels of the engine, the bound
        exchange tensors and real RCCL launches on the engine's stream - on a single GPU.
        bounds: explicit column boundaries of the shards, `world + 1` non-decreasing integers from 0 to n_variables (rank r
        holds columns [bounds[r], bounds[r+1]), at least one each) instead of the balanced split - GPUs with unequal free
        memory, and the tests' awkward shards.  The same on every rank."""
        import torch.distributed as dist
        self._dist = dist
        self.group = group
        self.rank = dist.get_rank(group)
        self.world = dist.get_world_size(group)
        self.exchange = self.world > 1 or bool(always_exchange)
        self.selftest_seconds = None       # seconds one Y-buffer all-reduce took in the transport's first-contact test (bind_engine)
        self.bounds = None
        err = None
        if bounds is not None:
            b = [int(t) for t in bounds]
            if len(b) != self.world + 1 or b[0] != 0 or any(b[k + 1] <= b[k] for k in range(self.world)):
                err = "bounds must be %d increasing column boundaries starting at 0" % (self.world + 1)
            else:
                self.bounds = b
        if self.world > 1:
            # "the same on every rank" is checked, not assumed: shard widths enter the padding of the gathers and the global column
            # map - ranks that disagree would hang or gather wrong columns without an error.  Every rank takes part (balanced split =
            # all -1), and the verdict is rank-identical, so all of them raise together.
            import torch
            mine = (self.bounds if self.bounds is not None else [-1] * (self.world + 1)) + [1 if err else 0]
            dev = torch.device("cuda", torch.cuda.current_device()) if dist.get_backend(group) == "nccl" else "cpu"
            t = torch.tensor(mine + [-v for v in mine], dtype=torch.int64, device=dev)
            dist.all_reduce(t, op=dist.ReduceOp.MAX, group=group)
            t = [int(v) for v in t.cpu()]
            hi, lo = t[:len(mine)], [-v for v in t[len(mine):]]
            if hi[-1]:
                raise ValueError(err or "another rank passed malformed shard bounds")
            if hi != lo:
                raise ValueError("rank %d: Comm(bounds=...) differs across the ranks: mine %r, elementwise max %r, min %r"
                                 % (self.rank, mine[:-1], hi[:-1], lo[:-1]))
        elif err:
            raise ValueError(err)

    # contiguous column ranges: balanced, or the caller's boundaries.  unit: shards begin at multiples of it (variables that must stay together)
    def shard(self, nv, rank=None, unit=1):
        r = self.rank if rank is None else rank
        if self.bounds is not None:
            if self.bounds[-1] != nv:
                raise ValueError("shard boundaries end at %d, the data have %d variables" % (self.bounds[-1], nv))
            if any(b % unit for b in self.bounds[:-1]):
                raise ValueError("shard boundaries %r: %d neighbouring variables must stay together" % (self.bounds, unit))
            return self.bounds[r], self.bounds[r + 1]
        if unit > 1 and self.world > 1:
            blocks = -(-nv // unit)
            if blocks < self.world:
                raise ValueError("%d variables in blocks of %d do not give each of %d ranks one" % (nv, unit, self.world))
            return blocks * r // self.world * unit, min(nv, blocks * (r + 1) // self.world * unit)
        return (nv * r) // self.world, (nv * (r + 1)) // self.world

    def allreduce(self, tensor):
        if self.exchange:
            self._dist.all_reduce(tensor, op=self._dist.ReduceOp.SUM, group=self.group)

    def allreduce_max(self, tensor):
        if self.exchange:
            self._dist.all_reduce(tensor, op=self._dist.ReduceOp.MAX, group=self.group)

    def barrier(self):
        if self.world > 1:
            self._dist.barrier(group=self.group)

    def bind_engine(self, backend, first_contact=True):
        """Move the exchange steps into the engine (include/lcx.h, 'exchange inside the library'): afterwards the levels of
        the C ABI all-reduce what they produce themselves and `lcx_iterate` serves several ranks.  Returns the transport
        name, or None when the backend has no in-library exchange (the NumPy test double) or LCX_EXCHANGE=torch asks for
        the host-sequenced path (torch.distributed between the level calls - kept selectable).

        RCCL group ("nccl"): the handle gets an RCCL communicator of its own - rank 0 draws the unique id, which travels
        through this group's broadcast - and issues ncclAllReduce on its stream.  Any other backend (gloo in the tests, two
        ranks sharing one GPU): a hook that runs this group's all_reduce on a zero-copy view of the device buffer."""
        import os
        mode = os.environ.get("LCX_EXCHANGE", "engine")
        if mode == "torch" or not self.exchange or not hasattr(backend, "comm_init"):
            return None
        with _FirstContactWatchdog(self.rank) as dog:
            return self._bind_engine(backend, first_contact, mode, dog)

    def _bind_engine(self, backend, first_contact, mode, dog):
        import os
        import sys
        import torch
        # first_contact=False: a temporary handle beside one whose transport already passed (same group, same kind).  That holds
        # literally for the hook (the same process group carries it); an RCCL handle owns a brand-new communicator from a fresh
        # ncclCommInitRank, so it is always tested
        run_selftest = bool(first_contact)
        if run_selftest:
            self.selftest_seconds = None

        def agreed(flag, dev):
            """MAX over the ranks of a local failure flag, on this group (every rank calls it at the same point)"""
            with backend.stream_context():
                bad = torch.tensor([1.0 if flag else 0.0], device=dev)
                self._dist.all_reduce(bad, op=self._dist.ReduceOp.MAX, group=self.group)
                return float(bad.item()) > 0

        def selftest(dev, what):
            """lcx_comm_selftest on every rank; its verdict is shared inside the test itself (rank-identical), the MAX over the
            ranks on top covers a rank that could not even run it"""
            err = None
            if (run_selftest or what == "rccl") and os.environ.get("LCX_COMM_SELFTEST", "1") not in ("", "0"):
                try:
                    if os.environ.get("LCX_TEST_FAIL_COMM_INIT") == "selftest" and what == "rccl":
                        raise RuntimeError("LCX_TEST_FAIL_COMM_INIT=selftest")
                    secs = backend.comm_selftest(self.rank)
                    if run_selftest:
                        self.selftest_seconds = secs
                except Exception as e:       # noqa: BLE001 - reported by the caller, on every rank
                    err = "lcx_comm_selftest (%s): %s" % (what, e)
            return err

        # (LCX_TEST_FORCE_RCCL_NEGOTIATION: a test hook - run the negotiation below on a non-RCCL group, where two ranks can share one
        # GPU, to exercise a ONE-SIDED failure; only meaningful together with a forced failure before ncclCommInitRank)
        negotiate = self._dist.get_backend(self.group) == "nccl" or bool(os.environ.get("LCX_TEST_FORCE_RCCL_NEGOTIATION"))
        if negotiate and mode != "hook":
            # The group agrees on every step BEFORE a rank commits to a collective the others might not enter:
            #   1. every rank probes librccl locally (dlopen) and the flags are MAX-reduced on this group - ncclCommInitRank is
            #      collective, a rank that raised before entering it would leave the others blocked inside it;
            #   2. rank 0 draws the id, which reaches every rank (or None) through the group's broadcast;
            #   3. after ncclCommInitRank the ranks MAX-reduce a failure flag (a failure INSIDE CommInitRank on some ranks only
            #      is fatal by RCCL's own contract - bounded by its timeout, not by this code);
            #   4. lcx_comm_selftest: the communicator must SUM at the real buffer size and give every rank the same bits.
            # If the library's own communicator is not to be had, every rank says so loudly and takes the hook transport below
            # (this group's RCCL all_reduce on the same device buffers, lcx_iterate still inside the library) - never a silent
            # or a one-sided change.
            dev = torch.device("cuda", backend.device)
            err, box = None, [None]
            forced = os.environ.get("LCX_TEST_FAIL_COMM_INIT", "")
            can = True
            dog.step("librccl probe (dlopen)")
            try:
                if forced == "probe" or forced == "probe:%d" % self.rank:
                    raise RuntimeError("LCX_TEST_FAIL_COMM_INIT=%s" % forced)
                backend.comm_probe()
            except Exception as e:           # noqa: BLE001
                can, err = False, "librccl probe: %s" % e
            dog.step("agreeing on the librccl probe (all_reduce on the process group)")
            if agreed(not can, dev):
                err = err or "another rank cannot load librccl"
            else:
                dog.step("unique id: ncclGetUniqueId on rank 0, broadcast on the process group")
                if self.rank == 0:
                    try:
                        if forced == "id":
                            raise RuntimeError("LCX_TEST_FAIL_COMM_INIT=id")
                        box = [backend.comm_unique_id()]
                    except Exception as e:       # noqa: BLE001 - reported below, on every rank
                        err = "lcx_comm_unique_id: %s" % e
                src = self._dist.get_global_rank(self.group, 0) if self.group is not None else 0
                self._dist.broadcast_object_list(box, src=src, group=self.group, device=dev)
                if box[0] is not None:
                    dog.step("ncclCommInitRank of the handle's own communicator (lcx_comm_init)")
                    try:
                        if forced == "init":
                            raise RuntimeError("LCX_TEST_FAIL_COMM_INIT=init")
                        if os.environ.get("LCX_TEST_HANG_COMM_INIT") in ("all", str(self.rank)):
                            import time          # test hook: this rank never arrives in ncclCommInitRank - the others block inside it
                            time.sleep(10 ** 6)
                        backend.comm_init(self.world, self.rank, box[0])
                    except Exception as e:       # noqa: BLE001
                        err = "lcx_comm_init: %s" % e
                elif err is None:
                    err = "rank 0 could not draw an RCCL unique id"
                dog.step("agreeing on the outcome of ncclCommInitRank (all_reduce on the process group)")
                if agreed(err is not None, dev):
                    err = err or "another rank failed"
                else:
                    dog.step("lcx_comm_selftest on the handle's RCCL communicator")
                    err = selftest(dev, "rccl")
                    dog.step("agreeing on the self-test (all_reduce on the process group)")
                    if agreed(err is not None, dev):
                        err = err or "another rank failed the self-test"
            if err is None:
                return "rccl"
            print("linearcorex_amd: rank %d: the engine's own RCCL communicator is not available (%s); every rank exchanges "
                  "through this process group's all_reduce instead (LCX_EXCHANGE=hook)" % (self.rank, err),
                  file=sys.stderr, flush=True)
            backend.set_exchange_hook(None)                  # drops a communicator this rank may have got

        class _View:                        # zero-copy: torch.as_tensor understands __cuda_array_interface__
            def __init__(self, ptr, count, dtype):
                self.__cuda_array_interface__ = {"shape": (count,), "typestr": "<f4" if dtype == 0 else "<f8",
                                                 "data": (ptr, False), "version": 2}

        streams = {}

        def allreduce(ptr, count, dtype, stream):
            # the stream the library hands over: its main stream (= backend.torch_stream), or the second stream of the pipelined
            # Y exchange (LCX_Y_PIPELINE=chunks) - the collective must be ordered with THAT one
            sid = int(stream or 0)
            if sid == backend.torch_stream.cuda_stream or sid == 0:
                ctx = backend.stream_context()
            else:
                if sid not in streams:
                    streams[sid] = torch.cuda.ExternalStream(sid, device=torch.device("cuda", backend.device))
                ctx = torch.cuda.stream(streams[sid])
            with ctx:
                t = torch.as_tensor(_View(ptr, count, dtype), device=torch.device("cuda", backend.device))
                self._dist.all_reduce(t, op=self._dist.ReduceOp.SUM, group=self.group)
        backend.set_exchange_hook(allreduce)
        # the hook transport gets the same first-contact test; here a failure has no fall-back left: raise on every rank
        dev = torch.device("cuda", backend.device)
        dog.step("lcx_comm_selftest through the hook (this process group's all_reduce)")
        err = selftest(dev, "hook")
        if agreed(err is not None, dev):
            raise RuntimeError("linearcorex_amd: rank %d: the exchange transport failed its self-test (%s)"
                               % (self.rank, err or "on another rank"))
        return "hook"

    def gather_columns(self, local, nv, like, unit=1):
        """All-gather per-rank column blocks (last axis, cut by `shard` with this unit) into the full array on every rank.
        `like` is a tensor on the device the group communicates on."""
        import torch
        if self.world == 1:
            return local
        widths = [b - a for a, b in (self.shard(nv, r, unit) for r in range(self.world))]
        wmax = max(widths)
        lead = local.shape[:-1]
        pad = np.zeros(lead + (wmax,), dtype=local.dtype)
        pad[..., :local.shape[-1]] = local
        # RCCL gathers device tensors; gloo (CPU tests, and two ranks sharing one GPU) gathers on the host
        dev = like.device if self._dist.get_backend(self.group) == "nccl" else "cpu"
        mine = torch.from_numpy(pad).to(dev)
        parts = [torch.empty_like(mine) for _ in range(self.world)]
        self._dist.all_gather(parts, mine, group=self.group)
        return np.concatenate([p.cpu().numpy()[..., :w] for p, w in zip(parts, widths)], axis=-1)


class SingleComm:
    """world size 1: no torch import, no collectives."""
    rank, world, exchange = 0, 1, False

    def shard(self, nv, rank=None, unit=1):
        return 0, nv

    def allreduce(self, tensor):
        pass

    def allreduce_max(self, tensor):
        pass

    def barrier(self):
        pass

    def bind_engine(self, backend, first_contact=True):
        return None

    def gather_columns(self, local, nv, like=None, unit=1):
        return local
