"""The preflight's agreement (mxtrain/parallel/preflight.py) with gloo stand-in children: every rank reads
the same verdict, also one that comes to it late -- rank 0, which hosts the store, waits for it."""
import os
import socket
import time

import pytest
import torch.multiprocessing as mp


def _port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


class _Late:
    """A store whose reader of the verdict is held up until it has long been there."""

    def __init__(self, store):
        self.store = store

    def __getattr__(self, name):
        return getattr(self.store, name)

    def get(self, key):
        if key == "verdict":
            while not self.store.check(["verdict"]):
                time.sleep(0.01)
            time.sleep(4.0)
        return self.store.get(key)


def _rank(rank, world, port, fail, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world),
                      LOCAL_RANK=str(rank), MXTRAIN_XGMI="auto", MXTRAIN_PREFLIGHT_CPU="1")
    if fail is not None:
        os.environ["MXTRAIN_PREFLIGHT_FAIL_RANK"] = str(fail)
    for k in ("MXTRAIN_XGMI_PREFLIGHT_DONE", "TORCHELASTIC_USE_AGENT_STORE"):
        os.environ.pop(k, None)
    from mxtrain.parallel import preflight
    if rank == world - 1:
        store = preflight._store
        preflight._store = lambda *a: (lambda s, base: (_Late(s), base))(*store(*a))
    v = preflight.run_preflight(world, rank, timeout_s=60)
    q.put((rank, v, os.environ["MXTRAIN_XGMI"]))


@pytest.mark.parametrize("fail", [None, 0])
def test_a_late_rank_reads_the_verdict(fail):
    ctx, world, port = mp.get_context("spawn"), 3, _port()
    q = ctx.Queue()
    ps = [ctx.Process(target=_rank, args=(r, world, port, fail, q)) for r in range(world)]
    for p in ps:
        p.start()
    out = {r: (v, m) for r, v, m in (q.get(timeout=150) for _ in ps)}
    for p in ps:
        p.join(30)
    for r in range(world):
        v, mode = out[r]
        assert (v["ok"], mode) == ((True, "auto") if fail is None else (False, "0")), out
        assert v["reason"] == out[0][0]["reason"], out
