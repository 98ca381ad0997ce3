"""The adapter operators where calls meet one another or the edges of their
types: captures on one batch replayed on another, calls from several threads,
infinities, the bits of rows without an adapter."""
import threading

import numpy as np
import pytest

from test_adapters import DT, LowRankCase, _batch, path  # noqa: F401 (a fixture)


def _threads(*work):
    """Runs the functions at once; the first exception of any of them is raised here."""
    errors = []

    def guard(f):
        try:
            f()
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    ts = [threading.Thread(target=guard, args=(f,)) for f in work]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    if errors:
        raise errors[0]


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [True, False])
@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_one_cluster_takes_many_units_with_and_without_rank(ctx, captured, x):
    # Tiles whose adapters have a rank, none, a rank in turn, with a base of their own, so that a cluster of the
    # CUDA-core kernel copies a unit between two that it sums: a call captured on an empty batch has one cluster for
    # all of them, more than 4096 tiles give a cluster three.
    import _lib
    import torch
    lib = _lib.load()
    prev = lib.sem_lowrank_path(1)
    count = 120 if captured else 5000
    lengths = [16 - i % 3 for i in range(count)] if captured else [1] * count
    ranks = [0 if i % 2 else 2 + 5 * (i % 4) for i in range(count)] if captured else [0 if i // 2048 == 1 else 1 + i % 3 for i in range(count)]
    c = LowRankCase(ctx, lengths, list(range(count)), ranks, 72, 40, x=x, seed=count)
    try:
        if captured:
            c.plan.set(np.zeros(1, np.int32), np.zeros(0, np.int32))
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                c.call(torch.cuda.current_stream().cuda_stream)
            c.plan.set(c.offs, c.use)
            torch.cuda.synchronize()
        first = None
        for _ in range(40):
            c.dy.fill_(77)
            torch.cuda.synchronize()
            if captured:
                graph.replay()
            else:
                c.call(ctx.stream)
            c.bank.check()
            if first is None:
                c.verify(c.dy)
                first = c.dy.clone()
            assert torch.equal(c.dy, first)
    finally:
        lib.sem_lowrank_path(prev)
    c.close()
