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


@pytest.mark.gpu
def test_int8_scales_are_checked_against_the_batch_they_meet(ctx):
    # One thread sets the plan to a batch of two sequences and to one of sixteen in turn, another calls with two
    # scales: a call is refused, or it runs on the batch of two. The scales behind the second one are NaN, which
    # would stay in y (a sum in place) for good.
    import _lib
    import torch
    import adapters as ad
    k, n, rows = 32, 32, 32
    rng = np.random.default_rng(0)
    bank = ad.LowRank(ctx, k, n, [rng.standard_normal((2, k)).astype(np.float32)],
                      [rng.standard_normal((n, 2)).astype(np.float32)], [1e-6], ad.F32)
    plan = ad.AdapterPlan(ctx, rows, 16)
    two, sixteen = ([0, 16, 32], [0, 0]), (list(range(0, 33, 2)), [0] * 16)
    codes = torch.randint(-127, 128, (rows, k), device="cuda").half()
    absmax = torch.full((16,), float("nan"), device="cuda")
    absmax[:2] = 1.0
    y = torch.zeros(rows, n, device="cuda")
    torch.cuda.synchronize()
    plan.set(*sixteen)
    done, took = threading.Event(), [0, 0]

    def setter():
        while not done.is_set():
            plan.set(*two)
            plan.set(*sixteen)

    def caller():
        try:
            for _ in range(20000):
                try:
                    bank.apply_int8(plan, codes.data_ptr(), absmax.data_ptr(), 2, y.data_ptr(), y.data_ptr())
                    took[0] += 1
                except _lib.SemError as e:
                    assert "2 activation scales for a plan of 16 sequences" in str(e)
                    took[1] += 1
        finally:
            done.set()

    _threads(setter, caller)
    bank.check()
    assert took[0] and took[1], took  # both batches were met
    assert torch.isfinite(y).all(), torch.isfinite(y).all(1)
    bank.close()
    plan.close()


@pytest.mark.gpu
def test_block_norm_runs_on_the_batch_it_was_checked_against(ctx):
    # The plan is set to 40 rows without an adapter and to 20 of adapter 0 in turn: a call over 40 rows is refused or
    # runs on the first. Adapter 0's gate is NaN, which would stay in the residual stream (in place) for good.
    import _lib
    import torch
    import adapters as ad
    dim, rows = 64, 40
    bn = ad.BlockNorm(ctx, dim, 1e-6, gates=np.full((1, dim), np.nan, np.float32))
    plan = ad.AdapterPlan(ctx, rows, 1)
    o, h = torch.zeros(rows, dim, device="cuda"), torch.ones(rows, dim, device="cuda")
    torch.cuda.synchronize()
    plan.set([0, 20], [0])
    done, took = threading.Event(), [0, 0]

    def setter():
        while not done.is_set():
            plan.set([0, 40], [-1])
            plan.set([0, 20], [0])

    def caller():
        try:
            for _ in range(20000):
                try:
                    bn.run(rows, o.data_ptr(), 0, h.data_ptr(), 0, h.data_ptr(), plan=plan)
                    took[0] += 1
                except _lib.SemError as e:
                    assert "40 rows, the plan has 20" in str(e)
                    took[1] += 1
        finally:
            done.set()

    _threads(setter, caller)
    torch.cuda.synchronize()
    assert took[0] and took[1], took
    assert (h == 1).all()
    bn.close()
    plan.close()
