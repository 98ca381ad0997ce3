"""The adapter operators where calls meet one another or the edges of their
types: captures on one batch replayed on another, calls from several threads,
infinities, the bits of rows without an adapter."""
import ctypes as C
import os
import subprocess
import threading

import numpy as np
import pytest

from conftest import ROOT
from test_adapters import BUILD, DT, LowRankCase, _batch, path  # noqa: F401 (a fixture)
from test_model_adapters import model, tensors  # noqa: F401 (fixtures)


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


@pytest.fixture(scope="module")
def scales_host():
    os.makedirs(BUILD, exist_ok=True)
    so = os.path.join(BUILD, "libscales_host.so")
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror",
                        os.path.join(ROOT, "tests", "adapters", "scales_host.cpp"), "-o", so],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lib = C.CDLL(so)
    lib.sh_scales.restype = C.c_char_p
    return lib


@pytest.mark.parametrize("n_absmax,n_seqs,captured,want", [
    (1, 1, False, 0), (1, 3, False, 0), (1, 0, False, 0), (3, 3, False, 1), (0, 0, False, 1),
    (1, 1, True, None), (1, 3, True, 0), (1, 0, True, 0), (3, 3, True, 1), (0, 0, True, 1),
    (-2, 1, True, 0), (-3, 1, True, 1), (-2, 5, False, 0), (-3, 5, True, 1), (-3, 0, True, 1),
    (0, 2, False, None), (3, 2, True, None), (2, 1, False, None), (-1, 2, False, None), (-1, 0, False, None),
])
def test_what_the_scales_belong_to(scales_host, n_absmax, n_seqs, captured, want):
    per_seq = C.c_int32(-7)
    why = scales_host.sh_scales(n_absmax, n_seqs, int(captured), C.byref(per_seq))
    assert (why == b"") == (want is not None)
    if want is not None:
        assert per_seq.value == want


def _captured(torch, c, call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(torch.cuda.current_stream().cuda_stream)
    return graph


@pytest.mark.gpu
@pytest.mark.parametrize("start", [0, 1, 3])
def test_captured_int8_call_keeps_its_scales_meaning(ctx, path, start):
    # captured on an empty batch, on one sequence or on three, replayed on batches of one, three and five
    import torch
    c = LowRankCase(ctx, [40, 3, 60, 20, 77], [0, 1, 0, -1, 1], [16, 8], 96, 160, x="f16", y="f32", codes=2)
    every = c.absmax.clone()
    batches = {0: ([], []), 1: ([90], [1]), 3: ([40, 3, 60], [0, 1, 0]), 5: ([40, 3, 60, 20, 77], [0, 1, 0, -1, 1])}

    def put(count):
        lengths, use = batches[count]
        c.offs, c.use = _batch(lengths, use)
        c.plan.set(c.offs, c.use)
        torch.cuda.synchronize()

    put(start)
    import adapters as ad
    for mode in (ad.ABSMAX_PER_SEQUENCE, ad.ABSMAX_ALL_ROWS):
        put(start)
        graph = _captured(torch, c, lambda st: c.bank.apply_int8(  # noqa: B023
            c.plan, c.dx.data_ptr(), c.dabs.data_ptr(), mode, c.dy.data_ptr(), c.dbase.data_ptr(), stream=st))  # noqa: B023
        for count in (1, 3, 5, 3):
            put(count)
            c.dy.fill_(77)
            graph.replay()
            c.bank.check()
            lengths, use = batches[count]
            rows = sum(lengths)
            c.seq = np.concatenate([np.repeat(np.arange(count), lengths), np.zeros(c.rows - rows, int)])
            c.adapter = np.concatenate([np.repeat(use, lengths), np.full(c.rows - rows, -1)])
            c.absmax = every if mode == ad.ABSMAX_PER_SEQUENCE else every[:1]
            c.codes = 2 if mode == ad.ABSMAX_PER_SEQUENCE else 1
            want, bound = c.oracle()
            assert ((c.dy[:rows].cpu().double() - want[:rows]).abs() <= bound[:rows]).all()
            assert (c.dy[rows:] == 77).all()
    c.close()


@pytest.mark.gpu
def test_one_scale_for_one_sequence_is_not_captured(ctx):
    # one number that says both "one for all rows" and "one per sequence": fine for a call, refused in a capture
    import _lib
    import torch
    c = LowRankCase(ctx, [40], [0], [16], 96, 160, x="f16", y="f32", codes=2)
    c.run(ctx)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        c.dy.fill_(77)
        with pytest.raises(_lib.SemError, match="captured with 1 activation scale for a plan of 1 sequence"):
            c.call(torch.cuda.current_stream().cuda_stream)
    c.run(ctx)
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("ranks", [(128, 40), (32, 27)])
def test_banks_of_other_ranks_at_the_same_time(ctx, ranks):
    # two threads, each with a bank, a plan and a stream of its own, on the CUDA cores: their kernels are one function
    # with different needs of shared memory
    import _lib
    import torch
    so = os.path.join(BUILD, "libcalls.so")
    os.makedirs(BUILD, exist_ok=True)
    r = subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-Wall", "-Werror",
                        os.path.join(ROOT, "tests", "adapters", "calls.cpp"), "-o", so], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    repeat = C.CDLL(so).repeat_apply
    repeat.argtypes = [C.c_void_p] * 7 + [C.c_int32]
    lib = _lib.load()
    prev = lib.sem_lowrank_path(1)
    cases = [LowRankCase(ctx, [3, 9], [0, -1], [r], 64, 64, seed=r) for r in ranks]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    failed = [None, None]

    def caller(i):
        c = cases[i]
        failed[i] = repeat(C.cast(lib.sem_lowrank_apply, C.c_void_p), c.bank.handle, c.plan.handle, c.dx.data_ptr(),
                           c.dbase.data_ptr(), c.dy.data_ptr(), streams[i].cuda_stream, 50000)

    try:
        _threads(lambda: caller(0), lambda: caller(1))
        assert failed == [0, 0]
        for c in cases:
            c.bank.check()
            c.verify(c.dy)
    finally:
        lib.sem_lowrank_path(prev)
    for c in cases:
        c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("x,y", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
def test_rows_without_an_adapter_keep_their_bits(ctx, path, x, y):
    # y = base for them: the sign of a zero and the bits of a NaN too
    import torch
    c = LowRankCase(ctx, [5, 20, 70, 3], [-1, 1, 0, 2], [0, 16, 4], 64, 96, x=x, y=y)
    word = torch.int32 if y == "f32" else torch.int16
    nan = torch.tensor([{"f32": 0x7fc12345, "f16": 0x7e45, "bf16": 0x7fc5}[y]], dtype=word).view(c.base.dtype)
    plain = torch.from_numpy(~np.isin(c.adapter, [1, 2]))
    assert plain.any() and not plain.all()
    c.base[plain, 1::3] = -0.0
    c.base[plain, 2::3] = nan
    c.dbase.copy_(c.base)
    torch.cuda.synchronize()
    c.call(ctx.stream)
    c.bank.check()
    got = c.dy.cpu()
    assert torch.equal(got[plain].view(word), c.base[plain].view(word))
    want, bound = c.oracle()
    assert ((got[~plain].double() - want[~plain]).abs() <= bound[~plain]).all()
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("x,y", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("w", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("short", [False, True])
def test_infinite_rows_give_the_formulas_infinities(ctx, path, x, y, w, short):
    # Rank 1 and one infinity in a row of x: every result of the row is infinite, with the formula's sign (no weight is
    # zero). Rank 3 with weights whose terms agree in sign the same; one infinity of each sign: NaN. `short`: float32
    # weights whose low parts are all zero.
    import torch
    import adapters as ad
    k, n = 70, 90
    c = LowRankCase(ctx, [40, 30], [0, 1], [1, 3], k, n, x=x, y=y, w=w, seed=5, scales=[-1.5, 2.0])
    inf = float("inf")

    def away(t):  # away from zero; of few bits with `short`
        t = t.float().sign() * (t.float().abs() + 0.01)
        return (t.to(torch.bfloat16) if short else t).to(t.dtype)

    c.a = [away(t).to(t.dtype) for t in c.a]
    c.b = [away(t).to(t.dtype) for t in c.b]
    c.a[1], c.b[1] = c.a[1].abs(), c.b[1].abs()
    host = lambda t: (t.view(torch.int16) if t.dtype == torch.bfloat16 else t).numpy()  # noqa: E731
    c.bank.close()
    c.bank = ad.LowRank(ctx, k, n, [host(t) for t in c.a], [host(t) for t in c.b], c.scales, DT[w])
    rows = {0: (3, inf), 7: (69, -inf), 20: (0, inf), 39: (64, -inf), 41: (5, inf), 50: (69, -inf), 69: (33, inf)}
    for r, (col, v) in rows.items():
        c.x[r, col] = v
    c.x[60, 2], c.x[60, 8] = inf, -inf
    c.dx.copy_(c.x)
    torch.cuda.synchronize()
    c.call(ctx.stream)
    c.bank.check()
    got = c.dy.cpu().double()
    for r, (col, v) in rows.items():
        i = int(c.adapter[r])
        t = torch.sign(c.a[i][:, col].double()) * v
        want = c.scales[i] * c.b[i].double() @ t
        assert torch.isinf(want).all()
        assert torch.equal(got[r], want), (r, got[r][:8], want[:8])
    assert torch.isnan(got[60]).all()
    finite = [r for r in range(c.rows) if r not in rows and r != 60]
    c.x[list(rows) + [60]] = 0
    want, bound = c.oracle()
    assert ((got[finite] - want[finite]).abs() <= bound[finite]).all()
    c.close()


@pytest.mark.gpu
def test_a_nan_of_any_payload_stays_one(ctx, path):
    # float32 rows are cut to 11 bits for the tensor cores: a NaN whose payload lies behind them is no infinity
    import torch
    c = LowRankCase(ctx, [64, 9], [0, 1], [1, 5], 64, 40, w="f32")
    bits = c.dx.view(torch.int32)
    bits[3, 7], bits[60, 63], bits[70, 0] = 0x7f800001, -0x7fffff, 0x7fc00000  # the second: a negative one
    assert torch.isnan(c.dx).sum() == 3
    torch.cuda.synchronize()
    c.call(ctx.stream)
    c.bank.check()
    got, bad = c.dy.cpu(), [3, 60, 70]
    assert torch.isnan(got[bad]).all()
    want, bound = c.oracle()
    rest = [i for i in range(73) if i not in bad]
    assert ((got[rest].double() - want[rest]).abs() <= bound[rest]).all()
    c.close()


@pytest.mark.gpu
def test_calls_on_the_contexts_stream_beside_captured_forwards(ctx, model, tensors):
    # One thread embeds batches of new shapes, whose forwards are captured on the context's stream; another makes
    # plans and calls operators there. Neither may end in the other's capture.
    import torch
    import adapters as ad
    import synth
    shapes = [[5 + i, 9, 30 + 2 * i] for i in range(60)]
    batches = [synth.token_batch(i, s, 64) for i, s in enumerate(shapes)]
    want = [model.forward_batch(*b) for b in batches[:4]]
    c = LowRankCase(ctx, [40, 3], [0, -1], [16], 96, 160)
    bn = ad.BlockNorm(ctx, 96, 1e-6, np.ones(96, np.float32), np.ones(96, np.float32))
    o, h = torch.randn(43, 96, device="cuda"), torch.randn(43, 96, device="cuda")
    ho, y = torch.empty_like(h), torch.empty_like(o)
    torch.cuda.synchronize()
    bn.run(43, o.data_ptr(), 0, h.data_ptr(), 0, ho.data_ptr(), y.data_ptr(), c.plan)
    c.bank.check()
    ho1, y1 = ho.clone(), y.clone()
    torch.cuda.synchronize()
    done, rounds, got = threading.Event(), [0], [None] * len(batches)

    def embed():
        try:
            for i, b in enumerate(batches):
                got[i] = model.forward_batch(*b)
        finally:
            done.set()

    def operators():
        while not done.is_set() or rounds[0] < 5:
            plan = ad.AdapterPlan(ctx, c.rows, 2)
            plan.set(c.offs, c.use)
            c.bank.apply(plan, c.dx.data_ptr(), 0, c.dy.data_ptr(), 0, c.dbase.data_ptr())
            bn.run(43, o.data_ptr(), 0, h.data_ptr(), 0, ho.data_ptr(), y.data_ptr(), plan)
            c.bank.check()
            c.verify(c.dy)
            assert torch.equal(ho, ho1) and torch.equal(y, y1)
            for t in (c.dy, ho, y):
                t.fill_(77)
            torch.cuda.current_stream().synchronize()
            plan.close()
            model.load_adapters([]).close()
            rounds[0] += 1

    _threads(embed, operators)
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            np.testing.assert_array_equal(a, b)
    c.dy.fill_(77)
    torch.cuda.synchronize()
    # the captured forwards hold nothing of the other thread's: replayed, they leave y alone
    for i, b in enumerate(batches[-8:]):
        for a, w in zip(model.forward_batch(*b), got[len(batches) - 8 + i]):
            np.testing.assert_array_equal(a, w)
    torch.cuda.synchronize()
    assert (c.dy == 77).all()
    bn.close()
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("x,w,k", [("f32", "f32", 768), ("f16", "bf16", 768), ("bf16", "bf16", 517)])
def test_a_sequence_alone_and_in_other_batches(ctx, path, x, w, k):
    # With one kernel for both, a sequence's rows have the same bits alone, in a small batch and in a large one. AUTO
    # takes the kernel that suits the whole batch: there the two are each within the bound of the operator.
    import torch
    lengths, use, ranks = [300, 20, 7, 150], [0, 1, 2, 1], [16, 24, 100]
    c = LowRankCase(ctx, lengths, use, ranks, k, 256, x=x, w=w)
    c.run(ctx)
    together, offs = c.dy.clone(), c.offs
    want, bound = c.oracle()

    def check(got, at):
        if path == "auto":
            assert ((got.cpu().double() - want[at]).abs() <= bound[at]).all()
        else:
            assert torch.equal(got, together[at])

    dx, dbase = c.dx, c.dbase
    for s, a in enumerate(use):
        at = slice(int(offs[s]), int(offs[s + 1]))
        c.plan.set([0, lengths[s]], [a])
        c.dx, c.dbase, c.dy = dx[at].clone(), dbase[at].clone(), torch.full_like(together[at], 77)
        torch.cuda.synchronize()
        c.call(ctx.stream)
        c.bank.check()
        check(c.dy, at)
    # behind 6000 other rows, in a plan with room for them
    import adapters as ad
    big = ad.AdapterPlan(ctx, 6000 + c.rows, 8)
    big.set(np.concatenate([[0], 6000 + offs]), [2] + use)
    c.plan.close()
    c.plan = big
    c.dx, c.dbase = torch.cat([dx[:1].expand(6000, -1), dx]), torch.cat([dbase[:1].expand(6000, -1), dbase])
    c.dy = torch.full_like(c.dbase, 77)
    torch.cuda.synchronize()
    c.call(ctx.stream)
    c.bank.check()
    check(c.dy[6000:], slice(None))
    c.close()
