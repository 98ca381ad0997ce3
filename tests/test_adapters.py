"""The adapter operators (sem_adapter_plan, sem_lowrank, sem_block_norm)
against their formulas in float64.

Bounds. A result is base + scale * sum_r (sum_k x a) b, computed with float32
products and sums. Every product's factors carry at least 21 bits (a factor of
more than 11 bits is split in two parts of at least 11 and 10; the product of
the two low parts, below 2^-22 of the whole, may be left out), so a product is
off by at most 2^-20 relative to its magnitude, twice over for the two products
in a term; each of the at most k + r additions is off by at most one step of
float32 of the running sum (2^-23, which covers sums that cut instead of
round). So |error| <= (2^-19 + (k + r + 8) 2^-23) * sum_r (sum_k |x||a|) |b| * |scale|
before the rounding of the result, half a step of its type.
"""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from conftest import ROOT

DT = {"f32": 0, "f16": 1, "bf16": 2}
BUILD = os.path.join(ROOT, "tests", "_build")


# ---------------------------------------------------------------------------
# Without a device: the plan's tiles, refusals
# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def plan_host():
    os.makedirs(BUILD, exist_ok=True)
    so = os.path.join(BUILD, "libplan_host.so")
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", "-fsanitize=undefined",
                        "-fno-sanitize-recover", "-static-libubsan",
                        os.path.join(ROOT, "tests", "adapters", "plan_host.cpp"), "-o", so],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lib = C.CDLL(so)
    lib.ph_check.restype = C.c_char_p
    lib.ph_check.argtypes = [C.c_void_p, C.c_void_p, C.c_int32, C.c_int64, C.c_int32, C.c_void_p]
    lib.ph_build.argtypes = [C.c_void_p, C.c_void_p, C.c_int32] + [C.c_void_p] * 5
    lib.ph_max_large.argtypes, lib.ph_max_large.restype = [C.c_int64, C.c_int32], C.c_int64
    return lib


def _batch(lengths, adapters):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32), np.asarray(adapters, dtype=np.int32)


BATCHES = [
    ([], []), ([0], [3]), ([1], [0]), ([0, 0, 5, 0], [1, -1, 1, 0]), ([16], [0]), ([17], [0]), ([128], [2]),
    ([129, 143, 144, 145], [0, 1, 2, 3]), ([64] * 8, [0, 1, 0, 1, -1, 2, 0, 1]), ([1] * 300, [i % 7 - 1 for i in range(300)]),
]


def _check_plan(lib, lengths, adapters):
    offs, ad = _batch(lengths, adapters)
    n, rows = len(lengths), int(offs[-1])
    cap = lib.ph_max_large(rows, n)
    order, pos = np.full(n, -9, np.int32), np.full(n + 1, -9, np.int32)
    large, small = np.zeros((cap + 1, 4), np.int32), np.zeros((n + 1, 4), np.int32)
    counts = np.zeros(4, np.int32)
    lib.ph_build(offs.ctypes.data, ad.ctypes.data, n, order.ctypes.data, pos.ctypes.data, large.ctypes.data,
                 small.ctypes.data, counts.ctypes.data)
    # the tile lists fit the room a plan of this size allocates
    assert counts[0] <= cap and counts[1] <= n and counts[2] == rows
    used = {int(a) for a, k in zip(adapters, lengths) if k}
    assert counts[3] == max(used, default=-1)
    assert sorted(order.tolist()) == list(range(n))
    row_at = np.concatenate([np.arange(offs[s], offs[s + 1]) for s in order] or [np.zeros(0)]).astype(int)
    adapter_of = np.repeat(ad, lengths) if n else np.zeros(0, int)
    seen = np.zeros(rows, int)
    for tiles, most in ((large[:counts[0]], lib.ph_tile_rows()), (small[:counts[1]], lib.ph_small_rows())):
        for a, p0, r, first in tiles:
            assert 0 < r <= most and 0 <= p0 and p0 + r <= rows
            at = row_at[p0:p0 + r]
            assert (adapter_of[at] == a).all()
            assert first == (at[0] if (np.diff(at) == 1).all() else -1)
            seen[at] += 1
    assert (seen == 1).all()
    for i, s in enumerate(order):
        assert pos[i + 1] - pos[i] == lengths[s]


def test_plan_tiles(plan_host):
    for lengths, adapters in BATCHES:
        _check_plan(plan_host, lengths, adapters)
    rng = np.random.default_rng(3)
    for _ in range(200):
        n = int(rng.integers(1, 60))
        lengths = rng.integers(0, int(rng.choice([2, 20, 140, 700])), n).tolist()
        _check_plan(plan_host, lengths, rng.integers(-1, int(rng.integers(1, 12)), n).tolist())


@pytest.mark.parametrize("offsets,adapters,rows,seqs,want,bad", [
    ([0, 4, 3], [0, 0], 10, 10, b"offsets must not decrease", 1),
    ([1, 4], [0], 10, 10, b"offsets[0] must be 0", -1),
    ([0, 4], [-2], 10, 10, b"an adapter is -1 (none) or an index", 0),
    ([0, 11], [0], 10, 10, b"more rows than the plan was created for", -1),
    ([0, 1, 2], [0, 0], 10, 1, b"more sequences than the plan was created for", -1),
    ([0, 10], [0], 10, 1, b"", -1),
])
def test_plan_refusals(plan_host, offsets, adapters, rows, seqs, want, bad):
    o, a = np.asarray(offsets, np.int32), np.asarray(adapters, np.int32)
    at = C.c_int32(-7)
    assert plan_host.ph_check(o.ctypes.data, a.ctypes.data, a.size, rows, seqs, C.byref(at)) == want
    assert at.value == bad
    assert plan_host.ph_check(None, None, -1, 1, 1, C.byref(at)) == b"negative sequence count"
    assert plan_host.ph_check(None, None, 1, 1, 1, C.byref(at)) == b"null argument"
    assert plan_host.ph_check(None, None, 0, 0, 0, C.byref(at)) == b""


def _create_lowrank(k=8, n=8, ranks=(4,), dtype=0, scales=True, weights=True):
    import _lib
    r = np.asarray(ranks, np.int32)
    s = np.ones(max(r.size, 1), np.float32)
    w = np.zeros(8 * 1024, np.float32)
    p = (C.c_void_p * max(r.size, 1))(*[w.ctypes.data if weights else None] * max(r.size, 1))
    h = C.c_void_p()
    _lib.check(_lib.load().sem_lowrank_create(None, k, n, r.size, r.ctypes.data, s.ctypes.data if scales else None, p,
                                              p, dtype, C.byref(h)))


@pytest.mark.parametrize("kw,want", [
    (dict(k=0), "both dimensions must be in 1..65536"),
    (dict(n=65537), "both dimensions must be in 1..65536"),
    (dict(dtype=3), "unknown element type 3"),
    (dict(ranks=(4, 129)), r"low-rank adapter 1: rank 129 out of range \(0..128\)"),
    (dict(ranks=(-1,)), r"low-rank adapter 0: rank -1 out of range"),
    (dict(scales=False), "null argument"),
    (dict(weights=False), "low-rank adapter 0: null weights"),
    (dict(), "null argument"),  # no context
])
def test_lowrank_refusals(kw, want):
    import _lib
    with pytest.raises(_lib.SemError, match=want) as e:
        _create_lowrank(**kw)
    assert e.value.code == _lib.SEM_EINVAL


@pytest.mark.parametrize("dim,eps,n,want", [
    (0, 1e-6, 0, "1..16384 are supported"), (16385, 1e-6, 0, "1..16384 are supported"),
    (8, -1.0, 0, "eps must be finite and not negative"), (8, float("nan"), 0, "eps must be finite"),
    (8, float("inf"), 0, "eps must be finite"), (8, 0.0, -1, "negative adapter count"), (8, 1e-6, 0, "null argument"),
])
def test_block_norm_refusals(dim, eps, n, want):
    import _lib
    h = C.c_void_p()
    with pytest.raises(_lib.SemError, match=want):
        _lib.check(_lib.load().sem_block_norm_create(None, dim, eps, None, None, n, None, None, C.byref(h)))


def test_lowrank_path_switch():
    import _lib
    lib = _lib.load()
    assert lib.sem_lowrank_path(2) == 0
    assert lib.sem_lowrank_path(3) == -1 and lib.sem_lowrank_path(-1) == -1
    assert lib.sem_lowrank_path(0) == 2


def test_calls_without_handles():
    import _lib
    lib = _lib.load()
    h = C.c_void_p()
    assert lib.sem_adapter_plan_create(None, 1, 1, C.byref(h)) == _lib.SEM_EINVAL
    assert lib.sem_adapter_plan_create(None, 1 << 31, 1, C.byref(h)) == _lib.SEM_EINVAL
    assert lib.sem_adapter_plan_create(None, -1, 1, C.byref(h)) == _lib.SEM_EINVAL
    assert lib.sem_adapter_plan_set(None, None, None, 0, None) == _lib.SEM_EINVAL
    assert lib.sem_lowrank_apply(None, None, None, 0, 0, None, 0, None, 0, 0, None) == _lib.SEM_EINVAL
    assert lib.sem_lowrank_apply_int8(None, None, None, None, 1, None, 0, None, 0, None) == _lib.SEM_EINVAL
    assert lib.sem_lowrank_check(None) == _lib.SEM_EINVAL
    assert lib.sem_block_norm_run(None, None, 1, None, 0, 0, None, 0, 0, None, 0, None, 0, None) == _lib.SEM_EINVAL
    # type pairs are refused before anything else is looked at
    for x, y in ((0, 1), (1, 2), (2, 1), (3, 3), (-1, 0)):
        assert lib.sem_lowrank_apply(None, None, None, x, 0, None, 0, None, y, 0, None) == _lib.SEM_EINVAL
        assert b"no form for inputs" in lib.sem_last_error()
        assert lib.sem_block_norm_run(None, None, 1, None, 0, x, None, 0, y, None, 0, None, 0, None) == _lib.SEM_EINVAL
        assert b"no form for block outputs" in lib.sem_last_error()
    for free in (lib.sem_adapter_plan_free, lib.sem_lowrank_free, lib.sem_block_norm_free):
        assert free(None) == _lib.SEM_OK


def test_python_weight_checks():
    import adapters as ad
    ctx = None
    a, b = np.zeros((4, 8), np.float32), np.zeros((6, 4), np.float32)
    with pytest.raises(ValueError, match="float32 weights for a bank of type 1"):
        ad.LowRank(ctx, 8, 6, [a], [b], [1.0], ad.F16)
    with pytest.raises(ValueError, match=r"shape \(4, 8\), want \(4, 9\)"):
        ad.LowRank(ctx, 9, 6, [a], [b], [1.0], ad.F32)
    with pytest.raises(ValueError, match="one of its two weights is missing"):
        ad.LowRank(ctx, 8, 6, [a], [None], [1.0], ad.F32)
    with pytest.raises(ValueError, match="1 a, 1 b and 2 scales"):
        ad.LowRank(ctx, 8, 6, [a], [b], [1.0, 2.0], ad.F32)
    with pytest.raises(ValueError, match="unknown element type 9"):
        ad.LowRank(ctx, 8, 6, [a], [b], [1.0], 9)
    with pytest.raises(ValueError, match="gates of shape"):
        ad.BlockNorm(ctx, 8, 1e-6, gates=np.zeros((2, 9)))
    with pytest.raises(ValueError, match="3 offsets for 1 sequences"):
        ad.AdapterPlan.set(None, [0, 1, 2], [0])


# ---------------------------------------------------------------------------
# On a device
# ---------------------------------------------------------------------------
def _torch(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _host(w):
    import torch
    return (w.view(torch.int16) if w.dtype == torch.bfloat16 else w).cpu().numpy()


@pytest.fixture(params=["auto", "cuda_cores", "tensor"])
def path(request):
    """Each kernel for the larger tiles (sem_lowrank_path): small test batches would all take the CUDA cores."""
    import _lib
    lib = _lib.load()
    prev = lib.sem_lowrank_path(["auto", "cuda_cores", "tensor"].index(request.param))
    yield request.param
    lib.sem_lowrank_path(prev)


class LowRankCase:
    """Inputs of one call on the device, its oracle in float64 and its bound."""

    def __init__(self, ctx, lengths, use, ranks, k, n, x="f32", y=None, w="f16", pads=(0, 0, 0), codes=0, seed=0,
                 scales=None):
        import torch
        import adapters as ad
        g = torch.Generator().manual_seed(seed)
        y = y or x
        self.offs, self.use = _batch(lengths, use)
        self.rows, self.k, self.n, self.xt, self.yt = int(self.offs[-1]), k, n, x, y
        rows = self.rows
        self.seq = np.repeat(np.arange(len(lengths)), lengths)
        self.adapter = self.use[self.seq] if rows else np.zeros(0, int)
        self.codes = codes
        if codes:
            xs = torch.randint(-127, 128, (rows, k), generator=g).to(torch.float32)
            self.absmax = torch.rand(len(lengths) if codes == 2 else 1, generator=g) * 5 + 0.5
        else:
            xs = torch.randn(rows, k, generator=g)
        self.x = torch.full((rows, k + pads[0]), float("nan")).to(_torch(x))
        self.x[:, :k] = xs.to(_torch(x))
        self.base = torch.full((rows, n + pads[1]), float("nan")).to(_torch(y))
        self.base[:, :n] = torch.randn(rows, n, generator=g).to(_torch(y))
        self.y = torch.full((rows, n + pads[2]), 77.0).to(_torch(y))
        self.a = [torch.randn(r, k, generator=g).mul(k ** -0.5).to(_torch(w)) if r else None for r in ranks]
        self.b = [torch.randn(n, r, generator=g).mul(r ** -0.5).to(_torch(w)) if r else None for r in ranks]
        self.scales = scales or [0.5 + 0.25 * i for i in range(len(ranks))]
        self.ranks = ranks
        self.dx, self.dbase, self.dy = self.x.cuda(), self.base.cuda(), self.y.cuda()
        self.bank = ad.LowRank(ctx, k, n, [None if t is None else _host(t) for t in self.a],
                               [None if t is None else _host(t) for t in self.b], self.scales, DT[w])
        self.plan = ad.AdapterPlan(ctx, max(rows, 1), max(len(lengths), 1))
        self.plan.set(self.offs, self.use)
        if codes:
            self.dabs = self.absmax.cuda()
        torch.cuda.synchronize()

    def oracle(self, with_base=True):
        import torch
        n, k = self.n, self.k
        out = self.base[:, :n].double() if with_base else torch.zeros(self.rows, n, dtype=torch.float64)
        size = torch.zeros(self.rows, n, dtype=torch.float64)
        x = self.x[:, :k].double()
        if self.codes:
            x = x * (self.absmax.double()[torch.from_numpy(self.seq)] if self.codes == 2 else self.absmax.double())[:, None] / 127
        for i, r in enumerate(self.ranks):
            at = torch.from_numpy(np.nonzero(self.adapter == i)[0])
            if r and len(at):
                a, b = self.a[i].double(), self.b[i].double()
                out[at] += self.scales[i] * (x[at] @ a.T) @ b.T
                size[at] += abs(self.scales[i]) * (x[at].abs() @ a.abs().T) @ b.abs().T
        c = 2.0 ** -19 + (k + max(self.ranks, default=0) + 8) * 2.0 ** -23
        half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[self.yt]
        # the last sum's own float32 rounding, and below the smallest normal the type's absolute step
        bound = c * size + (half + 2.0 ** -24) * (out.abs() + c * size) + (2.0 ** -25 if self.yt == "f16" else 0.0)
        return out, bound

    def call(self, stream, base="own", y=None):
        dy = self.dy if y is None else y
        d_base = {"own": self.dbase.data_ptr(), "none": 0, "y": dy.data_ptr()}[base]
        ld_base = dy.stride(0) if base == "y" else self.dbase.stride(0)
        if self.codes:
            self.bank.apply_int8(self.plan, self.dx.data_ptr(), self.dabs.data_ptr(), self.dabs.numel(), dy.data_ptr(),
                                 d_base, ld_base, dy.stride(0), stream)
        else:
            self.bank.apply(self.plan, self.dx.data_ptr(), DT[self.xt], dy.data_ptr(), DT[self.yt], d_base,
                            self.dx.stride(0), ld_base, dy.stride(0), stream)

    def verify(self, y, with_base=True):
        import torch
        want, bound = self.oracle(with_base)
        got = y.cpu()
        assert torch.isfinite(got[:, :self.n].float()).all()
        off = (got[:, :self.n].double() - want).abs() - bound
        assert (off <= 0).all(), (float(off.max()), float(bound.min()), np.argwhere(off.numpy() > 0)[:4])
        assert (got[:, self.n:] == 77).all()  # behind the rows' outputs nothing is written

    def run(self, ctx, base="own"):
        import torch
        if base == "y":
            self.dy[:, :self.n] = self.dbase[:, :self.n]
            torch.cuda.synchronize()
        self.call(ctx.stream, base)
        self.bank.check()
        self.verify(self.dy, base != "none")

    def close(self):
        self.bank.close()
        self.plan.close()


SHAPES = [
    # lengths, adapters, ranks
    ([1], [0], [1]),
    ([5, 1, 0, 9], [1, 0, 1, -1], [16, 8]),
    ([16, 17, 15, 33], [0, 1, 2, 3], [3, 5, 16, 64]),
    ([128, 129, 1, 200], [0, 1, -1, 0], [16, 128]),
    ([40, 300, 3, 250, 64], [2, 0, 1, 0, 3], [0, 33, 7, 100]),
]
TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")]


@pytest.mark.gpu
@pytest.mark.parametrize("x,y", TYPES)
@pytest.mark.parametrize("w", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_lowrank_types(ctx, path, shape, x, y, w):
    c = LowRankCase(ctx, *SHAPES[shape], k=96, n=160, x=x, y=y, w=w, seed=shape)
    c.run(ctx)
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("k,n", [(1, 1), (7, 3), (31, 129), (32, 128), (33, 127), (257, 64), (517, 1001), (768, 768),
                                 (1152, 256)])
@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_lowrank_sizes(ctx, path, k, n, x):
    c = LowRankCase(ctx, [1, 40, 130, 2, 260], [0, 1, 2, -1, 1], [4, 19, 128], k, n, x=x, w="bf16", seed=k)
    c.run(ctx)
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("pads", [(0, 0, 0), (1, 3, 5), (8, 8, 8), (4, 0, 12)])
@pytest.mark.parametrize("base", ["own", "none", "y"])
@pytest.mark.parametrize("x,y", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32")])
def test_lowrank_strides_and_base(ctx, path, pads, base, x, y):
    # rank 0 and no adapter: the row is the base (or zeros) whatever the kernel
    c = LowRankCase(ctx, [3, 60, 140, 20, 7], [0, 1, 2, 3, -1], [8, 0, 24, 40], 72, 136, x=x, y=y, w="f16", pads=pads)
    c.run(ctx, base)
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("x,y", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("start", [1, 2, 4])
def test_lowrank_rows_from_any_element(ctx, path, start, x, y):
    # strides of whole 16-byte pieces, but rows that start `start` elements behind one
    import torch
    c = LowRankCase(ctx, [3, 60, 140], [0, 1, 2], [8, 24, 40], 72, 136, x=x, y=y, pads=(8, 8, 8))

    def moved(t):
        wide = torch.empty(t.numel() + start, dtype=t.dtype, device="cuda")
        wide[start:] = t.flatten()
        return wide[start:].view(t.shape)

    c.dx, c.dbase, c.dy = moved(c.dx), moved(c.dbase), moved(c.dy)
    c.run(ctx)
    c.run(ctx, "y")
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("x,y", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("ld", [2 ** 37, 2 ** 40, 2 ** 40 + 1])
def test_lowrank_single_row_of_any_stride(ctx, path, ld, x, y):
    # no second row is there to be read at the stride
    import torch
    c = LowRankCase(ctx, [1], [0], [24], 72, 136, x=x, y=y)
    c.bank.apply(c.plan, c.dx.data_ptr(), DT[x], c.dy.data_ptr(), DT[y], c.dbase.data_ptr(), ld, ld, ld, ctx.stream)
    c.bank.check()
    c.verify(c.dy)
    torch.cuda.synchronize()
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [1, 2])
@pytest.mark.parametrize("w", ["f16", "f32"])
def test_lowrank_int8_codes(ctx, path, codes, w):
    c = LowRankCase(ctx, [64, 64, 5, 300, 64], [0, 1, 0, 2, -1], [16, 4, 32], 768, 256, x="f16", y="f32", w=w,
                    codes=codes)
    c.run(ctx)
    c.run(ctx, "y")
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [17, 23, 33, 64])
@pytest.mark.parametrize("k,n,x", [(768, 256, "bf16"), (32, 40, "f32")])
def test_lowrank_many_short_tiles(ctx, path, rows, k, n, x):
    # more tiles than SMs, each its own adapter's, most of them shorter than a full one; then a few full ones
    count = 700
    c = LowRankCase(ctx, [rows] * count + [200], [i % 40 if i % 7 else -1 for i in range(count)] + [40],
                    [3 + i % 30 for i in range(40)] + [8], k, n, x=x, w="f16", seed=rows)
    c.run(ctx)
    c.close()
    c = LowRankCase(ctx, [rows] * 60, list(range(60)), [8 + i % 3 for i in range(60)], k, n, x=x, w="bf16", seed=rows)
    c.run(ctx)
    c.close()


@pytest.mark.gpu
def test_lowrank_empty_batch_writes_nothing(ctx):
    import torch
    c = LowRankCase(ctx, [0, 0], [0, -1], [4], 8, 8)
    guard = torch.full((4, 8), 5.0, device="cuda")
    torch.cuda.synchronize()
    c.bank.apply(c.plan, guard.data_ptr(), 0, guard.data_ptr() + 64, 0, stream=ctx.stream)
    c.plan.set(np.zeros(1, np.int32), np.zeros(0, np.int32))
    c.bank.apply(c.plan, guard.data_ptr(), 0, guard.data_ptr() + 64, 0, stream=ctx.stream)
    c.bank.check()
    assert (guard == 5).all()
    c.close()


@pytest.mark.gpu
def test_lowrank_non_finite_rows_stay_their_own(ctx, path):
    # infinities and NaN in some rows of x: those rows are the formula's, every other row is finite and right
    import torch
    c = LowRankCase(ctx, [200, 10], [0, 1], [16, 8], 64, 64, w="f16")
    c.dx[3, 5], c.dx[130, 0], c.dx[205, 63] = float("inf"), float("nan"), float("-inf")
    torch.cuda.synchronize()
    c.call(ctx.stream)
    c.bank.check()
    got = c.dy.cpu()
    bad = [3, 130, 205]
    want, bound = c.oracle()
    keep = [i for i in range(210) if i not in bad]
    assert ((got[keep].double() - want[keep]).abs() <= bound[keep]).all()
    assert torch.isnan(got[130]).all()
    for row, adapter, col, sign in ((3, 0, 5, 1.0), (205, 1, 63, -1.0)):
        # x a^T is +-inf in every rank (no weight is zero), so a result is +-inf or NaN: never finite
        assert (c.a[adapter][:, col] != 0).all()
        assert not torch.isfinite(got[row]).any()
    c.close()


@pytest.mark.gpu
def test_lowrank_large_values_and_wide_range(ctx, path):
    # rows of very different magnitude: float32's whole range of exponents through the split operands
    import torch
    c = LowRankCase(ctx, [150, 6], [0, 1], [16, 8], 64, 96, w="f32", pads=(0, 0, 0))
    f = torch.logspace(-25, 25, 156)[:, None]
    c.x, c.base = c.x * f, c.base * f
    c.dx.copy_(c.x)
    c.dbase.copy_(c.base)
    torch.cuda.synchronize()
    c.run(ctx)
    c.close()


@pytest.mark.gpu
def test_lowrank_repeats_bit_for_bit_and_alone(ctx, path):
    # the same rows give the same bits again, and a sequence's rows do not depend on the batch around it
    import torch
    lengths, use, ranks = [300, 20, 7, 150], [0, 1, 2, 1], [16, 24, 8]
    c = LowRankCase(ctx, lengths, use, ranks, 768, 256, w="f16")
    c.run(ctx)
    first = c.dy.clone()
    c.dy.fill_(0)
    torch.cuda.synchronize()
    c.call(ctx.stream)
    c.bank.check()
    assert torch.equal(first, c.dy)
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n,x", [(64, 32, 40, "f32"), (33, 32, 40, "f32"), (33, 32, 160, "bf16"), (64, 256, 256, "f16")])
def test_lowrank_many_units_repeat(ctx, path, rows, k, n, x):
    # several short units per SM, so that slots of every ring are used again while their last reader may be late
    import torch
    count = 700
    c = LowRankCase(ctx, [rows] * count, [i % 40 if i % 7 else -1 for i in range(count)], [3 + i % 30 for i in range(40)],
                    k, n, x=x, w="f16", seed=rows)
    c.run(ctx)
    first = c.dy.clone()
    for _ in range(150):
        c.dy.fill_(77)
        torch.cuda.synchronize()
        c.call(ctx.stream)
        c.bank.check()
        assert torch.equal(c.dy, first)
    c.close()


@pytest.mark.gpu
def test_lowrank_streams_and_graph(ctx, path):
    # two calls at once on two streams with one bank and one plan, then a captured call replayed: first as it was
    # captured, then with other inputs, then with the plan set to another batch (both tile lists change)
    import torch
    c = LowRankCase(ctx, [200, 3, 64], [0, 1, 1], [16, 8], 96, 160)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    y1, y2 = torch.full_like(c.dy, 77), torch.full_like(c.dy, 77)
    torch.cuda.synchronize()
    for _ in range(20):
        c.call(s1.cuda_stream, y=y1)
        c.call(s2.cuda_stream, y=y2)
    c.bank.check()
    c.verify(y1)
    assert torch.equal(y1, y2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s1):
        c.call(torch.cuda.current_stream().cuda_stream)
        with pytest.raises(Exception, match="outside stream capture"):
            c.plan.set(c.offs, c.use, torch.cuda.current_stream().cuda_stream)
    c.dy.fill_(77)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.dy, y1)
    c.dx.mul_(2)
    c.x.mul_(2)
    graph.replay()
    c.bank.check()
    c.verify(c.dy)
    for lengths, use in (([267], [1]), ([5, 9, 2], [0, 1, -1]), ([100, 30, 130, 7], [1, 0, 1, -1])):
        c.offs, c.use = _batch(lengths, use)
        c.seq = np.repeat(np.arange(len(lengths)), lengths)
        rows = int(c.offs[-1])
        plan_rows = c.use[c.seq]
        if len(lengths) <= 3:
            c.plan.set(c.offs, c.use)
        else:
            with pytest.raises(Exception, match="more sequences"):
                c.plan.set(c.offs, c.use)
            continue
        torch.cuda.synchronize()
        c.dy.fill_(77)
        graph.replay()
        c.bank.check()
        assert (c.dy[rows:] == 77).all()  # rows behind the last sequence stay as they were
        c.adapter = np.concatenate([plan_rows, np.full(c.rows - rows, -1)])
        want, bound = c.oracle()
        assert ((c.dy[:rows].cpu().double() - want[:rows]).abs() <= bound[:rows]).all()
    c.close()


@pytest.mark.gpu
def test_lowrank_call_refusals(ctx):
    import _lib
    import torch
    c = LowRankCase(ctx, [20, 4], [0, 1], [8, 4], 16, 16)
    buf = torch.zeros(64 * 64, device="cuda")
    p = buf.data_ptr()
    cases = [
        (dict(ldx=15), "inputs: row stride 15 below the 16 values"), (dict(ldy=3), "outputs: row stride 3"),
        (dict(ld_base=1, d_base=p), "base: row stride 1"), (dict(d_y=p + 2), "not aligned to its element type"),
        (dict(d_base=p + 8, d_y=p + 8, ld_base=16, ldy=20), "one buffer with two row strides"),
    ]
    for kw, want in cases:
        args = dict(d_y=p)
        args.update(kw)
        with pytest.raises(_lib.SemError, match=want):
            c.bank.apply(c.plan, p, 0, args.pop("d_y"), 0, stream=ctx.stream, **args)
    with pytest.raises(_lib.SemError, match="null argument"):
        c.bank.apply(c.plan, 0, 0, p, 0)
    h = torch.zeros(64 * 16, device="cuda", dtype=torch.float16)
    for n in (0, 3, -1):
        with pytest.raises(_lib.SemError, match="activation scales for a plan of 2 sequences"):
            c.bank.apply_int8(c.plan, h.data_ptr(), p, n, p)
    c.plan.set(c.offs, np.array([0, 2], np.int32))
    with pytest.raises(_lib.SemError, match="the plan uses adapter 2, the bank has 2"):
        c.bank.apply(c.plan, p, 0, p + 4096, 0)
    with pytest.raises(_lib.SemError, match="more rows"):
        c.plan.set(np.array([0, 25], np.int32), np.array([0], np.int32))
    c.close()


def _norm_case(rows, dim, t, ht, n, post, pre, seed, pads=(0, 0, 0, 0)):
    import torch
    g = torch.Generator().manual_seed(seed)

    def mk(width, pad, dt, scale):
        v = torch.full((rows, width + pad), 77.0).to(_torch(dt))
        v[:, :width] = (torch.randn(rows, width, generator=g) * scale).to(_torch(dt))
        return v

    o, h = mk(dim, pads[0], t, 3.0), mk(dim, pads[1], ht, 5.0)
    ho, y = mk(dim, pads[2], ht, 0.0), mk(dim, pads[3], t, 0.0)
    vec = lambda: 1 + 0.3 * torch.randn(dim, generator=g)  # noqa: E731
    return o, h, ho, y, vec() if post else None, vec() if pre else None, \
        torch.randn(n, dim, generator=g) if n else None, 1 + 0.2 * torch.randn(n, generator=g) if n else None


def _norm_oracle(o, h, post, pre, gates, scales, adapter, eps, dim, t, ht):
    """Results in float64 and bounds. Squares are positive, so a float32 sum of dim of them in any order is off by at
    most dim 2^-24 relative (and a tree by far less), the root and reciprocal halve or keep that and add one rounding
    each; five more products and sums: (dim / 2 + 8) 2^-24 relative to the magnitudes that are added."""
    import torch
    c = (dim / 2 + 8) * 2.0 ** -24
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
    o, h = o[:, :dim].double(), h[:, :dim].double()
    if post is not None:
        o = o / (o.square().mean(1, keepdim=True) + eps).sqrt() * post.double()
    if gates is not None:
        at = torch.from_numpy(np.where(adapter < 0, len(gates), adapter).astype(np.int64))
        o = torch.cat([gates.double(), torch.ones(1, dim, dtype=torch.float64)])[at] * o
        h = torch.cat([scales.double(), torch.ones(1, dtype=torch.float64)])[at][:, None] * h
    out = h + o
    size = c * (h.abs() + o.abs())
    bounds = [size + half[ht] * (out.abs() + size) + (2.0 ** -25 if ht == "f16" else 0)]
    if pre is None:
        return [out], bounds
    inv = 1 / (out.square().mean(1, keepdim=True) + eps).sqrt()
    y = out * inv * pre.double()
    # the errors of one row's values move its root mean square by at most their own root mean square
    e = (size + size.square().mean(1, keepdim=True).sqrt() * (out * inv).abs()) * inv * pre.double().abs() + c * y.abs()
    bounds.append(e + half[t] * (y.abs() + e) + (2.0 ** -25 if t == "f16" else 0))
    return [out, y], bounds


def _run_norm(ctx, rows, dim, t, ht, n=0, use_plan=False, post=True, pre=True, seed=0, pads=(0, 0, 0, 0), alias=False,
              eps=1e-6):
    import torch
    import adapters as ad
    o, h, ho, y, wp, wq, gates, scales = _norm_case(rows, dim, t, ht, n, post, pre, seed, pads)
    rng = np.random.default_rng(seed)
    adapter, plan = np.zeros(rows, int), None
    if use_plan:
        lengths = []
        while sum(lengths) < rows:
            lengths.append(int(min(rng.integers(0, 40), rows - sum(lengths))))
        use = rng.integers(-1, n, len(lengths))
        offs, use = _batch(lengths, use)
        adapter = np.repeat(use, lengths)
        plan = ad.AdapterPlan(ctx, rows, len(lengths))
        plan.set(offs, use)
    bn = ad.BlockNorm(ctx, dim, eps, None if wp is None else wp.numpy(), None if wq is None else wq.numpy(),
                      None if gates is None else gates.numpy(), None if scales is None else scales.numpy())
    do, dh, dho, dy = o.cuda(), h.cuda(), ho.cuda(), y.cuda()
    if alias:
        dho, dy = dh, do
    torch.cuda.synchronize()
    bn.run(rows, do.data_ptr(), DT[t], dh.data_ptr(), DT[ht], dho.data_ptr(), dy.data_ptr() if pre else 0, plan,
           do.stride(0), dh.stride(0), dho.stride(0), dy.stride(0), ctx.stream)
    torch.cuda.synchronize()
    want, bound = _norm_oracle(o, h, wp, wq, gates, scales, adapter, eps, dim, t, ht)
    for got, w, b in zip((dho, dy), want, bound):
        got = got.cpu()
        off = (got[:, :dim].double() - w).abs() - b
        assert (off <= 0).all(), (float(off.max()), np.argwhere(off.numpy() > 0)[:4])
        assert (got[:, dim:] == 77).all()
    if not pre and not alias:
        assert torch.equal(dy.cpu(), y)
    bn.close()
    if plan:
        plan.close()


@pytest.mark.gpu
@pytest.mark.parametrize("t,ht", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("dim", [1, 7, 31, 64, 768, 1000, 1024, 1032, 1153, 4096, 4100, 16384])
def test_block_norm_types_and_widths(ctx, dim, t, ht):
    _run_norm(ctx, 37, dim, t, ht, n=3, use_plan=True, seed=dim)


@pytest.mark.gpu
@pytest.mark.parametrize("post,pre", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("n,use_plan", [(0, False), (1, False), (4, True), (4, False)])
@pytest.mark.parametrize("dim", [96, 97])
def test_block_norm_parts(ctx, post, pre, n, use_plan, dim):
    _run_norm(ctx, 130, dim, "bf16", "f32", n=n, use_plan=use_plan, post=post, pre=pre, seed=n)


@pytest.mark.gpu
@pytest.mark.parametrize("pads", [(1, 2, 3, 5), (8, 8, 8, 8), (0, 4, 0, 0)])
@pytest.mark.parametrize("t,ht", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("dim", [768, 2048])
def test_block_norm_strides(ctx, pads, t, ht, dim):
    _run_norm(ctx, 33, dim, t, ht, n=2, use_plan=True, pads=pads)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [33, 768, 2000, 8192])
def test_block_norm_in_place(ctx, dim):
    _run_norm(ctx, 50, dim, "f32", "f32", n=2, use_plan=True, alias=True)
    _run_norm(ctx, 50, dim, "bf16", "f32", n=2, use_plan=True, alias=True)


@pytest.mark.gpu
def test_block_norm_zero_rows_and_non_finite(ctx):
    import torch
    import adapters as ad
    dim = 128
    bn = ad.BlockNorm(ctx, dim, 1e-6, np.ones(dim), np.ones(dim))
    o, h = torch.randn(6, dim, device="cuda"), torch.randn(6, dim, device="cuda")
    o[0], h[0] = 0, 0           # a row of zeros stays zero
    o[2, 3], h[4, 7] = float("nan"), float("inf")
    ho, y = torch.full_like(h, 9.0), torch.full_like(o, 9.0)
    torch.cuda.synchronize()
    bn.run(0, 0, 0, 0, 0, 0, 0, stream=ctx.stream)  # no rows: nothing is read or written
    bn.run(6, o.data_ptr(), 0, h.data_ptr(), 0, ho.data_ptr(), y.data_ptr(), stream=ctx.stream)
    torch.cuda.synchronize()
    assert (ho[0] == 0).all() and (y[0] == 0).all()
    assert torch.isnan(ho[2]).all() and torch.isnan(y[2]).all()
    assert torch.isinf(ho[4, 7]) and torch.isnan(y[4, 7]) and (y[4, :7] == 0).all()
    for r in (1, 3, 5):
        assert torch.isfinite(ho[r]).all() and torch.isfinite(y[r]).all()
    bn.close()


@pytest.mark.gpu
def test_block_norm_call_refusals(ctx):
    import _lib
    import torch
    import adapters as ad
    dim = 16
    bn = ad.BlockNorm(ctx, dim, 1e-6, np.ones(dim), np.ones(dim), np.ones((2, dim)))
    plan = ad.AdapterPlan(ctx, 10, 4)
    plan.set([0, 4, 10], [0, 2])
    p = torch.zeros(1024, device="cuda").data_ptr()
    q = p + 2048

    def refused(want, rows=10, o=p, t=0, h=p, ht=0, ho=p, y=q, **kw):
        with pytest.raises(_lib.SemError, match=want):
            bn.run(rows, o, t, h, ht, ho, y, **kw)

    refused("the plan uses adapter 2, there are 2", plan=plan)
    refused("9 rows, the plan has 10", rows=9, plan=plan)
    refused("-1 rows", rows=-1)
    refused("null argument", o=0)
    refused("null argument", y=0)
    refused("block outputs: row stride 15", ldo=15)
    refused("residual: row stride 15", ldh=15)
    refused("one buffer with two row strides", ldh=17)
    refused("not aligned to its element type", y=q + 2)
    refused("no form for block outputs of type 0 and a residual of type 1", ht=1)
    bn.close()
    plan.close()


@pytest.mark.gpu
def test_projection_with_adapters_then_block_norm(ctx):
    """A run of them together, as a served block uses them: the shared Q8_0 projection, its adapters beside it on the
    same INT8 codes, then the block norm with the same adapters' gates."""
    import torch
    import adapters as ad
    import runtime
    import synth
    k = n = 768
    rng = np.random.default_rng(12)
    w = runtime.Q8Weight(ctx, synth.q8_0_blocks(rng, n, k), k, n)
    lengths, use = [200, 12, 64, 1, 130], [0, 1, -1, 2, 1]
    c = LowRankCase(ctx, lengths, use, [16, 8, 32], k, n, x="f32", w="f16", seed=4)
    rows = c.rows
    codes = torch.empty(rows, k, dtype=torch.float16, device="cuda")
    absmax = torch.zeros(1, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    w.run(c.dx.data_ptr(), rows, c.dbase.data_ptr(), codes.data_ptr(), absmax.data_ptr(), s.cuda_stream)
    c.bank.apply_int8(c.plan, codes.data_ptr(), absmax.data_ptr(), 1, c.dy.data_ptr(), c.dbase.data_ptr(),
                      stream=s.cuda_stream)
    gates = (1 + 0.2 * rng.standard_normal((3, n))).astype(np.float32)
    scales = np.array([1.0, 0.5, 0.75], np.float32)
    post, pre = np.full(n, 0.9, np.float32), np.full(n, 1.1, np.float32)
    bn = ad.BlockNorm(ctx, n, 1e-6, post, pre, gates, scales)
    h = torch.randn(rows, n, generator=torch.Generator().manual_seed(3))
    dh, dout = h.cuda(), torch.empty(rows, n, device="cuda")
    s.wait_stream(torch.cuda.current_stream())
    bn.run(rows, c.dy.data_ptr(), 0, dh.data_ptr(), 0, dh.data_ptr(), dout.data_ptr(), c.plan, stream=s.cuda_stream)
    c.bank.check()
    # the adapters: from the codes and the base that the projection wrote
    c.codes, c.x, c.absmax, c.base = 1, codes.float().cpu(), absmax.cpu(), c.dbase.cpu()
    c.verify(c.dy)
    want, bound = _norm_oracle(c.dy.cpu(), h, torch.from_numpy(post), torch.from_numpy(pre), torch.from_numpy(gates),
                               torch.from_numpy(scales), c.adapter, 1e-6, n, "f32", "f32")
    for got, x, b in zip((dh, dout), want, bound):
        assert ((got.cpu().double() - x).abs() <= b).all()
    # without an adapter the row is the projection's own, bit for bit
    none = torch.from_numpy(c.adapter == -1)
    assert torch.equal(c.dy.cpu()[none], c.base[none])
    bn.close()
    w.close()
    c.close()
