"""sem_embed_adapted: adapters of many requests in the model's forward, against
the forward written out in numpy (the oracle's quantiser, projections, norms,
softmax and GELU; the adapters in float64) on a small model.

Tolerance: the model's INT8 codes turn a float32 rounding difference into a
code now and then, as between the reference's own builds; the bound is the one
of the other forward tests (cosine >= 0.9995, max abs <= 2e-3).
"""
import ctypes as C

import numpy as np
import pytest

import synth
from conftest import cosine

H, F, HD, NH, LAYERS, VOCAB = 768, 1152, 256, 3, 2, 64
F32, F16, BF16, Q8 = 0, 1, 30, 8
SHAPES = {"attn_q": (H, NH * HD), "attn_k": (H, HD), "attn_v": (H, HD), "attn_output": (H, H), "ffn_gate": (H, F),
          "ffn_up": (H, F), "ffn_down": (F, H)}


def _model_tensors(seed=5):
    rng = np.random.default_rng(seed)
    t = {"token_embd.weight": (Q8, (H, VOCAB), synth.q8_0_blocks(rng, VOCAB, H))}

    def norm(name, n):
        t[name] = (F32, (n,), (1 + 0.1 * rng.standard_normal(n)).astype(np.float32))

    norm("output_norm.weight", H)
    for l in range(LAYERS):
        for p, (k, n) in SHAPES.items():
            t[f"blk.{l}.{p}.weight"] = (Q8, (k, n), synth.q8_0_blocks(rng, n, k))
        for p, n in (("attn_norm", H), ("ffn_norm", H), ("attn_q_norm", HD), ("attn_k_norm", HD),
                     ("post_attention_norm", H), ("post_ffw_norm", H)):
            norm(f"blk.{l}.{p}.weight", n)
    return t


def _adapter(rng, rank, dtype, projections=tuple(SHAPES), layers=range(LAYERS), gates=False, size=1.0):
    t = {}
    for l in layers:
        for p in projections:
            k, n = SHAPES[p]
            for half, shape, sigma in (("a", (rank, k), k ** -0.5), ("b", (n, rank), size * 0.3 * rank ** -0.5)):
                w = (rng.standard_normal(shape) * sigma).astype(np.float32)
                w = w.astype(np.float16) if dtype == F16 else (w.view(np.uint32) >> 16).astype(np.uint16) if dtype == BF16 else w
                t[f"blk.{l}.{p}.weight.lora_{half}"] = (dtype, shape[::-1], w)
        if gates:
            for b in ("attn_residual", "ffn_residual"):
                t[f"blk.{l}.{b}.gate"] = (F32, (H,), (1 + 0.3 * rng.standard_normal(H)).astype(np.float32))
                t[f"blk.{l}.{b}.scale"] = (F32, (1,), np.array([0.8], np.float32))
    return t


def _wide(dtype, w):
    return (w.astype(np.uint32) << 16).view(np.float32).astype(np.float64) if dtype == BF16 else w.astype(np.float64)


class Forward:
    """One sequence through the model with one adapter (or none), step by step."""

    def __init__(self, tensors):
        self.t = tensors

    def run(self, ids, adapter=None, alpha=0.0, dim=H):
        import oracle
        t = self.t
        ad = adapter or {}
        w = lambda n: t[n][2]  # noqa: E731

        def project(name, codes, sc):
            p = name.split(".")[2]
            y = oracle.matmul_q8_0_int8(w(name), codes, sc, SHAPES[p][1])
            a = ad.get(name + ".lora_a")
            if a is None:
                return y
            b = ad[name + ".lora_b"]
            x = codes.astype(np.float64) * np.float64(np.float32(sc))
            scale = alpha / a[2].shape[0] if alpha else 1.0
            return (y + scale * (x @ _wide(a[0], a[2]).T) @ _wide(b[0], b[2]).T).astype(np.float32)

        raw = w("token_embd.weight")[ids]
        d = np.ascontiguousarray(raw[:, :, :2]).view(np.float16).astype(np.float32)
        h = (raw[:, :, 2:].view(np.int8).astype(np.float32) * d).reshape(len(ids), H) * np.float32(np.sqrt(np.float64(H)))
        pos = np.arange(len(ids), dtype=np.float32)
        freq = np.array([1.0 / 10000.0 ** (2 * i / HD) for i in range(HD // 2)], np.float32)
        theta = (pos[:, None] * freq[None]).astype(np.float64)
        cs, sn = np.cos(theta).astype(np.float32), np.sin(theta).astype(np.float32)

        def rope(x):
            lo, hi = x[:, :HD // 2], x[:, HD // 2:]
            return np.concatenate([lo * cs - hi * sn, lo * sn + hi * cs], axis=1)

        for l in range(LAYERS):
            n = lambda s: f"blk.{l}.{s}"  # noqa: B023, E731
            codes, sc = oracle.quantize_sym_int8(oracle.rmsnorm(h, w(n("attn_norm.weight")), 1e-6))
            q = project(n("attn_q.weight"), codes, sc)
            k = rope(oracle.rmsnorm(project(n("attn_k.weight"), codes, sc), w(n("attn_k_norm.weight")), 1e-6))
            v = project(n("attn_v.weight"), codes, sc)
            out = np.empty((len(ids), NH * HD), np.float32)
            for j in range(NH):
                qj = rope(oracle.rmsnorm(np.ascontiguousarray(q[:, j * HD:(j + 1) * HD]), w(n("attn_q_norm.weight")), 1e-6))
                s = (qj.astype(np.float64) @ k.T.astype(np.float64) / 16).astype(np.float32)
                p = np.stack([oracle.softmax(r) for r in s])
                out[:, j * HD:(j + 1) * HD] = p.astype(np.float64) @ v
            for name, post, block in (("attn_output", "post_attention_norm", "attn_residual"),
                                      ("ffn_down", "post_ffw_norm", "ffn_residual")):
                if name == "ffn_down":
                    codes, sc = oracle.quantize_sym_int8(oracle.rmsnorm(h, w(n("ffn_norm.weight")), 1e-6))
                    out = oracle.gelu_quick(project(n("ffn_gate.weight"), codes, sc)) * project(n("ffn_up.weight"), codes, sc)
                codes, sc = oracle.quantize_sym_int8(out)
                o = oracle.rmsnorm(project(n(name + ".weight"), codes, sc), w(n(post + ".weight")), 1e-6)
                if n(block + ".gate") in ad:
                    o = o * ad[n(block + ".gate")][2]
                if n(block + ".scale") in ad:
                    h = h * ad[n(block + ".scale")][2]
                h = h + o
        e = oracle.rmsnorm(h, w("output_norm.weight"), 1e-6).astype(np.float64).mean(axis=0)[:dim]
        return e / np.linalg.norm(e)


@pytest.fixture(scope="module")
def tensors():
    return _model_tensors()


@pytest.fixture(scope="module")
def model(ctx, tensors):
    import _lib
    import runtime
    cfg = _lib.ModelConfig(VOCAB, H, LAYERS, NH, 1, HD, F, 2048, 1e-6, 10000.0, 1 / 16)
    m = runtime.load_model_from_views(ctx, cfg, tensors)
    yield m
    m.close()


def _near(got, want):
    assert cosine(got, want) >= 0.9995
    assert np.abs(got - want).max() <= 2e-3


LENGTHS = [20, 1, 40, 130, 12, 9]


@pytest.mark.gpu
def test_adapted_batch_matches_the_written_out_forward(model, tensors):
    # mixed types, ranks and alphas in one batch, one adapter with gates, short and long sequences, two without
    rng = np.random.default_rng(9)
    ads = [(_adapter(rng, 8, F16), 16.0), (_adapter(rng, 16, BF16, gates=True), 0.0),
           (_adapter(rng, 5, F32, projections=("attn_q", "ffn_down")), 5.0)]
    a = model.load_adapters(ads)
    ids, offs = synth.token_batch(3, LENGTHS, VOCAB)
    use, dims = [0, -1, 1, 0, 2, -1], [768, 512, 768, 256, 768, 768]
    got = model.forward_batch_adapted(a, ids, offs, use, dims)
    plain = model.forward_batch(ids, offs, dims)
    fw = Forward(tensors)
    for i, u in enumerate(use):
        seq = ids[offs[i]:offs[i + 1]]
        want = fw.run(seq, ads[u][0] if u >= 0 else None, ads[u][1] if u >= 0 else 0.0, dims[i])
        _near(got[i], want)
        if u >= 0:  # the adapter does something that the bound above would see
            assert np.abs(plain[i] - want).max() > 1e-2
        else:
            _near(plain[i], want)
    a.close()


@pytest.mark.gpu
@pytest.mark.parametrize("projection", list(SHAPES))
def test_each_projection(model, tensors, projection):
    rng = np.random.default_rng(21)
    ads = [(_adapter(rng, 12, F16, projections=(projection,), size=3.0), 12.0)]
    a = model.load_adapters(ads)
    ids, offs = synth.token_batch(8, [30, 17, 140], VOCAB)
    got = model.forward_batch_adapted(a, ids, offs, [0, 0, 0])
    plain = model.forward_batch(ids, offs)
    for i in range(3):
        want = Forward(tensors).run(ids[offs[i]:offs[i + 1]], ads[0][0], 12.0)
        _near(got[i], want)
        assert np.abs(plain[i] - want).max() > 2e-3
    a.close()


@pytest.mark.gpu
def test_none_and_zero_adapters_change_nothing(model):
    rng = np.random.default_rng(2)
    zero = _adapter(rng, 8, F16)
    for k in zero:
        if k.endswith("lora_b"):
            zero[k] = (F16, zero[k][1], np.zeros_like(zero[k][2]))
    a = model.load_adapters([(zero, 8.0), (_adapter(rng, 8, F16), 8.0)])
    ids, offs = synth.token_batch(4, LENGTHS, VOCAB)
    plain = model.forward_batch(ids, offs)
    for use in ([-1] * 6, [0, -1, 0, 0, -1, 0]):  # adding zeros to a float changes no bit (but a zero's sign)
        for x, y in zip(model.forward_batch_adapted(a, ids, offs, use), plain):
            np.testing.assert_array_equal(x, y)
    # beside another sequence's adapter, the others keep the model's result
    got = model.forward_batch_adapted(a, ids, offs, [1, -1, -1, -1, -1, -1])
    assert not np.array_equal(got[0], plain[0])
    for x, y in zip(got[1:], plain[1:]):
        np.testing.assert_array_equal(x, y)
    # the same batch again, a larger one (the plan and the workspace grow), then the model without adapters
    again = model.forward_batch_adapted(a, ids, offs, [1, -1, -1, -1, -1, -1])
    np.testing.assert_array_equal(got[0], again[0])
    ids2, offs2 = synth.token_batch(6, [200] * 8 + [5] * 30, VOCAB)
    model.forward_batch_adapted(a, ids2, offs2, [i % 3 - 1 for i in range(38)])
    again = model.forward_batch_adapted(a, ids, offs, [1, -1, -1, -1, -1, -1])
    np.testing.assert_array_equal(got[0], again[0])
    for x, y in zip(model.forward_batch(ids, offs), plain):
        np.testing.assert_array_equal(x, y)
    assert model.forward_batch_adapted(a, np.zeros(0, np.int32), np.zeros(1, np.int32), []) == []
    a.close()


@pytest.mark.gpu
def test_adapter_refusals(model, ctx, tensors):
    import _lib
    import runtime
    rng = np.random.default_rng(1)
    good = _adapter(rng, 4, F16, projections=("attn_q",), layers=[0])
    a, b = "blk.0.attn_q.weight.lora_a", "blk.0.attn_q.weight.lora_b"

    def refused(change, want, alpha=1.0):
        t = dict(good)
        t.update(change)
        t = {k: v for k, v in t.items() if v is not None}
        with pytest.raises(_lib.SemError, match=want):
            model.load_adapters([(good, 1.0), (t, alpha)])

    refused({b: None}, "adapter 1: .*lora_a without its other half")
    refused({a: None}, "adapter 1: .*lora_b without its other half")
    refused({"blk.7.attn_q.weight.lora_a": good[a]}, "adapter 1: unknown tensor blk.7.attn_q")
    refused({"blk.00.attn_q.weight.lora_a": good[a]}, "unknown tensor blk.00")
    refused({"output.weight.lora_a": good[a]}, "unknown tensor output.weight.lora_a")
    refused({a: (F16, (H, 3), good[a][2][:3])}, r"lora_b \{4,768\}")
    refused({a: (F16, (H - 1, 4), good[a][2])}, r"want \{768,rank\}")
    refused({a: (F16, (H, 129), np.zeros((129, H), np.float16)), b: (F16, (129, H), np.zeros((H, 129), np.float16))},
            "rank 1..128")
    refused({a: (Q8, good[a][1], good[a][2])}, "type 8, want F32, F16 or BF16")
    refused({a: (F32, good[a][1], good[a][2])}, "bytes")
    refused({"blk.1.ffn_residual.gate": (F32, (H - 1,), np.ones(H - 1, np.float32))}, "want 768 F32 values")
    refused({}, "alpha must be finite", float("inf"))
    ad = model.load_adapters([(good, 1.0)])
    ids, offs = synth.token_batch(4, [3, 4], VOCAB)
    for use in ([0, 1], [-2, 0]):
        with pytest.raises(_lib.SemError, match=r"adapter (1|-2) out of range \(-1..0\)"):
            model.forward_batch_adapted(ad, ids, offs, use)
    with pytest.raises(ValueError, match="1 adapters for 2 sequences"):
        model.forward_batch_adapted(ad, ids, offs, [0])
    with pytest.raises(ValueError, match="1 output widths for 2 sequences"):
        model.forward_batch_adapted(ad, ids, offs, [0, 0], [128])
    with pytest.raises(_lib.SemError, match="empty input"):
        model.forward_batch_adapted(ad, ids, np.array([0, 3, 3], np.int32), [0, 0])
    with pytest.raises(_lib.SemError, match="token ID out of range"):
        model.forward_batch_adapted(ad, ids + VOCAB, offs, [0, 0])
    cfg = _lib.ModelConfig(VOCAB, H, LAYERS, NH, 1, HD, F, 2048, 1e-6, 10000.0, 1 / 16)
    other = runtime.load_model_from_views(ctx, cfg, tensors)
    with pytest.raises(_lib.SemError, match="belong to another model"):
        other.forward_batch_adapted(ad, ids, offs, [0, 0])
    other.close()
    ad.close()


def test_calls_without_a_model():
    import _lib
    lib = _lib.load()
    h = C.c_void_p()
    assert lib.sem_model_adapters_create(None, None, -1, C.byref(h)) == _lib.SEM_EINVAL
    assert b"negative count -1" in lib.sem_last_error()
    assert lib.sem_model_adapters_create(None, None, 0, C.byref(h)) == _lib.SEM_EINVAL
    assert lib.sem_embed_adapted(None, None, None, None, 0, None, None, None) == _lib.SEM_EINVAL
    assert lib.sem_model_adapters_free(None) == _lib.SEM_OK
