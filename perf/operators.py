"""Cases of the per-request adapter operators: low-rank adapters beside a shared
projection, and the norms around a block fused with its gate and residual scale.

A served batch is packed sequences, each of which names an adapter (or none).
The low-rank operator adds scale_a * (x A_a^T) B_a^T to the rows of every
sequence of adapter a, next to the output of the projection they share; the
block-norm operator computes h' = s_a h + g_a * rmsnorm(o) w_post and
y = rmsnorm(h') w_pre, with the gate g_a and the residual scale s_a of the row's
adapter.

own = False runs the plain forms (elementary torch operations in 32 bits),
own = True the framework's operators.
"""
import math
import random

import torch

own = False

SIZE = {"f32": 4, "f16": 2, "bf16": 2, "int8": 2}  # int8 codes are held as fp16, the projections' operand type
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.float16}


def listed():
    return [
        # one short query of a tenant with its own adapter: latency
        lowrank("query_12x768_r8", 1, 12, 12, 1, 8, "f32", 768, 768),
        # 48 queries of 48 tenants, every one with its own adapter and rank, in half precision; some use none
        lowrank("tenants_48_r16", 48, 1, 24, 48, 16, "f16", 768, 1280, mixed=True, none=0.1),
        # a small request batch on the quantised path: the projection's INT8 codes, one scale per sequence
        lowrank("codes_8x64_r16", 8, 64, 64, 4, 16, "int8", 768, 2304),
        # odd widths, rows longer than the part that is read, ragged sequences and ranks
        lowrank("odd_517x1001", 37, 1, 300, 5, 23, "f32", 517, 1001, mixed=True, none=0.2, pad=3),
        # documents up to the model's context length, many adapters of mixed rank
        lowrank("ragged_bf16_r64", 100, 1, 2048, 33, 64, "bf16", 768, 2304, mixed=True, none=0.05),
        # wide ranks with full-precision weights
        lowrank("wide_32x512_r128", 32, 512, 512, 3, 128, "f16", 768, 1280, weights="f32"),
        # bulk indexing: 512-token documents, few adapters, full precision
        lowrank("bulk_128x512_r16", 128, 512, 512, 8, 16, "f32", 768, 768),
        # bulk indexing through the down projection on INT8 codes
        lowrank("bulk_codes_384x512_r32", 384, 512, 512, 8, 32, "int8", 1152, 768),
        # one token's residual step
        norm("row_1x768", 1, 1, 1, 0, "bf16", "bf16", 768),
        # a small batch with per-request gates
        norm("gated_8x64x768", 8, 64, 64, 4, "f32", "f32", 768),
        # wide half-precision rows over an fp32 residual stream, odd width, no norm before the next block's input
        norm("odd_1153_f16", 61, 1, 300, 7, "f16", "f32", 1153, none=0.2, pre=False),
        # bulk indexing
        norm("bulk_256x512x768", 256, 512, 512, 8, "f32", "f32", 768, none=0.1),
    ]


def lowrank(name, seqs, lo, hi, adapters, rank, dtype, k, n, mixed=False, none=0.0, pad=0, weights="f16", layout=1):
    """seqs sequences of lo..hi tokens; `adapters` adapters of rank up to `rank`; a share `none` of the sequences has no
    adapter; the rows of x are `pad` elements longer than the k that are read."""
    return {"name": name, "op": "lowrank", "seqs": seqs, "lo": lo, "hi": hi, "adapters": adapters, "rank": rank,
            "dtype": dtype, "k": k, "n": n, "mixed": mixed, "none": none, "pad": pad, "layout": layout,
            "weights": "bf16" if dtype == "bf16" and weights == "f16" else weights}


def norm(name, seqs, lo, hi, adapters, dtype, residual, dim, none=0.0, post=True, pre=True, layout=1):
    """`adapters` gates and residual scales (0: none), rows of `dim` in `dtype`, the residual stream in `residual`."""
    return {"name": name, "op": "norm", "seqs": seqs, "lo": lo, "hi": hi, "adapters": adapters, "dtype": dtype,
            "residual": residual, "dim": dim, "none": none, "post": post, "pre": pre, "layout": layout}


def spread(rng, lo, hi):
    """A whole number of lo..hi, even over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    seqs = spread(rng, 1, 256)
    hi = spread(rng, 1, 2048 if seqs <= 48 else 512)
    lo = rng.choice([1, hi, max(1, hi // 2)])
    layout = rng.randrange(1 << 30)
    none = rng.choice([0.0, 0.0, 0.1, 0.3])
    if rng.random() < 0.6:
        k, n = rng.choice([(768, 768), (768, 256), (768, 1280), (768, 2304), (1152, 768),
                           (spread(rng, 16, 1300), spread(rng, 16, 2400))])
        case = lowrank("", seqs, lo, hi, spread(rng, 1, 40), spread(rng, 1, 128), rng.choice(["f32", "f16", "bf16", "int8"]),
                       k, n, mixed=rng.random() < 0.5, none=none, pad=rng.choice([0, 0, 8, 5]),
                       weights=rng.choice(["f16", "f16", "bf16", "f32"]), layout=layout)
    else:
        dtype = rng.choice(["f32", "f16", "bf16"])
        case = norm("", seqs, lo, hi, rng.choice([0, 1, spread(rng, 2, 40)]), dtype, rng.choice([dtype, "f32"]),
                    rng.choice([768, 512, 1024, spread(rng, 8, 1600)]), none=none, post=rng.random() < 0.8,
                    pre=rng.random() < 0.8, layout=layout)
    del case["name"]
    return case


def shape(case):
    """(lengths, adapter of each sequence or -1, ranks): the batch's layout, by the case alone."""
    rng = random.Random(case["layout"] * 1000003 + case["seqs"])
    count = case["adapters"]
    lengths = [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    if count:
        use = [-1 if rng.random() < case["none"] else (i if case["seqs"] <= count else rng.randrange(count))
               for i in range(case["seqs"])]
    else:
        use = [-1] * case["seqs"]
    rank = case.get("rank", 0)
    ranks = [rng.randint(max(1, rank // 8), rank) if case.get("mixed") else rank for _ in range(count)]
    return lengths, use, ranks


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    lengths, use, ranks = shape(case)
    rows = sum(lengths)
    offsets = [0]
    for length in lengths:
        offsets.append(offsets[-1] + length)

    def rand(*size, dtype="f32", scale=1.0):
        return torch.empty(*size, device="cuda").normal_(generator=gen).mul_(scale).to(TORCH[dtype])

    s = {"case": case, "rows": rows, "offsets": offsets, "use": use, "ranks": ranks,
         "seq_of": torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths)).cuda()}
    s["adapter_of"] = torch.tensor(use, device="cuda")[s["seq_of"]]
    if case["op"] == "lowrank":
        k, n, dtype = case["k"], case["n"], case["dtype"]
        out = "f32" if dtype == "int8" else dtype
        if dtype == "int8":
            s["absmax"] = torch.empty(len(lengths), device="cuda").uniform_(2.0, 6.0, generator=gen)
            s["x"] = rand(rows, k).mul_(30).round_().clamp_(-127, 127).half()
        else:
            s["x"] = rand(rows, k + case["pad"], dtype=dtype)[:, :k]
        s["base"] = rand(rows, n, dtype=out)
        s["a"] = [rand(r, k, dtype=case["weights"], scale=k ** -0.5) for r in ranks]
        s["b"] = [rand(n, r, dtype=case["weights"], scale=0.1 * r ** -0.5) for r in ranks]
        s["scale"] = [2.0 / (1 + i % 3) for i in range(len(ranks))]
        s["y"] = torch.empty(rows, n, device="cuda", dtype=TORCH[out])
    else:
        dim, count = case["dim"], case["adapters"]
        s["o"], s["h"] = rand(rows, dim, dtype=case["dtype"], scale=3.0), rand(rows, dim, dtype=case["residual"], scale=5.0)
        s["post"] = 1 + rand(dim, scale=0.2) if case["post"] else None
        s["pre"] = 1 + rand(dim, scale=0.2) if case["pre"] else None
        s["gates"], s["scales"] = rand(count, dim, scale=0.3) + 0.5, rand(count, scale=0.1) + 1
        s["h_out"] = torch.empty_like(s["h"])
        s["y"] = torch.empty_like(s["o"]) if case["pre"] else None
    if own:
        handles(s)
    return s


_context = None


def handles(s):
    """The handles that a serving program keeps: the batch's plan, the adapters' weights on the device."""
    global _context
    import sys
    if "go-semantica_b200" not in sys.path:
        sys.path.insert(0, "go-semantica_b200")
    import _lib
    import adapters
    if _context is None:
        _context = _lib.Context(0)
    case = s["case"]
    code = {"f32": adapters.F32, "f16": adapters.F16, "bf16": adapters.BF16}
    s["plan"] = None
    if case["op"] == "lowrank" or case["adapters"] > 1 or (case["adapters"] and case["none"]):
        s["plan"] = adapters.AdapterPlan(_context, s["rows"], len(s["use"]))
        s["plan"].set(s["offsets"], s["use"])

    def host(w):
        return (w.view(torch.int16) if w.dtype == torch.bfloat16 else w).cpu().numpy()

    if case["op"] == "lowrank":
        s["lowrank"] = adapters.LowRank(_context, case["k"], case["n"], [host(a) for a in s["a"]],
                                        [host(b) for b in s["b"]], s["scale"], code[case["weights"]])
        if case["dtype"] != "int8":
            s["code"] = code[case["dtype"]]
    else:
        s["block"] = adapters.BlockNorm(_context, case["dim"], 1e-6, *(None if w is None else host(w) for w in
                                        (s["post"], s["pre"])), host(s["gates"]), host(s["scales"]))
        s["code"] = code[case["dtype"]], code[case["residual"]]


def run(s):
    case = s["case"]
    if own:
        # the framework takes 0 for its context's stream; 1 is CUDA's handle of the default stream, torch's current one
        stream = torch.cuda.current_stream().cuda_stream or 1
        if case["op"] == "lowrank":
            if case["dtype"] == "int8":
                s["lowrank"].apply_int8(s["plan"], s["x"].data_ptr(), s["absmax"].data_ptr(), len(s["use"]),
                                        s["y"].data_ptr(), d_base=s["base"].data_ptr(), stream=stream)
            else:
                s["lowrank"].apply(s["plan"], s["x"].data_ptr(), s["code"], s["y"].data_ptr(), s["code"],
                                   d_base=s["base"].data_ptr(), ldx=s["x"].stride(0), stream=stream)
            return s["y"]
        o, h = s["o"], s["h"]
        s["block"].run(s["rows"], o.data_ptr(), s["code"][0], h.data_ptr(), s["code"][1], s["h_out"].data_ptr(),
                       0 if s["y"] is None else s["y"].data_ptr(), plan=s["plan"], stream=stream)
        return [s["h_out"]] if s["y"] is None else [s["h_out"], s["y"]]
    return plain_lowrank(s) if case["op"] == "lowrank" else plain_norm(s)


def plain_lowrank(s):
    """Every row against every adapter's rows of A, the columns of other adapters set to zero, then against every B."""
    a = torch.cat([w.float() for w in s["a"]])
    b = torch.cat([w.float() for w in s["b"]], dim=1)
    owner = torch.repeat_interleave(torch.arange(len(s["ranks"])), torch.tensor(s["ranks"])).cuda()
    scale = torch.tensor(s["scale"], device="cuda")[owner]
    x = s["x"].float()
    if s["case"]["dtype"] == "int8":
        x = x * (s["absmax"] / 127)[s["seq_of"], None]
    t = torch.where(owner[None, :] == s["adapter_of"][:, None], (x @ a.T) * scale, 0.0)
    return (s["base"].float() + t @ b.T).to(s["base"].dtype)


def rms(x, w):
    return x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + 1e-6) * w


def plain_norm(s):
    o, h = s["o"].float(), s["h"].float()
    if s["post"] is not None:
        o = rms(o, s["post"])
    if s["case"]["adapters"]:
        gates = torch.cat([s["gates"], torch.ones_like(s["gates"][:1])])  # the last entry, -1: no adapter
        scales = torch.cat([s["scales"], torch.ones_like(s["scales"][:1])])
        o = gates[s["adapter_of"]] * o
        h = scales[s["adapter_of"], None] * h
    h = h + o
    out = [h.to(s["h"].dtype)]
    if s["pre"] is not None:
        out.append(rms(h, s["pre"]).to(s["o"].dtype))
    return out


def work(case):
    lengths, use, ranks = shape(case)
    rows = sum(lengths)
    if case["op"] == "lowrank":
        k, n = case["k"], case["n"]
        out = SIZE["f32" if case["dtype"] == "int8" else case["dtype"]]
        busy = sum(length for length, a in zip(lengths, use) if a >= 0)
        weights = sum(ranks[a] * (k + n) for a in set(use) if a >= 0) * SIZE[case["weights"]]
        flops = sum(2.0 * length * ranks[a] * (k + n) for length, a in zip(lengths, use) if a >= 0)
        return {"bytes": busy * k * SIZE[case["dtype"]] + 2 * rows * n * out + weights, "flops": flops}
    row = case["dim"] * (SIZE[case["dtype"]] * (1 + case["pre"]) + 2 * SIZE[case["residual"]])
    vectors = 4 * case["dim"] * (case["post"] + case["pre"] + len({a for a in use if a >= 0}))
    return {"bytes": rows * row + vectors, "flops": 12.0 * rows * case["dim"]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lowrank":
        y = s["base"].double()
        for i in {a for a in s["use"] if a >= 0}:
            at = (s["adapter_of"] == i).nonzero()[:, 0]
            x = s["x"][at].double()
            if case["dtype"] == "int8":
                x = x * s["absmax"][s["seq_of"][at]].double()[:, None] / 127
            y[at] += s["scale"][i] * torch.mm(torch.mm(x, s["a"][i].double().t()), s["b"][i].double().t())
        return y
    o, h, at = s["o"].double(), s["h"].double(), s["adapter_of"]
    if case["post"]:
        o = o / (o.square().sum(1, keepdim=True) / case["dim"] + 1e-6).sqrt() * s["post"].double()
    with_adapter = (at >= 0)[:, None]
    if case["adapters"]:
        o = torch.where(with_adapter, s["gates"].double()[at.clamp(min=0)] * o, o)
        h = torch.where(with_adapter, s["scales"].double()[at.clamp(min=0)][:, None] * h, h)
    h = h + o
    if not case["pre"]:
        return [h]
    return [h, h / (h.square().sum(1, keepdim=True) / case["dim"] + 1e-6).sqrt() * s["pre"].double()]
