"""The cases on which the expert and 8-bit matrix products are timed and checked.

Four ways a program reaches them:

* ``grouped``   one product per expert: rows sorted by expert times that expert's weights;
* ``backward``  the gradients of that product by its rows and by its weights;
* ``int8``      8-bit rows times 8-bit weights with a scale for each row and each channel,
                for one weight matrix (``experts == 0``) or one matrix for each expert;
* ``linear8``   the same from 16-bit rows: each row is quantized, then multiplied.

``run`` computes a case in its plain form (elementary torch operations in 32 bits, integer sums
in 64) or, where ``own`` is true, through :mod:`emmy_ptx_compiler_b200.products`.  ``exact``
computes the same outputs from the definitions in 64 bits.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed() -> list[dict]:
    """``tokens`` rows each go to ``topk`` of ``experts`` experts (``skew`` 0: evenly; larger: a few
    experts take most rows, some take none); weights are ``n`` outputs by ``k`` inputs."""
    return [
        # one sequence being decoded: eight experts read for one row each, latency counts
        {"name": "grouped_one_token", "op": "grouped", "dtype": "bfloat16", "tokens": 1, "topk": 8, "experts": 64,
         "n": 1024, "k": 2048, "skew": 0.0, "out": "bfloat16"},
        # a batch of sequences being decoded: nearly every expert's weights are read for a few rows
        {"name": "grouped_decode_batch", "op": "grouped", "dtype": "bfloat16", "tokens": 64, "topk": 8, "experts": 64,
         "n": 2048, "k": 4096, "skew": 0.0, "out": "bfloat16"},
        # a short prompt with an uneven router: ragged groups, sizes off every tile
        {"name": "grouped_ragged_prompt", "op": "grouped", "dtype": "float16", "tokens": 1777, "topk": 4,
         "experts": 24, "n": 1416, "k": 1000, "skew": 1.0, "out": "float32"},
        # the forward pass of a training step
        {"name": "grouped_train_forward", "op": "grouped", "dtype": "bfloat16", "tokens": 16384, "topk": 4,
         "experts": 16, "n": 4096, "k": 2048, "skew": 0.3, "out": "bfloat16"},
        # fine-tuning on a short sequence, with an odd number of channels; weight gradients kept in 32 bits
        {"name": "backward_short_odd", "op": "backward", "dtype": "bfloat16", "tokens": 511, "topk": 2, "experts": 8,
         "n": 777, "k": 1000, "skew": 0.5, "out": "float32"},
        # half-precision training of small experts on a few sequences
        {"name": "backward_small_experts", "op": "backward", "dtype": "float16", "tokens": 4096, "topk": 2,
         "experts": 32, "n": 512, "k": 1024, "skew": 0.5, "out": "float16"},
        # the backward pass of a training step
        {"name": "backward_train", "op": "backward", "dtype": "bfloat16", "tokens": 16384, "topk": 2, "experts": 16,
         "n": 4096, "k": 2048, "skew": 0.3, "out": "bfloat16"},
        # one token through a quantized dense layer
        {"name": "int8_one_token", "op": "int8", "dtype": "int8", "tokens": 1, "topk": 1, "experts": 0, "n": 4096,
         "k": 4096, "skew": 0.0, "out": "bfloat16", "bias": False},
        # a prompt through quantized experts
        {"name": "int8_experts", "op": "int8", "dtype": "int8", "tokens": 2048, "topk": 4, "experts": 16, "n": 2048,
         "k": 2048, "skew": 0.5, "out": "bfloat16", "bias": False},
        # long prompts through a wide quantized layer with a bias
        {"name": "int8_wide", "op": "int8", "dtype": "int8", "tokens": 8192, "topk": 1, "experts": 0, "n": 8192,
         "k": 8192, "skew": 0.0, "out": "float16", "bias": True},
        # a decode batch from 16-bit activations: the rows are quantized on the way
        {"name": "linear8_decode_batch", "op": "linear8", "dtype": "bfloat16", "tokens": 16, "topk": 1, "experts": 0,
         "n": 4096, "k": 4096, "skew": 0.0, "out": "bfloat16", "bias": True},
        # long prompts, a narrow output: reading and quantizing the rows weighs as much as the product
        {"name": "linear8_long_prompt", "op": "linear8", "dtype": "bfloat16", "tokens": 16381, "topk": 1,
         "experts": 0, "n": 1024, "k": 8192, "skew": 0.0, "out": "bfloat16", "bias": False},
    ]


def _log_uniform(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    """One more case of the same ranges: 1 to 16384 tokens, 1 to 8 of up to 64 experts, 256 to 8192
    channels, mostly whole 16-byte rows, sometimes any number."""
    while True:
        op = rng.choice(["grouped", "backward", "int8", "linear8"])
        eight = op in ("int8", "linear8")
        experts = rng.choice([0, 0, 8, 16]) if eight else rng.choice([8, 12, 16, 24, 32, 64])
        topk = 1 if experts == 0 else rng.choice([1, 2, 4, 8])
        tokens = _log_uniform(rng, 1, 16384)
        n, k = _log_uniform(rng, 256, 8192), _log_uniform(rng, 256, 8192)
        if rng.random() < 0.8:
            step = 16 if eight else 8
            n, k = n // step * step, k // step * step
        case = {"op": op, "dtype": rng.choice(["bfloat16", "float16"]), "tokens": tokens, "topk": topk,
                "experts": experts, "n": n, "k": k, "skew": 0.0 if experts == 0 else rng.choice([0.0, 0.5, 1.0])}
        if op == "int8":
            case["dtype"] = "int8"
            case["out"] = rng.choice(["bfloat16", "float16", "float32"])
        else:
            case["out"] = rng.choice([case["dtype"], case["dtype"], "float32"])
        if eight:
            case["bias"] = rng.random() < 0.5
        cost = work(case)
        if cost["flops"] <= 1.1e12 and cost["bytes"] <= 1.1e9 and max(1, experts) * n * k <= 1 << 29:
            return case


def _counts(case: dict, seed: int) -> list[int]:
    """Rows of each expert: every token takes its ``topk`` best of seeded router scores."""
    rng = np.random.default_rng(seed)
    t, e = case["tokens"], max(1, case["experts"])
    scores = rng.gumbel(size=(t, e)) - case["skew"] * np.log(np.arange(1, e + 1))
    best = np.argsort(-scores, axis=1)[:, :case["topk"]]
    return np.bincount(best.reshape(-1), minlength=e).tolist()


def _inputs(case: dict, seed: int) -> dict:
    """The seeded inputs of a case, on the GPU, with each group's rows one after the other."""
    counts = _counts(case, seed)
    rows, e, n, k = sum(counts), max(1, case["experts"]), case["n"], case["k"]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)

    s = {"case": dict(case), "counts": counts,
         "offsets": torch.tensor([0] + np.cumsum(counts).tolist(), dtype=torch.int32, device="cuda")}
    if case["op"] in ("grouped", "backward"):
        dt = DTYPES[case["dtype"]]
        s["w"] = normal(e, n, k, std=k ** -0.5, dtype=dt)
        s["x"] = normal(rows, k, dtype=dt)
        if case["op"] == "grouped":
            s["out"] = torch.empty(rows, n, dtype=DTYPES[case["out"]], device="cuda")
        else:
            s["dy"] = normal(rows, n, std=0.01, dtype=dt)
            s["dx"] = torch.empty(rows, k, dtype=dt, device="cuda")
            s["dw"] = torch.empty(e, n, k, dtype=DTYPES[case["out"]], device="cuda")
        return s
    # quantized weights: 8-bit values of a layer whose channels differ in size, a scale for each
    shape = (n, k) if case["experts"] == 0 else (e, n, k)
    s["wq"] = torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=g)
    s["ws"] = (normal(*shape[:-1]).abs() + 0.5) * (k ** -0.5 / 73.0)
    s["bias"] = normal(*shape[:-1]) if case["bias"] else None
    s["out"] = torch.empty(rows, n, dtype=DTYPES[case["out"]], device="cuda")
    # activations: a few channels are much larger than the others
    x = normal(rows, k)
    x *= 1.0 + 20.0 * (torch.rand(k, device="cuda", generator=g) < 0.01)
    if case["op"] == "linear8":
        s["x"] = x.to(DTYPES[case["dtype"]])
        s["xq"] = torch.empty(rows, k, dtype=torch.int8, device="cuda")
        s["xs"] = torch.empty(rows, dtype=torch.float32, device="cuda")
    else:
        s["xs"] = x.abs().amax(1) / 127.0
        s["xq"] = (x / s["xs"][:, None]).round().clamp(-127, 127).to(torch.int8)
    return s


def prepare(case: dict, seed: int) -> dict:
    s = _inputs(case, seed)
    if own and case["tokens"] <= 64 and case["op"] != "backward":
        _bind(s, _current_stream(s))
    return s


def _current_stream(s: dict) -> int:
    # what torch.cuda.current_stream().cuda_stream holds, without the 2 us of making its objects
    return torch._C._cuda_getCurrentRawStream(s["out"].device.index)


def _bind(s: dict, stream: int) -> None:
    """The calls of a decode loop, which works on the same buffers step after step and so binds them once;
    a bound call stays with its stream."""
    from emmy_ptx_compiler_b200 import products

    s["stream"] = stream
    if s["case"]["op"] == "grouped":
        s["calls"] = [products.bind_grouped_matmul(s["x"], s["w"], s["offsets"], s["out"], stream=stream)]
        return
    s["calls"] = [products.bind_int8_matmul(s["xq"], s["xs"], s["wq"], s["ws"], s["out"], offsets=_groups(s),
                                            bias=s["bias"], stream=stream)]
    if s["case"]["op"] == "linear8":
        s["calls"].insert(0, products.bind_quantize_rows(s["x"], s["xq"], s["xs"], stream=stream))


def _groups(s: dict):
    return None if s["case"]["experts"] == 0 else s["offsets"]


def _run_own(s: dict):
    from emmy_ptx_compiler_b200 import products

    op = s["case"]["op"]
    if "calls" in s:
        if s["stream"] != _current_stream(s):
            _bind(s, _current_stream(s))
        for call in s["calls"]:
            call()
        return s["out"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "grouped":
        products.grouped_matmul(s["x"], s["w"], s["offsets"], s["out"], stream=stream)
        return s["out"]
    if op == "backward":
        # the rows' gradient is the same product with the weights' two axes exchanged
        products.grouped_matmul(s["dy"], s["w"].transpose(1, 2), s["offsets"], s["dx"], stream=stream)
        products.grouped_matmul_dw(s["dy"], s["x"], s["offsets"], s["dw"], stream=stream)
        return s["dx"], s["dw"]
    if op == "linear8":
        products.quantize_rows(s["x"], s["xq"], s["xs"], stream=stream)
    products.int8_matmul(s["xq"], s["xs"], s["wq"], s["ws"], s["out"], offsets=_groups(s), bias=s["bias"],
                         stream=stream)
    return s["out"]


def run(s: dict):
    if own:
        return _run_own(s)
    case, op = s["case"], s["case"]["op"]
    ends = np.cumsum(s["counts"]).tolist()
    spans = [(i, b - c, b) for i, (c, b) in enumerate(zip(s["counts"], ends)) if c]
    if op == "grouped":
        parts = [s["x"][a:b].float() @ s["w"][i].float().t() for i, a, b in spans]
        return torch.cat(parts).to(DTYPES[case["out"]])
    if op == "backward":
        dx = torch.cat([s["dy"][a:b].float() @ s["w"][i].float() for i, a, b in spans])
        dw = torch.zeros(s["w"].shape, dtype=torch.float32, device=dx.device)
        for i, a, b in spans:
            dw[i] = s["dy"][a:b].float().t() @ s["x"][a:b].float()
        return dx.to(s["x"].dtype), dw.to(DTYPES[case["out"]])
    if op == "linear8":
        # torch multiplies by the rounded 1 / 127 in 32 bits, which is not the rounded quotient
        xs = (s["x"].abs().amax(1).double() / 127.0).float()
        # a quotient next to a half needs more than 32 bits to round to the right side of it
        xq = (s["x"].double() / xs.double()[:, None]).round().clamp(-127, 127)
        xq = torch.where(xs[:, None] > 0, xq, torch.zeros_like(xq))
    else:
        xs, xq = s["xs"], s["xq"].double()
    parts = []
    for i, a, b in spans:
        wq, ws, bias = s["wq"], s["ws"], s["bias"]
        if case["experts"]:
            wq, ws, bias = wq[i], ws[i], None if bias is None else bias[i]
        # sums of 8-bit products pass 24 bits, so the product runs in 64
        y = (xq[a:b] @ wq.double().t()).float() * xs[a:b, None] * ws
        parts.append(y if bias is None else y + bias)
    return torch.cat(parts).to(DTYPES[case["out"]])


def exact(case: dict, seed: int):
    """The outputs from the definitions, in 64 bits: every output is a sum over one contracted axis."""
    s = _inputs(case, seed)
    f64 = torch.float64
    expert = torch.repeat_interleave(torch.arange(len(s["counts"])), torch.tensor(s["counts"])).cuda()

    def rows_of(i):
        return (expert == i).nonzero()[:, 0]

    if case["op"] in ("grouped", "backward"):
        w = s["w"]
        y = torch.zeros(len(expert), case["n"] if case["op"] == "grouped" else case["k"], dtype=f64, device="cuda")
        dw = None if case["op"] == "grouped" else torch.zeros(w.shape, dtype=f64, device="cuda")
        for i in range(w.shape[0]):
            r = rows_of(i)
            x, wi = s["x"].index_select(0, r).to(f64), w[i].to(f64)
            if dw is None:
                y.index_copy_(0, r, torch.einsum("tk,nk->tn", x, wi))
            else:
                dy = s["dy"].index_select(0, r).to(f64)
                y.index_copy_(0, r, torch.einsum("tn,nk->tk", dy, wi))
                dw[i] = torch.einsum("tn,tk->nk", dy, x)
        return y if dw is None else (y, dw)
    e = max(1, case["experts"])
    wq, ws = s["wq"].view(e, case["n"], case["k"]), s["ws"].view(e, case["n"]).to(f64)
    if case["op"] == "linear8":
        # a row's scale is its largest magnitude over 127, held in 32 bits; ties round to the even integer
        peak = torch.maximum(s["x"].max(1).values, -s["x"].min(1).values)
        scale = (peak.to(f64) / 127.0).to(torch.float32).to(f64)
        q = torch.round(s["x"].to(f64) / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None])
        q = q.clamp_(-127, 127)
    else:
        scale, q = s["xs"].to(f64), s["xq"].to(f64)
    y = torch.zeros(len(expert), case["n"], dtype=f64, device="cuda")
    for i in range(e):
        r = rows_of(i)
        total = torch.einsum("tk,nk->tn", q.index_select(0, r), wq[i].to(f64))
        total = total * (scale.index_select(0, r)[:, None] * ws[i][None, :])
        if s["bias"] is not None:
            total = total + s["bias"].view(e, case["n"])[i].to(f64)
        y.index_copy_(0, r, total)
    return y


def work(case: dict) -> dict:
    """Bytes that have to move (each input read once, each output written once) and operations."""
    e, n, k = max(1, case["experts"]), case["n"], case["k"]
    rows = case["tokens"] * case["topk"]
    # experts that get a row, for an even router; an uneven one reaches no more of them
    active = e if e == 1 else e * (1.0 - (1.0 - case["topk"] / e) ** case["tokens"])
    out = DTYPES[case["out"]].itemsize
    flops = 2.0 * rows * n * k
    if case["op"] == "grouped":
        return {"bytes": 2.0 * rows * k + 2.0 * active * n * k + out * rows * n, "flops": flops}
    if case["op"] == "backward":
        return {"bytes": 2.0 * rows * (n + 2 * k) + (2.0 * active + out * e) * n * k, "flops": 2.0 * flops}
    size = 1.0 if case["op"] == "int8" else 2.0
    scales = 4.0 * (rows if case["op"] == "int8" else 0) + 4.0 * active * n * (2 if case["bias"] else 1)
    return {"bytes": size * rows * k + active * n * k + scales + out * rows * n, "flops": flops}
