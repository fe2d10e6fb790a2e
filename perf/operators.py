"""The gradient norm, clipping and embedding operators, as they are timed on one GPU.

``run`` computes them in their plain form (elementary torch operations in 32 bits or more) or, with ``own``, through
the calls that a training program makes: ``ops.grad_norm``, ``ops.clip_grad_norm``, ``ops.embedding`` and
``ops.embedding_grad``.

A case is a dict.  Of the gradient norm and of clipping:

  op        norm | clip
  layers    parameter lists: layers of two vectors and five matrices each; 0 = `count` flat buckets
  width     elements of a vector, rows of a matrix; of a bucket: its elements
  count     flat buckets
  dtype     element type of the gradients
  out       clip only: element type of the clipped gradients, "" = in place
  power     2 or 0 (the largest magnitude)
  below     clip only: the norm is below the bound, so that nothing is to be scaled
  offset    elements by which the storage misses its alignment

Of the embedding:

  op        lookup | grad | step (lookup and the gradient of its table through autograd)
  tokens    number of tokens
  rows      rows of the table
  width     elements of a row
  dtype     element type of the table (grad: of the table's gradient)
  out       element type of the looked-up rows (grad: of the rows' gradients)
  ids       element type of the tokens
  spread    zipf (frequencies that fall with the rank) | uniform
  add       grad only: added to what the table's gradient holds, as in a gradient bucket; else written whole
"""
import itertools
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16, "float64": torch.float64,
          "int32": torch.int32, "int64": torch.int64}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2, "float64": 8, "int32": 4, "int64": 8}
MIB = 1 << 20
SCALE = 45.25  # of a looked-up row: about the root of a width of 2048
EPS = 1e-6


def _grads(op, *, layers=0, width, count=0, dtype="float32", out="", power=2, below=False, offset=0):
    return {"op": op, "layers": layers, "width": width, "count": count, "dtype": dtype, "out": out, "power": power, "below": below,
            "offset": offset}


def _rows(op, tokens, rows, width, *, dtype="float32", out="bfloat16", ids="int64", spread="zipf", add=False):
    return {"op": op, "tokens": tokens, "rows": rows, "width": width, "dtype": dtype, "out": out, "ids": ids, "spread": spread,
            "add": add}


def listed():
    cases = {
        # A handful of small tensors: what a call costs by itself.
        "norm_f32_4KiB": _grads("norm", layers=1, width=12),
        # A model's list of gradients, 161 tensors of some 25 M values: the count and the size of ResNet-50's.
        "norm_f32_161_tensors": _grads("norm", layers=23, width=304),
        # Five 25 MiB gradient buckets in place, with a norm below the bound: most steps of a run.
        "clip_f32_buckets_below": _grads("clip", width=25 * MIB // 4, count=5, below=True),
        # 1 G parameters with gradients in bf16, clipped into the fp32 gradients of the optimizer: the largest.
        "clip_bf16_f32_1G": _grads("clip", layers=5, width=4096, dtype="bfloat16", out="float32"),
        # Odd widths and a storage off its boundary, fp16, into other tensors.
        "clip_f16_ragged": _grads("clip", layers=3, width=1001, dtype="float16", out="float16", offset=1),
        # One token for each of eight sequences that are being written.
        "lookup_bf16_8_tokens": _rows("lookup", 8, 32000, 4096, dtype="bfloat16"),
        # A batch of prompts, or the forward pass of training: fp32 weights, bf16 activations.
        "lookup_f32_bf16_16k": _rows("lookup", 16384, 50021, 2048),
        # Few tokens, an odd width, into a bucket.
        "grad_33_tokens_add": _rows("grad", 33, 10007, 770, add=True),
        # A training step's tokens into the fp32 bucket of a wide table.
        "grad_bf16_f32_16k_add": _rows("grad", 16384, 50021, 4096, add=True),
        # The whole gradient of a bf16 table, as autograd hands it on.
        "grad_bf16_8k_dense": _rows("grad", 8192, 100003, 2048, dtype="bfloat16", ids="int32"),
        # Rows of eight ranks, gathered instead of reduced.
        "grad_f32_131k_uniform_add": _rows("grad", 131072, 32000, 1024, out="float32", spread="uniform", add=True),
        # Lookup and gradient through autograd.
        "step_f32_bf16_8k": _rows("step", 8191, 32000, 2048),
    }
    return [dict(c, name=k) for k, c in cases.items()]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "clip", "clip", "lookup", "grad", "grad", "step"])
    if op in ("norm", "clip"):
        dtype = rng.choice(["float32", "float32", "bfloat16", "float16", "float64"])
        layers = rng.choice([0, _log_int(rng, 1, 40)])
        most = 256 * MIB // SIZE[dtype]
        if layers:
            width, count = _log_int(rng, 8, min(4096, int(math.sqrt(most / layers / 12)))), 0
        else:
            count = rng.randint(1, 8)
            width = _log_int(rng, 64, most // count)
        if width >= 64 and rng.random() < 0.5:
            width = width // 16 * 16
        outs = {"float32": ["", "float32", "bfloat16", "float16"], "bfloat16": ["", "bfloat16", "float32"],
                "float16": ["", "float16", "float32"], "float64": ["", "float64"]}[dtype]
        out = rng.choice(outs) if op == "clip" else ""
        return _grads(op, layers=layers, width=width, count=count, dtype=dtype, out=out, power=rng.choice([2, 2, 2, 0]),
                      below=op == "clip" and (out == "" or rng.random() < 0.25), offset=rng.choice([0, 0, 0, 1]))
    table, rows = rng.choice([("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("float16", "float16"),
                              ("float32", "float16"), ("bfloat16", "float32")])
    width = _log_int(rng, 64, 8192)
    if rng.random() < 0.75:
        width = width // 16 * 16
    tokens = _log_int(rng, 1, min(131072, 128 * MIB // width))
    return _rows(op, tokens, _log_int(rng, 100, min(200000, 256 * MIB // width)), width, dtype=table, out=rows,
                 ids=rng.choice(["int64", "int32"]), spread=rng.choice(["zipf", "uniform"]), add=op == "grad" and rng.random() < 0.6)


# ------------------------------------------------------------------ inputs
def _sizes(case):
    w = case["width"]
    if not case["layers"]:
        return [w] * (case["count"] - 1) + [w - w // 3]
    return [w, w, w * w, w * w, 2 * w * w, 4 * w * w, 4 * w * w] * case["layers"]


def _views(flat, sizes, esize, offset):
    """Tensors of `sizes` elements in one storage, each on a 16-byte boundary (plus `offset`)."""
    align = 16 // esize
    ends = itertools.accumulate((n + align - 1) // align * align for n in sizes)
    starts = [offset] + [offset + e for e in ends]
    return [flat[o:o + n] for o, n in zip(starts, sizes)]


def _storage(sizes, esize, offset):
    align = 16 // esize
    return offset + sum((n + align - 1) // align * align for n in sizes)


def _tokens(case, g):
    n, v = case["tokens"], case["rows"]
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    if case["spread"] == "zipf":
        t = (torch.exp(u * math.log(v + 1)) - 1).long().clamp_(0, v - 1)
    else:
        t = (u * v).long().clamp_(0, v - 1)
    gone = torch.rand(n, device="cuda", generator=g) < 1 / 64  # padded places
    return torch.where(gone, -1, t).to(DTYPES[case["ids"]])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if case["op"] in ("norm", "clip"):
        t, sizes, off = DTYPES[case["dtype"]], _sizes(case), case["offset"]
        flat = torch.zeros(_storage(sizes, SIZE[case["dtype"]], off), device="cuda", dtype=t)
        grads = _views(flat, sizes, SIZE[case["dtype"]], off)
        std = 0.5 if t == torch.float16 else 1e-3  # of fp16 gradients the loss was scaled
        [x.normal_(0, std / (1 + k % 5), generator=g) for k, x in enumerate(grads)]
        bound = 1e9 if case["below"] else std * (0.15 * math.sqrt(sum(sizes)) if case["power"] == 2 else 1)
        s = {"case": case, "flat": flat, "grads": grads, "outs": None, "out_flat": flat, "bound": bound}
        if case["out"]:
            s["out_flat"] = torch.zeros(_storage(sizes, SIZE[case["out"]], off), device="cuda", dtype=DTYPES[case["out"]])
            s["outs"] = _views(s["out_flat"], sizes, SIZE[case["out"]], off)
        return s
    v, d = case["rows"], case["width"]
    s = {"case": case, "tokens": _tokens(case, g)}
    if case["op"] in ("lookup", "step"):
        s["weight"] = torch.empty(v, d, device="cuda", dtype=DTYPES[case["dtype"]]).normal_(0, 0.02, generator=g)
    if case["op"] in ("grad", "step"):
        s["dy"] = torch.empty(case["tokens"], d, device="cuda", dtype=DTYPES[case["out"]]).normal_(0, 1e-3, generator=g)
    if case["op"] == "grad":
        s["table"] = torch.empty(v, d, device="cuda", dtype=DTYPES[case["dtype"]]).normal_(0, 1e-3, generator=g)
    if case["op"] == "step":
        s["weight"].requires_grad_(True)
    return s


# -------------------------------------------------------------- plain forms
def _plain_norm(grads, power):
    if power == 2:
        return torch.stack([x.double().square().sum() if x.dtype == torch.float64 else x.float().square().sum(dtype=torch.float64)
                            for x in grads]).sum().sqrt()
    return torch.stack([x.abs().amax().double() for x in grads]).amax()


def _plain_clip(grads, outs, bound, power):
    norm = _plain_norm(grads, power)
    c = torch.clamp(bound / (norm + EPS), max=1.0)
    [o.copy_(x * c if x.dtype == torch.float64 else x.float() * c.float()) for x, o in zip(grads, outs)]
    return norm


def _plain_lookup(tokens, weight, out):
    inside = (tokens >= 0) & (tokens < weight.shape[0])
    rows = weight[torch.where(inside, tokens, 0)].float() * SCALE
    return torch.where(inside[:, None], rows, 0.0).to(out)


def _plain_grad(tokens, dy, rows):
    inside = (tokens >= 0) & (tokens < rows)
    total = torch.zeros(rows, dy.shape[1], device=dy.device, dtype=torch.float32)
    return total.index_add_(0, tokens[inside], dy[inside].float()) * SCALE


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        import allreduce_proto_b200 as ar

        power = 2.0 if case.get("power") == 2 else math.inf
        if op == "norm":
            return ar.ops.grad_norm(state["grads"], norm_type=power)
        if op == "clip":
            norm = ar.ops.clip_grad_norm(state["grads"], state["bound"], out=state["outs"], norm_type=power)
            return norm, state["out_flat"]
        if op == "lookup":
            return ar.ops.embedding(state["tokens"], state["weight"], scale=SCALE, out_dtype=DTYPES[case["out"]])
        if op == "grad":
            return ar.ops.embedding_grad(state["tokens"], state["dy"], out=state["table"], accumulate=case["add"], scale=SCALE)
        state["weight"].grad = None
        y = ar.ops.embedding(state["tokens"], state["weight"], scale=SCALE, out_dtype=DTYPES[case["out"]])
        y.backward(state["dy"])
        return y.detach(), state["weight"].grad
    if op == "norm":
        norm = _plain_norm(state["grads"], case["power"])
        return norm if case["dtype"] == "float64" else norm.float()
    if op == "clip":
        norm = _plain_clip(state["grads"], state["outs"] or state["grads"], state["bound"], case["power"])
        return norm if case["dtype"] == "float64" else norm.float(), state["out_flat"]
    if op == "lookup":
        return _plain_lookup(state["tokens"], state["weight"], DTYPES[case["out"]])
    if op == "grad":
        total = _plain_grad(state["tokens"], state["dy"], case["rows"])
        return state["table"].copy_(state["table"].float() + total if case["add"] else total)
    weight = state["weight"].detach()
    y = _plain_lookup(state["tokens"], weight, DTYPES[case["out"]])
    return y, _plain_grad(state["tokens"], state["dy"], case["rows"]).to(weight.dtype)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "clip"):
        x = s["flat"].double()  # the places between the tensors are zero
        norm = torch.linalg.vector_norm(x, ord=2 if case["power"] == 2 else math.inf)
        if op == "norm":
            return norm
        c = min(1.0, s["bound"] / (float(norm) + EPS))
        if not case["out"] or SIZE[case["out"]] == SIZE[case["dtype"]]:
            return norm, x.mul_(c)
        whole = torch.zeros(s["out_flat"].numel(), device="cuda", dtype=torch.float64)
        torch._foreach_copy_(_views(whole, _sizes(case), SIZE[case["out"]], case["offset"]), [t.double().mul_(c) for t in s["grads"]])
        return norm, whole
    known = torch.nonzero((s["tokens"] >= 0) & (s["tokens"] < case["rows"])).flatten()
    ids = s["tokens"][known].long()
    y = g = None
    if op in ("lookup", "step"):
        y = torch.zeros(case["tokens"], case["width"], device="cuda", dtype=torch.float64)
        y[known] = s["weight"].detach().index_select(0, ids).double().mul_(SCALE)
    if op in ("grad", "step"):
        g = s["table"].double() if case["add"] else torch.zeros(case["rows"], case["width"], device="cuda", dtype=torch.float64)
        g.index_put_((ids,), s["dy"].index_select(0, known).double().mul_(SCALE), accumulate=True)
    return y if op == "lookup" else g if op == "grad" else (y, g)


# --------------------------------------------------------------------- work
def _touched(case):
    """Rows of the table that the tokens are expected to name."""
    n, v = case["tokens"] * 63 / 64, case["rows"]
    if case["spread"] == "uniform":
        return v * -math.expm1(n * math.log1p(-1 / v))
    k = torch.arange(v, dtype=torch.float64)
    p = torch.log((k + 2) / (k + 1)) / math.log(v + 1)
    return float((-torch.expm1(n * torch.log1p(-p))).sum())


def work(case):
    if case["op"] in ("norm", "clip"):
        n = sum(_sizes(case))
        written = SIZE[case["out"]] if case["out"] else 0 if case["below"] else SIZE[case["dtype"]]
        return {"bytes": n * (SIZE[case["dtype"]] + (written if case["op"] == "clip" else 0)) + 4,
                "flops": n * (2 if case["op"] == "norm" or not written else 3)}
    t, d, u = case["tokens"], case["width"], _touched(case)
    w, r = SIZE[case["dtype"]], SIZE[case["out"]]
    lookup = {"bytes": t * SIZE[case["ids"]] + u * d * w + t * d * r, "flops": t * d}
    grad = {"bytes": t * SIZE[case["ids"]] + t * d * r + (2 * u if case["add"] else case["rows"]) * d * w, "flops": t * d + u * d}
    if case["op"] == "step":
        return {k: lookup[k] + grad[k] for k in lookup}
    return lookup if case["op"] == "lookup" else grad
