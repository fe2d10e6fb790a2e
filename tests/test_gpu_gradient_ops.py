"""The gradient norm, clipping and the embedding on the GPU, against plain computations in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of fp32, `half(t)` half a step of t.
- norm: a load's squares are added in two chains of at most 8 fused steps and one addition, all terms positive, then in
  double: at most 9 u of the sum, 4.5 u of its root, and half a step for the result.
- clipping: the coefficient has the norm's error and one rounding, the product one, the result one: 6.5 u + half(t), and
  half of the smallest step of t where it is subnormal.
- lookup: the product is rounded to fp32, then to the result's type: u + half(t).
- gradient: m rows added one by one or in parts, a scale and an addition to the table: at most (m + 2) u of the sum of
  magnitudes, u of the old value, and half a step of the result."""
import ctypes as C
import math
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import allreduce_proto_b200 as ar

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent
U = 2.0 ** -24
F32, F64, F16, BF16 = torch.float32, torch.float64, torch.float16, torch.bfloat16


def half(t):
    return torch.finfo(t).eps / 2


def least(t):
    return torch.finfo(t).tiny * half(t)


def values(shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.empty(shape, device="cuda", dtype=F64).normal_(0, std, generator=g).to(dtype)


def whole(ts):
    return torch.cat([t.double().flatten() for t in ts])


def norm_of(ts, power):
    x = whole(ts)
    return x.norm() if power == 2 else x.abs().max()


def norm_rtol(dtype):
    return 1e-12 if dtype == F64 else 5.5 * U


def within(got, want, bound):
    """Where `want` is a number `got` is at most `bound` off; elsewhere both are the same."""
    got, want = got.double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    rest = ~fine & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest])
    bound = torch.as_tensor(bound, device=got.device, dtype=F64).expand_as(got)
    off = ((got - want).abs() - bound)[fine]
    assert off.numel() == 0 or off.max() <= 0, (off.max().item(), int((off > 0).sum()))


# Around a load (8 to 16 values), a thread's row of loads, a chunk (2048 to 8192 values) and several; nothing.
SIZES = [(1,), (0,), (7,), (31, 33), (2047,), (2048,), (4097,), (8192,), (3, 5, 1111), (300001,)]


@pytest.mark.parametrize("power", [2.0, math.inf])
@pytest.mark.parametrize("offset", [0, 1, 5])
@pytest.mark.parametrize("dtype", [F32, F64, F16, BF16])
def test_norm_of_lists(dtype, offset, power):
    ts = [values(offset + math.prod(s), dtype, i)[offset:].view(s) for i, s in enumerate(SIZES)]
    for chosen in (ts, ts[:1], ts[1:2], ts[-1:], ts[2:5]):
        norm = ar.ops.grad_norm(chosen, norm_type=power)
        assert norm.dtype == (F64 if dtype == F64 else F32) and norm.shape == ()
        want = norm_of(chosen, power) if whole(chosen).numel() else torch.zeros((), device="cuda", dtype=F64)
        within(norm, want, norm_rtol(dtype) * want.item())


@pytest.mark.parametrize("power", [2.0, math.inf])
@pytest.mark.parametrize("count", [17, 800, 801, 2500])
def test_norm_and_clipping_of_long_mixed_lists(count, power):
    # More tensors than a kernel's parameters hold.
    ts = [values((1 + 37 * i % 301,), (F32, BF16, F16)[i % 3], i) for i in range(count)]
    want = norm_of(ts, power)
    within(ar.ops.grad_norm(ts, norm_type=power), want, norm_rtol(F32) * want.item())
    c = 0.7 / (want.item() + 1e-6)
    before = [t.double() for t in ts]
    within(ar.ops.clip_grad_norm(ts, 0.7, norm_type=power), want, norm_rtol(F32) * want.item())
    for kind in (F32, BF16, F16):
        b = torch.cat([x for x, t in zip(before, ts) if t.dtype == kind]) * c
        within(torch.cat([t for t in ts if t.dtype == kind]), b, (6.5 * U + half(kind)) * b.abs() + least(kind))


def test_one_double_tensor_makes_the_norm_double():
    ts = [values((1000,), F32, 1), values((1000,), F64, 2), values((1000,), BF16, 3)]
    norm = ar.ops.grad_norm(ts)
    assert norm.dtype == F64
    within(norm, norm_of(ts, 2), 4.5 * U * norm.item())


@pytest.mark.parametrize("dtype,value", [(F32, 1e30), (F32, 3e38), (F32, 1e-30), (F32, 1e-44), (BF16, 1e38), (BF16, 1e-38), (F16, 65504.0),
                                         (F16, 6e-8), (F64, 1e-150), (F32, 0.0), (BF16, 0.0)])
def test_norms_beyond_the_range_of_fp32_squares(dtype, value):
    # The root of 5 times the value may pass fp32's range: then the norm is infinite, and nothing else is.
    x = torch.full((5,), value, device="cuda", dtype=dtype)
    want = whole([x]).norm()
    want = want if dtype == F64 else want.float()
    within(ar.ops.grad_norm([x]), want, norm_rtol(dtype) * want.item() + least(F32) if torch.isfinite(want) else 0.0)
    # Such a value among ordinary ones, in every place of a load.
    for place in (0, 7, 8, 15, 4000):
        y = values((5000,), dtype, place)
        y[place] = value
        want = norm_of([y], 2)
        within(ar.ops.grad_norm([y]), want, norm_rtol(dtype) * want.item())
        want = norm_of([y], math.inf)
        within(ar.ops.grad_norm([y], norm_type=math.inf), want, U * want.item())


@pytest.mark.parametrize("power", [2.0, math.inf])
@pytest.mark.parametrize("dtype", [F32, F64, F16, BF16])
def test_norms_that_are_not_finite(dtype, power):
    for place in (0, 9, 4999):
        for bad in (math.inf, -math.inf, math.nan, -math.nan):
            x = values((5000,), dtype, 3)
            x[place] = bad
            y = values((100,), dtype, 4)
            norm = ar.ops.grad_norm([x, y], norm_type=power)
            assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
            ar.ops.clip_grad_norm([x, y], 1.0, norm_type=power)
            if math.isnan(bad):
                assert torch.isnan(x).all() and torch.isnan(y).all()
            else:
                assert torch.isnan(x[place]) and int(torch.isnan(x).sum()) == 1
                assert not y.any() and not x[torch.arange(5000, device="cuda") != place].any()
            x[place], x[(place + 17) % 5000] = math.nan, math.inf
            assert math.isnan(ar.ops.grad_norm([y, x], norm_type=power))


PAIRS = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F64, F64)]


@pytest.mark.parametrize("offsets", [(0, 0), (1, 1), (3, 3), (1, 0), (0, 1), (8, 4)])
@pytest.mark.parametrize("types", PAIRS)
def test_clipping_into_other_tensors(types, offsets):
    a, b = types
    xs = [values(offsets[0] + math.prod(s), a, i)[offsets[0]:].view(s) for i, s in enumerate(SIZES)]
    guards = [torch.full((offsets[1] + math.prod(s) + 9,), 7.0, device="cuda", dtype=b) for s in SIZES]
    outs = [g[offsets[1]:offsets[1] + math.prod(s)].view(s) for g, s in zip(guards, SIZES)]
    before = [x.clone() for x in xs]
    want = norm_of(xs, 2)
    for bound in (1.5, 1e9, 0.0, math.inf):
        within(ar.ops.clip_grad_norm(xs, bound, out=outs), want, norm_rtol(a) * want.item())
        c = min(1.0, bound / (want.item() + 1e-6))
        step = norm_rtol(a) + 2 * half(a) if a == F64 else 6.5 * U
        for x, x0, o in zip(xs, before, outs):
            assert torch.equal(x, x0)
            if c == 1.0:
                assert torch.equal(o, x.to(b))
            else:
                w = x.double() * c
                within(o, w, (step + half(b)) * w.abs() + least(b))
        for g, s in zip(guards, SIZES):
            assert torch.all(g[:offsets[1]] == 7) and torch.all(g[offsets[1] + math.prod(s):] == 7)


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("dtype", [F32, F64, F16, BF16])
def test_clipping_in_place(dtype, offset):
    guards = [torch.full((offset + math.prod(s) + 9,), 7.0, device="cuda", dtype=dtype) for s in SIZES]
    xs = [g[offset:offset + math.prod(s)].view(s) for g, s in zip(guards, SIZES)]
    for i, x in enumerate(xs):
        x.copy_(values(tuple(x.shape), dtype, i))
    before = [x.clone() for x in xs]
    ar.ops.clip_grad_norm(xs, 1e9)
    assert all(torch.equal(x, b) for x, b in zip(xs, before))
    outs = [torch.empty_like(x) for x in xs]
    ar.ops.clip_grad_norm(xs, 2.0, out=outs)
    ar.ops.clip_grad_norm(xs, 2.0)
    assert all(torch.equal(x, o) for x, o in zip(xs, outs))
    for g, s in zip(guards, SIZES):
        assert torch.all(g[:offset] == 7) and torch.all(g[offset + math.prod(s):] == 7)


def test_dense_tensors_of_any_order():
    x = values((4, 6, 8, 10), F32, 1).contiguous(memory_format=torch.channels_last)
    y = values((50, 70), F32, 2).t()
    b = [x.clone(), y.clone()]
    within(ar.ops.grad_norm([x, y]), norm_of([x, y], 2), 5.5 * U * norm_of([x, y], 2).item())
    want = norm_of([x, y], 2).item()
    out = [torch.empty_like(x), torch.empty_like(y)]
    ar.ops.clip_grad_norm([x, y], 1.0, out=out)
    ar.ops.clip_grad_norm([x, y], 1.0)
    for t, o, t0 in zip([x, y], out, b):
        assert torch.equal(t, o)
        within(t, t0.double() / (want + 1e-6), 7.5 * U * t0.double().abs() / want)


def test_norm_is_the_same_whatever_runs_beside_it():
    xs = [values((n,), BF16, n) for n in (5000001, 333, 70000)]
    first = ar.ops.grad_norm(xs)
    side = torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(side):
            torch.randn(1 << 22, device="cuda").sin()
        assert torch.equal(ar.ops.grad_norm(xs), first)


def test_two_streams_and_two_graphs_at_once():
    # Every call has a workspace of its own: two that run at the same time do not disturb one another.
    sets = [[values((n,), F32, k * 10 + i) for i, n in enumerate((3000001, 77, 65536))] for k in range(2)]
    outs = [[torch.empty_like(x) for x in xs] for xs in sets]
    wants = [norm_of(xs, 2).item() for xs in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    norms = [[], []]
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                norms[k].append(ar.ops.clip_grad_norm(sets[k], 1.0, out=outs[k]))
    torch.cuda.synchronize()
    graphs, kept = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kept.append(ar.ops.clip_grad_norm(sets[k], 1.0, out=outs[k]))
        graphs.append(g)
    for xs in sets:
        for x in xs:
            x.mul_(2)
    torch.cuda.synchronize()
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
    torch.cuda.synchronize()
    for k in range(2):
        assert all(abs(n.item() - wants[k]) <= 5.5 * U * wants[k] for n in norms[k])
        assert abs(kept[k].item() - 2 * wants[k]) <= 11 * U * wants[k]
        for x, o in zip(sets[k], outs[k]):
            w = x.double() / (2 * wants[k] + 1e-6)
            within(o, w, 7.5 * U * w.abs())


@pytest.mark.parametrize("n", [700, 300000, 40000000])
@pytest.mark.parametrize("power", [2.0, math.inf])
def test_lists_of_every_size_in_a_graph(n, power):
    # One cluster, the kernel that holds what it read, and the two kernels of long lists.
    xs = [values((n,), F32, 1), values((n // 3,), BF16, 2)]
    outs = [torch.empty_like(x) for x in xs]
    ar.ops.clip_grad_norm(xs, 1.0, out=outs, norm_type=power)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ar.ops.grad_norm(xs, norm_type=power)
        clipped = ar.ops.clip_grad_norm(xs, 1.0, out=outs, norm_type=power)
        after = ar.ops.clip_grad_norm(outs, 0.5, norm_type=power)
    for x in xs:
        x.mul_(3)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    want = norm_of(xs, power).item()
    within(norm, torch.tensor(want, device="cuda"), norm_rtol(F32) * want)
    within(clipped, norm, 2 * norm_rtol(F32) * want)
    # The second clipping sees the first one's values, rounded to bf16 here and there.
    within(after, torch.ones((), device="cuda"), half(BF16) + 8 * U)
    for x, o in zip(xs, outs):
        w = x.double() * (0.5 / (want + 1e-6))
        within(o, w, (3 * half(BF16) + 20 * U) * w.abs() + 2 * least(x.dtype))


class TwoRanks:
    """What a communicator of two ranks does for the norm, seen from the first; `other` is the second's sum."""
    world_size, rank = 2, 0

    def __init__(self, other):
        self.other = other

    def all_gather(self, send, recv):
        recv[0:1].copy_(send)
        recv[1] = self.other


@pytest.mark.parametrize("power", [2.0, math.inf])
def test_norm_of_shards(power):
    xs, rest = [values((70001,), F32, 1), values((9,), BF16, 2)], values((5000,), F32, 3) * 3
    comm = TwoRanks(rest.double().square().sum() if power == 2 else rest.double().abs().max())
    want = norm_of(xs + [rest], power)
    within(ar.ops.grad_norm(xs, norm_type=power, comm=comm), want, 5.5 * U * want.item())
    before = [x.double() for x in xs]
    within(ar.ops.clip_grad_norm(xs, 0.25, norm_type=power, comm=comm), want, 5.5 * U * want.item())
    for x, b in zip(xs, before):
        w = b * (0.25 / (want.item() + 1e-6))
        within(x, w, (6.5 * U + half(x.dtype)) * w.abs() + least(x.dtype))
    # A rank whose part has no elements.
    within(ar.ops.grad_norm([torch.empty(0, device="cuda")], norm_type=power, comm=comm), norm_of([rest], power), 5.5 * U * want.item())


def test_gradient_buckets():
    shapes = [(300, 7), (5,), (640, 64), (1,)]
    for dtype in (F32, BF16):
        buckets = ar.GradientBuckets(shapes, dtype=dtype, bucket_bytes=8192, shardable=True)
        grads = [values(s, dtype, i) for i, s in enumerate(shapes)]
        buckets.load(grads)
        want = norm_of(grads, 2)
        within(buckets.grad_norm(), want, 5.5 * U * want.item())
        assert torch.equal(buckets.grad_norm(sharded=True), buckets.grad_norm())
        within(buckets.clip_grad_norm(0.5), want, 5.5 * U * want.item())
        for v, g in zip(buckets.views, grads):
            w = g.double() * (0.5 / (want.item() + 1e-6))
            within(v, w, (6.5 * U + half(dtype)) * w.abs())
        within(buckets.grad_norm(norm_type=math.inf), norm_of(buckets.views, math.inf), 0.0)


# ---------------------------------------------------------------- embedding
def tokens_of(n, rows, seed, dtype=torch.int64, shape=None):
    """Skewed towards the first rows, some outside of the table on both sides."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    u = torch.rand(n, device="cuda", generator=g, dtype=F64)
    t = (torch.exp(u * math.log(rows + 1)) - 1).long().clamp_(0, max(rows - 1, 0))
    pick = torch.randint(0, 16, (n,), device="cuda", generator=g)
    t = torch.where(pick == 0, -1, torch.where(pick == 1, rows, t))
    return t.to(dtype).view(shape or (n,))


def lookup_in_64_bits(tokens, weight, scale):
    inside = (tokens >= 0) & (tokens < weight.shape[0])
    rows = torch.zeros(*tokens.shape, weight.shape[1], device="cuda", dtype=F64)
    rows[inside] = weight.double()[tokens[inside].long()] * scale
    return rows


def grad_in_64_bits(tokens, grad, rows, scale, padding=None):
    """The gradient, and the bound of its error from the additions."""
    t, g = tokens.flatten().long(), grad.double().reshape(tokens.numel(), -1)
    keep = (t >= 0) & (t < rows)
    if padding is not None:
        keep &= t != padding
    t, g = t[keep], g[keep] * scale
    total = torch.zeros(rows, g.shape[1], device="cuda", dtype=F64).index_add_(0, t, g)
    size = torch.zeros(rows, g.shape[1], device="cuda", dtype=F64).index_add_(0, t, g.abs())
    count = torch.bincount(t, minlength=rows).double()[:, None]
    return total, (count + 2) * U * size


TYPES = [(F32, F32), (F32, BF16), (F32, F16), (BF16, F32), (BF16, BF16), (BF16, F16), (F16, F32), (F16, BF16), (F16, F16)]


@pytest.mark.parametrize("table,rows_type", TYPES)
@pytest.mark.parametrize("width", [1, 4, 8, 17, 64, 100, 1000, 2056])
def test_lookup(width, table, rows_type):
    for n, rows, offset in ((1, 1, 0), (5, 3, 1), (1000, 77, 0), (333, 5000, 4), (257, 100, 8)):
        w = values(offset + rows * width, table, width)[offset:].view(rows, width)
        for ids in (torch.int64, torch.int32):
            t = tokens_of(n, rows, n, ids)
            got = ar.ops.embedding(t, w, scale=1.5, out_dtype=rows_type)
            want = lookup_in_64_bits(t, w, 1.5)
            assert got.dtype == rows_type and got.shape == (n, width)
            within(got, want, (U + half(rows_type)) * want.abs() + least(rows_type))


def test_lookup_of_tokens_of_any_shape():
    w = values((50, 24), BF16, 1)
    for t in (tokens_of(24, 50, 1, shape=(2, 3, 4)), tokens_of(40, 50, 2, shape=(4, 10))[:, :-1], tokens_of(12, 50, 3, shape=(3, 4)).t(),
              torch.tensor(7, device="cuda"), tokens_of(1, 50, 4).expand(6), torch.empty(0, 3, dtype=torch.int64, device="cuda")):
        got = ar.ops.embedding(t, w)
        assert got.shape == (*t.shape, 24)
        assert torch.equal(got, lookup_in_64_bits(t, w, 1.0).to(BF16))
    # A table without rows, and one without columns.
    assert not ar.ops.embedding(torch.tensor([0, 3], device="cuda"), torch.empty(0, 8, device="cuda")).any()
    assert ar.ops.embedding(torch.tensor([0, 3], device="cuda"), torch.empty(4, 0, device="cuda")).shape == (2, 0)
    # Values that are not finite stay in their rows.
    w[3], w[4] = math.nan, math.inf
    got = ar.ops.embedding(torch.tensor([2, 3, 4, -1], device="cuda"), w)
    assert torch.isfinite(got[[0, 3]]).all() and torch.isnan(got[1]).all() and (got[2] == math.inf).all()


# Around a chunk of tokens, a sort's block, and several blocks; rows from one to more than one digit of the sort.
@pytest.mark.parametrize("n,rows", [(1, 1), (2, 1), (31, 3), (32, 1000), (33, 2), (64, 64), (100, 5000), (200, 1), (255, 3), (256, 40), (257, 1), (500, 1), (1000, 1023), (1000, 1024),
                                    (2047, 100), (2049, 200000), (5000, 7), (20000, 300), (70000, 1 << 20)])
@pytest.mark.parametrize("table,rows_type", [(F32, BF16), (F32, F32), (BF16, BF16), (F16, F32)])
def test_gradient_of_the_table(table, rows_type, n, rows):
    width = 8 if rows > 100000 else 136
    t = tokens_of(n, rows, n + rows)
    g = values((n, width), rows_type, n)
    want, bound = grad_in_64_bits(t, g, rows, 0.25)
    got = ar.ops.embedding_grad(t, g, num_rows=rows, dtype=table, scale=0.25)
    assert got.dtype == table and got.shape == (rows, width)
    within(got, want, bound + half(table) * want.abs() + least(table))
    # Added to what a bucket holds: rows that no token names keep their bits, whatever they are.
    old = values((rows, width), table, 5)
    named = torch.zeros(rows, dtype=torch.bool, device="cuda")
    inside = (t >= 0) & (t < rows)
    named[t[inside]] = True
    old[~named] = math.nan
    into = old.clone()
    assert ar.ops.embedding_grad(t, g, out=into, accumulate=True, scale=0.25) is into
    assert torch.equal(into[~named].view(torch.int16), old[~named].view(torch.int16))
    want, bound = (want + old.double())[named], bound[named]
    within(into[named], want, bound + (U * (old[named].double().abs() + want.abs()) + half(table) * want.abs()) + least(table))


@pytest.mark.parametrize("n,width", [(200003, 264), (700001, 264), (300001, 33)])
@pytest.mark.parametrize("table,rows_type", [(F32, BF16), (F32, F32), (BF16, BF16)])
def test_gradient_of_few_rows(table, rows_type, n, width):
    # Long runs: a warp's part of the list is longer than the 32 tokens that its lanes hold.
    rows = 40
    t, g = tokens_of(n, rows, n, torch.int32), values((n, width), rows_type, width)
    want, bound = grad_in_64_bits(t, g, rows, 0.5)
    within(ar.ops.embedding_grad(t, g, num_rows=rows, dtype=table, scale=0.5), want, bound + half(table) * want.abs())
    old = values((rows, width), table, 7)
    into = old.clone()
    ar.ops.embedding_grad(t, g, out=into, accumulate=True, scale=0.5)
    want = want + old.double()
    within(into, want, bound + U * (old.double().abs() + want.abs()) + half(table) * want.abs())


@pytest.mark.parametrize("table,rows_type", TYPES)
@pytest.mark.parametrize("width", [1, 3, 4, 8, 100, 129, 255, 256, 1000, 2056])
def test_gradient_widths_types_and_alignment(width, table, rows_type):
    for n, rows, offsets in ((100, 20, (0, 0)), (700, 30, (1, 0)), (700, 30, (0, 1)), (90, 3, (4, 4)), (700, 300, (8, 2))):
        t = tokens_of(n, rows, n, torch.int32)
        g = values(offsets[0] + n * width, rows_type, n)[offsets[0]:].view(n, width)
        guard = torch.full((offsets[1] + rows * width + 64,), 7.0, device="cuda", dtype=table)
        out = guard[offsets[1]:offsets[1] + rows * width].view(rows, width)
        want, bound = grad_in_64_bits(t, g, rows, 1.0)
        ar.ops.embedding_grad(t, g, out=out)
        within(out, want, bound + half(table) * want.abs() + least(table))
        old = values((rows, width), table, 9)
        out.copy_(old)
        ar.ops.embedding_grad(t, g, out=out, accumulate=True)
        want = want + old.double()
        within(out, want, bound + U * (old.double().abs() + want.abs()) + half(table) * want.abs() + least(table))
        assert torch.all(guard[:offsets[1]] == 7) and torch.all(guard[offsets[1] + rows * width:] == 7)


@pytest.mark.parametrize("n", [1, 40, 300, 9000, 100000, 600000])
def test_all_tokens_the_same_or_none(n):
    g = values((n, 72), F32, n)
    for token, rows in ((0, 1), (6, 9), (8, 9), (-1, 9), (9, 9), (-2 ** 31, 9), (2 ** 31 - 1, 9)):
        t = torch.full((n,), token, device="cuda", dtype=torch.int32)
        want, bound = grad_in_64_bits(t, g, rows, 1.0)
        within(ar.ops.embedding_grad(t, g, num_rows=rows), want, bound + U * want.abs())
    t = torch.full((n,), 2 ** 40 + 3, device="cuda")  # its lower half names a row
    assert not ar.ops.embedding_grad(t, g, num_rows=9).any()
    assert not ar.ops.embedding(t, torch.ones(9, 8, device="cuda")).any()


def test_gradient_without_tokens_rows_or_columns():
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    out = torch.ones(5, 8, device="cuda")
    ar.ops.embedding_grad(none, torch.empty(0, 8, device="cuda"), out=out, accumulate=True)
    assert torch.all(out == 1)
    ar.ops.embedding_grad(none, torch.empty(0, 8, device="cuda"), out=out)
    assert not out.any()
    one = torch.zeros(1, dtype=torch.int64, device="cuda")
    assert ar.ops.embedding_grad(one, torch.ones(1, 8, device="cuda"), num_rows=0).shape == (0, 8)
    assert ar.ops.embedding_grad(one, torch.ones(1, 0, device="cuda"), num_rows=3).shape == (3, 0)


@pytest.mark.parametrize("n", [50, 5000])
def test_padding_and_values_that_are_not_finite(n):
    rows = 40
    t = tokens_of(n, rows, 1)
    t[7], t[11], t[13] = 5, -1, 39
    g = values((n, 64), BF16, 2)
    outside = (t < 0) | (t >= rows) | (t == 5)
    g[outside] = math.nan  # of padded places: they reach no row
    g[13, 3] = math.inf
    got = ar.ops.embedding_grad(t, g, num_rows=rows, dtype=F32, padding_idx=5)
    want, bound = grad_in_64_bits(t, torch.where(torch.isfinite(g), g, 0.0), rows, 1.0, padding=5)
    assert got[39, 3] == math.inf and not got[5].any()
    got[39, 3] = want[39, 3].float()
    within(got, want, bound + U * want.abs())
    # The lookup reads the row all the same.
    assert ar.ops.embedding(torch.tensor([5], device="cuda"), torch.ones(rows, 8, device="cuda"), padding_idx=5).all()


def test_gradient_has_the_same_bits_every_time():
    t, g = tokens_of(30000, 500, 1), values((30000, 200), BF16, 2)
    first = ar.ops.embedding_grad(t, g, num_rows=500, dtype=F32)
    side = torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(side):
            torch.randn(1 << 22, device="cuda").sin()
        assert torch.equal(ar.ops.embedding_grad(t, g, num_rows=500, dtype=F32), first)


@pytest.mark.parametrize("n", [200, 5000, 30000, 40000])
def test_tables_of_many_rows(n):
    # Row numbers of 28 bits: three digits of the sort.
    rows = (1 << 27) + 3
    t = tokens_of(n, rows, n)
    t[:3] = torch.tensor([rows - 1, 0, rows - 1])
    g = torch.arange(1, n + 1, device="cuda", dtype=F32)[:, None] % 64
    out = torch.zeros(rows, 1, device="cuda", dtype=F32)
    ar.ops.embedding_grad(t, g, out=out, accumulate=True)
    inside = (t >= 0) & (t < rows)
    want = torch.zeros(rows, 1, device="cuda", dtype=F32).index_add_(0, t[inside], g[inside])  # whole numbers, exact
    assert torch.equal(out, want)


def test_largest_offsets():
    # More than 2^31 elements in the table and in the rows: a wide table whose last rows are named.
    rows, width = 270000, 8192
    w = torch.zeros(rows, width, device="cuda", dtype=BF16)
    w[-1], w[rows - 2] = 3.0, 2.0
    t = torch.full((270001,), rows - 2, device="cuda", dtype=torch.int32)
    t[-1] = rows - 1
    y = ar.ops.embedding(t, w)
    assert torch.all(y[-1] == 3) and torch.all(y[-2] == 2)
    ar.ops.embedding_grad(t, y, out=w, scale=2.0 ** -10, accumulate=True)
    # 270000 rows of 2 in parts, exact in fp32 up to 2^24.
    assert torch.all(w[rows - 2].double() == torch.tensor(2 + 540000 / 1024, dtype=F64).to(BF16).double())
    assert torch.all(w[-1].double() == torch.tensor(3 + 3 / 1024, dtype=F64).to(BF16).double()) and not w[:rows - 2].any()


@pytest.mark.parametrize("table,rows_type", [(F32, None), (F32, BF16), (BF16, None)])
def test_gradient_through_autograd(table, rows_type):
    rows, width = 60, 40
    w = values((rows, width), table, 1).requires_grad_(True)
    t = tokens_of(300, rows, 2, shape=(20, 15))
    y = ar.ops.embedding(t, w, scale=3.0, padding_idx=4, out_dtype=rows_type)
    dy = values((20, 15, width), y.dtype, 3)
    y.backward(dy)
    want, bound = grad_in_64_bits(t, dy, rows, 3.0, padding=4)
    assert w.grad.dtype == table
    within(w.grad, want, bound + half(table) * want.abs() + least(table))
    # Broadcast gradients, and two uses of one table.
    w.grad = None
    (ar.ops.embedding(t, w).sum() + ar.ops.embedding(t[0], w, scale=2.0).float().sum()).backward()
    one = torch.ones(20, 15, width, device="cuda")
    want = grad_in_64_bits(t, one, rows, 1.0)[0] + grad_in_64_bits(t[0], one[0], rows, 2.0)[0]
    within(w.grad, want, (U * 300 + 3 * half(table)) * want.abs())
    with torch.no_grad():
        assert not ar.ops.embedding(t, w).requires_grad


def test_what_autograd_refuses():
    w = values((20, 8), F32, 1).requires_grad_(True)
    t = tokens_of(30, 20, 2)
    y = ar.ops.embedding(t, w)
    dy = torch.ones_like(y).requires_grad_(True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(y, w, dy, create_graph=True, retain_graph=True)
    (g,) = torch.autograd.grad(y, w, dy, retain_graph=True)
    assert torch.equal(torch.autograd.grad(y, w, dy)[0], g)
    with pytest.raises(RuntimeError, match="retain_graph"):
        torch.autograd.grad(y, w, dy)
    y = ar.ops.embedding(t, w)
    t.zero_()  # what the backward pass needs has changed
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = ar.ops.embedding(t, w, grad_into=torch.zeros(20, 8, device="cuda", dtype=F16))
    y.sum().backward()
    assert w.grad is None
    # No tokens at all, and a table that is no leaf.
    ar.ops.embedding(t[:0], w).sum().backward()
    assert w.grad.shape == w.shape and not w.grad.any()
    half_table = w.detach().requires_grad_(True)
    ar.ops.embedding(t, half_table * 2).sum().backward()
    assert torch.equal(half_table.grad, 2 * grad_in_64_bits(t, torch.ones(30, 8, device="cuda"), 20, 1.0)[0].float())


def test_gradient_against_differences():
    # f is a polynomial of second degree in the weights: central differences have no error but rounding.
    rows, width = 7, 8
    w = values((rows, width), F32, 1).requires_grad_(True)
    t = tokens_of(50, rows, 2)
    a = values((50, width), F32, 3)
    f = lambda x: (ar.ops.embedding(t, x, scale=0.5).double().square() * a.double()).sum()  # noqa: E731
    f(w).backward()
    h = 2.0 ** -3
    size = (lookup_in_64_bits(t, w.detach(), 0.5).abs() + h).square().mul(a.double().abs()).sum().item()
    for v, d in ((0, 0), (1, 5), (6, 7)):
        e = torch.zeros(rows, width, device="cuda")
        e[v, d] = h
        diff = (f(w.detach() + e) - f(w.detach() - e)).item() / (2 * h)
        # Two roundings (the shifted weight, the product) in each factor of both sides' squares; 53 additions in the gradient.
        assert abs(diff - w.grad[v, d].item()) <= (8 / h + 60) * U * size


def test_gradient_into_a_bucket():
    shapes = [(50, 24), (24,)]
    buckets = ar.GradientBuckets(shapes, bucket_bytes=1 << 20)
    w = torch.nn.Parameter(values((50, 24), BF16, 1).float())
    b = torch.nn.Parameter(values((24,), F32, 2))
    t = tokens_of(500, 50, 3)
    dy = values((500, 24), BF16, 4)
    buckets.attach([w, b])
    for _ in range(2):  # gradients add up until zero_()
        (buckets.embedding(0, t, w, scale=2.0, out_dtype=BF16).float() + b).backward(dy.float())
    want, bound = grad_in_64_bits(t, dy, 50, 2.0)
    within(buckets.views[0], 2 * want, 2 * bound + 3 * U * want.abs())
    assert w.grad is buckets.views[0] or w.grad.data_ptr() == buckets.views[0].data_ptr()
    within(b.grad, 2 * dy.double().sum(0), 500 * 2 * U * dy.double().abs().sum(0))


@pytest.mark.parametrize("tied", [False, True])
def test_bucket_with_overlapped_allreduce(tied):
    # With another use of the table the bucket's hook runs after both gradients are in place.
    comm = ar.Communicator(1, 0)
    w = torch.nn.Parameter(values((64, 32), F32, 1))
    head = w if tied else torch.nn.Parameter(values((64, 32), F32, 2))
    params = [w] if tied else [w, head]
    t, y = tokens_of(200, 64, 3).clamp(0, 63), values((200, 64), F32, 4)
    plain = [p.detach().double().requires_grad_(True) for p in params]
    ((torch.nn.functional.embedding(t, plain[0]) * 2) @ plain[-1].t()).backward(y.double())
    buckets = ar.GradientBuckets([p.shape for p in params], comm=comm, bucket_bytes=64 * 32 * 4)
    buckets.overlap_with_backward(params)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for step in range(3):
        buckets.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # the lookup's stream is that of its gradient
            x = buckets.embedding(0, t, w, scale=2.0)
        x.register_hook(lambda g: torch.cuda._sleep(20_000_000))  # some 10 ms ahead of the table's gradient, on its stream
        torch.cuda.current_stream().wait_stream(side)
        (x.double() @ head.double().t()).backward(y.double())
        buckets.finish()
        for v, p in zip(buckets.views, plain):
            # 200 rows at most in a sum, and the roundings of the parts to fp32.
            size = p.grad.abs().max().item() + 200.0
            within(v, p.grad, 204 * U * size)
    buckets.remove_hooks()


def test_step_in_a_graph():
    rows, width = 200, 64
    w = values((rows, width), F32, 1).requires_grad_(True)
    t, dy = tokens_of(3000, rows, 2), values((3000, width), BF16, 3)
    into = torch.zeros(rows, width, device="cuda")

    def step():
        y = ar.ops.embedding(t, w, scale=2.0, out_dtype=BF16)
        (g,) = torch.autograd.grad(y, w, dy)
        ar.ops.embedding_grad(t, dy, out=into)
        return y.detach(), g, ar.ops.clip_grad_norm([into], 1.0)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    t.copy_(tokens_of(3000, rows, 20))
    dy.copy_(values((3000, width), BF16, 30))
    with torch.no_grad():
        w.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    want = step()
    for a, b in zip(kept, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_bucket_step_in_a_graph(dtype):
    # Lookup, backward pass into the bucket, allreduce, clipping: nothing of it is read back.
    buckets = ar.GradientBuckets([(50, 24), (24,)], dtype=dtype, comm=ar.Communicator(1, 0))
    w, h = torch.nn.Parameter(values((50, 24), dtype, 1)), torch.nn.Parameter(values((24,), dtype, 2))
    buckets.attach([w, h])
    t = tokens_of(500, 50, 3)

    def step():
        buckets.zero_()
        (buckets.embedding(0, t, w, scale=0.25) * h).sum().backward()
        buckets.allreduce()
        return buckets.clip_grad_norm(1.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = step()
    t.copy_(tokens_of(500, 50, 4))
    graph.replay()
    torch.cuda.synchronize()
    got = [norm.clone(), buckets.flat[0].clone()]
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want) and torch.equal(got[1], buckets.flat[0])
    inside = ((t >= 0) & (t < 50)).sum().item()
    assert 0 < inside < 500 and torch.isfinite(want)


IN_GRAPH = """
import torch
import allreduce_proto_b200 as ar
w = torch.randn(50, 16, device="cuda", requires_grad=True)
t = torch.randint(0, 50, (64,), device="cuda")
into = torch.zeros(50, 16, device="cuda")
alive = ar.ops.embedding(t, w, **KIND)   # an eager graph of the same leaf
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
graph = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(graph, stream=side):
        ar.ops.embedding(t, w, **KIND).sum().backward()
    graph.replay()
except (RuntimeError, ar.IbcommError) as e:
    print("refused", str(e)[:200])
torch.cuda.synchronize()
print("alive", into.sum().item() if KIND else w.grad.sum().item() if w.grad is not None else None)
"""


@pytest.mark.parametrize("kind", ["{}", "{'grad_into': into}"])
def test_backward_in_a_graph_beside_an_eager_graph_of_the_leaf(kind):
    p = subprocess.run([sys.executable, "-c", IN_GRAPH.replace("KIND", kind)], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=300)
    assert p.returncode == 0 and "alive" in p.stdout, (p.returncode, p.stdout, p.stderr[-2000:])


@pytest.mark.parametrize("ranks", [2, 3])
def test_a_step_of_several_ranks(ranks):
    # Lookup, gradient into buckets, mean over the ranks, clipping: and the same from the ranks' gathered rows.
    rows, width, n = 97, 40, 300
    world = ar.EmuWorld(ranks)
    w = values((rows, width), F32, 1)
    ts = [tokens_of(n, rows, 10 + r, torch.int32) for r in range(ranks)]
    dys = [values((n, width), F32, 20 + r) for r in range(ranks)]
    buckets = [ar.GradientBuckets([(rows, width), (width,)]) for _ in range(ranks)]
    bias = [values((width,), F32, 30 + r) for r in range(ranks)]
    for r in range(ranks):
        p = w.clone().requires_grad_(True)
        buckets[r].views[1].copy_(bias[r])
        buckets[r].embedding(0, ts[r], p, scale=2.0).backward(dys[r])
        assert p.grad is None
    world.allreduce([b.flat[0] for b in buckets], scale=1.0 / ranks)
    want, bound = grad_in_64_bits(torch.cat(ts), torch.cat(dys), rows, 2.0 / ranks)
    mean = sum(b.double() for b in bias) / ranks
    norm = torch.cat([want.flatten(), mean]).norm()
    bound = bound + 4 * U * torch.zeros_like(want).index_add_(0, torch.cat(ts).clamp(0, rows - 1).long(), torch.cat(dys).double().abs() * 2)
    c = 0.5 / (norm.item() + 1e-6)
    norms = [b.clip_grad_norm(0.5) for b in buckets]
    off = bound.norm().item() + 8 * U * norm.item()
    for b, got in zip(buckets, norms):
        assert torch.equal(got, norms[0]) and abs(got.item() - norm.item()) <= off
        within(b.views[0], want * c, bound * c + (off / norm.item() + 8 * U) * (want * c).abs())
    gathered = [torch.empty(ranks * n, dtype=torch.int32, device="cuda") for _ in range(ranks)]
    summed = [torch.empty(ranks * n * width, device="cuda") for _ in range(ranks)]
    world.all_gather(ts, gathered)
    world.all_gather([d.flatten() for d in dys], summed)
    for r in range(ranks):
        got = ar.ops.embedding_grad(gathered[r], summed[r].view(-1, width), num_rows=rows, scale=2.0 / ranks)
        within(got, want, bound + U * want.abs())


def test_what_is_refused_on_the_gpu():
    x, t = torch.ones(64, device="cuda"), torch.zeros(8, dtype=torch.int64, device="cuda")
    w = torch.ones(4, 8, device="cuda")

    def code_of(call):
        with pytest.raises(ar.IbcommError) as e:
            call()
        return e.value.code

    clip, norm = ar.ops.clip_grad_norm, ar.ops.grad_norm
    assert code_of(lambda: norm([x[::2]])) == ar.INVALID_ARGUMENT
    assert code_of(lambda: norm([x.int()])) == ar.NOT_SUPPORTED
    assert code_of(lambda: norm([x, x.cpu()])) == ar.INVALID_ARGUMENT
    assert code_of(lambda: norm([x.cpu(), x])) == ar.INVALID_ARGUMENT
    assert code_of(lambda: clip([x, x], 1.0)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: clip([x[:40], x[39:]], 1.0)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: clip([x[:32]], 1.0, out=[x[1:33]])) == ar.INVALID_ARGUMENT
    assert code_of(lambda: clip([x], 1.0, out=[x.double()])) == ar.NOT_SUPPORTED
    assert code_of(lambda: clip([x], 1.0, out=[x.view(8, 8)])) == ar.INVALID_ARGUMENT
    assert code_of(lambda: clip([x], -1.0)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding(t.cpu(), w)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding(t, w.double())) == ar.NOT_SUPPORTED
    assert code_of(lambda: ar.ops.embedding(t, w.t())) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding(t, w[0])) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding(t, w, scale=math.nan)) == ar.INVALID_ARGUMENT
    g = torch.ones(8, 8, device="cuda")
    assert code_of(lambda: ar.ops.embedding_grad(t, g, out=g)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding_grad(t, g[:7], out=w)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding_grad(t, g[:, :7], out=w)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding_grad(t, g, out=w.double())) == ar.NOT_SUPPORTED
    assert code_of(lambda: ar.ops.embedding_grad(t, g, out=torch.ones(8, 4, device="cuda").t())) == ar.INVALID_ARGUMENT
    torch.cuda.synchronize()
    assert torch.all(x == 1) and torch.all(w == 1)


@pytest.mark.parametrize("sharded", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_buckets_recover_from_a_step_that_is_not_a_number(dtype, sharded):
    # Every tensor leaves places up to the next 16 bytes, which only zero_() writes.
    shapes = [(5,), (7,), (3, 33)]
    buckets = ar.GradientBuckets(shapes, dtype=dtype, shardable=True)
    grads = [values(s, dtype, i) for i, s in enumerate(shapes)]
    buckets.load([torch.full_like(grads[0], math.nan)] + grads[1:])
    assert math.isnan(buckets.clip_grad_norm(1.0, sharded=sharded)) and torch.isnan(buckets.views[2]).all()
    buckets.load(grads)
    want = norm_of(grads, 2)
    within(buckets.grad_norm(), want, 5.5 * U * want.item())
    within(buckets.clip_grad_norm(0.5, sharded=sharded), want, 5.5 * U * want.item())
    for v, g in zip(buckets.views, grads):
        w = g.double() * (0.5 / (want.item() + 1e-6))
        within(v, w, (6.5 * U + half(dtype)) * w.abs())


@pytest.mark.parametrize("n", [20000, 40000])
def test_two_threads_with_tables_of_different_sizes(n):
    # The sorts of both tables are the same kernel (one cluster; cooperative), with digits of 8 and of 10 bits.
    wants, failures = [], []
    for rows in (200, 1000):
        t, g = tokens_of(n, rows, rows), values((n, 8), F32, rows)
        wants.append((t, g, rows, ar.ops.embedding_grad(t, g, num_rows=rows)))
    torch.cuda.synchronize()

    def loop(t, g, rows, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(500):
                    got = ar.ops.embedding_grad(t, g, num_rows=rows)
                assert torch.equal(got, want)
        except Exception as e:  # of another thread: pytest does not see it
            failures.append(repr(e))

    threads = [threading.Thread(target=loop, args=w) for w in wants for _ in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failures, failures


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("table", [F32, BF16])
@pytest.mark.parametrize("n", [200, 30000, 40000])
def test_gradients_of_every_sort_in_a_graph(n, table, accumulate):
    # One launch; the sort in a cluster; the cooperative sort: with what is launched early behind them.
    rows, width = 3001, 40
    t, g, out = tokens_of(n, rows, 1), values((n, width), BF16, 2), values((rows, width), table, 3)
    old = out.clone()
    ar.ops.embedding_grad(t, g, out=out, accumulate=accumulate)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ar.ops.embedding_grad(t, g, out=out, accumulate=accumulate)
    t.copy_(tokens_of(n, rows, 10))
    g.copy_(values((n, width), BF16, 20))
    want = old.clone()
    ar.ops.embedding_grad(t, g, out=want, accumulate=accumulate)
    for _ in range(3):
        out.copy_(old)
        graph.replay()
        assert torch.equal(out, want)
    assert not torch.equal(want, old)


class MeanOfTwo:
    """A communicator whose second rank has no gradients: the mean of a bucket is half of what it holds when the
    collective runs, on the stream that it is given."""
    world_size, rank = 2, 0

    def __init__(self):
        self.calls = []

    def allreduce(self, buf, *, scale, stream, algo, wire):
        self.calls.append(buf.data_ptr())
        with torch.cuda.stream(stream):
            buf.mul_(scale)


@pytest.mark.parametrize("tied", [False, True])
def test_overlapped_mean_sees_the_whole_gradient_of_the_table(tied):
    # The table's gradient comes some 10 ms late, on a stream of its own.  What is added behind the collective is not halved,
    # what the collective finds missing is lost to the sum only until then: either is off by half of a gradient.
    w = torch.nn.Parameter(values((64, 32), F32, 1))
    head = w if tied else torch.nn.Parameter(values((64, 32), F32, 2))
    params = [w] if tied else [w, head]
    t, y = tokens_of(200, 64, 3).clamp(0, 63), values((200, 64), F32, 4)
    plain = [p.detach().double().requires_grad_(True) for p in params]
    ((torch.nn.functional.embedding(t, plain[0]) * 2) @ plain[-1].t()).backward(y.double())
    comm = MeanOfTwo()
    buckets = ar.GradientBuckets([p.shape for p in params], comm=comm, symmetric=False, bucket_bytes=64 * 32 * 4)
    buckets.overlap_with_backward(params)
    side = torch.cuda.Stream()
    for step in range(1, 4):
        buckets.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            x = buckets.embedding(0, t, w, scale=2.0)
        x.register_hook(lambda g: torch.cuda._sleep(20_000_000))
        torch.cuda.current_stream().wait_stream(side)
        (x.double() @ head.double().t()).backward(y.double())
        buckets.finish()
        assert comm.calls == [b.data_ptr() for b in reversed(buckets.flat)] * step
        for v, p in zip(buckets.views, plain):
            # 200 rows at most in a sum, and the roundings of the parts to fp32; halving is exact.
            within(2 * v.double(), p.grad, 204 * U * (p.grad.abs().max().item() + 200.0))
    buckets.remove_hooks()


GRAPH_BESIDE_GRAPH = """
import torch
import allreduce_proto_b200 as ar
w = torch.randn(50, 16, device="cuda", requires_grad=True)
t = torch.randint(0, 50, (64,), device="cuda")
into = torch.zeros(50, 16, device="cuda")
if ATTACHED:
    w.grad = into   # as in a bucket
want = torch.bincount(t, minlength=50)[:, None].expand(50, 16).float()   # of the sum of all rows, exact
alive = ar.ops.embedding(t, w, **KIND)   # an eager graph of the same leaf, on the default stream
side = torch.cuda.Stream()

def attempt():
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            ar.ops.embedding(t, w, **KIND).sum().backward()
    except (RuntimeError, ar.IbcommError) as e:
        assert "captur" in str(e), e
        torch.cuda.synchronize()
        assert w.grad is (into if ATTACHED else None) and not into.any()   # nothing has run
        return "refused"
    assert not into.any()
    graph.replay()
    torch.cuda.synchronize()
    got = into if KIND else w.grad
    assert torch.equal(got, want), got
    return "right"

first = attempt()
if first == "refused":
    alive.sum().backward()   # the eager graph is whole
    got = into if KIND else w.grad
    assert torch.equal(got, want), got
    del got, alive
    into.zero_()
    w.grad = into if ATTACHED else None
    assert attempt() == "right"
print("done", first)
"""


@pytest.mark.parametrize("kind,attached", [("{}", False), ("{'grad_into': into}", False), ("{'grad_into': into}", True)])
def test_backward_in_a_graph_is_refused_or_right_beside_an_eager_graph(kind, attached):
    # Where autograd would make the eager graph's stream wait, CUDA ends the capture; without the eager graph it is captured.
    child = GRAPH_BESIDE_GRAPH.replace("KIND", kind).replace("ATTACHED", str(attached))
    p = subprocess.run([sys.executable, "-c", child], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=300)
    assert p.returncode == 0 and "done" in p.stdout, (p.returncode, p.stdout, p.stderr[-2000:])


def test_forward_derivatives_are_refused():
    w = values((20, 8), F32, 1).requires_grad_(True)
    t = tokens_of(30, 20, 2)
    forward = torch.autograd.forward_ad
    y = ar.ops.embedding(t, w)
    with forward.dual_level():
        with pytest.raises(ar.IbcommError, match="forward-mode"):
            ar.ops.embedding(t, forward.make_dual(w.detach(), torch.ones_like(w)))
        dy = forward.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, w, dy, retain_graph=True)
    (g,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert torch.equal(g, grad_in_64_bits(t, torch.ones(30, 8, device="cuda"), 20, 1.0)[0].float())
    # A table that is trained is refused by the tracer itself, which comes first.
    for table, words in ((w, "requires grad"), (w.detach(), "traced")):
        with pytest.raises(RuntimeError, match=words):
            torch.jit.trace(lambda x: ar.ops.embedding(x, table), t)


@pytest.mark.parametrize("overlap", [False, True])
def test_hooks_of_the_table_see_its_gradient(overlap):
    shapes = [(50, 24), (24,)]
    buckets = ar.GradientBuckets(shapes)
    w, b = torch.nn.Parameter(values(shapes[0], F32, 1)), torch.nn.Parameter(values(shapes[1], F32, 2))
    (buckets.overlap_with_backward if overlap else buckets.attach)([w, b])
    t, dy = tokens_of(500, 50, 3), values((500, 24), F32, 4)
    want, bound = grad_in_64_bits(t, dy, 50, 2.0)
    seen = []

    def step():
        buckets.zero_()
        (buckets.embedding(0, t, w, scale=2.0) + b).backward(dy)
        if overlap:
            buckets.finish()
        assert w.grad.data_ptr() == buckets.views[0].data_ptr()
        return buckets.views[0].clone()

    handle = w.register_hook(lambda g: seen.append(g.clone()) or 4 * g)  # scaling by a power of two is exact
    got = step()
    assert len(seen) == 1 and torch.equal(4 * seen[0], got)
    within(seen[0], want, bound + U * want.abs())
    handle.remove()
    within(step(), want, bound + 2 * U * want.abs())
    assert len(seen) == 1
    # Added to another tensor, or to that of a table which is no leaf: refused before anything is added.
    into = torch.zeros(50, 24, device="cuda")
    w.register_hook(lambda g: seen.append(g))
    with pytest.raises(RuntimeError, match="hook"):
        ar.ops.embedding(t, w, grad_into=into).sum().backward()
    table = w.detach().requires_grad_(True) * 1
    ar.ops.embedding(t, table, grad_into=into, scale=2.0).backward(dy)
    within(into, want, bound + 2 * U * want.abs())
    into.zero_()
    table.register_hook(lambda g: seen.append(g))
    with pytest.raises(RuntimeError, match="hook"):
        ar.ops.embedding(t, table, grad_into=into).sum().backward()
    assert len(seen) == 1 and not into.any()


@pytest.mark.parametrize("bound", [1e-3, 1e-7, 1e-30])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("n", [5, 70001, 40000001])
@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
def test_clipping_by_coefficients_below_the_normal_numbers(types, n, offset, bound):
    # The coefficient is 3e-42 or less; what it scales is an ordinary number all the same.
    a, b = types
    x = values((n + offset,), a, 1, 1e33)[offset:]
    x[3] = 3e38
    out = torch.empty(n + offset, device="cuda", dtype=b)[offset:]
    norm = norm_of([x], 2)
    within(ar.ops.clip_grad_norm(x, bound, out=out), norm, norm_rtol(a) * norm.item())
    want = x.double() * (bound / (norm.item() + 1e-6))
    assert want[3] > 0.99 * bound
    # One more rounding to a multiple of fp32's least number where the product is below its normal ones.
    within(out, want, (6.5 * U + half(b)) * want.abs() + least(F32) + least(b))
    if a == b:
        ar.ops.clip_grad_norm(x, bound)
        assert torch.equal(x, out)


class KernelNode(C.Structure):
    _fields_ = [("func", C.c_void_p), ("grid", C.c_uint * 3), ("block", C.c_uint * 3), ("smem", C.c_uint), ("params", C.c_void_p), ("extra", C.c_void_p),
                ("kernel", C.c_void_p), ("context", C.c_void_p)]


def grids_of(call):
    """(blocks, threads) of the kernels that a call launches."""
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    driver, raw, count = C.CDLL("libcuda.so.1"), C.c_void_p(graph.raw_cuda_graph()), C.c_size_t(0)
    assert driver.cuGraphGetNodes(raw, None, C.byref(count)) == 0
    nodes = (C.c_void_p * count.value)()
    assert driver.cuGraphGetNodes(raw, nodes, C.byref(count)) == 0
    found = []
    for node in nodes:
        kernel = KernelNode()
        assert driver.cuGraphKernelNodeGetParams_v2(C.c_void_p(node), C.byref(kernel)) == 0
        found.append((kernel.grid[0], kernel.block[0]))
    return found


@pytest.mark.parametrize("most", [0, 5, 40])
def test_where_a_grid_that_waits_does_not_fit(most):
    # As in a process that has a part of the GPU: kernels that do not wait, or a smaller grid, with the same results.
    xs = [values((3000001,), F32, 1), values((70001,), BF16, 2)]
    outs = [torch.empty_like(x) for x in xs]
    n, rows = 140001, 3001
    t, g = tokens_of(n, rows, 3), values((n, 24), BF16, 4)
    calls = [lambda: ar.ops.grad_norm(xs), lambda: ar.ops.clip_grad_norm(xs, 1.0, out=outs), lambda: ar.ops.embedding_grad(t, g, num_rows=rows, dtype=F32)]
    want, table = norm_of(xs, 2), calls[2]()
    assert len(grids_of(calls[0])) == len(grids_of(calls[1])) == 1 and max(b for b, threads in grids_of(calls[2]) if threads == 512) > 40
    ar.utils.set_tunable("IBCOMM_COOPERATIVE_CTAS", most)
    try:
        assert len(grids_of(calls[0])) == len(grids_of(calls[1])) == 2
        assert 1 <= max(b for b, threads in grids_of(calls[2]) if threads == 512) <= max(most, 1)
        within(calls[0](), want, 5.5 * U * want.item())
        within(calls[1](), want, 5.5 * U * want.item())
        for x, o in zip(xs, outs):
            w = x.double() / (want.item() + 1e-6)
            within(o, w, (6.5 * U + half(x.dtype)) * w.abs() + least(x.dtype))
        assert torch.equal(calls[2](), table)
    finally:
        ar.utils.set_tunable("IBCOMM_COOPERATIVE_CTAS", -1)


def test_a_hook_that_was_taken_out_refuses_nothing():
    t, into = tokens_of(30, 20, 2), torch.zeros(20, 8, device="cuda")
    want = grad_in_64_bits(t, torch.ones(30, 8, device="cuda"), 20, 1.0)[0].float()  # whole numbers
    for w in (values((20, 8), F32, 1).requires_grad_(True), values((20, 8), F32, 1).requires_grad_(True) * 1):
        w.register_hook(lambda g: 2 * g).remove()
        into.zero_()
        ar.ops.embedding(t, w, grad_into=into).sum().backward()
        assert torch.equal(into, want)
        w.register_hook(lambda g: 2 * g)
        with pytest.raises(RuntimeError, match="hook"):
            ar.ops.embedding(t, w, grad_into=into).sum().backward()
        assert torch.equal(into, want)
