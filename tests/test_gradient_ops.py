"""The gradient norm, clipping and the embedding without a GPU: the host path of the first two, and what the entry points
refuse before anything is launched."""
import ctypes as C
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import allreduce_proto_b200 as ar
from allreduce_proto_b200 import _native
from test_fastcall import outcomes

ROOT = Path(__file__).resolve().parent.parent


def lists(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g, dtype=torch.float64).to(dtype) for s in ((1,), (3, 5), (0,), (1000,), (7, 11, 13))]


@pytest.mark.parametrize("power", [2.0, math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_host_norm_and_clipping(dtype, power):
    ts = lists(dtype)
    whole = torch.cat([t.double().flatten() for t in ts])
    want = whole.norm() if power == 2 else whole.abs().max()
    # Sums in 64 bits, one rounding of the norm.
    rtol = 1e-12 if dtype == torch.float64 else 2.0 ** -24
    norm = ar.ops.grad_norm(ts, norm_type=power)
    assert norm.dtype == dtype and norm.dim() == 0
    torch.testing.assert_close(norm.double(), want, rtol=rtol, atol=0)
    outs = [torch.full_like(t, 7) for t in ts]
    before = [t.clone() for t in ts]
    assert torch.equal(ar.ops.clip_grad_norm(ts, 0.5, out=outs, norm_type=power), norm)
    c = 0.5 / (float(want) + 1e-6)
    # The coefficient and the product are rounded once each.
    step = torch.finfo(dtype).eps / 2
    for t, b, o in zip(ts, before, outs):
        assert torch.equal(t, b)
        torch.testing.assert_close(o.double(), b.double() * c, rtol=3 * step + 1e-12, atol=0)
    ar.ops.clip_grad_norm(ts, 0.5, norm_type=power)
    assert all(torch.equal(t, o) for t, o in zip(ts, outs))
    # Below the bound nothing changes.
    ar.ops.clip_grad_norm(ts, 1e3, norm_type=power)
    assert all(torch.equal(t, o) for t, o in zip(ts, outs))


def test_host_norms_that_are_not_finite():
    for power in (2.0, math.inf):
        for place in (0, 1, 2):
            x = torch.ones(3)
            x[place] = math.inf
            assert float(ar.ops.grad_norm([x], norm_type=power)) == math.inf
            x[(place + 1) % 3] = math.nan
            assert math.isnan(ar.ops.grad_norm([x], norm_type=power))
            ar.ops.clip_grad_norm([x], 1.0, norm_type=power)
            assert torch.isnan(x).all()
    # Squares beyond fp32's range.
    assert math.isclose(float(ar.ops.grad_norm(torch.full((4,), 1e30))), 2e30, rel_tol=1e-6)
    assert math.isclose(float(ar.ops.grad_norm(torch.full((4,), 1e-30))), 2e-30, rel_tol=1e-6)
    assert float(ar.ops.grad_norm([])) == 0 and float(ar.ops.grad_norm(torch.empty(0))) == 0
    x = torch.ones(4)
    ar.ops.clip_grad_norm(x, 0.0)
    assert torch.equal(x, torch.zeros(4))


@pytest.mark.parametrize("bound", [1e-3, 1e-7, 1e-30])
def test_host_clipping_by_coefficients_below_the_normal_numbers(bound):
    x = torch.tensor([3e38, -1e38, 1e30, 0.0])
    want = x.double() * (bound / (float(x.double().norm()) + 1e-6))
    out = torch.empty_like(x)
    ar.ops.clip_grad_norm(x, bound, out=out)
    # The product is rounded, to a multiple of the least number where it is below the normal ones.
    assert torch.all((out.double() - want).abs() <= 3 * 2.0 ** -24 * want.abs() + 2.0 ** -150), (out, want)
    ar.ops.clip_grad_norm(x, bound)
    assert torch.equal(x, out)


def test_buckets_on_the_host():
    shapes = [(300, 7), (5,), (64, 64)]
    buckets = ar.GradientBuckets(shapes, device="cpu", bucket_bytes=4096, shardable=True)
    grads = [torch.randn(s) for s in shapes]
    buckets.load(grads)
    want = torch.cat([g.double().flatten() for g in grads]).norm()
    torch.testing.assert_close(buckets.grad_norm().double(), want, rtol=2.0 ** -24, atol=0)
    assert torch.equal(buckets.grad_norm(), buckets.grad_norm(sharded=True))
    norm = buckets.clip_grad_norm(1.0)
    torch.testing.assert_close(norm.double(), want, rtol=2.0 ** -24, atol=0)
    for v, g in zip(buckets.views, grads):
        torch.testing.assert_close(v.double(), g.double() / (float(want) + 1e-6), rtol=3 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("sharded", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_buckets_recover_from_a_step_that_is_not_finite(bad, sharded):
    # Sizes that leave room up to the next 16 bytes behind every tensor, and gradients that are written through their views only.
    shapes = [(5,), (7,), (0,), (8,), (3, 3)]
    buckets = ar.GradientBuckets(shapes, device="cpu", shardable=True)
    params = [torch.nn.Parameter(torch.zeros(s)) for s in shapes]
    buckets.attach(params)
    ones, spoilt = [torch.ones(s) for s in shapes], [torch.ones(s) for s in shapes]
    spoilt[0][2] = bad
    for write in (buckets.load, lambda gs: [p.grad.add_(g) for p, g in zip(params, gs)]):
        write(spoilt)
        assert not math.isfinite(buckets.clip_grad_norm(1.0, sharded=sharded))
        torch.optim.SGD(params, lr=1.0).zero_grad(set_to_none=False)
        write(ones)
        want = torch.tensor(29.0, dtype=torch.float64).sqrt()
        for same in (False, True):
            torch.testing.assert_close(buckets.grad_norm(sharded=same).double(), want, rtol=2.0 ** -24, atol=0)
        buckets.clip_grad_norm(1.0, sharded=sharded)
        for v in buckets.views:
            torch.testing.assert_close(v.double(), torch.full_like(v, 1).double() / (want + 1e-6), rtol=3 * 2.0 ** -24, atol=0)
        torch.optim.SGD(params, lr=1.0).zero_grad(set_to_none=False)
    assert ar.GradientBuckets([], device="cpu").grad_norm() == 0 and ar.GradientBuckets([(0,)], device="cpu").grad_norm() == 0


SHARDED = """
import math, torch
import allreduce_proto_b200 as ar
comm = ar.Communicator.from_env()
torch.manual_seed(comm.rank)
mine = [torch.randn(100 + comm.rank), torch.randn(3, 2, dtype=torch.float64)]
whole = []
for r in range(comm.world_size):
    torch.manual_seed(r)
    whole += [torch.randn(100 + r).double(), torch.randn(3, 2, dtype=torch.float64).flatten()]
whole = torch.cat(whole)
for power, want in ((2.0, whole.norm()), (math.inf, whole.abs().max())):
    torch.testing.assert_close(ar.ops.grad_norm(mine, norm_type=power, comm=comm), want, rtol=1e-12, atol=0)
norm = ar.ops.clip_grad_norm(mine, 1.0, comm=comm)
both = [torch.zeros(comm.world_size, dtype=torch.float64)]
comm.all_gather(ar.ops.grad_norm(mine).reshape(1), both[0])
torch.testing.assert_close(both[0].norm(), torch.tensor(1.0, dtype=torch.float64), rtol=1e-5, atol=0)
buckets = ar.GradientBuckets([(50, 3), (7,)], dtype=torch.float32, device="cpu", comm=comm, shardable=True,
                             symmetric=False, bucket_bytes=128)
buckets.load([torch.full((50, 3), 1.0 + comm.rank), torch.full((7,), 2.0)])
buckets.reduce_scatter(average=True)
sharded = buckets.clip_grad_norm(1.0, sharded=True)
buckets.all_gather()
mean = 1.0 + (comm.world_size - 1) / 2
want = math.sqrt(150 * mean ** 2 + 28)
assert math.isclose(float(sharded), want, rel_tol=1e-6), (float(sharded), want)
assert math.isclose(float(buckets.grad_norm()), 1.0, rel_tol=1e-5)
comm.close()
"""


AFTER_NAN = """
import math, torch
import allreduce_proto_b200 as ar
comm = ar.Communicator.from_env()
shapes = [(5,), (7,), (1,), (9,)]   # blocks that begin and end inside of tensors, and between them
for bucket_bytes in (48, 1 << 20):
    buckets = ar.GradientBuckets(shapes, device="cpu", comm=comm, shardable=True, symmetric=False, bucket_bytes=bucket_bytes)
    for first in (math.nan, 1.0, 1.0):
        buckets.load([torch.full(s, first if i == 0 else 1.0) for i, s in enumerate(shapes)])
        buckets.reduce_scatter(average=True)
        norm = float(buckets.grad_norm(sharded=True))
        assert float(buckets.clip_grad_norm(1.0, sharded=True)) == norm or math.isnan(first)
        assert math.isnan(norm) if math.isnan(first) else math.isclose(norm, math.sqrt(22), rel_tol=2.0 ** -23), norm
        buckets.all_gather()
        for v in buckets.views:
            want = torch.full_like(v, first / math.sqrt(22))
            torch.testing.assert_close(v, want, rtol=1e-6, atol=0, equal_nan=True)
comm.close()
"""


@pytest.mark.parametrize("np_", [2, 3])
def test_shards_recover_from_a_step_that_is_not_finite(bins, np_, tmp_path):
    script = tmp_path / "after_nan.py"
    script.write_text(AFTER_NAN)
    p = subprocess.run(["timeout", "120s", bins["ibcomm_run"], "-np", str(np_), "-x", f"PYTHONPATH={ROOT}", sys.executable, str(script)],
                       stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
    assert p.returncode == 0, p.stderr[-3000:]


@pytest.mark.parametrize("np_", [2, 3])
def test_norm_of_shards_on_several_ranks(bins, np_, tmp_path):
    script = tmp_path / "sharded.py"
    script.write_text(SHARDED)
    p = subprocess.run(["timeout", "120s", bins["ibcomm_run"], "-np", str(np_), "-x", f"PYTHONPATH={ROOT}", sys.executable, str(script)],
                       stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
    assert p.returncode == 0, p.stderr[-3000:]


@pytest.mark.parametrize("mode", [[], ["--overlap"], ["--sharded"]])
def test_example_with_clipping(mode):
    port = 29660 + len(mode) + mode.count("--sharded")
    cmd = ["timeout", "300s", sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", "2", "--master-addr", "127.0.0.1",
           "--master-port", str(port), str(ROOT / "examples" / "ddp_gradient_buckets.py"), "--device", "cpu", "--steps", "2", "--clip", "0.1", *mode]
    p = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert p.returncode == 0, p.stdout[-3000:]
    assert p.stdout.count(": OK") == 2, p.stdout[-3000:]


def code_of(call):
    with pytest.raises(ar.IbcommError) as e:
        call()
    return e.value.code


def test_what_the_host_path_refuses():
    x, y = torch.ones(8), torch.ones(4, 8)
    clip, norm = ar.ops.clip_grad_norm, ar.ops.grad_norm
    assert code_of(lambda: norm([x], norm_type=1.0)) == ar.NOT_SUPPORTED
    assert code_of(lambda: norm([x.half()])) == ar.NOT_SUPPORTED
    assert code_of(lambda: norm([x.int()])) == ar.NOT_SUPPORTED
    assert code_of(lambda: norm([y.t()])) == ar.INVALID_ARGUMENT
    for bad in (-1.0, math.nan):
        assert code_of(lambda: clip([x], bad)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: clip([x], 1.0, out=[])) == ar.INVALID_ARGUMENT
    assert code_of(lambda: clip([x], 1.0, out=[torch.ones(7)])) == ar.INVALID_ARGUMENT
    assert code_of(lambda: clip([x], 1.0, out=[x.double()])) == ar.NOT_SUPPORTED
    # The same memory twice, or part of it.
    assert code_of(lambda: clip([x, x], 1.0)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: clip([x[:5], x[4:]], 1.0)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: clip([x[:4]], 1.0, out=[x[2:6]])) == ar.INVALID_ARGUMENT
    assert code_of(lambda: clip([y[0], y[1]], 1.0, out=[y[1], y[0]])) == ar.INVALID_ARGUMENT
    assert code_of(lambda: clip([y[0], y[1]], 1.0, out=[y[2], y[2]])) == ar.INVALID_ARGUMENT
    assert torch.equal(x, torch.ones(8)) and torch.equal(y, torch.ones(4, 8))
    clip([y[0], y[1]], 1.0, out=[y[0], y[3]])  # one in place, one not
    # Reading the same memory twice counts it twice.
    assert math.isclose(float(norm([x, x])), 4.0)
    with pytest.raises(TypeError):
        norm([None])


def test_what_the_embedding_refuses_without_a_gpu():
    t, w = torch.zeros(3, dtype=torch.int64), torch.ones(4, 8)
    assert code_of(lambda: ar.ops.embedding(t, w)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding(t.float(), w)) == ar.NOT_SUPPORTED
    assert code_of(lambda: ar.ops.embedding(t, w, padding_idx=4)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding(t, w, out_dtype=torch.float8_e4m3fn)) == ar.NOT_SUPPORTED
    assert code_of(lambda: ar.ops.embedding(t, w, grad_into=torch.ones(4, 7))) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding(t, w, grad_into=torch.ones(4, 8).double())) == ar.NOT_SUPPORTED
    g = torch.ones(3, 8)
    assert code_of(lambda: ar.ops.embedding_grad(t, g)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding_grad(t, g, num_rows=4, accumulate=True)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding_grad(t, g, num_rows=-1)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding_grad(t, g, out=w, num_rows=4)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding_grad(t, g, out=w, padding_idx=-2)) == ar.INVALID_ARGUMENT
    assert code_of(lambda: ar.ops.embedding_grad(t, g, out=w)) == ar.INVALID_ARGUMENT


def test_what_the_call_path_refuses_of_cuda_tensors():
    # `t` and `other` of the runner claim to be on two GPUs and have no memory.
    cases = {
        "fast.grad_norm([t, other], 2, None, 0)": "the tensors must live on one GPU",
        "fast.grad_norm([t, host], 2, None, 0)": "tensors must live on the GPU",
        "fast.grad_norm([], 2, None, 0)": "a tensor is expected at least",
        "fast.grad_norm([t.reshape(2, 4)[:, :3]], 2, None, 0)": "tensors must be dense",
        "fast.clip_grads([t], [t, t], 2, 1.0, None)": "one output per tensor is expected",
        "fast.clip_grads([t], [t[:7]], 2, 1.0, None)": "an output must match its tensor in shape and strides",
        "fast.clip_grads([t.reshape(2, 4)], [t.reshape(4, 2).t()], 2, 1.0, None)": "an output must match its tensor in shape and strides",
        "fast.clip_grads([t], [other], 2, 1.0, None)": "the tensors must live on one GPU",
        "fast.clip_grads([t], None, 2, 1.0, t)": "the ranks' sums must be float64 on the tensors' GPU",
        "fast.embedding(host, t.reshape(2, 4), -1, 1.0, -1, None)": "tensors must live on the GPU",
        "fast.embedding(other, t.reshape(2, 4), -1, 1.0, -1, None)": "tokens and table must live on the same GPU",
        "fast.embedding(t, t, -1, 1.0, -1, None)": "a table has rows and columns",
        "fast.embedding_grad(t, t, t, -1, 1.0, False)": "a table has rows and columns",
        "fast.embedding_grad(t[:3], t, t.reshape(2, 4), -1, 1.0, False)": "grad must hold a row of the table's width for every token",
        "fast.embedding_grad(other[:2], t.reshape(2, 4), t.reshape(2, 4), -1, 1.0, False)": "tokens, grad and table must live on the same GPU",
        "fast.embedding_grad(t[::4], t, t.reshape(2, 4), -1, 1.0, False)": "tensors must be contiguous",
    }
    for call, got in outcomes(list(cases)).items():
        assert cases[call] in got and got != "nothing", (call, got)


def test_derivatives_that_the_embedding_does_not_have_are_refused():
    # Before anything else is looked at, so on tensors of the host too.
    w, t = torch.ones(4, 8), torch.zeros(3, dtype=torch.int64)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ar.IbcommError, match="forward-mode") as e:
            ar.ops.embedding(t, torch.autograd.forward_ad.make_dual(w, w))
        assert e.value.code == ar.NOT_SUPPORTED
    with pytest.raises(ar.IbcommError, match="traced") as e:
        torch.jit.trace(lambda x: ar.ops.embedding(x, w), t)
    assert e.value.code == ar.NOT_SUPPORTED
    with pytest.raises(ar.IbcommError, match="on the GPU"):  # and nothing is left of either
        ar.ops.embedding(t, w)


def grad_tensors(*items):
    list_ = (_native.GradTensor * len(items))()
    for g, (p, o, n, a, b) in zip(list_, items):
        g.in_, g.out, g.len_elements, g.dtype_in, g.dtype_out = p, o, n, a, b
    return list_


def test_what_the_c_interface_refuses():
    # Addresses that nothing reads: the checks come before the launch.
    lib = _native.lib()
    one = grad_tensors((4096, 4096, 8, 0, 0))
    norm = lambda ts, power=2, sums=None, n=0, work=4096, dt=0: lib.ibcomm_grad_norm(ts, len(ts), power, sums, n, work, 4096, dt, None, None)  # noqa: E731
    clip = lambda ts, m=1.0, work=4096: lib.ibcomm_clip_grads(ts, len(ts), 2, m, None, 0, work, 4096, 0, None)  # noqa: E731
    assert norm(one, power=1) == ar.NOT_SUPPORTED
    assert norm(one, work=None) == ar.INVALID_ARGUMENT
    assert norm(one, sums=4096, n=0) == ar.INVALID_ARGUMENT
    assert norm(one, dt=4) == ar.NOT_SUPPORTED and norm(one, dt=9) == ar.INVALID_ARGUMENT
    assert norm(grad_tensors((None, None, 8, 0, 0))) == ar.INVALID_ARGUMENT
    assert norm(grad_tensors((4097, None, 8, 0, 0))) == ar.INVALID_ARGUMENT
    assert norm(grad_tensors((4096, None, 8, 2, 2))) == ar.NOT_SUPPORTED
    assert lib.ibcomm_grad_norm(one, -1, 2, None, 0, 4096, 4096, 0, None, None) == ar.INVALID_ARGUMENT
    assert lib.ibcomm_grad_norm(None, 1, 2, None, 0, 4096, 4096, 0, None, None) == ar.INVALID_ARGUMENT
    assert clip(one, m=-1.0) == ar.INVALID_ARGUMENT and clip(one, m=math.nan) == ar.INVALID_ARGUMENT
    assert clip(grad_tensors((4096, None, 8, 0, 0))) == ar.INVALID_ARGUMENT
    for a, b in ((4, 5), (5, 4), (0, 1), (1, 0)):
        assert clip(grad_tensors((4096, 8192, 8, a, b))) == ar.NOT_SUPPORTED
    assert clip(grad_tensors((4096, 4096, 8, 0, 5))) == ar.INVALID_ARGUMENT  # in place, of another type
    assert clip(grad_tensors((4096, 4096, 8, 0, 0), (4096 + 28, 4096 + 28, 8, 0, 0))) == ar.INVALID_ARGUMENT

    size = C.c_size_t(0)
    assert lib.ibcomm_embedding_grad_work(1000, 50, 64, C.byref(size)) == 0 and size.value > 0
    assert lib.ibcomm_embedding_grad_work(1000, 50, 64, None) == ar.INVALID_ARGUMENT
    grad = lambda tok=1 << 20, td=3, n=1000, g=1 << 21, gd=0, out=1 << 22, od=0, rows=50, width=64, pad=-1, s=1.0, work=1 << 23, b=size.value: (  # noqa: E731
        lib.ibcomm_embedding_grad(tok, td, n, g, gd, out, od, rows, width, pad, s, 0, work, b, None))
    assert grad(td=0) == ar.NOT_SUPPORTED and grad(gd=1) == ar.NOT_SUPPORTED and grad(od=2) == ar.NOT_SUPPORTED
    assert grad(tok=None) == ar.INVALID_ARGUMENT and grad(g=None) == ar.INVALID_ARGUMENT and grad(out=None) == ar.INVALID_ARGUMENT
    assert grad(rows=1 << 31) == ar.NOT_SUPPORTED and grad(n=1 << 31) == ar.NOT_SUPPORTED
    assert grad(pad=50) == ar.INVALID_ARGUMENT and grad(pad=-2) == ar.INVALID_ARGUMENT
    assert grad(s=math.nan) == ar.INVALID_ARGUMENT
    assert grad(b=size.value - 1) == ar.INVALID_ARGUMENT and grad(work=None) == ar.INVALID_ARGUMENT and grad(work=(1 << 23) + 4) == ar.INVALID_ARGUMENT
    assert grad(out=(1 << 21) + 256) == ar.INVALID_ARGUMENT  # the rows that are read are the table that is written
    look = lambda td=3, wd=0, od=0, out=1 << 22: lib.ibcomm_embedding(1 << 20, td, 100, 1 << 21, wd, 50, 64, out, od, 1.0, None)  # noqa: E731
    assert look(td=4) == ar.NOT_SUPPORTED and look(wd=1) == ar.NOT_SUPPORTED and look(od=3) == ar.NOT_SUPPORTED
    assert look(out=None) == ar.INVALID_ARGUMENT and look(out=1 << 21) == ar.INVALID_ARGUMENT


def test_what_is_not_aligned_is_refused():
    # A kernel would fault on it: nothing is launched.
    lib = _native.lib()
    one = grad_tensors((4096, 8192, 8, 0, 0))
    for off in (1, 2, 4):
        norm = lambda sums=None, work=4096, norm=4096, dt=1, sum_=4096: lib.ibcomm_grad_norm(one, 1, 2, sums, 1, work, norm, dt, sum_, None)  # noqa: E731
        assert norm(sums=4096 + off) == norm(work=4096 + off) == norm(norm=4096 + off) == norm(sum_=4096 + off) == ar.INVALID_ARGUMENT
        clip = lambda sums=None, work=4096, norm=4096: lib.ibcomm_clip_grads(one, 1, 2, 1.0, sums, 1, work, norm, 1, None)  # noqa: E731
        assert clip(sums=4096 + off) == clip(work=4096 + off) == clip(norm=4096 + off) == ar.INVALID_ARGUMENT
        look = lambda t=0, w=0, o=0: lib.ibcomm_embedding((1 << 20) + t, 3, 100, (1 << 21) + w, 0, 50, 64, (1 << 22) + o, 0, 1.0, None)  # noqa: E731
        assert look(t=off) == ar.INVALID_ARGUMENT
        grad = lambda t=0, g=0, o=0: lib.ibcomm_embedding_grad((1 << 20) + t, 3, 9, (1 << 21) + g, 0, (1 << 22) + o, 0, 50, 64, -1, 1.0, 0, None, 0, None)  # noqa: E731
        assert grad(t=off) == ar.INVALID_ARGUMENT
        if off < 4:
            assert look(w=off) == look(o=off) == grad(g=off) == grad(o=off) == ar.INVALID_ARGUMENT


def test_tensors_without_elements_share_no_memory():
    # Empty parts of the table that is written, or read: nothing to launch, and nothing to refuse.
    lib = _native.lib()
    for inside in (1 << 22, (1 << 22) + 64):
        assert lib.ibcomm_embedding_grad(inside, 3, 0, inside, 0, 1 << 22, 0, 50, 64, -1, 1.0, 1, None, 0, None) == 0
        assert lib.ibcomm_embedding(inside, 3, 0, 1 << 22, 0, 50, 64, inside, 0, 1.0, None) == 0
    # One that is not empty.
    assert lib.ibcomm_embedding_grad(1 << 20, 3, 9, (1 << 22) + 64, 0, 1 << 22, 0, 50, 64, -1, 1.0, 1, None, 0, None) == ar.INVALID_ARGUMENT
