"""How the operators over a vocabulary are called: from threads, on streams, and what the context says of it."""
import threading

import pytest
import torch

import linalg_b200 as lb

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(gpu):
    return lb.Context(0)


def test_long_rows_from_threads(ctx):
    """Vocabularies whose kernel takes more shared memory than any kernel may without asking, of several sizes, from threads
    at once: no call takes from another what it asked for."""
    jobs = []
    for v in (2_000_000, 1_400_000, 1_900_000, 1_500_000):
        x = torch.randn(1, v, device="cuda", generator=torch.Generator("cuda").manual_seed(v))
        ids, z = torch.arange(4, device="cuda").int()[None], torch.full((1, 4), -2.0, device="cuda")
        loss = torch.empty(1, device="cuda")
        jobs.append([lb.View.of(t) for t in (x, ids, z, loss)] + [torch.cuda.Stream().cuda_stream])
    torch.cuda.synchronize()
    want, failed = [], []
    for x, ids, z, loss, _ in jobs:
        lb.distill_loss(ctx, x, ids, z, 1.0, loss, tail=True)
        want.append(loss.owner.clone())
    torch.cuda.synchronize()
    start = threading.Barrier(len(jobs))

    def work(x, ids, z, loss, stream):
        start.wait()
        try:
            for _ in range(4000):
                lb.encode_distill_loss(ctx, stream, x, ids, z, 1.0, loss, tail=True)
        except lb.LinalgError as e:
            failed.append(str(e))

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for job, w in zip(jobs, want):
        assert torch.equal(job[3].owner, w)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("unit", [True, False])
def test_nan_of_a_teacher_shows(ctx, tail, unit):
    """A NaN among a teacher's entries makes the loss NaN, also where the student's row is masked throughout."""
    x = torch.randn(3, 500, device="cuda")
    x[1] = -float("inf")
    ids = torch.arange(3, device="cuda").int().expand(3, 3).contiguous()
    z = torch.full((3, 3), -2.0, device="cuda")
    z[:2, 1] = float("nan")
    if not unit:
        x = x.t().contiguous().t()
    only, loss, dx = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda"), torch.zeros_like(x)
    torch.cuda.synchronize()
    lb.distill_loss(ctx, x, ids, z, 1.0, only, tail=tail)
    lb.distill_grad(ctx, x, ids, z, 1.0, dx, loss=loss, tail=tail)
    for got in (only, loss):
        assert got.isnan().tolist() == [True, True, False]


def test_the_kernel_that_ran_is_the_one_recorded(ctx):
    """A vocabulary too long for a cluster's shared memory goes to the kernel for any strides, and the record says so."""
    x = torch.zeros(1, 4_300_001, device="cuda", dtype=torch.bfloat16)
    ids, z = torch.zeros(1, 1, device="cuda").int(), torch.full((1, 1), -1.0, device="cuda")
    loss, dx = torch.empty(1, device="cuda"), torch.empty_like(x)
    torch.cuda.synchronize()
    for n, way in ((x.shape[1], "strided"), (4_000_000, "rows")):
        lb.distill_loss(ctx, x[:, :n], ids, z, 1.0, loss, tail=True)
        lb.distill_grad(ctx, x[:, :n], ids, z, 1.0, dx[:, :n], tail=True)
        assert ctx.debug_launches()[-2:] == [f"distill_loss_{way}", f"distill_grad_{way}"]


def test_the_default_stream_by_its_object(ctx):
    """A call on torch's default stream, named by its object, comes after what torch has put there and before what follows."""
    n, v, k = 64, 30011, 8
    x = torch.randn(n, v, device="cuda")
    t = torch.zeros(n, dtype=torch.int32, device="cuda")
    lp, stats, ids = torch.empty(n, device="cuda"), torch.empty(n, 2, device="cuda"), torch.empty(n, k, device="cuda").int()
    late, dx, work = torch.zeros_like(x), torch.empty_like(x), torch.empty(1 << 28, device="cuda")
    stream = torch.cuda.current_stream()
    assert stream.cuda_stream == 0
    torch.cuda.synchronize()
    got = []
    for _ in range(2):
        late.zero_()
        for _ in range(4):
            work.zero_()  # a millisecond or so in which a kernel on another stream would read the zeros
        late.copy_(x)
        lb.encode_token_logprobs(ctx, stream, late, t, 1.0, logprob=lp, stats=stats, top_ids=ids)
        lb.encode_token_logprobs_backward(ctx, stream, late, t, 1.0, stats, lp, dx)
        got.append([y.clone() for y in (lp, stats, ids, dx)])
        late.zero_()
    want = torch.log_softmax(x.double(), 1)
    assert torch.equal(got[0][2].long(), x.topk(k, 1).indices)
    assert (got[0][0].double() - want[:, 0]).abs().max() < 1e-4
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_products_on_the_default_stream(ctx):
    """The other calls take the same object: products with a split sum among them, which need scratch."""
    stream = torch.cuda.current_stream()
    for dtype, (m, n, k) in ((torch.float32, (96, 64, 20000)), (torch.bfloat16, (128, 256, 16384)), (torch.bfloat16, (100, 36, 52))):
        a, b = torch.randn(m, k, device="cuda").to(dtype), torch.randn(k, n, device="cuda").to(dtype)
        own, c = (torch.zeros(m, n, device="cuda", dtype=dtype) for _ in range(2))
        turned = torch.zeros(n, m, device="cuda")
        torch.cuda.synchronize()
        lb.gemm(ctx, 1.0, a, b, 0.0, own)
        lb.encode_gemm(ctx, stream, 1.0, a, b, 0.0, c)
        lb.encode_materialize(ctx, stream, c.float().t(), turned)
        again = turned.clone()
        torch.cuda.synchronize()
        assert torch.equal(c, own) and torch.equal(again, c.float().t())
