"""Refusals of the operators over a vocabulary: every check runs before the context is looked at, so a call without one
shows them here.  Nothing is launched."""
import ctypes as C

import pytest

import linalg_b200 as lb

N, V, K = 6, 100, 4
SIZE = {lb.F32: 4, lb.BF16: 2, lb.F16: 2, lb.I32: 4, lb.U32: 4, lb.F64: 8}
_next = [1 << 20]


def view(shape, dtype=lb.F32, strides=None, base=None, offset=0):
    v = lb.lc_view()
    if base is None:
        _next[0] += 1 << 24
        base = _next[0]
    if strides is None:
        strides, s = [], 1
        for n in reversed(shape):
            strides.insert(0, s)
            s *= n
    v.data, v.offset, v.dtype, v.rank = base, offset, dtype, len(shape)
    last = offset + sum((n - 1) * s for n, s in zip(shape, strides)) if all(shape) else offset
    v.buffer_bytes = (last + 1) * SIZE[dtype]
    for i, (n, s) in enumerate(zip(shape, strides)):
        v.shape[i], v.strides[i] = n, s
    return v


def ref(v):
    return None if v is None else C.byref(v)


def said():
    return lb.load().lc_last_error().decode()


def scores(**kw):
    a = dict(logits=view([N, V], lb.BF16), targets=view([N], lb.I32), scale=1.0, logprob=view([N]), entropy=view([N]),
             stats=view([N, 2]), top_logprobs=view([N, K]), top_ids=view([N, K], lb.U32)) | kw
    return lb.load().lc_encode_token_logprobs(None, None, ref(a["logits"]), ref(a["targets"]), a["scale"], ref(a["logprob"]),
                                              ref(a["entropy"]), ref(a["stats"]), ref(a["top_logprobs"]), ref(a["top_ids"]))


def scores_grad(**kw):
    a = dict(logits=view([N, V], lb.BF16), targets=view([N], lb.I32), scale=1.0, stats=view([N, 2]), entropy=view([N]),
             d_logprob=view([N]), d_entropy=view([N]), dlogits=view([N, V], lb.BF16)) | kw
    return lb.load().lc_encode_token_logprobs_backward(None, None, ref(a["logits"]), ref(a["targets"]), a["scale"], ref(a["stats"]),
                                                       ref(a["entropy"]), ref(a["d_logprob"]), ref(a["d_entropy"]), ref(a["dlogits"]))


def distill_loss(**kw):
    a = dict(logits=view([N, V], lb.BF16), ids=view([N, K], lb.I32), teacher=view([N, K]), scale=1.0, tail=0, loss=view([N])) | kw
    return lb.load().lc_encode_distill_loss(None, None, ref(a["logits"]), ref(a["ids"]), ref(a["teacher"]), a["scale"], a["tail"],
                                            ref(a["loss"]))


def distill_grad(**kw):
    a = dict(logits=view([N, V], lb.BF16), ids=view([N, K], lb.I32), teacher=view([N, K]), scale=1.0, tail=1, d_loss=view([N]),
             loss=view([N]), dlogits=view([N, V], lb.BF16)) | kw
    return lb.load().lc_encode_distill_grad(None, None, ref(a["logits"]), ref(a["ids"]), ref(a["teacher"]), a["scale"], a["tail"],
                                            ref(a["d_loss"]), ref(a["loss"]), ref(a["dlogits"]))


def refused(code, text, want=lb.ERR_INVALID_ARGUMENT):
    assert code == want, (code, said())
    assert text in said(), said()


CALLS = [scores, scores_grad, distill_loss, distill_grad]


@pytest.mark.parametrize("call", CALLS)
def test_good_arguments_reach_the_context(call):
    refused(call(), "null context")


@pytest.mark.parametrize("call", CALLS)
def test_logits(call):
    refused(call(logits=None), "null logits")
    refused(call(logits=view([N, V], lb.F64)), "logits must be f32, f16 or bf16")
    refused(call(logits=view([N, V], lb.I32)), "logits must be f32, f16 or bf16")
    refused(call(logits=view([], lb.F32)), "vocabulary axis")
    refused(call(logits=view([N, 0], lb.F32)), "the vocabulary is empty")
    big = view([1, 4], lb.BF16)
    big.shape[1], big.strides[1] = 1 << 31, 0
    refused(call(logits=big), "exceeds 2^31 - 1")
    short = view([N, V], lb.BF16)
    short.buffer_bytes -= 2
    refused(call(logits=short), "buffer holds")


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("scale", [0.0, -1.0, float("inf"), float("nan")])
def test_scale(call, scale):
    refused(call(scale=scale), "scale must be positive and finite")


def test_scores_operands():
    none = dict(targets=None, logprob=None, entropy=None, stats=None, top_logprobs=None, top_ids=None)
    refused(scores(**none), "no output asked for")
    refused(scores(targets=None), "targets and logprob come together")
    refused(scores(logprob=None), "targets and logprob come together")
    refused(scores(**none | {"entropy": view([N])}), "null context")
    refused(scores(targets=view([N + 1], lb.I32)), "targets must have the logits' leading shape")
    refused(scores(targets=view([N, 1], lb.I32)), "targets must have the logits' leading shape")
    refused(scores(targets=view([N], lb.F32)), "targets must be i32 or u32")
    refused(scores(top_ids=view([N, K], lb.F32)), "top_ids must be i32 or u32")
    for name, shape in (("logprob", [N]), ("entropy", [N]), ("stats", [N, 2]), ("top_logprobs", [N, K])):
        refused(scores(**{name: view(shape, lb.BF16)}), "must be f32")
    refused(scores(stats=view([N, 3])), "stats must have the logits' leading shape and a last axis of 2")
    refused(scores(top_logprobs=view([N, K + 1])), "top_logprobs must have the logits' leading shape and a last axis of 4")
    refused(scores(top_ids=view([N], lb.U32)), "an axis of their own")
    for k, v in ((0, V), (129, 1000), (V + 1, V)):
        refused(scores(logits=view([N, v], lb.F32), top_logprobs=None, top_ids=view([N, k], lb.U32)), "1 to 128 and at most the vocabulary")


def test_scores_overlap():
    x = view([N, V], lb.F32)
    refused(scores(logits=x, logprob=view([N], base=x.data)), "logprob overlaps the logits", lb.ERR_OVERLAP)
    t = view([N], lb.I32)
    refused(scores(targets=t, entropy=view([N], base=t.data)), "overlaps", lb.ERR_OVERLAP)
    lp = view([N])
    refused(scores(logprob=lp, entropy=view([N], base=lp.data, offset=N - 1)), "overlaps", lb.ERR_OVERLAP)
    refused(scores(logprob=lp, entropy=view([N], base=lp.data, offset=N)), "null context")
    refused(scores(logprob=view([N], strides=[0])), "not injective")
    refused(scores(top_logprobs=view([N, K], strides=[2, 1])), "not injective")


def test_scores_grad_operands():
    refused(scores_grad(stats=None), "null stats or dlogits")
    refused(scores_grad(dlogits=None), "null stats or dlogits")
    refused(scores_grad(d_logprob=None, d_entropy=None), "neither d_logprob nor d_entropy")
    refused(scores_grad(targets=None), "d_logprob needs the targets")
    refused(scores_grad(entropy=None), "d_entropy needs the entropy")
    refused(scores_grad(d_entropy=None, entropy=None), "null context")
    refused(scores_grad(d_logprob=None, targets=None), "null context")
    refused(scores_grad(dlogits=view([N, V], lb.F32)), "dlogits must have the logits' type")
    refused(scores_grad(dlogits=view([N, V + 1], lb.BF16)), "dlogits must have the logits' leading shape")
    refused(scores_grad(stats=view([N, 2], lb.F16)), "must be f32")


@pytest.mark.parametrize("call", [scores_grad, distill_grad])
def test_grad_in_place_or_apart(call):
    x = view([N, V], lb.BF16)
    refused(call(logits=x, dlogits=x), "null context")
    refused(call(logits=x, dlogits=view([N, V], lb.BF16, base=x.data)), "null context")
    refused(call(logits=x, dlogits=view([N, V], lb.BF16, base=x.data, offset=1)), "dlogits overlaps the logits", lb.ERR_OVERLAP)
    refused(call(logits=x, dlogits=view([N, V], lb.BF16, base=x.data, strides=[1, N])), "dlogits overlaps the logits", lb.ERR_OVERLAP)
    refused(call(dlogits=view([N, V], lb.BF16, strides=[0, 1])), "not injective")
    # rows that lie upon one another can be read, not written
    same = view([N, V], lb.BF16, strides=[0, 1])
    refused(call(logits=same), "null context")
    refused(call(logits=same, dlogits=same), "not injective")


@pytest.mark.parametrize("call", [distill_loss, distill_grad])
def test_distill_operands(call):
    refused(call(ids=None), "null ids or teacher")
    refused(call(teacher=None), "null ids or teacher")
    refused(call(tail=2), "tail is 0")
    refused(call(tail=-1), "tail is 0")
    refused(call(ids=view([N], lb.I32)), "an axis of their own")
    refused(call(ids=view([N, 257], lb.I32), teacher=view([N, 257])), "at most 256")
    refused(call(ids=view([N, K + 1], lb.I32)), "teacher must have the logits' leading shape and a last axis of 5")
    refused(call(ids=view([N + 1, K], lb.I32)), "ids must have the logits' leading shape")
    refused(call(ids=view([N, K], lb.F32)), "ids must be i32 or u32")
    refused(call(teacher=view([N, K], lb.F64)), "teacher must be f32, f16 or bf16")
    refused(call(teacher=view([N, K], lb.U32)), "teacher must be f32, f16 or bf16")
    refused(call(loss=view([N], lb.BF16)), "must be f32")
    refused(call(loss=view([N + 1])), "loss must have the logits' leading shape")
    refused(call(ids=view([N, 0], lb.I32), teacher=view([N, 0])), "null context")


def test_distill_outputs():
    refused(distill_loss(loss=None), "null loss")
    refused(distill_grad(dlogits=None), "null dlogits")
    refused(distill_grad(loss=None, d_loss=None), "null context")
    refused(distill_grad(d_loss=view([N], lb.F64)), "must be f32")
    refused(distill_grad(dlogits=view([N, V], lb.F16)), "dlogits must have the logits' type")
    d = view([N])
    refused(distill_grad(d_loss=d, loss=view([N], base=d.data)), "overlaps", lb.ERR_OVERLAP)


@pytest.mark.parametrize("call", CALLS)
def test_no_rows_still_checked(call):
    refused(call(logits=view([0, V], lb.BF16)), "leading shape")


def test_tensors_elsewhere():
    """A tensor that does not lie on the context's device never reaches the library."""
    import torch

    class Ctx:
        h, device = None, 0

    x, t = torch.zeros(N, V), torch.zeros(N, dtype=torch.int32)
    n, n2, nk, ids = torch.zeros(N), torch.zeros(N, 2), torch.zeros(N, K), torch.zeros(N, K, dtype=torch.int32)
    for call in (lambda: lb.encode_token_logprobs(Ctx, None, x, t, 1.0, logprob=n),
                 lambda: lb.encode_token_logprobs_backward(Ctx, None, x, t, 1.0, n2, n, x),
                 lambda: lb.encode_distill_loss(Ctx, None, x, ids, nk, 1.0, n),
                 lambda: lb.encode_distill_grad(Ctx, None, x, ids, nk, 1.0, x)):
        with pytest.raises(lb.InvalidArgument, match="not on the context's device"):
            call()
