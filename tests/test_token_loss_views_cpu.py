"""Views that lie elsewhere than the context's device: refused before the library is called, whatever they are made from."""
import pytest
import torch

import linalg_b200 as lb


class Ctx:
    h, device = None, 0


def test_views_elsewhere():
    x, t, n, n2 = torch.zeros(6, 100), torch.zeros(6, dtype=torch.int32), torch.zeros(6), torch.zeros(6, 2)
    ids, z = torch.zeros(6, 4, dtype=torch.int32), torch.zeros(6, 4)
    for of in (lb.View.of, lambda y: lb.permute_view(y, list(range(y.dim()))),
               lambda y: lb.View.raw(y, 0, list(y.shape), list(y.stride()))):
        for call in (lambda: lb.encode_token_logprobs(Ctx, None, of(x), of(t), 1.0, logprob=of(n)),
                     lambda: lb.encode_token_logprobs_backward(Ctx, None, of(x), of(t), 1.0, of(n2), of(n), of(x)),
                     lambda: lb.encode_distill_loss(Ctx, None, of(x), of(ids), of(z), 1.0, of(n)),
                     lambda: lb.encode_distill_grad(Ctx, None, of(x), of(ids), of(z), 1.0, of(x))):
            with pytest.raises(lb.InvalidArgument, match="not on the context's device"):
                call()


def test_views_that_own_nothing_are_the_callers():
    """A view made by hand, with an address and no tensor, is taken at its word; the next check is the library's."""
    v = lb.lc_view()
    v.data, v.buffer_bytes, v.dtype, v.rank = 1 << 20, 4096, lb.F32, 2
    v.shape[0], v.shape[1], v.strides[0], v.strides[1] = 2, 100, 100, 1
    with pytest.raises(lb.InvalidArgument, match="no output asked for"):
        lb.encode_token_logprobs(Ctx, None, lb.View(v, None), None, 1.0)
