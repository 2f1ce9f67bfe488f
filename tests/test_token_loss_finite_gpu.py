"""Scores and losses over a vocabulary on rows with finite masks and large logits, against the plain forms in 64 bits of
test_token_loss_gpu.py, whose tolerances these tests take.

To the gradients' tolerances comes what 2^d loses below FLUSH = 2^-126, where it is 0: a probability is 2^d over a sum that is
at least 1, so a place misses at most FLUSH times what its probability is multiplied by.
"""
import pytest
import torch

import linalg_b200 as lb
from test_token_loss_gpu import TYPES, U, Plain, api, check_scores, close, outputs, plain_distill, randn, teacher_of, tiny

pytestmark = pytest.mark.gpu

FLUSH = 2.0 ** -126


@pytest.fixture(scope="module")
def ctx(gpu):
    return lb.Context(0)


FILLS = {"f32": [-1e9, -1e10, -1e12, -1e15, -1e18, -1e20, -1e30], "bf16": [-1e9, -1e10, -1e12, -1e15, -1e18, -1e20, -1e30],
         "f16": [-1e4, -60000.0]}


def rows_filled(v, dtype):
    """Ordinary rows in which a finite value forbids places: at the front, at the end, scattered, everywhere but in one or in
    five places, or everywhere."""
    base = randn(1, v, seed=15)[0] * 2
    at = torch.arange(v, device="cuda")
    rows = []
    for fill in FILLS[dtype]:
        for gone in (at < v // 2, at >= v // 2, at % 7 != 3, at != v // 3, at % max(1, v // 4) != 0, at >= 0):
            rows.append(torch.where(gone, fill, base))
    return torch.stack(rows).to(TYPES[dtype])


def rows_large(v, dtype):
    """Rows whose logits are all large, close together or not; and rows that step through the places where x scale log2 e
    passes powers of two between 2^18 and 2^26, upwards, downwards and in no order."""
    g = torch.Generator(device="cuda").manual_seed(16)
    wave, spread = torch.rand(v, generator=g, device="cuda"), randn(1, v, seed=17)[0]
    rows = []
    sizes = [1e4, 6e4] if dtype == "f16" else [1e4, 3e5, 1e6, 1e7, 1e8, 1e9, 2e9, 5e9, 1e10, 1e12, 1e15, 1e18, 1e20, 1e24]
    for m in sizes:
        for sign in (1.0, -1.0):
            rows.append(sign * m + spread * 3)
            rows.append(torch.where(wave < 0.3, sign * m, sign * m - m * wave * 1e-3))
    if dtype != "f16":
        for e in (18, 20, 22, 24, 26):
            edge = 2.0 ** e / 1.4426950408889634
            line = torch.linspace(-1, 1, v, device="cuda") * max(16.0, edge * 2.0 ** -18)
            for sign in (1.0, -1.0):
                rows += [sign * edge + line, sign * edge - line, sign * edge + line[torch.randperm(v, generator=g, device="cuda")]]
            rows.append(torch.linspace(-edge * 1.5, edge * 1.5, v, device="cuda"))
    return torch.stack(rows).to(TYPES[dtype])


def held(want, dtype):
    """What the type holds of a value: infinity from half a step beyond its largest number on (f16: 65,520)."""
    info = torch.finfo(dtype)
    return torch.where(want.abs() >= info.max * (1 + info.eps / 4), want.sign() * float("inf"), want)


def check_scores_grad(ctx, x, t, scale, g, h, what):
    """dlogits of one call from its statistics as they are given."""
    n, v = x.shape
    out = outputs(n)
    api.token_logprobs(ctx, x, t, scale, **out)
    dx = torch.full_like(x, 7.0)
    more = {} if h is None else {"entropy": out["entropy"], "d_entropy": h}
    api.token_logprobs_backward(ctx, x, t, scale, out["stats"], g, dx, **more)
    ref = Plain(x, scale)
    total, ent, gg = out["stats"][:, 1:].double(), out["entropy"].double()[:, None], g.double()[:, None]
    hh = torch.zeros_like(gg) if h is None else h.double()[:, None]
    lp = ref.d - total
    p = lp.exp()
    hot = torch.zeros_like(p).scatter_(1, t.long()[:, None], 1.0)
    want = ref.s * (gg * (hot - p) - hh * torch.where(p == 0, 0.0, p * (lp + ent)))
    # p as it is, and what flushing may take from it; beyond |d| = 130 nothing is left of either, so the factors are held there
    far, near = ref.absd.clamp(max=1e3), lp.abs().clamp(max=1e3)
    weight = gg.abs() + hh.abs() * (near + ent.abs() + total.abs() + far)
    tol = ref.s * U * p * weight * (3 * far + 24) + 4 * U * ref.s * gg.abs() * hot + ref.s * FLUSH * weight
    # d = x c2 - mc with mc = m c2 (c2 = s log2 e) as it rounds, so d at the largest logit is off = m c2 - mc and not 0,
    # |off| <= U |m c2|.  The row's constant takes bt off away again (|bt| <= s |h| p there), as it rounds: off by U |bt off|,
    # and by as much again in its own sum.  So even where everything else is 0 there may be 2 U |bt off| <= 2 U^2 s |h| |m c2|;
    # d is taken that way up to |m c2| = 2^20 alone.
    tol = tol + 2 * U * U * ref.s * hh.abs() * p * (ref.m.abs()[:, None] * (ref.s * 1.4427)).clamp(max=2.0 ** 20)
    close(dx, held(want, x.dtype), tol + want.abs() * (torch.finfo(x.dtype).eps / 2) + tiny(x.dtype), what + " dlogits")


def check_distill(ctx, x, ids, z, scale, tail, d_loss):
    """Loss alone, and loss and gradient of one call."""
    want_loss, tol_loss, want, tol = plain_distill(x, ids, z, scale, tail, d_loss)
    # outside the list 2^d is measured from the largest logit there and multiplied by sum P e^lead / S - r / St, |..| <= 2; in
    # the list q comes times sum P + r <= 1 (a little more by the rounding of P)
    tol = tol + FLUSH * 2 * scale * d_loss.double().abs()[:, None]
    only, loss, dx = torch.full_like(d_loss, -7.0), torch.full_like(d_loss, -7.0), torch.full_like(x, 7.0)
    api.distill_loss(ctx, x, ids, z, scale, only, tail=tail)
    close(only, want_loss, tol_loss, "loss alone")
    api.distill_grad(ctx, x, ids, z, scale, dx, d_loss=d_loss, loss=loss, tail=tail)
    close(loss, want_loss, tol_loss, "loss")
    close(dx, held(want, x.dtype), tol, "distill dlogits")


def check_far(ctx, x, scale, k=20):
    """All four operators on the rows."""
    n, v = x.shape
    t = torch.arange(n, device="cuda").int() * 7919 % v
    g, h = randn(n, seed=1), randn(n, seed=2)
    check_scores(ctx, x, t, scale, min(k, v))
    check_scores_grad(ctx, x, t, scale, g, h, "both")
    check_scores_grad(ctx, x, t, scale, g, None, "score")
    for tail in (False, True):
        # with a tail the list leaves a tenth: next to nothing, times the distance of a filled place, would be all rounding
        ids, z = teacher_of(x * scale, min(k, v), tail)
        check_distill(ctx, x, ids, z - 0.1, scale, tail, d_loss=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [9, 700, 20011, 200003])
def test_finite_masks(ctx, dtype, v):
    check_far(ctx, rows_filled(v, dtype), 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [9, 700, 20011, 200003])
def test_large_logits(ctx, dtype, v):
    check_far(ctx, rows_large(v, dtype), 1.0)


@pytest.mark.parametrize("scale", [0.01, 0.7, 40.0, 5000.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_far_scales(ctx, dtype, scale):
    check_far(ctx, torch.cat([rows_filled(9001, dtype), rows_large(9001, dtype)]), scale)


def test_finite_masks_strided(ctx):
    """A vocabulary that is not the unit axis gives the same."""
    x = torch.cat([rows_filled(3001, "f32"), rows_large(3001, "f32")])
    check_far(ctx, x.t().contiguous().t(), 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [9, 20011])
def test_largest_scale(ctx, dtype, v):
    """Only the largest logits of a row are left; every other place has weight and gradient 0."""
    x = (randn(8, v, seed=3) * 3).to(TYPES[dtype])
    x[1, :5] = x.max() + 1
    x[2] = 0.5
    x[3, 3:] = -1e4
    check_far(ctx, x, 2.0 ** 100)
