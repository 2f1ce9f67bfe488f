"""Scores and losses over a vocabulary (token_logprobs, distill and their gradients) on the device, against plain
implementations in 64 bits.

Tolerances count roundings.  U = 2^-24 is half a step of f32.  d = scale (x - m) takes a subtraction, a rounded constant and
a product (3 U |d|), and 2^d is within 4 U of its value, so one term of a sum is off by (3 |d| + 4) U of itself; a sum over
V places passes each term through at most CHAIN(V) roundings.  What is stored in 16 bits is off by half a step more.
"""
import math

import pytest
import torch

import linalg_b200 as lb

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF = float("inf")


def chain(v):
    """Roundings, in units of U, that a term of a row's sum passes.  A row is spread over 256 threads or over so many that
    none has more than 32 places; each step of a thread's sum may scale it (2^u within 4 U, a product) and adds to it; the
    merges of threads and blocks, at most 5 + 5 + 5 levels, take 10 each."""
    return 8 * max(math.ceil(v / 256), 13) + 152


class _Waits:
    """The waiting forms run on the context's own stream: what torch still does to their operands is waited for first."""

    def __getattr__(self, name):
        def call(*args, **kwargs):
            torch.cuda.synchronize()
            return getattr(lb, name)(*args, **kwargs)
        return call


api = _Waits()


@pytest.fixture(scope="module")
def ctx(gpu):
    return lb.Context(0)


def randn(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


def close(got, want, tol, what):
    got = got.double()
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, want.sign() * INF, want)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    ok = same | ((got - want).abs() <= tol)
    if not bool(ok.all()):
        at = (~ok).nonzero()[0].tolist()
        raise AssertionError(f"{what}{at}: {got[tuple(at)].item()} against {want[tuple(at)].item()}, {int((~ok).sum())} places off")


# ---- plain forms in 64 bits ------------------------------------------------------------------------------------------


class Plain:
    """Softmax of scale * x over the last axis, of rows [n, V]."""

    def __init__(self, x, scale):
        self.x = x.double()
        # the library's scale is an f32
        self.s = s = torch.tensor(scale, dtype=torch.float32).double().item()
        n, v = x.shape
        self.v = v
        self.m = self.x.amax(1)
        base = torch.where(self.m == -INF, 0.0, self.m)[:, None]
        self.d = (self.x - base) * s
        self.e = self.d.exp()
        self.sum = self.e.sum(1)
        self.total = self.sum.log()
        masked = (self.x == -INF) & ~self.total.isnan()[:, None]
        self.lp = torch.where(masked, -INF, self.d - self.total[:, None])
        self.p = torch.where(self.sum[:, None] == 0, 0.0, self.e / self.sum[:, None])
        dd = torch.where(masked, 0.0, self.d)
        self.absd = dd.abs()
        self.entropy = torch.where(self.m == -INF, 0.0, -(self.p * torch.where(masked, 0.0, self.lp)).sum(1))
        # weighted mean of |d|, and of |d|^2: how far the terms' own errors move the sums
        w1 = torch.nan_to_num((self.p * self.absd).sum(1))
        w2 = torch.nan_to_num((self.p * self.absd ** 2).sum(1))
        c = chain(v)
        self.tol_total = U * (3 * w1 + 4 + c + 2 * torch.nan_to_num(self.total, 0, 0, 0).abs())
        self.tol_lp = self.tol_total[:, None] + 8 * U * self.absd + 2 * U * torch.nan_to_num(self.lp, 0, 0, 0).abs()
        self.tol_entropy = self.tol_total + U * (3 * w2 + (8 + 2 * c) * w1) + 4 * U * torch.nan_to_num(self.total, 0, 0, 0).abs()

    def best(self, k):
        return torch.sort(self.x, dim=1, descending=True, stable=True).indices[:, :k]


def outputs(n, k=0):
    e = lambda *s, **kw: torch.full(s, -7, device="cuda", **kw)  # noqa: E731
    out = {"logprob": e(n, dtype=torch.float32), "entropy": e(n, dtype=torch.float32), "stats": e(n, 2, dtype=torch.float32)}
    if k:
        out |= {"top_logprobs": e(n, k, dtype=torch.float32), "top_ids": e(n, k, dtype=torch.int32)}
    return out


def check_scores(ctx, x, t, scale, k, what=""):
    """All outputs of one call against the plain form."""
    out = outputs(x.shape[0], k)
    api.token_logprobs(ctx, x, t, scale, **out)
    ref = Plain(x, scale)
    has = (t >= 0) & (t < x.shape[1])
    at = t.long().clamp(0, x.shape[1] - 1)[:, None]
    close(out["logprob"], torch.where(has, ref.lp.gather(1, at)[:, 0], 0.0), ref.tol_lp.gather(1, at)[:, 0], what + " logprob")
    close(out["entropy"], ref.entropy, ref.tol_entropy, what + " entropy")
    close(out["stats"][:, 0], ref.m, 0.0, what + " largest")
    close(out["stats"][:, 1], ref.total, ref.tol_total, what + " total")
    if k:
        best = ref.best(k)
        assert torch.equal(out["top_ids"].long(), best), what + " top_ids"
        close(out["top_logprobs"], ref.lp.gather(1, best), ref.tol_lp.gather(1, best), what + " top_logprobs")
    return out


def tokens(n, v, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    t[::5] = -1
    return t.int()


# ---- scores ------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k", [(3, 1, 1), (5, 2, 2), (1, 7, 3), (4, 8, 8), (130, 33, 5), (7, 255, 20), (9, 1000, 64),
                                   (2, 4099, 128), (33, 8192, 20), (1, 50001, 20), (300, 12345, 1), (2, 131075, 64),
                                   (3, 400003, 20)])
def test_scores(ctx, dtype, n, v, k):
    x = (randn(n, v, seed=n + v) * 3 + randn(n, 1, seed=v) * 10).to(TYPES[dtype])
    check_scores(ctx, x, tokens(n, v), 1.0, k)


@pytest.mark.parametrize("dtype,n,v,k", [("bf16", 301, 150001, 20), ("f32", 300, 140003, 64), ("f16", 1, 4300001, 128)])
def test_scores_long(ctx, dtype, n, v, k):
    """Rows so long that several steps of a block share what it notes for the alternatives."""
    x = (randn(n, v, seed=3) * 3).to(TYPES[dtype])
    x[0, : v - 4000] = -INF  # the best places side by side
    check_scores(ctx, x, tokens(n, v), 1.0, k)


@pytest.mark.parametrize("scale", [1e-6, 1e-3, 0.7, 1.0, 3.0, 200.0, 1e5])
def test_scores_scale(ctx, scale):
    x = randn(6, 5003, seed=2) * 4
    check_scores(ctx, x, tokens(6, 5003), scale, 7)


def test_scores_without_some_outputs(ctx):
    x = randn(5, 2049, seed=3)
    t = tokens(5, 2049)
    full = check_scores(ctx, x, t, 1.0, 9)
    for names in (["logprob"], ["entropy"], ["stats"], ["top_ids"], ["top_logprobs"], ["logprob", "top_ids"], ["entropy", "stats"]):
        out = {k: torch.empty_like(full[k]) for k in names}
        api.token_logprobs(ctx, x, t if "logprob" in names else None, 1.0, **out)
        for k in names:
            # the entropy's sum is the only one that may be left out, and nothing else goes by it
            assert torch.equal(out[k], full[k]), k


def rows_of_trouble(v, dtype):
    """Rows with masks that leave little or nothing, ties, extremes, NaN and infinities."""
    low = torch.finfo(TYPES[dtype]).min
    base = randn(1, v, seed=5)[0] * 2
    rows = [base.clone() for _ in range(16)]
    rows[0][:] = -INF                               # nothing left
    rows[1][:] = low                                # the type's lowest value throughout: even
    rows[2][:] = -INF
    rows[2][v // 2] = 1.5                           # one place left
    rows[3][torch.arange(v, device="cuda") % 3 != 0] = -INF
    rows[4][v // 3:] = low                          # masked with the lowest value
    rows[5][:] = 0.25                               # all equal
    rows[6] = torch.linspace(-5, 5, v, device="cuda")
    rows[7] = torch.linspace(5, -5, v, device="cuda")
    rows[8] = (base * 2).round()                    # many ties
    rows[9] = torch.where(torch.arange(v, device="cuda") % 2 == 0, 0.0, -0.0)
    rows[10][v // 2] = float("nan")
    rows[11][v // 4] = INF
    rows[12] = 100 + base * 1e-3                    # a narrow band
    rows[13][: v - v // 4] = -INF                   # only the end left
    rows[14][:] = -INF
    rows[14][: min(v, 3)] = 0.0
    rows[15][v - 1] = 60.0                          # nearly certain
    return torch.stack(rows).to(TYPES[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v,k", [(5, 5), (64, 20), (4097, 20), (20000, 64), (70001, 128)])
def test_scores_trouble(ctx, dtype, v, k):
    x = rows_of_trouble(v, dtype)
    t = torch.arange(16, device="cuda").int() * 7919 % v
    check_scores(ctx, x, t, 1.0, k)
    check_scores(ctx, x[2:4], t[2:4], 0.5, k)


def test_scores_extreme_range(ctx):
    """Differences that overflow f32 leave the far places without weight, not the row without a sum."""
    x = torch.tensor([[3e38, -3e38, 2.9e38, 0.0], [-3.3e38, -3.3e38, -INF, -3.4e38], [1e-40, 0.0, -1e-40, 2e-40]], device="cuda")
    check_scores(ctx, x, torch.tensor([0, 1, 2], device="cuda").int(), 1.0, 4)
    check_scores(ctx, x, torch.tensor([1, 0, 3], device="cuda").int(), 50.0, 4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,start", [(0, 1), (1, 0), (5, 3), (8, 8), (13, 7)])
def test_scores_alignment(ctx, dtype, pad, start):
    """Rows that start anywhere and step by any length."""
    n, v = 6, 3001
    buf = torch.full((n * (v + pad) + start + 9,), 77.0, device="cuda").to(TYPES[dtype])
    x = buf[start:start + n * (v + pad)].view(n, v + pad)[:, :v]
    x.copy_(randn(n, v, seed=pad) * 3)
    check_scores(ctx, x, tokens(n, v), 1.0, 20)


def test_scores_strides(ctx):
    """Leading axes in any order, a vocabulary that is not the unit axis, repeated rows, and strided outputs."""
    v, k = 517, 6
    full = randn(3, 4, v, 2, seed=8) * 3
    t = tokens(12, v).view(3, 4)
    for x in (full[..., 0], full[..., 1].transpose(0, 1), full.permute(3, 1, 0, 2)[1], randn(1, 1, v).expand(3, 4, v),
              randn(v, 3, 4).permute(1, 2, 0)):
        a, b = x.shape[:2]
        tt = t if (a, b) == (3, 4) else t.t()
        lp = torch.zeros(b, a, 3, device="cuda")[..., 1].t()
        ids = torch.zeros(a, b, k, 2, dtype=torch.int32, device="cuda")[..., 1]
        top = torch.zeros(k, a, b, device="cuda").permute(1, 2, 0)
        stats = torch.zeros(2, b, a, device="cuda").permute(2, 1, 0)
        api.token_logprobs(ctx, x, tt, 1.0, logprob=lp, stats=stats, top_logprobs=top, top_ids=ids)
        want = check_scores(ctx, x.reshape(a * b, v).contiguous(), tt.reshape(-1).contiguous(), 1.0, k)
        tol = Plain(x.reshape(a * b, v), 1.0).tol_lp.amax().item() * 2
        close(lp.reshape(-1), want["logprob"].double(), tol, "logprob")
        close(top.reshape(-1, k), want["top_logprobs"].double(), tol, "top")
        close(stats.reshape(-1, 2), want["stats"].double(), tol, "stats")
        assert torch.equal(ids.reshape(-1, k), want["top_ids"])


def test_scores_unsigned_tokens_and_one_row(ctx):
    v = 999
    x = randn(v, seed=4)
    t = torch.tensor([998], device="cuda").int()
    lp, ids = torch.empty((), device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda")
    tv = lb.View.raw(t, 0, [], [], lb.U32)
    iv = lb.View.raw(ids, 0, [4], [1], lb.U32)
    api.token_logprobs(ctx, x, tv, 1.0, logprob=lp, top_ids=iv)
    ref = Plain(x[None], 1.0)
    close(lp[None], ref.lp[:, 998], ref.tol_lp[:, 998], "logprob")
    assert torch.equal(ids.long(), ref.best(4)[0])


def test_no_rows(ctx):
    x = torch.empty(0, 100, device="cuda")
    api.token_logprobs(ctx, x, torch.empty(0, dtype=torch.int32, device="cuda"), 1.0, logprob=torch.empty(0, device="cuda"))
    api.distill_grad(ctx, x, torch.empty(0, 4, dtype=torch.int32, device="cuda"), torch.empty(0, 4, device="cuda"), 1.0,
                    torch.empty(0, 100, device="cuda"))


def test_rows_past_32_bits(ctx):
    """Rows whose elements lie beyond 2^32, reached by a row stride, forward and backward."""
    v, step = 1000, 2_200_000_001
    buf = torch.empty(2 * step + v, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((3, v), (step, 1))
    x.copy_(randn(3, v, seed=6) * 3)
    t = torch.tensor([5, 999, 0], device="cuda").int()
    out = check_scores(ctx, x, t, 1.0, 5)
    dx = torch.empty(3, v, dtype=torch.bfloat16, device="cuda")
    g = torch.ones(3, device="cuda")
    api.token_logprobs_backward(ctx, x, t, 1.0, out["stats"], g, dx)
    want = torch.empty_like(dx)
    api.token_logprobs_backward(ctx, x.contiguous(), t, 1.0, out["stats"], g, want)
    assert torch.equal(dx, want)
    api.token_logprobs_backward(ctx, x, t, 1.0, out["stats"], g, x)
    assert torch.equal(x, want)


# ---- gradient of the scores --------------------------------------------------------------------------------------------


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 1e-37


def check_scores_grad(ctx, x, t, scale, g, h, what="", in_place=False):
    n, v = x.shape
    out = outputs(n)
    api.token_logprobs(ctx, x, t, scale, **out)
    dx = x.clone() if in_place else torch.full_like(x, 7.0)
    api.token_logprobs_backward(ctx, dx if in_place else x, t, scale, out["stats"], g, dx, entropy=out["entropy"] if h is not None else None,
                               d_entropy=h)
    ref = Plain(x, scale)
    # from the statistics as they are given
    total = out["stats"][:, 1].double()[:, None]
    dead = (ref.m == -INF)[:, None]
    lp = torch.where((x == -INF) & ~dead, -INF, ref.d - total)
    p = torch.where(dead, 0.0, lp.exp())
    lp = torch.where(p == 0, 0.0, lp)
    has = ((t >= 0) & (t < v))[:, None] & ~dead
    gg = torch.where((t >= 0) & (t < v), g.double() if g is not None else 0.0, 0.0)[:, None]
    hh = (h.double() if h is not None else torch.zeros(n, device="cuda").double())[:, None]
    ent = out["entropy"].double()[:, None]
    hot = torch.zeros_like(p).scatter_(1, t.long().clamp(0, v - 1)[:, None], 1.0) * has
    want = ref.s * (torch.where(dead, 0.0, gg) * (hot - p) - hh * p * (lp + ent))
    big = p * (gg.abs() + hh.abs() * (lp.abs() + ent.abs() + total.nan_to_num(0, 0, 0).abs() + ref.absd))
    tol = ref.s * U * big * (3 * ref.absd + 24) + 4 * U * ref.s * gg.abs() * hot
    # d = x c2 - mc with mc = m c2 (c2 = s log2 e) as it rounds, so d at the largest logit is off = m c2 - mc and not 0,
    # |off| <= U |m c2|.  The row's constant takes bt off away again (|bt| <= s |h| p there), as it rounds: off by U |bt off|,
    # and by as much again in its own sum.  So even where everything else is 0 there may be 2 U |bt off| <= 2 U^2 s |h| |m c2|.
    m = torch.where(ref.m.isfinite(), ref.m, 0.0).abs()[:, None]
    tol = tol + 2 * U * U * ref.s * hh.abs() * p * m * (ref.s * 1.4427)
    tol = tol + want.abs() * (torch.finfo(x.dtype).eps / 2) + tiny(x.dtype)
    close(dx, want, tol, what + " dlogits")
    return dx


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v", [(3, 1), (5, 2), (1, 7), (130, 33), (7, 255), (9, 1000), (2, 4099), (33, 8192), (1, 50001),
                                 (40, 12345), (2, 131075)])
def test_scores_grad(ctx, dtype, n, v):
    x = (randn(n, v, seed=n + v) * 3 + randn(n, 1, seed=v) * 10).to(TYPES[dtype])
    t = tokens(n, v)
    g, h = randn(n, seed=11), randn(n, seed=12)
    check_scores_grad(ctx, x, t, 1.0, g, None, "score")
    check_scores_grad(ctx, x, t, 0.6, None, h, "entropy")
    check_scores_grad(ctx, x, t, 1.7, g, h, "both", in_place=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [5, 64, 4097, 20000])
def test_scores_grad_trouble(ctx, dtype, v):
    x = rows_of_trouble(v, dtype)
    t = torch.arange(16, device="cuda").int() * 7919 % v
    check_scores_grad(ctx, x, t, 1.0, randn(16, seed=1), randn(16, seed=2))


def test_scores_grad_against_differences():
    """The formula above against central differences of the plain form, in 64 bits."""
    x = (randn(2, 9, seed=3) * 2).double()
    t = torch.tensor([4, 0], device="cuda")
    g, h, s = torch.tensor([0.7, -1.3], device="cuda").double(), torch.tensor([0.4, 2.0], device="cuda").double(), 1.0

    def f(y):
        r = Plain(y, s)
        return (g * r.lp.gather(1, t[:, None])[:, 0] + h * r.entropy).sum()

    r = Plain(x, s)
    hot = torch.zeros_like(x).scatter_(1, t[:, None], 1.0)
    want = g[:, None] * (hot - r.p) - h[:, None] * r.p * (r.lp + r.entropy[:, None])
    for i in range(2):
        for j in range(9):
            e = torch.zeros_like(x)
            e[i, j] = 1e-5
            assert abs(((f(x + e) - f(x - e)) / 2e-5 - want[i, j]).item()) < 1e-8


def test_scores_grad_strides(ctx):
    v = 517
    full = randn(3, 4, v, 2, seed=8) * 3
    t = tokens(12, v).view(3, 4)
    x = full[..., 1]
    out = {"stats": torch.zeros(2, 3, 4, device="cuda").permute(1, 2, 0), "entropy": torch.zeros(4, 3, device="cuda").t()}
    api.token_logprobs(ctx, x, None, 1.0, **out)
    g, h = randn(4, 3, seed=2).t(), randn(1, 1, seed=3).expand(3, 4)
    dx = torch.full((v, 4, 3), 9.0, device="cuda").permute(2, 1, 0)
    api.token_logprobs_backward(ctx, x, t, 1.0, out["stats"], g, dx, entropy=out["entropy"], d_entropy=h)
    want = torch.empty(12, v, device="cuda")
    flat = x.reshape(12, v).contiguous()
    api.token_logprobs_backward(ctx, flat, t.reshape(-1), 1.0, out["stats"].reshape(12, 2).contiguous(), g.reshape(-1).contiguous(), want,
                               entropy=out["entropy"].reshape(-1).contiguous(), d_entropy=h.reshape(-1).contiguous())
    assert torch.equal(dx.reshape(12, v), want)
    # in place where the vocabulary is not the unit axis; what lies between stays
    other = full[..., 0].clone()
    api.token_logprobs_backward(ctx, x, t, 1.0, out["stats"], g, x, entropy=out["entropy"], d_entropy=h)
    assert torch.equal(x.reshape(12, v), want) and torch.equal(full[..., 0], other)


@pytest.mark.parametrize("dtype", TYPES)
def test_grad_leaves_the_padding(ctx, dtype):
    """Columns behind the vocabulary stay as they were, at every alignment of a row."""
    n, v, pad = 5, 1003, 9
    x = (randn(n, v, seed=1) * 2).to(TYPES[dtype])
    buf = torch.full((n, v + pad), 5.0, device="cuda", dtype=TYPES[dtype])
    t, g = tokens(n, v), randn(n, seed=2)
    stats = torch.empty(n, 2, device="cuda")
    api.token_logprobs(ctx, x, None, 1.0, stats=stats)
    api.token_logprobs_backward(ctx, x, t, 1.0, stats, g, buf[:, :v])
    assert bool((buf[:, v:] == 5).all())
    ids, z = torch.sort(x.float(), dim=1, descending=True).indices[:, :6].int(), torch.zeros(n, 6, device="cuda")
    buf.fill_(5)
    api.distill_grad(ctx, x, ids, z, 1.0, buf[:, :v])
    assert bool((buf[:, v:] == 5).all())


# ---- distillation ------------------------------------------------------------------------------------------------------


def plain_distill(x, ids, z, scale, tail, d_loss):
    """Loss and gradient in 64 bits with their tolerances, one row after the other."""
    ref = Plain(x, scale)
    n, v = x.shape
    s = ref.s
    loss, dx, tol_loss, tol_dx = [], [], [], []
    c = chain(v)
    for i in range(n):
        seen, ks = set(), []
        for k, j in enumerate(ids[i].tolist()):
            if 0 <= j < v and j not in seen:
                seen.add(j)
                ks.append(k)
        at = ids[i].long()[ks]
        zz = z[i].double()[ks]
        if tail:
            logp = zz
            P = logp.exp()
            r = max(0.0, 1.0 - P.sum().item()) if len(ks) else 1.0
        else:
            top = zz.max() if len(ks) else torch.tensor(0.0)
            y = (zz - (0.0 if top == -INF else top)) * s
            tot = y.exp().sum()
            logp = y - tot.log()
            P = torch.where(tot == 0, 0.0, y.exp() / tot)
            r = 0.0
        out = torch.ones(v, dtype=torch.bool, device=x.device)
        out[at] = False
        xt = ref.x[i][out]
        mt = xt.max() if xt.numel() else torch.tensor(-INF, device=x.device).double()
        ut = ((xt - (0.0 if mt == -INF else mt)) * s).exp()
        St = ut.sum()
        if St == 0:
            r = 0.0
        lead = s * (mt - ref.m[i]) if St > 0 else torch.tensor(0.0).double()
        total = P.sum() + r
        lq = ref.lp[i][at]
        terms = torch.where(P > 0, P * (logp - lq), 0.0)
        tail_term = r * (math.log(r) - (St.log() + lead - ref.total[i])) if r > 0 else 0.0
        loss.append(terms.sum() + tail_term)
        tl = (P * (ref.tol_lp[i][at] + 4 * U * torch.nan_to_num(logp, 0, 0, 0).abs() + 2 * U * torch.nan_to_num(lq, 0, 0, 0).abs())).sum()
        far = (ref.p[i] * ref.absd[i]).sum().nan_to_num()
        tl = tl + r * U * (2 * c + 32 + 6 * far + 4 * abs(float(lead)) + 4 * torch.nan_to_num(ref.total[i], 0, 0, 0).abs() + 4 * (abs(math.log(r)) if r > 0 else 0))
        tol_loss.append(tl + U * torch.nan_to_num(loss[-1], 0, 0, 0).abs() * 2)
        w = (float(d_loss[i]) if d_loss is not None else 1.0) * s
        row = torch.zeros(v, device=x.device).double()
        tol = torch.zeros(v, device=x.device).double()
        dead = ref.m[i] == -INF
        if not dead:
            q = ref.p[i]
            share = torch.zeros(v, device=x.device).double()
            if r > 0:
                share[out] = r * ut / St
            row = total * q - share
            row[at] -= P
            row *= w
            tol = abs(w) * U * (total * q + share) * (6 * ref.absd[i] + 3 * abs(float(lead)) + c + 32)
            tol[at] += abs(w) * 4 * U * P
        dx.append(row)
        tol_dx.append(tol)
    dx, tol_dx = torch.stack(dx), torch.stack(tol_dx)
    tol_dx = tol_dx + dx.abs() * (torch.finfo(x.dtype).eps / 2) + tiny(x.dtype)
    return torch.stack(loss), torch.stack(tol_loss), dx, tol_dx


def check_distill(ctx, x, ids, z, scale, tail, d_loss=None, what="", in_place=False):
    n, v = x.shape
    want_loss, tol_loss, want, tol = plain_distill(x, ids, z, scale, tail, d_loss)
    only = torch.full((n,), -7.0, device="cuda")
    api.distill_loss(ctx, x, ids, z, scale, only, tail=tail)
    close(only, want_loss, tol_loss, what + " loss alone")
    loss = torch.full((n,), -7.0, device="cuda")
    dx = x.clone() if in_place else torch.full_like(x, 7.0)
    api.distill_grad(ctx, dx if in_place else x, ids, z, scale, dx, d_loss=d_loss, loss=loss, tail=tail)
    close(loss, want_loss, tol_loss, what + " loss")
    close(dx, want, tol, what + " dlogits")
    again = torch.empty_like(dx)
    if not in_place:
        api.distill_grad(ctx, x, ids, z, scale, again, d_loss=d_loss, tail=tail)
        assert torch.equal(again, dx)
    return dx


def teacher_of(x, k, tail, seed=0):
    """A teacher near the student: its k best places with their log probabilities, or any values."""
    y = x.float().nan_to_num(0, 0, -50) + randn(*x.shape, seed=seed)
    lp = torch.log_softmax(y.double(), 1)
    best, ids = lp.topk(k, 1)
    return ids.int(), (best if tail else best * 2 + 5).float()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k", [(2, 1, 1), (3, 5, 2), (2, 9, 9), (20, 40, 7), (4, 257, 64), (3, 2500, 256), (5, 8192, 16),
                                   (2, 33001, 32), (1, 131075, 64), (2, 300007, 20)])
def test_distill(ctx, dtype, n, v, k, tail):
    x = (randn(n, v, seed=n + v) * 3 + randn(n, 1, seed=v) * 10).to(TYPES[dtype])
    ids, z = teacher_of(x, k, tail)
    check_distill(ctx, x, ids, z, 1.0, tail, d_loss=randn(n, seed=4))
    check_distill(ctx, x, ids, z, 0.5, tail, in_place=True)


@pytest.mark.parametrize("dtype,v,k,pad,dpad", [("bf16", 16384, 16, 0, 0), ("bf16", 50001, 40, 63, 0), ("f16", 33003, 256, 0, 5),
                                                ("f32", 40001, 64, 3, 0), ("f32", 8199, 1, 0, 0), ("bf16", 131075, 33, 5, 5)])
def test_distill_many_rows(ctx, dtype, v, k, pad, dpad):
    """More rows than the device takes at once, with lists of every length, masked rows among them, and rows of the logits
    and of the gradient that start at different places within 16 bytes."""
    n = 331
    buf = torch.zeros(n, v + pad, device="cuda", dtype=TYPES[dtype])
    x = buf[:, :v]
    x.copy_(randn(n, v, seed=v) * 3 + randn(n, 1, seed=k) * 10)
    x[5] = -INF
    x[7, 100:] = -INF
    x[9] = torch.finfo(TYPES[dtype]).min
    ids, z = teacher_of(x, k, True)
    ids[::3, k // 2:] = -1
    ids[11] = -1
    if k > 4:
        ids[13, 2] = ids[13, 0]
        ids[14, 0], ids[14, 1] = 0, v - 1
        z[14, :2] = -3.0
    d = randn(n, seed=4)
    want_loss, tol_loss, want, tol = plain_distill(x, ids, z, 1.0, True, d)
    out = torch.full((n, v + dpad), 5.0, device="cuda", dtype=TYPES[dtype])
    loss = torch.empty(n, device="cuda")
    for _ in range(2):
        api.distill_grad(ctx, x, ids, z, 1.0, out[:, :v], d_loss=d, loss=loss, tail=True)
        close(loss, want_loss, tol_loss, "loss")
        close(out[:, :v], want, tol, "dlogits")
        assert bool((out[:, v:] == 5).all())
    first = out[:, :v].clone()
    api.distill_grad(ctx, x, ids, z, 1.0, x, d_loss=d, tail=True)
    close(x, want, tol, "in place")
    if pad == dpad:
        assert torch.equal(x, first)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_longest(ctx, tail):
    """A vocabulary whose places' bits do not fit in a cluster's shared memory."""
    x = (randn(2, 4300001, seed=3) * 3).bfloat16()
    ids, z = teacher_of(x, 40, tail)
    check_distill(ctx, x, ids, z, 1.0, tail, d_loss=randn(2, seed=4))


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("ttype", TYPES)
def test_distill_padding_and_repeats(ctx, ttype, tail):
    """Entries outside the vocabulary are padding, of an index named twice the first entry stands, and a row may have no
    entry at all."""
    v, k = 1200, 24
    x = randn(6, v, seed=9) * 3
    ids, z = teacher_of(x, k, tail)
    z = z.to(TYPES[ttype])
    ids[0, 5:] = -1
    ids[1] = -1
    ids[2, 3:9] = ids[2, 1]
    ids[3, 0] = v
    ids[3, 1] = 2 ** 31 - 1
    ids[4, ::2] = ids[4, 1::2]
    check_distill(ctx, x, ids, z, 1.0, tail, d_loss=randn(6, seed=3))


@pytest.mark.parametrize("tail", [False, True])
def test_distill_empty_list(ctx, tail):
    x = randn(3, 700, seed=1)
    ids, z = torch.empty(3, 0, dtype=torch.int32, device="cuda"), torch.empty(3, 0, device="cuda")
    check_distill(ctx, x, ids, z, 1.0, tail)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v,k", [(6, 4), (300, 32), (5001, 64)])
def test_distill_trouble(ctx, dtype, v, k, tail):
    """Masked rows, extremes, NaN and infinities in the student; entries that say nothing in the teacher."""
    x = rows_of_trouble(v, dtype)
    keep = torch.ones(16, dtype=torch.bool, device="cuda")
    keep[10] = keep[11] = False  # a NaN or an infinity makes its row NaN, below
    ids, z = teacher_of(x, k, tail)
    check_distill(ctx, x[keep].contiguous(), ids[keep].contiguous(), z[keep].contiguous(), 1.0, tail, d_loss=randn(14, seed=3))
    z[:, ::3] = -INF
    check_distill(ctx, x[keep].contiguous(), ids[keep].contiguous(), z[keep].contiguous(), 1.0, tail)
    z[4] = -INF
    check_distill(ctx, x[4:5], ids[4:5], z[4:5], 1.0, tail)
    loss, dx = torch.zeros(2, device="cuda"), torch.zeros(2, v, device="cuda", dtype=x.dtype)
    api.distill_grad(ctx, x[10:12], ids[10:12], z[10:12], 1.0, dx, loss=loss, tail=tail)
    assert bool(loss.isnan().all()) and bool(dx[0].isnan().any()) and bool(dx[1].isnan().any())


def test_distill_far_tail(ctx):
    """A student that leaves next to nothing, or less than f32 can hold, outside the list still feels the tail."""
    v, k = 900, 8
    x = randn(5, v, seed=2)
    ids, z = teacher_of(x, k, True)
    for i, gap in enumerate([30.0, 80.0, 100.0, 300.0, 2000.0]):
        x[i].scatter_add_(0, ids[i].long(), torch.full((k,), gap, device="cuda"))
    check_distill(ctx, x, ids, z, 1.0, True)


def test_distill_whole_vocabulary(ctx):
    """A list that names every place leaves no tail, whatever the teacher's sum rounds to."""
    x = randn(4, 200, seed=2) * 2
    ids, z = teacher_of(x, 200, True)
    check_distill(ctx, x, ids, z, 1.0, True)


def test_distill_strides(ctx):
    v, k = 640, 12
    full = randn(2, 5, v, 2, seed=8) * 2
    x = full[..., 1]
    flat = x.reshape(10, v).contiguous()
    ids, z = teacher_of(flat, k, True)
    want_loss, want = torch.empty(10, device="cuda"), torch.empty_like(flat)
    d = randn(10, seed=3)
    api.distill_grad(ctx, flat, ids, z, 1.0, want, d_loss=d, loss=want_loss, tail=True)
    ids2 = torch.empty(k, 5, 2, dtype=torch.int32, device="cuda").permute(2, 1, 0).copy_(ids.view(2, 5, k))
    z2 = torch.empty(5, 2, k, device="cuda").transpose(0, 1).copy_(z.view(2, 5, k))
    loss = torch.empty(5, 2, device="cuda").t()
    dx = torch.empty(v, 2, 5, device="cuda").permute(1, 2, 0)
    api.distill_grad(ctx, x, ids2, z2, 1.0, dx, d_loss=d.view(2, 5), loss=loss, tail=True)
    # another order of the sums: both are within their tolerance of the same value
    _, tol_loss, _, tol = plain_distill(flat, ids, z, 1.0, True, d)
    close(loss.reshape(-1), want_loss.double(), 2 * tol_loss, "loss")
    close(dx.reshape(10, v), want.double(), 2 * tol, "dlogits")
    api.distill_grad(ctx, x, ids2, z2, 1.0, x, d_loss=d.view(2, 5), tail=True)
    assert torch.equal(x.reshape(10, v), dx.reshape(10, v))


@pytest.mark.parametrize("tail", [False, True])
def test_distill_grad_against_differences(tail):
    """The formula above against central differences of the plain loss, in 64 bits."""
    x = (randn(2, 11, seed=3) * 2).double()
    ids, z = teacher_of(x, 4, tail)
    f = lambda y: plain_distill(y, ids, z, 1.0, tail, None)[0].sum()  # noqa: E731
    want = plain_distill(x, ids, z, 1.0, tail, None)[2]
    for i in range(2):
        for j in range(11):
            e = torch.zeros_like(x)
            e[i, j] = 1e-5
            assert abs(((f(x + e) - f(x - e)) / 2e-5 - want[i, j]).item()) < 1e-8


# ---- as they are used --------------------------------------------------------------------------------------------------


def test_same_bits_again(ctx):
    x = (randn(70, 20011, seed=1) * 3).bfloat16()
    t = tokens(70, 20011)
    ids, z = teacher_of(x, 32, True)
    first = None
    for _ in range(3):
        out = outputs(70, 20)
        api.token_logprobs(ctx, x, t, 1.0, **out)
        dx, loss = torch.empty_like(x), torch.empty(70, device="cuda")
        api.distill_grad(ctx, x, ids, z, 1.0, dx, loss=loss, tail=True)
        got = list(out.values()) + [dx, loss]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_streams_and_graphs(ctx):
    """Two streams at once, and a captured call replayed on new inputs beside an eager one."""
    n, v, k = 48, 30011, 10
    xs = [(randn(n, v, seed=i) * 3).bfloat16() for i in range(2)]
    t = tokens(n, v)
    teach = [teacher_of(x, 16, True, seed=i) for i, x in enumerate(xs)]

    def call(x, ids, z, out, dx, dl, loss, stream):
        lb.encode_token_logprobs(ctx, stream, x, t, 1.0, **out)
        lb.encode_token_logprobs_backward(ctx, stream, x, t, 1.0, out["stats"], out["logprob"], dx, entropy=out["entropy"],
                                          d_entropy=out["logprob"])
        lb.encode_distill_grad(ctx, stream, x, ids, z, 1.0, dl, loss=loss, tail=True)

    want = []
    for x, (ids, z) in zip(xs, teach):
        got = (outputs(n, k), torch.empty_like(x), torch.empty_like(x), torch.empty(n, device="cuda"))
        torch.cuda.synchronize()
        call(x, ids, z, *got, None)
        want.append(got)
    ctx.sync()
    flat = lambda g: list(g[0].values()) + list(g[1:])  # noqa: E731
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    both = [(outputs(n, k), torch.empty_like(x), torch.empty_like(x), torch.empty(n, device="cuda")) for x in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            call(xs[i], *teach[i], *both[i], streams[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(flat(want[i]), flat(both[i])))
    # two graphs of the same calls, each with its own buffers, replayed at once on inputs that came after the capture
    held, graphs = [], []
    for i in range(2):
        x, (ids, z) = torch.zeros_like(xs[0]), (torch.zeros_like(teach[0][0]), torch.zeros_like(teach[0][1]))
        got = (outputs(n, k), torch.empty_like(x), torch.empty_like(x), torch.empty(n, device="cuda"))
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=streams[i]):
            call(x, ids, z, *got, streams[i])
        graphs.append(g)
        held.append((x, ids, z, got))
    for i in range(2):
        held[i][0].copy_(xs[i])
        held[i][1].copy_(teach[i][0])
        held[i][2].copy_(teach[i][1])
    torch.cuda.synchronize()
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        call(xs[0], *teach[0], *both[0], streams[0])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(flat(want[i]), flat(held[i][3])))
    assert all(torch.equal(a, b) for a, b in zip(flat(want[0]), flat(both[0])))


def test_graphs_of_many_rows(ctx):
    """Two captured calls over many rows, replayed at once, beside an eager one."""
    n, v = 200, 20000
    xs = [(randn(n, v, seed=i) * 3).bfloat16() for i in range(2)]
    teach = [teacher_of(x, 16, True, seed=i) for i, x in enumerate(xs)]
    want = []
    for x, (ids, z) in zip(xs, teach):
        dx, loss = torch.empty_like(x), torch.empty(n, device="cuda")
        api.distill_grad(ctx, x, ids, z, 1.0, dx, loss=loss, tail=True)
        want.append((dx, loss))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, held = [], []
    for i in range(2):
        x, ids, z = torch.zeros_like(xs[0]), torch.zeros_like(teach[0][0]), torch.zeros_like(teach[0][1])
        dx, loss = torch.empty_like(x), torch.empty(n, device="cuda")
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=streams[i]):
            lb.encode_distill_grad(ctx, streams[i], x, ids, z, 1.0, dx, loss=loss, tail=True)
        graphs.append(g)
        held.append((x, ids, z, dx, loss))
    for i in range(2):
        held[i][0].copy_(xs[i])
        held[i][1].copy_(teach[i][0])
        held[i][2].copy_(teach[i][1])
    dx, loss = torch.empty_like(xs[0]), torch.empty(n, device="cuda")
    torch.cuda.synchronize()
    for _ in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        lb.encode_distill_grad(ctx, None, xs[1], *teach[1], 1.0, dx, loss=loss, tail=True)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(held[i][3], want[i][0]) and torch.equal(held[i][4], want[i][1])
    assert torch.equal(dx, want[1][0]) and torch.equal(loss, want[1][1])


def test_output_layer_step(ctx):
    """A training step of an output layer: the product makes the logits, the score and its gradient go back through the
    products; then a teacher's best alternatives, as token_logprobs gives them, distil the same layer."""
    rows, width, v, k = 96, 128, 1500, 24
    h = (randn(rows, width, seed=1)).bfloat16()
    w = (randn(width, v, seed=2) * width ** -0.5 * 3).bfloat16()
    t = tokens(rows, v)
    logits = torch.empty(rows, v, dtype=torch.bfloat16, device="cuda")
    api.gemm(ctx, 1.0, h, w, 0.0, logits)
    out = outputs(rows, k)
    api.token_logprobs(ctx, logits, t, 1.0, **out)
    n = int((t >= 0).sum())
    g = torch.full((rows,), -1.0 / n, device="cuda")
    dlogits = torch.empty_like(logits)
    api.token_logprobs_backward(ctx, logits, t, 1.0, out["stats"], g, dlogits)
    dw, dh = torch.empty(width, v, dtype=torch.bfloat16, device="cuda"), torch.empty_like(h)
    api.gemm(ctx, 1.0, h.t(), dlogits, 0.0, dw)
    api.gemm(ctx, 1.0, dlogits, w.t(), 0.0, dh)
    # 64 bits from the same logits: each gradient is a sum of products of values rounded to bf16 (half a step each), and is
    # rounded once more
    ref = Plain(logits, 1.0)
    hot = torch.zeros_like(ref.p).scatter_(1, t.long().clamp(min=0)[:, None], 1.0)
    d = torch.where((t >= 0)[:, None], (ref.p - hot) / n, 0.0)
    step = torch.finfo(torch.bfloat16).eps / 2
    for got, a, b in ((dw, h.double().t(), d), (dh, d, w.double().t())):
        want, size = a @ b, a.abs() @ b.abs()
        # 2 U sqrt-free bound of the product's own f32 sums over at most 1500 terms
        close(got, want, step * want.abs() + size * (step * 1.01 + 1500 * 2 * U) + 1e-37, "gradient")
    # the teacher: its best alternatives as they come out; the student: the same layer, disturbed
    student = (logits.float() + randn(rows, v, seed=7)).bfloat16()
    loss, dstudent = torch.empty(rows, device="cuda"), torch.empty_like(student)
    api.distill_grad(ctx, student, out["top_ids"], out["top_logprobs"], 1.0, dstudent, loss=loss, tail=True)
    want_loss, tol_loss, want, tol = plain_distill(student, out["top_ids"], out["top_logprobs"], 1.0, True, None)
    close(loss, want_loss, tol_loss, "loss")
    close(dstudent, want, tol, "dlogits")
    assert float(loss.min()) > 0
    # a student that is the teacher has nothing to learn: what is left are the roundings of the logits and of the list
    api.distill_grad(ctx, logits, out["top_ids"], out["top_logprobs"], 1.0, dstudent, loss=loss, tail=True)
    want_loss, tol_loss, want, tol = plain_distill(logits, out["top_ids"], out["top_logprobs"], 1.0, True, None)
    close(loss, want_loss, tol_loss, "no loss")
    close(dstudent, want, tol, "no gradient")
