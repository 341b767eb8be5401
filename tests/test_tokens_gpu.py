"""The token operators (per-head norm with rotation, attention, gated linear layer) against plain 64-bit forms.

Tolerances are bounds, not fits: a sum of n terms in f32 is off by at most n half-steps (2^-24) of the sum of the terms'
absolute values, a rounding to bf16 by half a step (2^-8) of what is rounded. Every test counts them beside its check."""
import math

import pytest
import torch

import token_oracle as oracle
from token_oracle import U32, UBF

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _ops():
    from vegans.engine import ops
    return ops


def _rand(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


def _within(got, want, allowed, what):
    """|got - want| <= allowed, elementwise, and no NaN"""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), "%s is not finite" % what
    over = ((got - want).abs() - allowed).max().item() if got.numel() else -1.0
    assert over <= 0, "%s: off by up to %.3e, %.3e beyond its bound" % (what, (got - want).abs().max().item(), over)


# ------------------------------------------------------------------------------------------------------------------
# norm and rotation
# ------------------------------------------------------------------------------------------------------------------
ROTARY = [
    # B, T, Hq, Hk, D, axes, far, normed
    (1, 1, 1, 1, 8, (2,), 8, True),
    (2, 5, 3, 1, 16, (4, 6), 50, True),
    (1, 64, 4, 4, 64, (32, 32), 8, True),
    (3, 77, 6, 2, 72, (24, 24), 100000, True),           # part of the head unturned
    (2, 9, 16, 4, 128, (32, 48, 48), 1 << 30, True),     # three axes, far positions
    (2, 33, 5, 3, 24, (8, 2, 2, 6), 1000, True),         # four axes whose borders cut a lane's vector
    (1, 50, 2, 2, 256, (128, 128), 4096, True),
    (2, 13, 33, 1, 40, (40,), 300, True),                # more heads than a wave has room for
    (1, 21, 4, 2, 64, (64,), 77, False),                 # rotation alone
    (2, 21, 4, 2, 64, (), 1, True),                      # norm alone
    (1, 2100, 1, 1, 8, (8,), 5000, True),                # more token groups than one pass of waves
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", ROTARY, ids=str)
def test_rotary(gpu, case, dtype):
    b, t, hq, hk, d, axes, far, normed = case
    gen = torch.Generator().manual_seed(b * 1000 + t + d)
    packed = _rand(gen, b, t, hq + hk + 1, d, dtype=dtype, scale=1.7)
    wq, wk = (1 + 0.3 * torch.randn(d, generator=gen) for _ in range(2))
    shared = b == 1 or t % 2 == 1
    pos = torch.randint(0, far, (t, len(axes)) if shared else (b, t, len(axes)), generator=gen)
    if t % 3 == 0:
        pos = pos.int()
    gq, gk = _rand(gen, b, t, hq, d, dtype=dtype), _rand(gen, b, t, hk, d, dtype=dtype)
    dev = packed.cuda()
    q, k = dev[:, :, :hq].detach().requires_grad_(), dev[:, :, hq:hq + hk].detach().requires_grad_()
    w = [x.cuda().requires_grad_() if normed else None for x in (wq, wk)]
    yq, yk = _ops().qk_norm_rotary(q, k, *w, pos.cuda() if axes else None, axes, base=10000.0, eps=1e-6)
    leaves = [q, k] + ([*w] if normed else [])
    got = torch.autograd.grad((yq, yk), leaves, (gq.cuda(), gk.cuda()))
    place = pos.expand(b, t, len(axes)) if shared else pos
    for x, wx, y, gy, gx, gw, what in ((packed[:, :, :hq], wq, yq, gq, got[0], got[2] if normed else None, "q"),
                                       (packed[:, :, hq:hq + hk], wk, yk, gk, got[1], got[3] if normed else None, "k")):
        wx = wx.double() if normed else None
        y0, gx0, gw0 = oracle.rotary(x.double(), wx, place, axes, 10000.0, 1e-6, gy.double())
        # forward: the sum of D squares (D half-steps, halved by the root, then root, division, two products, sine, cosine
        # to 4 half-steps, product, sum): D / 2 + 16 of the pair's size; backward: two sums of D terms
        u = UBF if dtype == BF16 else U32
        size = y0.reshape(*y0.shape[:-1], d // 2, 2).norm(dim=-1, keepdim=True).expand(*y0.shape[:-1], d // 2, 2).reshape(y0.shape)
        _within(y, y0, u * y0.abs() + (d / 2 + 16) * U32 * size + 1e-30, what)
        reach = (gy.double().norm(dim=-1, keepdim=True) * (1 if wx is None else wx.abs().max()))
        if normed:
            reach = reach * (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        _within(gx, gx0, u * gx0.abs() + (2 * d + 32) * U32 * reach * 2, "g" + what)
        if normed:
            # terms |gn| |x r|, each off by D / 2 + 20 half-steps, and their sum over all rows
            xhat = x.double() * (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
            pairs = gy.double().reshape(*gy.shape[:-1], d // 2, 2).norm(dim=-1, keepdim=True).expand(*gy.shape[:-1], d // 2, 2)
            mag = (pairs.reshape(xhat.shape) * xhat.abs()).sum((0, 1, 2))
            _within(gw, gw0, (b * t * hq + d / 2 + 20) * U32 * mag, "gw" + what)


def test_rotary_gradient_against_differences(gpu):
    gen = torch.Generator().manual_seed(3)
    q, k = _rand(gen, 1, 6, 2, 16), _rand(gen, 1, 6, 1, 16)
    w = 1 + 0.3 * torch.randn(16, generator=gen)
    pos = torch.randint(0, 40, (1, 6, 2), generator=gen)
    gq, gk = _rand(gen, 1, 6, 2, 16), _rand(gen, 1, 6, 1, 16)
    leaves = [t.cuda().requires_grad_() for t in (q, k, w, w)]
    got = torch.autograd.grad(_ops().qk_norm_rotary(*leaves, pos.cuda(), (8, 6)), leaves, (gq.cuda(), gk.cuda()))

    def value(q, k, wq, wk):
        return sum((oracle.rotary(x, wx, pos, (8, 6), 10000.0, 1e-6) * g.double()).sum() for x, wx, g in ((q, wq, gq), (k, wk, gk)))

    _against_differences(value, [q, k, w, w], got, gen)


def _against_differences(value, inputs, got, gen, step=1e-5):
    """<gradient, v> against the central difference of the 64-bit form along v (its own error: step^2, 1e-10)."""
    for i, x in enumerate(inputs):
        v = torch.randn(x.shape, generator=gen).double()
        base = [t.double() for t in inputs]
        ends = []
        for sign in (1, -1):
            moved = list(base)
            moved[i] = base[i] + sign * step * v
            ends.append(value(*moved))
        want = ((ends[0] - ends[1]) / (2 * step)).item()
        g = got[i].detach().cpu().double()
        # a thousand f32 half-steps of what is summed, and the difference's own cancellation
        allowed = 1000 * U32 * (g.abs() * v.abs()).sum().item() + 1e-7 * max(1.0, abs(float(ends[0])))
        assert abs((g * v).sum().item() - want) <= allowed, (i, (g * v).sum().item(), want, allowed)


# ------------------------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------------------------
ATTENTION = [
    # B, Tq, Tk, Hq, Hk, D, ragged
    (1, 1, 1, 1, 1, 8, False),
    (1, 64, 64, 4, 4, 64, False),
    (2, 33, 65, 4, 2, 32, True),
    (3, 130, 129, 6, 2, 40, True),          # odd sizes, padded width
    (2, 1, 700, 8, 2, 64, False),           # one query: keys split, joined
    (2, 1, 1500, 4, 1, 128, True),          # one query, ragged keys in every split
    (1, 300, 5, 4, 4, 128, False),          # few keys: rows split for the keys' gradient
    (1, 1100, 70, 2, 1, 16, True),
    (1, 257, 1030, 1, 1, 72, False),        # both long, one head: both walks split
    (4, 20, 31, 12, 4, 96, True),
    (2, 160, 160, 3, 3, 128, False),
    (1, 7, 66, 21, 3, 24, False),           # group of seven heads
]


def _attention_case(case, dtype, seed=0):
    b, tq, tk, hq, hk, d, ragged = case
    gen = torch.Generator().manual_seed(b * 7919 + tq * 31 + tk + d + seed)
    q, k, v = _rand(gen, b, tq, hq, d, dtype=dtype), _rand(gen, b, tk, hk, d, dtype=dtype), _rand(gen, b, tk, hk, d, dtype=dtype)
    go = _rand(gen, b, tq, hq, d, dtype=dtype)
    ql = kl = None
    if ragged:
        ql = torch.randint(0, tq + 1, (b,), generator=gen, dtype=torch.int32)
        kl = torch.randint(0, tk + 1, (b,), generator=gen, dtype=torch.int32)
        kl[0] = max(1, tk // 3)
        if b > 1:
            kl[-1] = -3                      # an element without keys (below zero: clamped)
            ql[0], kl[0] = tq, tk + 50       # beyond the tensor: clamped
    return q, k, v, ql, kl, go


def _attention_allowed(want, dtype, case, name):
    """Half-steps of `name`: scores off by D + 4 half-steps of the largest |q||k| sum move every probability by as much;
    exponential and sum of Tk terms; then the sum over keys (rows). bf16: the probabilities (o, gv) or ds (gq, gk) are
    rounded once for the next product; and the output is rounded."""
    b, tq, tk, hq, hk, d, _ = case
    steps = 2 * (d + 4) * (want["scores_abs"] + 1) * 1.5 + 2 * tk + tq * (hq // hk) + d + 64
    allowed = steps * U32 * want["abs"][name] + 1e-30
    if dtype == BF16:
        allowed = allowed + UBF * want["abs"][name] * (1 + UBF) + UBF * want[name].abs() * 1.01
    return allowed


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", ATTENTION, ids=str)
def test_attention(gpu, case, dtype):
    q, k, v, ql, kl, go = _attention_case(case, dtype)
    want = oracle.attention(q.double(), k.double(), v.double(), ql, kl, None, go.double())
    if kl is not None:      # what takes no part may be anything
        for i in range(q.shape[0]):
            k[i, max(0, int(kl[i])):], v[i, max(0, int(kl[i])):] = float("nan"), float("inf")
            q[i, int(ql[i]):], go[i, int(ql[i]):] = float("inf"), float("nan")
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    lens = [t.cuda() if t is not None else None for t in (ql, kl)]
    o = _ops().attention(*leaves, *lens)
    got = dict(zip(("gq", "gk", "gv"), torch.autograd.grad(o, leaves, go.cuda())))
    got["o"] = o
    with torch.no_grad():
        assert torch.equal(_ops().attention(*leaves, *lens), o)
    for name in ("o", "gq", "gk", "gv"):
        _within(got[name], want[name], _attention_allowed(want, dtype, case, name), name)
    again = torch.autograd.grad(_ops().attention(*leaves, *lens), leaves, go.cuda())
    assert all(torch.equal(a, got[n]) for a, n in zip(again, ("gq", "gk", "gv"))), "a second run differs"


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_attention_strides_and_orders(gpu, dtype):
    """Heads-major tensors, slices of a packed projection, keys shared over the batch by a stride of zero."""
    case = (3, 50, 70, 4, 2, 32, False)
    q, k, v, _, _, go = _attention_case(case, dtype)
    k, v = k[:1].expand_as(k), v[:1].expand_as(v)
    want = oracle.attention(q.double(), k.double(), v.double(), None, None, None, go.double())
    packed = torch.zeros(3, 50, 7, 64, dtype=dtype)
    packed[:, :, 1:5, 16:48] = q
    qd = packed.cuda()[:, :, 1:5, 16:48].detach().requires_grad_()
    kd = k[:1].transpose(1, 2).contiguous().cuda().transpose(1, 2).requires_grad_()      # [1, heads, keys, width] in memory
    vd = v[:1].cuda().requires_grad_()
    o = _ops().attention(qd, kd.expand(3, -1, -1, -1), vd.expand(3, -1, -1, -1))
    gq, gk, gv = torch.autograd.grad(o, (qd, kd, vd), go.transpose(1, 2).contiguous().cuda().transpose(1, 2))
    _within(o, want["o"], _attention_allowed(want, dtype, case, "o"), "o")
    _within(gq, want["gq"], _attention_allowed(want, dtype, case, "gq"), "gq")
    # shared keys: autograd adds the three elements' gradients (two more roundings of partial sums)
    for g, n in ((gk, "gk"), (gv, "gv")):
        u = UBF if dtype == BF16 else U32
        _within(g, want[n].sum(0, keepdim=True), _attention_allowed(want, dtype, case, n).sum(0, keepdim=True) +
                2 * u * 1.01 * want[n].abs().sum(0, keepdim=True), n)


@pytest.mark.parametrize("scale", [-0.3, 1.7])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_attention_scales(gpu, dtype, scale):
    """A negative scale turns the order of the scores; ragged keys keep out under both."""
    case = (2, 40, 100, 4, 2, 32, True)
    q, k, v, ql, kl, go = _attention_case(case, dtype)
    want = oracle.attention(q.double(), k.double(), v.double(), ql, kl, scale, go.double())
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    o = _ops().attention(*leaves, ql.cuda(), kl.cuda(), scale=scale)
    got = dict(zip(("o", "gq", "gk", "gv"), (o,) + torch.autograd.grad(o, leaves, go.cuda())))
    for n in got:
        _within(got[n], want[n], _attention_allowed(want, dtype, case, n), n)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_attention_extreme_scores(gpu, dtype):
    """Scores far from zero on both sides, rows with one dominant key, equal scores."""
    gen = torch.Generator().manual_seed(5)
    q, k, v = _rand(gen, 1, 40, 2, 32, dtype=dtype, scale=12.0), _rand(gen, 1, 90, 2, 32, dtype=dtype, scale=12.0), _rand(gen, 1, 90, 2, 32, dtype=dtype)
    q[:, :4] = 0                                                  # all scores equal
    k[:, :, 0] = k[:, :, 0].abs()
    q[:, 4:8, 0] = -q[:, 4:8, 0].abs() * 4                        # every score of the row far below zero
    go = _rand(gen, 1, 40, 2, 32, dtype=dtype)
    case = (1, 40, 90, 2, 2, 32, False)
    want = oracle.attention(q.double(), k.double(), v.double(), None, None, 0.25, go.double())
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    o = _ops().attention(*leaves, scale=0.25)
    got = dict(zip(("o", "gq", "gk", "gv"), (o,) + torch.autograd.grad(o, leaves, go.cuda())))
    for n in got:
        _within(got[n], want[n], _attention_allowed(want, dtype, case, n), n)


def test_attention_gradient_against_differences(gpu):
    gen = torch.Generator().manual_seed(11)
    q, k, v, go = _rand(gen, 1, 9, 4, 16), _rand(gen, 1, 12, 2, 16), _rand(gen, 1, 12, 2, 16), _rand(gen, 1, 9, 4, 16)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(_ops().attention(*leaves), leaves, go.cuda())
    _against_differences(lambda q, k, v: (oracle.attention(q, k, v)["o"] * go.double()).sum(), [q, k, v], got, gen)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_attention_over_few_keys(gpu, dtype):
    """One key: the scores' gradients are exactly zero. Two and three keys: ds is a small difference of go v^T and delta, and
    delta must not carry the rounding of a bf16 o: in norm, ds is off by its own rounding and 2^-15 of |go| |v| instead."""
    for tk in (1, 2, 3):
        case = (2, 37, tk, 4, 2, 64, False)
        q, k, v, _, _, go = _attention_case(case, dtype)
        want = oracle.attention(q.double(), k.double(), v.double(), None, None, None, go.double())
        leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
        gq, gk, gv = torch.autograd.grad(_ops().attention(*leaves), leaves, go.cuda())
        if tk == 1:
            assert not gq.any() and not gk.any()
            continue
        for got, n in ((gq, "gq"), (gk, "gk")):
            u = UBF if dtype == BF16 else 64 * U32
            off = (got.cpu().double() - want[n]).norm()
            # ds rounded once, the output rounded once (each at most u of the value), delta at 2^-17 and the scores in f32
            assert off <= 2 * u * want[n].norm() + 2.0 ** -15 * u / UBF * want["abs"][n].norm(), (tk, n, off / want[n].norm())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_attention_of_nothing(gpu, dtype):
    ops = _ops()
    new = lambda *s: torch.ones(*s, dtype=dtype, device="cuda", requires_grad=True)  # noqa: E731
    q, k, v = new(2, 3, 2, 16), new(2, 0, 1, 16), new(2, 0, 1, 16)
    o = ops.attention(q, k, v)
    assert not o.any() and not torch.autograd.grad(o, q, torch.ones_like(o))[0].any()
    q, k, v = new(2, 0, 2, 16), new(2, 3, 1, 16), new(2, 3, 1, 16)
    o = ops.attention(q, k, v)
    gk, gv = torch.autograd.grad(o, (k, v), torch.ones_like(o))
    assert o.shape == (2, 0, 2, 16) and not gk.any() and not gv.any()
    assert ops.attention(new(0, 3, 2, 16), new(0, 3, 2, 16), new(0, 3, 2, 16)).shape == (0, 3, 2, 16)


@pytest.mark.parametrize("case", [
    (2, 700, 900, 2, 2, 24, False),        # both walks split
    (3, 640, 520, 4, 2, 64, True),
    (1, 1100, 1030, 2, 1, 96, True),
    (8, 300, 300, 16, 8, 32, False),       # keys whole, rows split
    (16, 256, 260, 16, 16, 64, True),      # both whole
    (8, 200, 200, 32, 32, 128, False),
], ids=str)
def test_attention_of_many_scores(gpu, case):
    """bf16 beyond 2^20 scores, where probabilities and ds are rounded to one bf16 term for their products."""
    assert case[0] * case[1] * case[2] * case[3] > 1 << 20
    q, k, v, ql, kl, go = _attention_case(case, BF16)
    want = oracle.attention(q.double(), k.double(), v.double(), ql, kl, None, go.double())
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    lens = [t.cuda() if t is not None else None for t in (ql, kl)]
    o = _ops().attention(*leaves, *lens)
    got = dict(zip(("o", "gq", "gk", "gv"), (o,) + torch.autograd.grad(o, leaves, go.cuda())))
    for name in got:
        _within(got[name], want[name], _attention_allowed(want, BF16, case, name), name)


def test_attention_over_few_keys_in_a_large_batch(gpu):
    """What test_attention_over_few_keys says, beyond 2^20 scores, for two and three keys."""
    for tk in (2, 3):
        case = (1024, 33, tk, 16, 16, 64, False)
        q, k, v, _, _, go = (t.cuda() if t is not None else None for t in _attention_case(case, BF16))
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        got = dict(zip(("gq", "gk"), torch.autograd.grad(_ops().attention(*leaves), leaves[:2], go)))
        some = slice(500, 503)
        want = oracle.attention(*(t[some].cpu().double() for t in (q, k, v)), None, None, None, go[some].cpu().double())
        for n in got:
            off = (got[n][some].cpu().double() - want[n]).norm()
            assert off <= 2 * UBF * want[n].norm() + 2.0 ** -15 * want["abs"][n].norm(), (tk, n, off / want[n].norm())


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("b, tq, tk", [(700, 33, 3), (64, 40, 37), (16, 130, 150), (64, 1, 1100)])
def test_attention_of_a_common_part(gpu, b, tq, tk, d):
    """bf16 beyond 2^20 scores, keys, values and output gradients of mean 3 and deviation 1. ds = p (go v^T - delta) is the small
    difference of two numbers near 9 d that have the values' common part in common: delta must not carry it rounded.

    In norm, independent roundings adding as squares: the result's (u of it), each ds' (u |ds_j| |k_j|), and each
    probability's: e_j p_j, |e_j| <= u, moves o by sum_j e_j p_j (v_j - o), delta by sum_j e_j ds_j (u |ds| in norm) and gq by that
    times the row's mean key. A rounding is at most u, 0.4 u in the mean: a factor of two to spare; f32 adds 64 half-steps
    of |go| |v| in delta."""
    gen = torch.Generator().manual_seed(d + tk)
    h, scale = 16, 0.02
    q, k, v, go = (_rand(gen, b, n, h, d) + mean for n, mean in ((tq, 0), (tk, 3), (tk, 3), (tq, 3)))
    q, k, v, go = (t.to(BF16).cuda() for t in (q, k, v, go))
    assert b * h * tq * tk >= 1 << 20
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = _ops().attention(*leaves, scale=scale)
    gq, gk, gv = torch.autograd.grad(o, leaves, go)
    Q, K, V, G = (t.double().transpose(1, 2).contiguous() for t in (q, k, v, go))
    p = torch.softmax(scale * Q @ K.transpose(2, 3).contiguous(), -1)
    O = p @ V
    ds = p * (G @ V.transpose(2, 3).contiguous() - (G * O).sum(-1, keepdim=True))
    want = scale * ds @ K
    squares = ds.square() @ K.square().sum(-1, keepdim=True) + ds.square().sum(-1, keepdim=True) * (p @ K).square().sum(-1, keepdim=True)
    delta = 64 * U32 * (G.abs() * (p @ V.abs())).sum(-1, keepdim=True) * (p @ K).norm(dim=-1, keepdim=True)
    allowed = UBF * (want.square().sum() + scale ** 2 * squares.sum()).sqrt() + scale * delta.norm()
    off = (gq.double().transpose(1, 2) - want).norm()
    assert off <= allowed, ((off / want.norm()).item(), (allowed / want.norm()).item())
    assert (o.double().transpose(1, 2) - O).norm() <= 1.5 * UBF * O.norm()


def test_attention_gradients_of_a_part(gpu):
    """Only what asks for a gradient gets one, and it is the same."""
    q, k, v, ql, kl, go = _attention_case((2, 33, 65, 4, 2, 32, True), F32)
    dev = [t.cuda() for t in (q, k, v)]
    full = [t.clone().requires_grad_() for t in dev]
    want = torch.autograd.grad(_ops().attention(*full, ql.cuda(), kl.cuda()), full, go.cuda())
    for i in range(3):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate(dev)]
        got = torch.autograd.grad(_ops().attention(*some, ql.cuda(), kl.cuda()), some[i], go.cuda())[0]
        assert torch.equal(got, want[i])


# ------------------------------------------------------------------------------------------------------------------
# gated linear layer
# ------------------------------------------------------------------------------------------------------------------
GATED = [
    # rows, in, out, act, bias
    (1, 8, 8, "silu", False),
    (5, 64, 96, "gelu", True),
    (33, 40, 31, "relu", True),           # odd output width
    (130, 129, 70, "sigmoid", True),      # nothing is a multiple of anything
    (257, 256, 200, "silu", True),
    (300, 1, 1, "silu", True),            # one feature in, one out
    (64, 1100, 64, "gelu", False),        # many features: pre-activations stored, not computed again
    (1000, 96, 16, "silu", True),         # few tiles, many rows: the weight gradient's sum is split
    (17, 72, 1030, "relu", False),        # few rows: the input gradient's sum is split
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", GATED, ids=str)
def test_gated(gpu, case, dtype):
    m, c, f, act, with_bias = case
    gen = torch.Generator().manual_seed(m + c + f)
    x, w = _rand(gen, m, c, dtype=dtype), _rand(gen, 2 * f, c, dtype=dtype, scale=c ** -0.5)
    bias = _rand(gen, 2 * f, scale=0.2) if with_bias else None
    gh = _rand(gen, m, f, dtype=dtype)
    want = oracle.gated(x.double(), w.double(), bias.double() if with_bias else None, act, gh.double())
    leaves = [t.cuda().requires_grad_() for t in (x, w) + ((bias,) if with_bias else ())]
    h = _ops().gated_linear(*leaves, **({} if with_bias else {"bias": None}), act=act)
    got = dict(zip(("gx", "gw", "gb"), torch.autograd.grad(h, leaves, gh.cuda())))
    got["h"] = h
    with torch.no_grad():
        assert torch.equal(_ops().gated_linear(*leaves, **({} if with_bias else {"bias": None}), act=act), h)
    # pre-activations: C + 2 half-steps of their sums over absolute values; gate and derivative 16 (erf, exp, division);
    # then sums over 2F, M or M terms. bf16: gz is rounded once for the products, and the output
    for n, terms in (("h", 0), ("gx", 2 * f), ("gw", m), ("gb", m)):
        if n not in got:
            continue
        allowed = (c + terms + 32) * U32 * want["abs"][n] + 1e-30
        if act == "relu" and n != "h":
            # a pre-activation within its error of zero may fall on either side
            near = (c + 4) * U32 * want["z_abs"][:, :f]
            g = (x.double() @ w.double().T + (bias.double() if with_bias else 0))[:, :f]
            assert not ((g.abs() <= near) & (g != 0)).any()
        if dtype == BF16 and n != "gb":
            u = want["gz_abs"][n] * UBF * (1 + UBF) if n != "h" else 0
            allowed = allowed + u + UBF * want[n].abs() * 1.01
        _within(got[n], want[n], allowed, n)


def test_gated_gradient_against_differences(gpu):
    gen = torch.Generator().manual_seed(21)
    for act in ("silu", "gelu", "sigmoid"):
        x, w, b, gh = _rand(gen, 7, 12), _rand(gen, 10, 12), _rand(gen, 10), _rand(gen, 7, 5)
        leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
        got = torch.autograd.grad(_ops().gated_linear(*leaves, act=act), leaves, gh.cuda())
        _against_differences(lambda x, w, b: (oracle.gated(x, w, b, act)["h"] * gh.double()).sum(), [x, w, b], got, gen)


def test_gated_of_nothing_and_extremes(gpu):
    ops = _ops()
    for dtype in (F32, BF16):
        x = torch.ones(0, 16, dtype=dtype, device="cuda", requires_grad=True)
        w, b = torch.ones(8, 16, dtype=dtype, device="cuda", requires_grad=True), torch.ones(8, device="cuda", requires_grad=True)
        h = ops.gated_linear(x, w, b)
        gx, gw, gb = torch.autograd.grad(h, (x, w, b), torch.ones_like(h))
        assert h.shape == (0, 4) and gx.shape == x.shape and not gw.any() and not gb.any()
    # gates far on both sides: silu and gelu end in 0 and in the gate itself, derivatives in 0 and 1
    x = torch.tensor([[-300.0], [300.0]], device="cuda", requires_grad=True)
    w = torch.tensor([[1.0], [1.0]], device="cuda")
    for act, far in (("silu", 90000.0), ("gelu", 90000.0), ("relu", 90000.0), ("sigmoid", 300.0)):
        h = ops.gated_linear(x, w, act=act)
        assert h[0].item() == 0 and h[1].item() == far
        g = torch.autograd.grad(h, x, torch.ones_like(h))[0]
        assert g[0].item() == 0 and g[1].item() == (1.0 if act == "sigmoid" else 600.0), act


def test_gated_f32_master_weight(gpu):
    """bf16 activations, f32 master weight: the products of the rounded weight, the gradient in f32."""
    gen = torch.Generator().manual_seed(2)
    x, w, gh = _rand(gen, 70, 64, dtype=BF16), _rand(gen, 96, 64), _rand(gen, 70, 48, dtype=BF16)
    xd, wd, wh = x.cuda().requires_grad_(), w.cuda().requires_grad_(), w.to(BF16).cuda().requires_grad_()
    h, h2 = _ops().gated_linear(xd, wd), _ops().gated_linear(xd, wh)
    assert torch.equal(h, h2)
    g, g2 = torch.autograd.grad(h, (xd, wd), gh.cuda()), torch.autograd.grad(h2, (xd, wh), gh.cuda())
    assert torch.equal(g[0], g2[0]) and g[1].dtype == F32 and torch.equal(g[1].to(BF16), g2[1])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_gated_takes_column_slices_and_refuses_other_strides(gpu, dtype):
    from vegans._hip import HipError
    gen = torch.Generator().manual_seed(6)
    wide_x, wide_w, gh = (_rand(gen, n, c, dtype=dtype).cuda() for n, c in ((70, 96), (24, 64), (70, 12)))
    x, w = wide_x[:, 16:64], wide_w[:, 2:50]
    dense, sliced = ([t.requires_grad_() for t in ts] for ts in ((x.clone(), w.clone()), (x.detach(), w.detach())))
    assert not sliced[0].is_contiguous() and not sliced[1].is_contiguous()
    h, want = _ops().gated_linear(*sliced), _ops().gated_linear(*dense)
    assert torch.equal(h, want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(h, sliced, gh), torch.autograd.grad(want, dense, gh)))
    x, w = dense[0].detach(), dense[1].detach()
    bad = [(x.T.contiguous().T, w), (x, w.T.contiguous().T), (x[:1].expand(70, -1), w), (x, w[:1].expand(24, -1)), (wide_x[:, :96:2], w)]
    if dtype == BF16:
        bad += [(wide_x[:, 1:49], w), (wide_x[:, :47], w[:, :47].contiguous())]
    for operands in bad:
        with pytest.raises(HipError):
            _ops().gated_linear(*operands)


@pytest.mark.parametrize("dtype, m, c, f, act", [
    (BF16, 130, 600, 72, "gelu"),          # pre-activations kept, small tiles
    (BF16, 200, 1024, 6400, "silu"),       # gx on small tiles, gw on large ones: two launches
    (BF16, 4099, 264, 4096, "gelu"),       # large tiles, pre-activations computed again
    (BF16, 4099, 520, 4720, "silu"),       # large tiles, pre-activations kept: over 256 MB, past the caches
    (F32, 4099, 60, 3300, "gelu"),         # the same in f32
], ids=str)
def test_gated_large(gpu, dtype, m, c, f, act):
    """What test_gated says, at the sizes where other tiles and the streaming kernels are chosen (the oracle on the GPU)."""
    gen = torch.Generator().manual_seed(m + c + f)
    x, w = _rand(gen, m, c, dtype=dtype).cuda(), _rand(gen, 2 * f, c, dtype=dtype, scale=c ** -0.5).cuda()
    bias, gh = _rand(gen, 2 * f, scale=0.2).cuda(), _rand(gen, m, f, dtype=dtype).cuda()
    leaves = [t.clone().requires_grad_() for t in (x, w, bias)]
    h = _ops().gated_linear(*leaves, act=act)
    got = dict(zip(("gx", "gw", "gb"), torch.autograd.grad(h, leaves, gh)))
    got["h"] = h.detach()
    want = oracle.gated(x.double(), w.double(), bias.double(), act, gh.double())
    for n, terms in (("h", 0), ("gx", 2 * f), ("gw", m), ("gb", m)):
        allowed = (c + terms + 32) * U32 * want["abs"][n] + 1e-30
        if dtype == BF16 and n != "gb":
            u = want["gz_abs"][n] * UBF * (1 + UBF) if n != "h" else 0
            allowed = allowed + u + UBF * want[n].abs() * 1.01
        _within(got[n].cpu(), want[n].cpu(), allowed.cpu(), n)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m, c, f", [(17, 72, 1030), (1000, 96, 16), (257, 256, 200), (130, 600, 72)])
def test_gated_gradients_of_a_part(gpu, dtype, m, c, f):
    """Only what asks for a gradient gets one, and it is the same: alone, two together, with and without slabs to sum."""
    gen = torch.Generator().manual_seed(8)
    dev = [t.cuda() for t in (_rand(gen, m, c, dtype=dtype), _rand(gen, 2 * f, c, dtype=dtype), _rand(gen, 2 * f))]
    gh = _rand(gen, m, f, dtype=dtype).cuda()
    full = [t.clone().requires_grad_() for t in dev]
    want = torch.autograd.grad(_ops().gated_linear(*full), full, gh)
    for part in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        some = [t.clone().requires_grad_(j in part) for j, t in enumerate(dev)]
        got = torch.autograd.grad(_ops().gated_linear(*some), [some[i] for i in part], gh)
        for i, g in zip(part, got):
            assert torch.equal(g, want[i]), (part, i)


# ------------------------------------------------------------------------------------------------------------------
# beyond 32-bit offsets
# ------------------------------------------------------------------------------------------------------------------
def test_attention_over_a_cache_of_four_gigabytes(gpu):
    """2^24 + 77 keys of 128 bf16: everything that counts lies in the last key and in one near the 2^31st element."""
    n, d = (1 << 24) + 77, 128
    k = torch.zeros(1, n, 1, d, dtype=BF16, device="cuda")
    v = torch.zeros(1, n, 1, d, dtype=BF16, device="cuda")
    q = torch.zeros(1, 3, 1, d, dtype=BF16, device="cuda")
    q[0, :, 0, 0] = 16.0
    places = (n - 1, (1 << 31) // d + 5)
    for i, at in enumerate(places):
        k[0, at, 0, 0] = 64.0                      # score 1024 / sqrt(128) = 90.5: all others together weigh 2^24 e^-90
        v[0, at, 0, i] = 2.0
    go = torch.ones(1, 3, 1, d, dtype=BF16, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = _ops().attention(*leaves)
    assert (o[0, :, 0, :2] == 1).all() and not o[0, :, 0, 2:].any()
    gq, gk, gv = torch.autograd.grad(o, leaves, go)
    for i, at in enumerate(places):
        assert (gv[0, at, 0] == 1.5).all()         # three rows with weight 1/2 each
    assert not gv[0, :1000].any() and gv.count_nonzero() == 2 * d
    # go v^T is 2 at both places and delta is 2: no gradient of scores
    assert not gq.any() and not gk.any()


def test_attention_gradients_over_a_cache_of_four_gigabytes(gpu):
    """As above, with output gradients under which the scores of the two keys have gradients: go v^T is 2 and -2, delta 0, ds
    therefore 1 and -1 (p = 1/2), and components of the keys that the queries do not see tell them apart."""
    n, d = (1 << 24) + 77, 128
    k = torch.zeros(1, n, 1, d, dtype=BF16, device="cuda")
    v = torch.zeros(1, n, 1, d, dtype=BF16, device="cuda")
    q = torch.zeros(1, 3, 1, d, dtype=BF16, device="cuda")
    q[0, :, 0, 0] = 16.0
    places = (n - 1, (1 << 31) // d + 5)
    for i, at in enumerate(places):
        k[0, at, 0, 0], k[0, at, 0, 2 + i] = 64.0, 8.0
        v[0, at, 0, i] = 2.0
    go = torch.zeros(1, 3, 1, d, dtype=BF16, device="cuda")
    go[..., 0], go[..., 1] = 1.0, -1.0
    leaves = [t.requires_grad_() for t in (q, k, v)]
    gq, gk, gv = torch.autograd.grad(_ops().attention(*leaves), leaves, go)
    assert gv.count_nonzero() == 4 and gk.count_nonzero() == 2 and gq.count_nonzero() == 6
    scale = torch.tensor(d ** -0.5)              # of three queries of 16, of keys of 8: far from a rounding border of bf16
    for i, (at, sign) in enumerate(zip(places, (1, -1))):
        assert gv[0, at, 0, :2].tolist() == [1.5, -1.5]
        assert gk[0, at, 0, 0].item() == sign * (48 * scale).to(BF16).item()
        assert gq[0, :, 0, 2 + i].tolist() == [sign * (8 * scale).to(BF16).item()] * 3


def test_strides_of_four_gigabytes(gpu):
    """Batch elements 2^31 elements apart."""
    store = torch.zeros((1 << 31) + 4096, dtype=BF16, device="cuda")
    gen = torch.Generator().manual_seed(8)
    x = _rand(gen, 2, 9, 4, 32, dtype=BF16).cuda()
    far = store.as_strided((2, 9, 4, 32), (1 << 31, 128, 32, 1))
    far.copy_(x)
    ops, w, pos = _ops(), torch.ones(32, device="cuda"), torch.arange(9, device="cuda")[:, None]
    with torch.no_grad():
        assert torch.equal(ops.attention(far, far, far), ops.attention(x, x, x))
        for a, b in zip(ops.qk_norm_rotary(far, far, w, w, pos, (32,)), ops.qk_norm_rotary(x, x, w, w, pos, (32,))):
            assert torch.equal(a, b)


def test_gated_rows_beyond_two_gigabytes(gpu):
    """2^20 + 3 rows of 2 x 1100 pre-activations: the last rows are what they are alone."""
    m, c, f = (1 << 20) + 3, 8, 1100
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(m, c, generator=gen, device="cuda").to(BF16).requires_grad_()
    w = torch.randn(2 * f, c, generator=gen, device="cuda").to(BF16).requires_grad_()
    gh = torch.randn(m, f, generator=gen, device="cuda").to(BF16)
    h = _ops().gated_linear(x, w)
    gx, gw = torch.autograd.grad(h, (x, w), gh)
    last = slice(m - 300, m)
    xl = x.detach()[last].clone().requires_grad_()
    hl = _ops().gated_linear(xl, w)
    (gxl,) = torch.autograd.grad(hl, xl, gh[last])
    assert torch.equal(h[last], hl)
    # the alone rows' products are split (and small enough for two terms): the same up to the roundings of [gg gu] and gx
    want = oracle.gated(xl.detach().cpu().double(), w.detach().cpu().double(), None, "silu", gh[last].cpu().double())
    for got in (gx[last], gxl):
        allowed = (c + 2 * f + 32) * U32 * want["abs"]["gx"] + UBF * (1 + UBF) * want["gz_abs"]["gx"] + UBF * want["gx"].abs() * 1.01
        _within(got, want["gx"], allowed, "gx")
    assert torch.isfinite(gw).all()


def test_gated_weight_gradient_beyond_two_gigabytes(gpu):
    """2^20 + 3 rows of 2 x 1100 pre-activations, output gradients around the 2^31st of them and in the last rows only: the
    weight gradient is that of these rows alone."""
    m, c, f = (1 << 20) + 3, 8, 1100
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(m, c, generator=gen, device="cuda").to(BF16).requires_grad_()
    w = torch.randn(2 * f, c, generator=gen, device="cuda").to(BF16).requires_grad_()
    border = (1 << 31) // (2 * f)
    some = torch.cat((torch.arange(border - 20, border + 20), torch.arange(m - 100, m))).cuda()
    gh = torch.zeros(m, f, dtype=BF16, device="cuda")
    gh[some] = torch.randn(len(some), f, generator=gen, device="cuda").to(BF16)
    gx, gw = torch.autograd.grad(_ops().gated_linear(x, w), (x, w), gh)
    want = oracle.gated(x.detach()[some].cpu().double(), w.detach().cpu().double(), None, "silu", gh[some].cpu().double())
    # as in test_gated: all other rows add zeros
    for n, got, terms in (("gw", gw, len(some)), ("gx", gx[some], 2 * f)):
        allowed = (c + terms + 32) * U32 * want["abs"][n] + UBF * (1 + UBF) * want["gz_abs"][n] + UBF * want[n].abs() * 1.01
        _within(got, want[n], allowed, n)
    assert gx.count_nonzero() == gx[some].count_nonzero()


@pytest.mark.parametrize("dtype, c, f", [(BF16, 16384, 65600), (F32, 8192, 65600)], ids=str)
@pytest.mark.parametrize("m", [65, 400])          # small tiles, large tiles (bf16)
def test_gated_weights_beyond_four_gigabytes(gpu, dtype, c, f, m):
    """2 x 65600 rows of 32 KB: all weights are zero but some gate rows and the matching value rows, among them the last, whose
    byte offsets pass 2^32. Those columns are the layer of these rows alone, all others and their gradients are zero."""
    gen = torch.Generator().manual_seed(m)
    rows = torch.tensor([0, 33, f // 2, f - 66, f - 2, f - 1])
    x, small = _rand(gen, m, c, dtype=dtype), _rand(gen, 2 * len(rows), c, dtype=dtype, scale=c ** -0.5)
    gh_small = _rand(gen, m, len(rows), dtype=dtype)
    at = torch.cat((rows, f + rows)).cuda()
    w = torch.zeros(2 * f, c, dtype=dtype, device="cuda")
    w[at] = small.cuda()
    gh = torch.ones(m, f, dtype=dtype, device="cuda")
    gh[:, rows.cuda()] = gh_small.cuda()
    leaves = [x.cuda().requires_grad_(), w.requires_grad_()]
    h = _ops().gated_linear(*leaves)
    gx, gw = torch.autograd.grad(h, leaves, gh)
    want = oracle.gated(x.double(), small.double(), None, "silu", gh_small.double())
    got = {"h": h[:, rows.cuda()], "gx": gx, "gw": gw[at]}
    # as in test_gated: the other columns add zeros to these sums
    for n, terms in (("h", 0), ("gx", 2 * len(rows)), ("gw", m)):
        allowed = (c + terms + 32) * U32 * want["abs"][n] + 1e-30
        if dtype == BF16:
            u = want["gz_abs"][n] * UBF * (1 + UBF) if n != "h" else 0
            allowed = allowed + u + UBF * want[n].abs() * 1.01
        _within(got[n], want[n], allowed, n)
    assert h.count_nonzero() == got["h"].count_nonzero() and gw.count_nonzero() == got["gw"].count_nonzero()


# ------------------------------------------------------------------------------------------------------------------
# together, on streams and in graphs
# ------------------------------------------------------------------------------------------------------------------
def _stage_inputs(dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    b, h, w, heads, kv, d, f = 2, 6, 5, 4, 2, 16, 40
    t, c = h * w, heads * d
    grid = torch.stack(torch.meshgrid(torch.arange(h), torch.arange(w), indexing="ij"), -1).reshape(t, 2)
    qkv = _rand(gen, b, t, heads + 2 * kv, d, dtype=dtype)
    wq, wk = 1 + 0.2 * torch.randn(d, generator=gen), 1 + 0.2 * torch.randn(d, generator=gen)
    wg, bg = _rand(gen, 2 * f, c, dtype=dtype, scale=c ** -0.5), _rand(gen, 2 * f, scale=0.1)
    lengths = torch.tensor([t, t - 7], dtype=torch.int32)
    gh = _rand(gen, b * t, f, dtype=dtype)
    return (qkv, wq, wk, wg, bg), grid, lengths, gh, (b, t, heads, kv, d)


def _stage(leaves, grid, lengths, sizes, packed=True):
    ops = _ops()
    qkv, wq, wk, wg, bg = leaves
    b, t, heads, kv, d = sizes
    if packed:
        o = ops.self_attention(qkv, heads, kv, wq, wk, grid, (8, 8), lengths)
    else:
        q, k, v = qkv.split((heads, kv, kv), 2)
        q, k = ops.qk_norm_rotary(q, k, wq, wk, grid, (8, 8))
        o = ops.attention(q, k, v, lengths, lengths)
    return ops.gated_linear(o.reshape(b * t, heads * d), wg, bg)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_the_operators_together(gpu, dtype):
    """A stage of a token network: packed norm, rotation and attention, then the gated layer. The packed form gives bit for
    bit what the separate operators give; both against the 64-bit forms chained."""
    cpu, grid, lengths, gh, sizes = _stage_inputs(dtype)
    b, t, heads, kv, d = sizes
    leaves = [x.cuda().requires_grad_() for x in cpu]
    h = _stage(leaves, grid.cuda(), lengths.cuda(), sizes)
    got = torch.autograd.grad(h, leaves, gh.cuda())
    h2 = _stage(leaves, grid.cuda(), lengths.cuda(), sizes, packed=False)
    got2 = torch.autograd.grad(h2, leaves, gh.cuda())
    assert torch.equal(h, h2) and all(torch.equal(x, y) for x, y in zip(got, got2))
    # 64 bits, chained
    qkv, wq, wk, wg, bg = (x.double() for x in cpu)
    q, k, v = qkv.split((heads, kv, kv), 2)
    pos = grid.expand(b, t, 2)
    yq, yk = oracle.rotary(q, wq, pos, (8, 8), 10000.0, 1e-6), oracle.rotary(k, wk, pos, (8, 8), 10000.0, 1e-6)
    o = oracle.attention(yq, yk, v, lengths, lengths)["o"]
    last = oracle.gated(o.reshape(b * t, heads * d), wg, bg, "silu", gh.double())
    att = oracle.attention(yq, yk, v, lengths, lengths, None, last["gx"].reshape(b, t, heads, d))
    _, gq, gwq = oracle.rotary(q, wq, pos, (8, 8), 10000.0, 1e-6, att["gq"])
    _, gk, gwk = oracle.rotary(k, wk, pos, (8, 8), 10000.0, 1e-6, att["gk"])
    want = [torch.cat((gq, gk, att["gv"]), 2), gwq, gwk, last["gw"], last["gb"]]
    # in norm: a chain of at most 8 stages, each off by at most 64 f32 half-steps of its input's size (times 8 for what the
    # norm and the softmax amplify), or in bf16 by the 8 roundings of 2^-8 between the stages
    tol = 8 * UBF if dtype == BF16 else 8 * 64 * 8 * U32
    for x, y, n in zip([h] + list(got), [last["h"]] + want, ("h", "gqkv", "gwq", "gwk", "gw", "gb")):
        off = (x.detach().cpu().double() - y).norm() / y.norm()
        assert off <= tol, (n, off.item(), tol)


@pytest.mark.parametrize("packed", [True, False], ids=["packed", "separate"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_padding_holds_anything(gpu, dtype, packed, eps):
    """Norm, rotation and attention of a padded batch whose padding is NaN, infinite or zero: results and gradients are those
    of any other padding, bit for bit, the padding's own gradient is zero."""
    ops = _ops()
    gen = torch.Generator().manual_seed(12)
    b, t, heads, kv, d = 4, 37, 4, 2, 24
    lengths = torch.tensor([37, 9, 0, 30], dtype=torch.int32)
    pad = torch.arange(t)[None, :] >= lengths[:, None]
    base = _rand(gen, b, t, heads + 2 * kv, d, dtype=dtype)
    wq, wk = (1 + 0.2 * torch.randn(d, generator=gen) for _ in range(2))
    pos, go = torch.randint(0, 99, (b, t, 1), generator=gen), _rand(gen, b, t, heads, d, dtype=dtype)
    found = []
    for filling in (1.5, float("nan"), float("inf"), 0.0):
        qkv = base.clone()
        qkv[pad] = filling
        leaves = [x.cuda().requires_grad_() for x in (qkv, wq, wk)]
        n = lengths.cuda()
        if packed:
            o = ops.self_attention(leaves[0], heads, kv, leaves[1], leaves[2], pos.cuda(), (16,), n, eps=eps)
        else:
            q, k, v = leaves[0].split((heads, kv, kv), 2)
            q, k = ops.qk_norm_rotary(q, k, leaves[1], leaves[2], pos.cuda(), (16,), eps=eps)
            o = ops.attention(q, k, v, n, n)
        found.append([o.detach()] + list(torch.autograd.grad(o, leaves, go.cuda())))
    assert not found[0][0][pad.cuda()].any() and not found[0][1][pad.cuda()].any()
    assert all(x.isfinite().all() and x.any() for x in found[0])
    for other in found[1:]:
        assert all(torch.equal(x, y) for x, y in zip(found[0], other))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("b, t", [(2, 0), (0, 5), (1, 1)])
def test_packed_of_nothing_and_one_token(gpu, dtype, b, t):
    gen = torch.Generator().manual_seed(13)
    leaves = [x.cuda().requires_grad_() for x in (_rand(gen, b, t, 4, 16, dtype=dtype), torch.ones(16), torch.ones(16))]
    o = _ops().self_attention(leaves[0], 2, 1, leaves[1], leaves[2], torch.zeros(t, 1, dtype=torch.int32, device="cuda"), (16,))
    assert o.shape == (b, t, 2, 16) and torch.equal(o, leaves[0][:, :, 3:].expand(b, t, 2, 16))
    gx, gq, gk = torch.autograd.grad(o, leaves, torch.ones_like(o))
    # one token attends to itself alone: its value's gradient is the sum over the heads, nothing else has one
    assert gx.shape == leaves[0].shape and not gq.any() and not gk.any() and not gx[:, :, :3].any() and (gx[:, :, 3:] == 2).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_gradients_at_any_address(gpu, dtype):
    """The gradient of a result may be a slice of another tensor, off every 16-byte border (what a concatenation hands back),
    or one number expanded."""
    ops = _ops()
    gen = torch.Generator().manual_seed(14)
    qkv, x, w = _rand(gen, 2, 7, 4, 16, dtype=dtype), _rand(gen, 9, 24, dtype=dtype), _rand(gen, 32, 24, dtype=dtype)
    scale, pos = torch.ones(16, device="cuda"), torch.arange(7, device="cuda")[:, None]
    calls = [lambda t: ops.self_attention(t, 2, 1, scale, scale, pos, (16,)), lambda t: ops.attention(t[:, :, :2], t[:, :, 2:3], t[:, :, 3:]),
             lambda t: ops.qk_norm_rotary(t[:, :, :2], t[:, :, 2:], scale, scale, pos, (16,))[0], lambda t: ops.gated_linear(t, w.cuda())]
    for call, t in zip(calls, (qkv, qkv, qkv, x)):
        leaf = t.cuda().requires_grad_()
        out = call(leaf)
        g = _rand(gen, *out.shape, dtype=dtype).cuda()
        want = torch.autograd.grad(out, leaf, g, retain_graph=True)[0]
        room = torch.zeros(g.numel() + 1, dtype=dtype, device="cuda")
        room[1:] = g.flatten()
        off = room[1:].view(g.shape)
        assert off.data_ptr() % 16 and off.is_contiguous()
        assert torch.equal(torch.autograd.grad(out, leaf, off, retain_graph=True)[0], want)
        one = torch.ones(1, dtype=dtype, device="cuda")
        want = torch.autograd.grad(out, leaf, torch.ones_like(out), retain_graph=True)[0]
        assert torch.equal(torch.autograd.grad(out, leaf, one.expand(out.shape))[0], want)


def test_on_other_streams_at_once(gpu):
    """Two streams run the operators at the same time (the second on other inputs): no scratch is shared."""
    sets = [_stage_inputs(F32, s) for s in (1, 2)]
    on = []
    for cpu, grid, lengths, gh, sizes in sets:
        leaves = [x.cuda().requires_grad_() for x in cpu]
        on.append((leaves, grid.cuda(), lengths.cuda(), gh.cuda(), sizes))
    want = []
    for leaves, grid, lengths, gh, sizes in on:
        h = _stage(leaves, grid, lengths, sizes)
        want.append([h.detach()] + list(torch.autograd.grad(h, leaves, gh)))
        del h
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in on]
    results = [[], []]
    for _ in range(4):
        for i, (leaves, grid, lengths, gh, sizes) in enumerate(on):
            with torch.cuda.stream(streams[i]):
                h = _stage(leaves, grid, lengths, sizes)
                results[i].append([h.detach()] + list(torch.autograd.grad(h, leaves, gh)))
    torch.cuda.synchronize()
    for i in range(2):
        for r in results[i]:
            assert all(torch.equal(x, y) for x, y in zip(r, want[i]))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_two_captured_graphs(gpu, dtype):
    """Forward and backward captured twice (other inputs each), replayed in turn between eager work: every replay equals the
    eager result."""
    graphs = []
    for seed in (3, 4):
        cpu, grid, lengths, gh, sizes = _stage_inputs(dtype, seed)
        leaves = [x.cuda().requires_grad_() for x in cpu]
        grid, lengths, gh = grid.cuda(), lengths.cuda(), gh.cuda()

        def step(leaves=leaves, grid=grid, lengths=lengths, gh=gh, sizes=sizes):
            h = _stage(leaves, grid, lengths, sizes)
            return [h.detach()] + list(torch.autograd.grad(h, leaves, gh))

        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs, want, step))
    for _ in range(3):
        for graph, outs, want, step in graphs:
            for o in outs:
                o.zero_()
            graph.replay()
            eager = step()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(outs, want)) and all(torch.equal(x, y) for x, y in zip(eager, want))


def test_capture_over_a_live_eager_graph_is_refused(gpu):
    """(refused in Python, before autograd reaches the leaf's accumulation node)"""
    from vegans._hip import HipError
    ops = _ops()
    x = torch.ones(4, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, 8, device="cuda", requires_grad=True)
    alive = ops.gated_linear(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(HipError, match="eager graph"):
        with torch.cuda.graph(graph):
            h = ops.gated_linear(x, w)
            torch.autograd.grad(h, (x, w), torch.ones_like(h))
    assert alive.shape == (4, 4)


def test_capture_over_a_live_graph_of_another_operation_is_refused(gpu):
    """The leaf's accumulation node was made by an eager operation that is none of the token operators."""
    from vegans._hip import HipError
    ops = _ops()
    x = torch.ones(4, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, 8, device="cuda", requires_grad=True)
    alive = x * 2
    torch.cuda.synchronize()
    with pytest.raises(HipError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            h = ops.gated_linear(x, w)
            torch.autograd.grad(h, (x, w), torch.ones_like(h))
    # without it the same capture works, and replays
    del alive, h
    want = torch.autograd.grad(ops.gated_linear(x, w), (x, w), torch.ones(4, 4, device="cuda"))
    torch.cuda.synchronize()
    graph, ones = torch.cuda.CUDAGraph(), torch.ones(4, 4, device="cuda")
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(ops.gated_linear(x, w), (x, w), ones)
    for _ in range(3):
        for g in got:
            g.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_second_derivative_is_refused(gpu):
    """A gradient taken with create_graph=True raises when it is differentiated, also behind a constant output gradient."""
    from vegans._hip import HipError
    ops = _ops()
    x = torch.ones(4, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, 8, device="cuda", requires_grad=True)
    t = torch.randn(2, 3, 4, 16, device="cuda", requires_grad=True)
    for out, leaf in ((ops.gated_linear(x, w), x), (ops.attention(t, t, t), t), (ops.self_attention(t, 2, 1), t),
                      (ops.qk_norm_rotary(t, t, torch.ones(16, device="cuda"))[0], t)):
        (g,) = torch.autograd.grad(out, leaf, torch.ones_like(out), create_graph=True)
        with pytest.raises(HipError, match="second derivatives"):
            g.square().sum().backward()


# ------------------------------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------------------------------
def test_refusals(gpu):
    from vegans._hip import HipError
    ops = _ops()
    z = lambda *s, dt=F32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    pos = torch.zeros(4, 1, dtype=torch.int32, device="cuda")
    q, k = z(2, 4, 2, 16), z(2, 4, 1, 16)
    bad = [
        lambda: ops.qk_norm_rotary(q, k.bfloat16(), None, None, pos, (4,)),
        lambda: ops.qk_norm_rotary(q.double(), k.double(), None, None, pos, (4,)),
        lambda: ops.qk_norm_rotary(q, z(2, 5, 1, 16), None, None, pos, (4,)),
        lambda: ops.qk_norm_rotary(z(2, 4, 2, 12), z(2, 4, 1, 12), None, None, pos, (4,)),
        lambda: ops.qk_norm_rotary(q, k, None, None, pos, (3,)),
        lambda: ops.qk_norm_rotary(q, k, None, None, pos, (18,)),
        lambda: ops.qk_norm_rotary(q, k, None, None, None, (4,)),
        lambda: ops.qk_norm_rotary(q, k, None, None, pos.float(), (4,)),
        lambda: ops.qk_norm_rotary(q, k, None, None, pos[:3], (4,)),
        lambda: ops.qk_norm_rotary(q, k, None, None, pos, (4,), base=0.0),
        lambda: ops.qk_norm_rotary(q, k, z(15), None, pos, (4,)),
        lambda: ops.qk_norm_rotary(q, k, z(16, dt=BF16), None, pos, (4,)),
        lambda: ops.qk_norm_rotary(z(2, 4, 2, 17)[..., 1:], k, None, None, pos, (4,)),
        lambda: ops.qk_norm_rotary(z(2, 4, 16, 2).transpose(2, 3), k, None, None, pos, (4,)),
        lambda: ops.attention(q, k, z(2, 4, 2, 16)),
        lambda: ops.attention(q, k.bfloat16(), k.bfloat16()),
        lambda: ops.attention(z(2, 4, 3, 16), z(2, 4, 2, 16), z(2, 4, 2, 16)),
        lambda: ops.attention(z(2, 4, 2, 136), z(2, 4, 1, 136), z(2, 4, 1, 136)),
        lambda: ops.attention(q, k, k, torch.zeros(2, dtype=torch.int64, device="cuda")),
        lambda: ops.attention(q, k, k, None, torch.zeros(3, dtype=torch.int32, device="cuda")),
        lambda: ops.attention(q, k, k, None, torch.zeros(2, dtype=torch.int32)),
        lambda: ops.attention(q, k, k, scale=math.inf),
        lambda: ops.attention(q, k, k, scale=0.0),
        lambda: ops.attention(q[0], k[0], k[0]),
        lambda: ops.self_attention(z(2, 4, 5, 16), 2),
        lambda: ops.self_attention(z(2, 4, 4, 16), 2, 0),
        lambda: ops.gated_linear(z(3, 8), z(5, 8)),
        lambda: ops.gated_linear(z(3, 8), z(4, 9)),
        lambda: ops.gated_linear(z(3, 8), z(4, 8, dt=BF16)),
        lambda: ops.gated_linear(z(3, 8), z(4, 8), z(3)),
        lambda: ops.gated_linear(z(3, 8), z(4, 8), act="tanh"),
        lambda: ops.gated_linear(z(2, 3, 8), z(4, 8)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(HipError):
            call()
            pytest.fail("call %d was not refused" % i)
