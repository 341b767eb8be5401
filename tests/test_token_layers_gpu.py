"""LayerSelfAttention and LayerGatedFeedForward inside generators and critics: against their formulas in 64 bits, through
fit()'s training step with replayed graphs, and what they refuse."""
import numpy as np
import pytest
import torch
from torch import nn

import token_oracle as oracle
from token_oracle import U32, UBF

pytestmark = pytest.mark.gpu


def _layers():
    from vegans.utils import layers
    return layers


def _bound(module):
    from vegans.engine import modules
    return modules.prepare_parameters(modules.bind(module.cuda()))


def _reference(layer, x, gy):
    """Output and gradients of a layer for a feature map in 64 bits, by the oracle's formulas chained."""
    layers = _layers()
    P = {n: p.detach().cpu().double() for n, p in layer.named_parameters()}
    n, c, h, w = x.shape
    rows, grow = x.permute(0, 2, 3, 1).reshape(-1, c).double(), gy.permute(0, 2, 3, 1).reshape(-1, c).double()
    found = {}
    if isinstance(layer, layers.LayerGatedFeedForward):
        mid = oracle.gated(rows, P["weight"], P.get("bias"), layer.activation, grow @ P["out.weight"])
        found.update(weight=mid["gw"], bias=mid["gb"])
        hidden, grows = mid["h"], mid["gx"]
    else:
        H, K, D = layer.heads, layer.kv_heads, layer.width
        pos = torch.stack(torch.meshgrid(torch.arange(h), torch.arange(w), indexing="ij"), -1).reshape(1, h * w, 2).expand(n, -1, -1)
        axes = (D // 4 * 2, D - D // 4 * 2)
        qkv = (rows @ P["qkv.weight"].T).view(n, h * w, H + 2 * K, D)
        q, k, v = qkv.split((H, K, K), 2)
        yq, yk = (oracle.rotary(t, s, pos, axes, layer.base, layer.eps) for t, s in ((q, P["q_scale"]), (k, P["k_scale"])))
        att = oracle.attention(yq, yk, v, go=(grow @ P["out.weight"]).view(n, h * w, H, D))
        _, gq, found["q_scale"] = oracle.rotary(q, P["q_scale"], pos, axes, layer.base, layer.eps, att["gq"])
        _, gk, found["k_scale"] = oracle.rotary(k, P["k_scale"], pos, axes, layer.base, layer.eps, att["gk"])
        gqkv = torch.cat((gq, gk, att["gv"]), 2).reshape(rows.shape[0], -1)
        found["qkv.weight"] = gqkv.T @ rows
        hidden, grows = att["o"].reshape(rows.shape[0], -1), gqkv @ P["qkv.weight"]
    out = hidden @ P["out.weight"].T + P["out.bias"]
    found.update({"out.weight": grow.T @ hidden, "out.bias": grow.sum(0)})
    if layer.residual:
        out, grows = out + rows, grows + grow
    back = lambda t: t.view(n, h, w, c).permute(0, 3, 1, 2)  # noqa: E731
    return back(out), back(grows), found


def _make(kind):
    layers = _layers()
    torch.manual_seed(3)
    if kind == "attention":
        layer = layers.LayerSelfAttention(32, 4, kv_heads=2, width=16, base=100.0)
    elif kind == "attention, no residual":
        layer = layers.LayerSelfAttention(24, 3, width=8, residual=False)
    elif kind == "feed-forward":
        layer = layers.LayerGatedFeedForward(32, 48, "gelu")
    else:
        layer = layers.LayerGatedFeedForward(40, 30, "silu", bias=False, residual=False)
    with torch.no_grad():
        for p in layer.parameters():
            if p.dim() == 1:
                p.add_(0.1 * torch.randn_like(p))
    return layer


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["attention", "attention, no residual", "feed-forward", "feed-forward, plain"])
def test_layer_against_its_formula(gpu, kind, mode):
    from vegans.engine import ops
    layer = _make(kind)
    gen = torch.Generator().manual_seed(9)
    x, gy = (torch.randn(3, layer.channels, 5, 6, generator=gen) for _ in range(2))
    want, want_gx, want_p = _reference(layer, x, gy)
    previous = ops.set_matmul_precision(mode)
    try:
        layer = _bound(layer)
        xd = x.cuda().contiguous(memory_format=torch.channels_last).requires_grad_()
        y = ops.as_f32(layer(xd))
        got = torch.autograd.grad(y, [xd] + list(layer.parameters()), gy.cuda().contiguous(memory_format=torch.channels_last))
    finally:
        ops.set_matmul_precision(previous)
    # in norm: a chain of at most 10 stages, each off by at most 64 f32 half-steps of its input's size, times 8 for what norm
    # and softmax amplify; bf16: by the 10 roundings of 2^-8 between the stages
    tol = 10 * UBF if mode == "bf16" else 10 * 64 * 8 * U32
    names = [n for n, _ in layer.named_parameters()]
    for a, b, n in [(y, want, "y"), (got[0], want_gx, "gx")] + [(g, want_p[n], n) for g, n in zip(got[1:], names)]:
        off = ((a.detach().cpu().double() - b).norm() / b.norm()).item()
        assert off <= tol, (n, off, tol)


def test_layers_take_tokens_and_rows(gpu):
    """A token tensor gives what the feature map of its tokens gives where rotation does not tell them apart, and rows what
    the tokens give."""
    ff = _bound(_make("feed-forward"))
    x = torch.randn(2, 32, 3, 4, device="cuda").contiguous(memory_format=torch.channels_last)
    t = x.permute(0, 2, 3, 1).reshape(2, 12, 32)
    with torch.no_grad():
        assert torch.equal(ff(t), ff(x).permute(0, 2, 3, 1).reshape(2, 12, 32))
        assert torch.equal(ff(t.reshape(24, 32)), ff(t).reshape(24, 32))
        att = _bound(_make("attention"))
        assert att(t).shape == t.shape
        # one row of pixels: the column half of every head turns as a sequence of half the width would
        assert att(x[:, :, :1].contiguous(memory_format=torch.channels_last)).shape == (2, 32, 1, 4)


def _reference_of_tokens(layer, x, gy):
    """What `_reference` gives, for a token tensor [batch, tokens, channels]: one axis, along the tokens."""
    if isinstance(layer, _layers().LayerGatedFeedForward):         # (tokens do not meet: any feature map of them)
        n, t, c = x.shape
        y, gx, found = _reference(layer, x.transpose(1, 2).reshape(n, c, 1, t), gy.transpose(1, 2).reshape(n, c, 1, t))
        return y.reshape(n, c, t).transpose(1, 2), gx.reshape(n, c, t).transpose(1, 2), found
    P = {n: p.detach().cpu().double() for n, p in layer.named_parameters()}
    H, K, D = layer.heads, layer.kv_heads, layer.width
    n, t, c = x.shape
    rows, grow = x.reshape(-1, c).double(), gy.reshape(-1, c).double()
    pos = torch.arange(t).view(1, t, 1).expand(n, -1, -1)
    q, k, v = (rows @ P["qkv.weight"].T).view(n, t, H + 2 * K, D).split((H, K, K), 2)
    yq, yk = (oracle.rotary(a, s, pos, (D,), layer.base, layer.eps) for a, s in ((q, P["q_scale"]), (k, P["k_scale"])))
    att = oracle.attention(yq, yk, v, go=(grow @ P["out.weight"]).view(n, t, H, D))
    _, gq, gqs = oracle.rotary(q, P["q_scale"], pos, (D,), layer.base, layer.eps, att["gq"])
    _, gk, gks = oracle.rotary(k, P["k_scale"], pos, (D,), layer.base, layer.eps, att["gk"])
    gqkv, hidden = torch.cat((gq, gk, att["gv"]), 2).reshape(n * t, -1), att["o"].reshape(n * t, -1)
    out, grows = hidden @ P["out.weight"].T + P["out.bias"], gqkv @ P["qkv.weight"]
    if layer.residual:
        out, grows = out + rows, grows + grow
    return out.view(x.shape), grows.view(x.shape), {"q_scale": gqs, "k_scale": gks, "qkv.weight": gqkv.T @ rows, "out.weight": grow.T @ hidden,
                                                   "out.bias": grow.sum(0)}


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["attention", "attention, no residual", "feed-forward"])
@pytest.mark.parametrize("shape", ["tokens", "one row of pixels"])
def test_layers_on_sequences_against_their_formulas(gpu, shape, kind, mode):
    """Token tensors (one axis of rotation) and feature maps of one row (all rows' places are zero): values and gradients."""
    from vegans.engine import ops
    layer = _make(kind)
    gen = torch.Generator().manual_seed(19)
    size = (3, 29, layer.channels) if shape == "tokens" else (3, layer.channels, 1, 29)
    x, gy = (torch.randn(size, generator=gen) for _ in range(2))
    want, want_gx, want_p = (_reference_of_tokens if shape == "tokens" else _reference)(layer, x, gy)
    previous = ops.set_matmul_precision(mode)
    try:
        layer = _bound(layer)
        form = torch.contiguous_format if shape == "tokens" else torch.channels_last
        xd = x.cuda().contiguous(memory_format=form).requires_grad_()
        y = layer(xd)
        assert y.shape == size
        y = ops.as_f32(y) if shape != "tokens" else ops.as_f32(y.reshape(-1, size[-1])).reshape(size)
        got = torch.autograd.grad(y, [xd] + list(layer.parameters()), gy.cuda().contiguous(memory_format=form))
    finally:
        ops.set_matmul_precision(previous)
    # as in test_layer_against_its_formula
    tol = 10 * UBF if mode == "bf16" else 10 * 64 * 8 * U32
    names = [n for n, _ in layer.named_parameters()]
    for a, b, n in [(y, want, "y"), (got[0], want_gx, "gx")] + [(g, want_p[n], n) for g, n in zip(got[1:], names)]:
        off = ((a.detach().cpu().double() - b).norm() / b.norm()).item()
        assert off <= tol, (n, off, tol)


def test_layers_train_after_inference_mode(gpu):
    """Sampling under torch.inference_mode() first, then a training step on the same grid: what the layer keeps between calls
    (the pixels' places) can be saved for the backward pass."""
    att = _bound(_make("attention"))
    x = torch.randn(2, 32, 3, 5, device="cuda").contiguous(memory_format=torch.channels_last)
    with torch.inference_mode():
        sampled = att(x)
    y = att(x)
    grads = torch.autograd.grad(y, list(att.parameters()), torch.ones_like(y))
    assert torch.equal(sampled, y) and all(g.isfinite().all() for g in grads)


def test_layers_refuse(gpu):
    layers = _layers()
    for bad in (lambda: layers.LayerSelfAttention(32, 3, 2), lambda: layers.LayerSelfAttention(30, 3), lambda: layers.LayerSelfAttention(512, 2),
                lambda: layers.LayerGatedFeedForward(8, 8, "tanh")):
        with pytest.raises(ValueError):
            bad()
    att = _bound(_make("attention"))
    with pytest.raises(ValueError, match="expected"):
        att(torch.zeros(2, 31, 3, 3, device="cuda"))
    with pytest.raises(ValueError, match="tokens"):
        att(torch.zeros(2, 32, device="cuda"))
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="first time"):
        with torch.cuda.graph(graph):
            att(torch.empty(2, 32, 7, 9, device="cuda"))


def _networks():
    layers = _layers()
    torch.manual_seed(11)
    G = nn.Sequential(nn.Linear(16, 32 * 16), layers.LayerReshape([32, 4, 4]), layers.LayerSelfAttention(32, 4, 2),
                      nn.BatchNorm2d(32), layers.LayerGatedFeedForward(32, 64), nn.ConvTranspose2d(32, 16, 4, 2, 1), nn.BatchNorm2d(16),
                      nn.ReLU(), nn.ConvTranspose2d(16, 3, 4, 2, 1), nn.Tanh())
    D = nn.Sequential(nn.Conv2d(3, 32, 4, 2, 1), nn.LeakyReLU(0.2), layers.LayerSelfAttention(32, 2, width=16), nn.BatchNorm2d(32),
                      layers.LayerGatedFeedForward(32, 32, "gelu", bias=False), nn.Conv2d(32, 1, 8, 1, 0), nn.Flatten(), nn.Identity())
    return G, D


def _model(algo, **extra):
    import vegans.GAN as gan
    G, D = _networks()
    if algo == "LSGAN":
        D[-1] = nn.Sigmoid()
    np.random.seed(4)
    torch.manual_seed(4)
    m = getattr(gan, algo)(G, D, x_dim=(3, 16, 16), z_dim=16, optim_kwargs={"Generator": {"lr": 1e-3}, "Adversariat": {"lr": 5e-4}},
                           folder=None, fixed_noise_size=4, **extra)
    m._create_steps(None)
    m.train()
    return m


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("algo", ["WassersteinGAN", "LSGAN"])
def test_training_step_replayed_equals_eager(gpu, algo, mode):
    """Generator and critic with both layers: parameters and losses after seven steps, replayed and eager, bit for bit."""
    import bench_configs as cfg
    from vegans.engine import graph, ops
    previous = ops.set_matmul_precision(mode)
    try:
        data = cfg.synthetic_images(8 * 7, (3, 16, 16), seed=8)
        gen = torch.Generator().manual_seed(12)
        zs = [torch.randn(8, 16, generator=gen) for _ in range(7)]
        states = []
        for use_graph in (False, True):
            m = _model(algo, **({"clip_val": 0.05} if algo == "WassersteinGAN" else {}))
            m.use_step_graph = use_graph
            losses = []
            for i, z in enumerate(zs):
                m.train_on_batch(m._to_device(data[i * 8:(i + 1) * 8]), z.cuda())
                losses.append({k: v.detach().clone() for k, v in m._losses.items()})
            torch.cuda.synchronize()
            if use_graph:
                entries = list(graph._graphs.get(m, {}).values())
                assert len(entries) == 1 and entries[0].graph is not None and not entries[0].failed
            states.append((losses, {n + k: v.clone() for n, net in m.neural_nets.items() for k, v in net.state_dict().items()}))
    finally:
        ops.set_matmul_precision(previous)
    (l0, s0), (l1, s1) = states
    for a, b in zip(l0, l1):
        for k in a:
            assert torch.isfinite(a[k]).all() and torch.equal(a[k], b[k]), k
    for k in s0:
        assert torch.equal(s0[k], s1[k]), k


def test_gradient_penalty_through_a_token_layer_is_refused(gpu):
    from vegans._hip import HipError
    import vegans.GAN as gan
    G, D = _networks()
    m = gan.WassersteinGANGP(G, D, x_dim=(3, 16, 16), z_dim=16, folder=None, fixed_noise_size=4)
    m._create_steps(None)
    m.train()
    m.use_step_graph = False
    with pytest.raises(HipError, match="second derivatives"):
        m.train_on_batch(m._to_device(np.zeros((4, 3, 16, 16), np.float32)), torch.zeros(4, 16, device="cuda"))


def test_fit_through_the_public_call(gpu):
    """fit() on a numpy array, and the layers' parameters come back in the caller's modules."""
    import contextlib
    import io
    m = _model("WassersteinGAN", clip_val=0.05)
    before = {k: v.detach().cpu().clone() for k, v in m.generator.state_dict().items()}
    X = np.random.RandomState(0).randn(32, 3, 16, 16).astype(np.float32)
    with contextlib.redirect_stdout(io.StringIO()):
        m.fit(X, epochs=1, batch_size=8, print_every=None, enable_tensorboard=False)
        samples, losses = m.get_training_results(by_epoch=False)
    assert np.isfinite(np.asarray(samples)).all()
    after = m.generator.state_dict()
    assert all(not torch.equal(before[k], after[k].cpu()) for k in before if k.endswith(("qkv.weight", "q_scale", "2.out.weight", "4.weight")))
