"""Helper layers users put inside their generator / adversary definitions (reference: vegans/utils/layers.py:4-33)."""
import math

import torch
from torch import nn


class LayerPrintSize(nn.Module):
    """Debug layer: prints the shape of what flows through it and passes it on unchanged."""

    def forward(self, x):
        print(tuple(x.shape))
        return x


class LayerReshape(nn.Module):
    """Reshape [batch, features] to [batch, *shape] (metadata only: no kernel runs)."""

    def __init__(self, shape):
        super().__init__()
        self.shape = list(shape) if not isinstance(shape, int) else [shape]

    def forward(self, x):
        return torch.reshape(x, (-1, *self.shape))

    def extra_repr(self):
        return "shape={}".format(self.shape)


class _LayerOnTokens(nn.Module):
    """A layer of the engine that works on the tokens of its input: the pixels of a feature map [batch, channels, height,
    width], the rows of a token tensor [batch, tokens, channels] or, where tokens do not meet, of [batch, channels]. What it
    computes is added to its input where `residual` is set."""

    def __init__(self, channels, residual):
        super().__init__()
        self.channels = channels
        self.residual = residual

    def _rows(self, x):
        """(rows [*, channels], batch, the tokens' grid)"""
        from ..engine import ops
        if x.dim() == 4 and x.shape[1] == self.channels:
            return ops.tokens(x), x.shape[0], (x.shape[2], x.shape[3])
        if x.dim() == 3 and x.shape[2] == self.channels:
            return x.reshape(-1, self.channels), x.shape[0], (x.shape[1],)
        if x.dim() == 2 and x.shape[1] == self.channels:
            return x, x.shape[0], ()
        raise ValueError("expected [batch, {0}, height, width], [batch, tokens, {0}] or [batch, {0}], got {1}".format(
            self.channels, tuple(x.shape)))

    def _back(self, rows, out, x):
        from ..engine import ops
        if self.residual:
            out = ops.add(rows, out)
        return ops.feature_map(out, x.shape) if x.dim() == 4 else out.reshape(x.shape)


class LayerSelfAttention(_LayerOnTokens):
    """Self-attention of the pixels of a feature map (or of the tokens of a sequence): projection to `heads` query heads and
    `kv_heads` key and value heads, norm of every query and key head with a learned scale, rotation by row and column (by
    place in a sequence), attention, projection back. Runs in generators and in critics, but not under a gradient penalty
    (the operators have no second derivative).

    Args:
        channels: of the input. heads: of the queries; kv_heads: of keys and values, heads is a multiple (default: heads).
        width: of a head, a multiple of 8 up to 128 (default: channels / heads). base: of the rotation's frequencies.
        residual: whether the input is added. eps: of the norm."""

    def __init__(self, channels, heads, kv_heads=None, width=None, base=10000.0, residual=True, eps=1e-6):
        super().__init__(channels, residual)
        kv_heads = heads if kv_heads is None else kv_heads
        width = channels // heads if width is None else width
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError("heads={} is not a multiple of kv_heads={}".format(heads, kv_heads))
        if width % 8 or not 8 <= width <= 128:
            raise ValueError("width={} of a head is not a multiple of 8 from 8 to 128".format(width))
        self.heads, self.kv_heads, self.width, self.base, self.eps = heads, kv_heads, width, base, eps
        self.qkv = nn.Linear(channels, (heads + 2 * kv_heads) * width, bias=False)
        self.out = nn.Linear(heads * width, channels)
        self.q_scale = nn.Parameter(torch.ones(width))
        self.k_scale = nn.Parameter(torch.ones(width))
        self._places = {}

    def __getstate__(self):
        return {**self.__dict__, "_places": {}}

    def _positions(self, grid, device):
        """Row and column of every pixel (place of every token), int32 on `device`; made once per grid."""
        got = self._places.get((grid, device))
        if got is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("LayerSelfAttention meets a grid of {} for the first time while a HIP graph is being captured: "
                                   "run it once before".format(grid))
            with torch.inference_mode(False):       # (a tensor made in inference mode cannot be saved for a backward pass)
                axes = torch.meshgrid(*[torch.arange(n, dtype=torch.int32) for n in grid], indexing="ij")
                got = self._places[(grid, device)] = torch.stack(axes, -1).reshape(-1, len(grid)).contiguous().to(device)
        return got

    def forward(self, x):
        from ..engine import ops
        rows, batch, grid = self._rows(x)
        if not grid:
            raise ValueError("attention needs tokens: got a [batch, channels] input")
        rows = ops.as_feature(rows)
        count = math.prod(grid)
        # half of a head turns with the rows, half with the columns (in steps of a pair)
        axes = (self.width,) if len(grid) == 1 else (self.width // 4 * 2, self.width - self.width // 4 * 2)
        packed = self.qkv(rows).view(batch, count, self.heads + 2 * self.kv_heads, self.width)
        mixed = ops.self_attention(packed, self.heads, self.kv_heads, self.q_scale, self.k_scale, self._positions(grid, x.device), axes,
                                   base=self.base, eps=self.eps)
        return self._back(rows, self.out(mixed.view(batch * count, self.heads * self.width)), x)

    def extra_repr(self):
        return "channels={}, heads={}, kv_heads={}, width={}, residual={}".format(self.channels, self.heads, self.kv_heads, self.width,
                                                                                  self.residual)


class LayerGatedFeedForward(_LayerOnTokens):
    """Gated feed-forward block on every pixel (token, row): act(x Wg^T + bg) * (x Wu^T + bu), then a projection back.
    `weight` and `bias` hold the gate's rows, then the values'. Not under a gradient penalty (no second derivative).

    Args:
        channels: of the input. hidden: features between the projections. activation: of the gate, "silu", "gelu", "relu" or
        "sigmoid". bias: whether the first projections have one. residual: whether the input is added."""

    def __init__(self, channels, hidden, activation="silu", bias=True, residual=True):
        super().__init__(channels, residual)
        from .._hip import GATES
        if activation not in GATES:
            raise ValueError("activation={!r}: expected one of {}".format(activation, sorted(GATES)))
        self.hidden, self.activation = hidden, activation
        self.weight = nn.Parameter(torch.empty(2 * hidden, channels))
        self.bias = nn.Parameter(torch.empty(2 * hidden)) if bias else None
        nn.init.uniform_(self.weight, -channels ** -0.5, channels ** -0.5)
        if bias:
            nn.init.uniform_(self.bias, -channels ** -0.5, channels ** -0.5)
        self.out = nn.Linear(hidden, channels)

    def forward(self, x):
        from ..engine import ops
        rows, _, _ = self._rows(x)
        rows = ops.as_feature(rows)
        return self._back(rows, self.out(ops.gated_linear(rows, self.weight, self.bias, self.activation)), x)

    def extra_repr(self):
        return "channels={}, hidden={}, activation={!r}, bias={}, residual={}".format(self.channels, self.hidden, self.activation,
                                                                                      self.bias is not None, self.residual)
