"""Token operators on the host: argument checks of the C entry points (nothing is launched) and of the Python operators
without a GPU."""
import ctypes
import glob
import os
import shutil
import subprocess

import pytest
import torch


def _layouts(g, heads, d):
    from vegans import _hip
    for name, _ in g._fields_:
        if isinstance(getattr(g, name), _hip.HeadsLayout):
            setattr(g, name, _hip.HeadsLayout(heads * d * 4, heads * d, d))
    return g


def _rotary(**kw):
    from vegans import _hip
    g = _hip.RotaryGeom(**{**dict(B=2, T=4, Hq=2, Hk=1, D=16, axes=1, eps=1e-6, base=1e4), **kw})
    g.width[0] = 8
    return _layouts(g, 3, 16)


def _attention(**kw):
    from vegans import _hip
    return _layouts(_hip.AttentionGeom(**{**dict(B=2, Tq=4, Tk=4, Hq=2, Hk=1, D=16, scale=0.25), **kw}), 3, 16)


DUMMY = ctypes.c_void_p(256)        # never dereferenced


def _text(lib):
    return lib.vg_last_error().decode()


def test_rotary_arguments_are_checked_before_any_launch():
    from vegans import _hip
    lib = _hip.load()

    def fwd(g, q=DUMMY, pos=DUMMY):
        return lib.vg_qk_norm_rotary_fwd(ctypes.byref(g), q, DUMMY, DUMMY, DUMMY, pos, DUMMY, DUMMY, None)

    for g, word in ((_rotary(D=12), "head width"), (_rotary(D=264), "head width"), (_rotary(axes=5), "axes"), (_rotary(Hq=0), "bad sizes"),
                    (_rotary(T=-1), "bad sizes"), (_rotary(B=1 << 16, T=1 << 15), "too many"), (_rotary(base=0.0), "base")):
        assert fwd(g) == -1 and word in _text(lib), _text(lib)
        assert lib.vg_qk_norm_rotary_workspace_bytes(ctypes.byref(g)) == 0
    g = _rotary()
    g.width[0] = 18
    assert fwd(g) == -1 and "more than the head width" in _text(lib)
    g.width[0] = 3
    assert fwd(g) == -1 and "not even" in _text(lib)
    assert fwd(_rotary(), q=None) == -1 and "null" in _text(lib)
    assert fwd(_rotary(), pos=None) == -1 and "null positions" in _text(lib)
    assert fwd(_rotary(), q=ctypes.c_void_p(264)) == -1 and "16-byte" in _text(lib)
    g = _rotary()
    g.q.sh = 18
    assert fwd(g) == -1 and "16-byte" in _text(lib)
    assert lib.vg_qk_norm_rotary_fwd(None, DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, None) == -1
    need = lib.vg_qk_norm_rotary_workspace_bytes(ctypes.byref(_rotary()))
    assert need > 0
    rc = lib.vg_qk_norm_rotary_bwd(ctypes.byref(_rotary()), *[DUMMY] * 11, DUMMY, 8, None)
    assert rc == -3 and "too small" in _text(lib)
    rc = lib.vg_qk_norm_rotary_bwd(ctypes.byref(_rotary()), DUMMY, DUMMY, None, DUMMY, *[DUMMY] * 7, DUMMY, need, None)
    assert rc == -1 and "not there" in _text(lib)
    assert fwd(_rotary(T=0), q=None) == 0       # nothing to do


def test_attention_arguments_are_checked_before_any_launch():
    from vegans import _hip
    lib = _hip.load()

    def fwd(g, q=DUMMY, ws=None, size=0):
        return lib.vg_attention_fwd(ctypes.byref(g), q, DUMMY, DUMMY, None, None, DUMMY, None, ws, size, None)

    for g, word in ((_attention(D=12), "head width"), (_attention(D=136), "head width"), (_attention(Hq=3, Hk=2), "multiple"),
                    (_attention(Tk=-1), "bad sizes"), (_attention(Hk=0), "bad sizes"), (_attention(scale=float("inf")), "finite"),
                    (_attention(Tq=1 << 29, Hq=4), "too many"), (_attention(Tk=1 << 30), "too many"),
                    (_attention(B=1 << 20, Tq=1 << 14), "too many")):
        assert fwd(g) == -1 and word in _text(lib), _text(lib)
        assert lib.vg_attention_workspace_bytes(ctypes.byref(g), 0, 0) == 0
    assert fwd(_attention(), q=None) == -1 and "null" in _text(lib)
    assert fwd(_attention(), q=ctypes.c_void_p(8)) == -1 and "16-byte" in _text(lib)
    # one query over many keys: the keys are split, and the partial results need space
    g = _attention(B=1, Tq=1, Tk=1 << 14)
    need = lib.vg_attention_workspace_bytes(ctypes.byref(g), 0, 0)
    assert need > 0
    assert fwd(g, ws=DUMMY, size=need - 1) == -3 and "are needed" in _text(lib)
    assert fwd(g, ws=ctypes.c_void_p(264), size=need) == -1 and "aligned" in _text(lib)
    assert fwd(_attention(B=0), q=None) == 0
    g = _attention()
    g.k.st = 1 << 26
    assert fwd(g) == -1 and "stride" in _text(lib)
    rc = lib.vg_attention_bwd(ctypes.byref(_attention()), *[DUMMY] * 8, DUMMY, DUMMY, None, DUMMY, 1 << 20, None)
    assert rc == -1 and "null" in _text(lib)                 # keys' gradient without values'
    rc = lib.vg_attention_bwd(ctypes.byref(_attention()), *[DUMMY] * 8, DUMMY, DUMMY, DUMMY, None, 0, None)
    assert rc == -3


def test_gated_arguments_are_checked_before_any_launch():
    from vegans import _hip
    lib = _hip.load()
    assert lib.vg_gated_linear_fwd(4, 8, 8, None, DUMMY, None, DUMMY, None, 3, None) == -1 and "null" in _text(lib)
    assert lib.vg_gated_linear_fwd(4, 8, 8, DUMMY, DUMMY, None, DUMMY, None, 4, None) == -1 and "activation" in _text(lib)
    assert lib.vg_gated_linear_fwd(4, 0, 8, DUMMY, DUMMY, None, DUMMY, None, 3, None) == -1 and "bad sizes" in _text(lib)
    assert lib.vg_gated_linear_fwd(1 << 30, 8, 8, DUMMY, DUMMY, None, DUMMY, None, 3, None) == -1 and "too many" in _text(lib)
    assert lib.vg_gated_linear_fwd(0, 8, 8, None, None, None, None, None, 3, None) == 0
    need = lib.vg_gated_linear_bwd_workspace_bytes(4096, 64, 32, 0)
    assert need >= 4096 * 64 * 4                        # at least the pre-activations' gradient
    assert lib.vg_gated_linear_bwd(4096, 64, 32, *[DUMMY] * 7, 1, None, 3, DUMMY, need - 1, None) == -3
    assert lib.vg_gated_linear_bwd(4096, 64, 32, DUMMY, DUMMY, None, None, DUMMY, DUMMY, DUMMY, 1, None, 3, DUMMY, need, None) == -1
    assert "pre-activations" in _text(lib)
    assert lib.vg_gated_linear_bwd(4096, 64, 32, None, *[DUMMY] * 6, 1, None, 3, DUMMY, need, None) == -1 and "null" in _text(lib)
    assert lib.vg_gated_linear_bwd(4096, 64, 32, *[DUMMY] * 7, 0, None, 3, DUMMY, need, None) == -1 and "f32" in _text(lib)
    # f32 keeps its pre-activations; bf16 where computing them again would cost more
    assert lib.vg_gated_linear_keeps_z(4096, 64, 32, 0) and not lib.vg_gated_linear_keeps_z(4096, 64, 32, 1)
    assert lib.vg_gated_linear_keeps_z(4096, 2048, 32, 1) and lib.vg_gated_linear_keeps_z(8, 64, 32, 1)


def test_operators_refuse_cpu_tensors():
    from vegans import _hip
    from vegans.engine import ops
    q = torch.zeros(1, 4, 2, 16)
    for call in (lambda: ops.qk_norm_rotary(q, q), lambda: ops.attention(q, q, q), lambda: ops.self_attention(torch.zeros(1, 4, 6, 16), 2),
                 lambda: ops.gated_linear(torch.zeros(4, 8), torch.zeros(6, 8))):
        with pytest.raises(_hip.HipError, match="GPU"):
            call()


class _Twice(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return 2 * x

    @staticmethod
    def backward(ctx, g):
        return 2 * g


def _checked():
    """A toy operator whose backward pass is guarded as the token operators' are."""
    from vegans.engine import ops

    class Checked(_Twice):
        backward = staticmethod(ops._first_order(_Twice.backward))

    return lambda x: ops._record(Checked, x)


def test_accumulation_nodes_from_outside_a_capture_are_refused(monkeypatch):
    """The capture's state is made up, nothing runs on a GPU. Whoever made a leaf's accumulation node before the operator met
    it in the capture, the captured backward pass is refused; a node that the operator itself makes there is fine, also
    for its next calls, and after the capture."""
    from vegans import _hip
    state = {"capturing": False, "stream": "eager"}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: state["stream"])
    op, one = _checked(), torch.ones(3)

    def captured(x, calls=1):
        state.update(capturing=True, stream="capture")
        try:
            return [torch.autograd.grad(y, x, one)[0].tolist() for y in [op(x) for _ in range(calls)]]
        finally:
            state.update(capturing=False, stream="eager")

    def leaf():
        return torch.nn.Parameter(torch.ones(3))

    assert captured(leaf(), calls=2) == [[2.0] * 3] * 2
    for eager in (op, lambda x: x * 3, lambda x: torch.autograd.graph.get_gradient_edge(x)):
        x = leaf()
        alive = eager(x)
        with pytest.raises(_hip.HipError, match="eager graph"):
            captured(x)
        del alive
        assert captured(x) == [[2.0] * 3]
    # the captured graph lives on, an eager one joins it: the node is still the capture's
    x = leaf()
    state.update(capturing=True, stream="capture")
    kept = op(x)
    state.update(capturing=False, stream="eager")
    assert torch.autograd.grad(op(x), x, one)[0].tolist() == [2.0] * 3 and captured(x) == [[2.0] * 3]
    assert kept.requires_grad


@pytest.mark.skipif(shutil.which("make") is None, reason="no make here")
def test_a_change_of_the_compiler_flags_compiles_every_kernel_again():
    """(nothing is run: what make would do after an edit of its file) Objects built with other flags must not be kept: they
    may hold the packed f32 instructions that the flags leave out."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gan-pytorch_amd", "csrc")
    lines = subprocess.run(["make", "-n", "-C", csrc, "-W", "Makefile"], capture_output=True, text=True, check=True).stdout.splitlines()
    compiled = {line.split(" -c ")[1].split()[0]: line for line in lines if " -c " in line}
    assert sorted(compiled) == sorted(os.path.basename(p) for p in glob.glob(os.path.join(csrc, "*.hip")))
    assert all("-packed-fp32-ops" in line for line in compiled.values())
