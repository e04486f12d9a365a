"""Host-side checks of the gated feed-forward block: refusals of the C ABI
(nothing launches) and of the Python layer, sizes, and the traced route."""
import ctypes

import pytest
import torch

import mps_deform_conv as mdc
from mps_deform_conv import _abi


def _desc(dtype=_abi.DCN_BFLOAT16, act=0, tokens=100, channels=64, hidden=128):
    return _abi.DcnFfnDesc(dtype, act, tokens, channels, hidden)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=5), "dtype"), (dict(act=4), "activation"), (dict(act=-1), "activation"), (dict(tokens=-1), "positive"),
    (dict(channels=0), "positive"), (dict(hidden=0), "positive"), (dict(channels=(1 << 20) + 1), "at most"),
    (dict(tokens=(1 << 30) + 1), "size limit"), (dict(tokens=1 << 29, hidden=1 << 12), "size limit"),
])
def test_descriptor_refusals(kw, needle):
    lib = _abi.load()
    d = _desc(**kw)
    assert lib.dcn_ffn_validate(ctypes.byref(d)) != _abi.DCN_OK
    assert needle in lib.dcn_last_error().decode()
    assert lib.dcn_ffn_saved_bytes(ctypes.byref(d)) == 0
    assert lib.dcn_ffn_forward_workspace_size(ctypes.byref(d), 1) == 0
    assert lib.dcn_ffn_backward_workspace_size(ctypes.byref(d)) == 0


def test_null_descriptor_and_sizes():
    lib = _abi.load()
    assert lib.dcn_ffn_validate(None) == _abi.DCN_ERR_INVALID_ARGUMENT
    d = _desc(tokens=0)
    assert lib.dcn_ffn_validate(ctypes.byref(d)) == _abi.DCN_OK
    assert lib.dcn_ffn_saved_bytes(ctypes.byref(d)) == 0
    for dt in (_abi.DCN_FLOAT32, _abi.DCN_FLOAT16, _abi.DCN_BFLOAT16):
        for m, c, f in ((1, 1, 1), (129, 63, 65), (5000, 64, 170)):
            d = _desc(dt, 0, m, c, f)
            # the hidden values, in panels of 128 rows and 8 columns, live in the saved state when there is one
            hidden = (3 if dt == _abi.DCN_FLOAT32 else 1) * (-(-m // 128) * 128) * (-(-f // 8) * 8) * 2
            if m > 32:
                assert lib.dcn_ffn_forward_workspace_size(ctypes.byref(d), 0) - \
                    lib.dcn_ffn_forward_workspace_size(ctypes.byref(d), 1) == hidden
            # up to 256 (fp32: 128) channels gate and up are computed again, not saved
            assert lib.dcn_ffn_saved_bytes(ctypes.byref(d)) == hidden
            assert lib.dcn_ffn_backward_workspace_size(ctypes.byref(d)) >= 2 * hidden
    for dt, c in ((_abi.DCN_FLOAT32, 128), (_abi.DCN_BFLOAT16, 256)):
        few, many = _desc(dt, 0, 1000, c, 64), _desc(dt, 0, 1000, c + 1, 64)
        gate_up = 1000 * 64 * 2 * (4 if dt == _abi.DCN_FLOAT32 else 2)
        assert lib.dcn_ffn_saved_bytes(ctypes.byref(many)) - lib.dcn_ffn_saved_bytes(ctypes.byref(few)) >= gate_up


def _tensors(**kw):
    t = _abi.DcnFfnTensors(*[0x10000 * (i + 1) for i in range(7)])
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def test_forward_refusals():
    lib = _abi.load()
    d = _desc()
    need = lib.dcn_ffn_forward_workspace_size(ctypes.byref(d), 0)
    saved = lib.dcn_ffn_saved_bytes(ctypes.byref(d))

    def call(t, y=0x100000, sv=None, sv_bytes=0, ws=0x200000, ws_bytes=need, desc=d):
        rc = lib.dcn_ffn_forward(ctypes.byref(desc), ctypes.byref(t) if t is not None else None, y, sv, sv_bytes, ws,
                                 ws_bytes, None)
        return rc, lib.dcn_last_error().decode()

    for t, kw, needle in ((None, {}, "NULL"), (_tensors(x=None), {}, "NULL"), (_tensors(w_down=None), {}, "NULL"),
                          (_tensors(b_up=None), {}, "go together"), (_tensors(w_up=0x10008), {}, "16-byte"),
                          (_tensors(), dict(y=None), "both NULL"), (_tensors(), dict(y=0x100008), "16-byte"),
                          (_tensors(), dict(ws=None), "workspace"), (_tensors(), dict(ws_bytes=need - 1), "workspace"),
                          (_tensors(), dict(ws=0x200010), "256-byte"),
                          (_tensors(), dict(sv=0x400000, sv_bytes=saved - 1), "saved state")):
        rc, msg = call(t, **kw)
        assert rc != _abi.DCN_OK and needle in msg, (needle, msg)
    assert call(None, desc=_desc(tokens=0))[0] == _abi.DCN_OK  # nothing to do


def test_backward_refusals():
    lib = _abi.load()
    d = _desc()
    need = lib.dcn_ffn_backward_workspace_size(ctypes.byref(d))
    saved = lib.dcn_ffn_saved_bytes(ctypes.byref(d))

    def call(t=_tensors(), dy=0x900000, sv=0x400000, sv_bytes=saved, g=_tensors(), ws=0x200000, ws_bytes=need):
        rc = lib.dcn_ffn_backward(ctypes.byref(d), ctypes.byref(t), dy, sv, sv_bytes,
                                  ctypes.byref(g) if g is not None else None, ws, ws_bytes, None,
                                  _abi.PARAMS_READY_FN(), None)
        return rc, lib.dcn_last_error().decode()

    for kw, needle in ((dict(g=None), "grads is NULL"), (dict(dy=None), "grad_y"), (dict(dy=0x900008), "grad_y"),
                       (dict(sv=None), "saved state"), (dict(sv_bytes=saved - 1), "saved state"),
                       (dict(ws_bytes=need - 1), "workspace"), (dict(g=_tensors(w_gate=0x10004)), "16-byte"),
                       (dict(t=_tensors(x=None)), "NULL")):
        rc, msg = call(**kw)
        assert rc != _abi.DCN_OK and needle in msg, (needle, msg)


def _args(m=6, c=8, f=12, device="cpu", bias=True):
    t = lambda *s: torch.zeros(s, device=device)  # noqa: E731
    return [t(m, c), t(f, c), t(f, c), t(c, f)] + ([t(f), t(f), t(c)] if bias else [None] * 3)


def test_python_refusals():
    with pytest.raises(ValueError, match="Input must be on CUDA device"):
        mdc.gated_feed_forward(*_args())
    with pytest.raises(ValueError, match="positive"):
        mdc.GatedFeedForward2d(0, 4)
    with pytest.raises(ValueError, match="activation"):
        mdc.GatedFeedForward2d(4, 4, activation="tanh")
    with pytest.raises(ValueError, match="4-D"):
        mdc.GatedFeedForward2d(4, 4)(torch.zeros(3, 4))
    a = _args(device="meta")
    for k, bad, needle in ((1, torch.zeros(12, 7, device="meta"), "w_gate"), (1, torch.zeros(8, device="meta"), "w_gate"),
                           (2, torch.zeros(11, 8, device="meta"), "w_up"), (3, torch.zeros(12, 8, device="meta"), "w_down"),
                           (4, None, "go together"), (5, torch.zeros(8, device="meta"), "b_up"),
                           (6, torch.zeros(12, device="meta"), "b_down"), (3, torch.zeros(8, 12), "same device")):
        b = list(a)
        b[k] = bad
        with pytest.raises(ValueError, match=needle):
            mdc.gated_feed_forward(*b)
    with pytest.raises(ValueError, match="activation"):
        mdc.gated_feed_forward(*a, activation="swish")
    with pytest.raises(ValueError, match="positive"):
        mdc.gated_feed_forward(*[t if t is None else t[..., :0] if t.dim() == 2 and i != 3 else t[:0] for i, t in
                                 enumerate(_args(device="meta", bias=False))])


def test_module_parameters():
    m = mdc.GatedFeedForward2d(16, 40)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {
        "w_gate": (40, 16), "w_up": (40, 16), "w_down": (16, 40), "b_gate": (40,), "b_up": (40,), "b_down": (16,)}
    assert set(mdc.GatedFeedForward2d(16, 40, bias=False).state_dict()) == {"w_gate", "w_up", "w_down"}
    for p in m.parameters():
        assert torch.isfinite(p).all() and p.abs().max() > 0


@pytest.mark.parametrize("bias", [True, False])
def test_meta_shapes_and_gradients(bias):
    a = [t if t is None else t.requires_grad_(True) for t in _args(device="meta", bias=bias)]
    a[0] = torch.zeros(2, 5, 3, 8, device="meta", requires_grad=True)
    y = mdc.gated_feed_forward(*a, activation="gelu")
    assert y.shape == (2, 5, 3, 8)
    grads = torch.autograd.grad(y.sum(), [t for t in a if t is not None])
    assert [g.shape for g in grads] == [t.shape for t in a if t is not None]


def test_module_compiles_to_one_graph_on_meta():
    graphs = []

    def backend(gm, example_inputs):
        graphs.append([str(n.target) for n in gm.graph.nodes if n.op == "call_function"])
        return gm.forward

    m = mdc.GatedFeedForward2d(8, 16).to("meta")
    x = torch.zeros(2, 8, 4, 4, device="meta")
    torch._dynamo.reset()
    y = torch.compile(m, backend=backend, fullgraph=True)(x)
    assert y.shape == x.shape
    assert any("gated_feed_forward" in t for t in graphs[0])
    torch._dynamo.reset()


@pytest.mark.parametrize("k", range(7))
def test_forward_mode_is_refused(k):
    """No input requires grad, so autograd sees no call: the tangent must not vanish silently."""
    a = _args(device="meta")
    with torch.autograd.forward_ad.dual_level():
        assert mdc.gated_feed_forward(*a).shape == (6, 8)  # nothing carries a tangent
        a[k] = torch.autograd.forward_ad.make_dual(a[k], torch.zeros_like(a[k]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            mdc.gated_feed_forward(*a)


@pytest.mark.parametrize("name", ["b_gate", "b_up", "b_down"])
@pytest.mark.parametrize("dtype,off", [(_abi.DCN_BFLOAT16, 1), (_abi.DCN_FLOAT32, 2)])
def test_biases_off_their_elements_are_refused(name, dtype, off):
    """A kernel's access there would fault the GPU."""
    lib = _abi.load()
    d = _desc(dtype)
    bad = _tensors(**{name: 0x70000 + off})
    rc = lib.dcn_ffn_forward(ctypes.byref(d), ctypes.byref(bad), 0x1000000, None, 0, 0x2000000, 1 << 40, None)
    assert rc == _abi.DCN_ERR_INVALID_ARGUMENT and "aligned" in lib.dcn_last_error().decode()
    for tensors, grads in ((bad, _tensors()), (_tensors(), bad)):
        rc = lib.dcn_ffn_backward(ctypes.byref(d), ctypes.byref(tensors), 0x9000000, 0x4000000, 1 << 40,
                                  ctypes.byref(grads), 0x2000000, 1 << 40, None, _abi.PARAMS_READY_FN(), None)
        assert rc == _abi.DCN_ERR_INVALID_ARGUMENT and "aligned" in lib.dcn_last_error().decode()
