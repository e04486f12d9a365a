"""Host-side checks of the optimizer step and the gradient norm: the refusals of
the C ABI (nothing launches) and of the Python layer."""
import ctypes

import pytest
import torch

from mps_deform_conv import _abi, optim


def _options(**kw):
    o = _abi.DcnAdamwOptions(1e-3, 0.9, 0.999, 1e-8, 0.01, None, None, 32, 0)
    for k, v in kw.items():
        setattr(o, k, v)
    return o


def _tensors(n=1, **kw):
    """`n` tensors of 64 elements at made-up, disjoint addresses."""
    t = (_abi.DcnAdamwTensor * n)()
    for i in range(n):
        base = 0x100000 * (i + 1)
        t[i] = _abi.DcnAdamwTensor(base, base + 0x10000, base + 0x20000, base + 0x30000, None, None, None,
                                   base + 0x50000, 64, _abi.DCN_FLOAT32, 0)
        for k, v in kw.items():
            setattr(t[i], k, v)
    return t


def _call(o, t, n):
    lib = _abi.load()
    rc = lib.dcn_adamw_step(ctypes.byref(o) if o is not None else None, t, n, None)
    return rc, lib.dcn_last_error().decode()


@pytest.mark.parametrize("kw,needle", [
    (dict(lr=-1.0), "lr must be"), (dict(lr=float("nan")), "lr must be"),
    (dict(beta1=1.0), "betas must be"), (dict(beta2=-0.1), "betas must be"),
    (dict(eps=-1e-8), "eps must be"), (dict(weight_decay=float("inf")), "weight_decay must be"),
    (dict(state_bits=16), "state_bits"),
])
def test_adamw_option_refusals(kw, needle):
    rc, msg = _call(_options(**kw), _tensors(), 1)
    assert rc != _abi.DCN_OK and needle in msg


@pytest.mark.parametrize("kw,bits,needle", [
    (dict(param=None), 32, "NULL"), (dict(grad=None), 32, "NULL"), (dict(exp_avg=None), 32, "NULL"),
    (dict(exp_avg_sq=None), 32, "NULL"), (dict(step=None), 32, "step counter"), (dict(dtype=9), 32, "dtype"),
    (dict(numel=-1), 32, "elements"), (dict(numel=1 << 41), 32, "elements"), (dict(), 8, "exp_avg_scale"),
    (dict(exp_avg=0x100000), 32, "overlap"),                 # the state is the parameter
    (dict(exp_avg_sq=0x120000 + 255), 32, "overlap"),        # the states overlap by one byte
    (dict(master=0x100000 + 252), 32, "overlap"),
])
def test_adamw_tensor_refusals(kw, bits, needle):
    rc, msg = _call(_options(state_bits=bits), _tensors(**kw), 1)
    assert rc != _abi.DCN_OK and needle in msg


def test_adamw_refuses_the_same_parameter_twice():
    t = _tensors(3)
    t[2].param = t[0].param
    rc, msg = _call(_options(), t, 3)
    assert rc == _abi.DCN_ERR_INVALID_ARGUMENT and "twice" in msg


@pytest.mark.parametrize("kw,options,needle", [
    (dict(grad=0x100000), {}, "tensor 0: grad"),                      # the gradient is the parameter
    (dict(grad=0x120000 + 255), {}, "tensor 0: grad"),                # and by one byte a state
    (dict(grad=0x120000 - 255), {}, "tensor 0: grad"),
    (dict(step=0x120000 + 8), {}, "tensor 0: step"),                  # the counter lies in a state
    (dict(step=0x120000 - 4), {}, "tensor 0: step"),
    (dict(), dict(grad_scale=0x100000 + 4), "grad_scale"),
    (dict(), dict(lr_device=0x120000 + 252), "lr_device"),
    (dict(), dict(grad_scale=0x150004), "grad_scale"),                # the counter's ticket
])
def test_adamw_refuses_inputs_in_written_memory(kw, options, needle):
    rc, msg = _call(_options(**options), _tensors(**kw), 1)
    assert rc == _abi.DCN_ERR_INVALID_ARGUMENT and needle in msg and "overlap" in msg


def test_adamw_refuses_counters_that_overlap():
    t = _tensors(2)
    t[1].step = t[0].step + 4
    rc, msg = _call(_options(), t, 2)
    assert rc == _abi.DCN_ERR_INVALID_ARGUMENT and "counters" in msg


def test_adamw_empty_lists():
    assert _call(_options(), None, 0)[0] == _abi.DCN_OK
    assert _call(None, None, 0)[0] == _abi.DCN_ERR_INVALID_ARGUMENT
    assert _call(_options(), None, 2)[0] == _abi.DCN_ERR_INVALID_ARGUMENT
    assert _call(_options(), _tensors(), -1)[0] == _abi.DCN_ERR_INVALID_ARGUMENT


def test_grad_norm_refusals_and_workspace():
    lib = _abi.load()
    ref = (_abi.DcnTensorRef * 2)(_abi.DcnTensorRef(0x1000, 100, _abi.DCN_FLOAT32, 0),
                                  _abi.DcnTensorRef(None, 0, _abi.DCN_BFLOAT16, 0))
    need = lib.dcn_grad_norm_workspace_size(ref, 2)
    assert need >= 8

    def call(max_norm=1.0, scale=1.0, norm=0x2000, factor=0x2004, ws=0x4000, size=need, n=2):
        rc = lib.dcn_grad_norm(ref, n, max_norm, scale, norm, factor, ws, size, None)
        return rc, lib.dcn_last_error().decode()

    for kw, needle in ((dict(scale=0.0), "loss_scale"), (dict(scale=float("inf")), "loss_scale"),
                       (dict(max_norm=float("nan")), "max_norm"), (dict(norm=None), "NULL output"),
                       (dict(factor=None), "NULL output"), (dict(ws=None), "workspace"),
                       (dict(size=need - 1), "workspace"), (dict(n=-1), "tensor list")):
        rc, msg = call(**kw)
        assert rc != _abi.DCN_OK and needle in msg, kw
    ref[1] = _abi.DcnTensorRef(None, 5, _abi.DCN_BFLOAT16, 0)
    assert "NULL pointer" in call()[1]
    ref[1] = _abi.DcnTensorRef(0x1000, 5, 7, 0)
    assert "dtype" in call()[1]
    assert lib.dcn_grad_norm_workspace_size(ref, 2) == 0


def test_python_layer_refuses_cpu_tensors_and_bad_arguments():
    p = torch.zeros(4)
    with pytest.raises(ValueError, match="must be on CUDA device"):
        optim.adamw_step([p], [p], [p], [p], [optim.new_step("cpu")], lr=1e-3)
    with pytest.raises(ValueError, match="must be on CUDA device"):
        optim.grad_norm([p])
    with pytest.raises(ValueError, match="holds no gradient"):
        optim.grad_norm([None])
    q = torch.nn.Parameter(torch.zeros(4))
    for kw, needle in ((dict(lr=-1.0), "lr"), (dict(betas=(1.0, 0.9)), "betas"), (dict(eps=-1.0), "eps"),
                       (dict(weight_decay=-1.0), "weight_decay"), (dict(state_bits=4), "state_bits")):
        with pytest.raises(ValueError, match=needle):
            optim.AdamW([q], **kw)
    q.grad = torch.zeros(4)
    with pytest.raises(ValueError, match="must be on CUDA device"):
        optim.AdamW([q]).step()


def test_state_layouts():
    w = torch.empty(6, 5, 3, 3).to(memory_format=torch.channels_last)
    m, s = optim.new_state(w, 32)
    assert s is None and m.dtype == torch.float32 and m.stride() == w.stride() and not m.any()
    c, s = optim.new_state(w, 8)
    assert c.dtype == torch.float8_e4m3fn and c.stride() == w.stride() and s.shape == (2,)  # 270 elements
    assert not c.float().any()
    with pytest.raises(ValueError, match="state_bits"):
        optim.new_state(w, 4)


@pytest.mark.parametrize("kw,bits,needle", [
    (dict(param=0x100002), 32, "aligned"), (dict(param=0x100001, dtype=_abi.DCN_BFLOAT16), 32, "aligned"),
    (dict(grad=0x110002), 32, "aligned"), (dict(exp_avg=0x120002), 32, "aligned"),
    (dict(exp_avg_sq=0x130001), 32, "aligned"), (dict(master=0x140002), 32, "aligned"), (dict(step=0x150002), 32, "aligned"),
    (dict(exp_avg_scale=0x160002, exp_avg_sq_scale=0x170000), 8, "aligned"),
    (dict(exp_avg_scale=0x160000, exp_avg_sq_scale=0x170001), 8, "aligned"),
])
def test_adamw_refuses_pointers_off_their_elements(kw, bits, needle):
    """A kernel's access there would fault the GPU."""
    rc, msg = _call(_options(state_bits=bits), _tensors(**kw), 1)
    assert rc == _abi.DCN_ERR_INVALID_ARGUMENT and needle in msg


@pytest.mark.parametrize("options", [dict(grad_scale=0x900002), dict(lr_device=0x900001)])
def test_adamw_refuses_scalars_off_their_elements(options):
    rc, msg = _call(_options(**options), _tensors(), 1)
    assert rc == _abi.DCN_ERR_INVALID_ARGUMENT and "aligned" in msg


def test_grad_norm_refuses_pointers_off_their_elements():
    lib = _abi.load()

    def call(data=0x1000, dtype=_abi.DCN_FLOAT32, norm=0x2000, factor=0x2004, ws=0x4000):
        ref = (_abi.DcnTensorRef * 1)(_abi.DcnTensorRef(data, 100, dtype, 0))
        rc = lib.dcn_grad_norm(ref, 1, 1.0, 1.0, norm, factor, ws, 1 << 16, None)
        return rc, lib.dcn_last_error().decode()

    for kw in (dict(data=0x1002), dict(data=0x1001, dtype=_abi.DCN_FLOAT16), dict(norm=0x2002), dict(factor=0x2005),
               dict(ws=0x4004), dict(ws=0x4010)):
        rc, msg = call(**kw)
        assert rc == _abi.DCN_ERR_INVALID_ARGUMENT and "aligned" in msg, kw


def test_loading_keeps_the_learning_rate_tensor():
    """A schedule writes the tensor that the optimizer was made with."""
    def make(lr, lr2=None):
        p = [torch.nn.Parameter(torch.zeros(4)) for _ in range(2)]
        groups = [dict(params=[p[0]]), dict(params=[p[1]], **({} if lr2 is None else dict(lr=lr2)))]
        return optim.AdamW(groups, lr=lr)

    lr = torch.tensor(0.5)
    opt = make(lr)
    opt.load_state_dict(make(torch.tensor(0.25)).state_dict())
    assert all(g["lr"] is lr for g in opt.param_groups) and float(lr) == 0.25
    opt.load_state_dict(make(0.125).state_dict())  # saved by an optimizer with a plain number
    assert all(g["lr"] is lr for g in opt.param_groups) and float(lr) == 0.125
    opt.load_state_dict(make(0.75, 0.5).state_dict())  # one tensor cannot hold two values
    assert opt.param_groups[0]["lr"] is lr and [float(g["lr"]) for g in opt.param_groups] == [0.75, 0.5]
    plain, source = make(0.5), torch.tensor(0.25)
    plain.load_state_dict(make(source).state_dict())
    assert all(isinstance(g["lr"], torch.Tensor) and g["lr"] is not source and float(g["lr"]) == 0.25
               for g in plain.param_groups)


def test_loading_states_of_another_memory_format():
    """32-bit states come to the parameter's format with their values; codes cannot, as their scales go by
    memory order.  Scales and counters have shapes of their own and are taken as they are."""
    w = torch.randn(6, 5, 3, 3)

    def make(fmt, bits):
        p = torch.nn.Parameter(w.clone().contiguous(memory_format=fmt))
        opt = optim.AdamW([p], state_bits=bits)
        m, s = optim.new_state(p, bits)
        v, t = optim.new_state(p, bits)
        opt.state[p] = dict(step=optim.new_step("cpu", 3), exp_avg=m, exp_avg_sq=v)
        if bits == 8:
            opt.state[p].update(exp_avg_scale=s, exp_avg_sq_scale=t)
        else:
            m.copy_(w)
            v.copy_(w * w)
        return p, opt

    for a, b in ((torch.contiguous_format, torch.channels_last), (torch.channels_last, torch.contiguous_format)):
        _, source = make(a, 32)
        p, opt = make(b, 32)
        opt.load_state_dict(source.state_dict())
        state = opt.state[p]
        assert torch.equal(state["exp_avg"], w) and torch.equal(state["exp_avg_sq"], w * w)
        assert state["exp_avg"].stride() == state["exp_avg_sq"].stride() == p.stride()
        assert state["step"].tolist() == [3, 0]
        _, source = make(a, 8)
        p, opt = make(b, 8)
        before = dict(opt.state[p])
        with pytest.raises(ValueError, match="memory format"):
            opt.load_state_dict(source.state_dict())
        assert all(opt.state[p][k] is t for k, t in before.items())  # nothing was loaded
        _, same = make(b, 8)
        opt.load_state_dict(same.state_dict())
        assert opt.state[p]["exp_avg"].stride() == p.stride() and opt.state[p]["exp_avg_scale"].shape == (2,)


@pytest.mark.parametrize("eps", [1e-40, 2.0 ** -127, 1e-60])
def test_adamw_refuses_an_eps_that_fp32_flushes(eps):
    """A zero gradient on a zero state would become 0 / 0 where the formula says 0 / eps."""
    rc, msg = _call(_options(eps=eps), _tensors(), 1)
    assert rc == _abi.DCN_ERR_INVALID_ARGUMENT and "eps must be 0 or" in msg


def test_scalars_reach_parameters_on_every_device(monkeypatch):
    """Parameters on two devices and one factor and learning rate: each call gets them on its own device (else
    the second would be refused after the first had been stepped).  Fake tensors stand in for two GPUs.  A host
    tensor is left to the refusal of adamw_step: it would make every step wait."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    calls = []
    monkeypatch.setattr(optim, "adamw_step", lambda params, *a, **kw: calls.append((params[0], kw["lr"], kw["grad_scale"])))
    monkeypatch.setattr(optim.AdamW, "_init_state", lambda self, p, group: dict(step=p, exp_avg=p, exp_avg_sq=p))
    with FakeTensorMode():
        params = [torch.nn.Parameter(torch.zeros(4, device=f"cuda:{k}")) for k in range(2)]
        for p in params:
            p.grad = torch.zeros_like(p)
        lr, factor = torch.ones((), device="cuda:0"), torch.ones((), device="cuda:1")
        optim.AdamW(params, lr=lr).step(grad_scale=factor)
        assert [c[0].device.index for c in calls] == [0, 1]
        assert all(c[1].device == c[2].device == c[0].device for c in calls)
        assert calls[0][1] is lr and calls[1][2] is factor  # no copy where they are
        calls.clear()
        host = torch.ones(())
        optim.AdamW(params, lr=host).step()
        assert all(c[1] is host and c[2] is None for c in calls)
