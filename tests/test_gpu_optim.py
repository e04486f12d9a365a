"""The optimizer step and the gradient norm against plain implementations in 64 bits.

Error bounds count roundings, with u = 2^-24 for an fp32 operation or constant:
  m' = b1 m + (1 - b1) g: constant, (grad_scale,) product and sum: at most 4 per term
  v' = b2 v + (1 - b2) g^2: constant, two scalings, square, product and sum: at most 6
  update = step_size m' / (sqrt(v') corr + eps): v' enters by half (3), the root 1, corr and
    its product 2, eps and the sum 2, the quotient 4 (two units in the last place), the step
    size and its product 2, the difference 1: 15, besides the error of m'
  p' = p decay - update: constant, product and difference: 3
A 16-bit parameter adds half of its type's eps.
"""
import math

import pytest
import torch

from mps_deform_conv import optim

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
HYPER = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-7, weight_decay=0.1)
SIZES = [1, 7, 255, 256, 257, 2048, 8191, 8192, 8193, 40000, 0, 70001]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _inputs(sizes, dtype, dev, bits=32, master=False, misalign=False, seed=0):
    """Lists for adamw_step; with `misalign` every tensor starts one element into its storage."""
    g = _gen(seed)

    def put(t, dt):
        if not misalign:
            return t.to(dev, dt)
        if dt == torch.float8_e4m3fn:
            buf = torch.zeros(t.numel() + 1, device=dev, dtype=torch.uint8).view(dt)
        else:
            buf = torch.zeros(t.numel() + 1, device=dev, dtype=dt)
        buf[1:].copy_(t.to(dev, dt))
        return buf[1:]

    s = dict(params=[], grads=[], exp_avgs=[], exp_avg_sqs=[], steps=[], masters=[], scales=[], sq_scales=[])
    for n in sizes:
        p = torch.randn(n, generator=g)
        grad = torch.randn(n, generator=g) * 0.1
        m, v = torch.randn(n, generator=g) * 0.02, (torch.randn(n, generator=g) * 0.05) ** 2
        if n > 3:  # a gradient of zero on a state of zero, and one outlier
            grad[1] = m[1] = v[1] = 0.0
            grad[2] = 30.0
        s["params"].append(put(p, dtype))
        s["grads"].append(put(grad, dtype))
        if master:
            s["masters"].append(put(p, torch.float32))
        if bits == 8:
            for key, sk, x in (("exp_avgs", "scales", m), ("exp_avg_sqs", "sq_scales", v.sqrt())):
                b = torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256)
                scale = torch.exp2(torch.floor(torch.log2(b.abs().amax(1))).clamp(-100, 127) - 7)
                s[key].append(put((b / scale[:, None]).view(-1)[:n].to(torch.float8_e4m3fn), torch.float8_e4m3fn))
                s[sk].append(scale.to(dev))
        else:
            s["exp_avgs"].append(put(m, torch.float32))
            s["exp_avg_sqs"].append(put(v, torch.float32))
        s["steps"].append(optim.new_step(dev, int(torch.randint(0, 50, (1,), generator=g))))
    return s


def _call(s, bits=32, **kw):
    args = dict(HYPER, masters=s["masters"] or None, exp_avg_scales=s["scales"] if bits == 8 else None,
                exp_avg_sq_scales=s["sq_scales"] if bits == 8 else None)
    args.update(kw)
    optim.adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s["steps"], **args)


def _decoded(codes, scale):
    return codes.cpu().float() * scale.cpu().repeat_interleave(256)[:codes.numel()]


def _reference(s, k, bits, gs, hyper=HYPER):
    """(p', |update|, m', v', terms) of tensor k in 64 bits, before rounding the parameter."""
    lr, (b1, b2), eps, wd = hyper["lr"], hyper["betas"], hyper["eps"], hyper["weight_decay"]
    p = (s["masters"][k] if s["masters"] else s["params"][k]).cpu().double()
    g = s["grads"][k].cpu().double() * gs
    if bits == 8:
        m = _decoded(s["exp_avgs"][k], s["scales"][k]).double()
        v = _decoded(s["exp_avg_sqs"][k], s["sq_scales"][k]).double() ** 2
    else:
        m, v = s["exp_avgs"][k].cpu().double(), s["exp_avg_sqs"][k].cpu().double()
    t = int(s["steps"][k][0]) + 1
    m_new, v_new = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    denom = (v_new / (1 - b2 ** t)).sqrt() + eps
    rate = lr / (1 - b1 ** t)
    terms = (b1 * m).abs() + ((1 - b1) * g).abs()
    return p * (1 - lr * wd) - rate * m_new / denom, p, rate / denom, m_new, v_new, terms


def _assert_param(got, ref, p, rate, m_new, terms, dtype):
    err = 3 * U * p.abs() + 15 * U * (rate * m_new).abs() + rate * 4.1 * U * terms
    if dtype != torch.float32:
        err = err + (ref.abs() + err) * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bad = (got.cpu().double() - ref).abs() > 1.01 * err + 1e-38
    assert not bad.any(), (int(bad.sum()), got.cpu()[bad][:4], ref[bad][:4])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("misalign", [False, True])
@pytest.mark.parametrize("scaled", [False, True])
def test_adamw_32bit_states(dtype, master, misalign, scaled, cuda):
    if master and dtype == "float32":
        master = False
    dt = DTYPES[dtype]
    s = _inputs(SIZES, dt, cuda, master=master, misalign=misalign, seed=3)
    gs = 0.37 if scaled else 1.0
    scale = torch.tensor(gs, device=cuda) if scaled else None
    gs = float(scale) if scaled else 1.0
    refs = [_reference(s, k, 32, gs) for k in range(len(SIZES))]
    taken = [int(t[0]) for t in s["steps"]]
    _call(s, grad_scale=scale)
    torch.cuda.synchronize()
    for k in range(len(SIZES)):
        ref, p, rate, m_new, v_new, terms = refs[k]
        assert ((s["exp_avgs"][k].cpu().double() - m_new).abs() <= 4.1 * U * terms).all()
        assert ((s["exp_avg_sqs"][k].cpu().double() - v_new).abs() <= 6.1 * U * v_new).all()
        _assert_param(s["params"][k], ref, p, rate, m_new, terms, dt)
        if master:
            _assert_param(s["masters"][k], ref, p, rate, m_new, terms, torch.float32)
            assert torch.equal(s["masters"][k].to(dt), s["params"][k])
        assert s["steps"][k].tolist() == [taken[k] + 1, 0]


@pytest.mark.parametrize("scaled", [False, True])
def test_adamw_states_round_each_product_and_sum(scaled, cuda):
    """fp32 states are bit for bit those of separate fp32 products and sums."""
    s = _inputs([100000, 70001], torch.float32, cuda, seed=21)
    f = torch.tensor(0.37) if scaled else torch.tensor(1.0)
    b1, b2 = HYPER["betas"]
    want = []
    for g, m, v in zip(s["grads"], s["exp_avgs"], s["exp_avg_sqs"]):
        g, m, v = g.cpu() * f, m.cpu(), v.cpu()
        want.append((m * torch.tensor(b1) + g * torch.tensor(1 - b1),
                     v * torch.tensor(b2) + (g * g) * torch.tensor(1 - b2)))
    _call(s, grad_scale=f.to(cuda) if scaled else None)
    for k, (m, v) in enumerate(want):
        assert torch.equal(s["exp_avgs"][k].cpu(), m) and torch.equal(s["exp_avg_sqs"][k].cpu(), v)


# ---------------------------------------------------------------- 8-bit states
M32 = 0xFFFFFFFF


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & M32
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & M32
    return x ^ (x >> 16)


def _codes(x, words, positive):
    """The e4m3 codes and scales of one tensor: floor of (pattern + word) as the operator defines it."""
    n = x.numel()
    b = torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256)
    w = torch.nn.functional.pad(words, (0, -n % 256)).view(-1, 256)
    top = torch.where(torch.isfinite(b), b.abs(), torch.zeros_like(b)).amax(1)
    e = ((top.view(torch.int32) >> 23) - 127).clamp(min=-100)
    z = b.abs() * torch.exp2((7 - e).float())[:, None] * 2.0 ** -120
    c = (z.view(torch.int32).long() + (w << 4)) >> 20
    if positive:
        c = torch.where(b > 0, c.clamp(min=1), c)
    c = torch.where(torch.isfinite(b), c, torch.full_like(c, 0x7F)) | (torch.signbit(b).long() << 7)
    return c.view(-1)[:n].to(torch.uint8), torch.exp2((e - 7).float())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("misalign", [False, True])
@pytest.mark.parametrize("master", [False, True])
def test_adamw_8bit_states_bit_for_bit(dtype, misalign, master, cuda):
    """Codes and scales equal those of the definition, computed with one fp32 operation at a time."""
    dt = DTYPES[dtype]
    s = _inputs(SIZES, dt, cuda, bits=8, master=master, misalign=misalign, seed=5)
    scale = torch.tensor(0.61, device=cuda)
    f = torch.tensor(0.61)
    b1, b2 = HYPER["betas"]
    seed = 77
    want, refs = [], []
    for k, n in enumerate(SIZES):
        refs.append(_reference(s, k, 8, float(f)))
        g = s["grads"][k].cpu().float() * f
        m = _decoded(s["exp_avgs"][k], s["scales"][k])
        r = _decoded(s["exp_avg_sqs"][k], s["sq_scales"][k])
        m = m * torch.tensor(b1) + g * torch.tensor(1 - b1)
        r = ((r * r) * torch.tensor(b2) + (g * g) * torch.tensor(1 - b2)).sqrt()
        t = int(s["steps"][k][0]) + 1
        key = _mix((seed + t * 0x9E3779B9) & M32)
        w = _mix(torch.arange(n) ^ key)
        want.append((_codes(m, w & 0xFFFF, False), _codes(r, w >> 16, True)))
    _call(s, bits=8, grad_scale=scale, seed=seed)
    torch.cuda.synchronize()
    for k, n in enumerate(SIZES):
        for codes, scales, (c, sc) in ((s["exp_avgs"][k], s["scales"][k], want[k][0]),
                                       (s["exp_avg_sqs"][k], s["sq_scales"][k], want[k][1])):
            assert torch.equal(codes.view(torch.uint8).cpu(), c), (k, n)
            assert torch.equal(scales.cpu(), sc), (k, n)
        ref, p, rate, m_new, v_new, terms = refs[k]
        _assert_param(s["params"][k], ref, p, rate, m_new, terms, dt)


def test_8bit_rounding_is_unbiased_and_within_one_step(cuda):
    """One value everywhere: codes are its two neighbours, and their mean is it (five standard errors)."""
    n = 1 << 16
    value = 0.3  # of a block whose first element is 1
    grad = torch.full((n,), value)
    grad[::256] = 1.0
    s = dict(params=[torch.zeros(n, device=cuda)], grads=[grad.to(cuda)], steps=[optim.new_step(cuda)], masters=None)
    s["exp_avgs"], s["scales"] = zip(optim.new_state(s["params"][0], 8))
    s["exp_avg_sqs"], s["sq_scales"] = zip(optim.new_state(s["params"][0], 8))
    _call(s, bits=8, betas=(0.0, 0.0))
    for codes, scales in ((s["exp_avgs"][0], s["scales"][0]), (s["exp_avg_sqs"][0], s["sq_scales"][0])):
        x = _decoded(codes, scales).view(-1, 256)
        assert (x[:, 0] == 1.0).all()
        x = x[:, 1:].double()
        step = 2.0 ** -2 / 8  # values in [1/4, 1/2) are 2^-2 / 8 apart
        lo = math.floor(value / step) * step
        assert set(x.unique().tolist()) == {lo, lo + step}
        up = (value - lo) / step
        assert abs(float(x.mean()) - value) <= 5 * step * math.sqrt(up * (1 - up) / x.numel()) + step * 2.0 ** -16


def test_8bit_second_moment_never_rounds_to_zero(cuda):
    """Beside an outlier small gradients keep a positive root, so no update divides by eps alone."""
    n = 4096
    grad = torch.full((n,), 1e-9)
    grad[::256] = 1.0
    s = dict(params=[torch.zeros(n, device=cuda)], grads=[grad.to(cuda)], steps=[optim.new_step(cuda)], masters=None)
    s["exp_avgs"], s["scales"] = zip(optim.new_state(s["params"][0], 8))
    s["exp_avg_sqs"], s["sq_scales"] = zip(optim.new_state(s["params"][0], 8))
    _call(s, bits=8)
    assert (_decoded(s["exp_avg_sqs"][0], s["sq_scales"][0]) > 0).all()


def test_8bit_same_call_same_bits_and_seed_matters(cuda):
    outs = []
    for seed in (1, 1, 2):
        s = _inputs([5000], torch.bfloat16, cuda, bits=8, seed=9)
        _call(s, bits=8, seed=seed)
        outs.append(s["exp_avgs"][0].view(torch.uint8).cpu())
    assert torch.equal(outs[0], outs[1]) and not torch.equal(outs[0], outs[2])


# ---------------------------------------------------------------- calls
@pytest.mark.parametrize("count", [12, 13, 400, 900])
def test_many_tensors_share_one_counter(count, cuda):
    """More tensors than one launch takes, one counter for all: read by every launch, advanced once."""
    sizes = [(i * 37) % 300 for i in range(count)]
    s = _inputs(sizes, torch.float32, cuda, seed=1)
    step = optim.new_step(cuda, 7)
    s["steps"] = [step] * count
    refs = [_reference(s, k, 32, 1.0) for k in range(count)]
    _call(s)
    assert step.tolist() == [8, 0]
    for k in range(count):
        ref, p, rate, m_new, _, terms = refs[k]
        _assert_param(s["params"][k], ref, p, rate, m_new, terms, torch.float32)


def test_mixed_dtypes_share_one_counter(cuda):
    parts = [_inputs([700, 300], dt, cuda, seed=i) for i, dt in enumerate(DTYPES.values())]
    s = {k: sum((p[k] for p in parts), []) for k in parts[0]}
    s["steps"] = [optim.new_step(cuda, 3)] * 6
    refs = [_reference(s, k, 32, 1.0) for k in range(6)]
    _call(s)
    assert s["steps"][0].tolist() == [4, 0]
    for k in range(6):
        ref, p, rate, m_new, _, terms = refs[k]
        _assert_param(s["params"][k], ref, p, rate, m_new, terms, s["params"][k].dtype)


def test_only_empty_tensors_advance(cuda):
    s = _inputs([0, 0], torch.float32, cuda)
    s["steps"] = [optim.new_step(cuda, 3), optim.new_step(cuda, 5)]
    _call(s)
    assert [t.tolist() for t in s["steps"]] == [[4, 0], [6, 0]]


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("bits", [32, 8])
def test_factor_that_is_not_finite_skips_the_step(bad, bits, cuda):
    s = _inputs([9000, 5], torch.bfloat16, cuda, bits=bits, master=True)
    s["grads"][0][3] = float("inf")
    tensors = lambda: [t.view(torch.uint8).clone() for k in s for t in s[k]]  # noqa: E731
    before = tensors()
    _call(s, bits=bits, grad_scale=torch.tensor(bad, device=cuda))
    assert all(torch.equal(a, b) for a, b in zip(before, tensors()))


def test_non_finite_gradients_stay_in_their_elements(cuda):
    for bits in (32, 8):
        s = _inputs([1000], torch.float32, cuda, bits=bits, seed=2)
        s["grads"][0][300] = float("inf")
        s["grads"][0][301] = float("nan")
        _call(s, bits=bits)
        bad = ~torch.isfinite(s["params"][0])
        assert bad.nonzero().view(-1).tolist() == [300, 301]
        states = s["exp_avgs"][0].float()
        assert (~torch.isfinite(states)).nonzero().view(-1).tolist() == [300, 301]


def test_memory_formats(cuda):
    """A channels_last parameter, with a gradient in its format and in the other one."""
    g = _gen(4)
    w = torch.randn(8, 6, 3, 3, generator=g)
    grad = torch.randn(8, 6, 3, 3, generator=g)
    out = []
    for fmt, gfmt in ((torch.contiguous_format, torch.contiguous_format), (torch.channels_last, torch.channels_last),
                      (torch.channels_last, torch.contiguous_format)):
        p = w.to(cuda).contiguous(memory_format=fmt)
        m, _ = optim.new_state(p)
        v, _ = optim.new_state(p)
        optim.adamw_step([p], [grad.to(cuda).contiguous(memory_format=gfmt)], [m], [v], [optim.new_step(cuda)], **HYPER)
        out.append(p.cpu().contiguous())
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])


def test_refusals(cuda):
    s = _inputs([64, 64], torch.float32, cuda)
    p = s["params"][0]

    def bad(needle, **kw):
        t = {k: list(v) for k, v in s.items()}
        t.update(kw)
        with pytest.raises((RuntimeError, ValueError), match=needle):
            _call(t)

    bad("grads has 1", grads=s["grads"][:1])
    bad("overlap", params=[p, p])
    bad("overlap", exp_avgs=[s["exp_avgs"][0], s["exp_avgs"][0]])
    bad("exp_avgs", exp_avgs=[t.half() for t in s["exp_avgs"]])
    bad("grads", grads=[t.half() for t in s["grads"]])
    bad("grads", grads=[t[:32] for t in s["grads"]])
    bad("steps", steps=[t.float() for t in s["steps"]])
    bad("steps", steps=[t[:1] for t in s["steps"]])
    bad("dense", params=[torch.zeros(128, device=cuda)[::2], s["params"][1]])
    bad("CUDA", grads=[t.cpu() for t in s["grads"]])
    bad("masters", masters=[t.bfloat16() for t in s["params"]])
    with pytest.raises(RuntimeError, match="grad_scale"):
        _call(s, grad_scale=torch.ones(2, device=cuda))
    with pytest.raises(RuntimeError, match="lr must be one float32"):
        _call(s, lr=torch.ones((), device=cuda, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="lr must be"):
        _call(s, lr=-1.0)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        q = torch.zeros(4, device=cuda, dtype=torch.float64)
        optim.adamw_step([q], [q.clone()], [torch.zeros(4, device=cuda)], [torch.zeros(4, device=cuda)],
                         [optim.new_step(cuda)], lr=1e-3)


def test_device_learning_rate_and_graph_replay(cuda):
    """A captured step follows the counter, the factor and the learning rate on the device."""
    ref = _inputs([5000, 100], torch.bfloat16, cuda, bits=8, master=True, seed=6)
    s = _inputs([5000, 100], torch.bfloat16, cuda, bits=8, master=True, seed=6)
    lr = torch.tensor(1e-3, device=cuda)
    factor = torch.tensor(0.5, device=cuda)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            _call(s, bits=8, lr=lr, grad_scale=factor, seed=3)
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in ((1e-3, 0.5), (2e-3, 0.25), (5e-4, float("nan")), (5e-4, 1.0)):
        lr.fill_(a)
        factor.fill_(b)
        graph.replay()
        _call(ref, bits=8, lr=float(lr), grad_scale=torch.tensor(b, device=cuda), seed=3)
    torch.cuda.synchronize()
    for k in ("params", "masters", "exp_avgs", "exp_avg_sqs", "steps", "scales", "sq_scales"):
        for x, y in zip(s[k], ref[k]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), k
    assert s["steps"][0][0] == ref["steps"][0][0]


def test_update_is_seen_by_the_weight_image_cache_and_autograd(cuda):
    """The step bumps version counters: a cached forward weight image is rebuilt, and a graph that
    saved the parameter refuses to run backward."""
    import mps_deform_conv as mdc
    torch.manual_seed(0)
    layer = mdc.DeformConv2d(64, 64, 3, padding=1, bias=False).to(cuda, torch.bfloat16)
    x = torch.randn(1, 64, 8, 8, device=cuda, dtype=torch.bfloat16)
    off = torch.zeros(1, 18, 8, 8, device=cuda, dtype=torch.bfloat16)
    opt = optim.AdamW(layer.parameters(), lr=0.1)
    mdc.set_weight_image_cache(True)
    try:
        with torch.no_grad():
            layer(x, off)
            layer.weight.grad = torch.randn_like(layer.weight)
            opt.step()
            cached = layer(x, off)
        mdc.set_weight_image_cache(False)
        with torch.no_grad():
            assert torch.equal(cached, layer(x, off))
    finally:
        mdc.set_weight_image_cache(False)
    y = (layer.weight * layer.weight).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("bits,master", [(32, False), (32, True), (8, True)])
def test_optimizer_class(bits, master, cuda):
    """The class takes the same steps as the function, keeps its state over a save and a load, skips
    parameters without a gradient, and captures."""
    torch.manual_seed(1)
    make = lambda: [torch.nn.Parameter(torch.randn(n, device=cuda, generator=torch.Generator(cuda).manual_seed(n)).to(dt))  # noqa: E731
                    for n, dt in ((300, torch.bfloat16), (77, torch.bfloat16), (1000, torch.float32))]
    a, b = make(), make()
    oa = optim.AdamW([dict(params=a[:2], weight_decay=0.0), dict(params=a[2:])], lr=1e-2, state_bits=bits,
                     master_weights=master, seed=4)
    ob = optim.AdamW([dict(params=b[:2], weight_decay=0.0), dict(params=b[2:])], lr=1e-2, state_bits=bits,
                     master_weights=master, seed=4)
    with pytest.raises(RuntimeError, match="take one step before capturing"):
        a[0].grad = torch.ones_like(a[0])
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            oa.step()
    oa.state.clear()
    for it in range(4):
        for k, (p, q) in enumerate(zip(a, b)):
            p.grad = None if (it == 1 and k == 1) else torch.randn_like(p)
            q.grad = p.grad
        oa.step()
        if it == 2:  # continue from a saved state
            ob.load_state_dict(ob.state_dict())
        if it == 1:
            saved = ob.state_dict()
            ob = optim.AdamW([dict(params=b[:2]), dict(params=b[2:])], lr=1.0, state_bits=bits, master_weights=master)
            ob.load_state_dict(saved)
        ob.step()
    torch.cuda.synchronize()
    assert oa.state[a[1]]["step"].tolist() == [3, 0] and oa.state[a[0]]["step"].tolist() == [4, 0]
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for key, value in oa.state[p].items():
            other = ob.state[q][key]
            assert value.dtype == other.dtype and torch.equal(value.view(torch.uint8), other.view(torch.uint8)), key
    assert ("master" in oa.state[a[0]]) == master and "master" not in oa.state[a[2]]
    assert oa.state[a[0]]["exp_avg"].dtype == (torch.float8_e4m3fn if bits == 8 else torch.float32)
    calls = []
    assert oa.step(closure=lambda: calls.append(1) or 5.0) == 5.0 and calls == [1]


# ---------------------------------------------------------------- gradient norm
def _norm_ref(grads):
    return math.sqrt(sum(float((g.cpu().double() ** 2).sum()) for g in grads))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("misalign", [False, True])
def test_grad_norm(dtype, misalign, cuda):
    """Sums of squares carry 9 fp32 roundings per 8 elements (halved by the root); one more at the end."""
    g = _gen(8)
    grads = []
    for n in SIZES + [300000]:
        t = torch.randn(n + 1, generator=g).to(cuda, DTYPES[dtype])
        grads.append(t[1:] if misalign else t[:n].clone())
    ref = _norm_ref(grads) / 4.0
    for max_norm in (None, 0.0, ref / 3, ref * 3):
        norm, factor = optim.grad_norm(grads, max_norm=max_norm, loss_scale=4.0)
        assert norm.shape == factor.shape == () and norm.dtype == torch.float32
        assert abs(float(norm) - ref) <= 6 * U * ref
        want = (1.0 if max_norm is None else min(1.0, max_norm / (ref + 1e-6))) / 4.0
        assert abs(float(factor) - want) <= 7 * U * want
        again = optim.grad_norm(grads, max_norm=max_norm, loss_scale=4.0)
        assert torch.equal(again[0], norm) and torch.equal(again[1], factor)


def test_grad_norm_range(cuda):
    """Squares outside fp32's range, zeros, and gradients that are not finite."""
    big = torch.full((5000,), 1e25, device=cuda)
    tiny = torch.full((5000,), 1e-30, device=cuda)
    for t in (big, tiny, big.bfloat16()):
        ref = _norm_ref([t])
        norm, factor = optim.grad_norm([t], max_norm=1.0)
        assert abs(float(norm) - ref) <= 6 * U * ref
        want = min(1.0, 1.0 / (ref + 1e-6))
        assert abs(float(factor) - want) <= 7 * U * want
    zero = torch.zeros(100, device=cuda)
    norm, factor = optim.grad_norm([zero, torch.empty(0, device=cuda)], max_norm=1.0)
    assert float(norm) == 0.0 and float(factor) == 1.0
    for bad in (float("inf"), float("nan")):
        t = torch.ones(10000, device=cuda)
        t[7777] = bad
        norm, factor = optim.grad_norm([zero, t], max_norm=1.0)
        assert not math.isfinite(float(norm)) and math.isnan(float(factor))
    huge = torch.full((100,), 3e38, device=cuda)  # the norm itself leaves fp32
    norm, factor = optim.grad_norm([huge], max_norm=1.0)
    assert math.isinf(float(norm)) and math.isnan(float(factor))


def test_grad_norm_many_tensors_and_strides(cuda):
    g = _gen(10)
    grads = [torch.randn((i * 31) % 97, generator=g).to(cuda, list(DTYPES.values())[i % 3]) for i in range(1500)]
    grads.append(torch.randn(64, 50, generator=g).to(cuda).t())           # dense, other order
    grads.append(torch.randn(64, 50, generator=g).to(cuda)[:, ::2])       # gaps
    grads.append(torch.randn(1, 5, generator=g).to(cuda).expand(7, 5))    # the same row seven times
    ref = _norm_ref(grads)
    norm, _ = optim.grad_norm(grads)
    assert abs(float(norm) - ref) <= 6 * U * ref
    with pytest.raises(ValueError, match="max_norm"):
        optim.grad_norm(grads, max_norm=-1.0)
    with pytest.raises(RuntimeError, match="loss_scale"):
        optim.grad_norm(grads, loss_scale=0.0)


def test_training_step_norm_then_adamw_on_a_side_stream(cuda):
    """The two as they are used: clip and step, on another stream than the tensors'."""
    s = _inputs([40000, 300], torch.float16, cuda, master=True, seed=12)
    ref_norm = _norm_ref(s["grads"]) / 8.0
    factor64 = min(1.0, 1.0 / (ref_norm + 1e-6)) / 8.0
    refs = [_reference(s, k, 32, factor64) for k in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm, factor = optim.grad_norm(s["grads"], max_norm=1.0, loss_scale=8.0)
        _call(s, grad_scale=factor)
    torch.cuda.current_stream().wait_stream(side)
    assert abs(float(norm) - ref_norm) <= 6 * U * ref_norm
    for k in range(2):
        ref, p, rate, m_new, _, terms = refs[k]
        # the factor's own error (7 roundings) enters the gradient once and its square's root once
        err = 3 * U * p.abs() + 30 * U * (rate * m_new).abs() + rate * 12 * U * terms
        assert ((s["masters"][k].cpu().double() - ref).abs() <= err).all()


def test_loading_a_checkpoint_mapped_to_the_cpu(cuda, tmp_path):
    """States and the learning rate come back to the device, the latter into the optimizer's own tensor."""
    def make():
        p = torch.nn.Parameter(torch.linspace(-1, 1, 3000, device=cuda).bfloat16())
        p.grad = torch.linspace(1, -1, 3000, device=cuda).bfloat16()
        return p, optim.AdamW([p], lr=torch.tensor(1e-2, device=cuda), state_bits=8, master_weights=True)

    p, opt = make()
    opt.step()
    opt.param_groups[0]["lr"].fill_(3e-2)
    torch.save([p.detach(), opt.state_dict()], tmp_path / "checkpoint")
    opt.step()
    q, other = make()
    lr = other.param_groups[0]["lr"]
    value, state = torch.load(tmp_path / "checkpoint", map_location="cpu")
    other.load_state_dict(state)
    with torch.no_grad():
        q.copy_(value)
    assert other.param_groups[0]["lr"] is lr
    other.step()
    assert torch.equal(p, q)
    assert all(torch.equal(a.view(torch.uint8), other.state[q][k].view(torch.uint8)) for k, a in opt.state[p].items())


def test_smallest_eps_divides_zero_by_it(cuda):
    p = torch.ones(300, device=cuda)
    zero = lambda: torch.zeros(300, device=cuda)  # noqa: E731
    optim.adamw_step([p], [zero()], [zero()], [zero()], [optim.new_step(cuda)], lr=1e-3, eps=2.0 ** -126, weight_decay=0.0)
    assert torch.equal(p, torch.ones_like(p))
