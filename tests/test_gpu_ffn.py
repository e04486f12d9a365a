"""The gated feed-forward block against the formulas in 64 bits.

Bounds are elementwise and count roundings:
  * a sum of n products carries at most one truncation of its running value per 16 terms
    (a matrix instruction's step) and a few more: ``_sum_err`` times the sum of the
    products' absolute values.  fp32 data runs six such passes, and drops terms below
    3 * 2^-24 of a product;
  * the hidden values and their gradients are rounded to the type (half of its eps) as
    operands (the bounds count it for the bias gradients' summands too); saved gate and up
    values of 16-bit data (more than 256 channels) to 11 bits;
  * errors of gate and up enter the activation by its largest slope, those of its derivative
    by the largest curvature (relu: a sign may change where gate is within its own error);
  * 16-bit data: the fast exponential and quotient leave 2^-19 of an activation's value, the
    fitted normal distribution function 2^-17; fp32: 2^-21.
"""
import math

import pytest
import torch

import mps_deform_conv as mdc

pytestmark = pytest.mark.gpu

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SLOPE = {"silu": 1.1, "gelu": 1.13, "relu": 1.0, "sigmoid": 0.25}
CURVE = {"silu": 0.5, "gelu": 0.8, "relu": 0.0, "sigmoid": 0.1}
NAMES = ["y", "dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down"]


def _sum_err(n, dtype):
    return ((6 if dtype == torch.float32 else 1) * math.ceil(n / 16) + 4) * 2.0 ** -23


def _act(x, kind):
    if kind == "relu":
        on = (x > 0).to(x.dtype)
        return x * on, on
    if kind == "gelu":
        c = torch.special.ndtr(x)
        return x * c, c + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(x)
    if kind == "sigmoid":
        return s, s * (1 - s)
    return x * s, s * (1 + x * (1 - s))


def _inputs(m, c, f, dtype, dev, bias=True, seed=0):
    g = torch.Generator(dev).manual_seed(seed)
    r = lambda *s, scale=1.0: (torch.randn(s, generator=g, device=dev) * scale).to(dtype)  # noqa: E731
    t = [r(m, c), r(f, c, scale=c ** -0.5), r(f, c, scale=c ** -0.5), r(c, f, scale=f ** -0.5)]
    return t + ([r(f, scale=0.3), r(f, scale=0.3), r(c, scale=0.3)] if bias else [None] * 3), r(m, c)


def _reference(args, dy, act, dtype):
    """[(value, bound)] of y and the gradients, in 64 bits."""
    x, wg, wu, wd, bg, bu, bd = [None if t is None else t.detach().double() for t in args]
    (m, c), f = x.shape, wg.shape[0]
    u = torch.finfo(dtype).eps / 2
    wide = dtype == torch.float32
    floor = 2.0 ** -25 if dtype == torch.float16 else 1e-38
    fast = 2.0 ** (-21 if wide else -17 if act == "gelu" else -19)
    z = lambda t: 0.0 if t is None else t  # noqa: E731
    ab = lambda t: 0.0 if t is None else t.abs()  # noqa: E731
    gate, up = x @ wg.t() + z(bg), x @ wu.t() + z(bu)
    e_g = _sum_err(c, dtype) * (x.abs() @ wg.abs().t() + ab(bg))
    e_u = _sum_err(c, dtype) * (x.abs() @ wu.abs().t() + ab(bu))
    a, da = _act(gate, act)
    e_a = SLOPE[act] * e_g + fast * (a.abs() + e_g)
    h = a * up
    e_h = e_a * (up.abs() + e_u) + a.abs() * e_u
    e_h = e_h + (0 if wide else u) * (h.abs() + e_h) + floor
    y = h @ wd.t() + z(bd)
    e_y = e_h @ wd.abs().t() + _sum_err(f, dtype) * (h.abs() @ wd.abs().t() + ab(bd))
    done = lambda v, e: (v, e + u * (v.abs() + e) + floor)  # noqa: E731
    out = [done(y, e_y)]
    if dy is None:
        return out
    dy = dy.double()
    dh = dy @ wd
    e_dh = _sum_err(c, dtype) * (dy.abs() @ wd.abs())
    if not wide and c > 256:  # gate and up come back from the saved state with 11 bits
        # (a subnormal's step where the largest of 16 columns is at least 2^-4, else relative to that)
        e_g = e_g + 2.0 ** -11 * (gate.abs() + e_g) + (2.0 ** -36 * gate.abs()).amax(1, keepdim=True).clamp(min=2.0 ** -25)
        e_u = e_u + 2.0 ** -11 * (up.abs() + e_u) + (2.0 ** -36 * up.abs()).amax(1, keepdim=True).clamp(min=2.0 ** -25)
        e_a = SLOPE[act] * e_g + fast * (a.abs() + e_g)
    e_da = CURVE[act] * e_g + fast * 2
    if act == "relu":
        e_da = e_da + (gate.abs() <= e_g).double()
    dup = dh * a
    e_dup = e_dh * (a.abs() + e_a) + dh.abs() * e_a + 2.0 ** -23 * dup.abs()
    dgate = dh * up * da
    e_dgate = (e_dh * (up.abs() + e_u) + dh.abs() * e_u) * (da.abs() + e_da) + (dh * up).abs() * e_da + 2.0 ** -22 * dgate.abs()
    if not wide:
        e_dup = e_dup + u * (dup.abs() + e_dup) + floor
        e_dgate = e_dgate + u * (dgate.abs() + e_dgate) + floor
    sm = _sum_err(m, dtype)
    dx = dgate @ wg + dup @ wu
    e_dx = e_dgate @ wg.abs() + e_dup @ wu.abs() + _sum_err(2 * f, dtype) * (dgate.abs() @ wg.abs() + dup.abs() @ wu.abs())
    out.append(done(dx, e_dx))
    for d, e in ((dgate, e_dgate), (dup, e_dup)):
        out.append(done(d.t() @ x, e.t() @ x.abs() + sm * (d.abs().t() @ x.abs())))
    out.append(done(dy.t() @ h, dy.abs().t() @ e_h + sm * (dy.abs().t() @ h.abs())))
    if bg is not None:
        lin = (m / 32 + 40) * 2.0 ** -24    # running sums of fp32 values
        out += [done(d.sum(0), e.sum(0) + lin * d.abs().sum(0)) for d, e in ((dgate, e_dgate), (dup, e_dup))]
    if bd is not None:
        out.append(done(dy.sum(0), (m / 32 + 40) * 2.0 ** -24 * dy.abs().sum(0)))
    return out


def _check(got, ref, what=""):
    names = NAMES if len(ref) == len(NAMES) else NAMES[:5]
    for name, t, (v, e) in zip(names, got, ref):
        assert t.shape == v.shape, (what, name)
        t = t.double()
        bad = ~((t - v).abs() <= e)
        assert not bad.any(), (f"{what} {name}: {int(bad.sum())} of {bad.numel()} outside; first at "
                               f"{bad.nonzero()[0].tolist()}: {t[bad][0].item()} for {v[bad][0].item()}, "
                               f"bound {e[bad][0].item():.3e}; rel {float((t - v).norm() / v.norm()):.2e}")


def _run(args, dy, act):
    """y and, with dy, the gradients of every given tensor, in NAMES' order."""
    if dy is None:
        with torch.no_grad():
            return [mdc.gated_feed_forward(*args, activation=act)]
    leaves = [t if t is None else t.detach().requires_grad_(True) for t in args]
    y = mdc.gated_feed_forward(*leaves, activation=act)
    return [y.detach(), *torch.autograd.grad(y, [t for t in leaves if t is not None], dy)]


SIZES = [(1, 8, 8), (1, 512, 2048), (2, 1, 1), (3, 5, 7), (31, 64, 64), (127, 64, 136), (128, 64, 128), (129, 72, 200),
         (300, 100, 267), (257, 24, 40), (640, 96, 255), (1000, 256, 1024), (700, 320, 33), (4100, 64, 170),
         (9000, 128, 512), (2000, 512, 300), (513, 264, 520), (90, 257, 65)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward_and_backward(size, dtype, cuda):
    dt = DTYPES[dtype]
    bias = size[0] % 2 == 1 or size[1] % 8 != 0
    args, dy = _inputs(*size, dt, cuda, bias, seed=sum(size))
    got = _run(args, dy, "silu")
    torch.cuda.synchronize()
    mdc._get_lib().device_status()
    _check(got, _reference(args, dy, "silu", dt), f"{size} {dtype}")
    _check(_run(args, None, "silu"), _reference(args, None, "silu", dt), f"{size} {dtype} forward alone")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("act", list(SLOPE))
@pytest.mark.parametrize("bias", [True, False])
def test_activations(act, bias, dtype, cuda):
    dt = DTYPES[dtype]
    args, dy = _inputs(200, 64, 96, dt, cuda, bias, seed=5)
    args[0] = args[0] * 6  # far into both tails
    _check(_run(args, dy, act), _reference(args, dy, act, dt), f"{act} {dtype}")
    few, _ = _inputs(5, 64, 96, dt, cuda, bias, seed=6)
    few[0] = few[0] * 6
    _check(_run(few, None, act), _reference(few, None, act, dt), f"{act} {dtype} few rows")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 64])
def test_few_rows(m, dtype, cuda):
    """Single vectors and small batches while serving, widths with and without remainders."""
    dt = DTYPES[dtype]
    for c, f in ((256, 1000), (520, 88), (64, 4096), (1000, 72), (2048, 512), (33, 31)):
        args, _ = _inputs(m, c, f, dt, cuda, f % 16 == 8, seed=m + c)
        _check(_run(args, None, "silu"), _reference(args, None, "silu", dt), f"{(m, c, f)}")


@pytest.mark.parametrize("channels,dtype", [(512, "bf16"), (64, "bf16"), (64, "fp16")])
def test_bias_gradients_sum_unrounded_values(channels, dtype, cuda):
    """Sums of mixed signs over many rows.  Their error is the result's own rounding, 1 in its units, beside
    values that keep at least three bits more than the type (saved gate and up: 2 x (1/8)^2 in squares); the
    norm over 1536 columns scatters by 1 / sqrt(2 x 1536) = 2 %, six of which are allowed for.  Summands
    rounded to the type would add as much as the result's rounding: 1.41."""
    dt = {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    args, dy = _inputs(20000, channels, 1536, dt, cuda, True, seed=21)
    got = _run(args, dy, "silu")
    ref = _reference(args, dy, "silu", dt)
    for name in ("db_gate", "db_up"):
        k = NAMES.index(name)
        exact = ref[k][0]
        own = float((got[k].double() - exact).norm())
        rounded = float((exact.to(dt).double() - exact).norm())
        assert own <= rounded * (1 + 2 / 64) ** 0.5 * 1.12, (name, own / rounded)


def test_strides_views_and_alignment(cuda):
    """Packed weights, transposed weights, strided rows, storages that start off a 16-byte boundary."""
    dt = torch.bfloat16
    args, dy = _inputs(150, 64, 96, dt, cuda, True, seed=3)
    ref = _reference(args, dy, "gelu", dt)
    packed = torch.cat([args[1], args[2]])
    wide = torch.zeros(150, 80, device=cuda, dtype=dt)
    wide[:, 8:72] = args[0]
    odd = torch.zeros(150 * 64 + 1, device=cuda, dtype=dt)
    odd[1:] = args[0].reshape(-1)
    variants = [
        [args[0], packed[:96], packed[96:], *args[3:]],
        [wide[:, 8:72], *args[1:]],
        [odd[1:].view(150, 64), *args[1:]],
        [args[0].t().contiguous().t(), args[1].t().contiguous().t(), *args[2:]],
        [args[0], args[1], args[2], args[3].t().contiguous().t(), *args[4:]],
    ]
    for v in variants:
        _check(_run(v, dy, "gelu"), ref, "layout variant")
    _check(_run(args, dy.t().contiguous().t(), "gelu"), ref, "strided grad")
    one = dy[:1].expand(150, 64)
    _check(_run(args, one, "gelu"), _reference(args, one, "gelu", dt), "broadcast grad")
    x5 = args[0].view(5, 3, 10, 64)
    leaves = [x5.detach().requires_grad_(True)] + args[1:]
    y = mdc.gated_feed_forward(*leaves, activation="gelu")
    gx, = torch.autograd.grad(y, leaves[:1], dy.view(5, 3, 10, 64))
    assert y.shape == x5.shape and gx.shape == x5.shape
    _check([y.detach().view(150, 64), gx.view(150, 64)], ref[:2])


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_no_rows(dtype, cuda):
    args, dy = _inputs(0, 16, 24, DTYPES[dtype], cuda, True)
    got = _run(args, dy, "silu")
    assert got[0].shape == (0, 16) and got[1].shape == (0, 16)
    for g, t in zip(got[2:], args[1:]):
        assert g.shape == t.shape and not g.any()


def test_gradients_by_need_and_training_cache(cuda):
    """Any subset of gradients has the bits of the full set, with and without the training cache."""
    args, dy = _inputs(260, 72, 104, torch.bfloat16, cuda, True, seed=8)
    full = _run(args, dy, "silu")
    masks = [[i == k for i in range(7)] for k in range(7)] + [[True, False, False, True, False, False, False],
                                                              [False, True, True, False, True, True, False]]
    try:
        for cache in (True, False):
            mdc.set_training_cache(cache)
            for a, b in zip(_run(args, dy, "silu"), full):
                assert torch.equal(a, b)
            for mask in masks:
                leaves = [t.detach().requires_grad_(n) for t, n in zip(args, mask)]
                y = mdc.gated_feed_forward(*leaves)
                got = torch.autograd.grad(y, [t for t, n in zip(leaves, mask) if n], dy)
                want = [g for g, n in zip(full[1:], mask) if n]
                assert all(torch.equal(a, b) for a, b in zip(got, want)), mask
    finally:
        mdc.set_training_cache(True)


def test_reproducible_bit_for_bit(cuda):
    for dt in DTYPES.values():
        args, dy = _inputs(5000, 128, 264, dt, cuda, True, seed=9)
        a, b = _run(args, dy, "silu"), _run(args, dy, "silu")
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_gradient_against_differences(act, cuda):
    """Directional differences of the fp32 forward: third order leaves eps^2 / 6 of the third derivative
    (estimated by halving eps), the forward's own error is divided by eps.  The errors of the output's
    elements are independent of the direction and add in quadrature (six standard deviations, each at
    most its element's bound)."""
    args, dy = _inputs(70, 40, 56, torch.float32, cuda, True, seed=10)
    grads = _run(args, dy, act)[1:]
    g = torch.Generator(cuda).manual_seed(1)

    def loss(ts):
        with torch.no_grad():
            return float((mdc.gated_feed_forward(*ts, activation=act).double() * dy.double()).sum())

    noise = 6 * float((_reference(args, None, act, torch.float32)[0][1] * dy.double()).norm())
    for k, t in enumerate(args):
        d = torch.randn(t.shape, generator=g, device=cuda)
        diff = []
        for eps in (2.0 ** -6, 2.0 ** -7):
            plus, minus = list(args), list(args)
            plus[k], minus[k] = t + eps * d, t - eps * d
            # the perturbed operands are themselves rounded to fp32
            step = (plus[k].double() - minus[k].double())
            scale = float((step * d.double()).sum() / (2 * (d.double() ** 2).sum()))
            diff.append((loss(plus) - loss(minus)) / (2 * scale))
        want = float((grads[k].double() * d.double()).sum())
        tol = 2 * abs(diff[0] - diff[1]) + 2 * noise / 2.0 ** -7
        assert abs(diff[1] - want) <= tol, (k, diff, want, tol)
        assert tol <= 0.05 * abs(want) + 0.05 * float(grads[k].norm() * d.norm())  # the check says something


def test_second_order_is_refused(cuda):
    args, dy = _inputs(8, 16, 16, torch.float32, cuda, False)
    x = args[0].requires_grad_(True)
    y = mdc.gated_feed_forward(x, *args[1:])
    g, = torch.autograd.grad(y, x, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_non_finite_rows_stay_in_their_rows(cuda):
    for dt in DTYPES.values():
        args, dy = _inputs(300, 64, 96, dt, cuda, True, seed=11)
        clean = _run(args, dy, "silu")
        x = args[0].clone()
        x[5, 3] = float("nan")
        x[299, 0] = float("inf")
        got = _run([x, *args[1:]], dy, "silu")
        keep = torch.ones(300, dtype=torch.bool, device=cuda)
        keep[5] = keep[299] = False
        assert got[0][5].isnan().all() and got[1][5].isnan().all() and not got[0][299].isfinite().any()
        assert torch.equal(got[0][keep], clean[0][keep]) and torch.equal(got[1][keep], clean[1][keep])
        # a NaN in one hidden unit's weights stays in that unit's weight gradients
        w = args[1].clone()
        w[40, 7] = float("nan")
        got = _run([args[0], w, *args[2:]], dy, "silu")
        rows = torch.ones(96, dtype=torch.bool, device=cuda)
        rows[40] = False
        for k in (2, 3):
            assert got[k][40].isnan().all() and torch.equal(got[k][rows], clean[k][rows])
        assert got[4][:, 40].isnan().all() and torch.equal(got[4][:, rows], clean[4][:, rows])


def test_far_tails_and_small_values_of_the_saved_state(cuda):
    """Gate and up many decades apart in one row, and beyond fp16's range in bf16."""
    dt = torch.bfloat16
    args, dy = _inputs(64, 32, 64, dt, cuda, False, seed=12)
    scale = torch.exp2(torch.linspace(-20, 20, 64, device=cuda)).to(dt)
    args[2] = args[2] * scale[:, None]
    args[1] = args[1] * scale.flip(0)[:, None]
    for act in ("silu", "relu"):
        _check(_run(args, dy, act), _reference(args, dy, act, dt), "decades")


def test_offsets_past_32_bits(cuda):
    """More than 2^31 hidden values: rows at both ends against the formulas."""
    m, c, f = 1_050_000, 16, 2056
    dt = torch.bfloat16
    args, dy = _inputs(m, c, f, dt, cuda, False, seed=13)
    got = _run(args, dy, "silu")
    rows = torch.cat([torch.arange(0, 40), torch.arange(m // 2, m // 2 + 40), torch.arange(m - 40, m)]).to(cuda)
    part = [args[0][rows], *args[1:]]
    ref = _reference(part, dy[rows], "silu", dt)
    _check([got[0][rows], got[1][rows]], ref[:2], "far rows")
    # weight gradients add over the rows: those of two halves give the whole
    halves = [_run([args[0][s], *args[1:]], dy[s], "silu")[2:] for s in (slice(0, m // 2), slice(m // 2, m))]
    for a, b, w in zip(*halves, got[2:]):
        s = a.double() + b.double()
        # four roundings to bf16 of terms that each carry the operands' roundings
        assert float((s - w.double()).norm() / s.norm()) <= 4 * 2.0 ** -8


def test_graph_capture_and_streams(cuda):
    """A captured training step replayed on new data has the eager step's bits, while an eager graph of the
    same leaves is alive; and a call on a side stream."""
    args, dy = _inputs(500, 64, 128, torch.bfloat16, cuda, True, seed=14)
    leaves = [t.detach().clone().requires_grad_(True) for t in args]
    eager_y = mdc.gated_feed_forward(*leaves)           # alive across the capture
    static_dy = dy.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    static = [t.detach().clone().requires_grad_(True) for t in args]
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(mdc.gated_feed_forward(*static), static, static_dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mdc.gated_feed_forward(*static)
        grads = torch.autograd.grad(y, static, static_dy)
    for seed in (20, 21):
        new, ndy = _inputs(500, 64, 128, torch.bfloat16, cuda, True, seed=seed)
        with torch.no_grad():
            for a, b in zip(static, new):
                a.copy_(b)
            static_dy.copy_(ndy)
        graph.replay()
        want = _run(new, ndy, "silu")
        assert all(torch.equal(a, b) for a, b in zip([y.detach(), *grads], want))
    eager = torch.autograd.grad(eager_y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(eager, _run(args, dy, "silu")[1:]))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(args, dy, "silu")
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got[1:], eager))


@pytest.mark.parametrize("size", [(300, 64, 96), (40, 512, 200), (3, 64, 96)], ids=str)
def test_first_call_of_a_thread(size, cuda):
    """A thread that has made no CUDA call yet has no current context; forward and backward work all the same."""
    import threading
    args, dy = _inputs(*size, torch.bfloat16, cuda, True, seed=33)
    want = _run(args, dy, "silu")
    _, saved = mdc._get_lib().gated_feed_forward_forward(*args, 0, True, False)
    torch.cuda.synchronize()
    out = {}

    def forward():
        out["y"] = mdc._get_lib().gated_feed_forward_forward(*args, 0)[0]

    def backward():
        out["g"] = mdc._get_lib().gated_feed_forward_backward(dy, *args, 0, saved, [True] * 7)

    for f in (forward, backward):
        t = threading.Thread(target=f)
        t.start()
        t.join()
    torch.cuda.synchronize()
    few = _run(args, None, "silu")[0]  # nothing saved: the form of few rows, where it applies
    assert torch.equal(out["y"], few)
    assert all(torch.equal(a, b) for a, b in zip(out["g"], want[1:]))


def test_few_rows_captured_and_on_two_streams(cuda):
    """The dependent launches of the few-row kernels replay from a graph, and two streams at once keep apart."""
    calls = []
    for m, c, f, dt in ((1, 512, 2048, torch.bfloat16), (8, 1024, 264, torch.float16), (5, 96, 200, torch.float32)):
        args, _ = _inputs(m, c, f, dt, cuda, True, seed=m)
        calls.append(args)
    want = [_run(a, None, "gelu")[0] for a in calls]
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        outs = [mdc.gated_feed_forward(*a, activation="gelu") for a in calls for _ in range(3)]
    for _ in range(20):
        for o in outs:
            o.zero_()
        graph.replay()
        assert all(torch.equal(o, want[i // 3]) for i, o in enumerate(outs))
    for k, args in enumerate(calls):  # new data in the captured inputs
        args[0].mul_(-0.5)
    graph.replay()
    for i, o in enumerate(outs):
        assert torch.equal(o, _run(calls[i // 3], None, "gelu")[0])
    big, dy = _inputs(3000, 320, 640, torch.bfloat16, cuda, True, seed=30)
    ref = _run(big, dy, "silu")
    small = _run(calls[0], None, "silu")[0]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got, few = [], []
    for _ in range(5):
        with torch.cuda.stream(streams[0]):
            got.append(_run(big, dy, "silu"))
        with torch.cuda.stream(streams[1]):
            few += [_run(calls[0], None, "silu")[0] for _ in range(10)]
            got.append(_run(big, dy, "silu"))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, ref))
    assert all(torch.equal(o, small) for o in few)


def test_captured_training_step_of_a_block(cuda):
    """Deformable layer, gated block, gradient norm and AdamW in one graph: replayed steps leave the parameters
    of the same steps taken one call at a time (forward and weight gradients are reproducible; the offsets'
    gradients, summed by atomics, do not reach a parameter here)."""
    def make():
        torch.manual_seed(5)
        layer = mdc.DeformConv2d(64, 64, 3, padding=1).to(cuda, torch.bfloat16)
        block = mdc.GatedFeedForward2d(64, 160).to(cuda, torch.bfloat16)
        params = [*layer.parameters(), *block.parameters()]
        return layer, block, params, mdc.optim.AdamW(params, lr=1e-2, state_bits=8, master_weights=True, seed=9)

    g = torch.Generator(cuda).manual_seed(1)
    x = torch.randn(2, 64, 9, 8, generator=g, device=cuda).to(torch.bfloat16).contiguous(memory_format=torch.channels_last)
    off = torch.randn(2, 18, 9, 8, generator=g, device=cuda).to(torch.bfloat16)
    go = torch.randn(2, 64, 9, 8, generator=g, device=cuda).to(torch.bfloat16)

    def step(layer, block, params, opt):
        for p in params:
            p.grad = None
        block(layer(x, off)).backward(go)
        _, factor = mdc.optim.grad_norm([p.grad for p in params], max_norm=1.0)
        opt.step(grad_scale=factor)

    eager = make()
    for _ in range(6):
        step(*eager)
    replayed = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(*replayed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*replayed)
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    for p, q in zip(eager[2], replayed[2]):
        assert torch.equal(p, q)
        assert eager[3].state[p]["step"].tolist() == [6, 0] == replayed[3].state[q]["step"].tolist()


def test_parameter_gradient_hook(cuda):
    args, dy = _inputs(130, 32, 40, torch.float32, cuda, True, seed=15)
    want = _run(args, dy, "silu")
    seen = []
    mdc.set_param_grad_hook(lambda w, b: seen.append((w, b)))
    try:
        got = _run(args, dy, "silu")
    finally:
        mdc.set_param_grad_hook(None)
    assert len(seen) == 3
    for k, (w, b) in enumerate(seen):
        assert torch.equal(w, want[2 + k]) and torch.equal(b, want[5 + k])
    assert torch.equal(got[1], want[1])

    def boom(w, b):
        raise KeyError("hook")

    mdc.set_param_grad_hook(boom)
    try:
        with pytest.raises(KeyError):
            _run(args, dy, "silu")
        e, edy = _inputs(0, 32, 40, torch.float32, cuda, True)
        with pytest.raises(KeyError):
            _run(e, edy, "silu")
    finally:
        mdc.set_param_grad_hook(None)


@pytest.mark.parametrize("fmt", [torch.contiguous_format, torch.channels_last])
def test_module_after_a_deformable_layer(fmt, cuda):
    """A backbone block: deformable layer, residual gated block, one optimizer step; the block against its
    formula on the layer's own output, memory formats kept."""
    torch.manual_seed(2)
    layer = mdc.ModulatedDeformConv2d(64, 64, 3, padding=1, offset_groups=2).to(cuda, torch.bfloat16)
    block = mdc.GatedFeedForward2d(64, 160, activation="gelu").to(cuda, torch.bfloat16)
    x = torch.randn(2, 64, 12, 10, device=cuda, dtype=torch.bfloat16).contiguous(memory_format=fmt)
    feat = layer(x)
    feat.retain_grad()
    out = block(feat)
    assert out.shape == feat.shape and out.is_contiguous(memory_format=fmt)
    go = torch.randn_like(out)
    params = [*layer.parameters(), *block.parameters()]
    out.backward(go)
    rows = lambda t: t.permute(0, 2, 3, 1).reshape(-1, 64)  # noqa: E731
    args = [rows(feat).detach(), block.w_gate, block.w_up, block.w_down, block.b_gate, block.b_up, block.b_down]
    got = [rows(out).detach(), rows(feat.grad), *[p.grad for p in (args[1:])]]
    _check(got, _reference(args, rows(go), "gelu", torch.bfloat16), str(fmt))
    before = [p.detach().clone() for p in params]
    opt = mdc.optim.AdamW(params, lr=1e-2, master_weights=True)
    norm, factor = mdc.optim.grad_norm([p.grad for p in params], max_norm=1.0)
    opt.step(grad_scale=factor)
    assert torch.isfinite(norm) and all(not torch.equal(a, p) for a, p in zip(before, params))
    with torch.no_grad():
        assert torch.isfinite(block(layer(x))).all()


def test_refusals_on_the_device(cuda):
    args, _ = _inputs(8, 16, 24, torch.bfloat16, cuda, True)
    with pytest.raises(RuntimeError, match="same dtype"):
        mdc.gated_feed_forward(args[0], args[1].float(), *args[2:])
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        mdc.gated_feed_forward(*[t.double() for t in args])
    with pytest.raises(ValueError, match="same device"):
        mdc.gated_feed_forward(args[0], args[1].cpu(), *args[2:])
    with pytest.raises(ValueError, match="w_down"):
        mdc.gated_feed_forward(args[0], args[1], args[2], args[3].t(), *args[4:])


def test_dtype_refusals_name_their_operator(cuda):
    """The helper is shared; each operator keeps its own prefix."""
    x, w = torch.zeros(1, 4, 5, 5, device=cuda).double(), torch.zeros(4, 4, 3, 3, device=cuda).double()
    offset = torch.zeros(1, 18, 5, 5, device=cuda).double()
    with pytest.raises(RuntimeError, match="^deform_conv2d: unsupported dtype"):
        mdc.deform_conv2d(x, offset, w, padding=1)
    v, u = torch.zeros(3, 8, device=cuda).double(), torch.zeros(16, 8, device=cuda).double()
    with pytest.raises(RuntimeError, match="^gated_feed_forward: unsupported dtype"):
        mdc.gated_feed_forward(v, u, u, u.t().contiguous())
    with pytest.raises(RuntimeError, match="^grad_norm: unsupported dtype"):
        mdc.optim.grad_norm([v])
    with pytest.raises(RuntimeError, match="^adamw_step: unsupported dtype"):
        mdc.optim.adamw_step([v], [v.clone()], [v.float()], [v.float()], [mdc.optim.new_step(cuda)], lr=1e-3)


def test_registered_operators(cuda):
    ops = torch.ops.mps_deform_conv
    for bias in (True, False):
        args, dy = _inputs(20, 16, 24, torch.float32, cuda, bias, seed=16)
        leaves = [t if t is None else t.requires_grad_(True) for t in args]
        torch.library.opcheck(ops.gated_feed_forward.default, (*leaves, 0))
        with torch.no_grad():
            torch.library.opcheck(ops.gated_feed_forward_backward.default, (dy, *args, 1),
                                  test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_compiled_module_matches_eager(backend, cuda):
    torch.manual_seed(4)
    mod = mdc.GatedFeedForward2d(64, 96).to(cuda, torch.bfloat16)
    x = torch.randn(2, 64, 6, 5, device=cuda, dtype=torch.bfloat16)
    go = torch.randn_like(x)

    def run(fn):
        xi = x.clone().requires_grad_(True)
        mod.zero_grad(set_to_none=True)
        out = fn(xi)
        out.backward(go)
        return [out.detach(), xi.grad, *[p.grad.clone() for p in mod.parameters()]]

    eager = run(mod)
    torch._dynamo.reset()
    got = run(torch.compile(mod, fullgraph=True, backend=backend))
    assert all(torch.equal(a, b) for a, b in zip(got, eager))
    torch._dynamo.reset()


@pytest.mark.parametrize("m,c,f,dtype,train", [
    (19000, 384, 1536, "bfloat16", True), (4 * 69 * 69, 320, 1280, "bfloat16", True), (19300, 64, 1024, "float16", True),
    (19201, 128, 2048, "bfloat16", False), (19300, 64, 1600, "bfloat16", False), (19300, 64, 256, "float32", True),
    (19201, 64, 170, "float32", True), (19300, 64, 512, "float32", False), (18945, 192, 512, "float32", False),
    (57200, 64, 256, "float32", True), (817, 408, 1096, "float16", True), (870, 424, 1696, "bfloat16", False)])
def test_products_cut_among_few_tiles(m, c, f, dtype, train, cuda):
    """A last wave of few tiles, cut along K among all SMs: an even share of less than one K block a slice
    (three tiles for 148 SMs), and shares that leave runs beside the slices."""
    dt = DTYPES[dtype]
    args, dy = _inputs(m, c, f, dt, cuda, train, seed=m % 1000 + c)
    dy = dy if train else None
    _check(_run(args, dy, "silu"), _reference(args, dy, "silu", dt), f"{(m, c, f)} {dtype}")


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_few_training_rows_do_not_depend_on_earlier_calls(dtype, cuda):
    """One tile with fewer rows than 128: what an earlier call left in shared memory where rows are missing
    does not reach a gradient's bits.  Weight rows many decades apart, so that the two ways of keeping gate
    and up for the backward (more than 256 channels) differ in the small ones."""
    dt = DTYPES[dtype]
    args, dy = _inputs(40, 512, 2048, dt, cuda, False, seed=41)
    decades = torch.exp2(torch.arange(2048, device=cuda) % 16 * -2.0).to(dt)
    args[1], args[2] = args[1] * decades[:, None], args[2] * decades.flip(0)[:, None]
    fill, _ = _inputs(128, 512, 2048, dt, cuda, False, seed=42)
    results = []
    for scale in (1.0, 1e4, 1.0, 1e-6, 0.0):
        other = [fill[0] * scale, *args[1:]]
        leaves = [t if t is None else t.detach().requires_grad_(True) for t in args]
        mdc._get_lib().gated_feed_forward_forward(*other, 0, True)
        y = mdc.gated_feed_forward(*leaves)
        results.append([y.detach(), *torch.autograd.grad(y, leaves[:4], dy)])
    for got in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got, results[0]))
    _check(results[0], _reference(args, dy, "silu", dt))


@pytest.mark.parametrize("m", [8, 449])
def test_gelu_keeps_its_lower_tail(m, cuda):
    """fp32, one channel with weights of 1 and up = 1 (its bias), so that y is gelu(x) and dx its derivative
    with no other rounding.  normcdff and expf are documented within 5 and 2 units in the last place (2^-23
    each at most); the product x Phi adds one rounding.  In the derivative Phi + x phi: x^2 / 2 carries two
    roundings into the exponent, phi's constant, two products and the sum four more."""
    x = torch.linspace(-10, -3, m, device=cuda).mul(64).round().div(64).view(m, 1)
    one, zero = torch.ones(1, 1, device=cuda), torch.zeros(1, 1, device=cuda)
    args = [x, one, zero, one, torch.zeros(1, device=cuda), torch.ones(1, device=cuda), None]
    v = x.double()  # torch's ndtr cancels there, in 64 bits too
    cdf, density = 0.5 * torch.special.erfc(v * -math.sqrt(0.5)), torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    y, dx = _run(args, None, "gelu")[0], _run(args, one.expand(m, 1), "gelu")[1]
    exact = v * cdf
    assert ((y.double() - exact).abs() <= (5 + 1) * 2.0 ** -23 * exact.abs()).all()
    assert ((_run(args, one.expand(m, 1), "gelu")[0].double() - exact).abs() <= (5 + 1) * 2.0 ** -23 * exact.abs()).all()
    err = 5 * 2.0 ** -23 * cdf + (v * density).abs() * (v * v * 2.0 ** -24 + 2 * 2.0 ** -23 + 4 * 2.0 ** -24)
    assert ((dx.double() - (cdf + v * density)).abs() <= err + 2.0 ** -24 * err).all()


def test_forward_mode_is_refused(cuda):
    args, _ = _inputs(6, 16, 24, torch.float32, cuda, True)
    for k, t in enumerate(args):
        def call(x):
            return mdc.gated_feed_forward(*args[:k], x, *args[k + 1:])  # noqa: B023

        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))


# The backward reads gate and up back above these many channels, and computes them again up to them.
SAVED_CHANNELS = [("float16", 264), ("bfloat16", 264), ("bfloat16", 512), ("float32", 136)]


def _reads_saved_values(args):
    """The state that the forward leaves is more than the hidden values in their panels."""
    (m, c), f = args[0].shape, args[1].shape[0]
    saved = mdc._get_lib().gated_feed_forward_forward(*args, 0, True)[1].numel()
    panels = (3 if args[0].dtype == torch.float32 else 1) * (-(-m // 128) * 128) * (-(-f // 8) * 8) * 2
    return saved >= panels + 2 * 2 * m * f


@pytest.mark.parametrize("dtype,c", SAVED_CHANNELS)
def test_saved_state_rows_keep_to_themselves(dtype, c, cuda):
    """Rows that are not finite, or far outside fp16's range, leave the others' results as they are, bit for
    bit, those of their own 32-row block too.  Hidden units many decades apart, so that the ways of keeping
    a block differ in the small ones."""
    dt = DTYPES[dtype]
    args, dy = _inputs(300, c, 96, dt, cuda, True, seed=51)
    decades = torch.exp2(torch.arange(96, device=cuda) % 16 * -2.0).to(dt)
    for k in (1, 2, 4, 5):
        args[k] = args[k] * (decades[:, None] if args[k].dim() == 2 else decades)
    assert _reads_saved_values(args)
    dy[5] = dy[299] = 0.0  # with finite values these rows then add nothing to the weights' gradients
    clean = _run(args, dy, "silu")
    _check(clean, _reference(args, dy, "silu", dt))
    keep = torch.ones(300, dtype=torch.bool, device=cuda)
    keep[5] = keep[299] = False
    big = 20.0 if dtype == "float16" else 3e4  # the hidden values of these rows stay finite
    for a, b in ((float("nan"), float("inf")), (big, -big), (0.0, 2.0 ** -14)):
        x = args[0].clone()
        x[5], x[299] = a, b
        got = _run([x, *args[1:]], dy, "silu")
        assert torch.equal(got[0][keep], clean[0][keep]) and torch.equal(got[1][keep], clean[1][keep])
        if not math.isfinite(a):
            assert got[0][5].isnan().all() and got[1][5].isnan().all() and not got[0][299].isfinite().any()
        else:
            assert all(torch.equal(p, q) for p, q in zip(got[2:], clean[2:])), (a, b)


@pytest.mark.parametrize("dtype,c", SAVED_CHANNELS)
def test_saved_state_far_tails_and_small_values(dtype, c, cuda):
    """Gate and up many decades apart in one row and between rows, beyond fp16's range where the type has it."""
    dt = DTYPES[dtype]
    reach = 6 if dtype == "float16" else 20
    args, dy = _inputs(96, c, 64, dt, cuda, False, seed=52)
    scale = torch.exp2(torch.linspace(-reach, reach, 64, device=cuda)).to(dt)
    args[2] = args[2] * scale[:, None]
    args[1] = args[1] * scale.flip(0)[:, None]
    for rows in (torch.zeros(96, device=cuda), torch.linspace(-4, 4, 96, device=cuda).round()):
        case = [(args[0].float() * torch.exp2(rows)[:, None]).to(dt), *args[1:]]
        assert _reads_saved_values(case)
        for act in ("silu", "relu"):
            got, ref = _run(case, dy, act), _reference(case, dy, act, dt)
            if dtype == "float16":  # rounds 65520 and above to inf
                for t, (v, e) in zip(got, ref):
                    assert (t[v.abs() - e >= 65520].double() == math.inf * v.sign()[v.abs() - e >= 65520]).all()
                    past = v.abs() + e >= 65504
                    assert past.float().mean() < 0.05  # the check says something
                    t[past], v[past] = 0.0, 0.0
            _check(got, ref, "decades")


@pytest.mark.parametrize("dtype,c", [("bfloat16", 264), ("bfloat16", 512), ("float32", 136)])
@pytest.mark.parametrize("power", [-30, 30])
def test_saved_state_outside_fp16(dtype, c, power, cuda):
    """All of gate and up near 2^30 or 2^-30 (relu, whose products scale with them exactly): the gradients are
    those of the same rows near 1, scaled.  Per factor and sum half a step of the type, and half a step of 11 bits of
    what was saved; the sums' own error is below another half step."""
    dt = DTYPES[dtype]
    args, dy = _inputs(96, c, 64, dt, cuda, False, seed=53)
    assert _reads_saved_values(args)
    scaled = [args[0] * 2.0 ** power, *args[1:]]
    ref = _reference(args, dy, "relu", dt)
    got = _run(scaled, dy, "relu")
    u = max(torch.finfo(dt).eps / 2, 0 if dt == torch.float32 else 2.0 ** -11)
    # y ~ s^2; dgate and dup ~ s, so dx ~ s and the gate and up gradients ~ s^2; dw_down ~ s^2
    for name, t, (v, _), order in zip(NAMES, got, ref, (2, 1, 2, 2, 2)):
        err = float((t.double() * 2.0 ** (-power * order) - v).norm() / v.norm())
        assert err <= 4 * u + (2.0 ** -20 if dt == torch.float32 else 2.0 ** -11), (name, err)
