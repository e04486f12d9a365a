"""What is measured of this package's training-block operators, beside their plain forms.

Three operators, named by a case's "op":

* ``ffn``    -- ``gated_feed_forward``: y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd over the
  channels of every pixel, and with ``train`` its gradients;
* ``adamw``  -- ``optim.adamw_step``: one AdamW step over all tensors of a network, states in
  32 bits or in 8 (float8 e4m3 codes with one power-of-two scale per 256 elements);
* ``norm``   -- ``optim.grad_norm``: the global gradient norm and the factor that clips it.

``own`` False: the plain forms below, elementary torch operations in 32 bits (64 where noted).
``own`` True: the calls a user makes.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 256        # elements that share one scale of an 8-bit state
ALIGN = 64         # tensors of one flat buffer start at multiples of this many elements
MASK32 = 0xFFFFFFFF


# ---------------------------------------------------------------- cases
def _ffn(name, tokens, channels, hidden, dtype, activation="silu", bias=False, train=False, packed=False):
    case = {"op": "ffn", "tokens": tokens, "channels": channels, "hidden": hidden, "dtype": dtype,
            "activation": activation, "bias": bias, "train": train, "packed": packed}
    return dict(case, name=name) if name else case


def _net(name, op, layers, channels, groups, offset_groups, hidden, dtype, bits=32, master=False, scaled=True):
    case = {"op": op, "layers": layers, "channels": channels, "groups": groups, "offset_groups": offset_groups,
            "hidden": hidden, "dtype": dtype}
    if op == "adamw":
        case.update(bits=bits, master=master, scaled=scaled)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one pooled feature vector through a block: the smallest call, launch latency
        _ffn("ffn_one_vector_bf16", 1, 512, 2048, "bf16"),
        # a handful of vectors through a wide block while serving: weights are read, little is computed
        _ffn("ffn_few_wide_bf16", 16, 4096, 14336, "bf16"),
        # the ResNet-50 C4-stage feature map (8 x 50 x 68 pixels), inference, with biases
        _ffn("ffn_backbone_bf16", 27200, 256, 1024, "bf16", "gelu", True),
        # the fp32 DCNv2 layer's feature map (2 x 64 x 64 pixels), training
        _ffn("ffn_train_fp32", 8192, 128, 512, "fp32", "silu", True, True),
        # video alignment (16 x 180 x 320 pixels), narrow block of 8/3 of the channels (odd rows), training
        _ffn("ffn_train_video_fp16", 921600, 64, 170, "fp16", "silu", False, True),
        # the large training step's feature map (64 x 38 x 38 pixels), gate and up stored as one tensor
        _ffn("ffn_train_bf16", 92416, 512, 2048, "bf16", "silu", True, True, True),
        # one modulated layer of 64 channels, fp32: a few small tensors, launch latency
        _net("adamw_layer_fp32", "adamw", 1, 64, 1, 1, 0, "fp32"),
        # twenty blocks of the large training step, bf16 parameters with fp32 master copies
        _net("adamw_net_master_bf16", "adamw", 20, 512, 2, 4, 2048, "bf16", 32, True),
        # the same network with 8-bit states and no master copies
        _net("adamw_net_8bit_bf16", "adamw", 20, 512, 2, 4, 2048, "bf16", 8),
        # odd widths (rows that end inside a block of 256), fp32 parameters, 8-bit states
        _net("adamw_odd_8bit_fp32", "adamw", 6, 100, 1, 1, 267, "fp32", 8),
        # the clipping norm of one layer and of the network
        _net("norm_layer_fp32", "norm", 1, 64, 1, 1, 0, "fp32"),
        _net("norm_net_bf16", "norm", 20, 512, 2, 4, 2048, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "ffn", "adamw", "adamw", "norm"])
    if op == "ffn":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        train = rng.random() < 0.5
        if rng.random() < 0.3:  # few vectors, wide blocks
            channels, train = _log(rng, 128, 4096), False
            hidden, tokens = int(channels * rng.uniform(1.5, 3.5)), _log(rng, 1, 64)
        else:
            channels = _log(rng, 24, 768)
            hidden = int(channels * rng.choice([2, 8 / 3, 4]) + rng.randrange(0, 3))
            most = min(9e7 / hidden, (1.5e12 if dtype != "fp32" else 3e11) / (18 * channels * hidden), 9e5)
            tokens = _log(rng, 1, max(2, int(most)))
        if rng.random() < 0.7:  # most widths are multiples of 8
            channels, hidden = max(8, channels // 8 * 8), max(8, hidden // 8 * 8)
        return _ffn(None, tokens, channels, hidden, dtype, rng.choice(["silu", "silu", "gelu", "relu", "sigmoid"]),
                    rng.random() < 0.5, train, rng.random() < 0.3)
    channels = _log(rng, 16, 512)
    if rng.random() < 0.7:
        channels = channels // 4 * 4
    og = 4 if channels % 4 == 0 and rng.random() < 0.5 else 1
    groups = 2 if channels % 2 == 0 and rng.random() < 0.5 else 1
    hidden = rng.choice([0, channels * 4, channels * 8 // 3])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    layers = rng.randrange(1, 13)
    if op == "norm":
        return _net(None, "norm", layers, channels, groups, og, hidden, dtype)
    return _net(None, "adamw", layers, channels, groups, og, hidden, dtype, rng.choice([8, 32]),
                dtype != "fp32" and rng.random() < 0.5, rng.random() < 0.7)


def _shapes(case):
    """The parameters of a stack of modulated deformable layers, each with a gated block when hidden > 0."""
    c, t = case["channels"], 9
    layer = [(c, c // case["groups"], 3, 3), (c,), (3 * t * case["offset_groups"], c, 3, 3), (3 * t * case["offset_groups"],)]
    if case["hidden"]:
        layer += [(case["hidden"], c), (case["hidden"], c), (c, case["hidden"])]
    return layer * case["layers"]


def _numel(shape):
    return math.prod(shape)


def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "ffn":
        m, c, f = case["tokens"], case["channels"], case["hidden"]
        weights, biases = 3 * c * f, (2 * f + c if case["bias"] else 0)
        fwd = 2 * m * c + weights + biases
        if not case["train"]:
            return {"bytes": b * fwd, "flops": 6.0 * m * c * f}
        # the step reads grad_y too and writes the gradients of x, the weights and the biases
        return {"bytes": b * (fwd + 2 * m * c + weights + biases), "flops": 18.0 * m * c * f}
    n = sum(_numel(s) for s in _shapes(case))
    if case["op"] == "norm":
        return {"bytes": b * n, "flops": 2.0 * n}
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * (2 * b + b + state + (4 + 4 - b if case["master"] else 0)), "flops": 20.0 * n}


# ---------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _flat(shapes, dtype):
    """One buffer for all tensors and their views in it, each starting at a multiple of ALIGN elements."""
    at, spans = 0, []
    for s in shapes:
        spans.append((at, s))
        at += -(-_numel(s) // ALIGN) * ALIGN
    buf = torch.zeros(at, device=DEV, dtype=dtype)
    return buf, [buf[a:a + _numel(s)].view(s) for a, s in spans]


def _fill(views, g, scale, like=None):
    for v in views:
        v.copy_(torch.randn(v.shape, generator=g, device=DEV) * scale)


def prepare(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * scale).to(dt)

    if case["op"] == "ffn":
        m, c, f = case["tokens"], case["channels"], case["hidden"]
        gate_up = randn(2 * f, c, scale=1 / math.sqrt(c))
        w_gate, w_up = (gate_up[:f], gate_up[f:]) if case["packed"] else (gate_up[:f].clone(), gate_up[f:].clone())
        args = [randn(m, c), w_gate, w_up, randn(c, f, scale=1 / math.sqrt(f))]
        args += [randn(f, scale=0.1), randn(f, scale=0.1), randn(c, scale=0.1)] if case["bias"] else [None] * 3
        if case["train"]:
            args = [t if t is None else t.detach().requires_grad_(True) for t in args]
        return {"case": case, "args": args, "grad": randn(m, c) if case["train"] else None}

    shapes = _shapes(case)
    grads, grad_views = _flat(shapes, dt)
    _fill(grad_views, g, 1e-2)
    if case["op"] == "norm":
        return {"case": case, "grads": grad_views}
    params, param_views = _flat(shapes, dt)
    _fill(param_views, g, 0.05)
    state = {"case": case, "grads": grad_views, "p": params, "params": param_views, "masters": None, "master": None}
    if case["master"]:
        state["master"], state["masters"] = _flat(shapes, torch.float32)
        for w, p in zip(state["masters"], param_views):
            w.copy_(p)
    m, state["exp_avgs"] = _flat(shapes, torch.float32)
    v, state["exp_avg_sqs"] = _flat(shapes, torch.float32)
    _fill(state["exp_avgs"], g, 3e-3)
    for t in state["exp_avg_sqs"]:  # squares spread over some decades, as layers' and channels' gradients are
        t.copy_((torch.randn(t.shape, generator=g, device=DEV) * 1e-2) ** 2)
    state["exp_avg"], state["exp_avg_sq"] = m, v
    if case["bits"] == 8:
        for key, root in (("exp_avg", False), ("exp_avg_sq", True)):
            scales, scale_views = _flat([(-(-_numel(s) // BLOCK),) for s in shapes], torch.float32)
            codes, code_views = _flat(shapes, torch.float8_e4m3fn)
            for k, t in enumerate(state[key + "s"]):
                x = _blocks(t.sqrt() if root else t)
                s = torch.exp2(torch.floor(torch.log2(x.abs().amax(1))).clamp(-100, 127) - 7)
                scale_views[k].copy_(s)
                code_views[k].copy_((x / s[:, None]).to(torch.float8_e4m3fn).view(-1)[:t.numel()].view(t.shape))
            state[key], state[key + "s"] = codes, code_views
            state[key + "_scale"], state[key + "_scales"] = scales, scale_views
    count = torch.randint(1, 1000, (1,), generator=g, device=DEV)
    state["steps"] = [torch.cat([count, count * 0]).to(torch.int32)] * len(shapes)  # (steps taken, 0), one for the network
    state["grad_scale"] = torch.rand((), generator=g, device=DEV) * 0.5 + 0.25 if case["scaled"] else None
    state["hyper"] = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    state["seed"] = 1234
    return state


# ---------------------------------------------------------------- plain forms
def _act(x, kind):
    """act(x) and its derivative."""
    if kind == "silu":
        s = 1 / (1 + torch.exp(-x))
        return x * s, s * (1 + x * (1 - s))
    if kind == "sigmoid":
        s = 1 / (1 + torch.exp(-x))
        return s, s * (1 - s)
    if kind == "relu":
        on = (x > 0).to(x.dtype)
        return x * on, on
    cdf = 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
    return x * cdf, cdf + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))


def _ffn_in(state, dtype, kind):
    """Outputs (and gradients) computed throughout in `dtype`, not rounded to the inputs' type."""
    x, wg, wu, wd, bg, bu, bd = [t if t is None else t.detach().to(dtype) for t in state["args"]]
    gate, up = x @ wg.t(), x @ wu.t()
    if bg is not None:
        gate, up = gate + bg, up + bu
    a, da = _act(gate, kind)
    h = a * up
    y = h @ wd.t()
    if bd is not None:
        y = y + bd
    if state["grad"] is None:
        return [y]
    dy = state["grad"].to(dtype)
    dh = dy @ wd
    dgate, dup = dh * up * da, dh * a
    out = [y, dgate @ wg + dup @ wu, dgate.t() @ x, dup.t() @ x, dy.t() @ h]
    if bd is not None:
        out += [dgate.sum(0), dup.sum(0), dy.sum(0)]
    return out


def _blocks(t):
    """The elements in rows of BLOCK, the last one filled up with zeros."""
    flat = t.reshape(-1)
    return torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)


def _mix(x):
    """A 32-bit integer hash (the published 'lowbias32' constants), on int64 tensors."""
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & MASK32
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & MASK32
    return x ^ (x >> 16)


def _dither(n, step, seed):
    """One 32-bit word per element, from the element's index, the step and the seed."""
    key = _mix((seed + step.to(torch.int64) * 0x9E3779B9) & MASK32)
    return _mix((torch.arange(n, device=DEV, dtype=torch.int64) ^ key) & MASK32)


def _quantize(x, words, keep_positive):
    """x [blocks, BLOCK] to e4m3 codes and power-of-two scales; rounded up with the probability of the
    remainder: a 16-bit word of `words` is added below the last kept bit of the scaled fp32 pattern."""
    top = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(1)
    e = ((top.view(torch.int32) >> 23) - 127).clamp(-100, 127)
    scale = torch.exp2((e - 7).float())
    z = x.abs() * torch.exp2((7 - e).float())[:, None] * 2.0 ** -120
    code = (z.view(torch.int32) + (words << 4).to(torch.int32)) >> 20
    if keep_positive:
        code = torch.where(x > 0, code.clamp(min=1), code)
    code = torch.where(torch.isfinite(x), code, torch.full_like(code, 0x7F))
    code = code | torch.where(x < 0, 0x80, 0)
    return code.to(torch.uint8).view(torch.float8_e4m3fn), scale


def _adamw_one(state, k):
    """One tensor's AdamW step, in place; every product and sum rounded to 32 bits on its own."""
    case, h = state["case"], state["hyper"]
    b1, b2 = h["betas"]
    p = (state["masters"] or state["params"])[k]
    t = state["steps"][k][:1].double() + 1
    step_size = (h["lr"] / (1 - b1 ** t)).float()
    root_corr = (1 - b2 ** t).rsqrt().float()
    g = state["grads"][k].float()
    if state["grad_scale"] is not None:
        g = g * state["grad_scale"]
    m, v = state["exp_avgs"][k], state["exp_avg_sqs"][k]
    shape, n = g.shape, g.numel()
    if case["bits"] == 8:
        ms, vs = state["exp_avg_scales"][k], state["exp_avg_sq_scales"][k]
        g = _blocks(g)
        m_new = _blocks(m.float()) * ms[:, None]
        root = _blocks(v.float()) * vs[:, None]
        m_new, v_new = m_new * b1 + g * (1 - b1), (root * root) * b2 + (g * g) * (1 - b2)
        root = v_new.sqrt()
        words = _dither(g.numel(), state["steps"][k][:1] + 1, state["seed"]).view(g.shape)
        for x, old, scales, w, keep in ((m_new, m, ms, words & 0xFFFF, False), (root, v, vs, words >> 16, True)):
            code, scale = _quantize(x, w, keep)
            old.copy_(code.view(-1)[:n].view(shape))
            scales.copy_(scale)
        m_new, root = m_new.view(-1)[:n].view(shape), root.view(-1)[:n].view(shape)
    else:
        m.copy_(m * b1 + g * (1 - b1))
        v.copy_(v * b2 + (g * g) * (1 - b2))
        m_new, root = m, v.sqrt()
    new = p.float() * (1 - h["lr"] * h["weight_decay"]) - step_size * (m_new / (root * root_corr + h["eps"]))
    p.copy_(new)
    if state["masters"]:
        state["params"][k].copy_(new)


def _norm_of(grads, max_norm, loss_scale):
    total = torch.stack([(g.double() ** 2).sum() for g in grads]).sum().sqrt() / loss_scale
    return [total.float(), ((max_norm / (total + 1e-6)).clamp(max=1.0) / loss_scale).float()]


MAX_NORM, LOSS_SCALE = 1.0, 8.0


def _updated(state):
    keys = ["p", "master", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"]
    return {k: state[k] for k in keys if state.get(k) is not None}


def _package():
    """This repository's package (the repository's root is the working folder)."""
    import os
    import sys

    at = os.path.abspath("mps-deform-conv_b200")
    if at not in sys.path:
        sys.path.insert(1, at)
    import mps_deform_conv

    return mps_deform_conv


def run(state):
    case = state["case"]
    if case["op"] == "ffn":
        if own:
            y = _package().gated_feed_forward(*state["args"], activation=case["activation"])
            if state["grad"] is None:
                return [y]
            return [y.detach(), *torch.autograd.grad(y, [t for t in state["args"] if t is not None], state["grad"])]
        with torch.no_grad():
            return [t.to(DTYPES[case["dtype"]]) for t in _ffn_in(state, torch.float32, case["activation"])]
    if case["op"] == "norm":
        if own:
            return list(_package().optim.grad_norm(state["grads"], max_norm=MAX_NORM, loss_scale=LOSS_SCALE))
        return _norm_of(state["grads"], MAX_NORM, LOSS_SCALE)
    if own:
        _package().optim.adamw_step(
            state["params"], state["grads"], state["exp_avgs"], state["exp_avg_sqs"], state["steps"],
            masters=state["masters"], exp_avg_scales=state.get("exp_avg_scales"),
            exp_avg_sq_scales=state.get("exp_avg_sq_scales"), grad_scale=state["grad_scale"], seed=state["seed"],
            **state["hyper"])
        return _updated(state)
    for k in range(len(state["params"])):
        _adamw_one(state, k)
    state["steps"][0].add_(torch.tensor([1, 0], device=DEV, dtype=torch.int32))
    return _updated(state)


# ---------------------------------------------------------------- 64 bits
def _act64(x, kind):
    """act and derivative, in the forms of the functions' definitions."""
    if kind == "relu":
        return torch.where(x > 0, x, 0.0), torch.where(x > 0, 1.0, 0.0).to(x.dtype)
    if kind == "gelu":
        cdf = torch.special.ndtr(x)
        return x * cdf, cdf + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    s = torch.special.expit(x)
    if kind == "sigmoid":
        return s, s * torch.special.expit(-x)
    return x * s, s + x * s * torch.special.expit(-x)


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "ffn":
            x, wg, wu, wd, bg, bu, bd = [t if t is None else t.detach().double() for t in state["args"]]
            F = torch.nn.functional
            gate, up = F.linear(x, wg, bg), F.linear(x, wu, bu)
            a, da = _act64(gate, case["activation"])
            y = F.linear(a * up, wd, bd)
            if state["grad"] is None:
                return [y]
            dy = state["grad"].double()
            dwd = torch.einsum("mc,mf->cf", dy, a * up)
            dh = torch.einsum("mc,cf->mf", dy, wd)
            dup = dh * a
            del a
            dgate = dh.mul_(up).mul_(da)
            del up, da, gate
            out = [y, torch.addmm(dgate @ wg, dup, wu), torch.einsum("mf,mc->fc", dgate, x), torch.einsum("mf,mc->fc", dup, x), dwd]
            return out + ([dgate.sum(0), dup.sum(0), dy.sum(0)] if bd is not None else [])
        if case["op"] == "norm":
            square = sum(float(torch.dot(g.double().view(-1), g.double().view(-1))) for g in state["grads"])
            total = math.sqrt(square) / LOSS_SCALE
            value = lambda v: torch.tensor(v, dtype=torch.float64, device=DEV)  # noqa: E731
            return [value(total), value(min(1.0, MAX_NORM / (total + 1e-6)) / LOSS_SCALE)]
        h, (b1, b2) = state["hyper"], state["hyper"]["betas"]
        scale = float(state["grad_scale"]) if case["scaled"] else 1.0
        t = int(state["steps"][0][0]) + 1
        if case["bits"] == 8:  # by tensor: the scales belong to the elements of one tensor
            shapes = _shapes(case)
            wide, views = {}, {}
            for key in ("exp_avg", "exp_avg_sq"):
                wide[key], views[key] = _flat(shapes, torch.float64)
                for v, c, s in zip(views[key], state[key + "s"], state[key + "_scales"]):
                    v.copy_((c.double().view(-1) * s.double().repeat_interleave(BLOCK)[:c.numel()]).view(c.shape))
            m, v = wide["exp_avg"], wide["exp_avg_sq"] ** 2
        else:
            m, v = state["exp_avg"].double(), state["exp_avg_sq"].double()
        grads, grad_views = _flat(_shapes(case), torch.float64)
        for a, b in zip(grad_views, state["grads"]):
            a.copy_(b)
        grads *= scale
        p = (state["master"] if case["master"] else state["p"]).double()
        m = torch.lerp(grads, m, b1)
        v = torch.lerp(grads * grads, v, b2)
        new = p * (1 - h["lr"] * h["weight_decay"]) - h["lr"] * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + h["eps"])
        out = {"p": new, "exp_avg": m, "exp_avg_sq": v}
        if case["master"]:
            out["master"] = new
        if case["bits"] == 8:  # codes are rounded at random within a step: they have no one value
            out.update(exp_avg=None, exp_avg_sq=None)
        return out
