"""Gated residual, norm and modulation, and their gradient, against the formulas in 64 bits, element by element.

Where the bounds come from.  A result is rounded once: u = ``finfo.eps / 2`` of its type, relative.  Everything before is fp32:
a few operations of 2^-24 and sums of up to 8,192 channels in trees of at most 64 sequential terms, all within 2^-17 of the sum
of the magnitudes that a result adds up (``W``); a layer norm's mean leaves 2^-24 of the row's largest value in every channel,
which is inside the same bound once the largest normalised value is counted.  Column sums add up to some thousand rows one
after the other: 1,000 x 2^-24 = 6e-5 of the sum of the magnitudes (``S``).  fp16 has no exponents below 2^-14: smaller values
are multiples of 2^-24, and off by 2^-25 (``_tiny``)."""

import pytest
import torch

W, S, EPS = 2.0 ** -17, 1e-4, 1e-6


def _tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def _normalise(t, kind):
    c = t - t.mean(-1, keepdim=True) if kind == "layer" else t
    r = 1 / (c.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    return c * r, r


def _inputs(lead, frames, width, dtype, mod, weighted, post, seed):
    """x [*lead, C]; modulation [*lead[:-1], frames, C]."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0, mean=0.0, kind=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * std + mean).to(kind)

    loud = torch.ones(width, device="cuda")
    loud[::7] = 12.0
    x = (torch.randn(*lead, width, generator=gen, device="cuda") * loud + 0.5).to(dtype)
    shape = (*lead[:-1], frames, width)
    t = dict(x=x, y=randn(*lead, width, mean=0.3), gate=randn(*shape, std=0.3, mean=0.2, kind=mod),
             scale=randn(*shape, std=0.2, kind=mod), shift=randn(*shape, std=0.2, kind=mod),
             weight=randn(width, std=0.1, mean=1.0) if weighted else None,
             post_weight=randn(width, std=0.1, mean=1.0) if weighted and post else None)
    return t, randn(*lead, width, std=0.1), randn(*lead, width, std=0.1)


def _spread(t, lead):
    """Modulation rows repeated for the tokens that share them."""
    if t.ndim == 1:
        return t.double()
    return t.double().repeat_interleave(lead[-1] // t.shape[-2], dim=-2)


def _check_forward(t, norm, post, got, lead):
    x_out, h = got
    u, tiny = torch.finfo(t["x"].dtype).eps / 2, _tiny(t["x"].dtype)
    gate, scale, shift = (_spread(t[k], lead) for k in ("gate", "scale", "shift"))
    y = t["y"].double()
    if post:
        y = _normalise(y, post)[0]
        y = y if t["post_weight"] is None else y * t["post_weight"].double()
    want = t["x"].double() + gate * y
    size = t["x"].double().abs() + (gate * y).abs() + gate.abs() * (y.abs().amax(-1, keepdim=True) if post else 0)
    assert ((x_out.double() - want).abs() <= u * want.abs() + W * size + tiny).all()
    a = _normalise(want, norm)[0]
    f = (1 + scale) if t["weight"] is None else (1 + scale) * t["weight"].double()
    h_want = a * f + shift
    size = (a.abs().amax(-1, keepdim=True) + 1) * f.abs() * (1 + size / want.abs().amax(-1, keepdim=True)) + shift.abs()
    assert ((h.double() - h_want).abs() <= u * h_want.abs() + W * size + tiny).all()


def _check_backward(t, d_x, d_h, norm, post, grads, lead, groups_dims):
    """``t["x"]`` is the stream behind the residual."""
    u, tiny = torch.finfo(t["x"].dtype).eps / 2, _tiny(t["x"].dtype)
    gate, scale = _spread(t["gate"], lead), _spread(t["scale"], lead)
    one = torch.ones((), dtype=torch.float64, device="cuda")
    w = one if t["weight"] is None else t["weight"].double()
    pw = one if t["post_weight"] is None else t["post_weight"].double()
    zero = torch.zeros_like(t["x"], dtype=torch.float64)
    d, e = (zero if g is None else g.double() for g in (d_h, d_x))

    def norm_gradient(g, a, r, kind):
        out = g - a * (g * a).mean(-1, keepdim=True)
        size = g.abs() + (a.abs() + 1) * (g * a).abs().mean(-1, keepdim=True)
        if kind == "layer":
            out = out - g.mean(-1, keepdim=True)
            size = size + g.abs().mean(-1, keepdim=True) * (1 + a.abs().amax(-1, keepdim=True))
        return out * r, size * r

    a, r = _normalise(t["x"].double(), norm)
    dx, size = norm_gradient(d * (1 + scale) * w, a, r, norm)
    dx, size = dx + e, size + e.abs()
    assert ((grads.x.double() - dx).abs() <= u * dx.abs() + W * size + tiny).all()
    y, q = (t["y"].double(), one) if not post else _normalise(t["y"].double(), post)
    if post:
        dy, dy_size = norm_gradient(gate * dx * pw, y, q, post)
        dy_size = dy_size + norm_gradient((gate * pw).abs() * size, y, q, post)[1]
    else:
        dy, dy_size = gate * dx, gate.abs() * size
    assert ((grads.y.double() - dy).abs() <= u * dy.abs() + W * dy_size + tiny).all()
    tops = a.abs().amax(-1, keepdim=True) if norm == "layer" else a.abs()
    y_tops = y.abs().amax(-1, keepdim=True) if post == "layer" else y.abs()

    def close(got, terms, sizes, like):
        if like.ndim == 1:
            want, size = terms.flatten(0, -2).sum(0), sizes.flatten(0, -2).sum(0)
        else:
            per = lead[-1] // like.shape[-2]
            want, size = (v.unflatten(-2, (-1, per)).sum(-2) for v in (terms, sizes))
        um = torch.finfo(got.dtype).eps / 2
        assert got.shape == like.shape and got.dtype == like.dtype
        assert ((got.double() - want).abs() <= um * want.abs() + S * size + _tiny(got.dtype)).all()

    close(grads.gate, dx * y * pw, (size * y_tops * pw).abs(), t["gate"])
    if d_h is not None:
        close(grads.scale, d * a * w, (d * tops * w).abs(), t["scale"])
        close(grads.shift, d, d.abs(), t["shift"])
        if t["weight"] is not None:
            close(grads.weight, d * (1 + scale) * a, (d * (1 + scale) * tops).abs(), t["weight"])
    if t["post_weight"] is not None:
        close(grads.post_weight, gate * dx * y, (gate * size * y_tops).abs(), t["post_weight"])


def _run(lead, frames, width, dtype, mod, weighted, norm, post, seed):
    from anemoi_b200.modulation import fused_gate_norm_modulate, fused_gate_norm_modulate_backward

    t, d_x, d_h = _inputs(lead, frames, width, dtype, mod, weighted, post, seed)
    args = [t[k] for k in ("x", "y", "gate", "scale", "shift", "weight", "post_weight")]
    kw = dict(eps=EPS, norm=norm, post_norm=post)
    _check_forward(t, norm, post, fused_gate_norm_modulate(*args, **kw), lead)
    back = [t[k] for k in ("x", "y", "gate", "scale", "weight", "post_weight")]
    grads = fused_gate_norm_modulate_backward(d_x, d_h, *back, **kw)
    _check_backward(t, d_x, d_h, norm, post, grads, lead, None)
    again = fused_gate_norm_modulate_backward(d_x, d_h, *back, **kw)
    assert all(a is None or torch.equal(a, b) for a, b in zip(grads, again))
    return t, d_x, d_h, back, kw


@pytest.mark.gpu
@pytest.mark.parametrize("width", [8, 64, 72, 256, 264, 520, 1024, 1032, 1160, 2048, 2056, 5376, 5640, 8192])
@pytest.mark.parametrize("dtype, mod, norm, post, weighted",
                         [(torch.bfloat16, torch.bfloat16, "rms", None, False), (torch.float16, torch.float32, "layer", "rms", True),
                          (torch.bfloat16, torch.float32, "rms", "layer", True), (torch.float16, torch.float16, "layer", None, True)])
def test_widths(native_library, width, dtype, mod, norm, post, weighted):
    _run((2, 33), 3, width, dtype, mod, weighted, norm, post, seed=width)


@pytest.mark.gpu
@pytest.mark.parametrize("lead, frames", [((1, 1), 1), ((1, 7), 7), ((1, 700), 1), ((3, 400), 1), ((2, 300), 100), ((2, 260), 260),
                                          ((1, 2500), 5), ((5, 1), 1)])
@pytest.mark.parametrize("width, weighted, post", [(136, True, "rms"), (1160, False, None), (5376, True, "rms")])
def test_rows_and_groups(native_library, lead, frames, width, weighted, post):
    """One token, one group, a group per token, more groups than blocks, groups that several blocks share."""
    _run(lead, frames, width, torch.bfloat16, torch.bfloat16, weighted, "rms", post, seed=lead[1])


@pytest.mark.gpu
def test_forms_of_the_modulation(native_library):
    """[C], one row per sample, chunks of one wider tensor, and rows repeated by expand give the same as their full form."""
    from anemoi_b200.modulation import (fused_gate_norm_modulate, fused_gate_norm_modulate_backward, fused_gate_residual,
                                        fused_norm_modulate)

    gen = torch.Generator(device="cuda").manual_seed(1)
    x, y, d = (torch.randn(2, 30, 256, generator=gen, device="cuda").bfloat16() for _ in range(3))
    wide = torch.randn(2, 6 * 256, generator=gen, device="cuda").bfloat16()
    shift, scale, gate, *_ = wide.chunk(6, dim=-1)                          # rows six widths apart
    want = fused_gate_norm_modulate(x, y, gate.contiguous(), scale.contiguous(), shift.contiguous())
    for form in (lambda t: t, lambda t: t[:, None], lambda t: t[:, None].expand(2, 30, 256)):
        got = fused_gate_norm_modulate(x, y, form(gate), form(scale), form(shift))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    grads = fused_gate_norm_modulate_backward(d, d, want[0], y, gate, scale)
    assert grads.gate.shape == (2, 256)
    # one row for all of gate, one per sample of scale: gate's gradient is the sum
    one = gate[0].contiguous()
    got = fused_gate_norm_modulate(x, y, one, scale, shift)
    full = fused_gate_norm_modulate(x, y, one.expand(2, 256).contiguous(), scale, shift)
    assert torch.equal(got[0], full[0]) and torch.equal(got[1], full[1])
    grads = fused_gate_norm_modulate_backward(d, d, got[0], y, one, scale)
    full = fused_gate_norm_modulate_backward(d, d, got[0], y, one.expand(2, 256).contiguous(), scale)
    assert grads.gate.shape == (256,) and torch.equal(grads.scale, full.scale)
    terms = full.gate.double().abs().sum(0)
    assert ((grads.gate.double() - full.gate.double().sum(0)).abs() <= 2.0 ** -8 * terms).all()
    # the parts alone
    assert torch.equal(fused_gate_residual(x, y, gate), want[0])
    h = fused_norm_modulate(x, scale, shift)
    a = _normalise(x.double(), "rms")[0] * (1 + scale.double()[:, None]) + shift.double()[:, None]
    assert ((h.double() - a).abs() <= 2.0 ** -8 * a.abs() + W * (a.abs().amax() + 1)).all()
    # odd offsets and rows of a wider tensor
    rows = torch.randn(60, 512, generator=gen, device="cuda").bfloat16()
    part = rows[:, 128:384].unflatten(0, (2, 30))
    assert torch.equal(fused_norm_modulate(part, scale, shift), fused_norm_modulate(part.contiguous(), scale, shift))
    odd = torch.randn(256 + 1, generator=gen, device="cuda").bfloat16()[1:]
    assert torch.equal(fused_norm_modulate(x, odd), fused_norm_modulate(x, odd.clone()))


@pytest.mark.gpu
def test_one_output_without_gradient_and_no_rows(native_library):
    from anemoi_b200.modulation import fused_gate_norm_modulate_backward

    t, d_x, d_h, back, kw = _run((2, 40), 2, 320, torch.bfloat16, torch.bfloat16, True, "rms", "rms", seed=3)
    grads = fused_gate_norm_modulate_backward(d_x, None, *back, **kw)
    _check_backward(t, d_x, None, "rms", "rms", grads, (2, 40), None)
    assert grads.scale is None and grads.weight is None
    grads = fused_gate_norm_modulate_backward(None, d_h, *back, **kw)
    _check_backward(t, None, d_h, "rms", "rms", grads, (2, 40), None)
    none = [v if v is None or v.ndim == 1 else v[:0] for v in back]
    grads = fused_gate_norm_modulate_backward(d_x[:0], d_h[:0], *none, **kw)
    assert grads.x.shape == (0, 40, 320) and not grads.weight.any() and grads.gate.shape == (0, 2, 320)


@pytest.mark.gpu
def test_rows_of_zeros_without_eps(native_library):
    """eps = 0 and a row of zeros is 0 / 0 in that row; the rows that fill a step up are no rows."""
    from anemoi_b200.modulation import fused_gate_norm_modulate_backward

    for width in (256, 1160, 5376):
        gen = torch.Generator(device="cuda").manual_seed(width)
        x, y, d = (torch.randn(1, 301, width, generator=gen, device="cuda").bfloat16() for _ in range(3))
        gate, w = torch.ones(width, device="cuda").bfloat16(), torch.ones(width, device="cuda").bfloat16()
        grads = fused_gate_norm_modulate_backward(d, d, x, y, gate, gate, w, w, eps=0.0, post_norm="rms")
        assert all(torch.isfinite(g).all() for g in grads if g is not None)


@pytest.mark.gpu
def test_autograd_matches_the_calls_and_differences(native_library):
    from anemoi_b200.modulation import fused_gate_norm_modulate, fused_gate_norm_modulate_backward

    t, d_x, d_h = _inputs((2, 12), 3, 72, torch.bfloat16, torch.float32, True, "rms", seed=5)
    names = ("x", "y", "gate", "scale", "shift", "weight", "post_weight")
    leaves = [t[k].clone().requires_grad_() for k in names]
    x_out, h = fused_gate_norm_modulate(*leaves, norm="layer", post_norm="rms")
    grads = torch.autograd.grad((x_out, h), leaves, (d_x, d_h))
    want = fused_gate_norm_modulate_backward(d_x, d_h, x_out.detach(), *(t[k] for k in ("y", "gate", "scale", "weight", "post_weight")),
                                             norm="layer", post_norm="rms")
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    # h alone, through an expanded gradient
    x_out, h = fused_gate_norm_modulate(*leaves, norm="layer", post_norm="rms")
    assert all(g is not None for g in torch.autograd.grad(h.sum(), leaves))
    # along a direction, against central differences of the formula in 64 bits
    gen = torch.Generator(device="cuda").manual_seed(2)

    def value(v):
        gate, scale, shift = (m.repeat_interleave(4, dim=-2) for m in v[2:5])
        stream = v[0] + gate * _normalise(v[1], "rms")[0] * v[6]
        out = _normalise(stream, "layer")[0] * v[5] * (1 + scale) + shift
        return (stream * d_x.double()).sum() + (out * d_h.double()).sum()

    at = [v.detach().double() for v in leaves]
    for i, g in enumerate(grads):
        step = torch.randn(at[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        up, down = (value([v + s * 1e-5 * step if j == i else v for j, v in enumerate(at)]) for s in (1, -1))
        slope, along = (up - down) / 2e-5, (g.double() * step).sum()
        # the saved stream is rounded (2^-9 of it, which moves the norm's gradient by as much), and so is each value of g
        assert (along - slope).abs() <= 8 * 2.0 ** -8 * g.double().norm() + 1e-4


@pytest.mark.gpu
def test_captured(native_library):
    from anemoi_b200.modulation import fused_gate_norm_modulate, fused_gate_norm_modulate_backward

    t, d_x, d_h = _inputs((1, 900), 1, 1160, torch.float16, torch.float16, True, "rms", seed=6)
    args = [t[k] for k in ("x", "y", "gate", "scale", "shift", "weight", "post_weight")]
    back = [t[k] for k in ("x", "y", "gate", "scale", "weight", "post_weight")]

    def both():
        return [*fused_gate_norm_modulate(*args, post_norm="rms"),
                *fused_gate_norm_modulate_backward(d_x, d_h, *back, post_norm="rms")]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    t["x"].copy_(torch.randn_like(t["x"]))
    graph.replay()
    torch.cuda.synchronize()
    assert all(a is None or torch.equal(a, b) for a, b in zip(got, both()))


@pytest.mark.gpu
def test_an_eps_that_changes_in_place(native_library):
    """Calls are told apart by the value of eps, not by the object."""
    from anemoi_b200.modulation import fused_norm_modulate

    x, eps = torch.ones(4, 64, device="cuda", dtype=torch.bfloat16), torch.tensor(0.0)
    for value in (1.0, 3.0):
        eps.fill_(value)
        assert torch.equal(fused_norm_modulate(x, eps=eps), fused_norm_modulate(x, eps=value))


@pytest.mark.gpu
def test_calls_of_two_threads(native_library):
    """Widths that one kernel serves with different amounts of shared memory."""
    import threading

    from anemoi_b200.modulation import fused_gate_norm_modulate_backward

    failed = []

    def work(width):
        try:
            t, d_x, d_h = _inputs((1, 64), 1, width, torch.bfloat16, torch.bfloat16, True, "rms", seed=width)
            back = [t[k] for k in ("x", "y", "gate", "scale", "weight", "post_weight")]
            with torch.cuda.stream(torch.cuda.Stream()):
                torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
                first = fused_gate_norm_modulate_backward(d_x, d_h, *back, post_norm="rms")
                for _ in range(300):
                    again = fused_gate_norm_modulate_backward(d_x, d_h, *back, post_norm="rms")
                    if not all(a is None or torch.equal(a, b) for a, b in zip(first, again)):
                        failed.append(width)
        except Exception as error:
            failed.append(error)

    threads = [threading.Thread(target=work, args=(width,)) for width in (1160, 2048, 4104, 5376)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failed


def _cpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_refusals():
    """The plan refuses what the kernels cannot take; its layouts name a device without touching it."""
    from anemoi_b200.modulation import _plan

    cuda = torch.device("cuda", 0)

    def layout(*shape, dtype=torch.bfloat16, stride=None):
        steps = stride or torch.empty(shape, device="meta").stride()
        return torch.Size(shape), tuple(steps), dtype, cuda

    x, c = layout(2, 30, 64), layout(64)

    def plan(x=x, y=x, gate=c, scale=c, shift=c, weight=None, post_weight=None, eps=1e-6, norm="rms", post=None):
        return _plan(x, y, gate, scale, shift, weight, post_weight, eps, norm, post)

    assert plan().groups == 1 and plan(gate=layout(2, 64), scale=c).groups == 2 and plan(gate=layout(2, 5, 64)).groups == 10
    wide = layout(2, 30, 12)
    for bad, match in ((dict(x=wide, y=wide), "multiple of 8"), (dict(x=layout(2, 8200), y=layout(2, 8200)), "at most 8192"),
                       (dict(y=layout(2, 30, 128)), "shape"), (dict(gate=layout(30, 64)), "got"), (dict(gate=layout(2, 7, 64)), "got"),
                       (dict(gate=layout(64, dtype=torch.float32)), "one dtype"), (dict(gate=layout(64, dtype=torch.float16)), "gate"),
                       (dict(gate=layout(2, 64), scale=layout(2, 5, 64)), "same tokens"), (dict(norm="batch"), "norm"), (dict(post="x"), "norm"),
                       (dict(eps=-1.0), "eps"), (dict(gate=None), "together"), (dict(post_weight=c), "post_norm"),
                       (dict(weight=layout(32)), "weight"), (dict(x=layout(2, 30, 64, stride=(5000, 64, 1))), "one stride"),
                       (dict(x=layout(2, 30, 64, stride=(30 * 68, 68, 1))), "16 bytes"),
                       (dict(x=layout(2, 30, 64, dtype=torch.float32)), "fp16 or bf16")):
        if "x" in bad and "y" not in bad:
            bad = dict(bad, y=x if bad["x"][2] == torch.bfloat16 else bad["x"])
        with pytest.raises(ValueError, match=match):
            plan(**bad)


def test_the_library_refuses(native_library):
    import ctypes as C

    from anemoi_b200 import native

    good = dict(rows=60, groups=2, width=64, norm=1, post=0, is_bf16=1, mod_is_fp32=0, eps=1e-6)
    at, odd = C.c_void_p(1 << 20), C.c_void_p((1 << 20) + 2)

    def call(x=at, gate=at, h=at, strides=(64, 64, 0, 0, 0), **change):
        return native_library.anemoi_sm100_gate_norm_modulate(
            C.byref(native.Rows(**{**good, **change})), x, at, gate, at, at, None, None, (C.c_int64 * 5)(*strides), at, h, None)

    for change in (dict(rows=-1), dict(groups=0), dict(groups=7), dict(width=60), dict(norm=0), dict(norm=3), dict(post=3),
                   dict(eps=-1.0), dict(eps=float("nan"))):
        assert call(**change) == -1, change
    assert call(width=8200) == -3
    assert call(x=None) == -1 and call(x=odd) == -1 and call(gate=None) == -1 and call(strides=(60, 64, 0, 0, 0)) == -1
    assert call(strides=(-64, 64, 0, 0, 0)) == -1
    assert call(rows=0) == 0
    assert native_library.anemoi_sm100_gate_norm_modulate_backward_workspace(C.byref(native.Rows(**good)), 1) > 0
