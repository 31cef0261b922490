"""qk-norm with axial rotary positions, and its gradient, against the formulas in 64 bits, element by element.

Where the bounds come from.  A result is rounded once: u = ``finfo.eps / 2``, relative.  Before that, fp32: the root (2^-22), a
few products (2^-24 each), and a cosine and sine that are off by 2^-20 at most, plus 2^-22 of a turn (2^-19 of an angle) where
positions are large: together within W = 2^-17 of the magnitudes that a result adds up.  A weight's gradient adds up to some
ten thousand rows in parts of a few hundred: 300 x 2^-24 = 2e-5, within S = 1e-4 of the sum of the magnitudes.  fp16 has no
exponents below 2^-14: smaller values are multiples of 2^-24, and off by 2^-25."""

import math

import pytest
import torch

W, S, EPS = 2.0 ** -17, 1e-4, 1e-6


def _turn(positions, rotary):
    """cos + i sin of every pair, [.., T, 1, P]."""
    columns, first, total = [], 0, sum(rotary.sections)
    for axis, n in enumerate(rotary.sections):
        for i in range(n):
            power = (first + i) / total if rotary.shared_frequencies else i / n
            columns.append(positions[..., axis].double() * rotary.theta ** -power)
        first += n
    if not columns:
        return torch.zeros(*positions.shape[:-1], 1, 0, dtype=torch.complex128, device=positions.device)
    angle = torch.stack(columns, -1).unsqueeze(-2)
    return torch.polar(torch.ones_like(angle), angle)


def _pairs(x, rotary):
    p = rotary.pairs
    if rotary.interleaved:
        return torch.view_as_complex(x[..., : 2 * p].unflatten(-1, (p, 2)).contiguous())
    return torch.complex(x[..., :p], x[..., p : 2 * p])


def _flat(z, rest, rotary):
    turned = torch.view_as_real(z).flatten(-2) if rotary.interleaved else torch.cat((z.real, z.imag), -1)
    return torch.cat((turned, rest), -1)


def _rotate(x, turn, rotary):
    return _flat(_pairs(x, rotary) * turn, x[..., 2 * rotary.pairs :], rotary)


def _pair_size(x, rotary):
    """|u| + |v| of each channel's pair."""
    z = _pairs(x, rotary)
    size = z.real.abs() + z.imag.abs()
    return _flat(torch.complex(size, size), x[..., 2 * rotary.pairs :].abs(), rotary)


def _inputs(b, t, hq, hk, d, dtype, normed, seed, packed=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * std + mean).to(dtype)

    def pair(std):
        if packed:
            both = randn(b, t, hq + hk, d, std=std)
            return both[:, :, :hq], both[:, :, hq:]
        return randn(b, t, hq, d, std=std), randn(b, t, hk, d, std=std) if hk else None

    weights = [randn(d, std=0.1, mean=1.0) if normed and n else None for n in (hq, hk)]
    return *pair(1.5), *weights, *pair(0.1)


def _check(b, t, hq, hk, d, dtype, rotary, positions, normed=True, seed=0, packed=False):
    from anemoi_b200.producer import fused_qknorm_axial_rope, fused_qknorm_axial_rope_backward

    q, k, qw, kw, dq, dk = _inputs(b, t, hq, hk, d, dtype, normed, seed, packed)
    u, tiny = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0
    out = fused_qknorm_axial_rope(q, k, qw, kw, positions, rotary, EPS)
    grads = fused_qknorm_axial_rope_backward(dq, dk, q, k, qw, kw, positions, rotary, EPS)
    turn = _turn(positions if positions.ndim == 3 else positions[None], rotary)
    for x, w, g, got, dx, dw in ((q, qw, dq, out[0], grads[0], grads[2]), (k, kw, dk, out[1], grads[1], grads[3])):
        if x is None:
            assert got is None and dx is None and dw is None
            continue
        x, g = x.double(), g.double()
        r = 1 / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        n = x if w is None else x * r * w.double()
        want = _rotate(n, turn, rotary)
        assert ((got.double() - want).abs() <= u * want.abs() + W * _pair_size(n, rotary) + tiny).all()
        back = _rotate(g, turn.conj(), rotary)
        size = _pair_size(g, rotary)
        if w is not None:
            gw, a = back * w.double(), x * r
            want = r * (gw - a * (gw * a).mean(-1, keepdim=True))
            wide = size * w.double().abs()
            size_x = r * (wide + a.abs() * (wide * a.abs()).mean(-1, keepdim=True))
            want_w, size_w = (back * a).sum((0, 1, 2)), (size * a.abs()).sum((0, 1, 2))
            assert ((dw.double() - want_w).abs() <= u * want_w.abs() + S * size_w + tiny).all()
        else:
            want, size_x = back, size
            assert dw is None
        assert ((dx.double() - want).abs() <= u * want.abs() + W * size_x + tiny).all()
    again = fused_qknorm_axial_rope_backward(dq, dk, q, k, qw, kw, positions, rotary, EPS)
    assert all(x is None or torch.equal(x, y) for x, y in zip(grads, again))
    return (q, k, qw, kw, dq, dk), out, grads


def _grid(t, b=None, spread=1, axes=3, kind=torch.int32):
    i = torch.arange(t, device="cuda")
    side = max(1, int(t ** (1 / 3)))
    columns = [i // (side * side), i // side % side, i % side, i % 5][:axes]
    p = torch.stack(columns, -1) * spread
    return (p if b is None else p.expand(b, t, axes) + torch.arange(b, device="cuda")[:, None, None] * 17).to(kind)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, interleaved", [(torch.bfloat16, False), (torch.float16, True)])
@pytest.mark.parametrize("b, t, hq, hk, d, sections", [
    (1, 1, 56, 56, 128, (8, 12, 12)), (1, 37, 3, 3, 128, (16, 24, 24)), (2, 300, 24, 8, 64, (8, 12, 12)), (1, 5, 1, 0, 64, (8,)),
    (3, 70, 7, 2, 128, (0, 40, 0)), (1, 130, 2, 1, 64, (4, 4)), (1, 64, 5, 5, 128, (0, 0)), (2, 41, 9, 4, 128, (16, 16, 16, 16)),
    (1, 3000, 12, 12, 128, (8, 12, 12)), (1, 1, 1, 1, 64, (8, 8, 8)), (4, 1, 130, 3, 64, (8, 8, 16))])
def test_against_the_formula(native_library, dtype, interleaved, b, t, hq, hk, d, sections):
    from anemoi_b200.producer import AxialRotary

    rotary = AxialRotary(sections, interleaved=interleaved)
    _check(b, t, hq, hk, d, dtype, rotary, _grid(t, b, axes=len(sections)), seed=t)
    _check(b, t, hq, hk, d, dtype, rotary, _grid(t, axes=len(sections)), normed=False, seed=t)


@pytest.mark.gpu
@pytest.mark.parametrize("kind, spread", [(torch.int32, 1), (torch.int32, -100_000), (torch.int32, 40_000_000), (torch.int64, 10 ** 9),
                                          (torch.float32, 0.37), (torch.float32, -1000.25)])
@pytest.mark.parametrize("shared, theta", [(False, 10000.0), (True, 1e6), (False, 0.5)])
def test_far_and_fractional_positions(native_library, kind, spread, shared, theta):
    from anemoi_b200.producer import AxialRotary

    positions = _grid(90, 2, kind=torch.float64).mul(spread).to(kind)
    # (a position of 5 * 10^9 times a frequency that is good to 2^-52: 10^-6 of an angle)
    rotary = AxialRotary((8, 12, 12), theta=theta, shared_frequencies=shared)
    _check(2, 90, 4, 2, 64, torch.bfloat16, rotary, positions, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_views_in_place_and_odd_weights(native_library, interleaved):
    from anemoi_b200.producer import AxialRotary, fused_qknorm_axial_rope

    rotary = AxialRotary((8, 12, 12), interleaved=interleaved)
    (q, k, qw, kw, *_), out, _ = _check(2, 130, 6, 3, 128, torch.bfloat16, rotary, _grid(130), seed=5, packed=True)
    both = torch.cat((q, k), dim=2)
    got = fused_qknorm_axial_rope(both[:, :, :6], both[:, :, 6:], qw, kw, _grid(130), rotary, EPS, inplace=True)
    assert got[0].data_ptr() == both.data_ptr()
    assert torch.equal(both[:, :, :6], out[0]) and torch.equal(both[:, :, 6:], out[1])
    odd = torch.empty(129, device="cuda", dtype=qw.dtype)[1:].copy_(qw)
    assert torch.equal(fused_qknorm_axial_rope(q, k, odd, kw, _grid(130), rotary, EPS)[0], out[0])
    # the same positions for each sample, and heads before tokens
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]
    got = fused_qknorm_axial_rope(*turned, qw, kw, _grid(130).expand(2, 130, 3), rotary, EPS)
    assert torch.equal(got[0], out[0]) and torch.equal(got[1], out[1])


@pytest.mark.gpu
def test_agrees_with_the_call_that_takes_tables(native_library):
    """Where one axis has all pairs, the tables of ``fused_qknorm_rope`` say the same; fp32 tables and arithmetic in another order
    move a value across a rounding border at most."""
    from anemoi_b200.producer import AxialRotary, fused_qknorm_axial_rope, fused_qknorm_rope

    q, k, qw, kw, *_ = _inputs(1, 50, 4, 4, 128, torch.bfloat16, True, 7)
    at = torch.arange(50, device="cuda", dtype=torch.int32)[:, None]
    out, _ = fused_qknorm_axial_rope(q, k, qw, kw, at, AxialRotary((32,)), EPS)
    angle = at.double() * 10000.0 ** -(torch.arange(32, device="cuda").double() / 32)
    tables = [f(angle).float().repeat(1, 2) for f in (torch.cos, torch.sin)]
    want = fused_qknorm_rope(q.clone(), qw, *tables, EPS)
    assert ((out.double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 1e-5).all()
    assert (out != want).float().mean() < 0.01


@pytest.mark.gpu
def test_zeros_without_eps_in_heads_that_fill_up(native_library):
    from anemoi_b200.producer import AxialRotary, fused_qknorm_axial_rope_backward

    q, k, qw, kw, dq, dk = _inputs(1, 33, 5, 3, 64, torch.bfloat16, True, 8)
    grads = fused_qknorm_axial_rope_backward(dq, dk, q, k, qw, kw, _grid(33), AxialRotary((8, 8, 8)), 0.0)
    assert all(torch.isfinite(g).all() for g in grads)


@pytest.mark.gpu
def test_autograd_and_differences(native_library):
    from anemoi_b200.producer import AxialRotary, fused_qknorm_axial_rope, fused_qknorm_axial_rope_backward

    rotary, at = AxialRotary((4, 8, 4), interleaved=True), _grid(20, 2)
    q, k, qw, kw, dq, dk = _inputs(2, 20, 4, 2, 64, torch.float16, True, 9)
    leaves = [t.clone().requires_grad_() for t in (q, k, qw, kw)]
    out = fused_qknorm_axial_rope(*leaves, at, rotary, EPS)
    grads = torch.autograd.grad(out, leaves, (dq, dk))
    want = fused_qknorm_axial_rope_backward(dq, dk, q, k, qw, kw, at, rotary, EPS)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    total = torch.autograd.grad(fused_qknorm_axial_rope(*leaves, at, rotary, EPS)[0].sum(), leaves[0])
    ones = fused_qknorm_axial_rope_backward(torch.ones_like(dq), dk, q, k, qw, kw, at, rotary, EPS)
    assert torch.equal(total[0], ones[0])
    with pytest.raises(ValueError, match="overwrites"):
        fused_qknorm_axial_rope(*leaves, at, rotary, EPS, inplace=True)
    gen = torch.Generator(device="cuda").manual_seed(1)
    turn = _turn(at, rotary)

    def value(v):
        total = 0
        for x, w, g in ((v[0], v[2], dq), (v[1], v[3], dk)):
            n = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w
            total = total + (_rotate(n, turn, rotary) * g.double()).sum()
        return total

    here = [t.double() for t in (q, k, qw, kw)]
    for i, g in enumerate(grads):
        step = torch.randn(here[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        up, down = (value([v + s * 1e-5 * step if j == i else v for j, v in enumerate(here)]) for s in (1, -1))
        # each value of g is off by half a step: a random sum of those, five times over
        assert ((up - down) / 2e-5 - (g.double() * step).sum()).abs() <= 5 * 2.0 ** -11 * g.double().norm() + 1e-6


@pytest.mark.gpu
def test_captured_and_no_tokens(native_library):
    from anemoi_b200.producer import AxialRotary, fused_qknorm_axial_rope, fused_qknorm_axial_rope_backward

    rotary, at = AxialRotary((8, 12, 12)), _grid(400)
    q, k, qw, kw, dq, dk = _inputs(1, 400, 6, 6, 128, torch.bfloat16, True, 10)

    def both():
        return [*fused_qknorm_axial_rope(q, k, qw, kw, at, rotary, EPS),
                *fused_qknorm_axial_rope_backward(dq, dk, q, k, qw, kw, at, rotary, EPS)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    q.copy_(torch.randn_like(q))
    at += 3
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, both()))
    out = fused_qknorm_axial_rope(q[:, :0], k[:, :0], qw, kw, at[:0], rotary, EPS)
    assert out[0].shape == (1, 0, 6, 128)
    grads = fused_qknorm_axial_rope_backward(dq[:, :0], dk[:, :0], q[:, :0], k[:, :0], qw, kw, at[:0], rotary, EPS)
    assert not grads[2].any() and grads[0].shape == (1, 0, 6, 128)


@pytest.mark.gpu
def test_an_eps_that_changes_and_places_that_are_shared(native_library):
    from anemoi_b200.producer import AxialRotary, fused_qknorm_axial_rope

    q, k, qw, kw, *_ = _inputs(1, 50, 4, 4, 128, torch.bfloat16, True, 8)
    rotary, at, eps = AxialRotary((8, 12, 12)), _grid(50), torch.tensor(0.0)
    for value in (0.5, 3.0):
        eps.fill_(value)
        got, want = (fused_qknorm_axial_rope(q, k, qw, kw, at, rotary, e) for e in (eps, value))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # in place: rows that lie on one another, and queries that are the keys
    one = q[:, :, :1].expand_as(q)
    for a, b in ((one, k), (q, one), (q, q)):
        with pytest.raises(ValueError, match="inplace"):
            fused_qknorm_axial_rope(a, b, qw, kw, at, rotary, EPS, inplace=True)
    assert fused_qknorm_axial_rope(one, k, qw, kw, at, rotary, EPS)[0].shape == q.shape


def test_refusals():
    from anemoi_b200.producer import AxialRotary, _axial_plan, fused_qknorm_axial_rope

    for bad in (dict(sections=()), dict(sections=(1,) * 5), dict(sections=(4, 2)), dict(sections=(-8, 16)), dict(sections=(72,)),
                dict(sections=(8.0,)), dict(sections=[8]), dict(sections=(8,), theta=0.0), dict(sections=(8,), theta=math.inf), dict(sections=(4,))):
        with pytest.raises(ValueError):
            AxialRotary(**bad)
    assert AxialRotary((4,), interleaved=True).pairs == 4
    cuda = torch.device("cuda", 0)

    def layout(*shape, dtype=torch.bfloat16, stride=None, device=cuda):
        return torch.Size(shape), tuple(stride or torch.empty(shape, device="meta").stride()), dtype, device

    q, w, at, rotary = layout(1, 4, 2, 64), layout(64), layout(4, 1, dtype=torch.int32), AxialRotary((32,))

    def plan(q=q, k=q, qw=w, kw=w, at=at, rotary=rotary, eps=1e-6):
        return _axial_plan(q, k, qw, kw, at, rotary, eps)

    odd = layout(1, 4, 2, 64, stride=(600, 132, 66, 1))
    for bad in (dict(q=layout(4, 2, 64)), dict(q=layout(1, 4, 2, 96)), dict(k=layout(1, 5, 2, 64)), dict(qw=None), dict(k=None),
                dict(qw=layout(32)), dict(at=layout(4, 2, dtype=torch.int32)), dict(at=layout(4, 1, dtype=torch.float64)),
                dict(at=layout(2, 4, 1, dtype=torch.int32)), dict(rotary=AxialRotary((64,))), dict(eps=-1.0), dict(q=odd, k=odd),
                dict(q=layout(1, 4, 0, 64)), dict(q=layout(1, 4, 2, 64, device=torch.device("cpu")))):
        with pytest.raises(ValueError):
            plan(**bad)
    with pytest.raises(TypeError):
        plan(rotary=(32,))
    t = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        fused_qknorm_axial_rope(t, t, None, None, torch.zeros(4, 1, dtype=torch.int32), rotary)


def test_the_library_refuses(native_library):
    import ctypes as C

    from anemoi_b200 import native

    good = dict(batch=1, tokens=4, q_heads=2, k_heads=2, head_dim=64, axes=1, sections=(C.c_int32 * 4)(32), interleaved=0,
                positions_type=0, is_bf16=1, eps=1e-6)
    at, odd = C.c_void_p(1 << 20), C.c_void_p((1 << 20) + 2)
    turns = (C.c_double * 32)()

    def call(q=at, kw=at, strides=(512, 128, 64) * 4, **change):
        return native_library.anemoi_sm100_axial_rope(
            C.byref(native.AxialRopeShape(**{**good, **change})), q, at, at, kw, at, 0, turns, (C.c_int64 * 12)(*strides), at, at,
            None)

    for change in (dict(batch=-1), dict(tokens=-1), dict(q_heads=0), dict(k_heads=-1), dict(head_dim=96), dict(axes=0), dict(axes=5),
                   dict(sections=(C.c_int32 * 4)(40)), dict(sections=(C.c_int32 * 4)(4)), dict(sections=(C.c_int32 * 4)(-8)),
                   dict(positions_type=3), dict(eps=-1.0)):
        assert call(**change) == -1, change
    for change in (dict(q_heads=5000), dict(tokens=1 << 30), dict(batch=70000)):
        assert call(**change) == -3, change
    assert call(q=odd) == -1 and call(q=None) == -1 and call(kw=None) == -1 and call(strides=(512, 128, 60) * 4) == -1
    assert call(tokens=0) == 0
