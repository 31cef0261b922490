"""The fused norms, the axial rotary and dense attention as they are used together: the block stack's forward pass and its
gradients, against the same formulas in 64 bits.

The bound: eager torch in the same 16-bit type rounds at every operation, the fused path at the end of each fused one, so that
its distance from 64 bits may be 1.5 times the eager one's at most (the tensor cores' 16-bit operands P and dS are roundings
that both have: torch's attention has them, too)."""

import pytest
import torch
import torch.nn.functional as F


def _eager(stack, x, positions, sections, kind):
    """The stack's formulas in ``kind``, differentiable."""
    c = stack.config

    def norm(t):
        t32 = t if kind == torch.float64 else t.float()
        return (t32 * torch.rsqrt(t32.pow(2).mean(-1, keepdim=True) + c.eps)).to(kind)

    columns = []
    for axis, n in enumerate(sections):
        columns.append(positions[:, axis : axis + 1].double() * 10000.0 ** -(torch.arange(n, device=x.device).double() / n))
    angle = torch.cat(columns, -1)[None, :, None]
    wide = torch.float64 if kind == torch.float64 else torch.float32
    cos, sin = torch.cos(angle).to(wide), torch.sin(angle).to(wide)
    p = sum(sections)

    def rope(t, w):
        t = norm(t).to(wide) * w.to(wide)
        a, b = t[..., :p], t[..., p : 2 * p]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, t[..., 2 * p :]), -1).to(kind)

    for blk in stack.blocks:
        w = {name: t.to(kind) for name, t in blk.items()}
        shift1, scale1, gate1, shift2, scale2, gate2 = w["mod"].unbind(0)
        h = norm(x) * (1 + scale1) + shift1
        q, k, v = ((h @ w[n]).view(*x.shape[:2], c.heads, c.head_dim) for n in ("wq", "wk", "wv"))
        q, k = rope(q, w["qn"]), rope(k, w["kn"])
        attn = F.scaled_dot_product_attention(*(t.transpose(1, 2) for t in (q, k, v))).transpose(1, 2)
        x = x + gate1 * (attn.reshape(*x.shape[:2], c.inner) @ w["wo"])
        h = norm(x) * (1 + scale2) + shift2
        x = x + gate2 * ((F.silu(h @ w["w1"]) * (h @ w["w3"])) @ w["w2"])
    return x


def _stack(dtype, head_dim):
    from anemoi_b200.h3_stack import H3BlockStack, H3StackConfig

    config = H3StackConfig(width=264, heads=4, head_dim=head_dim, ffn_width=512, rotary_dim=32, layers=2)
    stack = H3BlockStack(config, torch.device("cuda"), dtype=dtype, seed=1)
    gen = torch.Generator(device="cuda").manual_seed(2)
    for blk in stack.blocks:
        blk["mod"] = (torch.randn(6, config.width, generator=gen, device="cuda") * 0.3).to(dtype)
        for name in blk:
            blk[name] = blk[name].detach().requires_grad_()
    return stack, gen


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, head_dim", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float16, 64)])
def test_forward_and_gradients_of_the_stack(native_library, dtype, head_dim):
    from anemoi_b200 import VisualLayout
    from anemoi_b200.producer import AxialRotary, axial_positions

    stack, gen = _stack(dtype, head_dim)
    layout = VisualLayout((3, 6, 9), 17)
    positions, sections = axial_positions(layout, "cuda"), (4, 6, 6)
    tokens = positions.size(0)
    assert tokens == 17 + 3 * 6 * 9 and positions[16].tolist() == [16] * 3 and positions[-1].tolist() == [19, 22, 25]
    x = torch.randn(2, tokens, stack.config.width, generator=gen, device="cuda").to(dtype).requires_grad_()
    g = (torch.randn(2, tokens, stack.config.width, generator=gen, device="cuda") * 0.1).to(dtype)
    leaves = [x] + [t for blk in stack.blocks for t in blk.values()]

    def both(out):
        return [out.detach()] + list(torch.autograd.grad(out, leaves, g.to(out.dtype)))

    fused = both(stack.fused_step(x, positions, AxialRotary(sections)))
    eager = both(_eager(stack, x, positions, sections, dtype))
    exact = both(_eager(stack, x.double(), positions, sections, torch.float64))
    for i, (a, b, want) in enumerate(zip(fused, eager, exact)):
        size = want.double().norm()
        off, theirs = ((t.double() - want.double()).norm() / size for t in (a, b))
        assert off <= 1.5 * theirs + 1e-4, f"{i}: {off:.2e} off, eager {theirs:.2e}"


@pytest.mark.gpu
def test_a_tuning_step_captured_into_a_graph(native_library):
    """The whole forward and backward pass replays on new inputs, and the sparse call serves the same stack."""
    from anemoi_b200 import QuantConfig, SparseConfig, VisualLayout, anemoi_attention
    from anemoi_b200.producer import AxialRotary, axial_positions

    stack, gen = _stack(torch.bfloat16, 64)
    layout = VisualLayout((4, 16, 16), 0)
    positions, rotary = axial_positions(layout, "cuda"), AxialRotary((4, 6, 6))
    x = torch.randn(1, 1024, stack.config.width, generator=gen, device="cuda").bfloat16()
    leaves = [t for blk in stack.blocks for t in blk.values()]

    def step():
        out = stack.fused_step(x, positions, rotary)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, torch.ones_like(out)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.copy_(torch.randn(1, 1024, stack.config.width, generator=gen, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    want = step()
    for i, (a, b) in enumerate(zip(got, want)):
        # (library GEMMs may be chosen differently under capture: a 16-bit rounding apart)
        assert ((a.double() - b.double()).norm() <= 2.0 ** -7 * b.double().norm()), i

    def sparse(q, k, v):
        return anemoi_attention(q, k, v, layout=layout, layer=0, sparse_config=SparseConfig(64, 0.5, (), 0.0),
                                quant_config=QuantConfig(0.0, 0.0, 1.0, "fp16", "fp16"))

    with torch.no_grad():
        assert torch.isfinite(stack.fused_step(x, positions, rotary, sparse)).all()
