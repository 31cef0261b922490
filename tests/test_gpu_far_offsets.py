"""Elements that lie more than 2^31 elements behind a tensor's first: their results are those of the same rows in a tensor of
their own, bit for bit.  (Each row's arithmetic is its own; nothing is said here about values.)"""

import pytest
import torch

FAR = 2 ** 31


def _random(*shape, seed, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


@pytest.mark.gpu
def test_rows_of_the_modulation(native_library):
    from anemoi_b200.modulation import fused_gate_norm_modulate, fused_gate_norm_modulate_backward

    width, last = 5376, 1000
    rows = FAR // width + 2 * last
    x, y = _random(1, rows, width, seed=1), _random(1, rows, width, seed=2)
    gate, scale, shift = _random(3, width, seed=3).unbind(0)
    out = fused_gate_norm_modulate(x, y, gate, scale, shift)
    few = fused_gate_norm_modulate(x[:, -last:].clone(), y[:, -last:].clone(), gate, scale, shift)
    for got, want in zip(out, few):
        assert torch.equal(got[:, -last:], want)
    grads = fused_gate_norm_modulate_backward(x, y, out[0], y, gate, scale)
    few = fused_gate_norm_modulate_backward(x[:, -last:].clone(), y[:, -last:].clone(), out[0][:, -last:].clone(),
                                            y[:, -last:].clone(), gate, scale)
    assert torch.equal(grads.x[:, -last:], few.x) and torch.equal(grads.y[:, -last:], few.y)


@pytest.mark.gpu
def test_heads_of_the_rotary(native_library):
    from anemoi_b200.producer import AxialRotary, fused_qknorm_axial_rope, fused_qknorm_axial_rope_backward

    heads, last = 56, 500
    tokens = FAR // (heads * 128) + 2 * last
    rotary, w = AxialRotary((8, 12, 12)), _random(128, seed=4)
    q, d = _random(1, tokens, heads, 128, seed=5), _random(1, tokens, heads, 128, seed=6)
    at = torch.arange(3 * tokens, device="cuda").view(tokens, 3)
    out, _ = fused_qknorm_axial_rope(q, None, w, None, at, rotary)
    few, _ = fused_qknorm_axial_rope(q[:, -last:].clone(), None, w, None, at[-last:], rotary)
    assert torch.equal(out[:, -last:], few)
    del out
    dq = fused_qknorm_axial_rope_backward(d, None, q, None, w, None, at, rotary)[0]
    few = fused_qknorm_axial_rope_backward(d[:, -last:].clone(), None, q[:, -last:].clone(), None, w, None, at[-last:], rotary)[0]
    assert torch.equal(dq[:, -last:], few)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_queries_of_the_dense_attention(native_library, d):
    from anemoi_b200.dense import dense_attention, dense_attention_backward

    heads, last = 7168 // d, 640
    tokens = (FAR // (heads * d) // 128 + 10) * 128
    q, do = _random(1, tokens, heads, d, seed=7), _random(1, tokens, heads, d, seed=8)
    k, v = _random(2, 1, 70, heads // 8, d, seed=9).unbind(0)
    out, lse = dense_attention(q, k, v, return_lse=True)
    dq, dk, dv = dense_attention_backward(do, q, k, v, out, lse)
    tail = [t[:, -last:].clone() for t in (q, do)]
    few, few_lse = dense_attention(tail[0], k, v, return_lse=True)
    assert torch.equal(out[:, -last:], few) and torch.equal(lse[..., -last:], few_lse)
    assert torch.equal(dq[:, -last:], dense_attention_backward(tail[1], tail[0], k, v, few, few_lse)[0])
    assert torch.isfinite(dk).all() and torch.isfinite(dv).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_keys_far_apart(native_library, d):
    """Keys and values as rows of a long cache, each a long stride behind the one before."""
    from anemoi_b200.dense import dense_attention, dense_attention_backward

    tokens = 4000
    step = (FAR // tokens // 8 + 100) * 8
    cache = torch.zeros(tokens * step, device="cuda", dtype=torch.bfloat16)
    far = [cache[i * d:].as_strided((1, tokens, 1, d), (tokens * step, step, d, 1)) for i in range(2)]
    near = _random(2, 1, tokens, 1, d, seed=10).unbind(0)
    for a, b in zip(far, near):
        a.copy_(b)
    q, do = _random(1, 300, 2, d, seed=11), _random(1, 300, 2, d, seed=12)
    results = []
    for k, v in (far, near):
        out, lse = dense_attention(q, k, v, return_lse=True)
        results.append((out, lse, *dense_attention_backward(do, q, k, v, out, lse)))
    for got, want in zip(*results):
        assert torch.equal(got, want)
