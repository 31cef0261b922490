"""Dense attention and its gradient against the formulas in 64 bits, element by element.

Where the bounds come from (u: half a step of the type, ``finfo.eps / 2``).  The kernels round P and dS to the type as operands
and their results at the end; products are exact, sums are fp32.  fp32 sums over D <= 128 channels or up to a thousand tokens
and the exponentials (2^-22, of arguments below 2^6 that are good to 2^-17) stay within ``w = 1e-4`` of the sum of the magnitudes
(1,000 terms x 2^-24 = 6e-5, plus 2^-17 and 2^-22).  With s = the sum of magnitudes that a result adds up:

(longer sums: their terms x 2^-24.)
    out   u s(P |v|)                + u |out| + w s
    dV    u s(P |dO|)               + u |dV|  + w s
    e_ij  |error of dS_ij| <= u |dS_ij| + P_ij |delta_i given - delta_i| + w P_ij (|dO_i| . |v_j| + |dO_i| . |out_i|)
    dQ    scale s(e |k|) + u |dQ| + w scale s(|dS| |k|),  dK alike

delta is dO . out of the rounded ``out`` that the call is given, so its exact distance from the formula's is used.  fp16
operands below 2^-14 lose bits: P times 2^15 is off by 2^-25, P by 2^-40 (in the forward pass, times 2^7, by 2^-32); dS,
scaled so that 2 max|dO| max|v| lies above 2^13, by 2^-25 2^-13 2 max|dO| max|v|.
"""

import math

import pytest
import torch

W = 1e-4


def _mask(nq, nk, q_len, k_len, causal, device):
    i = torch.arange(nq, device=device)[:, None]
    j = torch.arange(nk, device=device)[None, :]
    seen = (i < q_len) & (j < k_len)
    return seen & (j <= i + k_len - q_len) if causal else seen


def _reference(q, k, v, do, out, scale, causal, q_lens, k_lens):
    """(values, bounds) of out, lse, dq, dk, dv; ``out``: the kernel's, None for the forward pass alone."""
    u = torch.finfo(q.dtype).eps / 2
    half = q.dtype == torch.float16
    b, nq, hq, d = q.shape
    nk, hk = k.shape[1:3]
    group = hq // hk
    w = max(W, max(nk, nq * group) * 2.0 ** -24)
    val = {n: torch.zeros(t.shape, dtype=torch.float64, device=q.device) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    bnd = {n: torch.zeros_like(t) for n, t in val.items()}
    val["lse"] = torch.full((b, hq, nq), -math.inf, dtype=torch.float64, device=q.device)
    for s in range(b):
        ql, kl = q_lens[s], k_lens[s]
        seen = _mask(nq, nk, ql, kl, causal, q.device)
        clean = [t.double().clone() for t in (q[s], k[s], v[s])]
        clean[0][ql:], clean[1][kl:], clean[2][kl:] = 0, 0, 0
        dos = torch.zeros_like(clean[0]) if do is None else do[s].double().clone()
        dos[ql:] = 0
        top_do = dos.norm(dim=-1).max()
        top_v = clean[2].norm(dim=-1).max()
        tiny_ds = 2.0 ** -37 * top_do * top_v if half else 0.0
        for h in range(hq):
            qs, ks, vs, g = clean[0][:, h], clean[1][:, h // group], clean[2][:, h // group], dos[:, h]
            sc = (qs @ ks.T * scale).masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(sc, -1)
            val["lse"][s, h] = lse
            p = torch.exp(sc - lse.clamp(min=-1e300)[:, None])
            p = torch.where(seen, p, 0.0)
            o = p @ vs
            val["out"][s, :, h] = o
            mag = p @ vs.abs()
            # (the forward pass: P relative to a kept maximum, times 2^7, so that 2^8 more is held)
            bnd["out"][s, :, h] = (u + w) * mag + u * o.abs() + (nk * 2.0 ** -32 if half else 0.0) * vs.abs().amax(0)
            if do is None:
                continue
            given = out[s, :, h].double()
            delta, used = (g * o).sum(-1), (g * given).sum(-1)
            dp = g @ vs.T
            ds = p * (dp - delta[:, None])
            wide = g.abs() @ vs.abs().T + (g.abs() * o.abs()).sum(-1)[:, None]
            e = u * ds.abs() + p * (used - delta).abs()[:, None] + w * p * wide + torch.where(seen, tiny_ds, 0.0)
            val["dq"][s, :, h] = scale * ds @ ks
            bnd["dq"][s, :, h] = scale * (e @ ks.abs() + w * ds.abs() @ ks.abs())
            val["dk"][s, :, h // group] += scale * ds.T @ qs
            bnd["dk"][s, :, h // group] += scale * (e.T @ qs.abs() + w * ds.abs().T @ qs.abs())
            val["dv"][s, :, h // group] += p.T @ g
            bnd["dv"][s, :, h // group] += (u + w) * p.T @ g.abs() + (2.0 ** -40 * g.abs().sum(0) if half else 0.0)
    for n in ("dq", "dk", "dv"):
        bnd[n] += u * (val[n].abs() + bnd[n])
        if half:
            bnd[n] += 2.0 ** -25
    if half:
        bnd["out"] += 2.0 ** -25
    return val, bnd


def _close(name, got, want, bound):
    assert torch.isfinite(got).all(), name
    off = (got.double() - want).abs() - bound
    assert off.max() <= 0, f"{name}: {off.max().item():.3e} beyond its bound at {torch.argmax(off).item()}"


def _inputs(b, nq, nk, hq, hk, d, dtype, seed, packed=False, do_std=0.1):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    if packed:
        both = randn(b, nq, hq + 2 * hk, d)
        q, k, v = both[:, :, :hq], both[:, :, hq : hq + hk], both[:, :, hq + hk :]
    else:
        q, k, v = randn(b, nq, hq, d), randn(b, nk, hk, d), randn(b, nk, hk, d)
    return q * 2 if not packed else q, k, v, randn(b, nq, hq, d, std=do_std)


def _run(q, k, v, do, scale=None, causal=False, q_lens=None, k_lens=None):
    from anemoi_b200.dense import dense_attention, dense_attention_backward

    lens = [None if n is None else torch.tensor(n, dtype=torch.int32, device="cuda") for n in (q_lens, k_lens)]
    kw = dict(scale=scale, causal=causal, query_lengths=lens[0], key_lengths=lens[1])
    out, lse = dense_attention(q, k, v, return_lse=True, **kw)
    grads = dense_attention_backward(do, q, k, v, out, lse, **kw)
    return out, lse, grads


def _check(q, k, v, do, scale=None, causal=False, q_lens=None, k_lens=None):
    b, nq, _, d = q.shape
    out, lse, grads = _run(q, k, v, do, scale, causal, q_lens, k_lens)
    clamp = lambda lens, n: [n] * b if lens is None else [min(max(x, 0), n) for x in lens]
    val, bnd = _reference(q, k, v, do, out, scale or d ** -0.5, causal, clamp(q_lens, nq), clamp(k_lens, k.shape[1]))
    _close("out", out, val["out"], bnd["out"])
    empty = val["lse"] == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert ((lse.double() - val["lse"])[~empty].abs() <= W * (1 + val["lse"][~empty].abs())).all()
    for name, got in zip(("dq", "dk", "dv"), grads):
        _close(name, got, val[name], bnd[name])
    return out, lse, grads


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b, nq, nk, hq, hk", [(1, 128, 128, 1, 1), (1, 256, 384, 2, 2), (2, 300, 200, 3, 1), (1, 1, 1, 2, 2),
                                               (1, 1, 700, 4, 2), (3, 77, 2, 2, 1), (1, 129, 127, 1, 1), (1, 1000, 65, 8, 2),
                                               (2, 513, 641, 2, 2)])
def test_against_the_formula(native_library, dtype, d, b, nq, nk, hq, hk):
    _check(*_inputs(b, nq, nk, hq, hk, d, dtype, seed=nq + nk + d))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float16, 128)])
@pytest.mark.parametrize("nq, nk", [(300, 300), (130, 400), (400, 130), (1, 5), (257, 256), (700, 700)])
def test_causal(native_library, dtype, d, nq, nk):
    """More queries than keys leave the first rows without a key."""
    _check(*_inputs(1, nq, nk, 2, 1, d, dtype, seed=nq), causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 64)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_lens, k_lens", [(None, [300, 0, 1, 128]), ([300, 0, 5, 129], None), ([300, 10, 129, 1], [1, 300, 127, 200]),
                                            ([999, -3, 300, 0], [-1, 999, 0, 300])])
def test_lengths_with_nan_behind_them(native_library, dtype, d, causal, q_lens, k_lens):
    q, k, v, do = _inputs(4, 300, 300, 4, 2, d, dtype, seed=7)
    for s in range(4):
        for lens, tensors in ((q_lens, (q, do)), (k_lens, (k, v))):
            if lens is not None:
                for t, fill in zip(tensors, (float("nan"), float("inf"))):
                    t[s, max(0, min(300, lens[s])):] = fill
    _check(q, k, v, do, causal=causal, q_lens=q_lens, k_lens=k_lens)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_strided_views(native_library, dtype, d):
    """Views of one q|k|v buffer, heads before tokens, and a slice of a wider batch."""
    q, k, v, do = _inputs(2, 333, 333, 4, 2, d, dtype, seed=3, packed=True)
    _check(q, k, v, do)
    q, k, v, do = _inputs(2, 200, 150, 4, 2, d, dtype, seed=4)
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, do)]
    a, b = _run(q, k, v, do), _run(*turned)
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[2], b[2]))


@pytest.mark.gpu
def test_small_gradients_survive_in_fp16(native_library):
    """Gradients of 1e-5 over 4,000 keys: P is about 2^-12 and dS about 2^-29, which fp16 does not have; the results, which it
    has, keep their bits."""
    q, k, v, do = _inputs(1, 200, 4000, 1, 1, 64, torch.float16, seed=5)
    do = torch.full_like(do, 2.0 ** -10) * torch.sign(do)
    _check(q * 0.25, k, v, do)
    out, lse, small = _run(q, k, v, do)
    _, _, large = _run(q, k, v, do * 1024)
    for a, b in zip(small, large):
        far = (a.double() - b.double() / 1024).abs()
        assert (far <= 2.0 ** -10 * a.double().abs() + 2.0 ** -24).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_key_has_no_gradient(native_library, dtype):
    q, k, v, do = _inputs(2, 50, 1, 2, 2, 64, dtype, seed=6)
    out, lse, (dq, dk, dv) = _run(q, k, v, do)
    assert torch.equal(out, v.expand_as(out)) and not dq.any() and not dk.any()
    wide = torch.finfo(dtype).eps * do.double().abs().sum(1, keepdim=True)
    assert ((dv.double() - do.double().sum(1, keepdim=True)).abs() <= wide).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nk", [120, 256, 900])
def test_small_probabilities_survive_in_fp16(native_library, d, nk):
    """One key whose value is zero has nearly all of the probability; what the others give, 2^-20.6 each, is the answer."""
    from anemoi_b200.dense import dense_attention

    gen = torch.Generator(device="cuda").manual_seed(15)
    q, k = torch.zeros(1, 200, 1, d, device="cuda"), torch.zeros(1, nk, 1, d, device="cuda")
    v = torch.rand(1, nk, 1, d, generator=gen, device="cuda") + 1.0
    q[..., 0], k[..., 0], k[:, 5, :, 0], v[:, 5] = 8.0, -10.28125, 4.0, 0.0
    q, k, v = (t.half() for t in (q, k, v))
    p = torch.softmax(0.125 * k[0, :, 0, 0].double() * 8.0, 0)
    want = p @ v[0, :, 0].double()
    u = torch.finfo(torch.float16).eps / 2
    # as above, with P relative to the largest times 2^7: off by 2^-25 below 2^-14, so by 2^-32 each
    bound = (2 * u + W) * want + nk * 2.0 ** -32 * v.max().double() + 2.0 ** -25
    got = dense_attention(q, k, v, scale=0.125)[0, :, 0].double()
    assert ((got - want).abs() <= bound).all()


@pytest.mark.gpu
def test_large_scores(native_library):
    """Scores of thousands, either sign: the running maximum moves far, no exponential overflows."""
    q, k, v, do = _inputs(1, 260, 700, 2, 2, 64, torch.bfloat16, seed=8)
    from anemoi_b200.dense import dense_attention

    out, lse = dense_attention(q * 64, k * 16, v, return_lse=True)
    sc = torch.einsum("bqhd,bkhd->bhqk", (q * 64).double(), (k * 16).double()) / 8
    want = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(sc, -1), v.double())
    # fp32 scores of 2^14: 2^-8 absolute, so probabilities to 1 %
    assert ((out.double() - want).abs() <= 0.02 + 0.02 * want.abs()).float().mean() > 0.99
    assert torch.isfinite(out).all() and ((lse.double() - torch.logsumexp(sc, -1)).abs() <= 0.05).all()


@pytest.mark.gpu
def test_equal_calls_give_equal_bits_and_splits_agree(native_library):
    q, k, v, do = _inputs(1, 260, 3000, 2, 1, 128, torch.bfloat16, seed=9)
    a, b = _run(q, k, v, do), _run(q, k, v, do)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(x, y) for x, y in zip(a[2], b[2]))
    _check(q, k, v, do)


@pytest.mark.gpu
def test_autograd_and_differences(native_library):
    from anemoi_b200.dense import dense_attention

    q, k, v, do = _inputs(2, 70, 90, 4, 2, 64, torch.bfloat16, seed=10)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = dense_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, do)
    _, _, want = _run(q, k, v, do)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    # an expanded gradient, as a sum's is
    total = torch.autograd.grad(dense_attention(*leaves).sum(), leaves)
    _, _, ones = _run(q, k, v, torch.ones_like(do))
    assert all(torch.equal(a, b) for a, b in zip(total, ones))
    # along a direction, against central differences of the formula in 64 bits
    gen = torch.Generator(device="cuda").manual_seed(1)

    def value(ts):
        kk, vv = (t.repeat_interleave(2, dim=2) for t in ts[1:])
        p = torch.softmax(torch.einsum("bqhd,bkhd->bhqk", ts[0], kk) / 8, -1)
        return (torch.einsum("bhqk,bkhd->bqhd", p, vv) * do.double()).sum()

    at = [t.double() for t in (q, k, v)]
    for which in range(3):
        step = torch.randn(at[which].shape, generator=gen, device="cuda", dtype=torch.float64)
        moved = [[t + sign * 1e-4 * step if i == which else t for i, t in enumerate(at)] for sign in (1, -1)]
        slope = (value(moved[0]) - value(moved[1])) / 2e-4
        along = (grads[which].double() * step).sum()
        # a random sum of rounded values: off by sqrt(n) half steps of a typical one, five times that
        size = grads[which].double().norm() * 2.0 ** -8 * 5
        assert (along - slope).abs() <= size + 1e-6


@pytest.mark.gpu
def test_captured_on_another_stream(native_library):
    q, k, v, do = _inputs(1, 300, 300, 2, 2, 64, torch.float16, seed=11)
    want = _run(q, k, v, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(q, k, v, do)
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for _ in range(2):  # two graphs of the same call, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(_run(q, k, v, do))
        graphs.append(graph)
    q2 = torch.randn_like(q)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for got in results:
        assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[2], want[2]))
    q.copy_(q2)
    want = _run(q, k, v, do)
    for graph, got in zip(graphs, results):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[2], want[2]))


@pytest.mark.gpu
def test_the_first_call_is_not_captured(native_library):
    """The status word that a graph would allocate is zero only once that graph has run."""
    from anemoi_b200 import executor
    from anemoi_b200.dense import dense_attention

    q, k, v, do = _inputs(1, 40, 40, 1, 1, 64, torch.float16, seed=13)
    _run(q, k, v, do)
    word = executor._STATUS.pop(q.device)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="before a capture"):
                dense_attention(q, k, v)
    finally:
        executor._STATUS[q.device] = word
    assert executor.last_status(q.device) == 0


@pytest.mark.gpu
def test_two_streams_at_once(native_library):
    """Calls of two streams run beside each other with workspaces of their own."""
    a, b = _inputs(1, 300, 2000, 2, 2, 64, torch.float16, seed=14), _inputs(2, 500, 100, 4, 2, 128, torch.bfloat16, seed=15)
    want = [_run(*t) for t in (a, b)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(5):
        for i, t in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i] = _run(*t)
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) and all(torch.equal(m, n) for m, n in zip(x[2], y[2]))


@pytest.mark.gpu
@pytest.mark.parametrize("nq, nk, hq, hk", [(40, 5000, 4, 4), (5000, 40, 8, 2), (300, 9000, 2, 1), (2000, 1000, 12, 12)])
def test_split_walks(native_library, nq, nk, hq, hk):
    """Few CTAs with long walks: parts of keys and of queries that are joined; some tiles whole beside tiles in parts."""
    _check(*_inputs(1, nq, nk, hq, hk, 64, torch.bfloat16, seed=nq, do_std=0.05))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nk", [1, 100, 300, 700])
@pytest.mark.parametrize("q_lens, k_lens", [(None, None), ([4200, 130, 0, 2001], None), ([4000, 4200, 128, 1], [0, 1, 130, 700])])
def test_short_walks_of_many_queries(native_library, dtype, d, causal, nk, q_lens, k_lens):
    """Enough query tiles that a CTA takes several, some without keys: at the start, between others or at the end."""
    q, k, v, do = _inputs(4, 4200, nk, 16, 4, d, dtype, 12)
    if q_lens is not None:
        for t, lens in ((q, q_lens), (do, q_lens), (k, k_lens), (v, k_lens)):
            for s in range(4 if lens is not None else 0):
                t[s, lens[s] :] = math.nan
    _check(q, k, v, do, causal=causal, q_lens=q_lens, k_lens=k_lens)


@pytest.mark.gpu
def test_empty_sides(native_library):
    q, k, v, do = _inputs(2, 5, 3, 2, 1, 64, torch.bfloat16, seed=12)
    out, lse, grads = _run(q, k[:, :0], v[:, :0], do)
    assert not out.any() and (lse == -math.inf).all() and not grads[0].any() and grads[1].shape == (2, 0, 1, 64)
    out, lse, grads = _run(q[:, :0], k, v, do[:, :0])
    assert out.shape == (2, 0, 2, 64) and not grads[1].any() and not grads[2].any()


@pytest.mark.gpu
def test_a_scale_that_changes_in_place(native_library):
    """Calls are told apart by the value of the scale, not by the object."""
    from anemoi_b200.dense import dense_attention

    q, k, v, _ = _inputs(1, 200, 300, 2, 2, 64, torch.float16, 14)
    scale = torch.tensor(0.1)
    for value in (0.125, 0.5):
        scale.fill_(value)
        assert torch.equal(dense_attention(q, k, v, scale=scale), dense_attention(q, k, v, scale=value))


def test_refusals():
    """What the call refuses before it looks for a GPU, and the library before it launches anything."""
    from anemoi_b200.dense import dense_attention

    t = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        dense_attention(t, t, t)


def test_the_library_refuses(native_library):
    import ctypes as C

    from anemoi_b200 import native

    good = dict(batch=1, q_heads=4, k_heads=2, q_tokens=8, k_tokens=8, head_dim=64, causal=0, is_bf16=1, scale=0.125)
    assert native_library.anemoi_sm100_dense_attention_backward_workspace(C.byref(native.DenseShape(**good)), 0) > 0
    for change in (dict(batch=0), dict(k_heads=3), dict(k_heads=0), dict(head_dim=96), dict(scale=0.0), dict(scale=-1.0),
                   dict(scale=float("nan")), dict(scale=float("inf")), dict(q_tokens=0), dict(k_tokens=-1)):
        shape = native.DenseShape(**{**good, **change})
        assert native_library.anemoi_sm100_dense_attention_workspace(C.byref(shape)) == -1, change
    for change in (dict(batch=5000), dict(q_tokens=1 << 30), dict(batch=4000, q_tokens=1 << 18)):
        shape = native.DenseShape(**{**good, **change})
        assert native_library.anemoi_sm100_dense_attention_workspace(C.byref(shape)) == -3, change
    shape, strides = native.DenseShape(**good), (C.c_int64 * 12)(*([2048, 256, 64] * 4))
    one, odd = C.c_void_p(1 << 20), C.c_void_p((1 << 20) + 2)

    def call(q=one, lse=None, steps=strides, status=one):
        return native_library.anemoi_sm100_dense_attention(C.byref(shape), q, one, one, None, None, steps, one, lse, None, 0,
                                                           status, None)

    assert call(q=None) == -1 and call(q=odd) == -1 and call(status=None) == -1
    for at, value in ((0, 0), (1, -256), (1, 4), (2, 65)):
        wrong = (C.c_int64 * 12)(*strides)
        wrong[at] = value
        if at == 0:
            continue  # one sample: its stride does not matter
        assert call(steps=wrong) == -1
