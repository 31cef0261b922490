"""The operators around and of a video block's attention, in the forms that training and serving call.

Three operators, each with its gradient.  ``fused_qknorm_axial_rope``: RMS norm per head, then rotary positions with
several axes (time, height, width).  ``fused_gate_norm_modulate``: the gated residual after a block, fused with the
norm and modulation before the next one.  ``dense_attention``: softmax attention whose backward pass recomputes the
probabilities.  Widths and heads are those of the block stack (width 5,376, 56 heads of 128 channels), token counts
those of its video layouts (21 x 30 x 52 video tokens behind 512 of text, and smaller ones); the other sizes are
generic.

A case names its ``path``; ``plain`` forms work in 32 bits (angles in 64) and round once at the end.
"""

from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6
_VIDEO = 21 * 30 * 52 + 512          # tokens of the 832x480 layout
_MOST_SCORES = _VIDEO ** 2 * 7 * 128  # dot products of the largest listed attention
_MOST_ROPE = _VIDEO * 112 * 128       # values that the largest listed rotary call turns
_MOST_NORM = _VIDEO * 5376            # values of the largest listed residual stream


def _rope(name, path, batch, tokens, q_heads, k_heads, dim, sections, dtype, *, interleaved=False, shared=False,
          normed=True, theta=10000.0, packed=False, spread=1):
    case = dict(path=path, batch=batch, tokens=tokens, q_heads=q_heads, k_heads=k_heads, dim=dim, sections=sections,
                dtype=dtype, interleaved=interleaved, shared=shared, normed=normed, theta=theta, packed=packed,
                spread=spread)
    return dict(case, name=name) if name else case


def _norm(name, path, batch, groups, rows, width, dtype, mod, *, norm="rms", post="", weighted=False):
    """``groups`` modulation rows per sample, ``rows`` tokens that share one."""
    case = dict(path=path, batch=batch, groups=groups, rows=rows, width=width, dtype=dtype, mod=mod, norm=norm,
                post=post, weighted=weighted)
    return dict(case, name=name) if name else case


def _attn(name, path, batch, q_tokens, k_tokens, q_heads, k_heads, dim, dtype, *, causal=False, q_cut=0, k_cut=0,
          packed=False):
    """Sample b has ``q_tokens - b * q_cut`` queries and ``k_tokens - b * k_cut`` keys (none below zero); without cuts
    no lengths are given."""
    case = dict(path=path, batch=batch, q_tokens=q_tokens, k_tokens=k_tokens, q_heads=q_heads, k_heads=k_heads, dim=dim,
                dtype=dtype, causal=causal, q_cut=q_cut, k_cut=k_cut, packed=packed)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one token of a streaming request through the norm between two blocks: latency only
        _norm("norm_token", "norm", 1, 1, 1, 5376, "bf16", "bf16"),
        # the residual stream of the 832x480 layer between attention and feed-forward, one modulation for all tokens
        _norm("norm_layer", "norm", 1, 1, _VIDEO, 5376, "bf16", "bf16"),
        # training with a noise level per frame: ragged frames, layer norm, weights, a norm behind the block, fp32 modulation
        _norm("norm_grad_frames", "norm_grad", 2, 13, 27 * 45, 1160, "fp16", "fp32", norm="layer", post="rms",
              weighted=True),
        # the gradient at the benchmark stack's size
        _norm("norm_grad_layer", "norm_grad", 1, 1, _VIDEO, 5376, "bf16", "bf16"),
        # queries and keys of one new token
        _rope("rope_token", "rope", 1, 1, 56, 56, 128, "8,12,12", "bf16"),
        # queries and keys of the 832x480 layer, views of one fused projection
        _rope("rope_layer", "rope", 1, _VIDEO, 56, 56, 128, "8,12,12", "bf16", packed=True),
        # gradient with shared key heads, small heads turned over their whole width, neighbours paired
        _rope("rope_grad", "rope_grad", 2, 13 * 27 * 45 + 333, 24, 8, 64, "8,12,12", "fp16", interleaved=True),
        # a preview-sized training step's backward call: latency counts
        _attn("attn_grad_preview", "attn_grad", 1, 1024, 1024, 4, 4, 64, "fp16"),
        # video queries on text keys of two prompts, the second one padded: long loops for few keys
        _attn("attn_grad_text", "attn_grad", 2, 7800, 512, 16, 16, 128, "bf16", k_cut=179),
        # forward and backward as training calls them: causal, shared key heads, ragged samples, odd lengths
        _attn("attn_train_causal", "attn_train", 2, 4111, 4111, 16, 4, 128, "bf16", causal=True, q_cut=1000, k_cut=1000),
        # the dense-first layers' attention, small heads, odd length
        _attn("attn_video", "attn", 1, 13 * 27 * 45 + 333, 13 * 27 * 45 + 333, 12, 12, 64, "fp16"),
        # one rank's share (7 of 56 heads) of the 832x480 layer, gradients, on the strided views of its q|k|v buffer
        _attn("attn_grad_video", "attn_grad", 1, _VIDEO, _VIDEO, 7, 7, 128, "bf16", packed=True),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    family = rng.choice(("norm", "norm_grad", "rope", "rope_grad", "attn", "attn_grad", "attn_grad", "attn_train"))
    dtype = rng.choice(("bf16", "fp16"))
    if family.startswith("norm"):
        width = 8 * _log(rng, 8, 1024)
        batch, groups = rng.choice((1, 1, 2, 3)), _log(rng, 1, 40)
        rows = _log(rng, 1, max(1, _MOST_NORM // (width * batch * groups)))
        return _norm(None, family, batch, groups, rows, width, dtype, rng.choice((dtype, "fp32")),
                     norm=rng.choice(("rms", "layer")), post=rng.choice(("", "rms", "layer")),
                     weighted=rng.random() < 0.5)
    if family.startswith("rope"):
        dim = rng.choice((64, 128))
        interleaved = rng.random() < 0.5
        pairs = 8 * rng.randint(1, dim // 16)
        first = rng.randint(0, pairs)
        second = rng.randint(0, pairs - first)
        k_heads = _log(rng, 1, 28)
        q_heads = k_heads * rng.randint(1, 56 // k_heads if k_heads > 7 else 8)
        batch = rng.choice((1, 1, 2, 3))
        tokens = _log(rng, 1, min(100_000, _MOST_ROPE // (batch * (q_heads + k_heads) * dim)))
        return _rope(None, family, batch, tokens, q_heads, k_heads, dim, f"{first},{second},{pairs - first - second}",
                     dtype, interleaved=interleaved, shared=rng.random() < 0.3, normed=rng.random() < 0.8,
                     theta=rng.choice((256.0, 10000.0, 1e6)), packed=rng.random() < 0.5,
                     spread=rng.choice((1, 1, 1000)))
    dim = rng.choice((64, 128))
    k_heads = _log(rng, 1, 24)
    q_heads = k_heads * rng.choice((1, 1, 1, 2, 4))
    batch = rng.choice((1, 1, 2, 3))
    room = _MOST_SCORES / (batch * q_heads * dim) / 2
    q_tokens = _log(rng, 1, 20_000)
    k_tokens = _log(rng, 1, max(1, min(20_000, int(room / q_tokens))))
    causal = rng.random() < 0.3
    if causal or rng.random() < 0.5:
        q_tokens = k_tokens = max(1, min(_log(rng, 1, 20_000), int(room ** 0.5)))
    return _attn(None, family, batch, q_tokens, k_tokens, q_heads, k_heads, dim, dtype, causal=causal,
                 q_cut=rng.choice((0, 0, q_tokens // 3)), k_cut=rng.choice((0, 0, k_tokens // 2, k_tokens)),
                 packed=rng.random() < 0.3)


# ---- shapes ----
def _lengths(case):
    return ([max(0, case["q_tokens"] - b * case["q_cut"]) for b in range(case["batch"])],
            [max(0, case["k_tokens"] - b * case["k_cut"]) for b in range(case["batch"])])


def _scores(case):
    """Query-key pairs that the mask leaves, of one head over all samples."""
    total = 0
    for nq, nk in zip(*_lengths(case)):
        if not case["causal"]:
            total += nq * nk
        else:
            # query i sees keys 0 .. i + nk - nq
            first = max(0, nq - nk)
            total += (nq - first) * (2 * nk - (nq - first) + 1) // 2
    return total


def work(case):
    size = 4 if case.get("dtype") == "fp32" else 2
    if case["path"] in ("norm", "norm_grad"):
        rows = case["batch"] * case["groups"] * case["rows"]
        values = rows * case["width"]
        per = 4 if case["mod"] == "fp32" else 2
        mods = case["batch"] * case["groups"] * case["width"]
        weights = (2 if case["post"] else 1) * case["width"] * size if case["weighted"] else 0
        if case["path"] == "norm":
            return {"bytes": 4 * values * size + 3 * mods * per + weights, "flops": 10 * values}
        return {"bytes": 6 * values * size + 5 * mods * per + 2 * weights, "flops": 24 * values}
    if case["path"] in ("rope", "rope_grad"):
        tokens = case["batch"] * case["tokens"]
        values = tokens * (case["q_heads"] + case["k_heads"]) * case["dim"]
        around = tokens * 3 * 4 + (2 * case["dim"] * size if case["normed"] else 0)
        # without a norm the gradient needs no inputs: the rotation turned back
        passes = 2 if case["path"] == "rope" or not case["normed"] else 3
        return {"bytes": passes * values * size + around, "flops": (8 if passes == 2 else 16) * values}
    dim, nq, nk = case["dim"], sum(_lengths(case)[0]), sum(_lengths(case)[1])
    q_bytes, k_bytes = nq * case["q_heads"] * dim * size, nk * case["k_heads"] * dim * size
    product = 2 * _scores(case) * case["q_heads"] * dim
    lse = 4 * nq * case["q_heads"]
    forward = {"bytes": 2 * q_bytes + 2 * k_bytes + (lse if case["path"] == "attn" else 0), "flops": 2 * product}
    # q, k, v, out, their gradients, the rows' statistics
    backward = {"bytes": 4 * q_bytes + 4 * k_bytes + lse, "flops": 5 * product}
    if case["path"] == "attn":
        return forward
    if case["path"] == "attn_grad":
        return backward
    return {"bytes": forward["bytes"] + backward["bytes"], "flops": forward["flops"] + backward["flops"]}


# ---- inputs ----
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    gen = _generator(seed)

    def randn(*shape, std=1.0, dtype=None):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype or _TYPES[case["dtype"]])

    state = dict(case=case)
    if case["path"] in ("norm", "norm_grad"):
        tokens, width = case["groups"] * case["rows"], case["width"]
        # the residual stream: a few channels far above the others, as trained blocks have them
        channel = torch.ones(width, device="cuda")
        channel[:: max(1, width // 6)] = 12.0
        x = (torch.randn(case["batch"], tokens, width, generator=gen, device="cuda") * 2.0 * channel).to(_TYPES[case["dtype"]])
        state.update(x=x, y=randn(case["batch"], tokens, width))
        for key, mean, std in (("gate", 0.2, 0.3), ("scale", 0.0, 0.2), ("shift", 0.0, 0.2)):
            value = mean + torch.randn(case["batch"], case["groups"], width, generator=gen, device="cuda") * std
            state[key] = value.to(_TYPES[case["mod"]])
        state["weight"] = (1 + 0.1 * torch.randn(width, generator=gen, device="cuda")).to(x.dtype) if case["weighted"] else None
        state["post_weight"] = ((1 + 0.1 * torch.randn(width, generator=gen, device="cuda")).to(x.dtype)
                                if case["weighted"] and case["post"] else None)
        if case["path"] == "norm_grad":
            state.update(d_x=randn(*x.shape, std=0.1), d_h=randn(*x.shape, std=0.1))
        return state
    if case["path"] in ("rope", "rope_grad"):
        b, t, hq, hk, d = (case[key] for key in ("batch", "tokens", "q_heads", "k_heads", "dim"))

        def pair(std):
            if case["packed"]:
                both = randn(b, t, hq + hk, d, std=std)
                return both[:, :, :hq], both[:, :, hq:]
            return randn(b, t, hq, d, std=std), randn(b, t, hk, d, std=std)

        state["q"], state["k"] = pair(1.5)
        if case["path"] == "rope_grad":
            state["d_q"], state["d_k"] = pair(0.1)
        for key in ("q_weight", "k_weight"):
            state[key] = (1 + 0.1 * torch.randn(d, generator=gen, device="cuda")).to(state["q"].dtype) if case["normed"] else None
        # a prefix at the origin's place in time, then frames of a grid; far positions with `spread`
        index = torch.arange(t, device="cuda")
        side = max(1, int(t ** (1 / 3)))
        grid = torch.stack((index // (side * side), index // side % side, index % side), dim=-1)
        offset = torch.randint(0, 32, (b, 1, 3), generator=gen, device="cuda")
        state["positions"] = ((grid + offset) * case["spread"]).to(torch.int32)
        if own:
            from anemoi_b200.producer import AxialRotary

            state["rotary"] = AxialRotary(_sections(case), theta=case["theta"], interleaved=case["interleaved"],
                                          shared_frequencies=case["shared"])
        return state
    b, nq, nk, hq, hk, d = (case[key] for key in ("batch", "q_tokens", "k_tokens", "q_heads", "k_heads", "dim"))
    if case["packed"] and nq == nk:
        packed = randn(b, nq, hq + 2 * hk, d, std=1.0)
        q, k, v = packed[:, :, :hq], packed[:, :, hq : hq + hk], packed[:, :, hq + hk :]
    else:
        q, k, v = randn(b, nq, hq, d), randn(b, nk, hk, d), randn(b, nk, hk, d)
    # scores with a spread of two, so that some keys of a row stand out
    q *= 2.0
    state.update(q=q, k=k, v=v, q_lengths=None, k_lengths=None)
    q_list, k_list = _lengths(case)
    if case["q_cut"]:
        state["q_lengths"] = torch.tensor(q_list, dtype=torch.int32, device="cuda")
    if case["k_cut"]:
        state["k_lengths"] = torch.tensor(k_list, dtype=torch.int32, device="cuda")
    if case["path"] != "attn":
        state["d_out"] = randn(b, nq, hq, d, std=0.05)
    if case["path"] == "attn_grad":
        state["out"], state["lse"] = _attention(state, case, torch.float32)
        state["out"] = state["out"].to(q.dtype)
        state["lse"] = state["lse"].float()
    if case["path"] == "attn_train" and own:
        for key in ("q", "k", "v"):
            state[key] = state[key].detach().requires_grad_()
    return state


# ---- plain forms ----
def _sections(case):
    return tuple(int(n) for n in case["sections"].split(","))


def _rms(x, kind):
    """The normalised rows and the factor that made them."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    return x * r, r


def _rms_grad(d_hat, hat, r, kind):
    g = d_hat - hat * (d_hat * hat).mean(-1, keepdim=True)
    if kind == "layer":
        g = g - d_hat.mean(-1, keepdim=True)
    return g * r


def _grouped(state, case):
    """Tensors with the tokens that share a modulation row in an axis of their own, in 32 bits."""
    shape = (case["batch"], case["groups"], case["rows"], case["width"])
    return {key: state[key].float().view(shape) for key in ("x", "y", "d_x", "d_h") if key in state}


def _norm_plain(state, case):
    t = _grouped(state, case)
    gate, scale, shift = (state[key].float().unsqueeze(2) for key in ("gate", "scale", "shift"))
    y = t["y"]
    if case["post"]:
        y = _rms(y, case["post"])[0]
        if case["weighted"]:
            y = y * state["post_weight"].float()
    x = t["x"] + gate * y
    h = _rms(x, case["norm"])[0]
    if case["weighted"]:
        h = h * state["weight"].float()
    h = h * (1 + scale) + shift
    shape = state["x"].shape
    return x.to(state["x"].dtype).view(shape), h.to(state["x"].dtype).view(shape)


def _norm_grad_plain(state, case):
    """``x`` is the stream behind the residual here: its rows are normalised as they are."""
    t = _grouped(state, case)
    kind = state["x"].dtype
    gate, scale = state["gate"].float().unsqueeze(2), state["scale"].float().unsqueeze(2)
    weight = state["weight"].float() if case["weighted"] else None
    hat, r = _rms(t["x"], case["norm"])
    normed = hat if weight is None else hat * weight
    d_normed = t["d_h"] * (1 + scale)
    d_hat = d_normed if weight is None else d_normed * weight
    d_x = t["d_x"] + _rms_grad(d_hat, hat, r, case["norm"])
    d_scale, d_shift = (t["d_h"] * normed).sum(2), t["d_h"].sum(2)
    d_weight = None if weight is None else (d_normed * hat).sum((0, 1, 2)).to(kind)
    d_y, d_post, post = gate * d_x, None, t["y"]
    if case["post"]:
        y_hat, y_r = _rms(t["y"], case["post"])
        post = y_hat
        if case["weighted"]:
            pw = state["post_weight"].float()
            d_post = (d_y * y_hat).sum((0, 1, 2)).to(kind)
            post, d_y = y_hat * pw, d_y * pw
        d_y = _rms_grad(d_y, y_hat, y_r, case["post"])
    d_gate = (d_x * post).sum(2)
    shape, mod = state["x"].shape, state["gate"].dtype
    out = [d_x.to(kind).view(shape), d_y.to(kind).view(shape), d_gate.to(mod), d_scale.to(mod), d_shift.to(mod)]
    return out + [g for g in (d_weight, d_post) if g is not None]


def _angles(state, case):
    """cos and sin of every pair of channels, ``[B, T, 1, pairs]``, from angles in 64 bits."""
    sections = _sections(case)
    pairs = sum(sections)
    columns, first = [], 0
    for axis, count in enumerate(sections):
        index = torch.arange(count, device="cuda", dtype=torch.float64)
        power = (index + first) / pairs if case["shared"] else index / max(count, 1)
        columns.append(state["positions"][..., axis : axis + 1].double() * case["theta"] ** -power)
        first += count
    angle = torch.cat(columns, -1).unsqueeze(-2)
    return torch.cos(angle), torch.sin(angle)


def _turn(x, cos, sin, interleaved):
    pairs = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0 : 2 * pairs : 2], x[..., 1 : 2 * pairs : 2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :pairs], x[..., pairs : 2 * pairs]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., 2 * pairs :]), dim=-1)


def _rope_plain(state, case):
    cos, sin = (t.float() for t in _angles(state, case))
    out = []
    for key in ("q", "k"):
        x = state[key].float()
        if case["normed"]:
            x = _rms(x, "rms")[0] * state[key + "_weight"].float()
        out.append(_turn(x, cos, sin, case["interleaved"]).to(state[key].dtype))
    return out


def _rope_grad_plain(state, case):
    cos, sin = (t.float() for t in _angles(state, case))
    grads, weights = [], []
    for key in ("q", "k"):
        g = _turn(state["d_" + key].float(), cos, -sin, case["interleaved"])
        if case["normed"]:
            hat, r = _rms(state[key].float(), "rms")
            weights.append((g * hat).sum((0, 1, 2)).to(state[key].dtype))
            g = _rms_grad(g * state[key + "_weight"].float(), hat, r, "rms")
        grads.append(g.to(state[key].dtype))
    return grads + weights


def _chunks(state, case, kind):
    """Sample, head, rows of queries and what they attend to: ``(b, h, slice, q, keys, k, v, mask)``."""
    group = case["q_heads"] // case["k_heads"]
    for b, (nq, nk) in enumerate(zip(*_lengths(case))):
        step = max(1, min(nq, (1 << 28) // max(nk, 1)))
        for h in range(case["q_heads"]):
            k, v = state["k"][b, :nk, h // group].to(kind), state["v"][b, :nk, h // group].to(kind)
            for begin in range(0, nq, step):
                rows = slice(begin, min(nq, begin + step))
                mask = None
                if case["causal"]:
                    i = torch.arange(rows.start, rows.stop, device="cuda")[:, None] + (nk - nq)
                    mask = torch.arange(nk, device="cuda")[None, :] > i
                yield b, h, rows, state["q"][b, rows, h].to(kind), k, v, mask


def _probabilities(q, k, mask):
    """Softmax rows (zeros where no key is left) and their log-sum-exps."""
    if k.shape[0] == 0:
        return q.new_zeros(q.shape[0], 0), q.new_full((q.shape[0],), -math.inf)
    s = (q @ k.T) * q.shape[-1] ** -0.5
    if mask is not None:
        s.masked_fill_(mask, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total > 0, m + torch.log(total), -math.inf)
    return p / torch.where(total > 0, total, 1.0), lse.squeeze(-1)


def _attention(state, case, kind):
    q = state["q"]
    out = torch.zeros(q.shape, dtype=kind, device="cuda")
    lse = torch.full((case["batch"], case["q_heads"], case["q_tokens"]), -math.inf, dtype=kind, device="cuda")
    for b, h, rows, qc, k, v, mask in _chunks(state, case, kind):
        p, row_lse = _probabilities(qc, k, mask)
        out[b, rows, h] = p @ v
        lse[b, h, rows] = row_lse
    return out, lse


def _attention_grad(state, case, kind):
    dq, dk, dv = (torch.zeros(state[key].shape, dtype=kind, device="cuda") for key in ("q", "k", "v"))
    group, scale = case["q_heads"] // case["k_heads"], case["dim"] ** -0.5
    for b, h, rows, qc, k, v, mask in _chunks(state, case, kind):
        if k.shape[0] == 0:
            continue
        p, _ = _probabilities(qc, k, mask)
        do = state["d_out"][b, rows, h].to(kind)
        dp = do @ v.T
        ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
        dq[b, rows, h] = ds @ k
        dk[b, : k.shape[0], h // group] += ds.T @ qc
        dv[b, : k.shape[0], h // group] += p.T @ do
    return dq, dk, dv


def _attention_plain(state, case):
    kind = state["q"].dtype
    if case["path"] == "attn":
        out, lse = _attention(state, case, torch.float32)
        return [out.to(kind), lse]
    grads = [t.to(kind) for t in _attention_grad(state, case, torch.float32)]
    if case["path"] == "attn_grad":
        return grads
    return [_attention(state, case, torch.float32)[0].to(kind)] + grads


_PLAIN = {"norm": _norm_plain, "norm_grad": _norm_grad_plain, "rope": _rope_plain, "rope_grad": _rope_grad_plain,
          "attn": _attention_plain, "attn_grad": _attention_plain, "attn_train": _attention_plain}


# ---- the framework's calls ----
def _own(state, case):
    path = case["path"]
    if path in ("norm", "norm_grad"):
        from anemoi_b200.modulation import fused_gate_norm_modulate, fused_gate_norm_modulate_backward

        options = dict(eps=_EPS, norm=case["norm"], post_norm=case["post"] or None)
        if path == "norm":
            return list(fused_gate_norm_modulate(state["x"], state["y"], state["gate"], state["scale"], state["shift"],
                                                 state["weight"], state["post_weight"], **options))
        grads = fused_gate_norm_modulate_backward(state["d_x"], state["d_h"], state["x"], state["y"], state["gate"],
                                                  state["scale"], state["weight"], state["post_weight"], **options)
        return [g for g in (grads.x, grads.y, grads.gate, grads.scale, grads.shift, grads.weight, grads.post_weight)
                if g is not None]
    if path in ("rope", "rope_grad"):
        from anemoi_b200.producer import fused_qknorm_axial_rope, fused_qknorm_axial_rope_backward

        if path == "rope":
            return list(fused_qknorm_axial_rope(state["q"], state["k"], state["q_weight"], state["k_weight"],
                                                state["positions"], state["rotary"], _EPS))
        grads = fused_qknorm_axial_rope_backward(state["d_q"], state["d_k"], state["q"], state["k"], state["q_weight"],
                                                 state["k_weight"], state["positions"], state["rotary"], _EPS)
        return [g for g in grads if g is not None]
    from anemoi_b200.dense import dense_attention, dense_attention_backward

    options = dict(causal=case["causal"], query_lengths=state["q_lengths"], key_lengths=state["k_lengths"])
    q, k, v = state["q"], state["k"], state["v"]
    if path == "attn":
        return list(dense_attention(q, k, v, return_lse=True, **options))
    if path == "attn_grad":
        return list(dense_attention_backward(state["d_out"], q, k, v, state["out"], state["lse"], **options))
    out = dense_attention(q, k, v, **options)
    return [out.detach()] + list(torch.autograd.grad(out, (q, k, v), state["d_out"]))


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    with torch.no_grad():
        return _PLAIN[case["path"]](state, case)


# ---- in 64 bits, from the definitions ----
def _exact_norm(state, case):
    """The gradients come from differentiating the definition: autograd's rules for sums, products and roots."""
    with_grad = case["path"] == "norm_grad"
    leaves = {}
    for key in ("x", "y", "gate", "scale", "shift", "weight", "post_weight"):
        if state[key] is not None:
            leaves[key] = state[key].double().requires_grad_(with_grad)
    per_row = {key: leaves[key].repeat_interleave(case["rows"], dim=1) for key in ("gate", "scale", "shift")}

    def normalised(t, kind):
        centred = t - t.sum(-1, keepdim=True) / case["width"] if kind == "layer" else t
        return centred / ((centred ** 2).sum(-1, keepdim=True) / case["width"] + _EPS).sqrt()

    y = leaves["y"]
    if case["post"]:
        y = normalised(y, case["post"]) * leaves.get("post_weight", 1.0)
    # the gradient's stream is the one behind the residual: x = before + gate * y
    stream = leaves["x"] + per_row["gate"] * (y - y.detach()) + (per_row["gate"] - per_row["gate"].detach()) * y.detach() \
        if with_grad else leaves["x"] + per_row["gate"] * y
    h = normalised(stream, case["norm"]) * leaves.get("weight", 1.0) * (1 + per_row["scale"]) + per_row["shift"]
    if not with_grad:
        return [stream, h]
    wanted = [key for key in ("x", "y", "gate", "scale", "shift", "weight", "post_weight") if key in leaves]
    total = (stream * state["d_x"].double()).sum() + (h * state["d_h"].double()).sum()
    return list(torch.autograd.grad(total, [leaves[key] for key in wanted]))


def _exact_rope(state, case):
    sections, (b, t) = _sections(case), state["positions"].shape[:2]
    pairs = sum(sections)
    turn = torch.ones(b, t, pairs, dtype=torch.complex128, device="cuda")
    for pair in range(pairs):
        axis = 0 if pair < sections[0] else 1 if pair < sections[0] + sections[1] else 2
        local, count = pair - sum(sections[:axis]), sections[axis]
        rate = math.exp(-math.log(case["theta"]) * (pair / pairs if case["shared"] else local / count))
        angle = state["positions"][..., axis].double() * rate
        turn[..., pair] = torch.polar(torch.ones_like(angle), angle)
    turn = turn.unsqueeze(2)
    results, weights = [], []
    for key in ("q", "k"):
        grad = case["path"] == "rope_grad"
        x = state[key].double().requires_grad_(grad)
        w = state[key + "_weight"].double().requires_grad_(grad) if case["normed"] else None
        n = x if w is None else x / ((x ** 2).mean(-1, keepdim=True) + _EPS).sqrt() * w
        span = n[..., : 2 * pairs]
        if case["interleaved"]:
            z = torch.view_as_complex(span.unflatten(-1, (pairs, 2)).contiguous()) * turn
            turned = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(span[..., :pairs], span[..., pairs:]) * turn
            turned = torch.cat((z.real, z.imag), -1)
        out = torch.cat((turned, n[..., 2 * pairs :]), -1)
        if not grad:
            results.append(out)
            continue
        got = torch.autograd.grad((out * state["d_" + key].double()).sum(), [x] if w is None else [x, w])
        results.append(got[0])
        weights += got[1:]
    return results + weights


def _exact_attention(state, case):
    """Head by head: probabilities, then the products of the chain rule, all rows of a block of queries at once."""
    q, k, v = (state[key] for key in ("q", "k", "v"))
    group, scale = case["q_heads"] // case["k_heads"], 1.0 / math.sqrt(case["dim"])
    grad, forward = case["path"] != "attn", case["path"] != "attn_grad"
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full((case["batch"], case["q_heads"], case["q_tokens"]), -math.inf, dtype=torch.float64, device="cuda")
    d_q, d_k, d_v = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (q, k, v))
    for b, (nq, nk) in enumerate(zip(*_lengths(case))):
        for h in range(case["q_heads"] if nk else 0):
            keys, values = k[b, :nk, h // group].double(), v[b, :nk, h // group].double()
            for begin in range(0, nq, 2048):
                rows = torch.arange(begin, min(nq, begin + 2048), device="cuda")
                queries = q[b, rows, h].double()
                scores = torch.mm(queries, keys.t()).mul_(scale)
                if case["causal"]:
                    hidden = torch.arange(nk, device="cuda") - nk > (rows - nq).unsqueeze(1)
                    scores[hidden] = -math.inf
                weight = torch.logsumexp(scores, dim=1)
                lse[b, h, rows] = weight
                scores.sub_(weight.clamp(min=-1e300).unsqueeze(1)).exp_()
                if forward:
                    out[b, rows, h] = torch.mm(scores, values)
                if grad:
                    given = state["d_out"][b, rows, h].double()
                    d_v[b, :nk, h // group] += torch.mm(scores.t(), given)
                    d_scores = torch.mm(given, values.t())
                    d_scores.sub_(torch.linalg.vecdot(scores, d_scores).unsqueeze(1)).mul_(scores).mul_(scale)
                    d_q[b, rows, h] = torch.mm(d_scores, keys)
                    d_k[b, :nk, h // group] += torch.mm(d_scores.t(), queries)
    if not grad:
        return [out, lse]
    return ([out] if forward else []) + [d_q, d_k, d_v]


def exact(case, seed):
    state = prepare(case, seed)
    for key, value in state.items():
        if isinstance(value, torch.Tensor):
            state[key] = value.detach()
    if case["path"].startswith("norm"):
        return _exact_norm(state, case)
    return (_exact_rope if case["path"].startswith("rope") else _exact_attention)(state, case)
