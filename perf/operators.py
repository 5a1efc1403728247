"""Workloads of the operators around ``slot_murmurate`` in a transformer block.

Three operators, each in a plain form (elementary torch operations in 32 bits) and through this
package's public functions:

- ``linear``:   y = act(x W^T + b) + residual, alone or with its gradients (``fused_linear``);
- ``qk``:       per-head RMS norm of queries and keys and the position rotation of both, alone or
                with its gradients (``qk_norm_rope``);
- ``rotary``:   rotation by positions of several axes (time, height, width), alone or with its
                gradient (``rotary``).

``listed()`` names the cases, ``draw(rng)`` makes further ones of the same ranges,
``prepare(case, seed)`` makes a case's inputs, ``run(state)`` is one pass, ``work(case)`` the bytes
and operations a pass cannot do without and ``exact(case, seed)`` the outputs in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_EPS, _BASE = 1e-6, 10000.0
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _linear(name, rows, k, n, dtype, activation, bias, residual, train):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "activation": activation,
            "bias": bias, "residual": residual, "train": train}


def _qk(name, batch, q_heads, k_heads, tokens, head_dim, rotary_dim, dtype, layout, interleaved, start, train):
    return {"name": name, "op": "qk", "batch": batch, "q_heads": q_heads, "k_heads": k_heads, "tokens": tokens,
            "head_dim": head_dim, "rotary_dim": rotary_dim, "dtype": dtype, "layout": layout,
            "interleaved": interleaved, "start": start, "train": train}


def _rotary(name, batch, heads, frames, height, width, head_dim, sections, dtype, layout, interleaved, spectrum, train):
    return {"name": name, "op": "rotary", "batch": batch, "heads": heads, "frames": frames, "height": height,
            "width": width, "head_dim": head_dim, "sections": sections, "dtype": dtype, "layout": layout,
            "interleaved": interleaved, "spectrum": spectrum, "train": train}


def listed():
    return [
        # the output projection with its residual, for the next token of four sequences
        _linear("linear_step", 4, 1024, 1024, "float16", "none", False, True, False),
        # a small model in fp32 on a ragged batch: nothing is a multiple of a tile or of 16 bytes
        _linear("linear_ragged_fp32", 777, 1001, 1111, "float32", "silu", True, True, False),
        # the first product of a block's feed-forward part over a long sequence, inference
        _linear("linear_up", 8192, 1024, 4096, "bfloat16", "gelu", True, False, False),
        # training step of the query or output projection over a long sequence
        _linear("linear_proj_train", 8192, 1024, 1024, "float16", "none", True, True, True),
        # training step of the feed-forward part's first product, a full batch
        _linear("linear_up_train", 32768, 1024, 4096, "bfloat16", "gelu_tanh", True, False, True),
        # queries and shared-head keys of the next token of eight sequences far into their contexts
        _qk("qk_step", 8, 16, 4, 1, 64, 64, "bfloat16", "token", False, 100000, False),
        # queries and keys of a long prompt, straight from the projections
        _qk("qk_prompt", 1, 16, 16, 8192, 64, 64, "float16", "token", False, 0, False),
        # fp32 training, an odd length, half of an odd head size rotated, adjacent pairs
        _qk("qk_odd_train", 3, 6, 2, 1021, 80, 40, "float32", "head", True, 17, True),
        # training step over a full batch with shared key heads
        _qk("qk_train", 8, 16, 4, 8192, 128, 128, "bfloat16", "token", False, 0, True),
        # one small image through a model with few heads: latency
        _rotary("rotary_image_small", 1, 8, 1, 16, 16, 64, "0,16,16", "float16", "token", False, "own", False),
        # a batch of images at two axes, an odd head size
        _rotary("rotary_images", 8, 16, 1, 64, 63, 72, "0,18,18", "bfloat16", "head", True, "own", False),
        # training on a video clip: time, height and width, one spectrum shared by the axes
        _rotary("rotary_video_train", 2, 24, 13, 45, 40, 128, "16,24,24", "bfloat16", "token", False, "shared", True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("linear", "qk", "rotary"))
    dtype = rng.choice(("float32", "float16", "bfloat16", "float16", "bfloat16"))
    train = rng.random() < 0.5
    layout = rng.choice(("token", "head"))
    if op == "linear":
        k, n = _log_int(rng, 96, 4096), _log_int(rng, 96, 4096)
        # most widths are multiples of 8, as models have them; the rest are odd
        if rng.random() < 0.7:
            k, n = k // 8 * 8, n // 8 * 8
        top = 32768 if dtype != "float32" else 4096
        rows = min(_log_int(rng, 1, top), max(1, 32768 * 1024 * 4096 // (k * n)))
        case = _linear("", rows, k, n, dtype, rng.choice(ACTIVATIONS), rng.random() < 0.6, rng.random() < 0.5, train)
    elif op == "qk":
        head_dim = rng.choice((16, 32, 64, 64, 72, 80, 96, 128, 128))
        rotary_dim = head_dim if rng.random() < 0.7 else head_dim // 4 * 2
        k_heads = rng.choice((1, 2, 3, 4, 8))
        q_heads = k_heads * rng.choice((1, 2, 3, 4))
        batch = rng.choice((1, 2, 3, 8))
        cap = 8 * 20 * 8192 * 128 // (batch * (q_heads + k_heads) * head_dim)
        if dtype == "float32":
            cap //= 2
        tokens = _log_int(rng, 1, min(16384, cap))
        case = _qk("", batch, q_heads, k_heads, tokens, head_dim, rotary_dim, dtype, layout, rng.random() < 0.5,
                   _log_int(rng, 1, 1000000) - 1, train)
    else:
        head_dim = rng.choice((32, 64, 72, 96, 128))
        frames, height, width = rng.choice((1, 1, 4, 13)), _log_int(rng, 4, 64), _log_int(rng, 4, 64)
        heads = rng.choice((1, 4, 8, 16, 24))
        pairs = head_dim // 2
        a = pairs // 3 if frames > 1 else 0
        b = (pairs - a) // 2
        batch = rng.choice((1, 2, 3))
        case = _rotary("", batch, heads, frames, height, width, head_dim, f"{a},{b},{pairs - a - b}", dtype, layout,
                       rng.random() < 0.5, rng.choice(("own", "shared")), train)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _heads(g, batch, heads, tokens, head_dim, dtype, layout):
    """[B, H, N, d], in the projection's [B, N, H, d] memory ("token") or contiguous ("head")."""
    if layout == "token":
        return _randn(g, (batch, tokens, heads, head_dim), dtype).transpose(1, 2)
    return _randn(g, (batch, heads, tokens, head_dim), dtype)


def _sections(case):
    return tuple(int(s) for s in case["sections"].split(","))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        st["x"] = _randn(g, (m, k), dt)
        st["weight"] = _randn(g, (n, k), dt, k ** -0.5)
        st["bias"] = _randn(g, (n,), dt, 0.1) if case["bias"] else None
        st["residual"] = _randn(g, (m, n), dt) if case["residual"] else None
        st["wrt"] = [st[name] for name in ("x", "weight", "bias", "residual") if st[name] is not None]
        if case["train"]:
            st["grad"] = _randn(g, (m, n), dt, 0.1)
    elif case["op"] == "qk":
        b, n, d = case["batch"], case["tokens"], case["head_dim"]
        st["q"] = _heads(g, b, case["q_heads"], n, d, dt, case["layout"])
        st["k"] = _heads(g, b, case["k_heads"], n, d, dt, case["layout"])
        st["q_weight"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt)
        st["k_weight"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt)
        first = case["start"] + torch.randint(0, 1000, (b, 1), generator=g, device="cuda")
        st["positions"] = first + torch.arange(n, device="cuda")
        st["freq"], st["axis"] = _frequencies(case["rotary_dim"], None, None, _BASE)
        st["wrt"] = [st["q"], st["k"], st["q_weight"], st["k_weight"]]
        if case["train"]:
            st["grad"] = (_heads(g, b, case["q_heads"], n, d, dt, case["layout"]),
                          _heads(g, b, case["k_heads"], n, d, dt, case["layout"]))
    else:
        f, h, w, d = case["frames"], case["height"], case["width"], case["head_dim"]
        st["x"] = _heads(g, case["batch"], case["heads"], f * h * w, d, dt, case["layout"])
        # each sequence starts at a frame of its own
        t0 = torch.randint(0, 100, (case["batch"], 1, 1, 1), generator=g, device="cuda")
        t = t0 + torch.arange(f, device="cuda").view(1, f, 1, 1)
        y = torch.arange(h, device="cuda").view(1, 1, h, 1)
        x = torch.arange(w, device="cuda").view(1, 1, 1, w)
        full = (case["batch"], f, h, w)
        st["positions"] = torch.stack([t.expand(full), y.expand(full), x.expand(full)], -1).reshape(
            case["batch"], f * h * w, 3)
        st["freq"], st["axis"] = _frequencies(d, _sections(case), case["spectrum"], _BASE)
        st["wrt"] = [st["x"]]
        if case["train"]:
            st["grad"] = _heads(g, case["batch"], case["heads"], f * h * w, d, dt, case["layout"])
    if case["train"]:
        for t in st["wrt"]:
            t.requires_grad_(True)
    return st


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
_SQRT_HALF, _SQRT_2_PI = math.sqrt(0.5), math.sqrt(2 / math.pi)


def _act(z, activation):
    if activation == "relu":
        return z * (z > 0)
    if activation == "silu":
        return z / (1 + torch.exp(-z))
    if activation == "gelu":
        return 0.5 * z * (1 + torch.erf(z * _SQRT_HALF))
    if activation == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(_SQRT_2_PI * (z + 0.044715 * z * z * z)))
    return z


def _act_grad(z, activation):
    if activation == "relu":
        return (z > 0).to(z.dtype)
    if activation == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if activation == "gelu":
        return 0.5 * (1 + torch.erf(z * _SQRT_HALF)) + z * torch.exp(-0.5 * z * z) * (0.5 * _SQRT_2_PI)
    if activation == "gelu_tanh":
        t = torch.tanh(_SQRT_2_PI * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * (_SQRT_2_PI * (1 + 3 * 0.044715 * z * z))
    return torch.ones_like(z)


def _plain_linear(st):
    case, dt = st["case"], st["x"].dtype
    x, w = st["x"].float(), st["weight"].float()
    z = x @ w.t()
    if st["bias"] is not None:
        z = z + st["bias"].float()
    y = _act(z, case["activation"])
    if st["residual"] is not None:
        y = y + st["residual"].float()
    out = [y.to(dt)]
    if case["train"]:
        dy = st["grad"].float()
        dz = dy if case["activation"] == "none" else dy * _act_grad(z, case["activation"])
        out += [(dz @ w).to(dt), (dz.t() @ x).to(dt)]
        if st["bias"] is not None:
            out.append(dz.sum(0).to(dt))
        if st["residual"] is not None:
            out.append(dy.to(dt))
    return out


def _frequencies(rotary_dim, sections, spectrum, base):
    """(frequency of each pair, axis of each pair). "shared": pair i of the head turns at
    base^(-2i/rotary_dim) whatever its axis; "own": each axis has a whole spectrum over its pairs.
    A program of plain torch keeps this small table beside its weights."""
    pairs = torch.arange(rotary_dim // 2, dtype=torch.float64, device="cuda")
    if sections is None:
        return base ** (-2 * pairs / rotary_dim), None
    axis = torch.cat([torch.full((s,), a, dtype=torch.int64) for a, s in enumerate(sections)]).cuda()
    if spectrum == "shared":
        return base ** (-2 * pairs / rotary_dim), axis
    own_pairs = [torch.arange(s, dtype=torch.float64) / max(s, 1) for s in sections]
    return base ** -torch.cat(own_pairs).cuda(), axis


def _cos_sin(positions, freq, axis):
    """[B, 1, N, pairs] tables. The angle itself needs 64 bits: at position 100000 a 32-bit
    product is off by 0.004 rad."""
    p = positions.double()
    angle = (p[:, :, None] if axis is None else p[:, :, axis]) * freq
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _rotate(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        rot = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        rot = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return rot if r == x.shape[-1] else torch.cat((rot, x[..., r:]), -1)


def _plain_qk(st):
    case = st["case"]
    cos, sin = _cos_sin(st["positions"], st["freq"], st["axis"])
    outs, grads, wgrads = [], [], []
    for i, name in enumerate(("q", "k")):
        x, w = st[name].float(), st[name + "_weight"].float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        outs.append(_rotate(x * r * w, cos, sin, case["interleaved"]).to(st[name].dtype))
        if case["train"]:
            g = _rotate(st["grad"][i].float(), cos, -sin, case["interleaved"])
            gw = g * w
            dx = r * (gw - x * (r * r) * (gw * x).mean(-1, keepdim=True))
            grads.append(dx.to(st[name].dtype))
            wgrads.append((g * x * r).sum((0, 1, 2)).to(st[name].dtype))
    return outs + grads + wgrads


def _plain_rotary(st):
    case = st["case"]
    cos, sin = _cos_sin(st["positions"], st["freq"], st["axis"])
    dt = st["x"].dtype
    out = [_rotate(st["x"].float(), cos, sin, case["interleaved"]).to(dt)]
    if case["train"]:
        out.append(_rotate(st["grad"].float(), cos, -sin, case["interleaved"]).to(dt))
    return out


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _own(st):
    from murmurative_attention_b200 import fused_linear, qk_norm_rope, rotary

    case = st["case"]
    if case["op"] == "linear":
        outs = (fused_linear(st["x"], st["weight"], st["bias"], activation=case["activation"],
                             residual=st["residual"]),)
        grads = (st["grad"],) if case["train"] else None
    elif case["op"] == "qk":
        outs = qk_norm_rope(st["q"], st["k"], st["positions"], st["q_weight"], st["k_weight"], eps=_EPS, base=_BASE,
                            rotary_dim=case["rotary_dim"], interleaved=case["interleaved"])
        grads = st["grad"] if case["train"] else None
    else:
        outs = (rotary(st["x"], st["positions"], base=_BASE, sections=_sections(case), spectrum=case["spectrum"],
                       interleaved=case["interleaved"]),)
        grads = (st["grad"],) if case["train"] else None
    if grads is None:
        return list(outs)
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, st["wrt"], grads))


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"linear": _plain_linear, "qk": _plain_qk, "rotary": _plain_rotary}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    train = case["train"]
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        read = m * k + n * k + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        elements = read + m * n
        if train:  # + dy, dx, dW, db
            elements += m * n + m * k + n * k + (n if case["bias"] else 0)
        return {"bytes": elements * size, "flops": 2 * m * k * n * (3 if train else 1)}
    if case["op"] == "qk":
        d = case["head_dim"]
        rows = case["batch"] * (case["q_heads"] + case["k_heads"]) * case["tokens"]
        # forward: x in, y out; training: + dy in, dx out
        elements = rows * d * (4 if train else 2) + 2 * d * (2 if train else 1)
        flops = rows * (4 * d + 3 * case["rotary_dim"]) * (3 if train else 1)
        return {"bytes": elements * size + 8 * case["batch"] * case["tokens"], "flops": flops}
    tokens = case["batch"] * case["frames"] * case["height"] * case["width"]
    elements = tokens * case["heads"] * case["head_dim"] * (2 if not train else 4)
    return {"bytes": elements * size + 8 * 3 * tokens, "flops": 3 * elements // 2}


# ---------------------------------------------------------------------------
# the outputs in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _rotation_matrices(angle):
    """[..., pairs, 2, 2] rotation matrices."""
    c, s = torch.cos(angle), torch.sin(angle)
    return torch.stack((torch.stack((c, -s), -1), torch.stack((s, c), -1)), -2)


def _apply_pairs(x, rot, interleaved, transpose):
    """Each pair of the rotated part of x [B, H, N, d] times its 2x2 matrix (or its transpose)."""
    pairs = rot.shape[-3]
    idx = torch.arange(2 * pairs, device=x.device)
    idx = idx.view(pairs, 2) if interleaved else idx.view(2, pairs).t()
    if transpose:
        rot = rot.transpose(-1, -2)
    y = x.clone()
    v = x[..., idx]  # [B, H, N, pairs, 2]
    for i in (0, 1):
        y[..., idx[:, i]] = rot[..., i, 0] * v[..., 0] + rot[..., i, 1] * v[..., 1]
    return y


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "linear":
            return _exact_linear(case, st)
        if case["op"] == "qk":
            half = case["rotary_dim"] // 2
            speed = torch.tensor([_BASE ** (-i / half) for i in range(half)], dtype=torch.float64, device="cuda")
            rot = _rotation_matrices(st["positions"].double().unsqueeze(1).unsqueeze(-1) * speed)
            outs, dxs, dws = [], [], []
            for i, name in enumerate(("q", "k")):
                x, w = st[name].double(), st[name + "_weight"].double()
                rms = torch.sqrt(torch.sum(x * x, -1, keepdim=True) / x.shape[-1] + _EPS)
                outs.append(_apply_pairs(x / rms * w, rot, case["interleaved"], False))
                if case["train"]:
                    g = _apply_pairs(st["grad"][i].double(), rot, case["interleaved"], True)
                    unit = x / rms
                    h = g * w
                    dxs.append((h - unit * (unit * h).mean(-1, keepdim=True)) / rms)
                    dws.append((g * unit).sum((0, 1, 2)))
            return outs + dxs + dws
        sections = _sections(case)
        speed, axis = [], []
        for a, count in enumerate(sections):
            for j in range(count):
                share = j / count if case["spectrum"] == "own" else len(speed) / sum(sections)
                speed.append(_BASE ** -share)
                axis.append(a)
        place = st["positions"].double()[:, None, :, :][..., torch.tensor(axis, device="cuda")]
        rot = _rotation_matrices(place * torch.tensor(speed, dtype=torch.float64, device="cuda"))
        out = [_apply_pairs(st["x"].double(), rot, case["interleaved"], False)]
        if case["train"]:
            out.append(_apply_pairs(st["grad"].double(), rot, case["interleaved"], True))
        return out


def _exact_linear(case, st):
    x, w = st["x"].double(), st["weight"].double()
    z = torch.einsum("mk,nk->mn", x, w)
    if case["bias"]:
        z += st["bias"].double()
    kind = case["activation"]
    normal_cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    inner = math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3)  # gelu_tanh(z) = z sigmoid(inner)
    if kind == "none":
        y, slope = z.clone(), None
    elif kind == "relu":
        y, slope = z.clamp(min=0), torch.where(z > 0, 1.0, 0.0).double()
    elif kind == "silu":
        s = torch.sigmoid(z)
        y, slope = z * s, s + z * s * torch.sigmoid(-z)
    elif kind == "gelu":
        y, slope = z * normal_cdf, normal_cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        s = torch.sigmoid(inner)
        y = z * s
        slope = s + z * s * torch.sigmoid(-inner) * math.sqrt(8 / math.pi) * (1 + 0.134145 * z * z)
    if case["residual"]:
        y += st["residual"].double()
    out = [y]
    if case["train"]:
        dy = st["grad"].double()
        dz = dy if slope is None else dy * slope
        out += [torch.einsum("mn,nk->mk", dz, w), torch.einsum("mn,mk->nk", dz, x)]
        if case["bias"]:
            out.append(dz.sum(0))
        if case["residual"]:
            out.append(dy)
    return out
