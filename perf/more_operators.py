"""What a conditioned layer is trained with, around its cross attention: what is measured, in plain form and as a user calls it.

Three operators:

* ``rotary``: positions turned into rotations of pairs of channels of q [B, S, H, D] and k [B, S, Hkv, D],
      (x1, x2) -> f * (x1 cos a - x2 sin a, x2 cos a + x1 sin a),  a = position * w[pair],
  over the first R channels of a head, as pairs (i, i + R/2) or (2i, 2i + 1); the other channels stay.  Frequencies
  w[i] = theta^(-2i/R), for a grid of positions in sections of their own, and for contexts longer than the trained ones
  scaled: all of them ("linear"), by another theta ("base"), or those of few turns over the trained length ("parts").
  With ``back`` the gradients of q and k for given gradients of the rotated ones too (the rotation the other way).
* ``norm``: y = (x - mean) / sqrt(var + eps) * w + b over the last axis, and with ``back`` the gradients of x, w and b.
* ``ortho``: the orthogonal factor of an update, approached by five steps x <- a x + (b g + c g g) x, g = x x^T, from
  x / |x|, the smaller side first, as the optimiser of the layer's matrices takes it.

``own`` False computes them with elementary torch operations in 32 bits, rounded once at the end (angles in 64); True makes
the calls that a user makes of ``minixmax_h3_b200``.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-5  # of the norm
STEPS, COEFFICIENTS, ORTHO_EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7


# ----------------------------------------------------------------------------- cases


def listed():
    return [
        # One new token of one sequence, far into its context: latency.
        {"name": "rotary-one-token", "kind": "rotary", "b": 1, "s": 1, "h": 24, "hkv": 24, "d": 128, "r": 128,
         "pairs": "halves", "axes": 1, "scaling": "none", "far": 100000, "dtype": "bf16", "back": False},
        # Ragged text tokens in a window stretched by eight, shared key heads, half of each head turned.
        {"name": "rotary-stretched", "kind": "rotary", "b": 3, "s": 1111, "h": 16, "hkv": 4, "d": 64, "r": 32,
         "pairs": "neighbours", "axes": 1, "scaling": "parts", "far": 30000, "dtype": "f16", "back": False},
        # The video tokens of a clip by their grid positions.
        {"name": "rotary-video", "kind": "rotary", "b": 1, "s": 32768, "h": 24, "hkv": 24, "d": 128, "r": 128,
         "pairs": "halves", "axes": 3, "scaling": "none", "far": 0, "dtype": "bf16", "back": False},
        # A training step on a clip: rotated and the gradients turned back.
        {"name": "rotary-train", "kind": "rotary", "b": 2, "s": 8192, "h": 24, "hkv": 8, "d": 128, "r": 128,
         "pairs": "halves", "axes": 3, "scaling": "base", "far": 0, "dtype": "bf16", "back": True},
        # One token's activations before a projection.
        {"name": "norm-one-token", "kind": "norm", "m": 1, "n": 4096, "dtype": "bf16", "weights": "f32",
         "affine": "both", "back": False},
        # The tokens of a clip.
        {"name": "norm-video", "kind": "norm", "m": 32768, "n": 4096, "dtype": "bf16", "weights": "bf16",
         "affine": "both", "back": False},
        # An odd width in 32 bits, forward and backward.
        {"name": "norm-train-odd", "kind": "norm", "m": 2049, "n": 1111, "dtype": "f32", "weights": "f32",
         "affine": "both", "back": True},
        # A training step on the tokens of a clip.
        {"name": "norm-train", "kind": "norm", "m": 16384, "n": 4096, "dtype": "bf16", "weights": "f32",
         "affine": "both", "back": True},
        # The smallest matrices of a layer: latency.
        {"name": "ortho-small", "kind": "ortho", "b": 1, "m": 96, "n": 250, "dtype": "f32"},
        # The update of each head of a projection by itself.
        {"name": "ortho-heads", "kind": "ortho", "b": 24, "m": 128, "n": 1024, "dtype": "bf16"},
        # A key and value projection, taller than wide, in 32 bits.
        {"name": "ortho-projection", "kind": "ortho", "b": 1, "m": 4096, "n": 1024, "dtype": "f32"},
        # A square projection of a wide layer.
        {"name": "ortho-wide", "kind": "ortho", "b": 1, "m": 4096, "n": 4096, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_rotary(rng):
    h = rng.choice([1, 4, 8, 16, 24, 32])
    d = rng.choice([64, 80, 96, 128, 256])
    c = {"kind": "rotary", "h": h, "hkv": max(1, h // rng.choice([1, 2, 4])), "d": d,
         "r": rng.choice([d, d, d // 2, d // 4]), "pairs": rng.choice(["halves", "neighbours"]),
         "axes": rng.choice([1, 3]), "scaling": rng.choice(["none", "linear", "base", "parts"]),
         "far": _log_int(rng, 1, 1000000), "dtype": rng.choice(["bf16", "f16", "f32"]), "back": rng.random() < 0.4}
    size = 4 if c["dtype"] == "f32" else 2
    c["b"] = rng.choice([1, 1, 2, 3, 4, 16])
    # no more bytes than the largest listed case
    most = 32768 * 48 * 128 * 2 // (c["b"] * (h + c["hkv"]) * d * size * (2 if c["back"] else 1))
    c["s"] = _log_int(rng, 1, max(1, min(32768, most)))
    return c


def _draw_norm(rng):
    c = {"kind": "norm", "n": _log_int(rng, 32, 16384), "dtype": rng.choice(["bf16", "f16", "f32"]),
         "affine": rng.choice(["both", "both", "weight", "none"]), "back": rng.random() < 0.5}
    c["weights"] = rng.choice([c["dtype"], "f32"])
    if rng.random() < 0.5:
        c["n"] = max(32, c["n"] // 32 * 32)
    size = 4 if c["dtype"] == "f32" else 2
    c["m"] = _log_int(rng, 1, max(1, min(65536, 16384 * 4096 * 2 // (c["n"] * size))))
    return c


def _draw_ortho(rng):
    c = {"kind": "ortho", "b": rng.choice([1, 1, 1, 2, 3, 8, 24]), "dtype": rng.choice(["bf16", "f16", "f32"])}
    most = 4 * 4096 ** 3 // (c["b"] * (3 if c["dtype"] != "bf16" else 1))
    while True:
        c["m"], c["n"] = _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)
        small, large = sorted((c["m"], c["n"]))
        if small * small * (3 * large + small) <= most:
            return c


def draw(rng):
    return {"rotary": _draw_rotary, "norm": _draw_norm, "ortho": _draw_ortho}[rng.choice(["rotary", "norm", "ortho"])](rng)


def work(c):
    size = DTYPES[c["dtype"]].itemsize
    if c["kind"] == "rotary":
        x = c["b"] * c["s"] * (c["h"] + c["hkv"])
        ways = 2 if c["back"] else 1
        # every channel read and written; three operations for each channel that is turned
        return {"bytes": ways * 2 * x * c["d"] * size + 4 * c["b"] * c["s"] * c["axes"], "flops": ways * 3 * x * c["r"]}
    if c["kind"] == "norm":
        x, w = c["m"] * c["n"], c["n"] * {"both": 2, "weight": 1, "none": 0}[c["affine"]] * DTYPES[c["weights"]].itemsize
        if not c["back"]:
            return {"bytes": 2 * x * size + w, "flops": 8 * x}
        # x and the gradient of y read, y and the gradient of x written; the weights read, their gradients written
        return {"bytes": 4 * x * size + 2 * w, "flops": 20 * x}
    small, large = sorted((c["m"], c["n"]))
    # two of the three products are symmetric: half of each is enough
    return {"bytes": 2 * c["b"] * c["m"] * c["n"] * size,
            "flops": STEPS * c["b"] * small * small * (large + small + 2 * large)}


# ----------------------------------------------------------------------------- frequencies


def _sections(c):
    """Channels turned by each axis of the grid: near thirds, each even, the first one the largest."""
    if c["axes"] == 1:
        return [c["r"]]
    third = c["r"] // 6 * 2
    return [c["r"] - 2 * third, third, third]


SCALE, TRAINED = 8.0, 4096  # how much longer the context is than the trained one, and that one's tokens
FAST, SLOW = 32.0, 1.0      # "parts": turns over the trained length above which nothing, below which all is scaled


def _frequencies(c):
    """Radians a position for each pair, in Python's 64 bits, and the factor of the rotated channels."""
    w = []
    for dims in _sections(c):
        theta = 10000.0
        if c["scaling"] == "base" and dims > 2:
            theta *= SCALE ** (dims / (dims - 2))
        for i in range(dims // 2):
            f = theta ** (-2 * i / dims)
            if c["scaling"] == "linear":
                f /= SCALE
            elif c["scaling"] == "parts":
                turns = TRAINED * f / (2 * math.pi)
                keep = min(1.0, max(0.0, (turns - SLOW) / (FAST - SLOW)))
                f = f / SCALE * (1 - keep) + f * keep
            w.append(f)
    return w, 0.1 * math.log(SCALE) + 1 if c["scaling"] == "parts" else 1.0


# ----------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _positions(c, gen):
    """int32 [b, s] (or [b, s, 3] on a grid): samples start at different places, the first one the farthest."""
    at = torch.arange(c["s"], device="cuda", dtype=torch.int32)
    if c["axes"] == 3:
        wide = max(1, round(math.sqrt(c["s"] / 4)))
        grid = torch.stack([at // (wide * wide), at // wide % wide, at % wide], dim=-1)
        return (grid[None] + torch.randint(0, 8 + c["far"], (c["b"], 1, 3), generator=gen, device="cuda",
                                           dtype=torch.int32)).contiguous()
    start = torch.tensor([c["far"] * (c["b"] - i) // c["b"] for i in range(c["b"])], device="cuda", dtype=torch.int32)
    return start[:, None] + at


def _rotary_inputs(c, seed):
    gen, dt = _generator(seed), DTYPES[c["dtype"]]
    # q, k and v are slices of one projection of the tokens
    qkv = _normal(gen, c["b"], c["s"], c["h"] + 2 * c["hkv"], c["d"], dtype=dt)
    w, factor = _frequencies(c)
    s = {"q": qkv[:, :, :c["h"]], "k": qkv[:, :, c["h"]:c["h"] + c["hkv"]], "positions": _positions(c, gen),
         "w": torch.tensor(w, dtype=torch.float64, device="cuda"), "factor": factor, "pairs": c["pairs"],
         "sections": [n // 2 for n in _sections(c)], "back": c["back"]}
    if c["back"]:
        s["dq"], s["dk"] = (_normal(gen, c["b"], c["s"], n, c["d"], dtype=dt) for n in (c["h"], c["hkv"]))
    if own:
        from minixmax_h3_b200 import ops

        scaling = {"none": None, "linear": "linear", "base": "base", "parts": "by_parts"}[c["scaling"]]
        s["rope"] = ops.Rotary.build(_sections(c), interleaved=c["pairs"] == "neighbours", scaling=scaling,
                                     scale=SCALE, trained_len=TRAINED, device="cuda")
    return s


def _norm_inputs(c, seed):
    gen, dt, wt = _generator(seed), DTYPES[c["dtype"]], DTYPES[c["weights"]]
    # activations of a residual stream: tokens of varying size with a mean of their own, a few channels much larger
    x = _normal(gen, c["m"], c["n"], dtype=dt)
    x *= (1 + 15 * (torch.rand(c["n"], generator=gen, device="cuda") < 0.01)).to(dt)
    x = x.mul_(torch.exp2(2 * torch.rand(c["m"], 1, generator=gen, device="cuda") - 1).to(dt))
    x += (0.5 * _normal(gen, c["m"], 1)).to(dt)
    s = {"x": x, "w": None, "b": None, "back": c["back"]}
    if c["affine"] != "none":
        s["w"] = (1 + 0.1 * _normal(gen, c["n"])).to(wt)
    if c["affine"] == "both":
        s["b"] = (0.1 * _normal(gen, c["n"])).to(wt)
    if c["back"]:
        s["dy"] = _normal(gen, c["m"], c["n"], dtype=dt)
    return s


def _ortho_inputs(c, seed):
    gen = _generator(seed)
    # an averaged gradient: a few directions carry most of it, the rest is noise; small values
    rank = min(4, c["m"], c["n"])
    g = torch.bmm(_normal(gen, c["b"], c["m"], rank), _normal(gen, c["b"], rank, c["n"]))
    return {"x": (1e-3 * (g + 0.5 * _normal(gen, c["b"], c["m"], c["n"]))).to(DTYPES[c["dtype"]])}


def prepare(case, seed):
    make = {"rotary": _rotary_inputs, "norm": _norm_inputs, "ortho": _ortho_inputs}
    s = make[case["kind"]](case, seed)
    s["kind"] = case["kind"]
    return s


# ----------------------------------------------------------------------------- plain forms


def _turn(x, cos, sin, neighbours):
    """cos and sin [b, s, 1, pairs] in 32 bits."""
    n = cos.shape[-1]
    y = x.float().clone()
    one, two = (y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if neighbours else (y[..., :n], y[..., n:2 * n])
    a, b = one * cos - two * sin, two * cos + one * sin
    one.copy_(a)
    two.copy_(b)
    return y.to(x.dtype)


def _plain_rotary(s):
    p = s["positions"]
    if p.dim() == 2:
        p = p[..., None]
    p = torch.cat([p[..., i:i + 1].expand(*p.shape[:2], n) for i, n in enumerate(s["sections"])], dim=-1)
    angle = (p.double() * s["w"])[:, :, None]  # 64 bits: a far position's angle has many whole turns
    cos, sin = (angle.cos() * s["factor"]).float(), (angle.sin() * s["factor"]).float()
    neighbours = s["pairs"] == "neighbours"
    out = {"q": _turn(s["q"], cos, sin, neighbours), "k": _turn(s["k"], cos, sin, neighbours)}
    if s["back"]:
        out["dq"], out["dk"] = _turn(s["dq"], cos, -sin, neighbours), _turn(s["dk"], cos, -sin, neighbours)
    return out


def _plain_norm(s):
    x = s["x"].float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    xhat = centred * rstd
    y = xhat
    if s["w"] is not None:
        y = y * s["w"].float()
    if s["b"] is not None:
        y = y + s["b"].float()
    out = {"y": y.to(s["x"].dtype)}
    if s["back"]:
        dy = s["dy"].float()
        g = dy if s["w"] is None else dy * s["w"].float()
        dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
        out["dx"] = dx.to(s["x"].dtype)
        if s["w"] is not None:
            out["dw"] = (dy * xhat).sum(0).to(s["w"].dtype)
        if s["b"] is not None:
            out["db"] = dy.sum(0).to(s["b"].dtype)
    return out


def _plain_ortho(s):
    x = s["x"].float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = x / (torch.sqrt((x.double() ** 2).sum((1, 2), keepdim=True)) + ORTHO_EPS).float()
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        g = torch.matmul(x, x.transpose(1, 2))
        x = a * x + torch.matmul(b * g + c * torch.matmul(g, g), x)
    return {"x": (x.transpose(1, 2) if tall else x).to(s["x"].dtype)}


# ----------------------------------------------------------------------------- as a user calls them


def _own_rotary(s):
    from minixmax_h3_b200 import ops

    q, k = ops.rotary(s["q"], s["k"], s["positions"], s["rope"])
    out = {"q": q, "k": k}
    if s["back"]:
        out["dq"], out["dk"] = ops.rotary(s["dq"], s["dk"], s["positions"], s["rope"], inverse=True)
    return out


def _own_norm(s):
    from minixmax_h3_b200 import ops

    if not s["back"]:
        return {"y": ops.layer_norm(s["x"], s["w"], s["b"], EPS)}
    stats = torch.empty(2, s["x"].shape[0], dtype=torch.float32, device="cuda")
    out = {"y": ops.layer_norm(s["x"], s["w"], s["b"], EPS, stats=stats)}
    out["dx"], dw, db = ops.layer_norm_bwd(s["dy"], s["x"], stats, s["w"], bias_grad=s["b"] is not None)
    if s["w"] is not None:
        out["dw"] = dw
    if s["b"] is not None:
        out["db"] = db
    return out


def _own_ortho(s):
    from minixmax_h3_b200 import ops

    return {"x": ops.orthogonalize(s["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=ORTHO_EPS)}


def run(state):
    if own:
        return {"rotary": _own_rotary, "norm": _own_norm, "ortho": _own_ortho}[state["kind"]](state)
    return {"rotary": _plain_rotary, "norm": _plain_norm, "ortho": _plain_ortho}[state["kind"]](state)


# ----------------------------------------------------------------------------- 64 bits


def _exact_turn(x, angle, factor, pairs):
    """As products of complex numbers."""
    n = angle.shape[-1]
    x = x.double()
    turned, rest = x[..., :2 * n], x[..., 2 * n:]
    z = turned.reshape(*turned.shape[:-1], n, 2) if pairs == "neighbours" else turned.reshape(*turned.shape[:-1], 2, n).mT
    z = torch.view_as_complex(z.contiguous()) * torch.polar(torch.full_like(angle, factor), angle)[:, :, None]
    z = torch.view_as_real(z)
    z = z.flatten(-2) if pairs == "neighbours" else z.mT.flatten(-2)
    return torch.cat([z, rest], dim=-1)


def _exact_rotary(c, s):
    p = s["positions"].double().reshape(c["b"], c["s"], c["axes"])
    angle = torch.empty(c["b"], c["s"], c["r"] // 2, dtype=torch.float64, device="cuda")
    at = 0
    for i, dims in enumerate(_sections(c)):
        angle[..., at:at + dims // 2] = p[..., i, None] * s["w"][at:at + dims // 2]
        at += dims // 2
    out = {n: _exact_turn(s[n], angle, s["factor"], c["pairs"]) for n in ("q", "k")}
    if c["back"]:
        out |= {n: _exact_turn(s[n], -angle, s["factor"], c["pairs"]) for n in ("dq", "dk")}
    return out


def _exact_norm(c, s):
    """The backward pass from the matrix of derivatives: dx = (J dy w), J = rstd (1 - 1/n - xhat xhat^T / n)."""
    x = s["x"].double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    xhat = (x - mean) * (var + EPS) ** -0.5
    w = torch.ones(c["n"], dtype=torch.float64, device="cuda") if s["w"] is None else s["w"].double()
    out = {"y": xhat * w + (0 if s["b"] is None else s["b"].double())}
    if c["back"]:
        dy = s["dy"].double()
        g = dy * w
        along = torch.einsum("mn,mn->m", g, xhat)[:, None]
        out["dx"] = (c["n"] * g - torch.einsum("mn->m", g)[:, None] - xhat * along) / (c["n"] * (var + EPS) ** 0.5)
        if s["w"] is not None:
            out["dw"] = torch.einsum("mn,mn->n", dy, xhat)
        if s["b"] is not None:
            out["db"] = torch.einsum("mn->n", dy)
    return out


def _exact_ortho(c, s):
    """One matrix after the other, the polynomial by Horner's rule from the side that is smaller."""
    a, b, k = COEFFICIENTS
    out = []
    for x in s["x"].double():
        x = x / (torch.linalg.matrix_norm(x) + ORTHO_EPS)
        one = torch.eye(min(x.shape), dtype=torch.float64, device="cuda")
        for _ in range(STEPS):
            if x.shape[0] <= x.shape[1]:
                g = x @ x.T
                x = (a * one + g @ (b * one + k * g)) @ x
            else:
                g = x.T @ x
                x = x @ (a * one + g @ (b * one + k * g))
        out.append(x)
    return {"x": torch.stack(out)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "norm": _exact_norm, "ortho": _exact_ortho}[case["kind"]](case, s)
