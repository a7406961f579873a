"""The operators around the attention of a video transformer block, as they are measured.

Three operators:

``rotate``  the query and key norm with the rotary positions over (time, height, width)
            that stand between the projections and ``Operator.attend``;
``norm``    the norm with scale and shift before a block;
``gate``    the gate and residual sum after a block, with the norm of the next one.

``run`` computes them from elementary torch operations in 32 bits (angles in 64), or, with
``own`` set, by the calls a user of ``recap_b200`` makes.
"""

import math

import torch

own = False

# A case's largest drawn size, in elements of all its inputs (the largest listed case has
# 731 million): a drawn case costs no more than a listed one and is quickly made.
DRAWN_ELEMENTS = 60_000_000


def _rotate(name, dtype, batch, q_heads, k_heads, dim, grid, text, text_first, layout, norm, pairs, ladder="axis",
            rotated=None, far=0, tokens=None):
    """``grid`` None: positions come as a tensor of the call (``tokens`` of them)."""
    t, h, w = grid or (0, 0, 0)
    return dict(name=name, op="rotate", dtype=dtype, batch=batch, q_heads=q_heads, k_heads=k_heads, dim=dim, t=t, h=h,
                w=w, text=text, text_first=text_first, layout=layout, norm=norm, pairs=pairs, ladder=ladder,
                rotated=rotated or dim, far=far, tokens=tokens or (t * h * w + text))


def _norm(name, dtype, out, batch, tokens, width, kind, affine, mod, per_token):
    return dict(name=name, op="norm", dtype=dtype, out=out, batch=batch, tokens=tokens, width=width, kind=kind,
                affine=affine, mod=mod, per_token=per_token)


def _gate(name, dtype, out, batch, tokens, width, kind, affine, mod, per_token, branch_kind):
    return dict(name=name, op="gate", dtype=dtype, out=out, batch=batch, tokens=tokens, width=width, kind=kind,
                affine=affine, mod=mod, per_token=per_token, branch_kind=branch_kind)


def listed():
    bf, hf, f32 = "bfloat16", "float16", "float32"
    return [
        # one token at a far position: the smallest call there is, all latency
        _rotate("rotate one token", bf, 1, 12, 12, 128, None, 0, False, "token", "rms", "interleaved", far=100000,
                tokens=1),
        # the first frame of the 480p layer in its packed projections: a small grid
        _rotate("rotate one frame", bf, 1, 12, 12, 128, (1, 30, 52), 0, False, "packed", "rms_across", "interleaved"),
        # a picture between two texts, halves paired, one ladder of frequencies over the
        # axes, fewer key heads, odd token count, 10 of 11 dims turned, fp32
        _rotate("rotate picture and text", f32, 2, 10, 2, 88, None, 0, False, "token", "none", "halves", "shared",
                rotated=80, far=4000, tokens=4099),
        # the 480p layer of the benchmark: 12 heads, the norm over all of them
        _rotate("rotate 480p layer", bf, 1, 12, 12, 128, (21, 30, 52), 0, False, "token", "rms_across", "interleaved"),
        # the 768p layer: two guidance branches, 64 dims, text first, layer norm; in fp16
        _rotate("rotate 768p pair", hf, 2, 48, 48, 64, (11, 48, 85), 226, True, "head", "layer", "interleaved"),
        # the 720p layer, the benchmark's headline: the largest
        _rotate("rotate 720p layer", bf, 1, 24, 24, 128, (33, 45, 80), 256, False, "packed", "rms", "interleaved"),
        # the norm of a handful of conditioning tokens
        _norm("norm few tokens", bf, bf, 2, 3, 1536, "layer", True, f32, False),
        # the 480p layer's residual stream kept in fp32, its norm in bf16
        _norm("norm 480p layer", f32, bf, 1, 32760, 1536, "layer", False, f32, False),
        # an odd batch of short clips, root-mean-square norm, each token its own modulation
        _norm("norm ragged clips", hf, hf, 3, 5003, 1352, "rms", True, hf, True),
        # the text stream of the 768p pair
        _gate("gate text tokens", bf, bf, 2, 226, 1920, "layer", True, bf, False, "none"),
        # the residual of a wide 480p layer in fp32
        _gate("gate wide 480p layer", f32, bf, 1, 32760, 5120, "layer", False, f32, False, "none"),
        # norms after and before the block, a gate for each token, odd count
        _gate("gate sandwich", bf, bf, 1, 17777, 2304, "rms", True, bf, True, "rms"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "norm", "gate"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    batch = rng.choice([1, 1, 2, 3])
    if op == "rotate":
        dim = rng.choice([40, 64, 72, 80, 96, 128, 128, 256])
        norm = rng.choice(["none", "rms", "layer", "rms_across"])
        layout = rng.choice(["packed", "token", "head"])
        q_heads = rng.randint(1, 40)
        k_heads = q_heads if layout == "packed" or rng.random() < 0.6 else rng.randint(1, q_heads)
        most = max(1, min(60000, DRAWN_ELEMENTS // (batch * (q_heads + 2 * k_heads) * dim)))
        tokens = _log(rng, 1, most)
        pairs = rng.choice(["interleaved", "halves"])
        rotated = rng.choice([dim, dim, dim - 8]) if dim > 40 else dim
        if rng.random() < 0.5:
            return {k: v for k, v in _rotate("", dtype, batch, q_heads, k_heads, dim, None, 0, False, layout, norm,
                                             pairs, rng.choice(["axis", "shared"]), rotated, _log(rng, 1, 200000),
                                             tokens).items() if k != "name"}
        text = rng.randint(0, min(300, tokens - 1))
        w = _log(rng, 1, max(1, min(90, tokens - text)))
        h = _log(rng, 1, max(1, min(60, (tokens - text) // w)))
        t = max(1, (tokens - text) // (w * h))
        return {k: v for k, v in _rotate("", dtype, batch, q_heads, k_heads, dim, (t, h, w), text, rng.random() < 0.5,
                                         layout, norm, pairs, rng.choice(["axis", "shared"]), rotated).items()
                if k != "name"}
    width = 8 * _log(rng, 8, 768)
    tokens = _log(rng, 1, max(1, min(60000, DRAWN_ELEMENTS // (2 * batch * width))))
    out = dtype if dtype != "float32" else rng.choice(["float32", "bfloat16", "float16"])
    kind, affine = rng.choice(["layer", "rms"]), rng.random() < 0.5
    mod, per_token = rng.choice([out, "float32"]), rng.random() < 0.3
    if op == "norm":
        case = _norm("", dtype, out, batch, tokens, width, kind, affine, mod, per_token)
    else:
        case = _gate("", dtype, out, batch, tokens, width, kind, affine, mod, per_token,
                     rng.choice(["none", "none", "rms", "layer"]))
    del case["name"]
    return case


def _axes(case):
    """Turned dims of each axis: time takes what height and width, a third each, leave."""
    third = 2 * (case["rotated"] // 6)
    return case["rotated"] - 2 * third, third, third


EPS = 1e-6
THETA = 10000.0


def _weights(g, n, dtype):
    return (1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    s = {"case": case}

    def normal(*shape, dtype=dtype):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    if case["op"] == "rotate":
        b, n, d, hq, hk = (case[k] for k in ("batch", "tokens", "dim", "q_heads", "k_heads"))
        spread = torch.exp(0.5 * normal(2, d, dtype=torch.float32)).to(dtype)  # channels differ in size
        offset = (0.5 * normal(d, dtype=torch.float32)).to(dtype)  # and the keys' are off centre
        if case["layout"] == "packed":
            qkv = normal(b, n, 3, hq, d)
            q, k = qkv[:, :, 0].transpose(1, 2), qkv[:, :, 1].transpose(1, 2)
        elif case["layout"] == "token":
            q, k = normal(b, n, hq, d).transpose(1, 2), normal(b, n, hk, d).transpose(1, 2)
        else:
            q, k = normal(b, hq, n, d), normal(b, hk, n, d)
        s["q"], s["k"] = q.mul_(spread[0]), k.mul_(spread[1]).add_(offset)
        s["q_weight"] = s["k_weight"] = s["q_bias"] = s["k_bias"] = None
        if case["norm"] != "none":
            across = case["norm"] == "rms_across"
            s["q_weight"] = _weights(g, hq * d if across else d, dtype)
            s["k_weight"] = _weights(g, hk * d if across else d, dtype)
            if case["norm"] == "layer":
                s["q_bias"], s["k_bias"] = (0.1 * normal(d, dtype=torch.float32)).to(dtype), \
                    (0.1 * normal(d, dtype=torch.float32)).to(dtype)
        s["positions"] = _given_positions(case, g) if not case["t"] else None
        if own:
            from recap_b200 import AxialRotary, Norm

            grid = (case["t"], case["h"], case["w"]) if case["t"] else None
            s["rotary"] = AxialRotary(d, _axes(case), theta=THETA, grid=grid, text_tokens=case["text"],
                                      text_first=case["text_first"], pairs=case["pairs"], ladder=case["ladder"])
            s["q_norm"] = s["k_norm"] = None
            if case["norm"] != "none":
                kind, across = case["norm"].split("_")[0], case["norm"] == "rms_across"
                s["q_norm"] = Norm(kind, s["q_weight"], s["q_bias"], eps=EPS, across_heads=across)
                s["k_norm"] = Norm(kind, s["k_weight"], s["k_bias"], eps=EPS, across_heads=across)
        return s
    b, n, c = case["batch"], case["tokens"], case["width"]
    out, mod = getattr(torch, case["out"]), getattr(torch, case["mod"])
    size = torch.exp(0.5 * normal(c, dtype=torch.float32))
    size[torch.randint(0, c, (3,), generator=g, device="cuda")] *= 20  # the few large channels of a residual stream
    s["x"] = normal(b, n, c).mul_(size.to(dtype)).add_(normal(c).mul_(0.3))
    rows = n if case["per_token"] else 1
    for name in ("scale", "shift", "gate"):
        s[name] = normal(b, rows, c, dtype=mod).mul_(0.3)
    s["weight"] = _weights(g, c, dtype) if case["affine"] else None
    s["bias"] = (0.1 * normal(c, dtype=torch.float32)).to(dtype) if case["affine"] and case["kind"] == "layer" else None
    if case["op"] == "gate":
        s["branch"] = normal(b, n, c, dtype=out)
        s["branch_weight"] = _weights(g, c, out) if case["branch_kind"] != "none" else None
    if own:
        from recap_b200 import Norm

        s["norm"] = Norm(case["kind"], s["weight"], s["bias"], eps=EPS)
        if case["op"] == "gate" and case["branch_kind"] != "none":
            s["branch_norm"] = Norm(case["branch_kind"], s["branch_weight"], eps=EPS)
    return s


def _given_positions(case, g):
    """Integer positions [batch, tokens, 3] of a text, a picture as near square as fits into
    half of the tokens, and a text again: text counts on all axes at once, the picture keeps
    its time and counts rows and columns. Every sample starts at a place of its own."""
    n, b = case["tokens"], case["batch"]
    side = max(1, math.isqrt(n // 2))
    before = (n - side * side) // 2 if n > 1 else 0
    i = torch.arange(n, device="cuda")
    j = (i - before).clamp(0, side * side - 1)
    picture = torch.stack((torch.zeros_like(j), j // side, j % side), -1) + before
    after = (i - side * side + side).unsqueeze(-1).expand(n, 3)
    p = torch.where((i < before).unsqueeze(-1), i.unsqueeze(-1).expand(n, 3), picture)
    p = torch.where((i >= before + side * side).unsqueeze(-1), after, p)
    start = torch.randint(0, case["far"] + 1, (b, 1, 1), generator=g, device="cuda")
    return (p + start).contiguous()


# ----------------------------------------------------------------------------- the plain form


def _plain_tables(s):
    """cos and sin [batch or 1, tokens, pairs] of every token's angles, computed in 64 bits."""
    case, device = s["case"], s["q"].device
    axes = _axes(case)
    turned = None
    if s["positions"] is None:
        i = torch.arange(case["tokens"], device=device)
        v = i - (case["text"] if case["text_first"] else 0)
        turned = (v >= 0) & (v < case["t"] * case["h"] * case["w"])
        place = torch.stack((v // (case["h"] * case["w"]), v // case["w"] % case["h"], v % case["w"]), -1).unsqueeze(0)
    else:
        place = s["positions"]
    half = torch.cat([torch.arange(0, d, 2, device=device, dtype=torch.float64) / d for d in axes])
    if case["ladder"] == "shared":
        half = torch.arange(sum(axes) // 2, device=device, dtype=torch.float64) * 2 / sum(axes)
    axis = torch.cat([torch.full((d // 2,), a, device=device) for a, d in enumerate(axes)])
    angle = place.double()[..., axis] * THETA ** -half
    if turned is not None:
        angle = angle * turned.unsqueeze(-1)
    return angle.cos().float(), angle.sin().float()


def _plain_norm(x, kind, weight, bias):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    if weight is not None:
        x = x * weight.float()
    return x if bias is None else x + bias.float()


def _plain_turn(x, kind, weight, bias, cos, sin, case):
    y = x.float()
    if kind == "rms_across":
        y = y * torch.rsqrt(y.square().mean((1, 3), keepdim=True) + EPS)
        y = y * weight.float().view(1, x.shape[1], 1, x.shape[3])
    elif kind != "none":
        y = _plain_norm(y, kind, weight, bias)
    r = case["rotated"]
    cos, sin = cos.unsqueeze(1), sin.unsqueeze(1)
    if case["pairs"] == "interleaved":
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = y[..., : r // 2], y[..., r // 2 : r]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, y[..., r:]), -1).to(x.dtype)


def _run_plain(s):
    case = s["case"]
    if case["op"] == "rotate":
        cos, sin = _plain_tables(s)
        return (_plain_turn(s["q"], case["norm"], s["q_weight"], s["q_bias"], cos, sin, case),
                _plain_turn(s["k"], case["norm"], s["k_weight"], s["k_bias"], cos, sin, case))
    out = getattr(torch, case["out"])
    x = s["x"].float()
    if case["op"] == "gate":
        y = s["branch"].float()
        if case["branch_kind"] != "none":
            y = _plain_norm(y, case["branch_kind"], s["branch_weight"], None)
        x = x + s["gate"].float() * y
    h = _plain_norm(x, case["kind"], s["weight"], s["bias"])
    h = (h * (1 + s["scale"].float()) + s["shift"].float()).to(out)
    return h if case["op"] == "norm" else (x.to(s["x"].dtype), h)


def _run_own(s):
    import recap_b200

    case = s["case"]
    if case["op"] == "rotate":
        return recap_b200.rotate_qk(s["q"], s["k"], s["rotary"], query_norm=s["q_norm"], key_norm=s["k_norm"],
                                    positions=s["positions"])
    if case["op"] == "norm":
        return recap_b200.modulated_norm(s["x"], s["norm"], scale=s["scale"], shift=s["shift"],
                                         out_dtype=getattr(torch, case["out"]))
    return recap_b200.gated_residual(s["x"], s["branch"], s["gate"], branch_norm=s.get("branch_norm"), norm=s["norm"],
                                     scale=s["scale"], shift=s["shift"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------------- floor and truth


def _bytes_of(name):
    return 4 if name == "float32" else 2


def work(case):
    if case["op"] == "rotate":
        n = case["batch"] * case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        bytes_ = 2 * n * _bytes_of(case["dtype"])
        if not case["t"]:
            bytes_ += case["batch"] * case["tokens"] * 3 * 8
        return {"bytes": bytes_, "flops": n * (3 if case["norm"] == "none" else 6)}
    n = case["batch"] * case["tokens"] * case["width"]
    x, out = _bytes_of(case["dtype"]), _bytes_of(case["out"])
    mod = case["batch"] * (case["tokens"] if case["per_token"] else 1) * case["width"] * _bytes_of(case["mod"])
    if case["op"] == "norm":
        return {"bytes": n * (x + out) + 2 * mod, "flops": 6 * n}
    return {"bytes": n * (2 * x + 2 * out) + 3 * mod, "flops": n * (8 if case["branch_kind"] == "none" else 12)}


def _exact_rows(x, kind, weight, bias, dims):
    """A norm over ``dims`` from the mean and the population variance, in 64 bits."""
    if kind == "none":
        return x
    var, mean = torch.var_mean(x, dims, correction=0, keepdim=True)
    if kind == "layer":
        y = (x - mean) / torch.sqrt(var + EPS)
    else:
        y = x / torch.sqrt(var + mean * mean + EPS)
    if weight is not None:
        y = y * weight
    return y if bias is None else y + bias


def _exact_rotate(s):
    """The turn as a product of complex numbers."""
    case = s["case"]
    axes = _axes(case)
    pairs = sum(axes) // 2
    powers, which = [], []
    for a, d in enumerate(axes):
        for i in range(d // 2):
            at = 2 * len(powers) / (2 * pairs) if case["ladder"] == "shared" else 2 * i / d
            powers.append(THETA ** -at)
            which.append(a)
    freq = torch.tensor(powers, dtype=torch.float64, device="cuda")
    outs = []
    for x, weight, bias in ((s["q"], s["q_weight"], s["q_bias"]), (s["k"], s["k_weight"], s["k_bias"])):
        b, h, n, d = x.shape
        got = torch.empty(b, h, n, d, dtype=torch.float64, device="cuda")
        step = max(1, 40_000_000 // (b * h * d))  # tokens at a time, to bound the 64-bit temporaries
        for lo in range(0, n, step):
            hi = min(n, lo + step)
            y = x[:, :, lo:hi].double()
            if case["norm"] == "rms_across":
                y = _exact_rows(y, "rms", weight.double().view(h, 1, d), None, (1, 3))
            else:
                y = _exact_rows(y, case["norm"], None if weight is None else weight.double(),
                                None if bias is None else bias.double(), (3,))
            if s["positions"] is not None:
                place = s["positions"][:, lo:hi].double()
            else:
                first = case["text"] if case["text_first"] else 0
                v = torch.arange(lo, hi, device="cuda") - first
                inside = (v >= 0) & (v < case["t"] * case["h"] * case["w"])
                v = v.clamp(min=0)
                rest, col = torch.div(v, case["w"], rounding_mode="floor"), v.remainder(case["w"])
                place = torch.stack((torch.div(rest, case["h"], rounding_mode="floor"), rest.remainder(case["h"]), col))
                place = (place * inside).T.unsqueeze(0).double()
            angle = place[..., which] * freq  # [batch or 1, tokens, pairs]
            turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)
            r = 2 * pairs
            if case["pairs"] == "interleaved":
                z = torch.complex(y[..., 0:r:2].contiguous(), y[..., 1:r:2].contiguous()) * turn
                y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
            else:
                z = torch.complex(y[..., :pairs].contiguous(), y[..., pairs:r].contiguous()) * turn
                y[..., :pairs], y[..., pairs:r] = z.real, z.imag
            got[:, :, lo:hi] = y
        outs.append(got)
    return tuple(outs)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(s)
    d = lambda t: None if t is None else t.double()  # noqa: E731
    x = s["x"].double()
    if case["op"] == "gate":
        y = _exact_rows(s["branch"].double(), case["branch_kind"], d(s["branch_weight"]), None, (2,))
        x = torch.addcmul(x, s["gate"].double(), y)
    h = _exact_rows(x, case["kind"], d(s["weight"]), d(s["bias"]), (2,))
    h = torch.addcmul(h, h, s["scale"].double()) + s["shift"].double()
    return h if case["op"] == "norm" else (x, h)
