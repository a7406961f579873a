"""The operators around the attention (``rotate_qk``, ``modulated_norm``, ``gated_residual``) on the
GPU against plain implementations in 64 bits, and a block of them around ``Operator.attend``.

Tolerances count roundings, u = 2^-24 of fp32 and eps(t) of the output type:

* the output is rounded once: eps(t) / 2 of its value (2^-25 more where fp16 is subnormal);
* in fp32, with M = the largest |x| of the row times what the norm and weight scale it by: a sum over
  n values taken in registers, lanes and warps is off by at most k u M where k counts the additions one
  value passes through (13 for a row of up to 256 values: 8 in the thread, 5 over lanes; 53 for a row of
  channels: 32 in the thread, 5 lanes, 16 warps), the mean taken off adds one, the mean square is off by
  (k + 2) u relatively and by 2 u M sqrt(n) through the rounded differences, of which the root
  halves the former; rsqrt 2 u, the products with weight and bias 3 u, scale and shift 3 u, the turn 3 u for
  its products and sums and 4 u for sine and cosine (2 ulp of sincospif, and 2^-25 of half a turn from
  the angle's rounding), or 15 u where the output has 16 bits (__sincosf on [-pi, pi]: 2^-21.19, under 8 u;
  the angle in radians off by 2^-25 pi from its turns and 2^-24 pi / 2 from the product, under 4 u; the rest is slack).
  Added up: (13 + 1 + 8 + 2 + 3) = 27, + 2 sqrt(256), + 7 or 18 u for ``rotate_qk`` within one head,
  and 53 + 1 + 28 + 2 + 3 + 3 = 90, + 2 sqrt(n), for the rows."""

import math

import pytest
import torch

from recap_b200 import AxialRotary, Norm, gated_residual, modulated_norm, rotate_qk

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0**-24
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def check(got, want, fp32_error):
    """got within half a step of its type and ``fp32_error`` (64 bits, broadcasting) of want."""
    assert got.shape == want.shape
    eps = torch.finfo(got.dtype).eps
    least = 2.0**-25 if got.dtype == HF else 0.0
    tol = eps / 2 * (want.abs() + fp32_error) + fp32_error + least
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).max()):.3g} of the tolerance"


# ----------------------------------------------------------------------------- rotate_qk


def ref_norm64(x, norm, dims):
    """(normalised x, M): 64-bit norm over ``dims`` and the size its fp32 errors scale with."""
    if norm is None:
        return x, x.abs()
    mean = x.mean(dims, keepdim=True) if norm.kind == "layer" else torch.zeros_like(x[..., :1])
    y = x - mean
    r = 1 / torch.sqrt((y * y).mean(dims, keepdim=True) + norm.eps)
    y, big = y * r, x.abs().amax(dims, keepdim=True) * r
    if norm.weight is not None:
        w = norm.weight.double().reshape(x.shape[1], 1, x.shape[3]) if norm.across_heads else norm.weight.double()
        y, big = y * w, big * w.abs()
    if norm.bias is not None:
        y, big = y + norm.bias.double(), big + norm.bias.double().abs()
    return y, big.expand_as(y)


def ref_rotate64(x, norm, rotary, positions, first_token=0, out_dtype=None):
    """64-bit reference of one tensor [b, h, s, d]: (result, fp32 error bound)."""
    turn = 3 + (4 if (out_dtype or x.dtype) == F32 else 15)
    x = x.double()
    y, big = ref_norm64(x, norm, (1, 3) if norm is not None and norm.across_heads else (3,))
    n = x.shape[1] * x.shape[3] if norm is not None and norm.across_heads else x.shape[3]
    # across heads: up to 64 more additions in the thread and 32 over groups
    k = 0 if norm is None else 27 + (96 if norm.across_heads else 0) + 2 * math.sqrt(n)
    if rotary is None:
        return y, k * U * big
    b, h, s, d = x.shape
    if positions is None:
        v = torch.arange(first_token, first_token + s, device=x.device)
        v = v - (rotary.text_tokens if rotary.text_first else 0)
        inside = (v >= 0) & (v < math.prod(rotary.grid))
        axes, rest = [], v
        for g in reversed(rotary.grid):
            axes.insert(0, rest % g)
            rest = rest // g
        pos = torch.stack(axes, -1).unsqueeze(0)
    else:
        pos = positions if positions.dim() == 3 else positions.unsqueeze(0)
        inside = torch.ones(s, dtype=torch.bool, device=x.device)
    angle = []
    total = sum(rotary.axis_dims)
    for a, dims in enumerate(rotary.axis_dims):
        for i in range(dims // 2):
            p = len(angle)
            f = rotary_theta(rotary) ** -((2 * p / total) if rotary.ladder == "shared" else (2 * i / dims))
            angle.append(pos[..., a].double() * f)
    angle = torch.stack(angle, -1) * inside.view(1, s, 1)  # [b or 1, s, pairs]
    c, sn = angle.cos().unsqueeze(1), angle.sin().unsqueeze(1)
    p = total // 2
    i0 = slice(0, total, 2) if rotary.pairs == "interleaved" else slice(0, p)
    i1 = slice(1, total, 2) if rotary.pairs == "interleaved" else slice(p, total)
    y0, y1, m = y[..., i0].clone(), y[..., i1].clone(), big.clone()
    y[..., i0], y[..., i1] = y0 * c - y1 * sn, y0 * sn + y1 * c
    m[..., i0] = m[..., i1] = big[..., i0] + big[..., i1]
    return y, (k + turn) * U * m


def rotary_theta(rotary):
    return 10000.0


def make_qk(g, layout, b, hq, hk, s, d, dtype):
    n = lambda *sh: (torch.randn(*sh, generator=g, device=DEV) * 1.5 + 0.25).to(dtype)  # noqa: E731
    if layout == "packed":
        assert hq == hk
        qkv = n(b, s, 3, hq, d)
        return qkv[:, :, 0].transpose(1, 2), qkv[:, :, 1].transpose(1, 2)
    if layout == "token":
        return n(b, s, hq, d).transpose(1, 2), n(b, s, hk, d).transpose(1, 2)
    return n(b, hq, s, d), n(b, hk, s, d)


def make_norms(g, kind, hq, hk, d, dtype):
    if kind == "none":
        return None, None
    across = kind == "across"

    def one(h):
        w = (1 + 0.3 * torch.randn(h * d if across else d, generator=g, device=DEV)).to(dtype)
        bias = (0.2 * torch.randn(d, generator=g, device=DEV)).to(dtype) if kind == "layer" else None
        return Norm("layer" if kind == "layer" else "rms", w, bias, eps=1e-6, across_heads=across)

    return one(hq), one(hk)


def check_rotate(q, k, rotary, qn, kn, positions=None, first_token=0, **kw):
    got = rotate_qk(q, k, rotary, query_norm=qn, key_norm=kn, positions=positions, first_token=first_token, **kw)
    for y, x, n in ((got[0], q, qn), (got[1], k, kn)):
        if x is None:
            assert y is None
            continue
        check(y, *ref_rotate64(x, n, rotary, positions, first_token, y.dtype))
    return got


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("kind", ["none", "rms", "layer", "across"])
@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("layout,b,hq,hk,d,dims", [
    ("packed", 1, 3, 3, 128, (44, 42, 42)),
    ("token", 2, 5, 2, 64, (16, 24, 24)),
    ("head", 2, 7, 1, 88, (32, 24, 24)),   # 80 of 88 turned
    ("token", 1, 1, 1, 8, (8,)),
    ("head", 1, 17, 9, 256, (64, 64, 64, 64)),
    ("token", 1, 33, 33, 40, (16, 8, 8)),  # 32 of 40
])
def test_rotate_on_a_grid(dtype, kind, pairs, layout, b, hq, hk, d, dims):
    g = _gen(1)
    grid = (3, 4, 5, 2)[:len(dims)]
    text = 7
    rotary = AxialRotary(d, dims, grid=grid, text_tokens=text, text_first=b == 2, pairs=pairs)
    q, k = make_qk(g, layout, b, hq, hk, rotary.sequence_tokens, d, dtype)
    check_rotate(q, k, rotary, *make_norms(g, kind, hq, hk, d, dtype))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("kind", ["none", "rms", "layer", "across"])
@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("layout,b,hq,hk,d,dims", [
    ("packed", 1, 12, 12, 128, (48, 40, 40)), ("head", 2, 33, 7, 40, (8, 16, 16)), ("token", 1, 17, 3, 256, (64, 64, 64)),
    ("head", 1, 20, 20, 64, (16, 24, 24))])
def test_rotate_many_tokens(dtype, kind, pairs, layout, b, hq, hk, d, dims):
    """Enough tokens that a group takes all heads of a token, text and the last tokens inside a block."""
    g = _gen(19)
    rotary = AxialRotary(d, dims, grid=(5, 24, 40), text_tokens=9, text_first=b == 2, pairs=pairs)
    q, k = make_qk(g, layout, b, hq, hk, rotary.sequence_tokens, d, dtype)
    check_rotate(q, k, rotary, *make_norms(g, kind, hq, hk, d, dtype))


@pytest.mark.parametrize("s", [1, 2, 15, 16, 17, 127, 129, 4097])
@pytest.mark.parametrize("kind", ["rms", "across"])
@pytest.mark.parametrize("bits,far", [(torch.int32, 2**31 - 5000), (torch.int64, 2**45), (torch.int64, 3)])
def test_rotate_given_positions(s, kind, bits, far):
    """Positions of any size and sign, a batch of its own or shared; fp32, so that the angle counts.
    The reference's own 64-bit angle is off by 2^-52 of itself: far positions are compared by what
    they share with near ones (below), here up to 2^31 and, past it, by a position's 64-bit product taken apart."""
    g = _gen(2)
    rotary = AxialRotary(64, (24, 20, 20), ladder="shared", pairs="halves")
    q, k = make_qk(g, "token", 2, 4, 2, s, 64, F32)
    qn, kn = make_norms(g, kind, 4, 2, 64, F32)
    p = torch.randint(-50, 5000, (2, s, 3), generator=g, device=DEV)
    if far < 2**40:
        p = p + far if far > 3 else p
        if far > 2**20:
            # 2^31 rad is 2^-22 off in the reference: fold the turns exactly instead
            check_far(q, k, rotary, qn, kn, p.clamp(max=2**31 - 1).to(bits))
            return
        check_rotate(q, k, rotary, qn, kn, positions=p.to(bits))
        check_rotate(q, k, rotary, qn, kn, positions=p[0].to(bits))
        check_rotate(q, k, rotary, qn, kn, positions=p[:1].to(bits))
        wide = torch.zeros(2, s, 5, dtype=bits, device=DEV)
        wide[..., 1:4] = p.to(bits)
        check_rotate(q, k, rotary, qn, kn, positions=wide[..., 1:4])
    else:
        check_far(q, k, rotary, qn, kn, p + far)


def check_far(q, k, rotary, qn, kn, p):
    """Against angles taken from the definition in whole turns: position * frequency in Python's
    exact fractions, cut to 64-bit floats at the end."""
    from fractions import Fraction

    got = rotate_qk(q, k, rotary, query_norm=qn, key_norm=kn, positions=p)
    s = q.shape[2]
    rows = sorted({0, s // 2, s - 1})
    total = sum(rotary.axis_dims)
    for t, (x, n) in enumerate(((q, qn), (k, kn))):
        y, big = ref_norm64(x.double(), n, (1, 3) if n.across_heads else (3,))
        dims = x.shape[1] * x.shape[3] if n.across_heads else x.shape[3]
        kk = 27 + (96 if n.across_heads else 0) + 2 * math.sqrt(dims) + 7
        for b in range(2):
            for row in rows:
                ang, ax = [], 0
                for a, dims_a in enumerate(rotary.axis_dims):
                    for _ in range(dims_a // 2):
                        f = Fraction(10000.0 ** -(2 * ax / total) / (2 * math.pi))
                        turn = int(p[b, row, a]) * f
                        ang.append(float(turn - math.floor(turn)) * 2 * math.pi)
                        ax += 1
                ang = torch.tensor(ang, dtype=torch.float64, device=DEV)
                y0, y1 = y[b, :, row, :total // 2], y[b, :, row, total // 2:total]
                want = torch.cat((y0 * ang.cos() - y1 * ang.sin(), y0 * ang.sin() + y1 * ang.cos(),
                                  y[b, :, row, total:]), -1)
                m = big[b, :, row].clone()
                m[:, :total // 2] = m[:, total // 2:total] = m[:, :total // 2] + m[:, total // 2:total]
                # the frequency itself, rounded to 53 bits of a turn on both sides, cancels; the
                # kernel's is cut to 2^-64 of a turn: |p| 2^-65
                size = abs(p[b, row]).max().item() * 2.0**-64 * 2 * math.pi
                check(got[t][b, :, row], want, (kk * U + size) * m)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_unturned_values_pass_unchanged(dtype):
    """Without a norm, text tokens and values past the turned ones keep their values, beside
    infinities and NaN too; a NaN stays a NaN (its payload is not kept by the type conversions)."""
    g = _gen(3)
    for pairs in ("interleaved", "halves"):
        rotary = AxialRotary(128, (40, 32, 32), grid=(2, 3, 4), text_tokens=9, pairs=pairs)
        q, k = make_qk(g, "token", 1, 3, 3, 33, 128, dtype)
        q[0, 1, 30, 5], q[0, 1, 30, 6], q[0, 2, 31, 100] = math.inf, math.nan, -math.inf
        q[0, 0, 3, 104], q[0, 0, 3, 105] = math.inf, math.nan  # past the turned 104 values
        qo, ko = rotate_qk(q, k, rotary)
        assert torch.allclose(qo[:, :, 24:], q[:, :, 24:], rtol=0, atol=0, equal_nan=True)
        assert torch.equal(ko[..., 104:], k[..., 104:]) and torch.equal(ko[:, :, 24:], k[:, :, 24:])
        assert qo[0, 0, 3, 104] == math.inf and qo[0, 0, 3, 105].isnan()
        assert bool(qo[0, :, :24, :104].isfinite().all())


def test_position_zero_is_the_norm_alone():
    g = _gen(4)
    q, k = make_qk(g, "head", 1, 4, 4, 50, 64, BF)
    qn, kn = make_norms(g, "rms", 4, 4, 64, BF)
    zero = torch.zeros(50, 3, dtype=torch.int32, device=DEV)
    turned = rotate_qk(q, k, AxialRotary(64, (24, 20, 20)), query_norm=qn, key_norm=kn, positions=zero)
    plain = rotate_qk(q, k, query_norm=qn, key_norm=kn)
    assert torch.equal(turned[0], plain[0]) and torch.equal(turned[1], plain[1])
    check_rotate(q, k, None, qn, kn)
    check_rotate(q, None, None, qn, None)
    check_rotate(q, k, None, Norm("layer"), Norm("layer"))


def test_rotate_shards_equal_the_whole():
    """Chunks with first_token give the same bits as one call (text in the middle of a chunk)."""
    g = _gen(5)
    rotary = AxialRotary(128, (44, 42, 42), grid=(3, 7, 11), text_tokens=13, text_first=True)
    s = rotary.sequence_tokens
    q, k = make_qk(g, "packed", 1, 4, 4, s, 128, BF)
    qn, kn = make_norms(g, "across", 4, 4, 128, BF)
    whole = rotate_qk(q, k, rotary, query_norm=qn, key_norm=kn)
    for step in (1, 61, 100):
        for lo in range(0, s, step):
            hi = min(s, lo + step)
            part = rotate_qk(q[:, :, lo:hi], k[:, :, lo:hi], rotary, query_norm=qn, key_norm=kn, first_token=lo)
            assert torch.equal(part[0], whole[0][:, :, lo:hi]) and torch.equal(part[1], whole[1][:, :, lo:hi])


@pytest.mark.parametrize("kind", ["rms", "across"])
def test_rotate_in_place_and_into_views(kind):
    g = _gen(6)
    rotary = AxialRotary(64, (16, 24, 24), grid=(2, 5, 7))
    q, k = make_qk(g, "packed", 2, 3, 3, 70, 64, BF)
    qn, kn = make_norms(g, kind, 3, 3, 64, BF)
    want = rotate_qk(q, k, rotary, query_norm=qn, key_norm=kn)
    # rows of a longer joint sequence: what stands before and behind stays
    joint = torch.full((2, 2, 3, 90, 64), 7.0, dtype=BF, device=DEV)
    rotate_qk(q, k, rotary, query_norm=qn, key_norm=kn, out=(joint[0][:, :, 11:81], joint[1][:, :, 11:81]))
    assert torch.equal(joint[0][:, :, 11:81], want[0]) and torch.equal(joint[1][:, :, 11:81], want[1])
    assert bool((joint[:, :, :, :11] == 7).all()) and bool((joint[:, :, :, 81:] == 7).all())
    v = q.clone()
    base = q._base if q._base is not None else q
    third = base[:, :, 2].clone() if base.dim() == 5 else None
    got = rotate_qk(q, k, rotary, query_norm=qn, key_norm=kn, out=(q, k))
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1]) and not torch.equal(q, v)
    if third is not None:
        assert torch.equal(base[:, :, 2], third)


def test_written_outputs_count_as_changed():
    """Autograd sees that a given tensor was written: a graph that saved it refuses its backward pass."""
    g = _gen(23)
    x = torch.randn(1, 4, 64, generator=g, device=DEV)
    w = torch.randn(64, generator=g, device=DEV, requires_grad=True)
    for write in (lambda t: modulated_norm(t, Norm("rms"), out=t),
                  lambda t: gated_residual(t, t.clone(), out=(t, None)),
                  lambda t: rotate_qk(t.view(1, 1, 4, 64), None, query_norm=Norm("rms"), out=(t.view(1, 1, 4, 64), None))):
        t = x.clone()
        loss = (t * w).sum()
        before = t._version
        write(t)
        assert t._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        t = x.clone()
        modulated_norm(t, Norm("rms"), out=t)


@pytest.mark.parametrize("dtype", [HF, F32])
def test_rotate_to_bf16(dtype):
    g = _gen(7)
    rotary = AxialRotary(64, (16, 24, 24), grid=(2, 5, 7))
    q, k = make_qk(g, "token", 1, 3, 3, 70, 64, dtype)
    qn, kn = make_norms(g, "layer", 3, 3, 64, F32)
    got = check_rotate(q, k, rotary, qn, kn, out_dtype=BF)
    assert got[0].dtype == BF and got[0].stride() == q.stride()


def test_rotate_expanded_inputs_and_same_tensor_twice():
    g = _gen(8)
    rotary = AxialRotary(64, (16, 24, 24), grid=(2, 5, 7))
    q = torch.randn(1, 1, 70, 64, generator=g, device=DEV).to(BF).expand(2, 3, 70, 64)
    check_rotate(q, q, rotary, None, None)


@pytest.mark.parametrize("d,heads", [(64, 256), (128, 128), (256, 64), (128, 40), (64, 31)])
def test_rotate_across_many_heads(d, heads):
    g = _gen(9)
    rotary = AxialRotary(d, (d // 2, d // 4, d // 4), grid=(1, 2, 3))
    for dtype in (BF, F32):
        q, k = make_qk(g, "token", 1, heads, 3, 6, d, dtype)
        check_rotate(q, k, rotary, *make_norms(g, "across", heads, 3, d, dtype))


@pytest.mark.parametrize("tokens", [3, 5000])
def test_rotate_norms_without_weight_or_with_bias_only(tokens):
    g = _gen(20)
    rotary = AxialRotary(64, (24, 20, 20), grid=(1, 1, tokens))
    for dtype in (BF, F32):
        q, k = make_qk(g, "token", 1, 6, 2, tokens, 64, dtype)
        bias = torch.randn(64, generator=g, device=DEV)
        w = 1 + 0.2 * torch.randn(6 * 64, generator=g, device=DEV)
        check_rotate(q, k, rotary, Norm("rms"), Norm("rms"))
        check_rotate(q, k, rotary, Norm("layer", None, bias), Norm("layer", None, bias))
        check_rotate(q, k, rotary, Norm("layer", bias), Norm("layer"))
        check_rotate(q, k, rotary, Norm("rms", across_heads=True), Norm("rms", across_heads=True))
        check_rotate(q, k, rotary, Norm("rms", w, across_heads=True), Norm("rms", across_heads=True))
        check_rotate(q, k, rotary, Norm("rms", across_heads=True, eps=0.3), Norm("rms", w[:128], across_heads=True))
        check_rotate(q, None, rotary, Norm("rms", w, across_heads=True), None)


def test_rotate_constant_and_zero_rows():
    """A row of equal values has a layer norm of about zero, a row of zeros an rms norm of zero: the epsilon
    keeps both finite."""
    q = torch.full((1, 2, 4, 64), 3.0, dtype=BF, device=DEV)
    got, _ = rotate_qk(q, None, query_norm=Norm("layer"))
    assert bool((got.abs() <= 0.05).all())  # 3 * 13 u rounded mean over sqrt(eps): 0.0023
    for n in (Norm("rms"), Norm("rms", across_heads=True)):
        assert bool((rotate_qk(torch.zeros_like(q), None, query_norm=n)[0] == 0).all())


@pytest.mark.parametrize("b,s", [(3000, 1), (700, 3), (420, 5)])
def test_many_short_samples(b, s):
    g = _gen(21)
    x, y = rows(g, F32, b, s, 264), rows(g, BF, b, s, 264)
    norm = row_norm(g, "layer", 264, F32)
    gate, scale = (0.4 * torch.randn(b, 1, 264, generator=g, device=DEV) for _ in range(2))
    got_x, got_h = gated_residual(x, y, gate, norm=norm, scale=scale)
    want = x.double() + gate.double() * y.double()
    err = 2 * U * (want.abs() + (want - x.double()).abs())
    check(got_x, want, err)
    check(got_h, *ref_modulated(want, norm, scale, None, err))


def test_rotate_empty():
    rotary = AxialRotary(64, (16, 24, 24), grid=(2, 5, 7))
    q = torch.empty(0, 3, 70, 64, dtype=BF, device=DEV)
    assert rotate_qk(q, q, rotary)[1].shape == q.shape
    q = torch.empty(1, 3, 0, 64, dtype=BF, device=DEV)
    assert rotate_qk(q, None, rotary)[0].shape == q.shape


def test_misaligned_rows_are_refused():
    x = torch.zeros(1, 2, 8, 66, dtype=BF, device=DEV)
    with pytest.raises(ValueError):
        rotate_qk(x[..., :64], None)
    with pytest.raises(ValueError):
        rotate_qk(torch.zeros(1025, dtype=BF, device=DEV)[1:].view(1, 2, 8, 64), None)
    with pytest.raises(ValueError):
        modulated_norm(x[0, 0, :, :64], Norm("rms"))
    one = torch.zeros(1, 1, 3, 66, dtype=BF, device=DEV)[:, :, :1, :64]  # one row: its strides do not count
    rotate_qk(one, None)


# ----------------------------------------------------------------------------- norm rows


def ref_rows(x, norm):
    """(norm(x) weight + bias in 64 bits, M)."""
    return ref_norm64(x, norm, (-1,))


def ref_modulated(x, norm, scale, shift, x_error):
    """Modulated norm of x in 64 bits; x itself is off by x_error (fp32) in the kernel."""
    y, big = ref_rows(x, norm)
    n = x.shape[-1]
    k = 87 + 2 * math.sqrt(n)
    err = k * U * big
    if x_error is not None:
        # an error e of x moves the norm by e r |w| and, through the statistics, by no more than
        # twice that of the largest in the row
        mean = x.mean(-1, keepdim=True) if norm.kind == "layer" else 0.0
        r = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + norm.eps)
        w = norm.weight.double().abs() if norm.weight is not None else 1.0
        err = err + x_error.amax(-1, keepdim=True) * r * w * (2 + y.abs().amax(-1, keepdim=True))
    s = 1 + scale.double() if scale is not None else torch.ones((), dtype=torch.float64, device=x.device)
    t = shift.double() if shift is not None else torch.zeros((), dtype=torch.float64, device=x.device)
    # y (1 + s) + t: the product as y s + y, three roundings
    return y * s + t, err * (1 + (s - 1).abs()) + 3 * U * (y.abs() * (1 + (s - 1).abs()) + t.abs())


def rows(g, dtype, *shape):
    x = torch.randn(*shape, generator=g, device=DEV) * torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=DEV))
    x[..., :2] *= 20
    return (x + 0.3).to(dtype)


def row_norm(g, kind, c, dtype, affine=True):
    w = (1 + 0.2 * torch.randn(c, generator=g, device=DEV)).to(dtype) if affine else None
    b = (0.1 * torch.randn(c, generator=g, device=DEV)).to(dtype) if affine and kind == "layer" else None
    return Norm(kind, w, b, eps=1e-6)


PAIRS = [(BF, BF), (HF, HF), (F32, F32), (F32, BF), (F32, HF)]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("xt,ht", PAIRS)
@pytest.mark.parametrize("b,s,c", [(1, 1, 8), (2, 3, 256), (1, 130, 264), (3, 7, 1352), (1, 5, 1536), (2, 2, 5120),
                                   (1, 3, 8192), (1, 2, 8200), (1, 2, 16384), (1, 1, 10008)])
def test_modulated_norm(kind, xt, ht, b, s, c):
    g = _gen(10)
    x = rows(g, xt, b, s, c)
    norm = row_norm(g, kind, c, xt, affine=c != 1536)
    for shape, mt in [(None, None), ((c,), ht), ((b, 1, c), F32), ((b, s, c), ht), ((1, s, c), BF)]:
        scale = shift = None
        if shape is not None:
            scale = (0.3 * torch.randn(*shape, generator=g, device=DEV)).to(mt)
            shift = (0.3 * torch.randn(*shape, generator=g, device=DEV)).to(mt)
        got = modulated_norm(x, norm, scale=scale, shift=shift, out_dtype=ht)
        assert got.dtype == ht
        check(got, *ref_modulated(x.double(), norm, scale, shift, None))
    check(modulated_norm(x, norm, scale=scale, out_dtype=ht), *ref_modulated(x.double(), norm, scale, None, None))
    check(modulated_norm(x, norm, shift=shift, out_dtype=ht), *ref_modulated(x.double(), norm, None, shift, None))
    check(modulated_norm(x[0], norm, scale=scale[0], shift=shift[0, :1], out_dtype=ht),
          *ref_modulated(x[0].double(), norm, scale[0], shift[0, :1], None))


@pytest.mark.parametrize("kind", ["none", "rms", "layer"])
@pytest.mark.parametrize("branch_kind", ["none", "rms", "layer"])
@pytest.mark.parametrize("xt,ht", PAIRS)
@pytest.mark.parametrize("b,s,c", [(1, 1, 8), (2, 9, 1920), (1, 33, 5120), (3, 5, 1352), (1, 2, 16384)])
def test_gated_residual(kind, branch_kind, xt, ht, b, s, c):
    g = _gen(11)
    x, y = rows(g, xt, b, s, c), rows(g, ht, b, s, c)
    norm = row_norm(g, kind, c, xt) if kind != "none" else None
    bnorm = row_norm(g, branch_kind, c, ht) if branch_kind != "none" else None
    for shape, mt in [(None, None), ((b, 1, c), F32), ((b, s, c), ht)]:
        gate = scale = shift = None
        if shape is not None:
            gate = (0.5 * torch.randn(*shape, generator=g, device=DEV)).to(mt)
            if norm is not None:
                scale, shift = ((0.3 * torch.randn(*shape, generator=g, device=DEV)).to(mt) for _ in range(2))
        got_x, got_h = gated_residual(x, y, gate, branch_norm=bnorm, norm=norm, scale=scale, shift=shift)
        yy, err = y.double(), torch.zeros((), dtype=torch.float64, device=DEV)
        if bnorm is not None:
            yy, big = ref_rows(yy, bnorm)
            err = (87 + 2 * math.sqrt(c)) * U * big
        gg = gate.double() if gate is not None else torch.ones((), dtype=torch.float64, device=DEV)
        want = x.double() + gg * yy
        err = err * gg.abs() + 2 * U * ((gg * yy).abs() + want.abs())
        assert got_x.dtype == xt
        check(got_x, want, err)
        if norm is None:
            assert got_h is None
        else:
            assert got_h.dtype == ht
            check(got_h, *ref_modulated(want, norm, scale, shift, err))


@pytest.mark.parametrize("xt,ht", PAIRS)
@pytest.mark.parametrize("c", [8, 264, 1352, 3080, 4096, 5120, 8192, 10008])
def test_many_rows(xt, ht, c):
    """Enough tokens for blocks of several, with a rest in each sample (701 = 4 * 175 + 1), modulations shared,
    of a sample, of a token in each type; what each call gives a row does not depend on its neighbours."""
    g = _gen(18)
    b, s = 3, 701
    x, y = rows(g, xt, b, s, c), rows(g, ht, b, s, c)
    norm, bnorm = row_norm(g, "layer", c, xt), row_norm(g, "rms", c, ht)
    for shape, mt in [((c,), ht), ((b, 1, c), F32), ((b, s, c), ht), ((b, s, c), F32), ((1, s, c), BF)]:
        gate, scale, shift = ((0.4 * torch.randn(*shape, generator=g, device=DEV)).to(mt) for _ in range(3))
        check(modulated_norm(x, norm, scale=scale, shift=shift, out_dtype=ht),
              *ref_modulated(x.double(), norm, scale, shift, None))
        got_x, got_h = gated_residual(x, y, gate, branch_norm=bnorm, norm=norm, scale=scale, shift=shift)
        yy, big = ref_rows(y.double(), bnorm)
        want = x.double() + gate.double() * yy
        err = (87 + 2 * math.sqrt(c)) * U * big * gate.double().abs() + 2 * U * ((gate.double() * yy).abs() + want.abs())
        check(got_x, want, err)
        check(got_h, *ref_modulated(want, norm, scale, shift, err))
        # few rows take blocks of one token: the same bits
        part = [t if t.dim() == 1 else t[1:2, 5:6] if t.shape[1] > 1 and t.shape[0] > 1 else
                t[:, 5:6] if t.shape[1] > 1 else t[1:2] for t in (gate, scale, shift)]
        one_x, one_h = gated_residual(x[1:2, 5:6], y[1:2, 5:6], part[0], branch_norm=bnorm, norm=norm, scale=part[1],
                                      shift=part[2])
        assert torch.equal(one_x, got_x[1:2, 5:6]) and torch.equal(one_h, got_h[1:2, 5:6])


@pytest.mark.parametrize("xt,ht", PAIRS)
@pytest.mark.parametrize("c", [768, 2568, 2816, 4104, 6144])
def test_rows_of_whole_blocks(xt, ht, c):
    """Rows that fill their threads' columns and rows that do not, at the widths where a block takes more tokens."""
    test_many_rows(xt, ht, c)


@pytest.mark.parametrize("captured", [False, True])
def test_modulations_written_by_the_call_before(captured):
    """Calls that follow one another without a gap: what one writes into the modulations, the next reads, also where
    the one before has read them on every multiprocessor.  The same calls, waited for one by one, give the bits."""
    g = _gen(31)
    c, n = 5120, 24
    x, y = rows(g, F32, 1, 4096, c), rows(g, BF, 1, 4096, c)
    sources = torch.randn(n, 1, 1, c, generator=g, device=DEV)
    q = rows(g, BF, 1, 2048, 8 * 64).view(1, 2048, 8, 64).transpose(1, 2)
    norm, rms = Norm("layer"), Norm("rms")
    m = torch.zeros(1, 1, c, device=DEV)
    w = m.view(-1)[:64]
    head = Norm("rms", w)

    def run(wait):
        got = []
        for i in range(n):
            modulated_norm(sources[i], rms, out=m)
            wait()
            _, h = gated_residual(x, y, m, norm=norm, scale=m, shift=m)
            wait()
            turned, _ = rotate_qk(q, None, query_norm=head)
            wait()
            got += [h[:, ::97, ::13].clone(), turned[:, :, ::61].clone()]
            wait()
        return got

    want = run(torch.cuda.synchronize)
    for _ in range(3):
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = run(lambda: None)
            graph.replay()
        else:
            got = run(lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert not torch.equal(want[0], want[2])


def test_rows_in_place_and_views():
    g = _gen(12)
    c = 384
    x, y = rows(g, F32, 2, 40, c), rows(g, BF, 2, 40, c)
    norm = row_norm(g, "layer", c, F32)
    mods = (0.3 * torch.randn(2, 6, c, generator=g, device=DEV)).chunk(6, 1)  # views of one projection
    want = gated_residual(x, y, mods[2], norm=norm, scale=mods[3], shift=mods[4])
    h1 = modulated_norm(x, norm, scale=mods[0], shift=mods[1])
    # rows inside a longer joint buffer: the rows around stay
    joint = torch.full((2, 60, c), 5.0, device=DEV)
    hj = torch.full((2, 60, c), 5.0, device=DEV, dtype=BF)
    joint[:, 10:50], hj[:, 10:50] = x, y
    got = gated_residual(joint[:, 10:50], hj[:, 10:50], mods[2], norm=norm, scale=mods[3], shift=mods[4],
                         out=(joint[:, 10:50], hj[:, 10:50]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for t in (joint, hj):
        assert bool((t[:, :10] == 5).all()) and bool((t[:, 50:] == 5).all())
    wide = torch.zeros(2, 40, 2 * c, device=DEV)
    modulated_norm(x, norm, scale=mods[0], shift=mods[1], out=wide[..., c:])
    assert torch.equal(wide[..., c:], h1) and bool((wide[..., :c] == 0).all())
    modulated_norm(x, norm, scale=mods[0], shift=mods[1], out=x)
    assert torch.equal(x, h1)


def test_rows_keep_to_their_own_row():
    """A NaN or infinite row spoils itself alone; a row of equal values has a finite layer norm."""
    g = _gen(13)
    x = rows(g, BF, 1, 9, 1536)
    norm = Norm("layer")
    clean = modulated_norm(x, norm)
    x[0, 3, 7], x[0, 5, 9] = math.nan, math.inf
    x[0, 7] = 3.0
    got = modulated_norm(x, norm)
    same = [0, 1, 2, 4, 6, 8]
    assert torch.equal(got[0, same], clean[0, same])
    assert bool(got[0, 3].isnan().all()) and bool(got[0, 5].isnan().any())
    assert bool((got[0, 7].abs() <= 1e-3).all())  # the mean of equal values, rounded: within 53 u * 3 * 1e3


def test_empty_rows():
    x = torch.empty(2, 0, 64, device=DEV)
    assert modulated_norm(x, Norm("rms")).shape == x.shape
    s, h = gated_residual(x, x, norm=Norm("rms"))
    assert s.shape == h.shape == x.shape


# ----------------------------------------------------------------------------- streams, graphs


def test_streams_and_graphs():
    """Another stream than the default; two graphs captured and replayed over new inputs in turn."""
    g = _gen(14)
    rotary = AxialRotary(128, (44, 42, 42), grid=(2, 9, 11))
    q, k = make_qk(g, "packed", 1, 6, 6, 198, 128, BF)
    qn, kn = make_norms(g, "across", 6, 6, 128, BF)
    x, y = rows(g, F32, 1, 198, 768), rows(g, BF, 1, 198, 768)
    gate = torch.randn(1, 1, 768, generator=g, device=DEV)
    norm = row_norm(g, "rms", 768, F32)

    def run():
        return (*rotate_qk(q, k, rotary, query_norm=qn, key_norm=kn), *gated_residual(x, y, gate, norm=norm, scale=gate))

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    for seed in (20, 21):
        h = _gen(seed)
        q.copy_(torch.randn(q.shape, generator=h, device=DEV))
        x.copy_(torch.randn(x.shape, generator=h, device=DEV))
        want = run()
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("s,c", [(3, 512), (700, 512), (9000, 1536)])
def test_calls_that_follow_one_another(s, c):
    """A chain of calls, each on what the one before wrote and some in place, torch kernels between them, queued
    without waiting: the bits of the same chain with a wait after every call."""
    g = _gen(22)
    heads = c // 64
    rotary = AxialRotary(64, (16, 24, 24), grid=(1, 1, s))
    x0, gate = rows(g, F32, 1, s, c), 0.1 * torch.randn(1, 1, c, generator=g, device=DEV)
    norm, qn = row_norm(g, "layer", c, F32), Norm("rms", across_heads=True)

    def chain(wait):
        x = x0.clone()
        for i in range(12):
            h = modulated_norm(x, norm, scale=gate, out_dtype=BF)
            wait()
            q = h.view(1, s, heads, 64).transpose(1, 2)
            if i % 3 == 0:
                h.mul_(0.5)
                wait()
            q, _ = rotate_qk(q, None, rotary, query_norm=qn, out=(q, None) if i % 2 else None)
            wait()
            x, y = gated_residual(x, q.transpose(1, 2).reshape(1, s, c), gate, norm=norm, out=(x, None))
            wait()
            x = x + y.float() if i % 4 == 1 else x
            wait()
        return x

    want = chain(torch.cuda.synchronize)
    for _ in range(5):
        assert torch.equal(chain(lambda: None), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(lambda: None)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_long_rows_pass_32_bit_offsets():
    """A view whose later rows lie past 2^31 elements of its buffer."""
    g = _gen(15)
    pitch, s = 2**24, 200  # elements between tokens: the last lies at 3.3e9
    buf = torch.empty(pitch * (s - 1) + 256, dtype=BF, device=DEV)
    q = buf.as_strided((1, 2, s, 128), (pitch * s, 128, pitch, 1))
    q.copy_(torch.randn(1, 2, s, 128, generator=g, device=DEV))
    rotary = AxialRotary(128, (44, 42, 42), grid=(2, 10, 10))
    out, _ = rotate_qk(q, None, rotary, out=(torch.empty(1, 2, s, 128, dtype=BF, device=DEV), None))
    check(out, *ref_rotate64(q, None, rotary, None))
    rotate_qk(q, None, rotary, out=(q, None))
    assert torch.equal(q, out)
    x = buf.as_strided((1, s, 256), (pitch * s, pitch, 1))
    got = modulated_norm(x, Norm("rms"), out=torch.empty(1, s, 256, dtype=BF, device=DEV))
    check(got, *ref_modulated(x.double(), Norm("rms"), None, None, None))


# ----------------------------------------------------------------------------- a block of them


@pytest.mark.parametrize("d,text_first", [(128, False), (64, True)])
def test_attend_with_rotary_is_rotate_then_attend(d, text_first):
    from recap_b200 import REFRESH, SPARSE, Operator, OperatorConfig
    from recap_b200.sparse import Layout, SparseGeometry, hilbert_permutation

    g = _gen(16)
    grid, text = (4, 12, 16), 40
    layout = Layout.from_permutation(hilbert_permutation(grid), text_tokens=text, text_first=text_first)
    rotary = AxialRotary(d, (d - 4 * (d // 6), 2 * (d // 6), 2 * (d // 6)), grid=grid, text_tokens=text,
                         text_first=text_first)
    ops = [Operator.build(OperatorConfig(head_density=0.25), SparseGeometry.build(layout, 128), n_layers=1)
           for _ in range(2)]
    for step, kind in enumerate(("exact", REFRESH, SPARSE, REFRESH, SPARSE)):
        for dtype in (BF, F32):
            q, k = make_qk(g, "packed", 1, 4, 4, rotary.sequence_tokens, d, dtype)
            v = torch.randn(q.shape, generator=g, device=DEV).to(dtype)
            qn, kn = make_norms(g, "rms", 4, 4, d, dtype)
            for op in ops:
                op.begin_step(step, kind)
            got = ops[0].attend(0, q, k, v, rotary=rotary, query_norm=qn, key_norm=kn)
            qr, kr = rotate_qk(q, k, rotary, query_norm=qn, key_norm=kn, out_dtype=BF)
            want = ops[1].attend(0, qr, kr, v.to(BF))
            assert got.dtype == dtype and torch.equal(got.to(BF), want)
    for op in ops:
        op.check_device_status()


def test_block_around_exact_attention():
    """norm -> projections -> rotate_qk -> attend -> projection -> gate, residual and next norm, as a
    block uses them, against the same in 64 bits.  Between the operators stand library products in
    bf16 and the attention in bf16, each of whose outputs is off by eps/2 of itself and by what its bf16 inputs
    were: with some ten such roundings, independent and of 2^-9 rms each, the branch is off by
    about sqrt(10) 2^-9 = 0.6 % rms; 2 % is asked of it, and of the sum what 2 % of the branch make."""
    from recap_b200 import EXACT, Operator, OperatorConfig
    from recap_b200.sparse import Layout, SparseGeometry, hilbert_permutation

    g = _gen(17)
    grid, text, heads, d = (3, 10, 12), 24, 4, 64
    c, s = heads * d, 3 * 10 * 12 + 24
    layout = Layout.from_permutation(hilbert_permutation(grid), text_tokens=text, text_first=False)
    rotary = AxialRotary(d, (16, 24, 24), grid=grid, text_tokens=text)
    op = Operator.build(OperatorConfig(), SparseGeometry.build(layout, 128), n_layers=1)
    op.begin_step(0, EXACT)
    x = torch.randn(1, s, c, generator=g, device=DEV)
    w_qkv = (torch.randn(c, 3 * c, generator=g, device=DEV) / math.sqrt(c)).to(BF)
    w_o = (torch.randn(c, c, generator=g, device=DEV) / math.sqrt(c)).to(BF)
    mods = (0.3 * torch.randn(1, 5, c, generator=g, device=DEV)).chunk(5, 1)
    qn, kn = make_norms(g, "rms", heads, heads, d, BF)
    norm = Norm("layer")
    with torch.no_grad():
        h = modulated_norm(x, norm, scale=mods[0], shift=mods[1], out_dtype=BF)
        qkv = (h @ w_qkv).view(1, s, 3, heads, d)
        q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
        o = op.attend(0, q, k, v, rotary=rotary, query_norm=qn, key_norm=kn)
        y = o.transpose(1, 2).reshape(1, s, c) @ w_o
        got_x, got_h = gated_residual(x, y, mods[2], norm=norm, scale=mods[3], shift=mods[4])
    op.check_device_status()
    h, _ = ref_modulated(x.double(), norm, mods[0], mods[1], None)
    qkv = (h @ w_qkv.double()).view(1, s, 3, heads, d)
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    q, k = ref_rotate64(q, qn, rotary, None)[0], ref_rotate64(k, kn, rotary, None)[0]
    o = torch.softmax(q @ k.transpose(-1, -2) / math.sqrt(d), -1) @ v
    y = o.transpose(1, 2).reshape(1, s, c) @ w_o.double()
    want_x = x.double() + mods[2].double() * y
    want_h, _ = ref_modulated(want_x, norm, mods[3], mods[4], None)
    branch = (mods[2].double() * y).norm()
    assert float((got_x.double() - want_x).norm() / branch) < 0.02
    # the norm divides by the sum's own size and its bf16 output adds 2^-9 rms
    assert float((got_h.double() - want_h).norm() / want_h.norm()) < 0.02 * float(branch / want_x.norm()) * 2 + 2.0**-8
