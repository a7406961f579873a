"""Forms of the operators around the attention beside the common ones: thetas, scales and starts of each axis, turned
values that end inside a lane's eight, streams that join right before a call.  Tolerances as in test_gpu_block_ops; a start adds
2^-32 of a turn, 0.03 u, to an angle's 3.6 u of the 4 u counted there."""

import math

import pytest
import torch
from test_gpu_block_ops import BF, DEV, F32, HF, U, _gen, check, make_norms, make_qk, ref_norm64, row_norm, rows

from recap_b200 import AxialRotary, Norm, gated_residual, modulated_norm, rotate_qk

pytestmark = pytest.mark.gpu


def ref_turn64(x, norm, dims, pos, inside, out_dtype, pairs="interleaved", ladder="axis", theta=1e4, scale=1.0, start=0.0):
    """64-bit reference of one tensor [b, h, s, d] at positions [b or 1, s, axes] and the fp32 error bound."""
    each = lambda v: v if isinstance(v, tuple) else (v,) * len(dims)  # noqa: E731
    theta, scale, start = each(theta), each(scale), each(start)
    x = x.double()
    across = norm is not None and norm.across_heads
    y, big = ref_norm64(x, norm, (1, 3) if across else (3,))
    n = x.shape[1] * x.shape[3] if across else x.shape[3]
    k = 0 if norm is None else 27 + (96 if across else 0) + 2 * math.sqrt(n)
    total, angle = sum(dims), []
    for a, d in enumerate(dims):
        for i in range(d // 2):
            f = theta[a] ** -(2 * len(angle) / total if ladder == "shared" else 2 * i / d)
            angle.append((pos[..., a].double() * scale[a] + start[a]) * f)
    angle = torch.stack(angle, -1) * inside.view(1, -1, 1)
    c, sn = angle.cos().unsqueeze(1), angle.sin().unsqueeze(1)
    i0, i1 = (slice(0, total, 2), slice(1, total, 2)) if pairs == "interleaved" else \
        (slice(0, total // 2), slice(total // 2, total))
    y0, y1, m = y[..., i0].clone(), y[..., i1].clone(), big.clone()
    y[..., i0], y[..., i1] = y0 * c - y1 * sn, y0 * sn + y1 * c
    m[..., i0] = m[..., i1] = big[..., i0] + big[..., i1]
    return y, (k + 3 + (4 if out_dtype == F32 else 15)) * U * m


def grid_positions(grid, text, text_first):
    pos = torch.stack(torch.meshgrid(*(torch.arange(g) for g in grid), indexing="ij"), -1).view(1, -1, len(grid)).to(DEV)
    blank = torch.zeros(1, text, len(grid), dtype=pos.dtype, device=DEV)
    inside = torch.ones(pos.shape[1], device=DEV), torch.zeros(text, device=DEV)
    return (torch.cat((blank, pos), 1), torch.cat((inside[1], inside[0]))) if text_first else \
        (torch.cat((pos, blank), 1), torch.cat(inside))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind", ["none", "rms", "layer", "across"])
@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("how", [
    dict(theta=(1e4, 500.0, 256.0)), dict(scale=(0.5, 1.25, -1.0)), dict(start=(0.0, -7.5, 3.25)),
    dict(theta=100.0, scale=-0.3, start=11.0, ladder="shared"),
    dict(theta=(1e6, 1.5, 10000.0), scale=(2.0, -0.125, 1e-3), start=(-100.0, 0.3, 1e-3)),
])
def test_theta_scale_and_start(dtype, kind, pairs, how):
    g = _gen(41)
    dims, grid, text = (16, 24, 16), (3, 7, 11), 6
    q, k = make_qk(g, "token", 1, 4, 2, 231 + text, 64, dtype)
    qn, kn = make_norms(g, kind, 4, 2, 64, dtype)
    for text_first in (False, True):
        pos, inside = grid_positions(grid, text, text_first)
        rotary = AxialRotary(64, dims, grid=grid, text_tokens=text, text_first=text_first, pairs=pairs, **how)
        got = rotate_qk(q, k, rotary, query_norm=qn, key_norm=kn)
        for y, x, n in ((got[0], q, qn), (got[1], k, kn)):
            check(y, *ref_turn64(x, n, dims, pos, inside, dtype, pairs, **how))
    pos = torch.randint(-3000, 3000, (1, q.shape[2], 3), generator=g, device=DEV)
    inside = torch.ones(q.shape[2], device=DEV)
    for bits in (torch.int32, torch.int64):
        got = rotate_qk(q, k, AxialRotary(64, dims, pairs=pairs, **how), query_norm=qn, key_norm=kn, positions=pos.to(bits))
        for y, x, n in ((got[0], q, qn), (got[1], k, kn)):
            check(y, *ref_turn64(x, n, dims, pos, inside, dtype, pairs, **how))


# interleaved pairs end anywhere: 5, 18, 63 and 3 pairs, in lanes of four
PARTS = [(16, (10,)), (40, (12, 14, 10)), (128, (44, 42, 40)), (64, (2, 2, 2)), (256, (62, 62, 62, 64))]


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("kind", ["none", "rms", "layer", "across"])
@pytest.mark.parametrize("d,dims", PARTS)
def test_turned_values_that_end_inside_a_lane(dtype, kind, d, dims):
    g = _gen(42)
    grid, text = (3, 5, 4, 2)[:len(dims)], 3
    rotary = AxialRotary(d, dims, grid=grid, text_tokens=text)
    q, k = make_qk(g, "token", 2, 5, 3, rotary.sequence_tokens, d, dtype)
    qn, kn = make_norms(g, kind, 5, 3, d, dtype)
    pos, inside = grid_positions(grid, text, False)
    got = rotate_qk(q, k, rotary, query_norm=qn, key_norm=kn)
    for y, x, n in ((got[0], q, qn), (got[1], k, kn)):
        check(y, *ref_turn64(x, n, dims, pos, inside, dtype))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("d,dims", PARTS)
@pytest.mark.parametrize("odd", [math.inf, -math.inf, math.nan])
def test_an_infinity_beside_the_last_turned_pair_stays_there(dtype, d, dims, odd):
    g = _gen(43)
    total, s = sum(dims), 37
    q, _ = make_qk(g, "head", 1, 3, 1, s, d, dtype)
    pos = torch.randint(1, 900, (1, s, len(dims)), generator=g, device=DEV)
    q[0, 1, 5, total], q[0, 2, 6, total + 1], q[0, 0, 7, d - 1] = odd, odd, odd
    got, _ = rotate_qk(q, None, AxialRotary(d, dims), positions=pos)
    assert torch.allclose(got[..., total:], q[..., total:], rtol=0, atol=0, equal_nan=True)
    plain = q.clone()
    plain[..., total:] = 0
    want, err = ref_turn64(plain, None, dims, pos, torch.ones(s, device=DEV), dtype)
    check(got[..., :total], want[..., :total], err[..., :total])


@pytest.mark.parametrize("captured", [False, True])
def test_streams_that_join_right_before_a_call(captured):
    """A side stream, kept busy, writes what the next calls on the main stream read: modulations, rows, a norm's weight; and
    reads what they wrote.  The same calls, waited for one by one, give the bits."""
    g = _gen(44)
    c, n = 4096, 12
    x, y = rows(g, F32, 1, 2048, c), rows(g, BF, 1, 2048, c)
    sources = torch.randn(n, 1, 1, c, generator=g, device=DEV)
    q0 = rows(g, BF, 1, 2048, 8 * 64).view(1, 2048, 8, 64).transpose(1, 2)
    work = rows(g, F32, 1, 8192, c)
    norm, rms = Norm("layer"), Norm("rms")
    bnorm = row_norm(g, "rms", c, BF)
    m = torch.zeros(1, 1, c, device=DEV)
    head = Norm("rms", m.view(-1)[:64])
    branch, q = torch.empty_like(y), torch.empty_like(q0)
    side = torch.cuda.Stream()

    def run(wait):
        main = torch.cuda.current_stream()
        got = []
        for i in range(n):
            side.wait_stream(main)
            with torch.cuda.stream(side):
                modulated_norm(work, norm, out=work)  # keeps it busy
                wait()
                modulated_norm(sources[i], rms, out=m)
                wait()
                modulated_norm(y, bnorm, scale=m, out=branch)
                wait()
                q.copy_(q0).mul_(1.0 / (i + 1))
                wait()
            main.wait_stream(side)
            _, h = gated_residual(x, branch, m, norm=norm, scale=m, shift=m)
            wait()
            turned, _ = rotate_qk(q, None, query_norm=head, out=(q, None))
            wait()
            side.wait_stream(main)
            with torch.cuda.stream(side):
                _, again = gated_residual(x, h, norm=norm, out=(None, h))
                wait()
            main.wait_stream(side)
            got += [again[:, ::97, ::13].clone(), turned[:, :, ::61].clone()]
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


def test_outputs_beside_the_input_in_another_order_and_in_place_through_another_view():
    g = _gen(45)
    w = torch.zeros(2, 2, 40 * 6 * 64, dtype=BF, device=DEV)
    q = w[:, 0].view(2, 40, 6, 64).transpose(1, 2)
    q.copy_(torch.randn(q.shape, generator=g, device=DEV))
    rotary = AxialRotary(64, (16, 24, 24), grid=(2, 4, 5))
    qn = Norm("layer")
    want, _ = rotate_qk(q, None, rotary, query_norm=qn)
    out = w[:, 1].view(2, 6, 40, 64)
    before = q.clone()
    rotate_qk(q, None, rotary, query_norm=qn, out=(out, None))
    assert torch.equal(out, want) and torch.equal(q, before)
    one = q[:1]
    rotate_qk(one, None, rotary, query_norm=qn, out=(one.as_strided(one.shape, (8, *one.stride()[1:]), one.storage_offset()), None))
    assert torch.equal(one, want[:1]) and torch.equal(q[1:], before[1:])


@pytest.mark.parametrize("text_first", [False, True])
def test_text_with_norms_of_its_own(text_first):
    """Text and video projected and normalised apart, each turned into its part of the joint queries and keys."""
    g = _gen(46)
    grid, text, heads, d = (3, 5, 7), 11, 4, 64
    video = math.prod(grid)
    dims = (16, 24, 24)
    parts = {"video": video, "text": text}
    qk = {n: [torch.randn(1, s, heads, d, generator=g, device=DEV).to(BF).transpose(1, 2) for _ in range(2)]
          for n, s in parts.items()}
    norms = {n: make_norms(g, "rms", heads, heads, d, BF) for n in parts}
    q, k = (torch.empty(1, video + text, heads, d, dtype=BF, device=DEV).transpose(1, 2) for _ in range(2))
    at = {"text": slice(0, text), "video": slice(text, None)} if text_first else \
        {"video": slice(0, video), "text": slice(video, None)}
    for n, rotary in (("video", AxialRotary(d, dims, grid=grid)), ("text", None)):
        rotate_qk(*qk[n], rotary, query_norm=norms[n][0], key_norm=norms[n][1], out=(q[:, :, at[n]], k[:, :, at[n]]))
    pos, inside = grid_positions(grid, 0, False)
    for i, joint in enumerate((q, k)):
        check(joint[:, :, at["video"]], *ref_turn64(qk["video"][i], norms["video"][i], dims, pos, inside, BF))
        y, big = ref_norm64(qk["text"][i].double(), norms["text"][i], (3,))
        check(joint[:, :, at["text"]], y, (27 + 2 * math.sqrt(d)) * U * big)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("s,c", [(3, 64), (2501, 64), (2501, 1352), (2100, 3080), (2050, 4104), (2050, 5120), (2048, 8200),
                                 (1, 16384), (2048, 16384)])
def test_one_tensor_in_several_places_written_in_place(dtype, s, c):
    """The calls that are taken though an input stands in two places and is replaced: the bits of the same calls on copies."""
    g = _gen(47)
    norm = row_norm(g, "layer", c, dtype)
    r0, y0 = rows(g, dtype, 1, s, c), (0.3 * torch.randn(1, s, c, generator=g, device=DEV)).to(dtype)

    def both(call):
        want = call(r0.clone(), r0.clone(), y0.clone(), y0.clone(), lambda *t: None)
        r, y = r0.clone(), y0.clone()
        got = call(r, r, y, y, lambda *t: t)
        assert all(torch.equal(a, b) for a, b in zip(got, want) if a is not None)

    both(lambda r, r2, y, y2, out: gated_residual(r, r2, r2, norm=norm, out=out(r, None)))
    both(lambda r, r2, y, y2, out: gated_residual(r, y, y2, norm=norm, scale=y2, shift=y2, out=out(r, y)))
    both(lambda r, r2, y, y2, out: gated_residual(r, y, norm=norm, scale=y2, shift=y2, out=out(None, y)))
    both(lambda r, r2, y, y2, out: (modulated_norm(y, norm, scale=y2, shift=y2, out=(out(y) or (None,))[0]),))
