"""Host side of the operators around the attention: the angles of ``AxialRotary`` against
64-bit arithmetic, and the refusals of every entry point (no GPU)."""

import math
import struct

import pytest
import torch

from recap_b200 import AxialRotary, Norm, _lib, gated_residual, modulated_norm, rotate_qk


def _angle(r: AxialRotary, p: int, position: int) -> float:
    """Angle of pair p at an integer position, as the kernel forms it: 64 wrapping bits, the top
    32 as a signed fraction of half a turn."""
    t = (position * r._struct.turns[p] + r._struct.phase[p]) % 2**64
    top = t >> 32
    return math.pi * (top - 2**32 if top >= 2**31 else top) * 2.0**-31


@pytest.mark.parametrize("ladder", ["axis", "shared"])
@pytest.mark.parametrize("scale,start", [(1.0, 0.0), ((0.5, 1.25, -1.0), (0.0, -7.5, 3.0))])
def test_angles_follow_the_definition(ladder, scale, start):
    dims = (16, 24, 24)
    r = AxialRotary(64, dims, theta=256.0, ladder=ladder, scale=scale, start=start)
    scales = (scale,) * 3 if isinstance(scale, float) else scale
    starts = (start,) * 3 if isinstance(start, float) else start
    p = 0
    for axis, d in enumerate(dims):
        for i in range(d // 2):
            f = 256.0 ** -((2 * p / 64) if ladder == "shared" else (2 * i / d))
            assert r._struct.axis[p] == axis
            for n in (0, 1, 79, 100003, -5):
                want = (n * scales[axis] + starts[axis]) * f
                # the top 32 bits cut 2^-32 of a turn; 64-bit floats of the reference: n * 2^-52
                err = math.remainder(_angle(r, p, n) - want, 2 * math.pi)
                assert abs(err) <= 2 * math.pi * 2.0**-32 + 4 * abs(want) * 2.0**-52 + 1e-15
            p += 1
    assert r._struct.pairs == p == 32


def test_far_positions_wrap_exactly():
    """A position of 2^40 + n turns the slowest pairs by the same step as n."""
    r = AxialRotary(128, (128,))
    for p in (0, 5, 63):
        step = _angle(r, p, 2**40 + 1) - _angle(r, p, 2**40)
        near = _angle(r, p, 1) - _angle(r, p, 0)
        assert abs(math.remainder(step - near, 2 * math.pi)) <= 4 * math.pi * 2.0**-32


def test_grid_of_a_layout():
    r = AxialRotary(128, (44, 42, 42), grid=(3, 4, 5), text_tokens=7, text_first=True)
    assert r.sequence_tokens == 67 and r._struct.video_offset == 7 and r._struct.video_tokens == 60
    assert list(r._struct.grid)[:3] == [3, 4, 5] and r._struct.axes == 3


def test_copies_of_a_rotary_stand_alone():
    """A copied or unpickled rotary has a struct of its own: it outlives the one it came from."""
    import copy
    import ctypes
    import pickle

    r = AxialRotary(96, (32, 24, 24), theta=(1e4, 500.0, 256.0), grid=(2, 3, 4), text_tokens=5, text_first=True,
                    pairs="halves", scale=(1.0, 0.5, 2.0), start=(0.0, -1.5, 3.0))
    copies = [copy.copy(r), copy.deepcopy(r), pickle.loads(pickle.dumps(r))]
    image = bytes(r._struct)
    for c in copies:
        assert bytes(c._struct) == image and c._spec[0] == ctypes.addressof(c._struct) != r._spec[0]
        assert c._spec[1:] == r._spec[1:] and (c.grid, c.axis_dims, c.sequence_tokens) == (r.grid, r.axis_dims, 29)


@pytest.mark.parametrize("bad", [
    dict(axis_dims=()), dict(axis_dims=(2,) * 5), dict(axis_dims=(15, 16)), dict(axis_dims=(0, 16)),
    dict(axis_dims=(64, 66)), dict(head_dim=68, axis_dims=(64,)), dict(head_dim=264, axis_dims=(64,)),
    dict(pairs="quarters"), dict(ladder="rope"), dict(pairs="halves", axis_dims=(30, 32)), dict(theta=0.0),
    dict(theta=(1e4, 1e4)), dict(theta=(1e4, 1e4, 5e3), ladder="shared"), dict(scale=float("nan")),
    dict(start=(0.0,)), dict(grid=(3, 4)), dict(grid=(3, 0, 4)), dict(grid=(2048, 2048, 512)), dict(text_tokens=5),
    dict(text_first=True), dict(grid=(2, 2, 2), text_tokens=-1),
])
def test_rotary_refuses(bad):
    args = dict(head_dim=128, axis_dims=(44, 42, 42))
    args.update(bad)
    with pytest.raises(ValueError):
        AxialRotary(args.pop("head_dim"), args.pop("axis_dims"), **args)


@pytest.mark.parametrize("bad", [dict(kind="batch"), dict(kind="rms", bias=torch.zeros(8)),
                                 dict(kind="layer", across_heads=True), dict(kind="rms", eps=-1.0),
                                 dict(kind="rms", eps=float("inf")), dict(kind="rms", eps=float("nan"))])
def test_norm_refuses(bad):
    with pytest.raises(ValueError):
        Norm(**bad)


def _q(b=1, h=2, s=5, d=64, dtype=torch.bfloat16):
    return torch.zeros(b, h, s, d, dtype=dtype)


GRID = dict(axis_dims=(16, 24, 24), grid=(1, 1, 5))


@pytest.mark.parametrize("call", [
    lambda: rotate_qk(_q()[0], _q()[0]),
    lambda: rotate_qk(_q(), _q(s=6)),
    lambda: rotate_qk(_q(), _q(d=72)),
    lambda: rotate_qk(_q(), _q(b=2)),
    lambda: rotate_qk(_q(), _q(h=0)),
    lambda: rotate_qk(_q(h=0), None),
    lambda: rotate_qk(_q(), _q(dtype=torch.float16)),
    lambda: rotate_qk(_q(dtype=torch.float64), None),
    lambda: rotate_qk(_q(d=60), None),
    lambda: rotate_qk(_q(d=264), None),
    lambda: rotate_qk(_q().transpose(2, 3), None),
    lambda: rotate_qk(_q(), _q(), out_dtype=torch.float16),
    lambda: rotate_qk(_q(), _q(), query_norm=Norm("rms")),
    lambda: rotate_qk(_q(), _q(), key_norm=Norm("rms")),
    lambda: rotate_qk(_q(), _q(), query_norm=Norm("rms"), key_norm=Norm("layer")),
    lambda: rotate_qk(_q(), _q(), query_norm=Norm("rms", torch.ones(32)), key_norm=Norm("rms")),
    lambda: rotate_qk(_q(), _q(), query_norm=Norm("rms", torch.ones(128)[::2]), key_norm=Norm("rms")),
    lambda: rotate_qk(_q(), _q(), query_norm=Norm("rms", torch.ones(64)),
                      key_norm=Norm("rms", torch.ones(64, dtype=torch.bfloat16))),
    lambda: rotate_qk(_q(), _q(), query_norm=Norm("layer", torch.ones(64), torch.ones(64, dtype=torch.float16)),
                      key_norm=Norm("layer")),
    lambda: rotate_qk(_q(h=257), None, query_norm=Norm("rms", across_heads=True)),
    lambda: rotate_qk(_q(), _q(), AxialRotary(128, (128,), grid=(5,))),
    lambda: rotate_qk(_q(s=6), None, AxialRotary(64, **GRID)),
    lambda: rotate_qk(_q(s=4), None, AxialRotary(64, **GRID), first_token=2),
    lambda: rotate_qk(_q(s=4), None, AxialRotary(64, **GRID), first_token=-1),
    lambda: rotate_qk(_q(), None, AxialRotary(64, **GRID), positions=torch.zeros(5, 3, dtype=torch.int32)),
    lambda: rotate_qk(_q(), None, AxialRotary(64, (16, 24))),
    lambda: rotate_qk(_q(), None, AxialRotary(64, (16, 24)), positions=torch.zeros(5, 3, dtype=torch.int32)),
    lambda: rotate_qk(_q(), None, AxialRotary(64, (16, 24)), positions=torch.zeros(5, 2)),
    lambda: rotate_qk(_q(), None, AxialRotary(64, (16, 24)), positions=torch.zeros(2, 5, 2, dtype=torch.int64)),
    lambda: rotate_qk(_q(), None, AxialRotary(64, (16, 24)), positions=torch.zeros(5, 2, dtype=torch.int32),
                      first_token=1),
    lambda: rotate_qk(_q(), None, positions=torch.zeros(5, 3, dtype=torch.int32)),
    lambda: rotate_qk(_q(), None, first_token=1),
    lambda: rotate_qk(_q(), None, out=(_q(s=6), None)),
    lambda: rotate_qk(_q(), None, out=(_q(dtype=torch.float16), None)),
    lambda: rotate_qk(_q(), _q(), out=(_q(), _q(dtype=torch.float16))),
    lambda: rotate_qk(_q(), _q(), out=(_q(), None)),
    lambda: rotate_qk(_q(), None, out=(torch.zeros(1, 1, 5, 64, dtype=torch.bfloat16).expand(1, 2, 5, 64), None)),
    lambda: rotate_qk(_q(), _q()),  # not on a GPU
])
def test_rotate_qk_refuses(call):
    with pytest.raises(ValueError):
        call()


def test_rotate_qk_refuses_overlapping_outputs():
    q, k = _q(), _q()
    with pytest.raises(ValueError, match="overlap"):  # the outputs of each other's inputs
        rotate_qk(q, k, out=(k, q))
    with pytest.raises(ValueError, match="overlap"):  # one tensor turned twice in place
        rotate_qk(q, q, out=(q, q))
    with pytest.raises(ValueError, match="overlap"):
        out = _q()
        rotate_qk(q, k, out=(out, out))
    wide = torch.zeros(1, 2, 6, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):  # shifted by a row
        rotate_qk(wide[:, :, :5], None, out=(wide[:, :, 1:], None))
    # the views of one packed projection do not overlap: only the missing GPU is refused
    qkv = torch.zeros(2, 5, 3, 2, 64, dtype=torch.bfloat16)
    q, k = qkv[:, :, 0].transpose(1, 2), qkv[:, :, 1].transpose(1, 2)
    with pytest.raises(ValueError, match="CUDA"):
        rotate_qk(q, k, out=(q, k))


def _x(*shape, dtype=torch.bfloat16):
    return torch.zeros(*(shape or (2, 3, 16)), dtype=dtype)


@pytest.mark.parametrize("call", [
    lambda: modulated_norm(_x(16), Norm("rms")),
    lambda: modulated_norm(_x(1, 2, 3, 16), Norm("rms")),
    lambda: modulated_norm(_x(3, 12), Norm("rms")),
    lambda: modulated_norm(_x(1, 16392), Norm("rms")),
    lambda: modulated_norm(_x(3, 0), Norm("rms")),
    lambda: modulated_norm(_x(dtype=torch.float64), Norm("rms")),
    lambda: modulated_norm(_x(), Norm("rms"), out_dtype=torch.float32),
    lambda: modulated_norm(_x(), Norm("rms"), out_dtype=torch.float16),
    lambda: modulated_norm(_x(2, 16, 3).transpose(1, 2), Norm("rms")),
    lambda: modulated_norm(_x(), Norm("rms", across_heads=True)),
    lambda: modulated_norm(_x(), Norm("rms", torch.ones(8))),
    lambda: modulated_norm(_x(), Norm("rms"), scale=_x(2, 16)),
    lambda: modulated_norm(_x(), Norm("rms"), scale=_x(3, 1, 16)),
    lambda: modulated_norm(_x(), Norm("rms"), scale=_x(2, 2, 16)),
    lambda: modulated_norm(_x(), Norm("rms"), scale=_x(8)),
    lambda: modulated_norm(_x(), Norm("rms"), scale=_x(1)),
    lambda: modulated_norm(_x(), Norm("rms"), scale=_x(32)[::2]),
    lambda: modulated_norm(_x(), Norm("rms"), scale=_x(16), shift=_x(16, dtype=torch.float32)),
    lambda: modulated_norm(_x(), Norm("rms"), scale=_x(16, dtype=torch.float64)),
    lambda: modulated_norm(_x(), Norm("rms"), out=_x(2, 4, 16)),
    lambda: modulated_norm(_x(), Norm("rms"), out=_x(1, 1, 16).expand(2, 3, 16)),
    lambda: modulated_norm(_x(), Norm("rms")),  # not on a GPU
    lambda: gated_residual(_x(), _x(2, 3, 24)),
    lambda: gated_residual(_x(), _x(3, 16)),
    lambda: gated_residual(_x(), _x(dtype=torch.float32)),
    lambda: gated_residual(_x(), _x(), scale=_x(16)),
    lambda: gated_residual(_x(), _x(), shift=_x(16)),
    lambda: gated_residual(_x(), _x(), out=(None, _x())),
    lambda: gated_residual(_x(), _x(), norm=Norm("rms"), out=(_x(dtype=torch.float32), None)),
    lambda: gated_residual(_x(dtype=torch.float32), _x(), norm=Norm("rms"), out=(None, _x(dtype=torch.float32))),
    lambda: gated_residual(_x(), _x(), branch_norm=Norm("rms", across_heads=True)),
    lambda: gated_residual(_x(), _x()),  # not on a GPU
])
def test_norm_rows_refuse(call):
    with pytest.raises(ValueError):
        call()


def test_norm_rows_refuse_overlapping_outputs():
    r, y, g = _x(), _x(), _x()
    n = Norm("rms")
    for out in [(y, None), (None, r), (r, r), (y, r), (g, None), (None, g)]:
        with pytest.raises(ValueError, match="overlap"):
            gated_residual(r, y, g, norm=n, out=out)
    for out in [(r, y), (r, None), (None, y), (_x(), _x())]:  # in place, or apart
        with pytest.raises(ValueError, match="CUDA"):
            gated_residual(r, y, g, norm=n, out=out)
    x = _x(4, 16)
    with pytest.raises(ValueError, match="overlap"):
        modulated_norm(x[:3], n, out=x[1:])


def test_gradients_are_refused_not_cut():
    w = torch.ones(64, requires_grad=True)
    q = _q().requires_grad_()
    for call in (lambda: rotate_qk(q, None), lambda: rotate_qk(_q(), None, query_norm=Norm("rms", w)),
                 lambda: modulated_norm(_x(3, 64), Norm("rms", w)),
                 lambda: modulated_norm(_x(3, 64), Norm("rms"), scale=w),
                 lambda: gated_residual(_x(3, 64), _x(3, 64).requires_grad_())):
        with pytest.raises(RuntimeError, match="no_grad"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            call()


def test_attend_with_rotary_still_refuses_cpu_tensors():
    from recap_b200 import Operator, OperatorConfig
    from recap_b200.sparse import Layout, SparseGeometry

    layout = Layout.from_permutation(torch.arange(5), text_tokens=0, text_first=False)
    op = Operator.build(OperatorConfig(), SparseGeometry.build(layout, 128), n_layers=1)
    with pytest.raises(ValueError, match="CUDA"):
        op.attend(0, _q(), _q(), _q(), rotary=AxialRotary(64, **GRID))


def _rotate_args(**kw):
    """Packed recap_rotate_qk_args of a valid call on made-up addresses (never launched)."""
    v = dict(q=4096, k=8192, qo=4096, ko=8192, strides=[640, 320, 64] * 4, positions=0, ps=[0, 0, 0], first=0, qw=0, qb=0,
             kw=0, kb=0, batch=1, hq=2, hk=2, S=5, D=64, it=0, ot=0, norm=0, wt=0, bits=0)
    v.update(kw)
    return struct.Struct("<4Q12qQ3qq4Q10i2f").pack(
        v["q"], v["k"], v["qo"], v["ko"], *v["strides"], v["positions"], *v["ps"], v["first"], v["qw"], v["qb"], v["kw"],
        v["kb"], v["batch"], v["hq"], v["hk"], v["S"], v["D"], v["it"], v["ot"], v["norm"], v["wt"], v["bits"], 1e-6, 1e-6)


def test_c_abi_rejects_before_any_device_call():
    lib = _lib.load()
    shape, unsupported = _lib.RECAP_ERR_SHAPE, _lib.RECAP_ERR_UNSUPPORTED
    on_grid, on_positions = AxialRotary(64, **GRID), AxialRotary(64, (16, 24))
    rotary, given = on_grid._spec[0], on_positions._spec[0]

    def rotate(rot=None, **kw):
        return lib.recap_rotate_qk(_rotate_args(**kw), rot, None)

    assert lib.recap_rotate_qk(None, None, None) == shape
    for kw in (dict(D=60), dict(D=264), dict(D=0), dict(hq=0), dict(hk=-1), dict(batch=-1), dict(S=-1), dict(norm=4),
               dict(norm=-1), dict(it=3), dict(wt=3), dict(q=4100), dict(ko=8200), dict(q=0), dict(qw=4),
               dict(strides=[640, 320, 63] + [640, 320, 64] * 3), dict(strides=[640, 320, 64] * 3 + [640, 324, 64])):
        assert rotate(**kw) == shape, kw
    assert rotate(ot=1) == unsupported
    assert rotate(norm=3, hq=257) == unsupported
    assert rotate(given) == shape  # no positions
    assert rotate(given, bits=16, positions=4096) == shape
    assert rotate(given, bits=64, positions=4100) == shape
    assert rotate(given, bits=32) == shape
    assert rotate(rotary, D=32) == shape  # more turned values than the head has
    # a call on nothing launches nothing
    assert rotate(rotary, S=0) == _lib.RECAP_OK and rotate(rotary, batch=0, q=0) == _lib.RECAP_OK

    def norm(**kw):
        v = dict(x=4096, branch=0, xo=0, h=4096, strides=[64, 16] * 4, mods=[0, 0, 0], ms=[0] * 6, w=[0] * 4, b=1, S=3, C=16,
                 xt=0, ht=0, norm=1, bn=0, wt=0, bwt=0, mt=0)
        v.update(kw)
        return lib.recap_norm_rows(struct.Struct("<4Q8q3Q6q4Q10i2f").pack(
            v["x"], v["branch"], v["xo"], v["h"], *v["strides"], *v["mods"], *v["ms"], *v["w"], v["b"], v["S"], v["C"],
            v["xt"], v["ht"], v["norm"], v["bn"], v["wt"], v["bwt"], v["mt"], 1e-6, 1e-6), None)

    assert lib.recap_norm_rows(None, None) == shape
    for kw in (dict(C=12), dict(C=0), dict(b=-1), dict(S=-1), dict(xt=3), dict(ht=-1), dict(norm=3), dict(bn=3),
               dict(norm=0), dict(x=4104), dict(h=0), dict(branch=4096), dict(strides=[64, 12] + [64, 16] * 3),
               dict(mods=[4104, 0, 0]), dict(mods=[0, 4096, 0], ms=[0, 0, 0, 12, 0, 0]), dict(w=[8, 0, 0, 0]),
               dict(b=65536, S=65536), dict(mt=3), dict(wt=3), dict(bwt=-1)):
        assert norm(**kw) == shape, kw
    assert norm(C=16392) == unsupported and norm(ht=2) == unsupported
    assert norm(S=0) == _lib.RECAP_OK and norm(b=0, x=0) == _lib.RECAP_OK


def test_packed_projections_apart():
    """The overlap test on views of one buffer: packed heads, chunks of tokens, batches."""
    apart = _lib.native().apart
    qkv = torch.zeros(2, 6, 3, 4, 16)
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    assert apart(q, k) and apart(k, q) and apart(q, v) and apart(v, k)
    assert not apart(q, q) and not apart(q, qkv[:, :, 0, 1:].transpose(1, 2))
    assert apart(qkv[0], qkv[1]) and not apart(q, qkv)
    head_major = torch.zeros(2, 4, 6, 16)
    assert not apart(head_major[:, :, :4], head_major[:, :, 2:])
    assert apart(head_major[:, :, :4], head_major[:, :, 4:]) and apart(head_major[:, :, 4:], head_major[:, :, :4])
    assert apart(head_major[:, :2], head_major[:, 2:]) and not apart(head_major[:, :3], head_major[:, 2:])
    joint = torch.zeros(3, 10, 8)
    assert apart(joint[:, :4], joint[:, 4:]) and not apart(joint[:, :5], joint[:, 4:])
    assert apart(joint[..., :4], joint[..., 4:]) and not apart(joint[..., :5], joint[..., 4:])
    assert not apart(joint[:1].expand(3, 10, 8), joint)
    # against the elements themselves, over all pairs of boxes of a small grid
    base = torch.arange(3 * 4 * 5).view(3, 4, 5)
    boxes = [base[a:b, c:d, e:f] for a, b in ((0, 2), (1, 3), (2, 3)) for c, d in ((0, 2), (2, 4), (1, 4))
             for e, f in ((0, 5), (0, 2), (2, 5), (1, 3))]
    for x in boxes:
        for y in boxes:
            assert apart(x, y) == (not set(x.flatten().tolist()) & set(y.flatten().tolist()))
    assert apart(torch.zeros(0, 4, 6, 16), head_major)
