"""Arguments of the operators around the attention that have to be refused, or told apart, before any device
call (no GPU): outputs that overlap, missing operands, foreign types."""

import random

import pytest
import torch

from recap_b200 import (AxialRotary, HostBankOperator, Norm, Operator, OperatorConfig, _lib, gated_residual,
                        modulated_norm, rotate_qk)
from recap_b200.sparse import Layout, SparseGeometry

CUDA_ONLY = "CUDA tensors only"  # what a call that is right but for its device meets


def _elements(t):
    at = torch.tensor(t.storage_offset())
    for n, step in zip(t.shape, t.stride()):
        at = at.unsqueeze(-1) + torch.arange(n) * step
    return set(at.flatten().tolist())


def test_apart_never_says_so_of_tensors_that_share_an_element():
    """Pairs of views of one buffer with strides of their own, against the elements themselves."""
    apart = _lib.native().apart
    rng = random.Random(5)
    buf = torch.zeros(4096)
    told = met = 0
    for _ in range(30000):
        n = rng.randint(1, 4)
        shape = [rng.randint(1, 4) for _ in range(n)]
        other = shape if rng.random() < 0.7 else [rng.randint(1, 4) for _ in range(n)]
        steps = rng.sample([1, 2, 3, 4, 6, 8, 12, 16, 24, 48, 64, 96], n)
        mixed = [s if rng.random() < 0.8 else rng.choice(steps + [0, 1, 8, 32]) for s in steps]
        x = buf.as_strided(shape, steps, rng.randint(0, 100))
        y = buf.as_strided(other, mixed, rng.randint(0, 100))
        meet = bool(_elements(x) & _elements(y))
        said = apart(x, y)
        assert not (said and meet), (x.shape, x.stride(), x.storage_offset(), y.shape, y.stride(), y.storage_offset())
        told += said
        met += meet
    assert told > 4000 and met > 4000  # the draw reaches both


def test_apart_of_other_orders_within():
    """The halves of each sample, one in token order and one in head order: apart, though their inner strides differ."""
    apart = _lib.native().apart
    w = torch.zeros(3, 2, 6 * 4 * 16)
    x = w[:, 0].view(3, 6, 4, 16).transpose(1, 2)
    y = w[:, 1].view(3, 4, 6, 16)
    assert apart(x, y) and apart(y, x)
    assert not apart(w[:, 0].view(3, 4, 6, 16), x)


def test_output_in_another_order_over_the_input_is_refused():
    w = torch.zeros(2, 6, 32)
    x, out = w[:, :, :16], w[1].view(6, 2, 16).transpose(0, 1)
    with pytest.raises(ValueError, match="overlap"):
        modulated_norm(x, Norm("rms"), out=out)
    with pytest.raises(ValueError, match=CUDA_ONLY):
        modulated_norm(x, Norm("rms"), out=w[:, :, 16:])


@pytest.mark.parametrize("strides", [(96, 8, 1), (8, 16, 1), (80, 16, 1), (0, 16, 1), (96, 0, 1)])
def test_output_that_holds_an_element_twice_is_refused(strides):
    out = torch.zeros(1024).as_strided((2, 6, 16), strides)
    with pytest.raises(ValueError, match="twice"):
        modulated_norm(torch.zeros(2, 6, 16), Norm("rms"), out=out)
    q = torch.zeros(1, 2, 6, 16)
    with pytest.raises(ValueError, match="twice"):
        rotate_qk(q, None, out=(out.unsqueeze(0), None))


@pytest.mark.parametrize("strides", [(96, 16, 1), (16, 32, 1), (1000, 64, 1), (16, 48, 1)])
def test_output_in_any_order_without_a_second_place_is_taken(strides):
    out = torch.zeros(4096).as_strided((2, 6, 16), strides)
    with pytest.raises(ValueError, match=CUDA_ONLY):
        modulated_norm(torch.zeros(2, 6, 16), Norm("rms"), out=out)


def test_outputs_over_parameters_or_positions_are_refused():
    """Blocks read a norm's weight and bias, and the positions, without waiting for one another's rows."""
    x, w = torch.zeros(2, 3, 16), torch.ones(16)
    calls = [
        lambda: modulated_norm(x, Norm("rms", x[0, 0]), out=x),
        lambda: modulated_norm(x, Norm("layer", w, x[1, 2]), out=x),
        lambda: modulated_norm(torch.zeros(1, 1, 16), Norm("rms", w), out=w.view(1, 1, 16)),
        lambda: gated_residual(x, torch.zeros(2, 3, 16), norm=Norm("rms", x[0, 1]), out=(x, None)),
        lambda: gated_residual(x, torch.zeros(2, 3, 16), branch_norm=Norm("layer", w, x[0, 1]), out=(x, None)),
    ]
    q, k = torch.zeros(1, 2, 5, 16), torch.zeros(1, 2, 5, 16)
    calls += [
        lambda: rotate_qk(q, k, query_norm=Norm("rms", q[0, 0, 0]), key_norm=Norm("rms"), out=(q, k)),
        lambda: rotate_qk(q, k, query_norm=Norm("rms", k[0, 0, 0]), key_norm=Norm("rms"), out=(q, k)),
        lambda: rotate_qk(q, k, query_norm=Norm("layer"), key_norm=Norm("layer", None, q[0, 1, 4]), out=(q, k)),
    ]
    flat = torch.zeros(160, dtype=torch.int32)
    rows = flat.view(torch.float32).view(1, 2, 5, 16)
    calls.append(lambda: rotate_qk(q, None, AxialRotary(16, (8,)), positions=flat[:5].view(5, 1), out=(rows, None)))
    for call in calls:
        with pytest.raises(ValueError, match="overlap"):
            call()
    with pytest.raises(ValueError, match=CUDA_ONLY):
        rotate_qk(q, k, AxialRotary(16, (8,)), positions=flat[:5].view(5, 1), query_norm=Norm("rms", w),
                  key_norm=Norm("rms", w), out=(q, k))


def test_in_place_through_another_view_of_one_sample():
    """The stride of a dim of one element says nothing about where the elements lie."""
    joint = torch.zeros(1, 60, 16)
    x = joint[:, 10:50]
    out = x.as_strided(x.shape, (8 * 16, 16, 1), x.storage_offset())
    with pytest.raises(ValueError, match=CUDA_ONLY):
        modulated_norm(x, Norm("rms"), out=out)
    q = joint.view(1, 1, 60, 16)
    with pytest.raises(ValueError, match=CUDA_ONLY):
        rotate_qk(q, None, out=(q.as_strided(q.shape, (16, 16, 16, 1)), None))


def test_a_residual_without_a_branch_is_refused():
    """Not answered by the norm alone, without the residual sum that was asked for."""
    x = torch.zeros(2, 3, 16)
    for kw in (dict(norm=Norm("rms")), dict(norm=Norm("rms"), gate=x), dict(branch_norm=Norm("rms"), norm=Norm("rms")),
               dict(), dict(norm=Norm("rms"), out=(x, None))):
        with pytest.raises(ValueError, match="branch must be a tensor"):
            gated_residual(x, None, **kw)
        with pytest.raises(ValueError, match="branch must be a tensor"):
            gated_residual(x, False, **kw)


def test_forward_mode_tangents_are_refused_not_cut():
    from torch.autograd import forward_ad

    x, q, w = torch.zeros(2, 3, 16), torch.zeros(1, 2, 5, 16), torch.ones(16)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: modulated_norm(dual(x), Norm("rms")), lambda: modulated_norm(x, Norm("rms", dual(w))),
                     lambda: modulated_norm(x, Norm("rms"), scale=dual(w)), lambda: gated_residual(x, dual(x)),
                     lambda: gated_residual(x, x, dual(w)), lambda: rotate_qk(dual(q), None),
                     lambda: rotate_qk(q, dual(q))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match=CUDA_ONLY):
            modulated_norm(forward_ad.unpack_dual(dual(x)).primal, Norm("rms"))
    with pytest.raises(ValueError, match=CUDA_ONLY):
        modulated_norm(x, Norm("rms"))


def test_foreign_objects_are_refused():
    x, q = torch.zeros(2, 3, 16), torch.zeros(1, 2, 5, 16)
    for other in (object(), "rms", torch.nn.LayerNorm(16), torch.zeros(16)):
        for call in (lambda: modulated_norm(x, other), lambda: gated_residual(x, x, norm=other),
                     lambda: gated_residual(x, x, branch_norm=other),
                     lambda: rotate_qk(q, None, query_norm=other)):
            with pytest.raises(ValueError, match="must be a Norm"):
                call()
        with pytest.raises(ValueError, match="must be an AxialRotary"):
            rotate_qk(q, None, other)


def test_misaligned_tensors_are_named():
    x, w = torch.zeros(2, 3, 16), torch.ones(16)
    q = torch.zeros(1, 2, 5, 16)
    odd = lambda t: torch.zeros(t.numel() + 2, dtype=t.dtype)[2:].view(t.shape)  # noqa: E731
    pitch = torch.zeros(2, 3, 18)[..., :16]  # 72 bytes between rows
    mods = torch.zeros(2, 3, 18)[..., :16]
    rms = Norm("rms")
    for what, call in [
        ("query must", lambda: rotate_qk(odd(q), None)),
        ("key must", lambda: rotate_qk(q, odd(q))),
        ("query's out", lambda: rotate_qk(q, q, out=(odd(q), torch.zeros_like(q)))),
        ("key's out", lambda: rotate_qk(q, q, out=(torch.zeros_like(q), odd(q)))),
        ("norm's weight", lambda: rotate_qk(q, None, query_norm=Norm("rms", odd(w)))),
        ("x must", lambda: modulated_norm(pitch, rms)),
        ("norm's out", lambda: modulated_norm(x, rms, out=pitch)),
        ("scale must", lambda: modulated_norm(x, rms, scale=mods)),
        ("shift must", lambda: modulated_norm(x, rms, shift=odd(w))),
        ("norm's bias", lambda: modulated_norm(x, Norm("layer", w, odd(w)))),
        ("residual must", lambda: gated_residual(pitch, x)),
        ("branch must", lambda: gated_residual(x, pitch)),
        ("gate must", lambda: gated_residual(x, x, mods)),
        ("sum's out", lambda: gated_residual(x, x, out=(odd(x), None))),
    ]:
        with pytest.raises(ValueError, match=what + ".*16 bytes"):
            call()
    with pytest.raises(ValueError, match=CUDA_ONLY):  # contiguous values in any shape
        modulated_norm(x, Norm("rms", torch.ones(16, 1)))
    # one row, one vector: strides that take no step do not count
    with pytest.raises(ValueError, match=CUDA_ONLY):
        modulated_norm(torch.zeros(1, 1, 18)[..., :16], rms, scale=mods[:1, :1])
    with pytest.raises(ValueError, match=CUDA_ONLY):
        modulated_norm(pitch[:0], rms)


@pytest.mark.parametrize("streamed", [False, True])
def test_attend_refuses_a_rotary_of_another_sequence(streamed):
    """A longer grid, or text in another place than the layout has it, would turn every token by wrong angles."""
    layout = Layout.from_permutation(torch.arange(12), text_tokens=5, text_first=True)
    cls = HostBankOperator if streamed else Operator
    op = cls.build(OperatorConfig(), SparseGeometry.build(layout, 128), n_layers=1)
    q = torch.zeros(1, 2, 17, 16)
    turn = lambda grid, **kw: op.attend(0, q, q, q, rotary=AxialRotary(16, (8, 8), grid=grid, **kw))  # noqa: E731
    for grid, kw in (((4, 6), {}), ((4, 4), dict(text_tokens=5, text_first=True)), ((4, 4), {}), ((3, 4), dict(text_tokens=5)),
                     ((2, 5), dict(text_tokens=7, text_first=True)), ((3, 4), dict(text_tokens=6, text_first=True))):
        with pytest.raises(ValueError, match="rotary positions of .* for a sequence of 17 with 12 from 5 on"):
            turn(grid, **kw)
    for right in (dict(grid=(3, 4), text_tokens=5, text_first=True), dict(grid=(17, 1)), dict(grid=None)):
        with pytest.raises(ValueError, match=CUDA_ONLY):
            turn(right.pop("grid"), **right)


def test_attend_takes_a_rotary_with_room_for_longer_text():
    """Text behind the video does not move it: a rotary for the longest text serves shorter ones."""
    layout = Layout.from_permutation(torch.arange(12), text_tokens=5, text_first=False)
    op = Operator.build(OperatorConfig(), SparseGeometry.build(layout, 128), n_layers=1)
    q = torch.zeros(1, 2, 17, 16)
    for text in (5, 9, 200):
        with pytest.raises(ValueError, match=CUDA_ONLY):
            op.attend(0, q, q, q, rotary=AxialRotary(16, (8, 8), grid=(3, 4), text_tokens=text))
    for text, first in ((4, False), (0, False), (5, True)):
        with pytest.raises(ValueError, match="for a sequence of 17 with 12 from 0 on"):
            op.attend(0, q, q, q, rotary=AxialRotary(16, (8, 8), grid=(3, 4), text_tokens=text, text_first=first))


def test_more_heads_than_32_bits_count_are_refused():
    row = torch.zeros(1, 1, 1, 8)
    for heads in (2**31 - 31, 2**31 - 1, 2**31):
        with pytest.raises(ValueError, match="heads"):
            rotate_qk(row.expand(1, heads, 1, 8), None)
    with pytest.raises(ValueError, match=CUDA_ONLY):
        rotate_qk(row.expand(1, 2**31 - 32, 1, 8), None)
    import struct

    args = lambda hq, hk: struct.Struct("<4Q12qQ3qq4Q10i2f").pack(  # noqa: E731
        4096, 8192, 4096, 8192, *[8] * 12, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, hq, hk, 1, 8, 0, 0, 0, 0, 0, 1e-6, 1e-6)
    for hq, hk in ((2**31 - 31, 1), (1, 2**31 - 1)):
        assert _lib.load().recap_rotate_qk(args(hq, hk), None, None) == _lib.RECAP_ERR_SHAPE


def test_one_tensor_in_two_places_with_an_output_over_it():
    """Query and key are turned by different blocks, and the norm after a residual sum reads its modulations when the
    sum is stored: the same tensor there may not be written in place."""
    q, other = torch.zeros(1, 2, 5, 16), torch.zeros(1, 2, 5, 16)
    r, y, rms = torch.zeros(2, 3, 16), torch.zeros(2, 3, 16), Norm("rms")
    one = torch.zeros(1, 16)
    for call in (lambda: rotate_qk(q, q, out=(q, other)), lambda: rotate_qk(q, q, out=(other, q)),
                 lambda: gated_residual(r, y, norm=rms, scale=r, out=(r, None)),
                 lambda: gated_residual(r, y, norm=rms, shift=r, out=(r, None)),
                 lambda: gated_residual(one, torch.zeros(1, 16), norm=Norm("rms", one), out=(one, None)),
                 lambda: modulated_norm(one, Norm("rms", one), out=one)):
        with pytest.raises(ValueError, match="overlap"):
            call()
    # where each element is read by the thread that writes it, before it does
    for call in (lambda: rotate_qk(q, q), lambda: rotate_qk(q, q, out=(other, torch.zeros(1, 2, 5, 16))),
                 lambda: gated_residual(r, r, r, out=(r, None)), lambda: gated_residual(r, y, y, norm=rms, out=(r, y)),
                 lambda: gated_residual(r, y, norm=rms, scale=y, shift=y, out=(None, y)),
                 lambda: modulated_norm(r, rms, scale=r, shift=r, out=r)):
        with pytest.raises(ValueError, match=CUDA_ONLY):
            call()
