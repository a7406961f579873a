"""The paths that call the operators around the attention: the sequence-parallel exchange that
turns each rank's own tokens, and the layer stack of the benchmark with conditioned blocks."""

import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF = torch.bfloat16


@pytest.mark.parametrize("mode", ["in_place", "push"])
@pytest.mark.parametrize("world,text,text_first,across", [(2, 64, False, False), (4, 96, True, True)])
def test_sharded_rotation_matches_the_gathered_one(world, text, text_first, across, mode):
    """Every rank turns its own tokens (``ShardedIO.rotate``, and ``push`` with a rotary) before the
    exchange: the attention of each rank's heads equals, bit for bit, turning the gathered
    projections of all heads and attending on the rank's."""
    from recap_b200 import REFRESH, SPARSE, AxialRotary, Norm, Operator, OperatorConfig, rotate_qk
    from recap_b200.sparse import Layout, SparseGeometry
    from recap_b200.ulysses import ShardedIO

    H, d, grid = 2 * world, 64, (5, 16, 32)
    nv = math.prod(grid)
    S = nv + text
    s, h = S // world, H // world
    layout = Layout.from_permutation(np.random.default_rng(3).permutation(nv), text_tokens=text, text_first=text_first)
    rotary = AxialRotary(d, (16, 24, 24), grid=grid, text_tokens=text, text_first=text_first)
    g = torch.Generator(device=DEV).manual_seed(7)
    n = H * d if across else d
    qn, kn = (Norm("rms", 1 + 0.1 * torch.randn(n, generator=g, device=DEV), across_heads=across) for _ in range(2))
    geo = SparseGeometry.build(layout, 128)
    for rank in (0, world - 1):
        plain, sharded = (Operator.build(OperatorConfig(head_density=0.25), geo, n_layers=1) for _ in range(2))
        heads = slice(rank * h, (rank + 1) * h)
        outs = [torch.zeros(s, H, d, dtype=BF, device=DEV) for _ in range(world)]
        recvs = [torch.zeros(S, 3, h, d, dtype=BF, device=DEV) for _ in range(world)]

        def peers(bufs, r):
            return SimpleNamespace(ptrs=[t.data_ptr() for t in bufs], world=world, rank=r, device=torch.device(DEV),
                                   nbytes=bufs[0].numel() * 2)

        for step, kind in enumerate((REFRESH, SPARSE)):
            full = torch.randn(S, 3, H, d, generator=g, device=DEV).to(BF)
            shards = [full[r * s:(r + 1) * s].clone() for r in range(world)]
            for r in range(world):  # every rank's own step, one after another
                if mode == "push":
                    ShardedIO(None, peers(outs, r), H, d, S, recv=peers(recvs, r)).push(
                        shards[r], rotary=rotary, query_norm=qn, key_norm=kn)
                else:
                    ShardedIO(peers(shards, r), peers(outs, r), H, d, S).rotate(shards[r], rotary, qn, kn)
            io = ShardedIO(peers(shards, rank), peers(outs, rank), H, d, S,
                           recv=peers(recvs, rank) if mode == "push" else None)
            q, k, v = (full[:, i].permute(1, 0, 2).unsqueeze(0) for i in range(3))
            q, k = rotate_qk(q, k, rotary, query_norm=qn, key_norm=kn)
            plain.begin_step(step, kind)
            want = plain.attend(0, q[:, heads], k[:, heads], v[:, heads])
            sharded.begin_step(step, kind)
            sharded.attend_sharded(0, io)
            got = torch.cat([o[:, heads] for o in outs]).permute(1, 0, 2).unsqueeze(0)
            assert torch.equal(got, want)
            assert all(torch.equal(shards[r][:, 2], full[r * s:(r + 1) * s, 2]) for r in range(world))
        plain.check_device_status()
        sharded.check_device_status()


def test_sharded_rotation_refuses():
    from recap_b200 import AxialRotary
    from recap_b200.ulysses import ShardedIO

    out = torch.zeros(32, 4, 64, dtype=BF, device=DEV)
    peer = SimpleNamespace(ptrs=[out.data_ptr()] * 2, world=2, rank=1, device=torch.device(DEV), nbytes=out.numel() * 2)
    io = ShardedIO(None, peer, 4, 64, 64)
    qkv = torch.zeros(32, 3, 4, 64, dtype=BF, device=DEV)
    with pytest.raises(ValueError):  # positions of another sequence
        io.rotate(qkv, AxialRotary(64, (16, 24, 24), grid=(1, 8, 7)))
    with pytest.raises(ValueError):  # positions without a grid
        io.rotate(qkv, AxialRotary(64, (16, 24, 24)))
    with pytest.raises(ValueError):
        io.rotate(qkv[:16], AxialRotary(64, (16, 24, 24), grid=(1, 8, 8)))


def test_conditioned_stack_is_its_operators_in_turn():
    """Two layers of the benchmark's stack with conditioned blocks, step by step against the public
    operators; without the conditioning the stack is what it was."""
    import sys
    from pathlib import Path

    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
    import bench
    from recap_b200 import EXACT, AxialRotary, Norm, Operator, OperatorConfig, gated_residual, modulated_norm, rotate_qk
    from recap_b200.sparse import Layout, SparseGeometry, hilbert_permutation

    w = dict(grid=(3, 8, 12), heads=4, dim=64, text=32, text_first=False, density=0.25, layers=2, hidden=256)
    layout = Layout.from_permutation(hilbert_permutation(w["grid"]), text_tokens=32, text_first=False)
    op = Operator.build(OperatorConfig(head_density=0.25), SparseGeometry.build(layout, 128), n_layers=2)
    dev = torch.device(DEV)
    x0 = bench.stack_hidden(w, range(320), 256, seed=0, device=dev)
    with torch.no_grad():
        op.begin_step(0, EXACT)
        plain = bench.AttentionStack(op, w, 1, None, dev)
        x = x0
        for layer in range(2):
            q, k, v = (x @ plain.w_qkv[layer]).view(320, 3, 4, 64).permute(1, 2, 0, 3).unsqueeze(1)
            x = x + op.attend(layer, q, k, v)[0].permute(1, 0, 2).reshape(320, 256) @ plain.w_o[layer]
        assert torch.equal(plain.step(x0), x)

        stack = bench.AttentionStack(op, w, 1, None, dev, conditioned=True)
        rotary = AxialRotary(64, (24, 20, 20), theta=256.0, grid=w["grid"], text_tokens=32)
        x, norm = x0, Norm("layer")
        for layer in range(2):
            scale, shift, gate = stack.mods[layer]
            h = modulated_norm(x, norm, scale=scale, shift=shift) if layer == 0 else h
            q, k, v = (h @ stack.w_qkv[layer]).view(320, 3, 4, 64).permute(1, 2, 0, 3).unsqueeze(1)
            q, k = rotate_qk(q, k, rotary, query_norm=stack.qk_norms[layer][0], key_norm=stack.qk_norms[layer][1])
            y = op.attend(layer, q, k, v)[0].permute(1, 0, 2).reshape(320, 256) @ stack.w_o[layer]
            nxt = stack.mods[min(layer + 1, 1)]
            x, h = gated_residual(x, y, gate, norm=norm, scale=nxt[0], shift=nxt[1])
        got = stack.step(x0)
        assert torch.equal(got, x) and bool(got.isfinite().all()) and not torch.equal(got, x0)
    op.check_device_status()


def test_streamed_banks_with_rotary():
    """An operator that streams its banks through host memory turns the projections as the resident one."""
    from recap_b200 import REFRESH, SPARSE, AxialRotary, HostBankOperator, Norm, Operator, OperatorConfig
    from recap_b200.sparse import Layout, SparseGeometry, hilbert_permutation

    g = torch.Generator(device=DEV).manual_seed(9)
    grid, d = (4, 16, 16), 64
    layout = Layout.from_permutation(hilbert_permutation(grid), text_tokens=0, text_first=False)
    geo = SparseGeometry.build(layout, 128)
    cfg = OperatorConfig(head_density=0.25)
    resident, streamed = Operator.build(cfg, geo, n_layers=2), HostBankOperator.build(cfg, geo, n_layers=2)
    streamed.hbm_budget = 0
    turn = dict(rotary=AxialRotary(d, (16, 24, 24), grid=grid), query_norm=Norm("rms"), key_norm=Norm("rms"))
    for step, kind in enumerate((REFRESH, SPARSE, REFRESH)):
        for op in (resident, streamed):
            op.begin_step(step, kind)
        for layer in range(2):
            q, k, v = (torch.randn(1, 2, 1024, d, generator=g, device=DEV).to(BF) for _ in range(3))
            with pytest.raises(ValueError):  # refused before anything is written
                resident.attend(layer, q, k, v, rotary=AxialRotary(d, (16, 24, 24), grid=(4, 16, 15)))
            assert torch.equal(streamed.attend(layer, q, k, v, **turn), resident.attend(layer, q, k, v, **turn))
    resident.check_device_status()
    streamed.check_device_status()
