"""Blocks whose residual steps are fused keep that under the parallel splits, whichever call comes first."""
import pytest
import torch
import torch.nn as nn


def holder_of(n=1, dim=512, heads=4, kvheads=2, dtype=torch.bfloat16, device="cpu"):
    from k2q import dit
    torch.manual_seed(17)
    h = nn.Module()
    h.blocks = nn.ModuleList([dit.SingleStreamBlock(dim, heads, 3, bias=True, kvheads=kvheads) for _ in range(n)])
    for p in h.parameters():
        p.data.normal_(0.0, 0.04)
    return h.to(dtype).to(device)


def inputs_of(dim=512, tokens=8, dtype=torch.bfloat16, device="cpu"):
    from k2q import dit
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, tokens, dim, generator=g).to(dtype).to(device)
    vec = (torch.randn(2, 1, 6 * dim, generator=g) * 0.1).to(dtype).to(device)
    pos = torch.arange(tokens, device=device)[None, :, None].expand(2, tokens, 3)
    return x, vec, dit.rope_tables(pos, [128 - 12 * 8, 48, 48], 1e4)


def shard(kind, holder):
    from k2q import parallel
    return parallel.shard_dit_columns(holder, 0, 1) if kind == "columns" else parallel.shard_dit_sequence(holder, 0, 1)


def apply(holder, args):
    x, vec, rope = args
    with torch.no_grad():
        for b in holder.blocks:
            x = b(x, vec, rope)
    return x


@pytest.mark.parametrize("kind", ["columns", "sequence"])
@pytest.mark.parametrize("fuse_first", [True, False])
def test_setting_survives_sharding(kind, fuse_first, monkeypatch):
    """Dense bf16 blocks on the CPU: the fused step is taken once per block, and the results are the unsharded fused
    blocks'."""
    from k2q import fused, modules
    args = inputs_of()
    whole = holder_of(2)
    assert modules.fuse_residual_norms(whole) == 2
    want = apply(whole, args)
    calls, real = [], fused.residual_norm
    monkeypatch.setattr(fused, "residual_norm", lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    h = holder_of(2)
    if fuse_first:
        modules.fuse_residual_norms(h)
    shard(kind, h)
    if not fuse_first:
        assert modules.fuse_residual_norms(h) == 2
    assert torch.equal(apply(h, args), want) and len(calls) == 2
    assert modules.fuse_residual_norms(h, fused=False) == 2
    plain = apply(holder_of(2), args)
    assert torch.equal(apply(h, args), plain) and len(calls) == 2 and not torch.equal(plain, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["columns", "sequence"])
@pytest.mark.parametrize("bits", [8, 4])
def test_quantised_sharded_blocks_equal_the_unsharded_fused_block(kind, bits):
    from k2q import modules, ops
    args = inputs_of(768, 72, device="cuda")
    h = holder_of(1, 768, 6, 3, device="cuda")
    modules.quantize_dit_convrot(h, bits=bits)
    plain = apply(h, args)
    modules.fuse_residual_norms(h)
    want = apply(h, args)
    shard(kind, h)
    got = apply(h, args)
    ops.check_status()
    assert torch.equal(got, want) and not torch.equal(plain, want)
    modules.fuse_residual_norms(h, fused=False)
    assert torch.equal(apply(h, args), plain)
