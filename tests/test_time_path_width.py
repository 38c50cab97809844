"""``quantize_time_path`` without a width takes the base's, so that a model quantised with either default can be saved."""
import pytest
import torch

CFG = dict(features=256, tdim=128, txtdim=128, heads=2, kvheads=1, multiplier=2, layers=1, patch=2, channels=16,
           txtheads=1, txtkvheads=1, txtlayers=3)


def model():
    from k2q import dit
    torch.manual_seed(2)
    return dit.SingleStreamDiT(dit.DiTConfig(**CFG)).to(torch.bfloat16).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("base", [8, 4, None])
def test_default_width_is_the_bases(base, tmp_path):
    from k2q import modules, serialize
    m = model()
    n = modules.quantize_dit_convrot(m, bits=base) if base else 0
    n += modules.quantize_time_path(m)
    quantised = serialize.convrot_modules(m)
    assert {q.bits for q in quantised.values()} == {base or 4} and len(quantised) == n
    path = str(tmp_path / "base.safetensors")
    assert serialize.save_quantized_base(m, path) == n
    fresh = model()
    assert serialize.load_quantized_base(fresh, path, device="cuda") == n
    for name, want in quantised.items():
        got = fresh.get_submodule(name)
        assert got.bits == want.bits and torch.equal(got.weight_q, want.weight_q) and torch.equal(got.scale, want.scale)
    t = torch.randn(2, CFG["tdim"], device="cuda").bfloat16()
    with torch.no_grad():
        assert torch.equal(m.tproj(m.tmlp(t)), fresh.tproj(fresh.tmlp(t)))


@pytest.mark.gpu
def test_explicit_width_is_kept():
    from k2q import modules
    m = model()
    modules.quantize_dit_convrot(m, bits=8)
    assert modules.quantize_time_path(m, bits=4) == 3
    assert {c.bits for seq in (m.tmlp, m.tproj) for c in seq if isinstance(c, modules.ConvRotLinear)} == {4}
