"""One adapter-training step and one sampling step of a small DiT with a 4-bit base, 4-bit time path, residual steps
fused and orthogonalised adapter updates, against the same model on the separate kernels."""
import copy
import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu

CFG = dict(features=256, tdim=128, txtdim=128, heads=2, kvheads=1, multiplier=2, layers=2, patch=2, channels=16,
           txtheads=1, txtkvheads=1, txtlayers=3)


def build(fused_residual):
    from k2q import dit, lora, modules
    m = dit.SingleStreamDiT(dit.DiTConfig(**CFG))
    for name, p in m.named_parameters():
        g = torch.Generator().manual_seed(zlib.crc32(name.encode()))
        p.data = (torch.randn(p.shape, generator=g) * 0.05).to(p.dtype)
    m = m.to(torch.bfloat16).cuda()
    assert modules.quantize_dit_convrot(m, bits=4, backward_copy=True) == 16
    assert modules.quantize_time_path(m) == 3
    ads = lora.inject_lora(m, rank=8, alpha=8.0)
    for name, ad in ads.items():
        g = torch.Generator().manual_seed(zlib.crc32(name.encode()))
        ad.lora_A.data.copy_(torch.randn(ad.lora_A.shape, generator=g) * 0.02)
        ad.lora_B.data.copy_(torch.randn(ad.lora_B.shape, generator=g) * 0.02)
    if fused_residual:
        assert modules.fuse_residual_norms(m) == 6
    return m, ads


def inputs():
    g = torch.Generator().manual_seed(3)
    b, gh, gw, l = 2, 8, 8, 24
    tm = torch.ones(b, l, dtype=torch.bool)
    tm[1, 20:] = False
    return dict(z0=torch.randn(b, gh * gw, 64, generator=g).cuda(), context=torch.randn(b, l, 3, 128, generator=g).bfloat16().cuda(),
                text_mask=tm.cuda(), grid_h=gh, grid_w=gw, t=torch.tensor([0.3, 0.8]).cuda(),
                noise=torch.randn(b, gh * gw, 64, generator=g).cuda())


def params_of(ads):
    return [p for ad in ads.values() for p in (ad.lora_A, ad.lora_B)]


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-30))


def test_training_step(monkeypatch):
    from k2q import dit, ops, parallel, trainer
    grads, used = [], {"rows": 0}
    few = ops.gemv_w4a8
    monkeypatch.setattr(ops, "gemv_w4a8", lambda *a, **k: (used.__setitem__("rows", used["rows"] + 1), few(*a, **k))[1])
    for fused_residual in (False, True):
        m, ads = build(fused_residual)
        m.train()
        params = params_of(ads)
        buckets = parallel.AdapterGradBuckets([params])
        opt = trainer.FusedOrthogonalStep(buckets, lr=0.02, momentum=0.9, weight_decay=0.1, max_grad_norm=1e9)
        buckets.zero()
        loss = dit.flow_training_step(m, **inputs())
        loss.backward()
        ops.check_status()
        grads.append(buckets.flat.clone())
        before = opt.param.clone()
        opt.step()
        assert float(opt.grad_norm()) == pytest.approx(float(grads[-1].norm()), rel=1e-5)
        assert (buckets.flat == 0).all() and all(p.grad is not None and (p.grad == 0).all() for p in params)
    assert used["rows"] >= 6                                     # the time path's three Linears, both models
    # the fused step rounds less than the chain of kernels: every tensor on the way differs by bf16 roundings
    assert rel(grads[1], grads[0]) <= 3e-2
    # the optimizer step: momentum 0 before, so u = (1 - beta)(1 + beta) g, whose scale does not matter; the slices the
    # modules hold are the flat buffer's
    layout = opt.layout
    x = ops.orthogonalize(grads[1] * (1 - 0.9) * (1 + 0.9), layout)
    off = 0
    for p in params:
        n = p.numel()
        want = before[off:off + n].double() * (1 - 0.02 * 0.1) - 0.02 * 0.2 * max(p.shape) ** 0.5 * x[off:off + n].double()
        assert p.data_ptr() == opt.param.data_ptr() + 4 * off
        # u reaches the kernel through three roundings more than here; a^5 bounds what the iteration makes of them
        assert float((p.detach().reshape(-1).double() - want).norm()) <= 0.02 * 0.2 * max(p.shape) ** 0.5 * 485 * 8 * 2.0 ** -24 + 4 * 2.0 ** -24 * float(want.norm())
        off += n
    sd = opt.state_dict()
    assert sd["step"] == 1 and torch.equal(sd["m"], opt.m)
    opt.load_state_dict({"step": 5, "m": torch.zeros_like(opt.m)})
    assert opt.step_count == 5 and (opt.m == 0).all()


def test_sampling_step():
    from k2q import dit, lora, modules, ops
    outs = []
    for fused_residual in (False, True):
        m = dit.SingleStreamDiT(dit.DiTConfig(**CFG))
        for name, p in m.named_parameters():
            g = torch.Generator().manual_seed(zlib.crc32(name.encode()))
            p.data = (torch.randn(p.shape, generator=g) * 0.05).to(p.dtype)
        m = m.to(torch.bfloat16).cuda().eval()
        modules.quantize_dit_convrot(m, bits=4)
        modules.quantize_time_path(m)
        if fused_residual:
            modules.fuse_residual_norms(m)
        i = inputs()
        pos, mask = dit.position_ids(8, 8, i["text_mask"])
        outs.append(dit.denoise_step(m, i["noise"].bfloat16(), i["context"], 1.0, 0.9, pos, mask))
        ops.check_status()
    assert rel(outs[1], outs[0]) <= 1e-2 and not torch.equal(outs[0], torch.zeros_like(outs[0]))
    assert modules.fuse_residual_norms(m, fused=False) == 6
    back = dit.denoise_step(m, i["noise"].bfloat16(), i["context"], 1.0, 0.9, pos, mask)
    assert torch.equal(back, outs[0])


def test_checkpointed_training_step_captures_nothing_stale():
    """Under gradient checkpointing the fused step is run again in the backward: the same gradients."""
    from k2q import dit
    grads = []
    for ckpt in (False, True):
        m, ads = build(True)
        m.train()
        m.gradient_checkpointing = ckpt
        dit.flow_training_step(m, **inputs()).backward()
        grads.append(torch.cat([p.grad.reshape(-1) for p in params_of(ads)]))
    assert torch.equal(grads[0], grads[1])


def test_time_path_is_quantised_whole_or_not_at_all():
    from k2q import dit, modules
    m = dit.SingleStreamDiT(dit.DiTConfig(**dict(CFG, features=192, heads=2, kvheads=2))).to(torch.bfloat16).cuda()
    with pytest.raises(ValueError):
        modules.quantize_time_path(m)
    assert all(type(c) is not modules.ConvRotLinear for seq in (m.tmlp, m.tproj) for c in seq)


def test_orthogonal_step_refuses_vectors_and_large_ranks():
    from k2q import parallel, trainer
    for shape in ((300,), (65, 70)):
        p = torch.nn.Parameter(torch.zeros(shape, device="cuda"))
        with pytest.raises(ValueError):
            trainer.FusedOrthogonalStep(parallel.AdapterGradBuckets([[p]]))


def test_time_path_is_saved_and_loaded_with_the_base(tmp_path):
    from k2q import dit, modules, serialize
    make = lambda: dit.SingleStreamDiT(dit.DiTConfig(**CFG)).to(torch.bfloat16).cuda()      # noqa: E731
    m = make()
    n = modules.quantize_dit_convrot(m, bits=4, backward_copy=False) + modules.quantize_time_path(m)
    assert modules.quantize_time_path(m) == 0                    # nothing is quantised twice
    path = str(tmp_path / "base.safetensors")
    assert serialize.save_quantized_base(m, path) == n
    fresh = make()
    assert serialize.load_quantized_base(fresh, path, device="cuda") == n
    for name, want in serialize.convrot_modules(m).items():
        got = fresh.get_submodule(name)
        assert torch.equal(got.weight_q, want.weight_q) and torch.equal(got.scale, want.scale)
    mixed = make()
    modules.quantize_dit_convrot(mixed, bits=8)
    modules.quantize_time_path(mixed, bits=4)
    with pytest.raises(ValueError, match="mixed bit widths"):
        serialize.save_quantized_base(mixed, path)
