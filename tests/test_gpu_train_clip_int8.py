"""Clipping and 8-bit inference where a program uses them: the recorded training loop with this package's clipping, then the
finalised model quantised and answering batches and single tokens; and the layer's 8-bit mode by itself."""
import json
import math

import pytest
import torch

from golden_io import Golden, rel_err
from test_gpu_int8 import _check, _exact
from test_gpu_train_loop import DEV, LOOP_TOL, TinyMLP, _build

pytestmark = pytest.mark.gpu


def _captured_inputs(model, x):
    """Output of the model and the input every SparseLinear saw."""
    seen, handles = {}, []
    for name, m in model.named_modules():
        if hasattr(m, "hardening_x"):
            handles.append(m.register_forward_hook(lambda mod, i, o, n=name: seen.__setitem__(n, (i[0], o))))
    with torch.no_grad():
        y = model(x)
    for h in handles:
        h.remove()
    return y, seen


def test_training_with_clipping_then_8_bit_inference():
    import sparseforge_b200 as sf
    from sparseforge_b200 import utils as U

    g = Golden("train_loop")
    hp = json.loads(str(g["hp_json"]))
    cfgd = json.loads(str(g["cfg_json"]))
    model, _ = _build(g, "init/")
    U.initialize_model(model)
    opt = sf.AdamW([model.fc1.weight, model.fc1.bias, model.fc2.weight], lr=hp["lr"], betas=tuple(hp["betas"]),
                   weight_decay=hp["weight_decay"], srste_decay=cfgd["srste_decay"])
    X, Yt = g["X"].to(DEV), g["Yt"].to(DEV)
    for it in range(hp["steps"]):
        lam = hp["lambda_mid_max"] * min(1.0, it / hp["lambda_mid_warmup"])
        loss = torch.nn.functional.mse_loss(model(X[it]), Yt[it]) + U.mid_penalty(model, lam)
        queue = [g[f"s{it}_probe{j}"].to(DEV).float() for j in range(2)]
        U._rademacher_like = lambda t, q=queue: q.pop(0)
        U.update_hessian_hutchinson(model, loss)
        loss.backward()
        gnorm = U.clip_grad_norm_(model.parameters(), hp["grad_clip"])
        assert float(gnorm) == pytest.approx(g.scalar(f"s{it}_gnorm"), rel=LOOP_TOL)
        U.update_model_grad_ema(model, update_hessian_with_grad2=False)
        opt.step(decay=cfgd["srste_decay"] * min(1.0, (it + 1) / hp["decay_ramp"]))
        opt.zero_grad(set_to_none=True)
        U.calculate_model_mask(model, it, lambda_mid=lam)
        for ln, layer in (("fc1", model.fc1), ("fc2", model.fc2)):
            assert rel_err(layer.weight.data, g[f"s{it}_{ln}_W"]) <= LOOP_TOL, (it, ln)
            assert rel_err(layer.mask.data, g[f"s{it}_{ln}_mask"]) <= 5 * LOOP_TOL, (it, ln)

    U.finalize_hard_masks(model)
    model.eval()
    U.optimize_sparse_model_for_inference(model, int8=True)
    assert model.fc1.mode == model.fc2.mode == "int8_forward"
    Xe = g["eval_X"].to(DEV)
    y, seen = _captured_inputs(model, Xe)
    for name, (inp, out) in seen.items():
        layer = dict(model.named_modules())[name]
        w = layer.weight.data
        assert torch.all((w == 0) | (layer.mask.data == 1))  # the zeros of the hard mask are in the quantised weight
        assert not layer._i8_weight[:, :layer.in_features][w == 0].any()
        _check(out.reshape(-1, out.shape[-1]), *_exact(inp.reshape(-1, inp.shape[-1]), w, layer.bias), torch.float32)
    assert y.shape == g["eval_Y"].shape and torch.isfinite(y).all()
    # one token at a time gives the same values as the batch
    flat = Xe.reshape(-1, Xe.shape[-1])
    with torch.no_grad():
        single = torch.cat([model(flat[i:i + 1]) for i in range(min(5, flat.shape[0]))])
    first = y.reshape(-1, y.shape[-1])[:single.shape[0]]
    assert torch.equal(single, first)


def _layer(k, n, dtype, bias=True, **cfg):
    import sparseforge_b200 as sf

    torch.manual_seed(k + n)
    c = dict(mask_type="structured", mask_update_period=1, sparsity_warmup_steps=0)
    c.update(cfg)
    layer = sf.SparseLinear(k, n, sparselinear_config=sf.SparseLinearConfig(**c), bias=bias).to(DEV).to(dtype)
    layer.mask.data.copy_(torch.rand_like(layer.mask))
    return layer.eval()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cfg", [dict(), dict(N=4, M=8), dict(mask_type="unstructured"), dict(mask_type="none"),
                                 dict(hard_mask_type="block16", sparsity_ratio=0.5)])
def test_layer_in_8_bit_mode_with_every_hard_view(cfg, dtype):
    layer = _layer(64, 48, dtype, **cfg)
    w = layer.weight.data * layer._hard_mask_from_soft(layer.mask.data).to(dtype)
    layer.quantize_for_inference()
    for shape in ((64,), (1, 64), (3, 1, 64), (2, 9, 64), (200, 64), (0, 64)):
        x = torch.randn(shape, device=DEV).to(dtype)
        with torch.no_grad():
            y = layer(x)
        assert y.shape == shape[:-1] + (48,) and y.dtype == dtype
        if x.numel():
            _check(y.reshape(-1, 48), *_exact(x.reshape(-1, 64), w, layer.bias.data), dtype)


def test_layer_in_8_bit_mode_inputs_and_errors():
    layer = _layer(64, 48, torch.bfloat16)
    with pytest.raises(RuntimeError, match="quantize_for_inference"):
        layer.mode = "int8_forward"
        with torch.no_grad():
            layer(torch.zeros(2, 64, device=DEV, dtype=torch.bfloat16))
    layer.quantize_for_inference()
    base = torch.randn(6, 130, device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        want = layer(base[:, :64].contiguous())
        assert torch.equal(layer(base[:, :64]), want)                         # strided rows
        assert torch.equal(layer(base[:, :64].t().contiguous().t()), want)    # columns contiguous
        assert torch.equal(layer(base[:1, :64].expand(6, 64)), want[:1].expand(6, 48))
        half = layer(base[:, :64].half())                                     # float16 goes through float32
        assert half.dtype == torch.float16
        w = layer.weight.data * layer._hard_mask_from_soft(layer.mask.data).to(torch.bfloat16)
        ref, mag = _exact(base[:, :64].half(), w, layer.bias.data)
        assert ((half.double() - ref).abs() <= 2.0 ** -11 * ref.abs() + 8 * 2.0 ** -24 * (mag + ref.abs()) + 2.0 ** -25).all()
    x = torch.randn(2, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="inference only"):
        layer(x)
    with pytest.raises(RuntimeError, match="inference only"):
        layer.train()(x.detach())
    # moving the module keeps the 8-bit form as it is
    q = layer._i8_weight.clone()
    layer.eval().to(torch.float32)
    assert torch.equal(layer._i8_weight, q) and layer._i8_scale.dtype == torch.float32
    with torch.no_grad():
        assert layer(base[:, :64].float()).dtype == torch.float32


def test_model_level_choice():
    from sparseforge_b200 import utils as U

    class Two(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.a, self.b = _layer(32, 40, torch.bfloat16), _layer(40, 24, torch.float32, bias=False)

    m = Two()
    dense_a = m.a.weight.data * m.a._hard_mask_from_soft(m.a.mask.data).bfloat16()
    with pytest.raises(ValueError, match="one of"):
        U.optimize_sparse_model_for_inference(m, compressed=True, int8=True)
    U.optimize_sparse_model_for_inference(m, int8=True)
    assert m.a.mode == m.b.mode == "int8_forward"
    assert torch.equal(m.a.weight.data, dense_a)
    deq = m.a._i8_weight[:, :32].double() * m.a._i8_scale.double()[:, None]
    assert ((deq - dense_a.double()).abs() <= (0.5 + 1e-4) * m.a._i8_scale.double()[:, None]).all()
    # with the low-rank bypass kept the layers stay masked, as for the other inference forms
    m2 = Two()
    U.optimize_sparse_model_for_inference(m2, use_slorb=True, int8=True)
    assert m2.a.mode == "sparse_forward"


def test_clipping_feeds_the_optimizer_like_torch_does():
    """bf16 layer: one step with each clipping from the same gradients. Each clipped gradient is off by at most a rounding
    (the norm differs by the gradients' dtype in torch's), so the two weights agree to the bf16 steps that follow from it."""
    import sparseforge_b200 as sf
    from sparseforge_b200 import utils as U

    states = []
    for clip in (U.clip_grad_norm_, torch.nn.utils.clip_grad_norm_):
        layer = _layer(64, 48, torch.float32).train()
        opt = sf.AdamW(layer.parameters(), lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1)
        x = torch.arange(40 * 64, device=DEV).reshape(40, 64).remainder(17).float() - 8
        layer(x).square().mean().backward()
        norm = clip([p for p in layer.parameters()], 0.1)
        opt.step(decay=1e-4)
        states.append((float(norm), layer.weight.data.clone(), layer.bias.data.clone()))
    (n1, w1, b1), (n2, w2, b2) = states
    # torch adds squares in fp32, a tree of at most 3120 terms
    assert abs(n1 - n2) <= 64 * 2.0 ** -24 * n2 and math.isfinite(n1) and n1 > 0.1
    assert (w1 - w2).abs().max() <= 1e-2 * 200 * 2.0 ** -24 + 2.0 ** -22 * w2.abs().max()
    assert (b1 - b2).abs().max() <= 1e-2 * 200 * 2.0 ** -24 + 2.0 ** -22 * b2.abs().max()


def test_training_on_outdates_the_8_bit_form():
    """An evaluation in 8 bits between training steps: the optimizer's kernel and the mask update write weight and mask
    where no version counter sees it; the layer refuses to answer from the old weights until it is quantised again."""
    import copy

    import sparseforge_b200 as sf
    from sparseforge_b200 import utils as U

    x = torch.randn(12, 64, device=DEV)

    def answers(layer):
        mode, layer.mode = layer.mode, "int8_forward"
        try:
            with torch.no_grad():
                return layer.eval()(x)
        finally:
            layer.mode = mode
            layer.train()

    for cfg in (dict(), dict(N=4, M=8), dict(mask_type="unstructured", hard_mask_type="block16", sparsity_ratio=0.5)):
        layer = _layer(64, 48, torch.float32, change_mask=True, mask_metric="magnitude", **cfg).train()
        opt = sf.AdamW(layer.parameters(), lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1)
        for step in range(3):
            layer.quantize_for_inference()
            layer.mode = "sparse_forward"
            first = answers(layer)
            assert torch.equal(answers(copy.deepcopy(layer)), first)
            layer(x).square().mean().backward()
            assert torch.equal(answers(layer), first)  # neither pass of a training step has moved anything yet
            opt.step()
            with pytest.raises(RuntimeError, match="changed"):
                answers(layer)
            layer.quantize_for_inference()
            layer.mode = "sparse_forward"
            answers(layer)
            U.calculate_model_mask(layer, step)
            with pytest.raises(RuntimeError, match="changed"):
                answers(layer)
            opt.zero_grad()
    m = torch.nn.Sequential(_layer(64, 48, torch.bfloat16))
    U.optimize_sparse_model_for_inference(m, int8=True)
    with torch.no_grad():
        y = m(x.bfloat16())
    state = {k: torch.randn_like(v) for k, v in m.state_dict().items()}
    m.load_state_dict(state)
    with pytest.raises(RuntimeError, match="changed"), torch.no_grad():
        m(x.bfloat16())
    U.optimize_sparse_model_for_inference(m, int8=True)
    w = m[0].weight.data
    with torch.no_grad():
        z = m(x.bfloat16())
    _check(z, *_exact(x.bfloat16(), w, m[0].bias.data), torch.bfloat16)
    assert not torch.equal(y, z)
