"""ltx_nn.quantize_fp8 on models that it cannot convert as a whole, and on parts that share layers (GPU)."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16 = torch.bfloat16


@pytest.mark.parametrize("other", ["fp16", "fp32", "cpu", "bias"])
def test_a_layer_of_another_kind_leaves_the_model_as_it_was(other):
    import ltx_nn

    model = torch.nn.ModuleList([ltx_nn.FeedForward(128), ltx_nn.FeedForward(128)]).to(DEV, BF16).requires_grad_(False)
    last = model[1]
    if other == "cpu":
        last.cpu()
    elif other == "bias":
        last.proj_out.bias = torch.nn.Parameter(last.proj_out.bias.float(), requires_grad=False)
    else:
        last.to(torch.float16 if other == "fp16" else torch.float32)
    with pytest.raises(ValueError, match="1.proj"):
        ltx_nn.quantize_fp8(model)
    assert all(type(layer) is torch.nn.Linear for ff in model for layer in (ff.proj_in, ff.proj_out))
    with pytest.raises(ValueError, match="bf16"):
        ltx_nn.Fp8Linear.of(last.proj_out)


def test_shared_layers_stay_shared():
    import ltx_nn

    ff, other = (ltx_nn.FeedForward(128).to(DEV, BF16).requires_grad_(False) for _ in range(2))
    other.proj_in = ff.proj_in
    both = torch.nn.ModuleList([ff, other]).eval()
    ltx_nn.quantize_fp8(both)
    assert type(ff.proj_in) is ltx_nn.Fp8Linear and ff.proj_in is other.proj_in and not ff.proj_in.training


def test_another_device_leaves_the_model_as_it_was(monkeypatch):
    """Kernels run on the current device: layers on another one are refused before any is replaced."""
    import ltx_nn

    ff = ltx_nn.FeedForward(128).to(DEV, BF16).requires_grad_(False)
    other = torch.nn.ModuleList([ltx_nn.FeedForward(128).to(DEV, BF16).requires_grad_(False), ff])
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ValueError, match="0.proj_in .* on cuda:0.*current GPU"):
        ltx_nn.quantize_fp8(other)
    with pytest.raises(ValueError, match="current GPU"):
        ltx_nn.Fp8Linear.of(ff.proj_in)
    assert all(type(layer) is torch.nn.Linear for f in other for layer in (f.proj_in, f.proj_out))
    monkeypatch.undo()
    assert ltx_nn.quantize_fp8(ff).takes_blocks
