"""The norms and the linear layer have no derivatives: inputs that require a gradient or carry a tangent, also those of a
functional transform, are refused instead of coming back without it."""
import pytest
import torch
from torch.autograd import forward_ad


def _calls(device):
    """name -> (operator on one tensor per argument, the arguments)"""
    from mindiesd import add_rms_norm, add_rms_norm_quant, linear_forward
    from mindiesd.layers.quant import token_quant_preprocess

    def t(*shape):
        return torch.ones(shape, device=device, dtype=torch.bfloat16)
    x8, w8 = t(4, 64).to(torch.float8_e4m3fn), t(32, 64).to(torch.float8_e4m3fn)
    s, ws = torch.ones(4, 1, device=device), torch.ones(32, device=device)
    return {"norm": (add_rms_norm, [t(4, 64), t(64), t(4, 64)]), "norm_quant": (add_rms_norm_quant, [t(4, 64), t(64), t(4, 64)]),
            "quant": (token_quant_preprocess, [t(4, 64)]),
            "linear": (lambda x, w, b, r, g: linear_forward(x, w, b, residual=r, gate=g), [t(4, 64), t(32, 64), t(32), t(4, 32), t(32)]),
            "linear_e4m3": (lambda s, ws: linear_forward(x8, w8, x_scale=s, weight_scale=ws), [s, ws])}


def _check(device):
    from mindiesd import ParametersInvalid
    for name, (fn, args) in _calls(device).items():
        for i in range(len(args)):
            for guard in (torch.enable_grad, torch.no_grad):  # a tangent goes on under no_grad
                with forward_ad.dual_level(), guard():
                    dual = list(args)
                    dual[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                    with pytest.raises(ParametersInvalid):
                        fn(*dual)
                        pytest.fail(f"{name} took a tangent on argument {i}")
                    view = list(args)
                    view[i] = dual[i].view(args[i].shape)
                    with pytest.raises(ParametersInvalid):
                        fn(*view)
                        pytest.fail(f"{name} took the view of a tensor with a tangent as argument {i}")
                    fn(*args)
                    with torch.inference_mode():  # where none is computed
                        fn(*dual)
            def of_one(v):
                out = fn(*args[:i], v, *args[i + 1:])
                return (out[0] if isinstance(out, tuple) else out).float().sum()
            with pytest.raises(ParametersInvalid):
                torch.func.jvp(of_one, (args[i],), (torch.ones_like(args[i]),))
                pytest.fail(f"{name} took the tangent of a transform on argument {i}")
            with pytest.raises(ParametersInvalid):
                torch.func.grad(of_one)(args[i])
                pytest.fail(f"{name} took a transform's input that wants a gradient as argument {i}")
            with pytest.raises(ParametersInvalid):
                of_one(args[i].clone().requires_grad_())
            # a transform of something else leaves the call alone
            other = torch.ones(3, device=device)
            value, tangent = torch.func.jvp(lambda u: u.sum() + 0 * of_one(args[i]), (other,), (other,))
            assert value.shape == tangent.shape == ()


def test_tangents_are_refused():
    _check("meta")


@pytest.mark.gpu
def test_tangents_are_refused_on_the_device():
    _check("cuda")
