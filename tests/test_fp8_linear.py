"""`FP8DynamicLinear`, and the operators around attention run together as a transformer block uses them: norm with
quantised output -> packed projection -> attention -> projection with gate and residual -> norm -> feed-forward.

Every step is compared with the 64-bit formula on what the step before it really produced, with the tolerance of that
step (test_linear_forward.py, test_add_rms_norm.py), so an error cannot hide behind the next step's rounding."""
import pytest
import torch

import test_add_rms_norm as tn
import test_linear_forward as tl
from oracle import attention as oa
from oracle import block_linear as ob


def test_refusals():
    from mindiesd import FP8DynamicLinear, ParametersInvalid
    w8 = torch.zeros(8, 16, dtype=torch.float8_e4m3fn, device="meta")
    for weights in (None, {}, {"p.weight": torch.zeros(8)}, {"p.weight": w8},
                    {"p.weight": torch.zeros(8, 16), "p.weight_scale": torch.zeros(8)},
                    {"p.weight": w8, "p.weight_scale": torch.zeros(7)}, {"p.weight": w8, "p.weight_scale": torch.zeros(8).half()},
                    {"p.weight": torch.zeros(8, 16)}):  # quantising needs a CUDA device
        with pytest.raises(ParametersInvalid):
            FP8DynamicLinear("p", weights)
    layer = FP8DynamicLinear("p", {"p.weight": w8, "p.weight_scale": torch.zeros(8, 1, device="meta")})
    q = torch.zeros(3, 16, dtype=torch.float8_e4m3fn, device="meta")
    for x in ((q,), (q, None), (q, torch.zeros(2, 1, device="meta")), [q], torch.zeros(3, 15, dtype=torch.bfloat16, device="meta"),
              torch.zeros(3, 16, device="meta").double()):
        with pytest.raises(ParametersInvalid):
            layer(x)
    assert layer((q, torch.zeros(3, 1, device="meta"))).shape == (3, 8)
    assert layer(torch.zeros(3, 16, dtype=torch.float16, device="meta")).dtype == torch.float16
    assert layer(torch.zeros(3, 16, device="meta")).dtype == torch.bfloat16
    assert set(layer.state_dict()) == {"weight", "weight_scale"}


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 5, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer(m, dtype):
    from mindiesd import FP8DynamicLinear
    from mindiesd.layers.quant import token_quant_preprocess
    linear = torch.nn.Linear(384, 264, device="cuda", dtype=dtype)
    layer = FP8DynamicLinear.from_linear(linear)
    tn._close_quant(layer.weight, layer.weight_scale[:, None], linear.weight.detach().double())
    x = tn._randn(m, 2, m, 384, dtype=dtype)
    q, scale = token_quant_preprocess(x)
    kw = dict(x_scale=scale, weight_scale=layer.weight_scale, bias=layer.bias)
    got = layer(x)
    tl._check(got, q, layer.weight, dtype, 384, **kw)
    assert torch.equal(layer((q, scale), out_dtype=dtype), got)
    r = tn._randn(m + 1, 2, m, 264, dtype=dtype)
    g = tn._randn(m + 2, 2, 1, 264)
    tl._check(layer(x, activation="silu", residual=r, gate=g), q, layer.weight, dtype, 384, act="silu", residual=r, gate=g, **kw)
    again = FP8DynamicLinear("a", {"a.weight": layer.weight, "a.weight_scale": layer.weight_scale, "a.bias": layer.bias})
    assert torch.equal(again(x), got)
    # the layer as a whole stays close to the one it was made from: e4m3 on both sides, 384 products of independent
    # rounding errors of at most 2^-4 each per operand
    err = (got.double() - linear(x).detach().double()).norm() / linear(x).detach().double().norm()
    assert err < 2 * 2.0 ** -4


def _block(x, shift, p, heads, quantised):
    """One pass through a block; returns every intermediate."""
    from mindiesd import add_rms_norm, add_rms_norm_quant, attention_forward, linear_forward
    b, s, dim = x.shape
    got = {}
    if quantised:
        got["h"], got["total"] = (lambda r: (r[:2], r[2]))(add_rms_norm_quant(shift, p["norm1"], x))
        got["qkv"] = p["qkv8"](got["h"])
    else:
        got["h"], got["total"] = add_rms_norm(shift, p["norm1"], x)
        got["qkv"] = linear_forward(got["h"], p["qkv"], p["qkv_bias"])
    q, k, v = got["qkv"].view(b, s, 3, heads, 128).unbind(2)  # read in place, head slices of the packed projection
    got["attn"] = attention_forward(q, k, v)
    flat = got["attn"].reshape(b, s, dim)
    got["x1"] = linear_forward(flat, p["out"], p["out_bias"], residual=got["total"], gate=p["gate1"])
    if quantised:
        got["h2"] = add_rms_norm_quant(got["x1"], p["norm2"])
        got["up"] = p["up8"](got["h2"], activation="gelu_tanh")
        got["x2"] = p["down8"](got["up"], residual=got["x1"], gate=p["gate2"])
    else:
        got["h2"] = add_rms_norm(got["x1"], p["norm2"])
        got["up"] = linear_forward(got["h2"], p["up"], p["up_bias"], activation="gelu_tanh")
        got["x2"] = linear_forward(got["up"], p["down"], None, residual=got["x1"], gate=p["gate2"])
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("b,s", [(1, 1), (2, 77), (1, 700)])
def test_block(b, s, quantised):
    from mindiesd import FP8DynamicLinear
    from mindiesd.layers.quant import token_quant_preprocess
    t, heads, dim, ff = torch.bfloat16, 2, 256, 1024

    def w(seed, n, k):
        return tn._randn(seed, n, k, dtype=t, scale=k ** -0.5)
    p = {"norm1": 1 + 0.1 * tn._randn(1, dim), "norm2": tn._randn(2, dim, dtype=t), "qkv": w(3, 3 * dim, dim),
         "qkv_bias": tn._randn(4, 3 * dim, dtype=t), "out": w(5, dim, dim), "out_bias": tn._randn(6, dim), "up": w(7, ff, dim),
         "up_bias": tn._randn(8, ff, dtype=t), "down": w(9, dim, ff), "gate1": tn._randn(10, b, 1, dim), "gate2": tn._randn(11, b, 1, dim)}
    p["qkv8"] = FP8DynamicLinear("m", {"m.weight": p["qkv"], "m.bias": p["qkv_bias"]})
    p["up8"] = FP8DynamicLinear("m", {"m.weight": p["up"], "m.bias": p["up_bias"]})
    p["down8"] = FP8DynamicLinear("m", {"m.weight": p["down"]})
    x, shift = tn._randn(12, b, s, dim, dtype=t), tn._randn(13, b, s, dim, dtype=t)
    g = _block(x, shift, p, heads, quantised)

    y, total = ob.rms_norm(shift, p["norm1"], x)
    tn._close(g["total"], total, t)
    y2, _ = ob.rms_norm(g["x1"], p["norm2"])
    if quantised:
        tn._close_quant(*g["h"], y)
        tl._check(g["qkv"], g["h"][0], p["qkv8"].weight, t, dim, x_scale=g["h"][1], weight_scale=p["qkv8"].weight_scale, bias=p["qkv_bias"])
        tn._close_quant(*g["h2"], y2)
        tl._check(g["up"], g["h2"][0], p["up8"].weight, t, dim, act="gelu_tanh", x_scale=g["h2"][1],
                  weight_scale=p["up8"].weight_scale, bias=p["up_bias"])
        q, scale = token_quant_preprocess(g["up"])
        tl._check(g["x2"], q, p["down8"].weight, t, ff, residual=g["x1"], gate=p["gate2"], x_scale=scale,
                  weight_scale=p["down8"].weight_scale)
    else:
        tn._close(g["h"], y, t)
        tl._check(g["qkv"], g["h"], p["qkv"], t, dim, bias=p["qkv_bias"])
        tn._close(g["h2"], y2, t)
        tl._check(g["up"], g["h2"], p["up"], t, dim, act="gelu_tanh", bias=p["up_bias"])
        tl._check(g["x2"], g["up"], p["down"], t, ff, residual=g["x1"], gate=p["gate2"])
    q, k, v = (z.contiguous() for z in g["qkv"].view(b, s, 3, heads, 128).unbind(2))
    want = oa.attention_math(q.cpu(), k.cpu(), v.cpu(), head_first=False)
    assert (g["attn"].float().cpu() - want.float()).abs().max().item() <= 2e-2 * max(1.0, want.float().abs().max().item())
    tl._check(g["x1"], g["attn"].reshape(b, s, dim), p["out"], t, dim, bias=p["out_bias"], residual=g["total"], gate=p["gate1"])

    # the whole block in one graph, replayed on new data
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _block(x, shift, p, heads, quantised)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _block(x, shift, p, heads, quantised)["x2"]
    x.copy_(tn._randn(14, b, s, dim, dtype=t))
    graph.replay()
    assert torch.equal(captured, _block(x, shift, p, heads, quantised)["x2"])


@pytest.mark.gpu
def test_calls_back_to_back():
    """The start of each kernel may overlap the end of the one before it.  A chain in which every call reads what
    the call before has just written, into memory that an earlier one has just read, gives the same bits as
    the chain with a synchronisation after every call -- eager, and replayed as one graph."""
    from mindiesd import add_rms_norm, linear_forward
    from mindiesd.layers.quant import token_quant_preprocess
    for m in (1, 70, 600):
        w1, w2 = tn._randn(1, 1024, 256, dtype=torch.bfloat16, scale=1 / 16), tn._randn(2, 256, 1024, dtype=torch.bfloat16, scale=1 / 32)
        w8, ws = token_quant_preprocess(w2)
        start = tn._randn(3, m, 256, dtype=torch.bfloat16)

        def chain(x, pause):
            total = x
            for _ in range(12):
                y, total = add_rms_norm(x, None, total)
                pause()
                h = linear_forward(y, w1, activation="silu")
                pause()
                q, s = token_quant_preprocess(h)
                pause()
                x = linear_forward(q, w8, x_scale=s, weight_scale=ws, residual=total)
                pause()
                x = x + 0.5 * linear_forward(h, w2)  # torch's own kernels in between
                pause()
                del y, h, q, s
            return x
        want = chain(start, torch.cuda.synchronize)
        for _ in range(5):
            assert torch.equal(chain(start, lambda: None), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = chain(start, lambda: None)
        for _ in range(5):
            got.zero_()
            graph.replay()
            assert torch.equal(got, want)


@pytest.mark.parametrize("convert,bias_dtype", [(lambda m: m.to(torch.bfloat16), torch.bfloat16), (lambda m: m.half(), torch.float16),
                                                (lambda m: m.float(), torch.float32), (lambda m: m.to("cpu", torch.float16), torch.float16),
                                                (lambda m: m.type(torch.bfloat16), torch.bfloat16), (lambda m: m.half().bfloat16(), torch.bfloat16)])
def test_dtype_conversions_leave_the_stored_weights(convert, bias_dtype):
    """Of a module that holds the layer, and of the layer itself: the e4m3 values and their scales keep type and bits."""
    from mindiesd import FP8DynamicLinear
    g = torch.Generator().manual_seed(1)
    weight = torch.randn(8, 16, generator=g).to(torch.float8_e4m3fn)
    scale, bias = torch.rand(8, generator=g), torch.randn(8, generator=g)
    for wrap in (lambda layer: layer, lambda layer: torch.nn.Sequential(torch.nn.Linear(16, 16), layer)):
        layer = FP8DynamicLinear("p", {"p.weight": weight, "p.weight_scale": scale, "p.bias": bias})
        convert(wrap(layer))
        assert layer.weight.dtype == torch.float8_e4m3fn and torch.equal(layer.weight.float(), weight.float())
        assert layer.weight_scale.dtype == torch.float32 and torch.equal(layer.weight_scale, scale)
        assert layer.bias.dtype == bias_dtype
    layer.to("meta")
    assert layer.weight.is_meta and layer.weight_scale.is_meta and layer.weight.dtype == torch.float8_e4m3fn
    assert layer(torch.zeros(3, 16, dtype=bias_dtype, device="meta")).shape == (3, 8)
    layer.to_empty(device="cpu")
    assert layer.weight.device.type == "cpu" and layer.weight.dtype == torch.float8_e4m3fn and layer.weight_scale.dtype == torch.float32


@pytest.mark.gpu
def test_converted_layer_runs():
    from mindiesd import FP8DynamicLinear
    linear = torch.nn.Linear(384, 264, device="cuda", dtype=torch.bfloat16)
    layer = FP8DynamicLinear.from_linear(linear)
    x = tn._randn(1, 5, 384, dtype=torch.bfloat16)
    want = layer(x)
    for convert in (lambda m: m.to(torch.float32), lambda m: m.to(torch.bfloat16), lambda m: m.cpu().bfloat16().cuda()):
        convert(torch.nn.Sequential(layer))
        assert layer.weight.is_cuda and layer.weight_scale.is_cuda
        assert torch.equal(layer(x), want)
