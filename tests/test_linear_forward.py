"""`linear_forward`: refusals on the host, values on a GPU against the 64-bit formula.

Tolerances: one last rounding (half a step relative to the value), plus the fp32 accumulation: products of two-byte
or e4m3 values are exact in fp32, a tensor-core instruction adds at least 8 of them to a running sum that may be
truncated, so each step is off by at most 2^-23 of the largest partial sum, which the sum of |x||w| bounds:
(K/8 + 8) 2^-23 sum|x||w| (carried through the epilogue by the oracle).  The activations' own error is below 2^-15
relative: their exponent's argument is rounded to fp32 (|v| < 90 times 2^-24 times log2 e) and erfc amplifies its
argument's rounding by v^2."""
import ctypes

import pytest
import torch

from oracle import block_linear as ob

ACT_SLACK = 2.0 ** -15


def _randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _operands(seed, m, k, n, dtype):
    """(x, weight, keyword arguments): e4m3 operands come with their scales."""
    if dtype != torch.float8_e4m3fn:
        return _randn(seed, m, k, dtype=dtype), _randn(seed + 1, n, k, dtype=dtype, scale=k ** -0.5), {}
    from mindiesd.layers.quant import token_quant_preprocess
    x, xs = token_quant_preprocess(_randn(seed, m, k))
    w, ws = token_quant_preprocess(_randn(seed + 1, n, k, scale=k ** -0.5))
    return x, w, dict(x_scale=xs, weight_scale=ws)


def _check(got, x, w, out_dtype, k, **kw):
    want, size = ob.linear(x, w, **kw)
    assert got.dtype == out_dtype and got.shape == want.shape
    tol = want.abs() * (ob.half_step(out_dtype) + ACT_SLACK) + ob.smallest_half_step(out_dtype) + size * (k / 8 + 8) * 2.0 ** -23
    worst = ((got.double() - want).abs() - tol).max().item()
    assert worst <= 0, worst


# ---- host ------------------------------------------------------------------------------------------

def test_codes_without_a_gpu(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path
    from mindiesd import _cabi
    fn = _cabi.lib().mindiesd_linear_fwd
    a = _cabi.LinearArgs()
    assert fn(None, None) == -1 and fn(ctypes.byref(a), None) == -1
    a.x = a.weight = a.out = 4096
    assert fn(ctypes.byref(a), None) == -2
    a.m, a.n, a.k = 4, 64, 64
    a.x_stride = a.weight_stride = a.out_stride = 64
    for field, value, code in [("in_dtype", _cabi.FP32, -3), ("out_dtype", _cabi.FP32, -3), ("in_dtype", _cabi.E4M3, -1),
                               ("x_scale", 4096, -5), ("activation", 5, -5), ("activation", -1, -5), ("x_stride", 0, -4),
                               ("x_stride", 63, -4), ("weight_stride", 0, -4), ("out_stride", 32, -4), ("out", 4097, -4),
                               ("m", 0x7fffffff, -7), ("n", 0, -2), ("k", -1, -2)]:
        b = _cabi.LinearArgs.from_buffer_copy(a)
        setattr(b, field, value)
        assert fn(ctypes.byref(b), None) == code, (field, value)
    b = _cabi.LinearArgs.from_buffer_copy(a)
    b.bias, b.bias_dtype = 4096, _cabi.E4M3
    assert fn(ctypes.byref(b), None) == -3
    b.bias, b.bias_dtype = 4098, _cabi.FP32
    assert fn(ctypes.byref(b), None) == -4
    b = _cabi.LinearArgs.from_buffer_copy(a)
    b.gate = 4096
    assert fn(ctypes.byref(b), None) == -5  # no rows per gate
    b.rows_per_gate, b.gate_stride = 4, -64
    assert fn(ctypes.byref(b), None) == -4
    cc = shutil.which("gcc")
    if cc:
        src = tmp_path / "s.c"
        src.write_text('#include <stdio.h>\n#include "mindiesd_b200.h"\nint main(void){printf("%zu",sizeof(mindiesd_linear_args));return 0;}\n')
        inc = Path(__file__).resolve().parent.parent / "include"
        subprocess.run([cc, "-I", str(inc), str(src), "-o", str(tmp_path / "s")], check=True)
        assert int(subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout) == \
            ctypes.sizeof(_cabi.LinearArgs)


def _refused(device):
    """(calls that are refused, calls that are not) with every tensor on `device`."""
    def t(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype, device=device)
    x, w = t(2, 5, 64), t(32, 64)
    x8, w8 = t(2, 5, 64, dtype=torch.float8_e4m3fn), t(32, 64, dtype=torch.float8_e4m3fn)
    s, ws = t(2, 5, 1, dtype=torch.float32), t(32, dtype=torch.float32)
    bad = [
        dict(x=[1.0], weight=w), dict(x=x, weight=None), dict(x=x, weight=t(32, 63)), dict(x=x, weight=t(32, 64, 1)),
        dict(x=x, weight=t(0, 64)), dict(x=t(5, 0), weight=t(32, 0)), dict(x=t(), weight=w), dict(x=x.float(), weight=w.float()),
        dict(x=x, weight=w.half()), dict(x=x, weight=torch.zeros(32, 64, dtype=torch.bfloat16)),
        dict(x=torch.zeros(5, 64, dtype=torch.bfloat16), weight=torch.zeros(32, 64, dtype=torch.bfloat16)),
        dict(x=x, weight=w, activation="swish"), dict(x=x, weight=w, activation=None), dict(x=x, weight=w, out_dtype=torch.float32),
        dict(x=x, weight=w, bias=t(33)), dict(x=x, weight=w, bias=t(1, 32)), dict(x=x, weight=w, bias=t(32, dtype=torch.float64)),
        dict(x=x, weight=w, bias=torch.zeros(32)), dict(x=x, weight=w, bias=0.0),
        dict(x=x, weight=w, residual=t(2, 5, 33)), dict(x=x, weight=w, residual=t(10, 32)), dict(x=x, weight=w, residual=t(2, 5, 32).half()),
        dict(x=x, weight=w, residual=torch.zeros(2, 5, 32, dtype=torch.bfloat16)),
        dict(x=x, weight=w, gate=t(31)), dict(x=x, weight=w, gate=t(3, 1, 32)), dict(x=x, weight=w, gate=t(2, 5, 32)),
        dict(x=x, weight=w, gate=t(5, 32)), dict(x=x, weight=w, gate=t(32, dtype=torch.int32)), dict(x=t(64), weight=w, gate=t(2, 32)),
        dict(x=x, weight=w, x_scale=s, weight_scale=ws), dict(x=x8, weight=w8), dict(x=x8, weight=w8, x_scale=s),
        dict(x=x8, weight=w, x_scale=s, weight_scale=ws), dict(x=x8, weight=w8, x_scale=s.half(), weight_scale=ws),
        dict(x=x8, weight=w8, x_scale=t(10, dtype=torch.float32), weight_scale=ws),
        dict(x=x8, weight=w8, x_scale=s, weight_scale=t(31, dtype=torch.float32)),
        dict(x=x8, weight=w8, x_scale=s, weight_scale=1.0), dict(x=x8, weight=w8, x_scale=s, weight_scale=torch.zeros(32)),
        dict(x=x8, weight=w8, x_scale=s, weight_scale=ws, residual=t(2, 5, 32, dtype=torch.float32)),
        dict(x=x, weight=torch.nn.Parameter(w)), dict(x=x, weight=w, bias=t(32).requires_grad_()),
        dict(x=x.clone().requires_grad_(), weight=w), dict(x=x, weight=w, gate=t(32).requires_grad_()),
    ]
    good = [dict(x=x, weight=w), dict(x=x8, weight=w8, x_scale=s, weight_scale=ws), dict(x=x, weight=w, gate=t(1, 1, 1, 32)),
            dict(x=x8, weight=w8, x_scale=s[..., 0], weight_scale=ws[:, None], residual=t(2, 5, 32).half())]
    return bad, good


def test_refusals():
    from mindiesd import ParametersInvalid, linear_forward
    bad, good = _refused("meta")
    for kw in bad:
        with pytest.raises(ParametersInvalid):
            linear_forward(**kw)
    assert [linear_forward(**kw).dtype for kw in good] == [torch.bfloat16, torch.bfloat16, torch.bfloat16, torch.float16]
    assert all(linear_forward(**kw).shape == (2, 5, 32) for kw in good)
    with torch.no_grad():
        assert linear_forward(good[0]["x"][0, 0], torch.nn.Parameter(good[0]["weight"])).shape == (32,)


@pytest.mark.gpu
def test_refusals_on_the_device():
    """The operator makes the checks itself on the way to the kernel; nothing is launched for a refused call."""
    from mindiesd import ParametersInvalid, linear_forward
    bad, good = _refused("cuda")
    for i, kw in enumerate(bad):
        with pytest.raises(ParametersInvalid):
            linear_forward(**kw)
            pytest.fail(f"call {i} was taken")
    for kw in good:
        assert linear_forward(**kw).shape == (2, 5, 32)
    torch.cuda.synchronize()


# ---- GPU -------------------------------------------------------------------------------------------

# Both kernels, one and several blocks or tiles along every side, shares of k down to a step, every width of tile.
SHAPES = [(1, 256, 5120), (2, 64, 16), (1, 1, 1), (3, 8, 130), (16, 1001, 129), (17, 200, 1000), (64, 1536, 1536), (100, 4096, 257),
          (128, 72, 256), (129, 72, 256), (200, 520, 33), (256, 64, 256), (257, 1024, 1000), (300, 1536, 1001), (513, 5120, 640),
          (1000, 333, 514), (2048, 128, 2048), (5000, 256, 96),
          (1, 20480, 640), (33, 9000, 700), (150, 2000, 1100), (260, 15000, 100), (512, 1024, 2560), (1100, 512, 3500),
          (1500, 64, 9000), (4100, 768, 24), (700, 1536, 6144), (2500, 640, 5000)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
def test_product(m, k, n, dtype):
    from mindiesd import linear_forward
    x, w, kw = _operands(m + k + n, m, k, n, dtype)
    for out_dtype in (torch.bfloat16, torch.float16):
        _check(linear_forward(x, w, out_dtype=out_dtype, **kw), x, w, out_dtype, k, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(2, 200, 264), (48, 136, 129), (258, 320, 200), (600, 64, 333)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_epilogue(m, k, n, dtype, act):
    from mindiesd import linear_forward
    x, w, kw = _operands(m, m, k, n, dtype)
    for bias_dtype, gate_dtype, out_dtype in [(torch.bfloat16, torch.float32, torch.bfloat16), (torch.float32, torch.float16, torch.float16),
                                              (None, torch.bfloat16, torch.bfloat16), (torch.float16, None, torch.float16)]:
        full = dict(kw)
        if bias_dtype is not None:
            full["bias"] = _randn(5, n, dtype=bias_dtype, scale=2.0)
        if gate_dtype is not None:
            full["gate"] = _randn(6, n, dtype=gate_dtype)
        full["residual"] = _randn(7, m, n, dtype=out_dtype)
        got = linear_forward(x, w, activation=act, out_dtype=out_dtype, **full)
        _check(got, x, w, out_dtype, k, act=act, **full)
        del full["residual"]
        got = linear_forward(x, w, activation=act, out_dtype=out_dtype, **full)
        _check(got, x, w, out_dtype, k, act=act, **full)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,rows", [(2, 3), (3, 40), (2, 300), (5, 130), (7, 1)])
def test_gate_per_sample(batch, rows):
    from mindiesd import linear_forward
    x, w, _ = _operands(9, batch * rows, 192, 136, torch.bfloat16)
    x = x.view(batch, rows, 192)
    gate, residual = _randn(10, batch, 1, 136), _randn(11, batch, rows, 136, dtype=torch.bfloat16)
    got = linear_forward(x, w, gate=gate, residual=residual)
    _check(got, x, w, torch.bfloat16, 192, gate=gate, residual=residual)
    assert torch.equal(got, linear_forward(x, w, gate=gate[:, 0], residual=residual))
    flat = linear_forward(x.reshape(-1, 192), w, gate=gate.expand(batch, rows, 136).reshape(-1, 136), residual=residual.reshape(-1, 136))
    assert torch.equal(flat.view_as(got), got)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 300])
def test_strides_and_alignment(m):
    """Slices of packed projections, transposes, broadcast rows, odd starts: read in place or copied, same answer."""
    from mindiesd import linear_forward
    k, n = 128, 72
    pool = _randn(20, m, 3 * k + 8, dtype=torch.float16)
    wpool = _randn(21, n, 2 * k + 8, dtype=torch.float16, scale=0.1)
    rpool = _randn(22, m, 2 * n + 1, dtype=torch.float16)
    for x in (pool[:, k:2 * k], pool[:, 3:3 + k], pool[:, :3 * k:3], pool[:1, :k].expand(m, k), _randn(23, k, m, dtype=torch.float16).t()):
        for w in (wpool[:, k:2 * k], wpool[:, 1:1 + k], wpool[:1, :k].expand(n, k)):
            for r in (rpool[:, :n], rpool[:, n:2 * n], rpool[:, :2 * n:2], rpool[:1, :n].expand(m, n)):
                _check(linear_forward(x, w, residual=r), x, w, torch.float16, k, residual=r)
    bias = _randn(24, 2 * n + 1)
    for b in (bias[1:1 + n], bias[:2 * n:2]):
        _check(linear_forward(pool[:, :k], wpool[:, :k], b), pool[:, :k], wpool[:, :k], torch.float16, k, bias=b)


@pytest.mark.gpu
def test_single_scales_and_three_dimensions():
    from mindiesd import linear_forward
    for m in (6, 400):
        x = _randn(30, 2, m // 2, 96).to(torch.float8_e4m3fn)
        w = _randn(31, 40, 96).to(torch.float8_e4m3fn)
        kw = dict(x_scale=torch.tensor([0.37], device="cuda"), weight_scale=torch.tensor(0.11, device="cuda"))
        _check(linear_forward(x, w, **kw), x, w, torch.bfloat16, 96, **kw)
    x, w, _ = _operands(32, 1, 96, 40, torch.bfloat16)
    assert torch.equal(linear_forward(x[0], w), linear_forward(x, w)[0])
    assert linear_forward(x[:0], w).shape == (0, 40)
    assert linear_forward(x.view(1, 1, 96)[:, :0], w, gate=_randn(33, 40)).shape == (1, 0, 40)


@pytest.mark.gpu
def test_rows_do_not_depend_on_their_neighbours():
    """A NaN or an infinity stays in its row (or in its column, when it is in the weights)."""
    from mindiesd import linear_forward
    for m in (9, 300):
        x, w, _ = _operands(40, m, 320, 200, torch.bfloat16)
        clean = linear_forward(x, w)
        x2, w2 = x.clone(), w.clone()
        x2[3, 17] = float("nan")
        w2[11, 5] = float("inf")
        got = linear_forward(x2, w2)
        assert torch.isnan(got[3].float()).all() and not torch.isfinite(got[:, 11].float()).any()
        keep = torch.ones_like(got, dtype=torch.bool)
        keep[3] = False
        keep[:, 11] = False
        assert torch.equal(got[keep], clean[keep])


@pytest.mark.gpu
def test_repeatable_on_streams_and_in_graphs():
    from mindiesd import linear_forward
    for m in (4, 700):
        x, w, _ = _operands(50, m, 4096, 384, torch.bfloat16)
        first = linear_forward(x, w)
        streams = [torch.cuda.Stream() for _ in range(3)]
        outs = []
        for s in streams:  # several calls at once, of both kernels: nothing is shared between them
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs += [linear_forward(x, w) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(first, o) for o in outs)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = linear_forward(x, w)
        x.copy_(_randn(51, m, 4096, dtype=torch.bfloat16))
        graph.replay()
        assert torch.equal(captured, linear_forward(x, w))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 700])
def test_withheld_copies_give_up_cleanly(m):
    from mindiesd import _cabi, linear_forward
    assert _cabi.device_status() == 0
    x, w, _ = _operands(60, m, 1024, 2048, torch.bfloat16)
    out = torch.zeros(m, 2048, dtype=torch.bfloat16, device="cuda")
    a = _cabi.LinearArgs()
    a.x, a.weight, a.out = x.data_ptr(), w.data_ptr(), out.data_ptr()
    a.x_stride = a.weight_stride = 1024
    a.out_stride, a.m, a.n, a.k = 2048, m, 2048, 1024
    a.in_dtype = a.out_dtype = _cabi.BF16
    a.wait_limit_us, a.test_withhold = 20000, 1
    _cabi.check(_cabi.lib().mindiesd_linear_fwd(ctypes.byref(a), _cabi.current_stream_ptr(x.device)), "mindiesd_linear_fwd")
    torch.cuda.synchronize()
    assert torch.isnan(out.float()).all()
    assert torch.isnan(linear_forward(x, w).float()).all()  # while the word is set, later launches mark their rows too
    assert _cabi.device_status() == 105 and _cabi.device_status() == 0
    _check(linear_forward(x, w), x, w, torch.bfloat16, 1024)
    assert _cabi.device_status() == 0


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    from mindiesd import linear_forward
    x = torch.zeros(1100000, 64, dtype=torch.bfloat16, device="cuda")
    x[-2:] = _randn(70, 2, 64, dtype=torch.bfloat16)
    w = _randn(71, 2048, 64, dtype=torch.bfloat16)
    out = linear_forward(x, w)  # 2.25e9 elements
    _check(out[-2:], x[-2:], w, torch.bfloat16, 64)
    assert torch.count_nonzero(out[-300:-2]).item() == 0


@pytest.mark.gpu
def test_first_calls_of_a_process_may_be_captured():
    """Nothing that the operators set up once (limits, tables) needs a call before the capture."""
    import subprocess
    import sys
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    code = (
        "import sys, torch; sys.path.insert(0, 'mindie-sd_b200')\n"
        "from mindiesd import add_rms_norm_quant, linear_forward\n"
        "x, w = torch.ones(700, 512, device='cuda', dtype=torch.bfloat16), torch.ones(256, 512, device='cuda', dtype=torch.bfloat16)\n"
        "torch.cuda.synchronize(); g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g):\n"
        "    a, b, (q, s) = linear_forward(x, w), linear_forward(x[:3], w), add_rms_norm_quant(x)\n"
        "g.replay(); torch.cuda.synchronize()\n"
        "assert (a == 512).all() and (b == 512).all() and (q.float() * s - 1).abs().max() < 1e-5\n"
        "print('captured')\n")
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=200)
    assert run.returncode == 0 and "captured" in run.stdout, run.stderr[-2000:]


@pytest.mark.gpu
def test_threads_call_at_once():
    """Calls of different sizes from several host threads, each on its own stream."""
    import threading
    from mindiesd import linear_forward
    work = [_operands(80 + i, m, 512, n, torch.bfloat16)[:2] for i, (m, n) in enumerate([(1, 640), (300, 256), (40, 1000), (900, 128)])]
    want = [linear_forward(x, w) for x, w in work]
    torch.cuda.synchronize()
    wrong = []

    def loop(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                if not torch.equal(linear_forward(*work[i]), want[i]):
                    wrong.append(i)
    threads = [threading.Thread(target=loop, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(1, 136), (7, 136), (100, 131), (300, 200), (300, 131), (515, 520)])
def test_strided_output_leaves_the_rest_alone(m, n):
    """Through the C ABI: an output whose rows lie in wider ones, residual and gate with strides of their own; columns and
    rows beyond the product keep what they held."""
    from mindiesd import _cabi
    k = 192
    x, w, _ = _operands(90, m, k, n, torch.bfloat16)
    for start, pad in ((0, 24), (8, 40), (3, 17)):
        wide = torch.full((m + 5, n + pad), 7.0, dtype=torch.bfloat16, device="cuda")
        out = wide[2:2 + m, start:start + n]
        r, g = _randn(91, m, n + 9, dtype=torch.bfloat16)[:, 1:1 + n], _randn(92, m, n + 3)[:, :n]
        a = _cabi.LinearArgs()
        a.x, a.weight, a.out, a.residual, a.gate = x.data_ptr(), w.data_ptr(), out.data_ptr(), r.data_ptr(), g.data_ptr()
        a.x_stride = a.weight_stride = k
        a.out_stride, a.residual_stride, a.gate_stride = wide.stride(0), r.stride(0), g.stride(0)
        a.m, a.n, a.k, a.rows_per_gate = m, n, k, 1
        a.in_dtype = a.out_dtype = _cabi.BF16
        a.gate_dtype = _cabi.FP32
        _cabi.check(_cabi.lib().mindiesd_linear_fwd(ctypes.byref(a), _cabi.current_stream_ptr(x.device)), "mindiesd_linear_fwd")
        _check(out, x, w, torch.bfloat16, k, residual=r, gate=g)
        keep = torch.ones_like(wide, dtype=torch.bool)
        keep[2:2 + m, start:start + n] = False
        assert (wide[keep] == 7).all()


@pytest.mark.gpu
def test_fork_and_join_in_a_graph():
    """Calls with several predecessors: a captured side stream that joins the main one."""
    from mindiesd import add_rms_norm, linear_forward
    for m in (3, 400):
        x, w, _ = _operands(95, m, 256, 256, torch.bfloat16)

        def run():
            main = torch.cuda.current_stream()
            y = add_rms_norm(x)
            side.wait_stream(main)
            with torch.cuda.stream(side):
                z = linear_forward(y, w)
            u = linear_forward(y, w, activation="silu")
            main.wait_stream(side)
            return add_rms_norm(linear_forward(u, w, residual=z), None, z)[1]
        side = torch.cuda.Stream()
        want = run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
        for _ in range(3):
            got.zero_()
            graph.replay()
            assert torch.equal(got, want)


@pytest.mark.gpu
def test_failed_launch_leaves_no_error_behind():
    """An address that the copy engine cannot take is refused by its code, and the next call is not disturbed."""
    from mindiesd import _cabi, linear_forward
    x, w, _ = _operands(97, 8, 64, 64, torch.bfloat16)
    out = torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    a = _cabi.LinearArgs()
    a.x, a.weight, a.out = x.data_ptr() + 2, w.data_ptr(), out.data_ptr()
    a.x_stride = a.weight_stride = a.out_stride = 64
    a.m, a.n, a.k = 7, 64, 64
    a.in_dtype = a.out_dtype = _cabi.BF16
    assert _cabi.lib().mindiesd_linear_fwd(ctypes.byref(a), _cabi.current_stream_ptr(x.device)) == -4
    torch.cuda.synchronize()
    assert torch.count_nonzero(out).item() == 0
    _check(linear_forward(x, w), x, w, torch.bfloat16, 64)


def test_copy_rows_refusals_without_a_gpu(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path
    from mindiesd import _cabi
    fn = _cabi.lib().mindiesd_copy_rows

    def code(**changes):
        a = _cabi.CopyRowsArgs(src=1 << 20, dst=2 << 20, rows=4, row_bytes=100, src_stride=100, dst_stride=128)
        for name, value in changes.items():
            setattr(a, name, value)
        return fn(ctypes.byref(a), None)
    assert fn(None, None) == -1 and code(src=None) == -1 and code(dst=None) == -1
    assert code(rows=0) == -2 and code(row_bytes=0) == -2 and code(row_bytes=-1) == -2
    assert code(rows=1 << 31) == -7 and code(row_bytes=1 << 34) == -7
    assert code(rows=0x7fffffff, row_bytes=1 << 24, dst_stride=1 << 24) == -7  # more blocks than a grid has
    assert code(src_stride=-100) == -4 and code(dst_stride=96) == -4 and code(dst_stride=120) == -4 and code(dst=(2 << 20) + 8) == -4
    assert code(dst=(1 << 20) + 384) == -5 and code(src=(2 << 20) + 3 * 128 + 111) == -5  # they overlap by a byte
    cc = shutil.which("gcc")
    if cc:
        src = tmp_path / "s.c"
        src.write_text('#include <stdio.h>\n#include "mindiesd_b200.h"\nint main(void){printf("%zu",sizeof(mindiesd_copy_rows_args));return 0;}\n')
        inc = Path(__file__).resolve().parent.parent / "include"
        subprocess.run([cc, "-I", str(inc), str(src), "-o", str(tmp_path / "s")], check=True)
        assert int(subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout) == ctypes.sizeof(_cabi.CopyRowsArgs)


@pytest.mark.gpu
@pytest.mark.parametrize("row_bytes", [1, 2, 12, 40, 511, 512, 2048, 2064, 4098, 10001])
@pytest.mark.parametrize("start,gap", [(0, 0), (1, 0), (2, 6), (4, 12), (8, 8), (16, 48)])
def test_copy_rows(row_bytes, start, gap):
    """Every width of piece, one segment of a row and several: the rows, zeros up to 16 bytes, and nothing behind."""
    from mindiesd import _cabi
    rows, stride, wide = 37, row_bytes + gap, (row_bytes + 15) // 16 * 16 + 32
    buf = torch.randint(0, 256, (start + rows * stride,), dtype=torch.uint8, device="cuda")
    src = buf[start:].view(rows, stride)[:, :row_bytes]
    for step in (stride, 0):
        dst = torch.full((rows + 1, wide), 7, dtype=torch.uint8, device="cuda")
        a = _cabi.CopyRowsArgs(src.data_ptr(), dst.data_ptr(), rows, row_bytes, step, wide)
        _cabi.check(_cabi.lib().mindiesd_copy_rows(ctypes.byref(a), _cabi.current_stream_ptr(dst.device)), "mindiesd_copy_rows")
        assert torch.equal(dst[:rows, :row_bytes], src if step else src[:1].expand(rows, -1))
        assert (dst[:rows, row_bytes:wide - 32] == 0).all() and (dst[:rows, wide - 32:] == 7).all() and (dst[rows] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("m,k,n", [(4096, 2056, 2100), (20000, 1544, 1536), (600, 4104, 9000), (300, 520, 400)])
def test_rows_that_start_within_a_sector(m, k, n, dtype):
    """Rows on odd multiples of 16 bytes, which are copied first where that pays: the same bits as on aligned rows, whichever
    operand is so, on a stream of its own and replayed."""
    from mindiesd import linear_forward
    e = torch.empty(0, dtype=dtype).element_size()
    k = k if e == 2 else k + 8
    s = dict(x_scale=torch.full((1,), 0.5, device="cuda"), weight_scale=torch.full((1,), 2.0, device="cuda")) if e == 1 else {}

    def at(t, stride):
        wide = torch.zeros(t.shape[0], stride, dtype=torch.uint8, device="cuda").view(dtype)
        wide[:, :t.shape[1]].copy_(t)
        return wide[:, :t.shape[1]]
    x, w = (_randn(seed, rows, k, scale=0.1).to(dtype) for seed, rows in ((110, m), (111, n)))
    even, odd = (k * e + 127) // 128 * 128, (k * e + 127) // 128 * 128 + 16
    xe, xo, we, wo = at(x, even), at(x, odd), at(w, even), at(w, odd)
    want = linear_forward(xe, we, **s)
    for a, b in ((xo, wo), (xo, we), (xe, wo), (x, w)):
        assert torch.equal(linear_forward(a, b, **s), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [linear_forward(xo, wo, **s) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = linear_forward(xo, wo, **s)
    xo.copy_(_randn(112, m, k, scale=0.1).to(dtype))
    graph.replay()
    assert torch.equal(captured, linear_forward(at(xo, even), we, **s))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [256, 264, 260, 258, 257, 287])
def test_rows_of_every_piece(n, dtype):
    """Outputs and residuals whose rows can be moved 32, 16, 8 or 4 bytes at a time, or start between words in turn, each
    with the other on an address of its own; what surrounds the output stays."""
    from mindiesd import _cabi
    m, k = 4400, 64
    x, w, _ = _operands(120, m, k, n, dtype)
    for out_start, out_pad, res_start, res_pad in ((0, 0, 0, 0), (16, 32, 0, 16), (8, 8, 4, 4), (4, 4, 2, 2), (2, 2, 1, 1), (1, 1, 0, 3), (1, 16, 16, 16)):
        wide = torch.full((m + 2, n + out_pad + out_start), 7.0, dtype=dtype, device="cuda")
        out = wide[1:1 + m, out_start:out_start + n]
        r = _randn(121, m, n + res_pad + res_start, dtype=dtype)[:, res_start:res_start + n]
        a = _cabi.LinearArgs()
        a.x, a.weight, a.out, a.residual = x.data_ptr(), w.data_ptr(), out.data_ptr(), r.data_ptr()
        a.x_stride = a.weight_stride = k
        a.out_stride, a.residual_stride = wide.stride(0), r.stride(0)
        a.m, a.n, a.k = m, n, k
        a.in_dtype = a.out_dtype = _cabi.dtype_code(dtype)
        _cabi.check(_cabi.lib().mindiesd_linear_fwd(ctypes.byref(a), _cabi.current_stream_ptr(x.device)), "mindiesd_linear_fwd")
        _check(out, x, w, dtype, k, residual=r)
        keep = torch.ones_like(wide, dtype=torch.bool)
        keep[1:1 + m, out_start:out_start + n] = False
        assert (wide[keep] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m", [3, 700])
def test_activations_over_their_range(act, m):
    """One product per value (the other operand is the unit matrix), so the activation's own error shows: a fine sweep of
    both signs, the largest arguments, and what must come of an infinity and a NaN."""
    from mindiesd import linear_forward
    n = 128
    eye = torch.eye(n, dtype=torch.bfloat16, device="cuda")
    values = torch.cat([torch.linspace(-14, 14, m * n - 40, device="cuda"), torch.logspace(-30, 3, 20, device="cuda"),
                        -torch.logspace(-30, 3, 20, device="cuda")]).to(torch.bfloat16).view(m, n)
    _check(linear_forward(values, eye, activation=act), values, eye, torch.bfloat16, n, act=act)
    x = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    bias = torch.zeros(n, device="cuda")
    bias[1], bias[2], bias[5] = float("inf"), float("nan"), -40.0
    y = linear_forward(x, eye, bias, activation=act)
    assert (y[:, 1] == float("inf")).all() and y[:, 2].isnan().all()
    assert (y[:, 5].float().abs() < 1e-15).all() and (y[:, [0, 3, 4, 6]] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(5, 1024, 40), (100, 520, 131), (4400, 64, 264), (4400, 320, 257)])
def test_scales_whose_product_is_out_of_range(m, k, n):
    """A row scale and a column scale are finite each, but their product may be subnormal or infinite in fp32 where the result
    is neither: rows of the quantiser's smallest scale, and zeros under two large ones."""
    from mindiesd import linear_forward
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w = ((200 + 248 * torch.rand(rows, k, generator=g, device="cuda")).to(torch.float8_e4m3fn) for rows in (m, n))
    xs = (1 + torch.rand(m, 1, generator=g, device="cuda")) * 2.0 ** -126
    ws = (1 + torch.rand(n, generator=g, device="cuda")) * 2.0 ** -18
    kw = dict(x_scale=xs, weight_scale=ws)
    got = linear_forward(x, w, **kw)
    _check(got, x, w, torch.bfloat16, k, **kw)
    x[3], xs[3], ws[7] = 0, 2.0 ** 100, 2.0 ** 100
    got = linear_forward(x, w, **kw)
    assert (got[3] == 0).all()
    keep = [i for i in range(m) if i != 3]
    _check(got[keep], x[keep], w, torch.bfloat16, k, x_scale=xs[keep], weight_scale=ws)
