"""Both kernels of `linear_forward` at every way of cutting a product up, against the 64-bit formula: the sizes of a call
choose between them, and sizes small enough for a test are mostly cut in few ways (pair tiles of 32, 64, 96 and 256 columns).
Here the cut is given: tiles of 256 rows and 32..256 columns by two-SM MMAs ("pair"), or 16..128 rows with k split over one to
eight thread blocks ("swap").  Tolerances are those of test_linear_forward.py."""
import ctypes

import pytest
import torch

import test_linear_forward as tl
from mindiesd import _cabi
from oracle import block_linear as ob

PAIR = [(0, tile, 1, 1) for tile in range(32, 257, 32)]
SWAP = [(1, tile, split, per_sm) for tile in range(16, 129, 16) for split in range(1, 9) for per_sm in (1, 2)
        if per_sm == 1 or tile <= 80]
FEW = [(0, 32, 1, 1), (0, 128, 1, 1), (0, 160, 1, 1), (0, 192, 1, 1), (0, 256, 1, 1), (1, 16, 1, 2), (1, 48, 3, 1), (1, 128, 2, 1)]


def _arguments(x, weight, out, bias=None, act="none", residual=None, gate=None, x_scale=None, weight_scale=None):
    """gate: [G, N], every m / G rows sharing one."""
    a = _cabi.LinearArgs()
    a.x, a.weight, a.out = x.data_ptr(), weight.data_ptr(), out.data_ptr()
    a.x_stride, a.weight_stride, a.out_stride = x.stride(0), weight.stride(0), out.stride(0)
    (a.m, a.k), a.n = x.shape, weight.shape[0]
    a.in_dtype, a.out_dtype = _cabi.dtype_code(x.dtype), _cabi.dtype_code(out.dtype)
    a.activation = _cabi.ACTIVATIONS[act]
    if bias is not None:
        a.bias, a.bias_dtype = bias.data_ptr(), _cabi.dtype_code(bias.dtype)
    if residual is not None:
        a.residual, a.residual_stride = residual.data_ptr(), residual.stride(0)
    if gate is not None:
        a.gate, a.gate_dtype, a.gate_stride = gate.data_ptr(), _cabi.dtype_code(gate.dtype), gate.stride(0)
        a.rows_per_gate = -(-x.shape[0] // gate.shape[0])
    if x_scale is not None:
        a.x_scale, a.weight_scale = x_scale.data_ptr(), weight_scale.data_ptr()
        a.x_scale_single, a.weight_scale_single = x_scale.numel() == 1, weight_scale.numel() == 1
    return a


def _run(cut, x, weight, out, **kw):
    a, c = _arguments(x, weight, out, **kw), _cabi.LinearCut(*cut)
    _cabi.check(_cabi.lib().mindiesd_linear_fwd_as(ctypes.byref(a), ctypes.byref(c), _cabi.current_stream_ptr(x.device)), str(cut))
    return out


def _checked(cut, x, weight, out_dtype, **kw):
    """Runs the product into the middle of a larger buffer; the values, and that nothing around them changed."""
    m, n = x.shape[0], weight.shape[0]
    wide = torch.full((m + 2, n), 7.0, dtype=out_dtype, device="cuda")
    got = _run(cut, x, weight, wide[1:1 + m], **kw)
    gate = kw.pop("gate", None)
    if gate is not None:  # one row for each row of the product
        kw["gate"] = gate.repeat_interleave(-(-m // gate.shape[0]), 0)[:m]
    tl._check(got, x, weight, out_dtype, x.shape[1], **kw)
    assert (wide[0] == 7).all() and (wide[-1] == 7).all()
    return got


# ---- host ------------------------------------------------------------------------------------------

def test_cuts_that_are_refused():
    """Refused before anything is launched; the addresses are never read."""
    a = _cabi.LinearArgs()
    a.x, a.weight, a.out = 1 << 20, 2 << 20, 3 << 20
    a.m, a.n, a.k, a.in_dtype, a.out_dtype = 40, 100, 512, _cabi.BF16, _cabi.BF16
    a.x_stride = a.weight_stride = 512
    a.out_stride = 100
    fn = _cabi.lib().mindiesd_linear_fwd_as
    assert fn(ctypes.byref(a), None, None) == -1 and fn(None, ctypes.byref(_cabi.LinearCut(0, 64, 1, 1)), None) == -1
    for cut in [(0, 0, 1, 1), (0, 16, 1, 1), (0, 48, 1, 1), (0, 160, 1, 1), (0, 288, 1, 1), (0, 64, 2, 1), (0, 64, 1, 2), (0, -32, 1, 1),
                (1, 0, 1, 1), (1, 8, 1, 1), (1, 24, 1, 1), (1, 64, 1, 1), (1, 144, 1, 1), (1, 16, 0, 1), (1, 16, 9, 1), (1, 16, 5, 1),
                (1, 16, 1, 0), (1, 16, 1, 3), (2, 64, 1, 1), (-1, 64, 1, 1)]:
        assert fn(ctypes.byref(a), ctypes.byref(_cabi.LinearCut(*cut)), None) == -5, cut
    a.m = 128
    assert fn(ctypes.byref(a), ctypes.byref(_cabi.LinearCut(1, 128, 1, 2)), None) == -5  # two blocks would have one stage each


def test_struct_layout(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "mindiesd_b200.h"\nint main(void){printf("%zu",sizeof(mindiesd_linear_cut));return 0;}\n')
    inc = Path(__file__).resolve().parent.parent / "include"
    subprocess.run([cc, "-I", str(inc), str(src), "-o", str(tmp_path / "s")], check=True)
    assert int(subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout) == ctypes.sizeof(_cabi.LinearCut)


# ---- GPU -------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("m,n,k", [(300, 520, 208), (257, 271, 64), (1, 256, 2064), (4400, 1064, 144), (700, 1501, 1040)])
def test_every_pair_tile(m, n, k, dtype):
    """One and several tiles along each side, more tiles than blocks, whole and ragged last ones, one k step and many."""
    x, w, kw = tl._operands(m + n, m, k, n, dtype)
    outs = [_checked(cut, x, w, torch.bfloat16, **kw) for cut in PAIR]
    for o in outs[1:]:  # every output element is summed in the same order
        assert torch.equal(o, outs[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("m,n", [(128, 264), (261, 129), (113, 1000)])
def test_every_swap_tile_and_split(m, n, dtype):
    k = 1296 if dtype == torch.bfloat16 else 2320  # 21 and 19 steps
    x, w, kw = tl._operands(m + n, m, k, n, dtype)
    for cut in SWAP:
        _checked(cut, x, w, torch.bfloat16, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("cut", FEW)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_epilogue(cut, dtype, act):
    """Every type of bias, gate and output, with and without a residual, at widths whose rows move 32, 16, 8 and 4 bytes
    at a time; the gate is one for all rows."""
    for m, n in ((300, 256), (258, 264), (400, 268), (290, 271)):
        x, w, kw = tl._operands(m, m, 784, n, dtype)
        for bias_dtype, gate_dtype, out_dtype in [(torch.bfloat16, torch.float32, torch.bfloat16), (torch.float32, torch.float16, torch.float16),
                                                  (None, torch.bfloat16, torch.bfloat16), (torch.float16, None, torch.float16)]:
            full = dict(kw, act=act)
            if bias_dtype is not None:
                full["bias"] = tl._randn(5, n, dtype=bias_dtype, scale=2.0)
            if gate_dtype is not None:
                full["gate"] = tl._randn(6, 1, n, dtype=gate_dtype)
            _checked(cut, x, w, out_dtype, **full)
            _checked(cut, x, w, out_dtype, **dict(full, residual=tl._randn(7, m, n, dtype=out_dtype)))


@pytest.mark.gpu
@pytest.mark.parametrize("cut", FEW)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_gates_that_change_within_a_tile(cut, dtype):
    """Samples of 1, 7, 40, 100 and 256 rows: a warp's 32 rows share a gate, or do not.  Gates of each type, their rows
    on 16 bytes or not."""
    for m, n, per in ((300, 264, 1), (301, 256, 7), (520, 271, 40), (300, 264, 100), (600, 256, 256)):
        x, w, kw = tl._operands(m, m, 784, n, dtype)
        residual = tl._randn(8, m, n, dtype=torch.bfloat16)
        for gate_dtype in (torch.float32, torch.float16, torch.bfloat16):
            for pad in (0, 3, 8):
                gate = tl._randn(9, -(-m // per), n + pad, dtype=gate_dtype)[:, :n]
                wide = torch.full((m, n), 7.0, dtype=torch.bfloat16, device="cuda")
                a = _arguments(x, w, wide, residual=residual, gate=gate, **kw)
                a.rows_per_gate = per
                _cabi.check(_cabi.lib().mindiesd_linear_fwd_as(ctypes.byref(a), ctypes.byref(_cabi.LinearCut(*cut)),
                                                               _cabi.current_stream_ptr(x.device)), str(cut))
                tl._check(wide, x, w, torch.bfloat16, 784, residual=residual, gate=gate.repeat_interleave(per, 0)[:m], **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("cut", FEW)
@pytest.mark.parametrize("n", [256, 264, 268, 258, 257])
def test_strided_rows_of_every_piece(cut, n):
    """Operands, residual and output that lie in wider rows, on addresses of every kind; what surrounds the output stays."""
    m, k = 290, 392
    for x_pad, out_start, out_pad, res_start, res_pad in ((0, 0, 0, 0, 0), (8, 16, 32, 0, 16), (16, 8, 8, 4, 4), (64, 4, 4, 2, 2), (8, 2, 2, 1, 1), (24, 1, 1, 0, 3)):
        x, w = tl._randn(1, m, k + x_pad, dtype=torch.float16)[:, :k], tl._randn(2, n, k + x_pad, dtype=torch.float16, scale=0.1)[:, :k]
        wide = torch.full((m + 2, n + out_pad + out_start), 7.0, dtype=torch.float16, device="cuda")
        out = wide[1:1 + m, out_start:out_start + n]
        residual = tl._randn(3, m, n + res_pad + res_start, dtype=torch.float16)[:, res_start:res_start + n]
        _run(cut, x, w, out, residual=residual)
        tl._check(out, x, w, torch.float16, k, residual=residual)
        keep = torch.ones_like(wide, dtype=torch.bool)
        keep[1:1 + m, out_start:out_start + n] = False
        assert (wide[keep] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("cut", FEW)
@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
def test_activations_over_their_range(cut, act):
    m, n = 400, 384
    eye = torch.eye(n, dtype=torch.bfloat16, device="cuda")
    values = torch.cat([torch.linspace(-14, 14, m * n - 40, device="cuda"), torch.logspace(-30, 3, 20, device="cuda"),
                        -torch.logspace(-30, 3, 20, device="cuda")]).to(torch.bfloat16).view(m, n)
    _checked(cut, values, eye, torch.bfloat16, act=act)
    bias = torch.zeros(n, device="cuda")
    bias[1], bias[2], bias[5] = float("inf"), float("nan"), -40.0
    out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    y = _run(cut, torch.zeros(m, n, dtype=torch.bfloat16, device="cuda"), eye, out, bias=bias, act=act)
    assert (y[:, 1] == float("inf")).all() and y[:, 2].isnan().all()
    assert (y[:, 5].float().abs() < 1e-15).all() and (y[:, [0, 3, 4, 6]] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("cut", FEW)
def test_rows_and_columns_stay_apart(cut):
    """A NaN stays in its row or column, and so do scales of one and of each row."""
    m, n, k = 300, 270, 784
    x, w, _ = tl._operands(40, m, k, n, torch.bfloat16)
    clean = _run(cut, x, w, torch.empty(m, n, dtype=torch.bfloat16, device="cuda"))
    x2, w2 = x.clone(), w.clone()
    x2[3, 17] = float("nan")
    x2[299, 783] = float("inf")
    w2[11, 5] = float("inf")
    got = _run(cut, x2, w2, torch.empty_like(clean))
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[3], bad[299], bad[:, 11] = True, True, True
    assert not torch.isfinite(got[bad].float()).any() and torch.equal(got[~bad], clean[~bad])
    x8, w8, kw = tl._operands(41, m, k, n, torch.float8_e4m3fn)
    one = torch.tensor([0.37], device="cuda")
    for scales in (kw, dict(x_scale=one, weight_scale=kw["weight_scale"]), dict(x_scale=kw["x_scale"], weight_scale=one),
                   dict(x_scale=one, weight_scale=one)):
        _checked(cut, x8, w8, torch.bfloat16, **scales)


@pytest.mark.gpu
@pytest.mark.parametrize("cut", FEW)
def test_at_once_captured_and_replayed(cut):
    m, n, k = 700, 384, 1024
    x, w, _ = tl._operands(50, m, k, n, torch.bfloat16)
    residual = tl._randn(51, m, n, dtype=torch.bfloat16)

    def call():
        return _run(cut, x, w, torch.full((m, n), 7.0, dtype=torch.bfloat16, device="cuda"), residual=residual, act="gelu")
    first = call()
    tl._check(first, x, w, torch.bfloat16, k, residual=residual, act="gelu")
    torch.cuda.synchronize()
    outs = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            outs += [call() for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    x.copy_(tl._randn(52, m, k, dtype=torch.bfloat16))
    graph.replay()
    assert torch.equal(captured, call())


@pytest.mark.gpu
@pytest.mark.parametrize("cut", [(0, 96, 1, 1), (1, 32, 2, 1)])
@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_activations_relative_accuracy(cut, act, dtype):
    """The other operand is the unit matrix, so a sum is one product and exact, and the tolerance is the activation's alone: its
    2^-15 and the last rounding, both relative, and |v| 2^-126, where the reciprocal and the exponential flush to zero."""
    n = 256
    eye = torch.eye(n, dtype=dtype, device="cuda")
    edge = {"relu": 1.0, "silu": 87.34, "gelu": 13.22, "gelu_tanh": 10.0}[act]
    v = torch.cat([torch.linspace(-1.2 * edge, 0, 40 * n, device="cuda"), torch.linspace(-1.05 * edge, -0.95 * edge, 20 * n, device="cuda"),
                   torch.linspace(0, 100, 20 * n, device="cuda"), -torch.logspace(-4, 2, 20 * n, device="cuda")]).to(dtype).view(-1, n)
    out = _run(cut, v, eye, torch.empty(v.shape, dtype=dtype, device="cuda"), act=act)
    want = ob.activation(v.double(), act)
    tol = want.abs() * (ob.half_step(dtype) + tl.ACT_SLACK) + ob.smallest_half_step(dtype) + v.double().abs() * 2.0 ** -126
    worst = ((out.double() - want).abs() - tol).max().item()
    assert worst <= 0, worst
