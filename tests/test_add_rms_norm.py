"""Residual addition + RMS norm, its e4m3 form and the per-token quantiser: refusals on the host, values on
a GPU against the 64-bit formula.

Tolerances: the last rounding is off by at most half a step of the output's type relative to the value
(half a subnormal step below its normal range).  The fp32 arithmetic before it: a thread adds at most 48
squares, then at most 10 + 32 partial sums (rows beyond 49152 channels: one addition per 1024 channels
more), all positive, so the sum is off by less than 128 roundings of 2^-24, its root by half of that;
with the root's own 2 ulp, the addition, three products and a division: less than 2^-17 in all."""
import ctypes

import pytest
import torch

from oracle import block_linear as ob

F32_SLACK = 2.0 ** -17


def _close(got, want, dtype):
    want = want.double()
    tol = want.abs() * (ob.half_step(dtype) + F32_SLACK) + ob.smallest_half_step(dtype)
    worst = ((got.double() - want).abs() - tol).max().item()
    assert worst <= 0, worst


def _close_quant(q, scale, y):
    want = ob.token_scale(y)
    assert ((scale.double() - want).abs() <= want * F32_SLACK).all()
    stored = q.double()
    ideal = y / scale.double()
    # e4m3: half a step of 2^-4 relative, 2^-10 below its normal range; the quotient itself is off by F32_SLACK
    tol = ideal.abs() * (2.0 ** -4 + F32_SLACK) + 2.0 ** -10
    assert ((stored - ideal).abs() <= tol).all()
    assert stored.abs().max() <= 448


def _randn(seed, *shape, dtype=torch.float32, scale=1.0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=device) * scale).to(dtype)


# ---- host ------------------------------------------------------------------------------------------

def test_struct_layout_and_codes_without_a_gpu(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path
    from mindiesd import _cabi
    lib = _cabi.lib()
    a = _cabi.NormArgs()
    fn = lib.mindiesd_add_rms_norm
    assert fn(None, None) == -1 and fn(ctypes.byref(a), None) == -1
    a.x = a.out = 4096
    assert fn(ctypes.byref(a), None) == -2  # no rows
    a.rows, a.dim, a.dtype, a.out_dtype, a.eps = 4, 64, 7, 0, 1e-6
    assert fn(ctypes.byref(a), None) == -3
    a.dtype = _cabi.BF16
    a.out_dtype = _cabi.FP16
    assert fn(ctypes.byref(a), None) == -3  # the output has the type of x, or is e4m3
    a.out_dtype = _cabi.E4M3
    assert fn(ctypes.byref(a), None) == -1  # e4m3 without scales
    a.out_dtype, a.eps = _cabi.BF16, 0.0
    assert fn(ctypes.byref(a), None) == -5
    a.eps = 1e-6
    a.residual = 4096
    assert fn(ctypes.byref(a), None) == -1  # a residual without a place for the sum
    a.residual_out, a.residual_dtype = 4096, _cabi.FP16
    assert fn(ctypes.byref(a), None) == -3
    a.residual_dtype, a.residual_stride = _cabi.BF16, -64
    assert fn(ctypes.byref(a), None) == -4
    a.residual_stride, a.x = 64, 4097
    assert fn(ctypes.byref(a), None) == -4
    a.x, a.quant_only = 4096, 1
    assert fn(ctypes.byref(a), None) == -5  # the quantiser alone takes neither weight nor residual
    cc = shutil.which("gcc")
    if cc:
        src = tmp_path / "s.c"
        src.write_text('#include <stdio.h>\n#include "mindiesd_b200.h"\nint main(void){printf("%zu",sizeof(mindiesd_norm_args));return 0;}\n')
        inc = Path(__file__).resolve().parent.parent / "include"
        subprocess.run([cc, "-I", str(inc), str(src), "-o", str(tmp_path / "s")], check=True)
        assert int(subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout) == \
            ctypes.sizeof(_cabi.NormArgs)


@pytest.mark.parametrize("written,read", [("out", "x"), ("out", "residual"), ("residual_out", "x"), ("residual_out", "residual")])
def test_outputs_over_inputs_are_refused(written, read):
    """Addresses that overlap by one element; refused before anything reads them, so no device is needed."""
    from mindiesd import _cabi
    for delta in (0, 2 * (3 * 80 + 64) - 2, -(2 * 4 * 64 - 2)):  # the same address, the input's last element, its first
        a = _cabi.NormArgs()
        a.rows, a.dim, a.eps = 4, 64, 1e-6
        a.dtype = a.out_dtype = a.residual_dtype = _cabi.BF16
        a.x, a.residual, a.out, a.residual_out = 1 << 20, 2 << 20, 3 << 20, 4 << 20
        a.x_stride = a.residual_stride = 80
        setattr(a, written, getattr(a, read) + delta)
        assert _cabi.lib().mindiesd_add_rms_norm(ctypes.byref(a), None) == -5


def _refused(device):
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=device)
    return x, [
        dict(x=[1.0]), dict(x=x.double()), dict(x=torch.zeros(4, 0, dtype=torch.bfloat16, device=device)),
        dict(x=torch.zeros((), device=device)), dict(x=torch.zeros(4, 64)),  # not on a CUDA device
        dict(x=x, weight=torch.zeros(63, device=device)), dict(x=x, weight=torch.zeros(64, dtype=torch.float16, device=device)),
        dict(x=x, weight=torch.zeros(64)), dict(x=x, weight=3.0), dict(x=x, weight=torch.zeros(1, 64, device=device)),
        dict(x=x, residual=x[:3]), dict(x=x, residual=x.half()), dict(x=x, residual=torch.zeros(4, 64)), dict(x=x, residual=0),
        dict(x=x, eps=0.0), dict(x=x, eps=-1e-6), dict(x=x, eps=1e-50), dict(x=x, eps=float("nan")), dict(x=x, eps="1"),
        dict(x=x, weight=torch.zeros(64, device=device, requires_grad=True)), dict(x=x.clone().requires_grad_()),
        dict(x=x, residual=x.clone().requires_grad_()),
    ]


def _check_refusals(device):
    from mindiesd import ParametersInvalid, add_rms_norm, add_rms_norm_quant
    from mindiesd.layers.quant import token_quant_preprocess
    x, bad = _refused(device)
    for i, kw in enumerate(bad):
        for fn in (add_rms_norm, add_rms_norm_quant):
            with pytest.raises(ParametersInvalid):
                fn(**kw)
                pytest.fail(f"call {i} was taken")
    for t in ([1.0], torch.zeros(4, 64), x.double(), torch.zeros((), device=device), x.float().requires_grad_()):
        with pytest.raises(ParametersInvalid):
            token_quant_preprocess(t)
    with torch.no_grad():
        assert add_rms_norm(x, torch.nn.Parameter(torch.zeros(64, device=device))).shape == x.shape


def test_refusals():
    _check_refusals("meta")


@pytest.mark.gpu
def test_refusals_on_the_device():
    _check_refusals("cuda")


def test_fake_shapes():
    from mindiesd import add_rms_norm, add_rms_norm_quant
    from mindiesd.layers.quant import token_quant_preprocess
    x = torch.zeros(2, 5, 64, dtype=torch.float16, device="meta")
    r = torch.zeros(2, 5, 64, device="meta")
    y, total = add_rms_norm(x, None, r)
    assert y.dtype == torch.float16 and y.shape == x.shape and total.dtype == torch.float32 and total.shape == r.shape
    q, s = add_rms_norm_quant(x)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and s.shape == (2, 5, 1) and s.dtype == torch.float32
    q, s = token_quant_preprocess(x)
    assert q.shape == x.shape and s.shape == (2, 5, 1)


# ---- GPU -------------------------------------------------------------------------------------------

DIMS = [1, 3, 8, 31, 64, 100, 128, 1001, 1004, 1536, 5120, 6143, 8192, 20480]


@pytest.mark.gpu
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_values(dim, dtype):
    from mindiesd import add_rms_norm, add_rms_norm_quant
    for rows, weight, residual in [(1, None, None), (7, dtype, dtype), (33, torch.float32, torch.float32), (260, dtype, None)]:
        x = _randn(dim + rows, rows, dim, dtype=dtype)
        w = None if weight is None else _randn(1, dim, dtype=weight)
        r = None if residual is None else _randn(2, rows, dim, dtype=residual, scale=3.0)
        y64, v64 = ob.rms_norm(x, w, r)
        got = add_rms_norm(x, w, r)
        quant = add_rms_norm_quant(x, w, r)
        if r is not None:
            got, total = got
            assert total.dtype == residual and torch.equal(quant[2], total)
            _close(total, v64, residual)
        assert got.dtype == dtype and got.shape == x.shape
        _close(got, y64, dtype)
        _close_quant(quant[0], quant[1], y64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [1, 65, 72, 1536, 5120])
def test_token_quant(dim, dtype):
    from mindiesd.layers.quant import token_quant_preprocess
    x = _randn(dim, 2, 19, dim, dtype=dtype)
    x[0, 3] = 0
    x[1, 4] *= 1e-4
    q, s = token_quant_preprocess(x)
    assert s.shape == (2, 19, 1) and s[0, 3].item() == 1.0 and torch.count_nonzero(q[0, 3].float()) == 0
    _close_quant(q, s, x.double())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [8, 64, 128, 200, 1000, 1536, 5120, 10240, 16384, 24576])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_many_rows(dim, dtype):
    """Enough rows that the blocks of the launch walk several each, ragged at the end; every row is looked at."""
    from mindiesd import add_rms_norm, add_rms_norm_quant
    rows = {8: 200001, 64: 70003, 128: 40005, 200: 30001}.get(dim, 2503)
    for weight, residual in [(None, None), (dtype, dtype), (torch.float32, torch.float32)]:
        x = _randn(dim, rows, dim, dtype=dtype)
        w = None if weight is None else _randn(1, dim, dtype=weight)
        r = None if residual is None else _randn(2, rows, dim, dtype=residual, scale=3.0)
        y64, v64 = ob.rms_norm(x, w, r)
        got, quant = add_rms_norm(x, w, r), add_rms_norm_quant(x, w, r)
        if r is not None:
            got, total = got
            assert torch.equal(quant[2], total)
            _close(total, v64, residual)
        _close(got, y64, dtype)
        _close_quant(quant[0], quant[1], y64)


@pytest.mark.gpu
def test_many_strided_rows():
    from mindiesd import add_rms_norm
    packed = _randn(3, 6000, 3 * 1536, dtype=torch.bfloat16)
    weight = _randn(4, 1536, dtype=torch.bfloat16)
    for part in (packed[:, :1536], packed.narrow(1, 1536, 1536), packed[:1, :1536].expand(6000, 1536)):
        y, total = add_rms_norm(part, weight, packed[:, -1536:])
        y64, v64 = ob.rms_norm(part, weight, packed[:, -1536:])
        _close(y, y64, torch.bfloat16)
        _close(total, v64, torch.bfloat16)


@pytest.mark.gpu
def test_long_rows():
    from mindiesd import add_rms_norm, add_rms_norm_quant
    for dim, dtype in ((70001, torch.bfloat16), (70000, torch.float32), (6145, torch.float16)):
        x, r = _randn(3, 5, dim, dtype=dtype), _randn(4, 5, dim, dtype=dtype)
        w = _randn(5, dim)
        y64, v64 = ob.rms_norm(x, w, r)
        y, total = add_rms_norm(x, w, r)
        _close(y, y64, dtype)
        _close(total, v64, dtype)
        q, s, _ = add_rms_norm_quant(x, w, r)
        _close_quant(q, s, y64)


@pytest.mark.gpu
def test_strided_rows_and_empty_inputs():
    from mindiesd import add_rms_norm, add_rms_norm_quant
    from mindiesd.layers.quant import token_quant_preprocess
    packed = _randn(7, 3, 50, 3 * 384, dtype=torch.bfloat16)
    for part in (packed[..., :384], packed[..., 384:768], packed[..., 5:389], packed[:, ::2, :384], packed.transpose(0, 1)[..., 384:],
                 packed[..., ::3], packed[:1].expand(3, 50, 1152)):
        r = _randn(8, *part.shape, dtype=torch.bfloat16)
        y, total = add_rms_norm(part, None, r)
        y64, v64 = ob.rms_norm(part, None, r)
        _close(y, y64, torch.bfloat16)
        _close(total, v64, torch.bfloat16)
        y2, total2 = add_rms_norm(r, None, part)
        assert torch.equal(y2, y) and torch.equal(total2, total)  # a sum does not depend on the order of two terms
    one = _randn(9, 384, dtype=torch.float16)
    _close(add_rms_norm(one), ob.rms_norm(one)[0], torch.float16)
    empty = torch.empty(0, 384, dtype=torch.bfloat16, device="cuda")
    assert add_rms_norm(empty).shape == (0, 384)
    q, s, t = add_rms_norm_quant(empty, None, empty)
    assert q.shape == (0, 384) and s.shape == (0, 1) and t.shape == (0, 384)
    assert token_quant_preprocess(empty)[1].shape == (0, 1)


@pytest.mark.gpu
def test_unusual_values():
    """A row of zeros, one of the type's largest and smallest values, and rows with a NaN or an infinity stay apart."""
    from mindiesd import add_rms_norm, add_rms_norm_quant
    from mindiesd.layers.quant import token_quant_preprocess
    for dim in (128, 129):
        x = _randn(11, 8, dim, dtype=torch.bfloat16)
        x[1] = 0
        x[2, 5] = float("nan")
        x[4, 7] = float("inf")
        x[6] *= 1e-30
        keep = [0, 1, 3, 5, 6, 7]
        y = add_rms_norm(x)
        q, s = add_rms_norm_quant(x)
        y64 = ob.rms_norm(x)[0]
        _close(y[keep], y64[keep], torch.bfloat16)
        _close_quant(q[keep], s[keep], y64[keep])
        assert s[1].item() == 1.0 and torch.isnan(s[2]) and torch.isnan(s[4])
        assert torch.isnan(y[2].float()).all() and torch.isnan(y[4, 7]) and torch.isnan(q[2].float()).all()
        tiny = torch.full((2, dim), 1e-40, device="cuda")
        tiny[1] = torch.finfo(torch.float32).max
        q, s = token_quant_preprocess(tiny)
        _close_quant(q, s, tiny.double())
        assert s[0].item() == 2.0 ** -126 and (q[1].float() == 448).all()
        q, s = token_quant_preprocess(x)
        assert torch.isnan(s[2]) and torch.isinf(s[4]) and torch.isfinite(s[keep]).all()


@pytest.mark.gpu
def test_many_short_rows_and_rows_beyond_32_bit_offsets():
    from mindiesd import add_rms_norm, add_rms_norm_quant
    x = _randn(12, 70001, 128, dtype=torch.float16)
    w = _randn(13, 128, dtype=torch.float16)
    _close(add_rms_norm(x, w), ob.rms_norm(x, w)[0], torch.float16)
    x = torch.zeros(270000, 8192, dtype=torch.bfloat16, device="cuda")  # 2.2e9 elements
    x[-3:] = _randn(14, 3, 8192, dtype=torch.bfloat16)
    q, s = add_rms_norm_quant(x)
    _close_quant(q[-3:], s[-3:], ob.rms_norm(x[-3:])[0])
    assert s[-4].item() == 1.0


@pytest.mark.gpu
def test_streams_graphs_and_repeatability():
    from mindiesd import add_rms_norm_quant
    x, r = _randn(15, 300, 1536, dtype=torch.bfloat16), _randn(16, 300, 1536)
    first = add_rms_norm_quant(x, None, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = add_rms_norm_quant(x, None, r)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a.float(), b.float())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = add_rms_norm_quant(x, None, r)
    x.copy_(_randn(17, 300, 1536, dtype=torch.bfloat16))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, add_rms_norm_quant(x, None, r)):
        assert torch.equal(a.float(), b.float())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [5, 9, 15, 18, 98, 100, 179, 514, 1003, 1004, 4097, 6143, 10999, 11002])
def test_packed_rows_of_uneven_width(dim, dtype):
    """Rows that start anywhere in a 16-byte run and share runs with their neighbours: the values, the last row at the very
    end of its memory, and neighbours of a NaN as if it were not there.  Rows apart from one another agree."""
    from mindiesd import add_rms_norm, add_rms_norm_quant
    for rows, weight, residual in [(1, dtype, dtype), (2, None, torch.float32), (45, torch.float32, None), (4003, dtype, dtype),
                                   (3001, None, torch.float32)]:
        x = _randn(dim + rows, rows, dim, dtype=dtype)
        w = None if weight is None else _randn(1, dim, dtype=weight)
        r = None if residual is None else _randn(2, rows, dim, dtype=residual, scale=3.0)
        keep = torch.ones(rows, dtype=torch.bool, device="cuda")
        if rows > 2:
            x[rows // 2, 0] = x[rows // 3, dim - 1] = float("nan")
            keep[rows // 2] = keep[rows // 3] = False
        y64, v64 = ob.rms_norm(x, w, r)
        got, quant = add_rms_norm(x, w, r), add_rms_norm_quant(x, w, r)
        if r is not None:
            got, total = got
            assert torch.equal(quant[2].nan_to_num(), total.nan_to_num()) and torch.equal(total.isnan(), v64.isnan())
            _close(total.nan_to_num(), v64.nan_to_num(), residual)
        assert got[~keep].isnan().all() and quant[1][~keep].isnan().all()
        _close(got[keep], y64[keep], dtype)
        _close_quant(quant[0][keep], quant[1][keep], y64[keep])
        # the same rows lying apart take another kernel, whose sums run in another order
        wide = torch.zeros(rows, dim + 3, dtype=dtype, device="cuda")[:, :dim].copy_(x)
        apart = add_rms_norm(wide, w, r)
        _close((apart if r is None else apart[0])[keep], y64[keep], dtype)


@pytest.mark.gpu
def test_packed_rows_of_uneven_width_write_nothing_else():
    """Through the C ABI: what lies before and behind the outputs stays, at every position of the last element in a run."""
    from mindiesd import _cabi
    for dim in range(33, 42):
        for rows in (1, 2, 7):
            x, r = _randn(1, rows, dim, dtype=torch.bfloat16), _randn(2, rows, dim, dtype=torch.float32)
            w = _randn(3, dim, dtype=torch.bfloat16)
            for e4m3 in (False, True):
                buf = torch.full((rows * dim + 64,), 7.0, device="cuda").to(torch.float8_e4m3fn if e4m3 else torch.bfloat16)
                total, scales = torch.full((rows * dim + 64,), 7.0, device="cuda"), torch.full((rows + 2,), 7.0, device="cuda")
                a = _cabi.NormArgs()
                a.x, a.residual, a.weight = x.data_ptr(), r.data_ptr(), w.data_ptr()
                a.out, a.residual_out = buf[32:].data_ptr(), total[32:].data_ptr()
                a.scales = scales[1:].data_ptr() if e4m3 else None
                a.rows, a.dim, a.x_stride, a.residual_stride, a.eps = rows, dim, dim, dim, 1e-6
                a.dtype = a.weight_dtype = _cabi.BF16
                a.residual_dtype, a.out_dtype = _cabi.FP32, _cabi.E4M3 if e4m3 else _cabi.BF16
                _cabi.check(_cabi.lib().mindiesd_add_rms_norm(ctypes.byref(a), _cabi.current_stream_ptr(x.device)), "mindiesd_add_rms_norm")
                y64, v64 = ob.rms_norm(x, w, r)
                n = rows * dim
                _close(total[32:32 + n].view(rows, dim), v64, torch.float32)
                if e4m3:
                    _close_quant(buf[32:32 + n].view(rows, dim), scales[1:-1, None], y64)
                    assert scales[0] == 7 and scales[-1] == 7
                else:
                    _close(buf[32:32 + n].view(rows, dim), y64, torch.bfloat16)
                for t in (buf.float(), total):
                    assert (t[:32] == 7).all() and (t[32 + n:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,dim,apart", [(9, 128, 0), (9, 5120, 0), (70003, 128, 0), (2503, 5120, 0), (600, 1004, 4), (600, 1001, 3),
                                            (600, 1001, 0), (9, 6143, 0), (5, 70001, 0)])
def test_quantised_rows_of_tiny_values(rows, dim, apart, dtype):
    """Rows whose 448 / max|v w| is infinite in fp32 although 1 / sqrt(mean + eps) and 1 / scale are finite: their values keep
    their size, their zeros stay zero, and the rows beside them do not change.  Few rows and many, packed, apart, uneven,
    long.  (What an fp16 row holds is at least 6e-8, so there the weight makes the products tiny, by a power of two.)"""
    from mindiesd import add_rms_norm_quant
    x = torch.zeros(rows, dim + apart, dtype=dtype, device="cuda")[:, :dim].copy_(_randn(dim, rows, dim, dtype=dtype))
    plain = add_rms_norm_quant(x)
    tops = [1.5e-36, 1.2e-36, 1e-37, 3e-38, 1e-39]
    tiny = list(range(min(rows, 5))) + ([rows // 2, rows - 1] if rows > 10 else [])
    factor = 1.0 if dtype != torch.float16 else 2.0 ** -110
    for i, row in enumerate(tiny):
        x[row] *= tops[i % 5] / factor / x[row].abs().max().float()
        x[row, ::3] = 0
        x[row, 1] = tops[i % 5] / factor
    weight = None if dtype != torch.float16 else torch.full((dim,), factor, device="cuda")
    q, s = add_rms_norm_quant(x, weight)
    y64, _ = ob.rms_norm(x[tiny], weight)
    assert torch.isfinite(s).all() and not q.float().isnan().any()
    assert torch.count_nonzero(q[tiny][:, ::3].float()) == 0
    _close_quant(q[tiny], s[tiny], y64)
    if weight is None:
        keep = torch.ones(rows, dtype=torch.bool, device="cuda")
        keep[tiny] = False
        assert torch.equal(q[keep].float(), plain[0][keep].float()) and torch.equal(s[keep], plain[1][keep])
    else:
        _close_quant(q, s, ob.rms_norm(x, weight)[0])


@pytest.mark.parametrize("written,other,bytes_of_other", [("out", "weight", 128), ("residual_out", "weight", 128), ("scales", "x", 608), ("scales", "residual", 608),
                                                          ("scales", "weight", 128), ("scales", "out", 256), ("scales", "residual_out", 512), ("out", "residual_out", 512)])
def test_outputs_over_weights_and_each_other_are_refused(written, other, bytes_of_other):
    """Addresses that overlap by one element; refused before anything reads them, so no device is needed."""
    from mindiesd import _cabi

    def code(**where):
        a = _cabi.NormArgs()
        a.rows, a.dim, a.eps = 4, 64, 1e-6
        a.dtype = a.residual_dtype = a.weight_dtype = _cabi.BF16
        a.out_dtype = _cabi.E4M3
        a.x, a.residual, a.weight, a.out, a.residual_out = 1 << 20, 2 << 20, 5 << 20, 3 << 20, 4 << 20
        a.scales = 6 << 20
        a.x_stride = a.residual_stride = 80
        for name, at in where.items():
            setattr(a, name, at)
        return _cabi.lib().mindiesd_add_rms_norm(ctypes.byref(a), None)
    place = {"x": 1 << 20, "residual": 2 << 20, "weight": 5 << 20, "out": 3 << 20, "residual_out": 4 << 20}[other]
    size = {"out": 256, "residual_out": 512, "scales": 16}[written]
    for delta in (0, bytes_of_other - 4, -(size - 4)):
        assert code(**{written: place + delta}) == -5


@pytest.mark.gpu
def test_operands_side_by_side_are_taken():
    """Inputs and outputs that follow one another in one buffer without a gap."""
    from mindiesd import _cabi
    rows, dim = 4, 64
    x, w = _randn(31, rows, dim, dtype=torch.bfloat16), _randn(32, dim, dtype=torch.bfloat16)
    sizes = {"x": 512, "out": 256, "residual": 512, "residual_out": 512, "weight": 128, "scales": 16}
    for order in (list(sizes), list(sizes)[::-1]):
        buf, at = torch.zeros(sum(sizes.values()), dtype=torch.uint8, device="cuda"), {}
        for name in order:
            at[name] = buf[sum(t.numel() for t in at.values()):][:sizes[name]]
        for name, t in (("x", x), ("residual", x), ("weight", w)):
            at[name].copy_(t.view(torch.uint8).flatten())
        a = _cabi.NormArgs()
        for name, t in at.items():
            setattr(a, name, t.data_ptr())
        a.rows, a.dim, a.x_stride, a.residual_stride, a.eps = rows, dim, dim, dim, 1e-6
        a.dtype = a.residual_dtype = a.weight_dtype = _cabi.BF16
        a.out_dtype = _cabi.E4M3
        _cabi.check(_cabi.lib().mindiesd_add_rms_norm(ctypes.byref(a), _cabi.current_stream_ptr(x.device)), "mindiesd_add_rms_norm")
        y64, v64 = ob.rms_norm(x, w, x)
        _close(at["residual_out"].view(torch.bfloat16).view(rows, dim), v64, torch.bfloat16)
        _close_quant(at["out"].view(torch.float8_e4m3fn).view(rows, dim), at["scales"].view(torch.float32)[:, None], y64)
        assert torch.equal(at["x"], x.view(torch.uint8).flatten()) and torch.equal(at["weight"], w.view(torch.uint8).flatten())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim,apart", [(4, 1, 0), (4, 128, 0), (9, 5120, 0), (2503, 5120, 0), (600, 1001, 3), (600, 1001, 0), (4, 70001, 0)])
def test_rows_around_the_largest_sum_of_squares(rows, dim, apart):
    """A root mean square of 0.9 and of 1.1 times sqrt(largest fp32 / dim): the values, and zeros with a scale of 1."""
    from mindiesd import add_rms_norm, add_rms_norm_quant
    bound = (torch.finfo(torch.float32).max / dim) ** 0.5
    x = torch.empty(rows, dim + apart, device="cuda")[:, :dim]
    sign = torch.randint(0, 2, (rows, dim), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * 2.0 - 1
    x.copy_(sign * 0.9 * bound)
    x[rows // 2] *= 1.1 / 0.9
    keep = torch.arange(rows, device="cuda") != rows // 2
    y64 = ob.rms_norm(x)[0]
    y, (q, s) = add_rms_norm(x), add_rms_norm_quant(x)
    _close(y[keep], y64[keep], torch.float32)
    _close_quant(q[keep], s[keep], y64[keep])
    assert (y[~keep] == 0).all() and (q[~keep].float() == 0).all() and (s[~keep] == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [8188, 8192, 8196, 10996, 11000, 11004])
def test_packed_rows_that_four_divides(dim, dtype):
    """On both sides of the longest row that runs of four elements keep in registers, and of the longest that shared
    memory keeps the weights of."""
    from mindiesd import add_rms_norm, add_rms_norm_quant
    for rows, weight in ((3, dtype), (1301, torch.float32), (700, None)):
        x = _randn(dim + rows, rows, dim, dtype=dtype)
        w = None if weight is None else _randn(1, dim, dtype=weight)
        y64 = ob.rms_norm(x, w)[0]
        _close(add_rms_norm(x, w), y64, dtype)
        _close_quant(*add_rms_norm_quant(x, w), y64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [591, 592, 593])
def test_wide_rows_around_the_change_of_kernels(rows, dtype):
    """The count of rows from which blocks walk several of them, without a residual, at widths of three to six runs."""
    from mindiesd import add_rms_norm, add_rms_norm_quant
    e = torch.empty(0, dtype=dtype).element_size()
    for runs in (376, 385, 512, 640, 760, 1536, 1544):
        dim = runs * 16 // e
        x, w = _randn(dim, rows, dim, dtype=dtype), _randn(1, dim, dtype=dtype)
        y64 = ob.rms_norm(x, w)[0]
        _close(add_rms_norm(x, w), y64, dtype)
        _close_quant(*add_rms_norm_quant(x, w), y64)
