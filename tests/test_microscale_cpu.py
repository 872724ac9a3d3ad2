"""Block-scaled formats without a GPU: the oracle's own definitions, host checks and refusals."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from krea2_svdquant_b200 import _lib, microscale as M, ops
from oracle import mx_oracle as O


@pytest.fixture(scope="module", autouse=True)
def built():
    from krea2_svdquant_b200 import build
    build.build()


def test_oracle_tables():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(O.E4M3, t)
    e = torch.arange(256, dtype=torch.uint8).view(torch.float8_e8m0fnu).double().numpy()
    np.testing.assert_array_equal(O.E8M0, e)


@pytest.mark.parametrize("fmt", sorted(O.BLOCK))
def test_oracle_codes_round_trip(fmt):
    """Values that codes stand for quantise to themselves."""
    rng = np.random.default_rng(0)
    table = O.E4M3[:127] if fmt == "mxfp8" else O.E2M1[:8]
    q = rng.choice(np.concatenate([table, -table]), (20, 256))
    q[:, ::16] = table[-1]
    s = 2.0 ** rng.integers(-5, 5, (20, 256 // O.BLOCK[fmt]))
    x = (q.reshape(20, -1, O.BLOCK[fmt]) * s[..., None]).reshape(20, 256)
    codes, byte = O.quantize(x, fmt)
    np.testing.assert_array_equal(O.values(codes, byte, fmt), x)


def test_oracle_ties_go_to_even():
    x = np.array([[6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, 0]])
    codes, byte = O.quantize(x, "nvfp4")
    assert byte[0, 0] == 0x38  # 1.0
    want = [6, 0, 1, 1, 2, 2, 4, 4, 0, -1, -1, -2, -2, -4, -4, 0]
    np.testing.assert_array_equal(O.values(codes, byte, "nvfp4")[0, :16], want)


@pytest.mark.parametrize("fmt", sorted(O.BLOCK))
@pytest.mark.parametrize("rows,k", [(1, 1), (128, 128), (129, 130), (4352, 6144)])
def test_scale_layout_sizes(fmt, rows, k):
    n = ops.mx_scales_numel(rows, k, fmt)
    assert n == _lib.lib().svdq_mx_scale_bytes(rows, k, ops.MX_FORMATS[fmt])
    at = O.scale_index(rows, O.k_pad(k) // O.BLOCK[fmt])
    assert at.max() < n and np.unique(at).size == at.size


def test_scale_bytes_of_nothing():
    L = _lib.lib()
    assert L.svdq_mx_scale_bytes(0, 64, 0) == 0 and L.svdq_mx_scale_bytes(4, 0, 0) == 0
    assert L.svdq_mx_scale_bytes(4, 64, 3) == 0 and L.svdq_mx_scale_bytes(-1, 64, 0) == 0


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        M.quantize(x, "nvfp4")
    with pytest.raises(ValueError, match="CUDA"):
        M.tensor_scale(x)
    with pytest.raises(ValueError, match="CUDA"):
        M.rms_norm(x)
    t = M.MicroTensor(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8), "nvfp4", (4, 64))
    with pytest.raises(ValueError, match="CUDA"):
        M.dequantize(t)
    with pytest.raises(ValueError, match="CUDA"):
        M.matmul(t, t)


def test_operand_checks():
    """The checks of an operand's tensors, on the host."""
    c, s = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8)
    g = torch.ones(1)
    ops._mx_check("t", c, s, "nvfp4", 100, g)
    for bad in (dict(fmt="int4"), dict(k=200), dict(fmt="mxfp8"), dict(fmt="mxfp4"), dict(scales=s[:-1]),
                dict(codes=c[:, ::2]), dict(codes=c.float()), dict(scales=s.view(2, 512)), dict(g=torch.ones(2)),
                dict(g=torch.ones(1, dtype=torch.float64)), dict(codes=torch.zeros(4, 128, dtype=torch.uint8)[:, ::2])):
        a = dict(codes=c, scales=s, fmt="nvfp4", k=100, g=g, **{}) | bad
        with pytest.raises(ValueError):
            ops._mx_check("t", a["codes"], a["scales"], a["fmt"], a["k"], a["g"])
    with pytest.raises(ValueError, match="tensor scale"):
        ops._mx_check("t", c, torch.zeros(512, dtype=torch.uint8), "mxfp4", 100, g)
    for a, w in (("nvfp4", "mxfp4"), ("mxfp8", "nvfp4"), ("mxfp8", "mxfp8"), ("int4", "int4")):
        with pytest.raises(ValueError, match="no product"):
            ops._mx_gemm_check("t", a, w, 8, None, torch.bfloat16)
    with pytest.raises(ValueError, match="bias"):
        ops._mx_gemm_check("t", "nvfp4", "nvfp4", 8, torch.zeros(8), torch.bfloat16)
    with pytest.raises(ValueError, match="output"):
        ops._mx_gemm_check("t", "nvfp4", "nvfp4", 8, None, torch.float64)


def test_layer_refusals():
    w = M.MicroTensor(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8), "nvfp4", (4, 64))
    with pytest.raises(ValueError, match="activation format"):
        M.MicroscaledLinear(w, act="int8")
    with pytest.raises(ValueError, match="mxfp4 weight"):
        M.MicroscaledLinear(w, act="mxfp8")
    with pytest.raises(ValueError, match="tensor scale"):
        M.MicroscaledLinear(M.MicroTensor(w.codes, w.scales, "mxfp4", (4, 64)), act="mxfp4", act_scale=torch.ones(1))
    layer = M.MicroscaledLinear(w)
    with pytest.raises(ValueError, match="takes nvfp4"):
        layer(M.MicroTensor(w.codes, w.scales, "mxfp4", (4, 64)))
    with pytest.raises(ValueError, match="do not match"):
        M.matmul(M.MicroTensor(w.codes, w.scales, "nvfp4", (4, 128)), w)


def test_c_abi_refusals():
    """Bad calls come back as a status before any CUDA call."""
    L = _lib.lib()
    p = ctypes.c_void_p(4096)

    def last():
        return L.svdq_last_error().decode()

    assert L.svdq_mx_quantize(p, 64, 0, 4, 64, 3, None, p, p, None) == 1 and "format" in last()
    assert L.svdq_mx_quantize(p, 64, 5, 4, 64, 0, None, p, p, None) == 1
    assert L.svdq_mx_quantize(p, 63, 0, 4, 64, 0, None, p, p, None) == 1
    assert L.svdq_mx_quantize(p, 64, 0, 4, 64, 1, p, p, p, None) == 1 and "tensor scale" in last()
    assert L.svdq_mx_quantize(p, 64, 0, 4, 64, 0, None, ctypes.c_void_p(4100), p, None) == 1 and "aligned" in last()
    assert L.svdq_mx_quantize(ctypes.c_void_p(4097), 64, 0, 4, 64, 0, None, p, p, None) == 1 and "elements" in last()
    assert L.svdq_mx_quantize(p, 64, 0, 4, 64, 0, ctypes.c_void_p(4098), p, p, None) == 1
    assert L.svdq_mx_dequantize(p, p, 0, None, 4, 64, ctypes.c_void_p(4098), 64, 2, None) == 1
    assert L.svdq_mx_tensor_scale(ctypes.c_void_p(4098), 64, 2, 4, 64, p, None) == 1
    assert L.svdq_mx_quantize(None, 64, 0, 4, 64, 0, None, p, p, None) == 1
    assert L.svdq_mx_quantize(p, 1 << 20, 0, 1 << 20, 1 << 20, 0, None, p, p, None) == 2
    assert L.svdq_mx_quantize(ctypes.c_void_p(4097), 64, 0, 4, 64, 0, None, p, p, None) == 1 and "elements" in last()
    assert L.svdq_mx_quantize(p, 64, 0, 4, 64, 0, ctypes.c_void_p(4098), p, p, None) == 1
    assert L.svdq_mx_dequantize(p, p, 0, None, 4, 64, ctypes.c_void_p(4098), 64, 2, None) == 1
    assert L.svdq_mx_tensor_scale(ctypes.c_void_p(4098), 64, 2, 4, 64, p, None) == 1
    assert L.svdq_mx_quantize(None, 64, 0, 0, 64, 0, None, None, None, None) == 0  # no rows: nothing to do
    assert L.svdq_mx_dequantize(p, p, 0, None, 4, 64, p, 60, 0, None) == 1
    assert L.svdq_mx_dequantize(p, p, 7, None, 4, 64, p, 64, 0, None) == 1
    assert L.svdq_mx_tensor_scale(p, 64, 9, 4, 64, p, None) == 1
    assert L.svdq_mx_tensor_scale(p, 64, 0, 4, 64, None, None) == 1

    def gemm(a_fmt=0, w_fmt=0, out=p, dt=0, ldo=64, m=4, n=64, k=64, codes=p, ga=None, bias=None):
        return L.svdq_mx_gemm(codes, p, a_fmt, ga, p, p, w_fmt, None, bias, out, dt, ldo, m, n, k, None)

    assert gemm(a_fmt=0, w_fmt=1) == 1 and "operands" in last()
    assert gemm(a_fmt=2, w_fmt=2) == 1 and gemm(a_fmt=1, w_fmt=2) == 1
    assert gemm(dt=3) == 1 and gemm(ldo=63) == 1 and gemm(n=0) == 1 and gemm(k=0) == 1 and gemm(m=-1) == 1
    assert gemm(codes=ctypes.c_void_p(4096 + 16)) == 1 and "aligned" in last()
    assert gemm(codes=None) == 1 and gemm(out=None) == 1
    assert gemm(out=ctypes.c_void_p(4097)) == 1 and gemm(bias=ctypes.c_void_p(4097)) == 1
    assert gemm(a_fmt=1, w_fmt=1, ga=p) == 1
    assert gemm(m=1 << 25) == 2
    assert gemm(m=0) == 0

    def lin(x=p, a_fmt=0, w_fmt=0, ws=p, nws=1 << 20, m=4, n=64, ldx=64, ldo=64, w=p, dt=0):
        return L.svdq_mx_linear(x, ldx, dt, a_fmt, None, w, p, w_fmt, None, None, p, 0, ldo, m, n, 64, ws, nws, None)

    need = L.svdq_mx_linear_workspace_bytes
    assert lin(a_fmt=5) == 1 and lin(m=5, ws=None) == 1 and lin(m=5, ws=ctypes.c_void_p(4096 + 16)) == 1
    assert lin(m=5, nws=need(5, 64, 0) - 1) == 1 and "workspace" in last()
    assert lin(w_fmt=1) == 1 and "operands" in last()
    assert lin(x=ctypes.c_void_p(4097)) == 1 and lin(w=None) == 1 and lin(w=ctypes.c_void_p(4096 + 16)) == 1
    assert lin(ldo=60) == 1 and lin(n=0) == 1 and lin(ldx=60) == 1 and lin(x=None) == 1 and lin(dt=7) == 1
    assert lin(m=0) == 0 and lin(m=0, ws=None) == 0
    assert need(0, 64, 0) == 0 and need(4, 64, 0) == 0 and need(5, 64, 9) == 0 and need(5, 64, 0) == 512 + 128 * 8
    assert need(300, 1000, 2) == 300 * 1024 + 384 * 32

    def norm(x=p, r=None, s=None, dt=0, eps=1e-6, m=4, h=64, ldx=64, ldr=64, lds=64):
        return L.svdq_rms_norm_mx(x, ldx, r, ldr, None, dt, eps, m, h, p, p, s, lds, None)

    assert norm(r=p) == 1 and norm(s=p) == 1 and norm(dt=4) == 1 and norm(eps=-1.0) == 1 and norm(ldx=60) == 1
    assert norm(x=ctypes.c_void_p(4097)) == 1 and norm(r=ctypes.c_void_p(4097), s=p) == 1
    assert norm(x=None) == 1 and norm(h=0) == 1 and norm(r=p, s=p, ldr=60) == 1 and norm(m=0) == 0


def test_a_launch_makes_its_device_current(monkeypatch):
    """A launch for another device than the current one runs inside that device's guard, on its stream."""
    seen, here = [], [0]

    class Lib:
        def svdq_probe(self, *args):
            seen.append((here[0], args))
            return 0

    class Guard:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.was, here[0] = here[0], self.dev.index

        def __exit__(self, *exc):
            here[0] = self.was

    monkeypatch.setattr(ops._lib, "lib", lambda: Lib())
    monkeypatch.setattr(ops, "_current_device", lambda: here[0])
    monkeypatch.setattr(ops, "_current_stream", lambda i: 100 + i)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 100 + dev.index)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    ops._launch(torch.device("cuda", 0), "svdq_probe", 7)
    ops._launch(torch.device("cuda", 1), "svdq_probe", 8)
    assert seen == [(0, (7, 100)), (1, (8, 101))] and here[0] == 0


def test_a_failing_launch_raises_the_library_error(monkeypatch):
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    monkeypatch.setattr(ops, "_current_stream", lambda i: None)
    with pytest.raises(_lib.SVDQError, match="format"):
        ops._launch(torch.device("cuda", 0), "svdq_mx_quantize", 4096, 64, 0, 4, 64, 9, None, 4096, 4096)


def test_rows_of_any_layout_are_taken_or_copied():
    x = torch.arange(60.0).view(5, 12)
    assert M._rows(x) is x and M._rows(x[:, 2:9]).data_ptr() == x[:, 2:9].data_ptr()
    for v in (x.t(), x[:1].expand(4, 12), x[:, ::2], x[None, :, 3:], x[0], x[:, 4]):
        r = M._rows(v)
        assert r.dim() == 2 and torch.equal(r.reshape(v.shape), v)
        ops._mx_rows("t", r)
    with pytest.raises(ValueError, match="dimension"):
        M._rows(torch.tensor(1.0))
    for bad in (x.double(), x.int(), x[0], x.t(), x[:1].expand(4, 12), x[:, :0]):
        with pytest.raises(ValueError):
            ops._mx_rows("t", bad)
