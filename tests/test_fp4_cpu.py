"""4-bit floating point without a GPU: the numpy definition against its own inverse, sizes of the layout, exported
symbols, and calls that are refused before any device work."""
import ctypes as C
import os
import re

import numpy as np
import pytest

from tests import fp4_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 0x1000  # never dereferenced: every call below is refused first


def _lib():
    from lidar_ai_solution_b200 import cabi
    return cabi, cabi.lib()


def test_library_exports_every_declared_symbol():
    cabi, lib = _lib()
    header = open(os.path.join(ROOT, "include", "spconvb_fp4.h")).read()
    declared = set(re.findall(r"SPCONVB_API[^;(]*?\b(spconvb_\w+)\s*\(", header))
    assert len(declared) == 9
    for name in sorted(declared):
        assert hasattr(lib, name) and name in cabi.SYMBOLS, name


@pytest.mark.parametrize("fmt", [ref.MX, ref.NV])
@pytest.mark.parametrize("channels", [1, 63, 64, 65, 128, 192, 200, 320, 4096])
def test_sizes_of_the_layout(fmt, channels):
    cabi, lib = _lib()
    assert lib.spconvb_fp4_code_pitch(channels) == ref.cpad(channels) // 2
    assert lib.spconvb_fp4_scale_pitch(fmt, channels) == ref.pitch(fmt, channels)
    assert ref.pitch(fmt, channels) % 4 == 0
    chunks = -(-ref.cpad(channels) // 256)
    words = 2 if fmt == ref.MX and ref.cpad(channels) != 64 else 4
    assert lib.spconvb_fp4_packed_bytes(fmt, channels, 130, 1) == 2 * chunks * (16384 + 512 * words)
    assert lib.spconvb_fp4_packed_bytes(fmt, channels, 64, 27) == -(-27 * ref.cpad(channels) // 256) * (16384 + 512 * words)


def test_sizes_that_are_not_offered():
    cabi, lib = _lib()
    for c in (0, -1, 65537):
        assert lib.spconvb_fp4_code_pitch(c) == 0 and lib.spconvb_fp4_scale_pitch(0, c) == 0
        assert lib.spconvb_fp4_packed_bytes(0, c, 64, 1) == 0 and lib.spconvb_fp4_packed_bytes(0, 64, c, 1) == 0
    assert lib.spconvb_fp4_scale_pitch(2, 64) == 0 and lib.spconvb_fp4_packed_bytes(-1, 64, 64, 1) == 0
    assert lib.spconvb_fp4_packed_bytes(1, 64, 64, 0) == 0 and lib.spconvb_fp4_packed_bytes(1, 64, 64, 28) == 0
    sup = lib.spconvb_fp4_conv_supported
    assert sup(1, 1, 1) and sup(64, 64, 27) and sup(128, 128, 27) and sup(256, 128, 27) and sup(193, 17, 5)
    assert not sup(129, 64, 27) and not sup(192, 64, 27) and not sup(257, 64, 1)
    assert not sup(64, 129, 1) and not sup(64, 64, 28) and not sup(0, 64, 1) and not sup(64, 0, 1) and not sup(64, 64, 0)


def test_refusals_of_rows():
    cabi, lib = _lib()

    def quantize(fmt=0, x=FAKE, kind=cabi.F16, ch=64, g=1.0, n=FAKE, rows=10, codes=FAKE, scales=FAKE):
        return lib.spconvb_fp4_quantize(fmt, x, kind, 1.0, ch, g, n, rows, codes, scales, None)

    def dequantize(fmt=0, out=FAKE, kind=cabi.F16, ch=64, g=1.0, n=FAKE, rows=10, codes=FAKE, scales=FAKE):
        return lib.spconvb_fp4_dequantize(fmt, codes, scales, ch, g, kind, n, rows, out, None)
    for f in (quantize, dequantize):
        assert f(fmt=2) == f(fmt=-1) == f(kind=3) == f(ch=0) == f(ch=65537) == -1
        assert f(n=None) == f(rows=0) == f(codes=None) == f(scales=None) == -1
        assert f(codes=FAKE + 8) == f(scales=FAKE + 4) == -1                       # 16-byte alignment
        assert f(g=2.0) == -1                                                      # MXFP4 has no tensor scale
        for g in (0.0, -1.0, float("nan"), float("inf"), 1e-40, 1e38):
            assert f(fmt=1, g=g) == -1
    assert quantize(x=None) == quantize(x=FAKE + 1) == quantize(kind=cabi.F32, x=FAKE + 2) == -1
    assert dequantize(out=None) == dequantize(out=FAKE + 1) == dequantize(kind=cabi.I8) == -1
    assert lib.spconvb_fp4_pack_weights(0, 64, 64, 1, None, FAKE, FAKE, None) == -1
    assert lib.spconvb_fp4_pack_weights(0, 64, 64, 1, FAKE, FAKE, FAKE + 8, None) == -1
    assert lib.spconvb_fp4_pack_weights(2, 64, 64, 1, FAKE, FAKE, FAKE, None) == -1
    assert lib.spconvb_fp4_pack_weights(0, 64, 64, 28, FAKE, FAKE, FAKE, None) == -1


def test_refusals_of_products():
    cabi, lib = _lib()

    def params(**kw):
        p = cabi.Fp4Params()
        p.format, p.cin, p.cout, p.kvol, p.alpha, p.in_rows = 0, 64, 64, 1, 1.0, 10
        for k, v in kw.items():
            setattr(p, k, v)
        return C.byref(p)

    def linear(p=None, codes=FAKE, scales=FAKE, n=FAKE, rows=10, w=FAKE, bias=None, out=FAKE, **kw):
        return lib.spconvb_fp4_linear(params(**kw) if p is None else p, codes, scales, n, rows, w, bias, out, None, None)

    def conv(p=None, codes=FAKE, scales=FAKE, n=FAKE, cap=10, w=FAKE, bias=None, out=FAKE, m=FAKE, **kw):
        return lib.spconvb_fp4_conv(params(**kw) if p is None else p, codes, scales, m, cap, n, 0, w, bias, out, None,
                                    None)
    for f in (linear, conv):
        assert f(codes=None) == f(scales=None) == f(n=None) == f(w=None) == f(out=None) == -1
        assert f(codes=FAKE + 8) == f(scales=FAKE + 8) == f(w=FAKE + 4) == f(out=FAKE + 1) == f(bias=FAKE + 2) == -1
        assert f(format=2) == f(cin=0) == f(cout=0) == f(cin=65537) == f(act=2) == -1
        assert f(out_fp4=1) == f(out_fp4=1, out_scales=FAKE, out_format=5) == -1
        assert f(out_fp4=1, out_scales=FAKE, out_format=1, out_tensor_scale=0.0) == -1
        assert f(out_fp4=1, out_scales=FAKE + 4, out_format=1, out_tensor_scale=1.0) == -1
        assert f(out_fp4=1, out_scales=FAKE, out_format=1, out_tensor_scale=1.0, out=FAKE + 8) == -1
    assert linear(kvol=2) == linear(rows=0) == linear(rows=0x7fffffff) == linear(res=FAKE) == -1
    assert linear(cout=65536, rows=0x7fffff00) == -2                               # more tiles than a grid has
    assert conv(m=None) == conv(m=FAKE + 2) == conv(cap=0) == conv(cap=0x80000000) == conv(res=FAKE + 1) == conv(in_rows=0) == -1
    assert conv(cin=192) == conv(cout=129) == conv(kvol=28) == -5


def test_python_calls_check_what_they_are_given():
    torch = pytest.importorskip("torch")
    from lidar_ai_solution_b200 import ops
    x = torch.zeros(8, 64, dtype=torch.float16)
    n = torch.tensor([8], dtype=torch.int32)
    for bad in (x.double(), x[:, ::2], x[0]):
        with pytest.raises(ValueError):
            ops.fp4_quantize(bad, n, ops.NVFP4)
    with pytest.raises(ValueError):
        ops.fp4_quantize(x, n.long(), ops.NVFP4)
    with pytest.raises(ValueError):           # not on the current device
        ops.fp4_quantize(x, n, ops.NVFP4)
    codes, scales = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8)
    q = ops.Fp4Rows(codes, scales, 64, ops.NVFP4, 0.5)
    assert (q.channels, q.fmt, q.tensor_scale) == (64, ops.NVFP4, 0.5)
    for args in ((codes[:, :16], scales, 64), (codes, scales[:4], 64), (codes, scales, 65), (codes.int(), scales, 64),
                 (codes, scales, 0)):
        with pytest.raises(ValueError):
            ops.Fp4Rows(*args, ops.NVFP4)
    for fmt, g in ((ops.NVFP4, 0.0), (ops.NVFP4, -1.0), (ops.NVFP4, float("nan")), (ops.NVFP4, float("inf")), (ops.MXFP4, 0.5)):
        with pytest.raises(ValueError):
            ops.Fp4Rows(codes, scales, 64, fmt, g)
        with pytest.raises(ValueError):
            ops.Fp4Weights(torch.zeros(4, 64), fmt, g, device="cpu")
    with pytest.raises(ValueError):
        ops.fp4_dequantize(q, n)
    with pytest.raises(ValueError):
        ops.Fp4Weights(torch.zeros(4, 4, 4, 4), ops.NVFP4, device="cpu")


@pytest.mark.parametrize("fmt", [ref.MX, ref.NV])
def test_definition_keeps_what_it_can_hold(fmt):
    """Values that codes and scales hold come back; others come back as the nearest of their block's."""
    rng = np.random.default_rng(0)
    x = ref.VALUES[rng.integers(0, 16, (20, 128))].astype(np.float32)
    x[:, ::16] = 6.0
    assert np.array_equal(ref.values(*ref.quantize(x, fmt), fmt, 128), x)
    x = rng.standard_normal((50, 100)).astype(np.float32)
    codes, scales = ref.quantize(x, fmt, 1.0 if fmt == ref.MX else 0.01)
    got = ref.values(codes, scales, fmt, 100, 1.0 if fmt == ref.MX else 0.01)
    s = np.repeat(ref.scale_values(scales, fmt, 100), (32, 16)[fmt], 1)[:, :100] * (1.0 if fmt == ref.MX else 0.01)
    grid = np.sort(np.unique(ref.VALUES))
    nearest = np.abs(x[..., None] / s[..., None] - grid).min(2)
    assert np.allclose(np.abs(x - got) / s, nearest, atol=1e-6)


@pytest.mark.parametrize("fmt", [ref.MX, ref.NV])
@pytest.mark.parametrize("cin,cout,kvol", [(192, 64, 27), (129, 64, 2), (320, 64, 27), (64, 129, 27), (257, 1, 3)])
def test_weights_that_no_product_takes_are_refused_when_they_are_laid_out(fmt, cin, cout, kvol):
    torch = pytest.importorskip("torch")
    from lidar_ai_solution_b200 import ops
    cabi, lib = _lib()
    assert lib.spconvb_fp4_pack_weights(fmt, cin, cout, kvol, FAKE, FAKE, FAKE, None) == -5
    for w in (torch.zeros(cout, kvol, cin), torch.zeros(cout, kvol, cin).numpy()):
        with pytest.raises(ValueError, match="the convolution takes no"):
            ops.Fp4Weights(w, fmt, device="cpu")
    with pytest.raises(ValueError, match="the convolution takes no"):
        ops.Fp4Weights((cout, kvol, cin), fmt, rows=ops.Fp4Rows.empty(cout * kvol, cin, fmt, device="cpu"))


def test_factors_that_are_not_finite_are_refused():
    cabi, lib = _lib()
    p = cabi.Fp4Params()
    p.format, p.cin, p.cout, p.kvol, p.in_rows = 1, 64, 64, 1, 10
    for alpha in (float("inf"), float("-inf"), float("nan")):
        p.alpha = alpha
        assert lib.spconvb_fp4_linear(C.byref(p), FAKE, FAKE, FAKE, 10, FAKE, None, FAKE, None, None) == -1
        assert lib.spconvb_fp4_conv(C.byref(p), FAKE, FAKE, FAKE, 10, FAKE, 0, FAKE, None, FAKE, None, None) == -1


def test_tensor_scales_that_the_library_does_not_take_are_refused_at_once():
    torch = pytest.importorskip("torch")
    from lidar_ai_solution_b200 import ops
    codes, scales = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8)
    for g in (1e-39, 1e-45, 7.7e35, 1e37):
        with pytest.raises(ValueError, match="tensor scale"):
            ops.Fp4Rows(codes, scales, 64, ops.NVFP4, g)
        with pytest.raises(ValueError, match="tensor scale"):
            ops.Fp4Weights((8, 64), ops.NVFP4, g, rows=ops.Fp4Rows(codes, scales, 64, ops.NVFP4, 1.0))
    for g in (1.2e-38, 7.5e35, 1):
        assert ops.Fp4Rows(codes, scales, 64, ops.NVFP4, g).tensor_scale == g


@pytest.mark.parametrize("rows", [2 ** 32, 2 ** 32 + 5, 2 ** 40])
def test_rows_beyond_32_bits_are_refused_and_not_cut_off(rows):
    torch = pytest.importorskip("torch")
    from lidar_ai_solution_b200 import ops
    meta = dict(dtype=torch.uint8, device="meta")          # shapes without memory
    with pytest.raises(ValueError, match="32 bits"):
        ops.Fp4Rows(torch.empty(rows, 32, **meta), torch.empty(rows, 4, **meta), 64, ops.NVFP4)
    with pytest.raises(ValueError, match="32 bits"):
        ops.Fp4Rows.empty(rows, 64, ops.NVFP4, device="meta")
    with pytest.raises(ValueError, match="32 bits"):
        ops.fp4_conv(None, torch.empty(1, rows, dtype=torch.int32, device="meta"), None,
                     type("Weights", (), dict(kvol=1, device_index=0)))
    assert ops.Fp4Rows.empty(2 ** 32 - 1, 64, ops.NVFP4, device="meta").rows == 2 ** 32 - 1
