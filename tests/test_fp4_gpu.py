"""4-bit floating-point rows and products on the GPU against their definition in numpy."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests import fp4_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu

FORMATS = [ref.MX, ref.NV]
IDS = ["mx", "nv"]


def _ops():
    from lidar_ai_solution_b200 import ops
    return ops


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _features(rows, channels, seed, spread=1.0):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, channels)) * np.exp(spread * rng.standard_normal((rows, 1)))
    x[rng.random((rows, channels)) < 0.1] = 0.0
    if rows > 3:
        x[rows // 2] = 0.0
    return x.astype(np.float32)


def _scale(x, fmt):
    top = float(np.abs(x).max()) or 1.0
    return 1.0 if fmt == ref.MX else float(np.float32(top / 2688))


def _quantized(x, fmt, g):
    """Rows on the GPU made by the reference, and the values they stand for without g."""
    ops = _ops()
    codes, scales = ref.quantize(x, fmt, g)
    q = ops.Fp4Rows(_dev(codes), _dev(scales), x.shape[1], fmt, g)
    return q, ref.values(codes, scales, fmt, x.shape[1])


def _check_codes(got, want_codes, want_scales):
    assert np.array_equal(got.scales.cpu().numpy(), want_scales)
    assert np.array_equal(ref.magnitude_codes(got.codes.cpu().numpy()), ref.magnitude_codes(want_codes))


# ------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("kind", ["f16", "f32", "i8"])
@pytest.mark.parametrize("rows,channels", [(1, 1), (1, 64), (3, 16), (33, 72), (257, 128), (1000, 63), (65, 192),
                                           (129, 100), (7, 1000), (2049, 256)])
def test_quantize_is_the_definition(fmt, kind, rows, channels):
    ops = _ops()
    x = _features(rows, channels, rows + channels)
    in_scale = 1.0
    if kind == "i8":
        in_scale = float(np.float32(np.abs(x).max() / 127)) or 1.0
        xi = np.clip(np.rint(x / np.float32(in_scale)), -128, 127).astype(np.int8)
        dev, x = _dev(xi), xi.astype(np.float32) * np.float32(in_scale)
    elif kind == "f16":
        x = x.astype(np.float16)
        dev, x = _dev(x), x.astype(np.float32)
    else:
        dev = _dev(x)
    g = _scale(x, fmt)
    codes, scales = ref.quantize(x, fmt, g)
    q = ops.fp4_quantize(dev, ops.device_count(rows), fmt, g, in_scale=in_scale)
    _check_codes(q, codes, scales)
    for out_kind, dt in ((ops.F16, np.float16), (ops.F32, np.float32)):
        with np.errstate(over="ignore"):
            want = ref.values(codes, scales, fmt, channels, g).astype(np.float32).astype(dt)
        got = ops.fp4_dequantize(q, ops.device_count(rows), out_kind).cpu().numpy()
        assert np.array_equal(got, want)


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_quantize_borders_and_extremes(fmt):
    """Values on and beside the borders between codes, blocks that saturate, vanish, or are not finite."""
    ops = _ops()
    near = np.concatenate([ref.BORDERS, ref.MAGNITUDES])
    near = np.concatenate([near, np.nextafter(near.astype(np.float32), np.float32(9)),
                           np.nextafter(near.astype(np.float32), np.float32(-9))]).astype(np.float32)
    rows = []
    for s in (1.0, 1.125, 0.6875, 2.0 ** -9, 448.0, 3 * 2.0 ** -9):
        r = np.zeros(64, np.float32)
        r[: len(near)] = near * np.float32(s)
        r[63] = 6 * s
        r[15] = r[31] = r[47] = 6 * s        # every block's largest magnitude is 6 s
        rows += [r, -r]
    big = np.full(64, 1e30, np.float32)
    tiny = np.full(64, 1e-42, np.float32)
    rows += [big, tiny, np.full(64, 65504, np.float32), np.full(64, -3.4e38, np.float32), 0 * big]
    for bad in (np.nan, np.inf, -np.inf):
        r = np.linspace(-3, 3, 64).astype(np.float32)
        r[5] = bad
        rows.append(r)
    x = np.stack(rows)
    for g in ((1.0,) if fmt == ref.MX else (1.0, 0.0078125, 1e-30, 1e30, 0.3)):
        codes, scales = ref.quantize(x, fmt, g)
        q = ops.fp4_quantize(_dev(x), ops.device_count(len(x)), fmt, g)
        _check_codes(q, codes, scales)
        got = ops.fp4_dequantize(q, ops.device_count(len(x)), ops.F32).cpu().numpy()
        with np.errstate(over="ignore"):
            want = ref.values(codes, scales, fmt, 64, g).astype(np.float32)
        assert np.array_equal(got, want, equal_nan=True)
        b = (32, 16)[fmt]
        assert np.isnan(got[-3:, :b]).all() and not np.isnan(got[-3:, b:]).any()


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("n", [0, 1, 5, 40, 1000])
def test_rows_behind_the_count_stay(fmt, n):
    """Also where the count is larger than the buffers."""
    ops = _ops()
    cap, ch = 40, 72
    x = _features(cap, ch, 1)
    g = _scale(x, fmt)
    out = ops.Fp4Rows.empty(cap, ch, fmt, g)
    out.codes.fill_(0xa5)
    out.scales.fill_(0x5a)
    ops.fp4_quantize(_dev(x), ops.device_count(n), fmt, g, out=out)
    codes, scales = ref.quantize(x, fmt, g)
    k = min(n, cap)
    assert np.array_equal(out.scales.cpu().numpy()[:k], scales[:k]) and bool((out.scales[k:] == 0x5a).all())
    assert bool((out.codes[k:] == 0xa5).all())
    full, v = _quantized(x, fmt, g)
    y = torch.full((cap, ch), 7.0, dtype=torch.float16, device="cuda")
    ops.fp4_dequantize(full, ops.device_count(n), out=y)
    assert bool((y[k:] == 7).all()) and not bool((y[:k] == 7).all(1).any())
    w = _features(24, ch, 2)
    wq = ops.Fp4Weights(w, fmt, _scale(w, fmt))
    y = torch.full((cap, 24), 7.0, dtype=torch.float16, device="cuda")
    ops.fp4_linear(full, ops.device_count(n), wq, out=y)
    assert bool((y[k:] == 7).all()) and not bool((y[:k] == 7).all(1).any())


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("offset", [1, 8, 16])
@pytest.mark.parametrize("channels", [64, 72, 40, 33])
def test_rows_at_any_element(fmt, offset, channels):
    """Inputs and outputs that start anywhere in their buffers."""
    ops = _ops()
    rows = 50
    x = _features(rows, channels, channels).astype(np.float16)
    flat = torch.zeros(rows * channels + 32, dtype=torch.float16, device="cuda")
    view = flat[offset:offset + rows * channels].view(rows, channels)
    view.copy_(_dev(x))
    g = _scale(x.astype(np.float32), fmt)
    codes, scales = ref.quantize(x, fmt, g)
    n = ops.device_count(rows)
    q = ops.fp4_quantize(view, n, fmt, g)
    _check_codes(q, codes, scales)
    back = torch.full_like(flat, 9.0)
    out = back[offset:offset + rows * channels].view(rows, channels)
    ops.fp4_dequantize(q, n, out=out)
    want = ref.values(codes, scales, fmt, channels, g).astype(np.float32).astype(np.float16)
    assert np.array_equal(out.cpu().numpy(), want)
    assert bool((back[:offset] == 9).all()) and bool((back[offset + rows * channels:] == 9).all())
    w = _features(channels, channels, 3)
    wq = ops.Fp4Weights(w, fmt, _scale(w, fmt))
    straight = ops.fp4_linear(q, n, wq)
    back.fill_(9.0)
    ops.fp4_linear(q, n, wq, out=out)
    assert torch.equal(out, straight)
    assert bool((back[:offset] == 9).all()) and bool((back[offset + rows * channels:] == 9).all())


# ---------------------------------------------------------------------------- products
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("rows,cin,cout", [
    (1, 64, 64), (1, 1, 1), (3, 16, 8), (128, 64, 64), (127, 256, 64), (129, 320, 65), (50, 200, 136), (300, 72, 130),
    (1, 4096, 512), (5, 4100, 100), (2, 200, 9), (4, 64, 130), (8, 1000, 264), (9, 300, 72), (64, 16384, 64), (130, 9000, 300), (7, 8200, 1000), (130, 2048, 256), (1000, 512, 300), (20000, 64, 64), (19000, 192, 128),
    (19100, 128, 200), (40000, 256, 256), (5000, 448, 1000)])
def test_linear(fmt, rows, cin, cout):
    ops = _ops()
    x, w = _features(rows, cin, 1, 0.3), _features(cout, cin, 2, 0.3) / np.float32(np.sqrt(cin))
    gx, gw = _scale(x, fmt), _scale(w, fmt)
    q, xv = _quantized(x, fmt, gx)
    wc, ws = ref.quantize(w, fmt, gw)
    bias = np.random.default_rng(3).standard_normal(cout).astype(np.float32)
    st = ops.new_status()
    for relu, b in ((False, None), (True, bias)):
        wq = ops.Fp4Weights(w, fmt, gw, b)
        got = ops.fp4_linear(q, ops.device_count(rows), wq, act=ops.ACT_RELU if relu else ops.ACT_NONE, status=st)
        y, off = ref.product(xv, ref.values(wc, ws, fmt, cin), float(np.float32(gx * gw)), b, relu)
        got = got.cpu().numpy().astype(np.float64)
        assert (np.abs(got - y) <= off).all(), float((np.abs(got - y) / off).max())
        assert int(st[0]) == 0


def _map(n, kvol, seed, live=0.25, n_in=None):
    """A neighbour map [kvol, n] into n_in rows: the centre tap is the row itself, others are there with probability `live`."""
    rng = np.random.default_rng(seed)
    n_in = n if n_in is None else n_in
    m = rng.integers(0, max(n_in, 1), (kvol, n)).astype(np.int32)
    m[rng.random((kvol, n)) >= live] = -1
    if n_in == n:
        m[kvol // 2] = np.arange(n)
    return m


def _gather(xv, m):
    """[n, kvol * cin] of the neighbours' values, zeros where there is none."""
    x = np.concatenate([xv, np.zeros((1, xv.shape[1]))])
    return x[m.T].reshape(m.shape[1], -1)


def _conv_problem(fmt, n, cin, cout, kvol, seed=0):
    ops = _ops()
    x = _features(n, cin, seed, 0.3)
    w = _features(cout * kvol, cin, seed + 1, 0.3) / np.float32(np.sqrt(kvol * cin))
    gx, gw = _scale(x, fmt), _scale(w, fmt)
    q, xv = _quantized(x, fmt, gx)
    wc, ws = ref.quantize(w, fmt, gw)
    wv = ref.values(wc, ws, fmt, cin).reshape(cout, kvol * cin)
    bias = np.random.default_rng(seed + 2).standard_normal(cout).astype(np.float32)
    wq = ops.Fp4Weights(w.reshape(cout, kvol, cin), fmt, gw, bias)
    return q, xv, wq, wv, float(np.float32(gx * gw)), bias


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("n,cin,cout,kvol", [
    (1, 64, 64, 27), (33, 64, 64, 27), (200, 128, 128, 27), (1000, 256, 128, 27), (777, 48, 24, 27), (500, 100, 100, 27),
    (5000, 64, 64, 27), (9000, 64, 128, 27), (30000, 64, 32, 27), (29000, 128, 128, 27), (24000, 128, 64, 9),
    (3000, 256, 64, 3), (4000, 64, 64, 1), (2000, 33, 1, 8), (60000, 64, 64, 3)])
def test_conv(fmt, n, cin, cout, kvol):
    ops = _ops()
    q, xv, wq, wv, alpha, bias = _conv_problem(fmt, n, cin, cout, kvol)
    m = _map(n, kvol, 5)
    dm, n_ptr, st = _dev(m), ops.device_count(n), ops.new_status()
    res = np.random.default_rng(6).standard_normal((n, cout)).astype(np.float16)
    cols = _gather(xv, m)
    for relu, r, rr in ((False, None, False), (True, res, True)):
        got = ops.fp4_conv(q, dm, n_ptr, wq, act=ops.ACT_RELU if relu else ops.ACT_NONE,
                           res=None if r is None else _dev(r), res_relu=rr, status=st)
        y, off = ref.product(cols, wv, alpha, bias, relu, None if r is None else r.astype(np.float64), rr)
        got = got.cpu().numpy().astype(np.float64)
        assert int(st[0]) == 0
        assert (np.abs(got - y) <= off).all(), float((np.abs(got - y) / off).max())


def _exact_rows(rows, channels, seed):
    """Rows whose blocks all have the scale 1 in either format (largest magnitude 6, tensor scale 1): products of such rows are
    multiples of 1/4 and their sums exact in fp32, whatever the order."""
    rng = np.random.default_rng(seed)
    v = ref.VALUES[rng.integers(0, 16, (rows, ref.cpad(channels)))]
    v[:, ::16] = 6.0
    v[:, 15::16] = -6.0
    return v[:, :channels].astype(np.float32)


@pytest.mark.parametrize("out_fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("rows,cin,cout", [(1, 64, 64), (130, 128, 72), (37, 320, 256), (257, 64, 24), (5, 2048, 130),
                                           (20000, 64, 64), (19000, 64, 200), (40000, 128, 256)])
def test_linear_to_4_bits_is_the_definition(fmt, out_fmt, rows, cin, cout):
    """Sums that are exact: every code and scale is that of the definition."""
    ops = _ops()
    x, w = _exact_rows(rows, cin, 1), _exact_rows(cout, cin, 2)
    q, xv = _quantized(x, fmt, 1.0)
    bias = np.random.default_rng(3).integers(-64, 64, cout).astype(np.float32) / 4
    g = 1.0 if out_fmt == ref.MX else 0.0625
    for relu in (False, True):
        got = ops.fp4_linear(q, ops.device_count(rows), ops.Fp4Weights(w, fmt, 1.0, bias),
                             act=ops.ACT_RELU if relu else ops.ACT_NONE, out_fmt=out_fmt, out_tensor_scale=g)
        y = xv @ w.T.astype(np.float64) + bias
        y = np.maximum(y, 0) if relu else y
        _check_codes(got, *ref.quantize(y.astype(np.float32), out_fmt, g))


@pytest.mark.parametrize("out_fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("n,cin,cout", [(1, 64, 64), (100, 64, 64), (3000, 64, 24), (3001, 128, 128), (30000, 64, 100),
                                        (5000, 128, 40), (700, 256, 128)])
def test_conv_to_4_bits_is_the_definition(fmt, out_fmt, n, cin, cout):
    ops = _ops()
    kvol = 27
    x, w = _exact_rows(n, cin, 1), _exact_rows(cout * kvol, cin, 2).reshape(cout, kvol, cin)
    q, xv = _quantized(x, fmt, 1.0)
    rng = np.random.default_rng(3)
    bias = rng.integers(-64, 64, cout).astype(np.float32) / 4
    m = _map(n, kvol, 4, 0.1)
    y = _gather(xv, m) @ w.reshape(cout, -1).T.astype(np.float64) + bias
    g = 1.0 if out_fmt == ref.MX else 0.5
    dm, n_ptr, wq = _dev(m), ops.device_count(n), ops.Fp4Weights(w, fmt, 1.0, bias)
    got = ops.fp4_conv(q, dm, n_ptr, wq, act=ops.ACT_RELU, out_fmt=out_fmt, out_tensor_scale=g)
    _check_codes(got, *ref.quantize(np.maximum(y, 0).astype(np.float32), out_fmt, g))
    # with a residual: both sums as fp16 stores them
    res = (rng.integers(-512, 512, (n, cout)) / 4).astype(np.float16)
    got = ops.fp4_conv(q, dm, n_ptr, wq, res=_dev(res), res_relu=True, out_fmt=out_fmt, out_tensor_scale=g)
    y = y.astype(np.float16).astype(np.float32) + res.astype(np.float32)
    _check_codes(got, *ref.quantize(np.maximum(y, 0), out_fmt, g))


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_not_finite_blocks_stay_visible(fmt):
    """A block that is not finite makes exactly the results that read it NaN, through ReLU and into 4 bits."""
    ops = _ops()
    rows, cin, cout, kvol = 300, 128, 64, 27
    x = _features(rows, cin, 1, 0.3)
    x[7, 100], x[250, 3] = np.inf, np.nan
    q, _ = _quantized(x, fmt, 1.0)
    w = _features(cout * kvol, cin, 2, 0.3)
    bad = np.zeros(rows, bool)
    bad[[7, 250]] = True
    n = ops.device_count(rows)
    y = ops.fp4_linear(q, n, ops.Fp4Weights(w[:cout], fmt), act=ops.ACT_RELU)
    assert np.array_equal(torch.isnan(y).all(1).cpu().numpy(), bad) and int(torch.isnan(y).sum()) == 2 * cout
    h = ops.fp4_linear(q, n, ops.Fp4Weights(w[:cout], fmt), act=ops.ACT_RELU, out_fmt=fmt)
    assert torch.equal(torch.isnan(ops.fp4_dequantize(h, n)), torch.isnan(y))
    m = _map(rows, kvol, 3, 0.05)
    hit = np.isin(m, [7, 250]).any(0)
    wq = ops.Fp4Weights(w.reshape(cout, kvol, cin), fmt)
    y = ops.fp4_conv(q, _dev(m), n, wq, act=ops.ACT_RELU)
    assert np.array_equal(torch.isnan(y).all(1).cpu().numpy(), hit) and int(torch.isnan(y).sum()) == hit.sum() * cout
    h = ops.fp4_conv(q, _dev(m), n, wq, act=ops.ACT_RELU, out_fmt=fmt)
    assert torch.equal(torch.isnan(ops.fp4_dequantize(h, n)), torch.isnan(y))


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("n", [0, 1, 31, 500, 10 ** 6])
@pytest.mark.parametrize("cap", [500, 504])
def test_conv_rows_behind_the_count_stay(fmt, n, cap):
    """Also where the count is larger than the buffers; launch_rows only sizes the grid."""
    ops = _ops()
    q, xv, wq, wv, alpha, bias = _conv_problem(fmt, cap, 64, 40, 27)
    m = _map(cap, 27, 5)
    y, off = ref.product(_gather(xv, m), wv, alpha, bias, False)
    k = min(n, cap)
    for launch_rows in (0, 64, cap + 100):
        out = torch.full((cap, 40), 7.0, dtype=torch.float16, device="cuda")
        ops.fp4_conv(q, _dev(m), ops.device_count(n), wq, out=out, launch_rows=launch_rows)
        out = out.cpu().numpy().astype(np.float64)
        assert (out[k:] == 7).all() and (np.abs(out - y)[:k] <= off[:k]).all()
    h = ops.Fp4Rows.empty(cap, 40, fmt)
    h.codes.fill_(0xa5)
    h.scales.fill_(0x5a)
    ops.fp4_conv(q, _dev(m), ops.device_count(n), wq, out_fmt=fmt, out=h)
    assert bool((h.codes[k:] == 0xa5).all()) and bool((h.scales[k:] == 0x5a).all())


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_strided_conv_reads_other_rows_than_it_writes(fmt):
    """A rulebook of the framework's own: a stride-2 convolution between two sets of rows."""
    from lidar_ai_solution_b200 import scenes
    ops = _ops()
    grid, n = (21, 120, 120), 6000
    coords = scenes.make_coords(n, grid, 1)
    k3, s2, p1 = (3, 3, 3), (2, 2, 2), (1, 1, 1)
    dc, n_ptr = _dev(coords), ops.device_count(n)
    _, n_out, m, _, _ = ops.down_map(dc, n_ptr, grid, None, k3, s2, p1, want_table=False)
    count = int(n_out)
    q, xv, wq, wv, alpha, bias = _conv_problem(fmt, n, 64, 128, 27)
    got = ops.fp4_conv(q, m, n_out, wq)[:count].cpu().numpy().astype(np.float64)
    y, off = ref.product(_gather(xv, m.cpu().numpy()[:, :count]), wv, alpha, bias, False)
    assert (np.abs(got - y) <= off).all() and count > 100
