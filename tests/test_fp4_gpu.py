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
    (1, 64, 64), (1, 1, 1), (3, 16, 8), (128, 64, 64), (127, 256, 64), (129, 320, 65), (50, 200, 136), (300, 72, 130), (300, 72, 131), (9000, 72, 330),
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
    (1, 64, 64, 27), (33, 64, 64, 27), (200, 128, 128, 27), (1000, 256, 128, 27), (777, 48, 24, 27), (500, 100, 100, 27), (1500, 64, 50, 27), (1500, 64, 33, 27), (1500, 128, 105, 9),
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


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("n,cin,cout,kvol", [
    (60000, 64, 64, 1), (60000, 64, 40, 8),    # one stage a tile, four tiles a CTA
    (60000, 64, 64, 9), (40000, 128, 64, 5),   # two
    (40000, 64, 64, 17), (40000, 256, 24, 5),  # three
    (20001, 128, 64, 27), (20001, 256, 64, 11),  # seven and six, weights that do not stay
    (40000, 128, 128, 1), (20001, 128, 104, 5),
])
def test_conv_of_few_and_many_stages(fmt, n, cin, cout, kvol):
    """Tiles of one stage, of even and of odd numbers of them, several to a CTA: sums that are exact, so every bit counts.  A launch's
    stages may be ready in any order; ten launches have to agree."""
    ops = _ops()
    x, w = _exact_rows(n, cin, 1), _exact_rows(cout * kvol, cin, 2).reshape(cout, kvol, cin)
    q, xv = _quantized(x, fmt, 1.0)
    m = _map(n, kvol, 4, 0.3)
    rng = np.random.default_rng(5)
    bias = rng.integers(-64, 64, cout).astype(np.float32) / 4
    wq, n_ptr, dm = ops.Fp4Weights(w, fmt, 1.0, bias), ops.device_count(n), _dev(m)
    # on the device, in 64 bits, tap by tap
    xd, wd = _dev(xv), _dev(w.astype(np.float64))
    y = _dev(bias.astype(np.float64)).expand(n, cout).clone()
    for k in range(kvol):
        there = torch.nonzero(dm[k] >= 0).flatten()
        y[there] += xd[dm[k][there].long()] @ wd[:, k].T
    want = y.to(torch.float16)
    res = _dev((rng.integers(-512, 512, (n, cout)) / 4).astype(np.float16))
    want_res = (want.float() + res.float()).to(torch.float16)
    st = ops.new_status()
    for _ in range(10):
        assert torch.equal(ops.fp4_conv(q, dm, n_ptr, wq, status=st), want)
        assert torch.equal(ops.fp4_conv(q, dm, n_ptr, wq, res=res, status=st), want_res)
    assert int(st[0]) == 0


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


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("rows,cin,cout,counts", [
    (1300, 1100, 1800, (1300, 0, 1, 128, 129, 257, 1000)),  # tiles of 256 x 256: the last one of 20 rows, of 8 channels
    (1281, 1281, 1928, (1281, 1280)),                       # the last one of 1 row, of 136 channels
    (20000, 2304, 256, (20000, 18945)),                     # several tiles a pair of SMs
])
def test_large_linear_layers(fmt, rows, cin, cout, counts):
    ops = _ops()
    x, w = _features(rows, cin, 1, 0.3), _features(cout, cin, 2, 0.3) / np.float32(np.sqrt(cin))
    gx, gw = _scale(x, fmt), _scale(w, fmt)
    q, xv = _quantized(x, fmt, gx)
    wc, ws = ref.quantize(w, fmt, gw)
    bias = np.random.default_rng(3).standard_normal(cout).astype(np.float32)
    wq = ops.Fp4Weights(w, fmt, gw, bias)
    y, off = ref.product(xv, ref.values(wc, ws, fmt, cin), float(np.float32(gx * gw)), bias, True)
    st = ops.new_status()
    for n in counts:
        out = torch.full((rows, cout), 7.0, dtype=torch.float16, device="cuda")
        ops.fp4_linear(q, ops.device_count(n), wq, act=ops.ACT_RELU, out=out, status=st)
        got = out.cpu().numpy().astype(np.float64)
        assert (np.abs(got[:n] - y[:n]) <= off[:n]).all(), n
        assert (got[n:] == 7.0).all(), n
        assert int(st[0]) == 0


@pytest.mark.parametrize("out_fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_large_linear_layers_to_4_bits(fmt, out_fmt):
    ops = _ops()
    rows, cin, cout = 1300, 1100, 1800
    x, w = _exact_rows(rows, cin, 1), _exact_rows(cout, cin, 2)
    q, xv = _quantized(x, fmt, 1.0)
    g = 1.0 if out_fmt == ref.MX else 0.0625
    got = ops.fp4_linear(q, ops.device_count(rows), ops.Fp4Weights(w, fmt, 1.0), out_fmt=out_fmt, out_tensor_scale=g)
    _check_codes(got, *ref.quantize((xv @ w.T.astype(np.float64)).astype(np.float32), out_fmt, g))


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_large_linear_layers_replayed_on_two_streams(fmt):
    """Captured, replayed with other inputs and counts while another stream runs a layer of its own: the bits of a call alone."""
    ops = _ops()
    rows, cin, cout = 1300, 1100, 1800
    xs = [_features(rows, cin, i, 0.3) for i in range(3)]
    g = max(_scale(x, fmt) for x in xs)
    w = _features(cout, cin, 5, 0.3) / np.float32(np.sqrt(cin))
    wq = ops.Fp4Weights(w, fmt, _scale(w, fmt))
    qs = [_quantized(x, fmt, g)[0] for x in xs]
    alone = [ops.fp4_linear(q, ops.device_count(rows), wq).cpu() for q in qs]
    q, n_ptr = _quantized(xs[0], fmt, g)[0], ops.device_count(rows)
    side = torch.cuda.Stream()
    out = torch.empty((rows, cout), dtype=torch.float16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.fp4_linear(q, n_ptr, wq, out=out)
    for i, n in ((1, 1300), (2, 700), (0, 1), (1, 0), (2, 1300)):
        q.codes.copy_(qs[i].codes)
        q.scales.copy_(qs[i].scales)
        n_ptr.fill_(n)
        out.fill_(3.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            other = [ops.fp4_linear(qs[0], ops.device_count(rows), wq) for _ in range(4)]
        graph.replay()
        torch.cuda.synchronize()
        got = out.cpu()
        assert torch.equal(got[:n], alone[i][:n]) and (got[n:] == 3.0).all()
        assert all(torch.equal(o.cpu(), alone[0]) for o in other)


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


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_conv_takes_rows_beyond_the_input_as_missing(fmt):
    """Entries of the map that no row of the input has: nothing is read for them."""
    ops = _ops()
    n_in, n = 300, 900
    q, xv, wq, wv, alpha, bias = _conv_problem(fmt, n_in, 64, 64, 27)
    m = _map(n, 27, 5, n_in=n_in)
    rng = np.random.default_rng(1)
    bad = m.copy()
    bad[rng.random(m.shape) < 0.2] = rng.choice([n_in, n_in + 1, 2 ** 31 - 1, -2, -2 ** 31])
    bad[0, :4] = (n_in, 2 ** 31 - 1, -2 ** 31, -7)
    clean = np.where((bad < 0) | (bad >= n_in), -1, bad)
    y, off = ref.product(_gather(xv, clean), wv, alpha, bias, False)
    got = ops.fp4_conv(q, _dev(bad), ops.device_count(n), wq).cpu().numpy().astype(np.float64)
    assert (np.abs(got - y) <= off).all()


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_missing_neighbours_add_nothing_whatever_lay_there(fmt):
    """After rows of large values in every stage: rows with no neighbour at all, and rows whose only one is zero, give the bias;
    the map may start at any word."""
    ops = _ops()
    n = 3000
    q, xv, wq, wv, alpha, bias = _conv_problem(fmt, n, 64, 64, 27)
    x = _features(n, 64, 9, 0.3)
    x[::7] = 0.0
    q0, _ = _quantized(x, fmt, _scale(x, fmt))
    big, _ = _quantized(np.full((n, 64), 6e4, np.float32), fmt, 1.0)
    n_ptr = ops.device_count(n)
    every = _dev(_map(n, 27, 1, live=1.1))
    flat = torch.full((27 * n + 1,), -1, dtype=torch.int32, device="cuda")
    none = flat[1:].view(27, n)
    m = np.full((27, n), -1, np.int32)
    m[5] = np.arange(n) // 7 * 7
    for lone in (none, _dev(m)):
        ops.fp4_conv(big, every, n_ptr, wq)
        y = ops.fp4_conv(q0, lone, n_ptr, wq)
        assert torch.equal(y, torch.from_numpy(bias).half().cuda().expand(n, 64))


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_residual_may_be_the_output(fmt):
    ops = _ops()
    n = 3001
    q, xv, wq, wv, alpha, bias = _conv_problem(fmt, n, 64, 104, 27)
    m, n_ptr = _dev(_map(n, 27, 5)), ops.device_count(n)
    res = torch.randn(n, 104, device="cuda").half()
    want = ops.fp4_conv(q, m, n_ptr, wq, res=res, res_relu=True)
    ops.fp4_conv(q, m, n_ptr, wq, res=res, res_relu=True, out=res)
    assert torch.equal(res, want)


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("n", [40000, 39990, 31])
def test_wide_conv_over_its_own_residual(fmt, n):
    """The residual is the output, rows behind the count stay, a slice of a larger buffer around them does too."""
    ops = _ops()
    cap, c = 40000, 128
    q, xv, wq, wv, alpha, bias = _conv_problem(fmt, cap, c, c, 3)
    m, n_ptr = _dev(_map(cap, 3, 5)), ops.device_count(n)
    buf = torch.randn((cap + 2, c), dtype=torch.float32, device="cuda").to(torch.float16)
    buf[:1], buf[-1:] = 7.0, 9.0
    before = buf.clone()
    apart = ops.fp4_conv(q, m, n_ptr, wq, res=before[1:-1].contiguous(), res_relu=True)
    mine = buf[1:-1]
    assert ops.fp4_conv(q, m, n_ptr, wq, res=mine, res_relu=True, out=mine) is mine
    assert torch.equal(buf[1:n + 1], apart[:n])
    assert torch.equal(buf[n + 1:], before[n + 1:]) and torch.equal(buf[:1], before[:1])


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_weights_quantised_elsewhere(fmt):
    """Codes and scales of the weights that the caller has, and arrays in fp16."""
    ops = _ops()
    cout, kvol, cin = 72, 27, 100
    w = (_features(cout * kvol, cin, 1, 0.3) / 50).astype(np.float16)
    g = _scale(w.astype(np.float32), fmt)
    codes, scales = ref.quantize(w.astype(np.float32), fmt, g)
    rows = ops.Fp4Rows(_dev(codes), _dev(scales), cin, fmt, g)
    given = ops.Fp4Weights((cout, kvol, cin), fmt, g, rows=rows)
    made = ops.Fp4Weights(w.reshape(cout, kvol, cin), fmt, g)
    q, _ = _quantized(_features(500, cin, 2), fmt, 1.0)
    m, n = _dev(_map(500, kvol, 3)), ops.device_count(500)
    assert torch.equal(ops.fp4_conv(q, m, n, given), ops.fp4_conv(q, m, n, made))
    with pytest.raises(ValueError):
        ops.Fp4Weights((cout, kvol, cin + 1), fmt, g, rows=rows)
    with pytest.raises(ValueError):
        ops.Fp4Weights(w.reshape(cout, kvol, cin), fmt, g, bias=np.zeros(cout + 1))


def test_products_refuse_what_does_not_fit():
    ops = _ops()
    q, _ = _quantized(_features(8, 64, 1), ref.NV, 0.01)
    n = ops.device_count(8)
    wq = ops.Fp4Weights(_features(24, 64, 2), ref.NV, 0.01)
    other = ops.Fp4Weights(_features(24, 64, 2), ref.MX)
    wide = ops.Fp4Weights(_features(24, 128, 2), ref.NV, 0.01)
    m = torch.zeros((1, 8), dtype=torch.int32, device="cuda")
    for bad in (other, wide):
        with pytest.raises(ValueError):
            ops.fp4_linear(q, n, bad)
    for kw in (dict(out=torch.empty(8, 25, dtype=torch.float16, device="cuda")),
               dict(out=torch.empty(8, 24, device="cuda")), dict(out=torch.empty(8, 24, dtype=torch.float16)),
               dict(out_fmt=ref.MX, out=ops.Fp4Rows.empty(8, 24, ref.NV)), dict(status=torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.fp4_linear(q, n, wq, **kw)
    with pytest.raises(ValueError):
        ops.fp4_linear(q, torch.tensor([8], dtype=torch.int32), wq)
    with pytest.raises(ValueError):
        ops.fp4_conv(q, m.long(), n, wq)
    with pytest.raises(ValueError):
        ops.fp4_conv(q, m, n, wq, res=torch.zeros(8, 25, dtype=torch.float16, device="cuda"))
    with pytest.raises(RuntimeError):        # a tensor scale for MXFP4
        ops.fp4_quantize(torch.zeros(4, 64, device="cuda"), n, ref.MX, 2.0)
    w192 = ops.Fp4Weights(_features(24, 192, 2), ref.NV, 0.01)
    q192, _ = _quantized(_features(8, 192, 1), ref.NV, 0.01)
    with pytest.raises(RuntimeError):        # rows of 96 bytes: the convolution does not take them
        ops.fp4_conv(q192, m, n, w192)
    assert ops.fp4_quantize(torch.zeros(0, 64, device="cuda"), n, ref.NV).codes.shape == (0, 32)


def _chain(ops, x, n, m, ws, fmt, g):
    """How they are used together: rows to 4 bits, a residual block, a pointwise layer, back to fp16."""
    q = ops.fp4_quantize(x, n, fmt, g[0])
    h = ops.fp4_conv(q, m, n, ws[0], act=ops.ACT_RELU, out_fmt=fmt, out_tensor_scale=g[1])
    y = ops.fp4_conv(h, m, n, ws[1], res=x, res_relu=True)
    p = ops.fp4_linear(ops.fp4_quantize(y, n, fmt, g[2]), n, ws[2], out_fmt=fmt, out_tensor_scale=g[3])
    return h, y, ops.fp4_dequantize(p, n)


def _chain_problem(fmt, n, c, seed):
    ops = _ops()
    x = _features(n, c, seed, 0.2).astype(np.float16)
    g = [_scale(x.astype(np.float32), fmt)] + [1.0 if fmt == ref.MX else 0.004] * 3
    w = [_features(c * 27, c, 2, 0.3).reshape(c, 27, c) / 20, _features(c * 27, c, 3, 0.3).reshape(c, 27, c) / 20,
         _features(200, c, 4, 0.3) / 8]
    gw = [_scale(v, fmt) for v in w]
    rng = np.random.default_rng(5)
    bias = [rng.standard_normal(v.shape[0]).astype(np.float32) for v in w]
    ws = [ops.Fp4Weights(v, fmt, s, b) for v, s, b in zip(w, gw, bias)]
    wv = [ref.values(*ref.quantize(v.reshape(-1, c), fmt, s), fmt, c).reshape(v.shape[0], -1)
          for v, s in zip(w, gw)]
    return x, _map(n, 27, seed + 7, 0.2), ws, wv, g, gw, bias


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("n,c", [(2500, 64), (700, 128)])
def test_a_run_of_them_together(fmt, n, c):
    """Each stage against 64 bits on what the stage before left (a code that lies on a border may fall either way)."""
    ops = _ops()
    x, m, ws, wv, g, gw, bias = _chain_problem(fmt, n, c, 0)
    h, y, z = _chain(ops, _dev(x), ops.device_count(n), _dev(m), ws, fmt, g)
    xq = ref.values(*ref.quantize(x.astype(np.float32), fmt, g[0]), fmt, c)
    y1, off1 = ref.product(_gather(xq, m), wv[0], float(np.float32(g[0] * gw[0])), bias[0], True)
    codes, scales = ref.quantize(y1.astype(np.float32), fmt, g[1])
    assert (ref.magnitude_codes(h.codes.cpu().numpy()) != ref.magnitude_codes(codes)).mean() < 1e-3
    assert (h.scales.cpu().numpy() != scales).mean() < 1e-3
    hv = ref.values(h.codes.cpu().numpy(), h.scales.cpu().numpy(), fmt, c)
    y2, off2 = ref.product(_gather(hv, m), wv[1], float(np.float32(g[1] * gw[1])), bias[1], False,
                           x.astype(np.float64), True)
    got = y.cpu().numpy().astype(np.float64)
    assert (np.abs(got - y2) <= off2).all()
    yv = ref.values(*ref.quantize(y.cpu().numpy().astype(np.float32), fmt, g[2]), fmt, c)
    y3, _ = ref.product(yv, wv[2], float(np.float32(g[2] * gw[2])), bias[2], False)
    codes, scales = ref.quantize(y3.astype(np.float32), fmt, g[3])
    want = ref.values(codes, scales, fmt, 200, g[3]).astype(np.float32).astype(np.float16)
    assert (z.cpu().numpy() != want).mean() < 2e-3


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_captured_and_replayed_on_other_inputs_and_counts(fmt):
    """Two graphs of the same chain, on another stream, replayed beside one another's and with other rows and counts."""
    ops = _ops()
    n, c = 1500, 64
    problems = [_chain_problem(fmt, n, c, s) for s in (0, 1, 2)]
    ws, g = problems[0][2], problems[0][4]
    side = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(side):
        for k in range(2):
            x, m, cnt = _dev(problems[k][0]), _dev(problems[k][1]), ops.device_count(n)
            _chain(ops, x, cnt, m, ws, fmt, g)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = _chain(ops, x, cnt, m, ws, fmt, g)
            graphs.append((graph, x, m, cnt, out))
    torch.cuda.synchronize()
    for _ in range(2):
        for k, (graph, x, m, cnt, out) in enumerate(graphs):
            p = problems[k + 1]
            x.copy_(_dev(p[0]))
            rows = n if k else 777
            m.copy_(_dev(np.where(p[1] < rows, p[1], -1)))      # a rulebook points at rows below the count
            cnt.fill_(rows)
            torch.cuda.synchronize()
            graph.replay()
        torch.cuda.synchronize()
        for k, (graph, x, m, cnt, out) in enumerate(graphs):
            rows = int(cnt)
            want = _chain(ops, x.clone(), cnt, m.clone(), ws, fmt, g)
            for a, b in zip(out, want):
                a, b = (v.codes if isinstance(v, ops.Fp4Rows) else v for v in (a, b))
                assert torch.equal(a[:rows], b[:rows])


def test_two_streams_at_once_give_what_one_gives():
    ops = _ops()
    problems = [_chain_problem(ref.NV, 2500, 64, s) for s in (0, 1)]
    args = [(_dev(p[0]), ops.device_count(2500), _dev(p[1]), p[2], ref.NV, p[4]) for p in problems]
    want = [_chain(ops, *a)[1] for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(_chain(ops, *args[k])[1])
    torch.cuda.synchronize()
    assert all(torch.equal(v, want[k]) for k in range(2) for v in got[k])


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_bounded_waits_run_out_and_the_context_survives(fmt):
    """Producers that withhold a stage: the launch ends with the status bit, and the next one is right."""
    from lidar_ai_solution_b200 import cabi
    ops = _ops()
    n = 2000
    q, xv, wq, wv, alpha, bias = _conv_problem(fmt, n, 64, 64, 27)
    m, n_ptr = _dev(_map(n, 27, 5)), ops.device_count(n)
    good = ops.fp4_conv(q, m, n_ptr, wq)
    lin = ops.Fp4Weights(_features(64, 64, 3), fmt, 1.0)
    tall = ops.Fp4Weights(_features(64, 16384, 3), fmt, 1.0)
    qt, _ = _quantized(_features(40, 16384, 4, 0.1), fmt, 1.0)
    nt = ops.device_count(40)
    good_lin, good_tall = ops.fp4_linear(q, n_ptr, lin), ops.fp4_linear(qt, nt, tall)
    for call in (lambda st, w: ops.fp4_conv(q, m, n_ptr, wq, status=st, wait_test=w),
                 lambda st, w: ops.fp4_linear(q, n_ptr, lin, status=st, wait_test=w),
                 lambda st, w: ops.fp4_linear(qt, nt, tall, status=st, wait_test=w)):
        st = ops.new_status()
        call(st, 1)
        torch.cuda.synchronize()
        assert int(st[0]) == cabi.ST_TIMEOUT
    st = ops.new_status()
    assert torch.equal(ops.fp4_conv(q, m, n_ptr, wq, status=st), good)
    assert torch.equal(ops.fp4_linear(q, n_ptr, lin, status=st), good_lin)
    assert torch.equal(ops.fp4_linear(qt, nt, tall, status=st), good_tall)
    assert int(st[0]) == 0


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
def test_bounded_waits_of_a_large_linear_layer(fmt):
    """Copies withheld at the first chunk, inside a tile and at a later tile: the launch ends with the status bit, the next one is right."""
    from lidar_ai_solution_b200 import cabi
    ops = _ops()
    rows, cin, cout = 20000, 2304, 256
    q, _ = _quantized(_features(rows, cin, 1, 0.1), fmt, 1.0)
    wq, n_ptr = ops.Fp4Weights(_features(cout, cin, 2, 0.1), fmt, 1.0), ops.device_count(rows)
    good = ops.fp4_linear(q, n_ptr, wq)
    for at in (1, 4, 9):
        st = ops.new_status()
        ops.fp4_linear(q, n_ptr, wq, status=st, wait_test=at)
        torch.cuda.synchronize()
        assert int(st[0]) == cabi.ST_TIMEOUT
    st = ops.new_status()
    assert torch.equal(ops.fp4_linear(q, n_ptr, wq, status=st), good)
    assert int(st[0]) == 0


def test_the_same_call_gives_the_same_bits():
    ops = _ops()
    q, xv, wq, wv, alpha, bias = _conv_problem(ref.NV, 9000, 128, 128, 27)
    m, n_ptr = _dev(_map(9000, 27, 5)), ops.device_count(9000)
    first = ops.fp4_conv(q, m, n_ptr, wq)
    w = ops.Fp4Weights(_features(300, 9000, 2, 0.1), ref.MX)
    qx, _ = _quantized(_features(100, 9000, 3, 0.1), ref.MX, 1.0)
    n2 = ops.device_count(100)
    second = ops.fp4_linear(qx, n2, w)
    for _ in range(10):
        assert torch.equal(ops.fp4_conv(q, m, n_ptr, wq), first)
        assert torch.equal(ops.fp4_linear(qx, n2, w), second)


def test_offsets_beyond_32_bits():
    """140 M rows: codes, scales and fp16 rows whose last ones lie beyond 2^32 bytes."""
    ops = _ops()
    rows, ch = 140_000_000, 64
    x = torch.zeros((rows, ch), dtype=torch.int8, device="cuda")
    at = torch.tensor([0, 1, 67_108_863, 67_108_864, 134_217_728, rows - 2, rows - 1], device="cuda")
    piece = torch.randint(-127, 128, (len(at), ch), device="cuda").to(torch.int8)
    x[at] = piece
    g, s = 0.0009765625, 0.0078125
    n = ops.device_count(rows)
    q = ops.fp4_quantize(x, n, ref.NV, g, in_scale=s)
    want = ref.quantize(piece.cpu().numpy().astype(np.float32) * np.float32(s), ref.NV, g)
    codes, scales = q.codes[at].cpu().numpy(), q.scales[at].cpu().numpy()
    assert np.array_equal(scales, want[1])
    assert np.array_equal(ref.magnitude_codes(codes), ref.magnitude_codes(want[0]))
    del x
    w = _features(8, ch, 2)
    wq = ops.Fp4Weights(w, ref.NV, 0.01)
    y = ops.fp4_linear(q, n, wq)[at].cpu().numpy().astype(np.float64)
    wv = ref.values(*ref.quantize(w, ref.NV, 0.01), ref.NV, ch)
    full, off = ref.product(ref.values(*want, ref.NV, ch), wv, float(np.float32(g * 0.01)), None, False)
    assert (np.abs(y - full) <= off).all()
    back = ops.fp4_dequantize(q, n)
    exact = ref.values(*want, ref.NV, ch, g).astype(np.float32).astype(np.float16)
    assert np.array_equal(back[at].cpu().numpy(), exact)
    # a convolution that reads the far ones
    m = at.to(torch.int32).repeat(3, 1).contiguous()
    m[1] = -1
    cw = ops.Fp4Weights(_features(24, ch, 4).reshape(8, 3, ch), ref.NV, 0.01)
    got = ops.fp4_conv(q, m, ops.device_count(len(at)), cw).cpu().numpy().astype(np.float64)
    cv = ref.values(*ref.quantize(_features(24, ch, 4), ref.NV, 0.01), ref.NV, ch).reshape(8, -1)
    mm = np.tile(np.arange(len(at)), (3, 1))
    mm[1] = -1
    y, off = ref.product(_gather(ref.values(*want, ref.NV, ch), mm), cv, float(np.float32(g * 0.01)), None, False)
    assert (np.abs(got - y) <= off).all()


@pytest.mark.parametrize("rows,cin,cout", [(1, 512, 64), (8, 300, 41), (64, 16384, 64), (300, 200, 131), (20000, 1024, 256)])
def test_every_form_of_the_linear_layer_is_captured_and_replayed(rows, cin, cout):
    """Few rows, a split K, odd channels, wide tiles: a graph gives what calls give, on rows that came later."""
    ops = _ops()
    w = ops.Fp4Weights(_features(cout, cin, 1, 0.1), ref.NV, 0.01)
    q, _ = _quantized(_features(rows, cin, 2, 0.1), ref.NV, 0.01)
    later, _ = _quantized(_features(rows, cin, 3, 0.1), ref.NV, 0.01)
    n = ops.device_count(rows)
    ops.fp4_linear(q, n, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.fp4_linear(q, n, w, act=ops.ACT_RELU)
    want = ops.fp4_linear(later, n, w, act=ops.ACT_RELU)
    q.codes.copy_(later.codes)
    q.scales.copy_(later.scales)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_few_rows_of_extreme_scales():
    """Blocks whose scales' product is beyond fp32, with and without products of codes."""
    ops = _ops()
    x = np.zeros((2, 64), np.float32)
    x[0, 0], x[1, 1] = 6 * 2.0 ** 100, 3 * 2.0 ** -100
    w = np.zeros((8, 64), np.float32)
    w[0, 2], w[1, 0], w[2, 1] = 2.0 ** 60, 2.0 ** -100, 2.0 ** 100
    q, _ = _quantized(x, ref.MX, 1.0)
    for rows in (2, 9):                      # on the CUDA cores, and on the tensor cores
        codes, scales = ref.quantize(np.concatenate([x, np.zeros((rows - 2, 64), np.float32)]), ref.MX)
        q = ops.Fp4Rows(_dev(codes), _dev(scales), 64, ref.MX)
        y = ops.fp4_linear(q, ops.device_count(rows), ops.Fp4Weights(w, ref.MX)).cpu().numpy()
        assert np.array_equal(y[:2], (x.astype(np.float64) @ w.T.astype(np.float64)).astype(np.float16)), rows
        assert not y[2:].any()


@pytest.mark.parametrize("g,top", [(1e-20, 1e20), (1e-20, 1e19), (1e-27, 1e29), (2e-28, 3.4e38), (1e-27, 2e3), (1e-20, 3e18), (1.0, 3e38)])
def test_scales_saturate_however_far_a_block_is_from_its_tensor_scale(g, top):
    """amax / (6 g) up to the border of fp32 and beyond it is 448, and not NaN: of rows in fp32 and scaled int8."""
    ops = _ops()
    x = np.zeros((5, 100), np.float32)
    x[0], x[1, ::16] = np.linspace(-top, top, 100), top
    x[2], x[3, 7] = 6 * 448 * np.float32(g) * np.linspace(-1, 1, 100), np.float32(top) / 2
    codes, scales = ref.quantize(x, ref.NV, g)
    assert (scales[:2, :7] == 0x7e).all() and not (scales == 0x7f).any()
    n = ops.device_count(5)
    q = ops.fp4_quantize(_dev(x), n, ref.NV, g)
    _check_codes(q, codes, scales)
    assert torch.isfinite(ops.fp4_dequantize(q, n, ops.F32)).all()
    xi = np.arange(-100, 100, 1, np.int8).reshape(2, 100)
    in_scale = float(np.float32(top / 128))
    codes, scales = ref.quantize(xi.astype(np.float32) * np.float32(in_scale), ref.NV, g)
    _check_codes(ops.fp4_quantize(_dev(xi), ops.device_count(2), ref.NV, g, in_scale=in_scale), codes, scales)


@pytest.mark.parametrize("rows", [37, 20000])
def test_outputs_saturate_however_far_they_are_from_their_tensor_scale(rows):
    """The same of a product's 4-bit rows: sums that are exact, times 2^80."""
    ops = _ops()
    x, w = _exact_rows(rows, 64, 1), _exact_rows(72, 64, 2)
    codes, scales = ref.quantize(x, ref.NV, 1.0)
    big = ops.Fp4Rows(_dev(codes), _dev(scales), 64, ref.NV, 2.0 ** 40)
    wr = ops.fp4_quantize(_dev(w), ops.device_count(72), ref.NV, 1.0)
    wq = ops.Fp4Weights((72, 64), ref.NV, 2.0 ** 40, rows=ops.Fp4Rows(wr.codes, wr.scales, 64, ref.NV, 2.0 ** 40))
    y = (x.astype(np.float64) @ w.T.astype(np.float64) * 2.0 ** 80).astype(np.float32)
    for g in (2.0 ** -66, 2.0 ** -80, 2.0 ** 60, 2.0 ** 80):
        got = ops.fp4_linear(big, ops.device_count(rows), wq, out_fmt=ref.NV, out_tensor_scale=g)
        _check_codes(got, *ref.quantize(y, ref.NV, g))
    cw = ops.Fp4Weights((72, 1, 64), ref.NV, 2.0 ** 40, rows=ops.Fp4Rows(wr.codes, wr.scales, 64, ref.NV, 2.0 ** 40))
    m = torch.arange(rows, dtype=torch.int32, device="cuda")[None].contiguous()
    got = ops.fp4_conv(big, m, ops.device_count(rows), cw, out_fmt=ref.NV, out_tensor_scale=2.0 ** -66)
    _check_codes(got, *ref.quantize(y, ref.NV, 2.0 ** -66))


@pytest.mark.parametrize("rows", [1, 2, 4, 8, 9])
def test_scales_that_bring_each_other_back(rows):
    """Blocks near either end of fp32 whose products lie in the middle of it (every sum is exact), on the CUDA cores and the tensor cores."""
    ops = _ops()
    x, w = np.zeros((rows, 96), np.float32), np.zeros((24, 96), np.float32)
    for r in range(rows):
        x[r, 32 * (r % 3):32 * (r % 3) + 32] = 6 * 2.0 ** ((-122, 120, -118)[r % 3])
    w[0, :32], w[1, :32], w[2, :32] = 6 * 2.0 ** 122, 2.0 ** 110, -6 * 2.0 ** 121
    w[3, 32:64], w[4, 32:64], w[5, 32:64] = 6 * 2.0 ** -120, 2.0 ** -123, -3 * 2.0 ** -119
    w[6, 64:], w[7, 64:], w[8, 64:], w[9, 64:] = 6 * 2.0 ** 118, 3 * 2.0 ** 119, -2.0 ** 117, np.nan
    q, xv = _quantized(x, ref.MX, 1.0)
    wv = ref.values(*ref.quantize(w, ref.MX), ref.MX, 96)
    y = ops.fp4_linear(q, ops.device_count(rows), ops.Fp4Weights(w, ref.MX)).cpu().numpy()
    with np.errstate(invalid="ignore"):
        want = (xv @ wv.T).astype(np.float16)
    assert np.isfinite(np.delete(want, 9, 1)).all() and np.abs(want[0, :3]).min() > 0 and np.isnan(want[:, 9]).all()
    assert np.array_equal(y, want, equal_nan=True)


def _random_product(fmt, rows, cin, cout):
    """Rows, weights and their codes of a layer whose sums are exact: scales of 1, a fifth of the codes not zero."""
    ops = _ops()
    gen = torch.Generator(device="cuda").manual_seed(rows + cin + cout)

    def some(n):
        q = ops.Fp4Rows.empty(n, cin, fmt)
        keep = torch.rand(q.codes.shape, generator=gen, device="cuda") < 0.2
        q.codes.copy_(torch.randint(0, 256, q.codes.shape, generator=gen, device="cuda", dtype=torch.uint8) * keep)
        q.codes.view(n, -1, 32)[:, cin // 64:, (cin % 64 + 1) // 2:] = 0
        q.scales.fill_(127 if fmt == ref.MX else 56)
        return q
    return some(rows), some(cout)


def _exact_values(q):
    table = torch.tensor(ref.VALUES, device="cuda")
    return table[torch.stack((q.codes & 15, q.codes >> 4), 2).long()].view(q.rows, -1)[:, :q.channels]


def _time(f, launches=10):
    """Device microseconds of a launch among others, the median of five."""
    took = []
    for _ in range(6):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        torch.cuda._sleep(1_000_000)
        a.record()
        for _ in range(launches):
            f()
        b.record()
        torch.cuda.synchronize()
        took.append(a.elapsed_time(b) / launches * 1e3)
    return sorted(took[1:])[2]


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("rows,cin,cout", [(64, 57600, 256), (64, 57664, 256), (30, 65536, 200), (300, 65536, 512), (9, 65536, 128),
                                           (2, 65536, 100), (8, 32768, 65), (5, 16384, 130), (40, 64, 65536)])
def test_linear_of_the_widest_layers(fmt, rows, cin, cout):
    """Up to the most channels there are, bit for bit: quarters whose sums stay below 2^22."""
    ops = _ops()
    q, w = _random_product(fmt, rows, cin, cout)
    wq = ops.Fp4Weights((cout, cin), fmt, rows=w)
    st = ops.new_status()
    got = ops.fp4_linear(q, ops.device_count(rows), wq, status=st)
    x, y = _exact_values(q), _exact_values(w)
    assert float((x.abs() @ y.abs().T).max()) < 2 ** 22
    assert torch.equal(got, (x @ y.T).to(torch.float16)) and int(st[0]) == 0


@pytest.mark.parametrize("rows,cout", [(64, 256), (300, 512), (1000, 1024)])
def test_a_split_of_k_does_not_end_where_k_gets_longer(rows, cout):
    """57 664 channels are one chunk in 226 more than 57 600, and take as long but for that (twice is a wrong choice of tiles)."""
    ops = _ops()
    took = []
    for cin in (57600, 57664):
        q, w = _random_product(ref.NV, rows, cin, cout)
        wq, n = ops.Fp4Weights((cout, cin), ref.NV, rows=w), ops.device_count(rows)
        out = ops.fp4_linear(q, n, wq)
        took.append(_time(lambda: ops.fp4_linear(q, n, wq, out=out)))
    assert took[1] < 1.5 * took[0], took


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("rows,cin,cout", [(8, 65536, 128), (4, 65536, 64), (8, 32768, 8), (8, 32768, 256)])
def test_fewer_rows_of_a_long_k_take_no_longer(fmt, rows, cin, cout):
    """Few rows never take much longer than nine, which have all SMs split K (half as long again is a wrong choice of kernel)."""
    ops = _ops()
    took = []
    for r in (rows, 9):
        q, w = _random_product(fmt, r, cin, cout)
        wq, n = ops.Fp4Weights((cout, cin), fmt, rows=w), ops.device_count(r)
        out = ops.fp4_linear(q, n, wq)
        took.append(_time(lambda: ops.fp4_linear(q, n, wq, out=out)))
    assert took[0] < 1.5 * took[1], took


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("cin,cout", [(64, 64), (100, 128), (256, 40)])
def test_conv_of_no_rows_gives_the_bias(fmt, cin, cout):
    """An input without rows, whatever the map says: act(bias) and the residual."""
    ops = _ops()
    cap, kvol = 300, 27
    rng = np.random.default_rng(1)
    bias = rng.standard_normal(cout).astype(np.float32)
    wq = ops.Fp4Weights(_features(cout * kvol, cin, 2, 0.3).reshape(cout, kvol, cin), fmt, 1.0, bias)
    empty, n = ops.Fp4Rows.empty(0, cin, fmt), ops.device_count(cap)
    m = rng.integers(-3, 9, (kvol, cap)).astype(np.int32)
    m[0, :3] = 0, 2 ** 31 - 1, -2 ** 31
    want = torch.from_numpy(np.maximum(bias, 0)).cuda().half().expand(cap, cout)
    got = ops.fp4_conv(empty, _dev(m), n, wq, act=ops.ACT_RELU)
    assert torch.equal(got, want)
    res = torch.randn(cap, cout, device="cuda").half()
    got = ops.fp4_conv(empty, _dev(m), n, wq, act=ops.ACT_RELU, res=res, res_relu=True)
    assert torch.equal(got, torch.relu((want.float() + res.float()).half()))
    got = ops.fp4_conv(ops.fp4_quantize(torch.zeros(0, cin, device="cuda"), n, fmt), _dev(m), n, wq, out_fmt=fmt)
    _check_codes(got, *ref.quantize(np.broadcast_to(bias, (cap, cout)), fmt))


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("cin,cout", [(64, 64), (128, 128), (128, 98)])
@pytest.mark.parametrize("launch_rows", [1, 31, 200])
def test_conv_processes_the_count_whatever_rows_the_launch_is_for(fmt, cin, cout, launch_rows):
    """A hint far below the count and the capacity: all rows of the count are written, with and without a residual and in 4 bits."""
    ops = _ops()
    cap, n = 3000, 2790
    q, xv, wq, wv, alpha, bias = _conv_problem(fmt, cap, cin, cout, 9)
    m, n_ptr = _dev(_map(cap, 9, 5)), ops.device_count(n)
    res = torch.randn(cap, cout, device="cuda").half()
    for kw in (dict(), dict(res=res, res_relu=True)):
        out = torch.full((cap, cout), 7.0, dtype=torch.float16, device="cuda")
        ops.fp4_conv(q, m, n_ptr, wq, out=out, launch_rows=launch_rows, **kw)
        assert torch.equal(out[:n], ops.fp4_conv(q, m, n_ptr, wq, **kw)[:n]) and bool((out[n:] == 7).all())
    h = ops.Fp4Rows.empty(cap, cout, fmt)
    h.codes.fill_(0xa5)
    h.scales.fill_(0x5a)
    ops.fp4_conv(q, m, n_ptr, wq, out_fmt=fmt, out=h, launch_rows=launch_rows)
    want = ops.fp4_conv(q, m, n_ptr, wq, out_fmt=fmt)
    assert torch.equal(h.codes[:n], want.codes[:n]) and torch.equal(h.scales[:n], want.scales[:n])
    assert bool((h.codes[n:] == 0xa5).all()) and bool((h.scales[n:] == 0x5a).all())


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("cin,cout", [(64, 64), (128, 128), (256, 72)])
def test_conv_reads_no_row_behind_the_input(fmt, cin, cout):
    """Every kind of entry that is no row of the input, one by one, beside rows of NaN right behind it: reading any of them would show."""
    ops = _ops()
    n_in, n, kvol = 300, 900, 27
    q, xv, wq, wv, alpha, bias = _conv_problem(fmt, n_in, cin, cout, kvol)
    codes = torch.full((2 * n_in, q.codes.shape[1]), 0x77, dtype=torch.uint8, device="cuda")
    scales = torch.full((2 * n_in, q.scales.shape[1]), 0xff if fmt == ref.MX else 0x7f, dtype=torch.uint8, device="cuda")
    codes[:n_in], scales[:n_in] = q.codes, q.scales
    mine = ops.Fp4Rows(codes[:n_in], scales[:n_in], cin, fmt, q.tensor_scale)
    m = _map(n, kvol, 5, n_in=n_in)
    rng = np.random.default_rng(1)
    at = rng.random(m.shape) < 0.2
    m[at] = rng.choice([n_in, n_in + 1, n_in + 2, 2 * n_in - 1, 2 ** 31 - 1, -2, -2 ** 31], at.sum())
    for v in (n_in, n_in + 1, -2):
        assert (m == v).sum() > 100
    m[4, :9] = n_in - 1                       # the last row is one of the input's
    y, off = ref.product(_gather(xv, np.where((m < 0) | (m >= n_in), -1, m)), wv, alpha, bias, False)
    got = ops.fp4_conv(mine, _dev(m), ops.device_count(n), wq).cpu().numpy().astype(np.float64)
    assert (np.abs(got - y) <= off).all()
    # and the guard is one: an input of one row more has it
    m[:] = -1
    m[0, ::2] = n_in
    more = ops.Fp4Rows(codes[:n_in + 1], scales[:n_in + 1], cin, fmt, q.tensor_scale)
    got = torch.isnan(ops.fp4_conv(more, _dev(m), ops.device_count(n), wq)).all(1).cpu().numpy()
    assert got[::2].all() and not got[1::2].any()


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("cin,cout", [(64, 64), (128, 128), (256, 72)])
def test_a_block_of_weights_that_is_not_finite_shows_in_every_row(fmt, cin, cout):
    """Its output channel is NaN, in rows without that neighbour too, and no other channel is."""
    ops = _ops()
    n, kvol = 300, 27
    q, _ = _quantized(_features(n, cin, 1, 0.3), fmt, 1.0)
    w = _features(cout * kvol, cin, 2, 0.3).reshape(cout, kvol, cin)
    w[5, 3, 7], w[cout - 1, 26, cin - 1] = np.nan, np.inf
    m = _map(n, kvol, 3, 0.05)
    assert 0 < (m[3] >= 0).sum() < n
    bad = torch.isnan(ops.fp4_conv(q, _dev(m), ops.device_count(n), ops.Fp4Weights(w, fmt))).cpu().numpy()
    assert bad[:, [5, cout - 1]].all() and bad.sum() == 2 * n
    for rows in (3, 300):                     # the linear layer: on the CUDA cores, and on the tensor cores
        few = ops.Fp4Rows(q.codes[:rows], q.scales[:rows], cin, fmt)
        bad = torch.isnan(ops.fp4_linear(few, ops.device_count(rows), ops.Fp4Weights(w[:, 3].copy(), fmt))).cpu().numpy()
        assert bad[:, 5].all() and bad.sum() == rows


def test_tensor_scales_whose_product_is_beyond_fp32():
    """Refused where results would be wrong: above fp32, where a sum of 0 would be NaN, and below it for 4-bit rows."""
    ops = _ops()
    n, m = ops.device_count(40), torch.zeros((1, 40), dtype=torch.int32, device="cuda")
    codes, scales = ref.quantize(_features(40, 64, 1), ref.NV, 0.01)
    wr = ops.fp4_quantize(_dev(_features(24, 64, 2)), ops.device_count(24), ref.NV, 0.01)
    bias = np.linspace(-1, 1, 24).astype(np.float32)

    def both(gx, gw, **kw):
        q = ops.Fp4Rows(_dev(codes), _dev(scales), 64, ref.NV, gx)
        w = ops.Fp4Weights((24, 64), ref.NV, gw, bias, rows=ops.Fp4Rows(wr.codes, wr.scales, 64, ref.NV, gw))
        return [lambda: ops.fp4_linear(q, n, w, **kw), lambda: ops.fp4_conv(q, m, n, w, **kw)]
    for gx, gw in ((1e30, 1e30), (7.5e35, 1e3)):
        for kw in ({}, dict(out_fmt=ref.MX), dict(out_fmt=ref.NV, out_tensor_scale=1e30)):
            for call in both(gx, gw, **kw):
                with pytest.raises(ValueError, match="beyond fp32"):
                    call()
    for gx, gw in ((1e-30, 1e-30), (1e-20, 1e-19)):
        for call in both(gx, gw, out_fmt=ref.MX):
            with pytest.raises(ValueError, match="beyond fp32"):
                call()
        for call in both(gx, gw):             # in fp16 the sums are 0 beside the bias
            assert torch.equal(call(), _dev(bias).half().expand(40, 24))


def test_a_status_block_is_four_words():
    """A smaller one, or one of another type, would be written past its end when a wait runs out."""
    ops = _ops()
    q, _ = _quantized(_features(8, 64, 1), ref.NV, 0.01)
    n, m = ops.device_count(8), torch.zeros((1, 8), dtype=torch.int32, device="cuda")
    w = ops.Fp4Weights(_features(24, 64, 2), ref.NV, 0.01)
    for bad in (torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.uint8, device="cuda"),
                torch.zeros(8, dtype=torch.int32, device="cuda")[::2], torch.zeros(4, device="cuda")):
        for call in (lambda: ops.fp4_linear(q, n, w, status=bad), lambda: ops.fp4_conv(q, m, n, w, status=bad)):
            with pytest.raises(ValueError, match="status block"):
                call()
    for good in (ops.new_status(), torch.zeros(9, dtype=torch.int32, device="cuda")[3:]):
        ops.fp4_linear(q, n, w, status=good)
        ops.fp4_conv(q, m, n, w, status=good)
        assert not bool(good.any())


@pytest.mark.parametrize("fmt", FORMATS, ids=IDS)
@pytest.mark.parametrize("kind", ["f16", "f32", "i8"])
@pytest.mark.parametrize("channels", [65536, 65535, 65432, 65473])
def test_rows_of_the_most_channels(fmt, kind, channels):
    """Rows of 128 KB of fp16: flat, aligned and staged ways, there and back, and rows behind the count."""
    ops = _ops()
    rows, n = 7, 5
    x = _features(rows, channels, channels)
    in_scale = 1.0
    if kind == "i8":
        in_scale = float(np.float32(np.abs(x).max() / 127))
        xi = np.clip(np.rint(x / np.float32(in_scale)), -128, 127).astype(np.int8)
        dev, x = _dev(xi), xi.astype(np.float32) * np.float32(in_scale)
    else:
        dev = _dev(x.astype(np.float16 if kind == "f16" else np.float32))
        x = dev.cpu().numpy().astype(np.float32)
    g = _scale(x, fmt)
    codes, scales = ref.quantize(x, fmt, g)
    out = ops.Fp4Rows.empty(rows, channels, fmt, g)
    out.codes.fill_(0xa5)
    out.scales.fill_(0x5a)
    count = ops.device_count(n)
    ops.fp4_quantize(dev, count, fmt, g, in_scale=in_scale, out=out)
    assert np.array_equal(out.scales[:n].cpu().numpy(), scales[:n])
    assert np.array_equal(ref.magnitude_codes(out.codes[:n].cpu().numpy()), ref.magnitude_codes(codes[:n]))
    assert bool((out.codes[n:] == 0xa5).all()) and bool((out.scales[n:] == 0x5a).all())
    for out_kind, dt in ((ops.F16, np.float16), (ops.F32, np.float32)):
        want = ref.values(codes, scales, fmt, channels, g).astype(np.float32).astype(dt)
        y = torch.full((rows, channels), 7.0, dtype=torch.float16 if out_kind == ops.F16 else torch.float32, device="cuda")
        ops.fp4_dequantize(out, count, out_kind, out=y)
        assert np.array_equal(y[:n].cpu().numpy(), want[:n]) and bool((y[n:] == 7).all())
