"""Performance cases of the 4-bit floating-point operators, as plain data and functions.

* ``roundtrip`` rows to 4-bit codes with block scales and back to fp16: how features enter 4 bits, and how
                one looks at what that costs in accuracy.
* ``expand``    4-bit rows to fp16 rows: a layer that stays in fp16 reads rows that are kept in 4 bits.
* ``linear``    4-bit rows times 4-bit weights, bias and ReLU: one row (a single token or a pooled
                feature), BEV cells, many rows with wide layers.
* ``conv``      a sparse convolution, 3x3x3 submanifold, over a neighbour map.
* ``block``     two of them in a row as in a residual block: the first leaves 4-bit rows behind.

Formats: ``mx`` blocks of 32 channels with power-of-two scales, ``nv`` blocks of 16 with e4m3 scales and one
fp32 scale a tensor.  Rows are stored as codes [rows][cpad / 2] (even channel in the low nibble, cpad the
channels rounded up to 64) and scales [rows][pitch], a multiple of 4 bytes.

With ``own`` false ``run`` computes everything from elementary torch operations in fp32.
"""
import functools
import math

import numpy as np
import torch

own = False

GRID = (41, 1440, 1440)                       # the backbone's grid, z, y, x
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"f16": torch.float16, "f32": torch.float32}
DEV = "cuda"


# ------------------------------------------------------------------------------- the cases
def _rows(what, fmt, rows, channels, kind="f16", **name):
    return dict(name, what=what, fmt=fmt, rows=rows, channels=channels, kind=kind)


def _linear(fmt, rows, cin, cout, relu, **name):
    return dict(name, what="linear", fmt=fmt, rows=rows, cin=cin, cout=cout, relu=relu)


def _conv(what, fmt, voxels, cin, cout, residual, **name):
    return dict(name, what=what, fmt=fmt, voxels=voxels, cin=cin, cout=cout, residual=residual)


def listed():
    return [
        # one feature vector: launches and latency
        _rows("roundtrip", "nv", 1, 256, name="roundtrip_nv_1x256"),
        # a benchmark frame's widest rows, as the fp16 layer before leaves them
        _rows("roundtrip", "mx", 120000, 128, name="roundtrip_mx_120kx128"),
        # a batch of eight frames, kept in int8 so far
        _rows("roundtrip", "nv", 960000, 64, "i8", name="roundtrip_nv_i8_960kx64"),
        # rows that are kept in 4 bits, read by an fp16 layer; odd sizes
        _rows("expand", "nv", 200000, 128, name="expand_nv_200kx128"),
        _rows("expand", "mx", 50001, 72, name="expand_mx_50001x72"),
        # a single row through a wide layer: the weights' bytes
        _linear("nv", 1, 4096, 4096, False, name="linear_nv_1x4096x4096"),
        # the cells of a 180 x 180 BEV map of 256 channels
        _linear("nv", 32400, 256, 512, True, name="linear_nv_32400x256x512"),
        # odd sizes
        _linear("mx", 1001, 200, 136, True, name="linear_mx_1001x200x136"),
        # many rows, wide layers: arithmetic
        _linear("mx", 8192, 4096, 4096, False, name="linear_mx_8192x4096x4096"),
        # a small frame
        _conv("conv", "mx", 14000, 64, 64, False, name="conv_mx_14k_c64"),
        # a benchmark frame in the widest layers of the backbone
        _conv("conv", "nv", 120000, 128, 128, True, name="conv_nv_120k_c128"),
        # a residual block of the middle layers
        _conv("block", "nv", 60000, 64, 64, True, name="block_nv_60k_c64"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    what = rng.choice(["roundtrip", "expand", "linear", "linear", "conv", "conv", "block"])
    fmt = rng.choice(["mx", "nv"])
    if what in ("roundtrip", "expand"):
        channels = rng.choice([16, 32, 48, 64, 72, 100, 128, 256, 512, _log_int(rng, 16, 1024)])
        rows = min(_log_int(rng, 1, 960000), 61440000 // channels)
        return _rows(what, fmt, rows, channels,
                     rng.choice(["f16", "f16", "f32", "i8"]) if what == "roundtrip" else "f16")
    if what == "linear":
        cin, cout = (rng.choice([64, 128, 256, 512, 1024, 2048, 4096, _log_int(rng, 20, 4096)])
                     for _ in range(2))
        rows = min(_log_int(rng, 1, 260000), 8192 * 4096 * 4096 // (cin * cout))
        return _linear(fmt, rows, cin, cout, rng.random() < 0.5)
    if what == "conv":
        return _conv(what, fmt, _log_int(rng, 1000, 200000), rng.choice([48, 64, 100, 128]),
                     rng.choice([24, 32, 64, 96, 128]), rng.random() < 0.5)
    c = rng.choice([64, 128])
    return _conv(what, fmt, _log_int(rng, 1000, 100000), c, c, True)


# ---------------------------------------------------------------------------- the plain form
def _block(fmt):
    return 32 if fmt == "mx" else 16


def _cpad(channels):
    return -(-channels // 64) * 64


def _pitch(fmt, channels):
    cpad = _cpad(channels)
    return 4 * -(-cpad // 128) if fmt == "mx" else cpad // 16


def _quantize(x, fmt, g):
    """fp32 [rows, channels] -> (code indices with sign as values [rows, cpad], block scales [rows, blocks] without g)."""
    rows, channels = x.shape
    b, cpad = _block(fmt), _cpad(channels)
    xb = torch.nn.functional.pad(x, (0, cpad - channels)).reshape(rows, cpad // b, b)
    amax = xb.abs().amax(2)
    bad = ~torch.isfinite(amax)
    if fmt == "mx":
        e = torch.frexp(amax)[1].float() - 3.0            # floor(log2 amax) - 2
        s = torch.where(amax > 0, torch.exp2(e.clamp(-126, 127)), torch.full_like(amax, 2.0 ** -126))
        whole = s
    else:
        s = (amax / (6.0 * torch.full_like(amax, g))).clamp(max=448.0).to(torch.float8_e4m3fn).float()
        whole = s * g
    q = xb / whole[..., None]
    q = torch.where((whole > 0)[..., None], q, torch.zeros_like(q))
    a = q.abs()
    i = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
         + (a >= 3.5).int() + (a > 5.0).int())
    v = torch.tensor(MAGNITUDES, device=x.device)[i.long()]
    v = torch.where(q < 0, -v, v)
    v = torch.where(bad[..., None], torch.zeros_like(v), v)
    s = torch.where(bad, torch.full_like(s, float("nan")), s)
    return v.reshape(rows, cpad), s


def _values(v, s, fmt, g, channels):
    """What codes and scales stand for, fp32 [rows, channels]."""
    whole = s if fmt == "mx" else s * g
    rows = v.shape[0]
    return (v.reshape(rows, s.shape[1], -1) * whole[..., None]).reshape(rows, -1)[:, :channels]


def _pack(v, s, fmt):
    """Code values and scales -> the stored bytes."""
    i = torch.bucketize(v.abs(), torch.tensor(MAGNITUDES, device=v.device)).to(torch.uint8)
    i = i | (torch.signbit(v).to(torch.uint8) << 3)
    codes = i[:, 0::2] | (i[:, 1::2] << 4)
    if fmt == "mx":
        sb = (torch.frexp(s)[1] + 126).to(torch.uint8)
        pitch = _pitch(fmt, v.shape[1])
        sb = torch.nn.functional.pad(sb, (0, pitch - sb.shape[1]))
    else:
        sb = s.to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.contiguous(), sb.contiguous()


def _unpack(codes, scales, fmt, g, channels):
    """The stored bytes -> fp32 values [rows, channels], with g left to the caller when g is None."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    v = table[torch.stack((codes & 15, codes >> 4), 2).long()].reshape(codes.shape[0], -1)
    blocks = v.shape[1] // _block(fmt)
    s = scales[:, :blocks]
    s = torch.exp2(s.float() - 127.0) if fmt == "mx" else s.view(torch.float8_e4m3fn).float()
    return _values(v, s, fmt, 1.0 if g is None else g, channels)


def _plain_linear(x, w, alpha, bias, relu):
    y = (x @ w.t()) * alpha + bias
    return torch.relu(y) if relu else y


def _plain_conv(x, m, w, alpha, bias):
    xp = torch.cat((x, torch.zeros_like(x[:1])))          # index -1: the row of zeros
    return (xp[m.t().long()].reshape(m.shape[1], -1) @ w.t()) * alpha + bias


# ----------------------------------------------------------------------------- the inputs
def _features(rows, channels, gen):
    """Activations after a normalised layer: normal, a spread of row and channel magnitudes, a third of them cut to zero."""
    x = torch.randn(rows, channels, generator=gen, device=DEV)
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device=DEV))
    x *= torch.exp(0.5 * torch.randn(1, channels, generator=gen, device=DEV))
    return torch.where(x < -0.43, torch.zeros_like(x), x)


@functools.lru_cache(maxsize=4)
def _keys(n, seed):
    """n voxels of the benchmark law: 70 % on a ground band, density 1/r, 30 % in 8 x 4 x 4 boxes; sorted cells."""
    gz, gy, gx = GRID
    rng = np.random.default_rng(seed)
    boxes = max(1, round(50 * n / 20000))
    o = [rng.integers(0, g - b + 1, boxes) for g, b in zip(GRID, (4, 4, 8))]
    m = 4 * n
    b = rng.integers(0, boxes, m)
    z, y, x = (o[i][b] + rng.integers(0, s, m) for i, s in enumerate((4, 4, 8)))
    inside = np.unique((z * gy + y) * gx + x)
    inside = rng.permutation(inside)[: int(0.3 * n)]
    r, t = rng.random(m) * gy / 2, rng.random(m) * 2 * np.pi
    y = np.clip((gy / 2 + r * np.sin(t)).astype(np.int64), 0, gy - 1)
    x = np.clip((gx / 2 + r * np.cos(t)).astype(np.int64), 0, gx - 1)
    band = np.setdiff1d((rng.integers(2, 7, m) * gy + y) * gx + x, inside)
    return np.concatenate((inside, rng.permutation(band)[: n - len(inside)]))


def _map(keys):
    """The 3x3x3 submanifold neighbour map of the cells `keys` (int64 [n], any order): int32 [27, n]."""
    gz, gy, gx = GRID
    order = torch.argsort(keys)
    ranked = keys[order]
    x, y, z = keys % gx, keys // gx % gy, keys // (gx * gy)
    d = torch.arange(27, device=keys.device)
    nz, ny, nx = (v[None] + o[:, None] - 1 for v, o in ((z, d // 9), (y, d // 3 % 3), (x, d % 3)))
    fits = (nz >= 0) & (nz < gz) & (ny >= 0) & (ny < gy) & (nx >= 0) & (nx < gx)
    want = (nz * gy + ny) * gx + nx
    at = torch.searchsorted(ranked, want).clamp(max=len(keys) - 1)
    found = fits & (ranked[at] == want)
    return torch.where(found, order[at], -1).to(torch.int32).contiguous()


@functools.lru_cache(maxsize=64)
def _pairs(n):
    """Neighbour pairs of n voxels."""
    keys = np.sort(_keys(n, 0))
    gz, gy, gx = GRID
    pairs = 0
    for dz in (-1, 0, 1):
        for dy in (-1, 0, 1):
            for dx in (-1, 0, 1):
                want = keys + (dz * gy + dy) * gx + dx
                at = np.minimum(np.searchsorted(keys, want), len(keys) - 1)
                pairs += int((keys[at] == want).sum())
    return pairs


def _tensor_scale(top, fmt):
    """The tensor scale that a program keeps for values up to `top`: 8 significant bits, so that a value lies
    on the border between two codes or well off it."""
    return 1.0 if fmt == "mx" else float(torch.tensor(top / (6 * 448)).bfloat16())


def _weights(cout, taps, cin, fmt, gen):
    """Kaiming weights in fp16, their tensor scale, and their 4-bit values without it, fp32 [cout, taps * cin]."""
    w = torch.randn(cout, taps, cin, generator=gen, device=DEV) * math.sqrt(2.0 / (taps * cin))
    w = w.half()
    g = _tensor_scale(float(w.abs().max()), fmt)
    v, s = _quantize(w.float().reshape(cout * taps, cin), fmt, g)
    return w, g, _values(v, s, fmt, 1.0, cin).reshape(cout, taps * cin)




def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    what, fmt = case["what"], case["fmt"]
    s = dict(case)
    if what in ("roundtrip", "expand"):
        x = _features(case["rows"], case["channels"], gen)
        s["in_scale"] = 1.0
        if case["kind"] == "i8":
            s["in_scale"] = float(np.float32(float(x.abs().max()) / 127))
            x = torch.round(x / s["in_scale"]).clamp(-128, 127).to(torch.int8)
            s["g"] = _tensor_scale(127 * s["in_scale"], fmt)
        else:
            x = x.to(DTYPES[case["kind"]])
            s["g"] = _tensor_scale(float(x.abs().max()), fmt)
        s["n_ptr"] = torch.tensor([case["rows"]], dtype=torch.int32, device=DEV)
        if what == "roundtrip":
            s["x"] = x
        else:
            s["codes"], s["scales"] = _pack(*_quantize(x.float(), fmt, s["g"]), fmt)
    else:
        if what == "linear":
            rows, taps = case["rows"], 1
        else:
            rows, taps = case["voxels"], 27
            s["map"] = _map(torch.from_numpy(_keys(rows, seed)).to(DEV))
        cin, cout = case["cin"], case["cout"]
        x = _features(rows, cin, gen)
        s["g"] = _tensor_scale(float(x.abs().max()), fmt)
        s["codes"], s["scales"] = _pack(*_quantize(x, fmt, s["g"]), fmt)
        s["w"], s["gw"], s["wv"] = _weights(cout, taps, cin, fmt, gen)
        s["bias"] = 0.1 * torch.randn(cout, generator=gen, device=DEV)
        s["n_ptr"] = torch.tensor([rows], dtype=torch.int32, device=DEV)
        if case.get("residual"):
            s["res"] = _features(rows, cout, gen).half()
        if what == "block":
            s["g1"] = _tensor_scale(16.0, fmt)
            s["w2"], s["gw2"], s["wv2"] = _weights(cout, taps, cout, fmt, gen)
            s["bias2"] = 0.1 * torch.randn(cout, generator=gen, device=DEV)
    if own:
        from lidar_ai_solution_b200 import ops
        f = ops.MXFP4 if fmt == "mx" else ops.NVFP4
        s["f"] = f
        if "codes" in s:
            s["q"] = ops.Fp4Rows(s["codes"], s["scales"], case.get("channels", case.get("cin")), f, s["g"])
        if "w" in s:
            s["wq"] = ops.Fp4Weights(s["w"], f, s["gw"], s["bias"])
        if what == "block":
            s["wq2"] = ops.Fp4Weights(s["w2"], f, s["gw2"], s["bias2"])
    return s


# --------------------------------------------------------------------------------- a pass
def _run_own(s):
    from lidar_ai_solution_b200 import ops
    what = s["what"]
    if what == "roundtrip":
        q = ops.fp4_quantize(s["x"], s["n_ptr"], s["f"], s["g"], in_scale=s["in_scale"])
        return ops.fp4_dequantize(q, s["n_ptr"])
    if what == "expand":
        return ops.fp4_dequantize(s["q"], s["n_ptr"])
    if what == "linear":
        return ops.fp4_linear(s["q"], s["n_ptr"], s["wq"], act=ops.ACT_RELU if s["relu"] else ops.ACT_NONE)
    if what == "conv":
        return ops.fp4_conv(s["q"], s["map"], s["n_ptr"], s["wq"], act=ops.ACT_RELU, res=s.get("res"))
    h = ops.fp4_conv(s["q"], s["map"], s["n_ptr"], s["wq"], act=ops.ACT_RELU, out_fmt=s["f"],
                     out_tensor_scale=s["g1"])
    return ops.fp4_conv(h, s["map"], s["n_ptr"], s["wq2"], res=s["res"], res_relu=True)


def run(state):
    s = state
    if own:
        return _run_own(s)
    what, fmt = s["what"], s["fmt"]
    if what == "roundtrip":
        x = s["x"].float()
        x = x * s["in_scale"] if s["kind"] == "i8" else x
        return _values(*_quantize(x, fmt, s["g"]), fmt, s["g"], s["channels"]).half()
    if what == "expand":
        return _unpack(s["codes"], s["scales"], fmt, s["g"], s["channels"]).half()
    x = _unpack(s["codes"], s["scales"], fmt, None, s["cin"])
    alpha = s["g"] * s["gw"]
    if what == "linear":
        return _plain_linear(x, s["wv"], alpha, s["bias"], s["relu"]).half()
    y = torch.relu(_plain_conv(x, s["map"], s["wv"], alpha, s["bias"]))
    if what == "conv":
        return (y.half().float() + s["res"].float() if s["residual"] else y).half()
    h = _values(*_quantize(y, fmt, s["g1"]), fmt, 1.0, s["cout"])
    y = _plain_conv(h, s["map"], s["wv2"], s["g1"] * s["gw2"], s["bias2"])
    return torch.relu(y.half().float() + s["res"].float()).half()


def work(case):
    fmt = case["fmt"]
    stored = lambda c: _cpad(c) // 2 + _pitch(fmt, c)  # noqa: E731  bytes of a row
    if case["what"] in ("roundtrip", "expand"):
        rows, c = case["rows"], case["channels"]
        size = {"f16": 2, "f32": 4, "i8": 1}[case["kind"]]
        into = rows * c * size if case["what"] == "roundtrip" else 0
        return {"bytes": into + rows * stored(c) + 2 * rows * c, "flops": 0}
    cin, cout = case["cin"], case["cout"]
    if case["what"] == "linear":
        rows = case["rows"]
        return {"bytes": (rows + cout) * stored(cin) + 4 * cout + 2 * rows * cout,
                "flops": 2 * rows * cin * cout}
    n, convs = case["voxels"], 2 if case["what"] == "block" else 1
    b = n * stored(cin) + convs * (27 * 4 * n + cout * 27 * stored(cin) + 4 * cout)
    b += 2 * n * cout * (2 if case["residual"] else 1) + (2 * n * stored(cout) if convs == 2 else 0)
    return {"bytes": b, "flops": convs * 2 * _pairs(n) * cin * cout}


# ------------------------------------------------------------------------- in 64 bits, apart
def _exact_values(x, fmt, g):
    """float64 [rows, channels] -> the values its codes and scales stand for."""
    b = 32 if fmt == "mx" else 16
    rows, channels = x.shape
    out = torch.zeros(rows, -(-channels // b) * b, dtype=torch.float64, device=x.device)
    out[:, :channels] = x
    blocks = out.reshape(-1, b)
    top = blocks.abs().max(1).values
    if fmt == "mx":
        scale = torch.ldexp(torch.ones_like(top), (torch.frexp(top)[1] - 3).clamp(-127, 127))
    else:
        t = top / (6 * g)
        step = torch.ldexp(torch.ones_like(t), (torch.frexp(t)[1] - 1).clamp(-6, 8) - 3)
        scale = (torch.round(t / step) * step).clamp(max=448) * g
    ratio = blocks / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]
    m = ratio.abs().clamp(max=6)
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0)).double()
    near = (torch.round(m / step) * step).clamp(max=6)     # half to even: codes alternate with the step's multiples
    return (torch.sign(ratio) * near * scale[:, None]).reshape(rows, -1)[:, :channels]


def _exact_read(s, cin, g):
    """float64 values of stored rows, byte by byte."""
    codes, scales, fmt = s["codes"], s["scales"], s["fmt"]
    nib = torch.stack([codes % 16, codes // 16], -1).reshape(len(codes), -1)[:, :cin].double()
    i = nib % 8
    mag = torch.where(i < 2, i / 2, torch.ldexp(1 + (i % 2) / 2, torch.div(i, 2, rounding_mode="floor") - 1))
    val = torch.where(nib >= 8, -mag, mag)
    by = torch.arange(cin, device=codes.device) // (32 if fmt == "mx" else 16)
    raw = scales[:, by].double()
    if fmt == "mx":
        return val * torch.ldexp(torch.ones_like(raw), raw - 127)
    e, f = torch.div(raw, 8, rounding_mode="floor"), raw % 8
    return val * torch.where(e > 0, torch.ldexp(1 + f / 8, e - 7), torch.ldexp(f / 8, torch.full_like(e, -6))) * g


def _exact_conv(x, m, w, bias):
    taps, cin = m.shape[0], x.shape[1]
    y = bias.double().repeat(m.shape[1], 1)
    for k in range(taps):
        to = (m[k] >= 0).nonzero()[:, 0]
        y[to] += x[m[k][to].long()] @ w[:, k * cin:(k + 1) * cin].t()
    return y


def exact(case, seed):
    s = prepare(case, seed)
    what, fmt = case["what"], case["fmt"]
    if what == "roundtrip":
        return _exact_values(s["x"].double() * (s["in_scale"] if case["kind"] == "i8" else 1.0), fmt, s["g"])
    if what == "expand":
        return _exact_read(s, case["channels"], s["g"])
    x = _exact_read(s, case["cin"], s["g"])

    def weights(w, g):
        return _exact_values(w.double().reshape(-1, w.shape[2]), fmt, g).reshape(w.shape[0], -1)

    w = weights(s["w"], s["gw"])
    if what == "linear":
        y = x @ w.t() + s["bias"].double()
        return y.clamp(min=0) if case["relu"] else y
    y = _exact_conv(x, s["map"], w, s["bias"]).clamp(min=0)
    if what == "conv":
        return y + s["res"].double() if case["residual"] else y
    y = _exact_conv(_exact_values(y, fmt, s["g1"]), s["map"], weights(s["w2"], s["gw2"]), s["bias2"])
    return (y + s["res"].double()).clamp(min=0)
