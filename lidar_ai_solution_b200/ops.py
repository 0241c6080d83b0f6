"""Thin torch-tensor wrappers over the kernel-level C ABI.

torch is used only to own device memory and streams; every function here ends
in exactly one ``spconvb_*`` call on the current CUDA stream.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

from . import cabi
from .cabi import ACT_NONE, ACT_RELU, F16, F32, I8, MXFP4, NVFP4  # noqa: F401


# torch's own way to the current stream's handle, a microsecond cheaper a call; not a public one
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _stream():
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device())


def _ptr(t):
    return t.data_ptr() if t is not None else None


def kind_of(t: torch.Tensor) -> int:
    return I8 if t.dtype == torch.int8 else F16


def new_status(device="cuda"):
    return torch.zeros(4, dtype=torch.int32, device=device)


def device_count(n: int, device="cuda") -> torch.Tensor:
    """A row count in device memory (what kernels read instead of a host value)."""
    return torch.tensor([n], dtype=torch.int32, device=device)


def hash_build(coords, n_ptr, grid, batch=1, status=None, launch_rows=0):
    cap = coords.shape[0]
    slots = cabi.lib().spconvb_hash_slots_fast(cap)
    table = torch.empty(slots, dtype=torch.int64, device=coords.device)
    cabi.check(cabi.lib().spconvb_hash_build(_ptr(coords), _ptr(n_ptr), cap, launch_rows,
                                             cabi.i3(grid), batch, _ptr(table), slots, 0,
                                             _ptr(status), _stream()), "hash_build")
    return table


def subm_map(coords, n_ptr, grid, table, ksize=(3, 3, 3), dilation=(1, 1, 1), batch=1,
             status=None, launch_rows=0):
    cap = coords.shape[0]
    kvol = math.prod(ksize)
    m = torch.empty((kvol, cap), dtype=torch.int32, device=coords.device)
    cabi.check(cabi.lib().spconvb_subm_map(_ptr(coords), _ptr(n_ptr), cap, launch_rows,
                                           cabi.i3(grid), batch, cabi.i3(ksize),
                                           cabi.i3(dilation), _ptr(table), table.numel(), _ptr(m),
                                           _ptr(status), _stream()), "subm_map")
    return m


def out_grid(grid, ksize, stride, pad, dilation=(1, 1, 1)):
    return [int(cabi.lib().spconvb_out_extent(int(g), int(k), int(s), int(p), int(d)))
            for g, k, s, p, d in zip(grid, ksize, stride, pad, dilation)]


def down_map(coords, n_ptr, grid, table, ksize, stride, pad, dilation=(1, 1, 1), cap_out=None,
             batch=1, status=None, want_table=True, launch_rows=0, return_ws=False, in_ws=None):
    """Returns (out_coords, n_out_ptr, map, out_table, out_grid) and, with ``return_ws``,
    the workspace (bitmap + rank prefix of the outputs) as a sixth item.  ``table`` is not
    needed any more and may be None.  ``in_ws``: the workspace of the down_map call that made
    ``coords``; the map is then looked up by rank from the output side
    (spconvb_down_map_ranked), with the same result."""
    dev = coords.device
    cap_in = coords.shape[0]
    og = out_grid(grid, ksize, stride, pad, dilation)
    if cap_out is None:
        cap_out = max(1, min(cap_in * math.prod(ksize), batch * math.prod(og)))
    kvol = math.prod(ksize)
    ws = torch.empty(cabi.lib().spconvb_down_workspace_bytes(cabi.i3(og), batch),
                     dtype=torch.uint8, device=dev)
    oc = torch.zeros((cap_out, 4), dtype=torch.int32, device=dev)
    n_out = torch.zeros(1, dtype=torch.int32, device=dev)
    m = torch.full((kvol, cap_out), -1, dtype=torch.int32, device=dev)
    slots = cabi.lib().spconvb_hash_slots(cap_out) if want_table else 0
    otab = torch.empty(slots, dtype=torch.int64, device=dev) if want_table else None
    if in_ws is not None:
        cabi.check(cabi.lib().spconvb_down_map_ranked(
            _ptr(coords), _ptr(n_ptr), cap_in, launch_rows, cabi.i3(grid), batch, cabi.i3(ksize),
            cabi.i3(stride), cabi.i3(pad), cabi.i3(dilation), _ptr(in_ws), _ptr(ws),
            _ptr(oc), _ptr(n_out), cap_out, _ptr(m), _ptr(otab), slots, 0, _ptr(status),
            _stream()), "down_map_ranked")
    else:
        cabi.check(cabi.lib().spconvb_down_map(
            _ptr(coords), _ptr(n_ptr), cap_in, launch_rows, cabi.i3(grid), batch, cabi.i3(ksize),
            cabi.i3(stride), cabi.i3(pad), cabi.i3(dilation), _ptr(table),
            table.numel() if table is not None else 0, _ptr(ws),
            _ptr(oc), _ptr(n_out), cap_out, _ptr(m), _ptr(otab), slots, 0, _ptr(status),
            _stream()), "down_map")
    if return_ws:
        return oc, n_out, m, otab, og, ws
    return oc, n_out, m, otab, og


def subm_map_ranked(coords, n_ptr, grid, ws, ksize=(3, 3, 3), dilation=(1, 1, 1), batch=1,
                    status=None, launch_rows=0):
    """SubM map of rows that came out of ``down_map`` (ranked in its workspace ``ws``)."""
    cap = coords.shape[0]
    kvol = math.prod(ksize)
    m = torch.empty((kvol, cap), dtype=torch.int32, device=coords.device)
    cabi.check(cabi.lib().spconvb_subm_map_ranked(_ptr(coords), _ptr(n_ptr), cap, launch_rows,
                                                  cabi.i3(grid), batch, cabi.i3(ksize),
                                                  cabi.i3(dilation), _ptr(ws), _ptr(m),
                                                  _ptr(status), _stream()), "subm_map_ranked")
    return m


def inverse_map(coords, n_ptr, grid, ws, cap_coarse, ksize, stride, pad, dilation=(1, 1, 1),
                batch=1, status=None, launch_rows=0):
    """Map of the inverse conv of a strided rulebook: ``coords`` are the rows that went INTO
    ``down_map`` (with ``return_ws=True``), ``ws`` its workspace, ``cap_coarse`` its cap_out."""
    cap = coords.shape[0]
    kvol = math.prod(ksize)
    m = torch.empty((kvol, cap), dtype=torch.int32, device=coords.device)
    cabi.check(cabi.lib().spconvb_inverse_map(_ptr(coords), _ptr(n_ptr), cap, launch_rows,
                                              cabi.i3(grid), batch, cabi.i3(ksize), cabi.i3(stride),
                                              cabi.i3(pad), cabi.i3(dilation), _ptr(ws), cap_coarse,
                                              _ptr(m), _ptr(status), _stream()), "inverse_map")
    return m


class ConvWeights:
    """Device copies of one layer's parameters in both kernel formats."""

    def __init__(self, w, compute, scale=None, bias=None, device="cuda"):
        # w: numpy [cout, kvol, cin] int8 (compute I8) or float16 (compute F16)
        w = np.ascontiguousarray(w)
        self.compute = compute
        self.cout, self.kvol, self.cin = w.shape
        assert w.dtype == (np.int8 if compute == I8 else np.float16)
        self.plain = torch.from_numpy(w.copy()).to(device)
        self.packed = None
        lib = cabi.lib()
        if lib.spconvb_conv_supported(compute, self.cin, self.cout):
            nbytes = lib.spconvb_conv_packed_bytes(compute, self.cin, self.cout, self.kvol)
            host = np.zeros(nbytes, np.uint8)
            cabi.check(lib.spconvb_conv_pack_weights(compute, self.cin, self.cout, self.kvol,
                                                     w.ctypes.data_as(C.c_void_p),
                                                     host.ctypes.data_as(C.c_void_p)), "pack")
            self.packed = torch.from_numpy(host).to(device)
        self.scale = None if scale is None else torch.from_numpy(
            np.ascontiguousarray(scale, np.float32)).to(device)
        self.bias = None if bias is None else torch.from_numpy(
            np.ascontiguousarray(bias, np.float32)).to(device)


def conv_forward(x, m, n_out_ptr, wts: ConvWeights, act=ACT_NONE, out_kind=F16,
                 inv_out_scale=1.0, res=None, res_scale=1.0, mid_kind=F16, mid_inv_scale=1.0,
                 mid_scale=1.0, res_relu=False, force_simt=False, status=None, launch_rows=0,
                 out=None, wait_test=0, n_in_ptr=None):
    """``n_in_ptr`` (device row count of ``x``) is a hint; results do not depend on it."""
    cap = m.shape[1]
    p = cabi.ConvParams(
        wts.compute, wts.cin, wts.cout, wts.kvol, act, out_kind, inv_out_scale, _ptr(res),
        kind_of(res) if res is not None else F16, res_scale, mid_kind, mid_inv_scale, mid_scale,
        int(res_relu), int(force_simt), int(wait_test))
    if n_in_ptr is not None:
        p.n_in_ptr, p.cap_in = n_in_ptr.data_ptr(), x.shape[0]
    if out is None:
        out = torch.empty((cap, wts.cout), dtype=torch.int8 if out_kind == I8 else torch.float16,
                          device=x.device)
    cabi.check(cabi.lib().spconvb_conv_forward(
        C.byref(p), _ptr(x), _ptr(m), cap, _ptr(n_out_ptr), launch_rows, _ptr(wts.plain),
        _ptr(wts.packed), _ptr(wts.scale), _ptr(wts.bias), _ptr(out), _ptr(status), _stream()),
        "conv_forward")
    return out


def add(a, a_scale, b, b_scale, n_ptr, relu, out_kind, inv_out_scale=1.0):
    rows, ch = a.shape
    out = torch.empty((rows, ch), dtype=torch.int8 if out_kind == I8 else torch.float16,
                      device=a.device)
    cabi.check(cabi.lib().spconvb_add(_ptr(a), kind_of(a), a_scale, _ptr(b), kind_of(b), b_scale,
                                      ch, _ptr(n_ptr), rows, int(relu), out_kind, inv_out_scale,
                                      _ptr(out), _stream()), "add")
    return out


def relu(x, n_ptr):
    out = torch.empty_like(x)
    cabi.check(cabi.lib().spconvb_relu(_ptr(x), kind_of(x), x.shape[1], _ptr(n_ptr), x.shape[0],
                                       _ptr(out), _stream()), "relu")
    return out


def convert(x, out_kind, cout_pad, scale_or_inv, n_ptr):
    rows, cin = x.shape
    out = torch.empty((rows, cout_pad), dtype=torch.int8 if out_kind == I8 else torch.float16,
                      device=x.device)
    cabi.check(cabi.lib().spconvb_convert(_ptr(x), kind_of(x), cin, out_kind, cout_pad,
                                          scale_or_inv, _ptr(n_ptr), rows, _ptr(out), _stream()),
               "convert")
    return out


def scatter_dense(feat, coords, n_ptr, grid, batch=1, in_scale=1.0, perm=None):
    ch = feat.shape[1]
    g = [grid[p] for p in perm] if perm is not None else list(grid)
    out = torch.empty((batch, ch, g[0], g[1], g[2]), dtype=torch.float16, device=feat.device)
    cabi.check(cabi.lib().spconvb_scatter_dense(
        _ptr(feat), kind_of(feat), in_scale, _ptr(coords), _ptr(n_ptr), feat.shape[0], ch, batch,
        cabi.i3(grid), cabi.i3(perm) if perm is not None else None, _ptr(out), _stream()),
        "scatter_dense")
    return out


LAYOUTS = {"NCHW": 1, "NCHW32": 2, "NHWzC": 3}


def scatter_dense_layout(feat, coords, n_ptr, grid, layout="NCHW", dynamic_range=0.0, batch=1,
                         in_scale=1.0, perm=None):
    """ScatterDense into ``layout``; int8 with scale ``dynamic_range / 127`` when the range is
    positive, else fp16.  Returns the tensor with the dimensions as they lie in memory."""
    ch = feat.shape[1]
    g = [grid[p] for p in perm] if perm is not None else list(grid)
    lay = LAYOUTS[layout]
    i8 = dynamic_range > 0
    if lay == 2:
        shape = (batch, (ch * g[0] + 31) // 32, g[1], g[2], 32)
    elif lay == 3:
        shape = (batch, g[1], g[2], g[0], ch)
    else:
        shape = (batch, ch, g[0], g[1], g[2])
    out = torch.empty(shape, dtype=torch.int8 if i8 else torch.float16, device=feat.device)
    lib = cabi.lib()
    pp = cabi.i3(perm) if perm is not None else None
    assert lib.spconvb_dense_bytes(ch, batch, cabi.i3(grid), pp, lay, 1 if i8 else 0) == \
        out.numel() * out.element_size()
    inv = float(np.float32(127.0) / np.float32(dynamic_range)) if i8 else 1.0
    cabi.check(lib.spconvb_scatter_dense_layout(
        _ptr(feat), kind_of(feat), in_scale, _ptr(coords), _ptr(n_ptr), feat.shape[0], ch, batch,
        cabi.i3(grid), pp, lay, 1 if i8 else 0, inv, _ptr(out), _stream()), "scatter_dense_layout")
    return out


def voxel_params(prange, vsize, grid_xyz, num_features=5, points_kind=0, max_pts=10,
                 max_voxels=160000, order=0):
    p = cabi.VoxelParams()
    for i in range(3):
        p.range_min[i], p.range_max[i] = prange[i], prange[3 + i]
        p.voxel_size[i], p.grid[i] = vsize[i], grid_xyz[i]
    p.num_features, p.points_kind = num_features, points_kind
    p.max_points_per_voxel, p.max_voxels, p.order = max_pts, max_voxels, order
    return p


def voxelize(points, params, status=None):
    """points: cuda tensor [n, F] float32/float16.  Returns (features, indices, n_ptr)."""
    n = points.shape[0]
    lib = cabi.lib()
    dev = points.device
    p = C.byref(params)
    ws = torch.empty(max(256, lib.spconvb_voxelize_workspace_bytes(p, max(n, 1))),
                     dtype=torch.uint8, device=dev)
    feat = torch.empty((params.max_voxels, params.num_features), dtype=torch.float16, device=dev)
    idx = torch.empty((params.max_voxels, 4), dtype=torch.int32, device=dev)
    n_ptr = torch.empty(1, dtype=torch.int32, device=dev)
    cabi.check(lib.spconvb_voxelize_flags(p, _ptr(points), n, _ptr(ws), _ptr(feat), _ptr(idx),
                                          _ptr(n_ptr), cabi.FLAG_CLEAR_TAIL, _ptr(status),
                                          _stream()), "voxelize")
    return feat, idx, n_ptr


# ------------------------------------------------------------- 4-bit floating point
_FP4_KIND = {torch.float16: F16, torch.float32: F32, torch.int8: I8}
_FP4_MAX_CHANNELS = 65536
_FP4_SCALES = 2.0 ** -126, 3.4e38 / 448         # the tensor scales that the library takes
_FP32_NORMAL, _FP32_MAX = 2.0 ** -126, (2 - 2.0 ** -23) * 2.0 ** 127
_INT32, _FLOAT16, _empty_strided = torch.int32, torch.float16, torch.empty_strided


def _fp4_pitches(fmt, channels):
    """Bytes of a row's codes and scales, as spconvb_fp4_code_pitch() and spconvb_fp4_scale_pitch()."""
    if fmt not in (MXFP4, NVFP4) or not 1 <= channels <= _FP4_MAX_CHANNELS:
        raise ValueError("no 4-bit rows of %s channels in format %s" % (channels, fmt))
    k = (channels + 63) // 64
    return 32 * k, 4 * ((k + 1) // 2 if fmt == MXFP4 else k)


def _fp4_device(dev, count, *others):
    """Checks a tensor's device, which has to be the current one (the library enqueues there) and that of the row
    count (int32) and of the others."""
    if dev < 0 or dev != _current_device():
        raise ValueError("a tensor on device %d where the current CUDA device's is wanted" % dev)
    if count.dtype is not _INT32 or count.get_device() != dev or not count.numel():
        raise ValueError("a row count is an int32 on the rows' device (device_count)")
    for o in others:
        if o is not None and o.get_device() != dev:
            raise ValueError("tensors of different devices")


def _fp4_status(status):
    if status.dtype is not _INT32 or status.numel() < 4 or not status.is_contiguous():
        raise ValueError("a status block is four int32 in a row (new_status)")


def _fp4_tensor_scale(fmt, g):
    if not (g == 1 if fmt == MXFP4 else _FP4_SCALES[0] <= g <= _FP4_SCALES[1]):
        raise ValueError("a tensor scale is a positive number from 1.2e-38 to 7.5e35, and 1 for MXFP4")


def _fp4_stream(dev):
    return _stream() if _raw_stream is None else _raw_stream(dev)


def _fp4_rows(rows):
    if rows > 0xffffffff:  # the library counts in 32 bits, and ctypes would cut it off
        raise ValueError("more rows than 32 bits count")
    return rows


def _fp4_tensor(t, dtype, rows, width, what):
    if t.dtype != dtype or t.dim() != 2 or not t.is_contiguous() or t.shape[0] != rows or t.shape[1] != width:
        raise ValueError("%s: a contiguous %s [%d, %d] is wanted" % (what, dtype, rows, width))


class Fp4Rows:
    """Rows in 4 bits: ``codes`` uint8 [rows, cpad / 2], ``scales`` uint8 [rows, pitch], the format
    (``MXFP4`` or ``NVFP4``), the channels, and the tensor scale (1 for ``MXFP4``)."""

    __slots__ = ("rows", "channels", "fmt", "tensor_scale", "device_index", "codes_ptr", "scales_ptr", "_hold",
                 "_pitches")

    def __init__(self, codes, scales, channels, fmt, tensor_scale=1.0):
        cp, sp = self._pitches = _fp4_pitches(fmt, channels)
        self.rows = _fp4_rows(codes.shape[0]) if codes.dim() else -1
        _fp4_tensor(codes, torch.uint8, self.rows, cp, "codes")
        _fp4_tensor(scales, torch.uint8, self.rows, sp, "scales")
        if codes.device != scales.device:
            raise ValueError("codes and scales of different devices")
        _fp4_tensor_scale(fmt, tensor_scale)
        self._hold = codes, scales
        self.channels, self.fmt, self.tensor_scale = channels, fmt, float(tensor_scale)
        self.device_index, self.codes_ptr, self.scales_ptr = codes.get_device(), codes.data_ptr(), scales.data_ptr()

    @classmethod
    def empty(cls, rows, channels, fmt, tensor_scale=1.0, device="cuda"):
        """Rows with uninitialised contents."""
        t = torch.empty(0, dtype=torch.uint8, device=device)
        return cls._beside(t, rows, channels, fmt, tensor_scale, t.get_device())

    @classmethod
    def _beside(cls, t, rows, channels, fmt, tensor_scale, dev):
        """Uninitialised rows on t's device: one buffer, of which ``codes`` and ``scales`` are made when asked for."""
        _fp4_rows(rows)
        q = cls.__new__(cls)
        cp, sp = q._pitches = _fp4_pitches(fmt, channels)
        q._hold = buf = t.new_empty(rows * (cp + sp), dtype=torch.uint8)
        q.codes_ptr = at = buf.data_ptr()
        q.scales_ptr = at + rows * cp
        q.rows, q.channels, q.fmt, q.tensor_scale, q.device_index = rows, channels, fmt, float(tensor_scale), dev
        return q

    @property
    def codes(self):
        cp = self._pitches[0]
        return self._hold[0] if type(self._hold) is tuple else self._hold[:self.rows * cp].view(self.rows, cp)

    @property
    def scales(self):
        cp, sp = self._pitches
        return self._hold[1] if type(self._hold) is tuple else self._hold[self.rows * cp:].view(self.rows, sp)

    def _buffer(self):
        return self._hold[0] if type(self._hold) is tuple else self._hold

    def _check(self, rows, channels, fmt, tensor_scale, dev):
        if (self.rows, self.channels, self.fmt, self.tensor_scale, self.device_index) != (
                rows, channels, fmt, float(tensor_scale), dev):
            raise ValueError("out: rows of another shape, format, scale or device")
        return self


def fp4_quantize(x, n_ptr, fmt, tensor_scale=1.0, in_scale=1.0, out=None):
    """Rows [rows, channels] fp16, fp32 or int8 (times ``in_scale``) to :class:`Fp4Rows`; ``out``:
    rows to write into, whose format and tensor scale have to be the same."""
    kind = _FP4_KIND.get(x.dtype)
    if kind is None or x.dim() != 2 or not x.is_contiguous():
        raise ValueError("x: a contiguous [rows, channels] tensor of fp16, fp32 or int8")
    dev = x.get_device()
    _fp4_device(dev, n_ptr)
    rows, ch = x.shape
    if out is None:
        out = Fp4Rows._beside(x, rows, ch, fmt, tensor_scale, dev)
    else:
        out._check(rows, ch, fmt, tensor_scale, dev)
    if rows:
        code = cabi.lib().spconvb_fp4_quantize(
            fmt, x.data_ptr(), kind, in_scale, ch, tensor_scale, n_ptr.data_ptr(), rows,
            out.codes_ptr, out.scales_ptr, _fp4_stream(dev))
        if code:
            cabi.check(code, "fp4_quantize")
    return out


def fp4_dequantize(q, n_ptr, out_kind=F16, out=None):
    """What the codes and scales of ``q`` stand for: [rows, channels] fp16 or fp32."""
    rows, dt = q.rows, torch.float32 if out_kind == F32 else torch.float16
    if out is None:
        buf = q._buffer()
        out = _empty_strided((rows, q.channels), (q.channels, 1), dtype=dt, device=buf.device)
    else:
        _fp4_tensor(out, dt, rows, q.channels, "out")
    dev = out.get_device()
    _fp4_device(dev, n_ptr)
    if q.device_index != dev:
        raise ValueError("tensors of different devices")
    if rows:
        code = cabi.lib().spconvb_fp4_dequantize(
            q.fmt, q.codes_ptr, q.scales_ptr, q.channels, q.tensor_scale, out_kind,
            n_ptr.data_ptr(), rows, out.data_ptr(), _fp4_stream(dev))
        if code:
            cabi.check(code, "fp4_dequantize")
    return out


class Fp4Weights:
    """One layer's weights in 4 bits, laid out for ``fp4_linear`` (kvol 1) and ``fp4_conv``.  ``w``:
    [cout, kvol, cin] or [cout, cin], a tensor or an array of fp16 or fp32; ``rows``: the same
    weights quantised already, as :class:`Fp4Rows` of cout * kvol rows (``w`` is then the
    shape).  ``bias``: [cout] or None."""

    def __init__(self, w, fmt, tensor_scale=1.0, bias=None, rows=None, device="cuda"):
        lib = cabi.lib()
        if rows is None:
            w = torch.as_tensor(w)
            if w.dtype not in (torch.float16, torch.float32):
                raise ValueError("weights in fp16 or fp32")
            shape = w.shape
        else:
            shape = tuple(w)
        if len(shape) == 2:
            shape = (shape[0], 1, shape[1])
        if len(shape) != 3:
            raise ValueError("weights are [cout, kvol, cin] or [cout, cin]")
        self.cout, self.kvol, self.cin = (int(v) for v in shape)
        _fp4_tensor_scale(fmt, tensor_scale)
        self.fmt, self.tensor_scale = fmt, float(tensor_scale)
        nbytes = lib.spconvb_fp4_packed_bytes(fmt, self.cin, self.cout, self.kvol)
        if nbytes == 0:
            raise ValueError("no 4-bit weights [%d, %d, %d] in format %s" % (self.cout, self.kvol, self.cin, fmt))
        if self.kvol > 1 and not lib.spconvb_fp4_conv_supported(self.cin, self.cout, self.kvol):
            raise ValueError("the convolution takes no 4-bit weights [%d, %d, %d]" % (self.cout, self.kvol, self.cin))
        flat = self.cout * self.kvol
        if rows is None:
            w = w.to(device).reshape(flat, self.cin).contiguous()
            rows = fp4_quantize(w, device_count(flat, w.device), fmt, tensor_scale)
        else:
            rows._check(flat, self.cin, fmt, tensor_scale, torch.cuda.current_device())
        self.packed = rows._buffer().new_empty(nbytes, dtype=torch.uint8)
        self.device_index, self._device = rows.device_index, self.packed.device
        cabi.check(lib.spconvb_fp4_pack_weights(fmt, self.cin, self.cout, self.kvol, rows.codes_ptr, rows.scales_ptr,
                                                _ptr(self.packed), _stream()), "fp4_pack")
        self.bias = None
        if bias is not None:
            self.bias = torch.as_tensor(bias).to(self.packed.device, torch.float32).contiguous()
            if self.bias.shape != (self.cout,):
                raise ValueError("bias is [cout]")
        # what every call's parameters start from
        self._params = cabi.Fp4Params(fmt, self.cin, self.cout, self.kvol, 1.0)


def _fp4_product(q, wts, act, rows, out_fmt, out_tensor_scale, out):
    """Parameters, output, and the address of its codes or fp16 rows."""
    if q.fmt != wts.fmt or q.channels != wts.cin or q.device_index != wts.device_index:
        raise ValueError("rows and weights of different formats, channels or devices")
    p = cabi.Fp4Params.from_buffer_copy(wts._params)
    alpha = p.alpha = q.tensor_scale * wts.tensor_scale
    # (below fp32's normal numbers every sum is 0 in fp16 all the same)
    if alpha > _FP32_MAX or alpha < _FP32_NORMAL and out_fmt is not None:
        raise ValueError("the product of the tensor scales is beyond fp32")
    if act:
        p.act = act
    if out_fmt is None:
        if out is None:
            out = _empty_strided((rows, wts.cout), (wts.cout, 1), dtype=_FLOAT16, device=wts._device)
        else:
            _fp4_tensor(out, torch.float16, rows, wts.cout, "out")
            if out.get_device() != wts.device_index:
                raise ValueError("tensors of different devices")
        return p, out, out.data_ptr()
    if out is None:
        out = Fp4Rows._beside(wts.packed, rows, wts.cout, out_fmt, out_tensor_scale, wts.device_index)
    else:
        out._check(rows, wts.cout, out_fmt, out_tensor_scale, wts.device_index)
    p.out_fp4, p.out_format, p.out_tensor_scale, p.out_scales = 1, out_fmt, out_tensor_scale, out.scales_ptr
    return p, out, out.codes_ptr


def fp4_linear(q, n_ptr, wts: Fp4Weights, act=ACT_NONE, out_fmt=None, out_tensor_scale=1.0, out=None,
               status=None, wait_test=0):
    """act(x W^T + bias) of 4-bit rows: fp16 [rows, cout], or :class:`Fp4Rows` of ``out_fmt``."""
    rows = q.rows
    dev = wts.device_index
    _fp4_device(dev, n_ptr, status)
    if status is not None:
        _fp4_status(status)
    p, out, at = _fp4_product(q, wts, act, rows, out_fmt, out_tensor_scale, out)
    if wait_test:
        p.wait_test = wait_test
    if rows:
        code = cabi.lib().spconvb_fp4_linear(
            C.byref(p), q.codes_ptr, q.scales_ptr, n_ptr.data_ptr(), rows, wts.packed.data_ptr(),
            _ptr(wts.bias), at, _ptr(status), _fp4_stream(dev))
        if code:
            cabi.check(code, "fp4_linear")
    return out


def fp4_conv(q, m, n_out_ptr, wts: Fp4Weights, act=ACT_NONE, res=None, res_relu=False, out_fmt=None,
             out_tensor_scale=1.0, out=None, status=None, launch_rows=0, wait_test=0):
    """Sparse convolution of 4-bit rows over the map ``m`` [kvol, cap] (as ``conv_forward``): bias,
    activation, fp16 residual [cap, cout]; fp16 [cap, cout] or :class:`Fp4Rows` of ``out_fmt``.  ``launch_rows`` only sizes
    the grid."""
    if m.dtype != torch.int32 or m.dim() != 2 or m.shape[0] != wts.kvol or not m.is_contiguous():
        raise ValueError("m is a contiguous int32 [kvol, cap]")
    cap = _fp4_rows(m.shape[1])
    dev = wts.device_index
    _fp4_device(dev, n_out_ptr, m, res, status)
    if status is not None:
        _fp4_status(status)
    p, out, at = _fp4_product(q, wts, act, cap, out_fmt, out_tensor_scale, out)
    if res is not None:
        _fp4_tensor(res, torch.float16, cap, wts.cout, "res")
        p.res, p.res_relu = res.data_ptr(), res_relu
    if not q.rows:  # the library wants a row: one of zeros adds nothing, whatever the map says of it
        q = Fp4Rows._beside(wts.packed, 1, q.channels, q.fmt, q.tensor_scale, dev)
        q._hold.zero_()
    p.in_rows = q.rows
    if wait_test:
        p.wait_test = wait_test
    if cap:
        code = cabi.lib().spconvb_fp4_conv(
            C.byref(p), q.codes_ptr, q.scales_ptr, m.data_ptr(), cap, n_out_ptr.data_ptr(), launch_rows,
            wts.packed.data_ptr(), _ptr(wts.bias), at, _ptr(status), _fp4_stream(dev))
        if code:
            cabi.check(code, "fp4_conv")
    return out
