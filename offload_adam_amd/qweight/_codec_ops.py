"""HIP codec launches: quantise into existing payload buffers, dequantise into a
fresh (or given) tensor.  GPU tensors only; every function enqueues on the
current stream of the tensor's device and returns without synchronising.
"""

from ctypes import c_int, c_int64

import torch

from .. import _lib

_nvfp4_ws = {}


def _amax_workspace(device, stream_id):
    key = (device.index, stream_id)
    ws = _nvfp4_ws.get(key)
    if ws is None:
        ws = torch.zeros(_lib.load().oa_norm_workspace_bytes(), dtype=torch.uint8, device=device)
        _nvfp4_ws[key] = ws
    return ws


def _rows_view(t):
    """2-D float tensor -> (tensor with unit column stride, row stride in elements)."""
    if t.dim() != 2:
        raise ValueError(f"expected a 2-D weight, got shape {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError("HIP codecs work on GPU tensors")
    if t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    stride = t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)
    return t, stride


def _payload(t, name, dtype, shape):
    if t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous() or not t.is_cuda:
        raise ValueError(
            f"{name}: need a contiguous GPU tensor of {dtype} with shape {tuple(shape)}, "
            f"got {t.dtype} {tuple(t.shape)}"
        )


def _call(name, device, *args):
    lib = _lib.load()
    with _lib.device_guard(device):
        code = getattr(lib, name)(*args, _lib.current_stream_ptr())
    _lib.check(code, name)


# -------------------------------------------------------------------- int8


def mark_written(*tensors):
    """The kernels write payload tensors through raw pointers, which autograd's
    version counters do not see; bump them, as an in-place torch op would, so
    that anything keyed on a payload's version (the dequantisation cache of the
    linear layers) notices."""
    for t in tensors:
        torch.autograd.graph.increment_version(t)


def quantize_int8_into(src, weight, scales):
    """Per-row symmetric int8 codes of ``src`` into ``weight`` (R,C) int8 and
    ``scales`` (R,) float."""
    src, stride = _rows_view(src)
    rows, cols = src.shape
    _payload(weight, "weight", torch.int8, (rows, cols))
    _payload(scales, "scales", scales.dtype, (rows,))
    _call("oa_quant_int8", src.device, _lib.ptr(src), c_int(_lib.dtype_code(src.dtype)),
          c_int64(stride), c_int64(rows), c_int64(cols), _lib.ptr(weight), _lib.ptr(scales),
          c_int(_lib.dtype_code(scales.dtype)))
    mark_written(weight, scales)


def dequantize_int8(weight, scales, out_dtype=None):
    rows, cols = weight.shape
    out = torch.empty((rows, cols), dtype=out_dtype or scales.dtype, device=weight.device)
    _payload(weight, "weight", torch.int8, (rows, cols))
    _payload(scales, "scales", scales.dtype, (rows,))
    _call("oa_dequant_int8", weight.device, _lib.ptr(weight), _lib.ptr(scales),
          c_int(_lib.dtype_code(scales.dtype)), c_int64(rows), c_int64(cols), _lib.ptr(out),
          c_int(_lib.dtype_code(out.dtype)), c_int64(max(cols, 1)))
    return out


# -------------------------------------------------------------------- int4


def quantize_int4_into(src, group_size, qweight, scales):
    """Group-wise symmetric int4 of ``src`` into ``qweight`` (C/8,R) int32 and
    ``scales`` (C/group,R)."""
    src, stride = _rows_view(src)
    rows, cols = src.shape
    _payload(qweight, "qweight", torch.int32, (cols // 8, rows))
    _payload(scales, "scales", scales.dtype, (cols // group_size, rows))
    _call("oa_quant_int4", src.device, _lib.ptr(src), c_int(_lib.dtype_code(src.dtype)),
          c_int64(stride), c_int64(rows), c_int64(cols), c_int64(group_size),
          _lib.ptr(qweight), _lib.ptr(scales), c_int(_lib.dtype_code(scales.dtype)))
    mark_written(qweight, scales)


def dequantize_int4(qweight, scales, group_size, out_dtype=None):
    rows = qweight.shape[1]
    cols = qweight.shape[0] * 8
    _payload(qweight, "qweight", torch.int32, (cols // 8, rows))
    _payload(scales, "scales", scales.dtype, (cols // group_size, rows))
    out = torch.empty((rows, cols), dtype=out_dtype or scales.dtype, device=qweight.device)
    _call("oa_dequant_int4", qweight.device, _lib.ptr(qweight), _lib.ptr(scales),
          c_int(_lib.dtype_code(scales.dtype)), c_int64(rows), c_int64(cols),
          c_int64(group_size), _lib.ptr(out), c_int(_lib.dtype_code(out.dtype)),
          c_int64(max(cols, 1)))
    return out


# --------------------------------------------------------------------- NF4


def quantize_nf4_into(src, blocksize, packed, absmax):
    src, stride = _rows_view(src)
    rows, cols = src.shape
    _payload(packed, "weight_packed", torch.uint8, (rows, cols // 2))
    _payload(absmax, "absmax", torch.float32, (rows * (cols // blocksize),))
    _call("oa_quant_nf4", src.device, _lib.ptr(src), c_int(_lib.dtype_code(src.dtype)),
          c_int64(stride), c_int64(rows), c_int64(cols), c_int64(blocksize), _lib.ptr(packed),
          _lib.ptr(absmax))
    mark_written(packed, absmax)


def dequantize_nf4(packed, absmax, in_f, blocksize, out_dtype):
    rows = packed.shape[0]
    _payload(packed, "weight_packed", torch.uint8, (rows, in_f // 2))
    _payload(absmax, "absmax", torch.float32, (rows * (in_f // blocksize),))
    out = torch.empty((rows, in_f), dtype=out_dtype, device=packed.device)
    _call("oa_dequant_nf4", packed.device, _lib.ptr(packed), _lib.ptr(absmax), c_int64(rows),
          c_int64(in_f), c_int64(blocksize), _lib.ptr(out), c_int(_lib.dtype_code(out_dtype)),
          c_int64(max(in_f, 1)))
    return out


# ------------------------------------------------------------------- NVFP4


def quantize_nvfp4_into(src, packed, block_scale_fp8, global_scale):
    src, stride = _rows_view(src)
    rows, cols = src.shape
    _payload(packed, "weight_packed", torch.uint8, (rows, cols // 2))
    _payload(block_scale_fp8, "block_scale_fp8", torch.float8_e4m3fn, (rows, cols // 16))
    _payload(global_scale, "global_scale", torch.float32, ())
    with _lib.device_guard(src.device):
        ws = _amax_workspace(src.device, _lib.current_stream_id())
    _call("oa_quant_nvfp4", src.device, _lib.ptr(src), c_int(_lib.dtype_code(src.dtype)),
          c_int64(stride), c_int64(rows), c_int64(cols), _lib.ptr(packed),
          _lib.ptr(block_scale_fp8), _lib.ptr(global_scale), _lib.ptr(ws))
    mark_written(packed, block_scale_fp8, global_scale)


def dequantize_nvfp4(packed, block_scale_fp8, global_scale, in_f, out_dtype):
    rows = packed.shape[0]
    _payload(packed, "weight_packed", torch.uint8, (rows, in_f // 2))
    _payload(block_scale_fp8, "block_scale_fp8", torch.float8_e4m3fn, (rows, in_f // 16))
    _payload(global_scale, "global_scale", torch.float32, ())
    out = torch.empty((rows, in_f), dtype=out_dtype, device=packed.device)
    _call("oa_dequant_nvfp4", packed.device, _lib.ptr(packed), _lib.ptr(block_scale_fp8),
          _lib.ptr(global_scale), c_int64(rows), c_int64(in_f), _lib.ptr(out),
          c_int(_lib.dtype_code(out_dtype)), c_int64(max(in_f, 1)))
    return out


# --------------------------------------------------------------------- FP8

FP8_BLOCK = 128


def _fp8_payload(codes, scale):
    rows, cols = codes.shape
    if not (codes.is_cuda and codes.dtype is torch.float8_e4m3fn and codes.is_contiguous()
            and scale.dtype is torch.float8_e8m0fnu and scale.is_contiguous()
            and scale.shape == (-(-rows // FP8_BLOCK), -(-cols // FP8_BLOCK))
            and scale.device == codes.device):
        _payload(codes, "weight", torch.float8_e4m3fn, (rows, cols))
        _payload(scale, "block_scale", torch.float8_e8m0fnu,
                 (-(-rows // FP8_BLOCK), -(-cols // FP8_BLOCK)))
        raise ValueError("weight and block_scale must be on the same GPU")
    return rows, cols


def _addr(t):
    return None if t is None else t.data_ptr()


def quantize_fp8_into(src, codes, scale):
    src, stride = _rows_view(src)
    rows, cols = _fp8_payload(codes, scale)
    if tuple(src.shape) != (rows, cols) or src.device != codes.device:
        raise ValueError(f"cannot encode {tuple(src.shape)} on {src.device} into a "
                         f"{rows} x {cols} weight on {codes.device}")
    _call("oa_quant_fp8", src.device, src.data_ptr(), _lib.dtype_code(src.dtype), stride, rows,
          cols, codes.data_ptr(), scale.data_ptr())
    mark_written(codes, scale)


def dequantize_fp8(codes, scale, out_dtype):
    rows, cols = _fp8_payload(codes, scale)
    out = torch.empty((rows, cols), dtype=out_dtype, device=codes.device)
    _call("oa_dequant_fp8", codes.device, codes.data_ptr(), scale.data_ptr(), rows, cols,
          out.data_ptr(), _lib.dtype_code(out_dtype), max(cols, 1))
    return out


def _fp8_workspace(device, *sizes):
    nbytes = _lib.load().oa_fp8_linear_workspace_bytes(*sizes)
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def fp8_linear_forward(x, codes, scale, bias):
    """x (T, in) -> (T, out) in x's dtype."""
    x, ldx = _rows_view(x)
    out_f, in_f = _fp8_payload(codes, scale)
    dt = _lib.dtype_code(x.dtype)
    tokens, dev = x.shape[0], x.device
    y = torch.empty((tokens, out_f), dtype=x.dtype, device=dev)
    if y.numel() == 0:
        return y
    ws = _fp8_workspace(dev, tokens, in_f, out_f, 0, 0, 0, 0)
    _call("oa_fp8_linear_forward", dev, x.data_ptr(), ldx, dt, tokens, codes.data_ptr(),
          scale.data_ptr(), _addr(bias), out_f, in_f, y.data_ptr(), ws.data_ptr(), ws.numel())
    return y


def fp8_linear_backward(grad, x, codes, scale, want_dx, want_dw, want_db):
    """grad (T, out), x (T, in) -> (dx, dw, db) in x's dtype, None where not wanted."""
    grad, ldg = _rows_view(grad)
    x, ldx = _rows_view(x)
    out_f, in_f = _fp8_payload(codes, scale)
    dt = _lib.dtype_code(x.dtype)
    tokens, dev = x.shape[0], x.device
    make = torch.empty if tokens and out_f else torch.zeros
    dx = make((tokens, in_f), dtype=x.dtype, device=dev) if want_dx else None
    dw = make((out_f, in_f), dtype=x.dtype, device=dev) if want_dw else None
    db = make((out_f,), dtype=x.dtype, device=dev) if want_db else None
    if tokens and out_f and (want_dx or want_dw or want_db):
        ws = _fp8_workspace(dev, tokens, in_f, out_f, 1, int(want_dx), int(want_dw), int(want_db))
        _call("oa_fp8_linear_backward", dev, grad.data_ptr(), ldg, x.data_ptr(), ldx, dt, tokens,
              codes.data_ptr(), scale.data_ptr(), out_f, in_f, _addr(dx), _addr(dw), _addr(db),
              ws.data_ptr(), ws.numel())
    return dx, dw, db
