"""Operators on the channel vectors of dense features: layer norm (forward, backward, delta form) and the 4-bit microscaled
format MXFP4 (quantisation, products, a linear layer with gradients).

A tensor is seen as rows x channels: a 4-D tensor is a feature map (N, C, H, W) in channels-last memory, one row per pixel;
any other tensor is (..., C), contiguous, one row per token. Types are float32, float16 and bfloat16 (the delta form: those of
the delta path, float32 and float16). As everywhere in this package there is no CPU path, a wrong device, type or
memory format raises before a launch, and launches go to torch's current stream on the tensor's device; an argument is never
copied to make it fit, except an incoming gradient, whose layout the caller cannot choose. Gradients are those of a backward pass,
once; forward-mode tangents are refused. Every wait inside a product is bounded: one that runs out makes ``lib.dc_umma_error()``
non-zero (which synchronises), and leaves its tile of the result unwritten, or NaN where the tile is shared along k.
"""
import functools

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib
from ._lib import lib, check
from .cuda_kernels import _check_feature, _check_like, _check_mask

_CODES = {torch.float32: _lib.DC_F32, torch.float16: _lib.DC_F16, torch.bfloat16: _lib.DC_BF16}


# what torch.cuda.current_stream(i).cuda_stream and torch.cuda.current_device() give, at a fortieth and half of the time
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _launch(op, fn, t, *args):
    """Calls a library entry point on t's device and that device's current stream."""
    index = t.get_device()
    if index == _current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        check(status, op)


@functools.lru_cache(maxsize=4096)
def _bytes_wanted(query, index, *sizes):
    """A workspace query of the library (its answer depends on the sizes and on the device's SMs)."""
    with torch.cuda.device(index):
        return getattr(lib, query)(*sizes)


def _fail(op, text):
    raise RuntimeError(f"deltacnn_b200.{op}: {text}")


def _no_tangent(op, *tensors):
    """A dual tensor does not ask for a gradient: without this its tangent would be dropped and read as a derivative of zero."""
    if _forward_ad._current_level < 0:
        return
    for t in tensors:
        if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
            _fail(op, "there is no forward-mode derivative")


def _code(t, op, name):
    code = _CODES.get(t.dtype)
    if code is None:
        _fail(op, f"{name} has unsupported dtype {t.dtype} (float32, float16 and bfloat16 only)")
    return code


def _rows(x, op, name="x"):
    """(rows, channels) of a feature map or token tensor."""
    if not x.is_cuda:
        _fail(op, f"{name} must be a CUDA tensor (there is no CPU path)")
    if x.dim() == 4:
        if not x.is_contiguous(memory_format=torch.channels_last):
            _fail(op, f"{name} is 4-D and must be a channels_last contiguous feature map (N, C, H, W)")
        n, c, h, w = x.shape
        rows = n * h * w
    else:
        if x.dim() == 0 or not x.is_contiguous():
            _fail(op, f"{name} must be a contiguous (..., channels) tensor or a 4-D channels_last feature map")
        c = x.shape[-1]
        rows = x.numel() // c if c > 0 else 0
    if c == 0:
        _fail(op, f"{name} has no channels")
    return rows, c


def _like_rows(g, x):
    """An incoming gradient in x's layout."""
    if x.dim() == 4:
        return g.contiguous(memory_format=torch.channels_last)
    return g.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


class _Once(torch.autograd.Function):
    """The gradients of an operator that is differentiable once, tied to what they depend on (``of``): whoever asks for their own
    gradients comes through here and is refused, instead of getting a sum without its second-order part."""

    @staticmethod
    def forward(ctx, op, count, *grads_and_of):
        ctx.op = op
        return grads_and_of[:count]

    @staticmethod
    def backward(ctx, *_):
        _fail(ctx.op, "differentiable once: the gradients have no gradients")


def _once(op, grads, *of):
    return _Once.apply(op, len(grads), *grads, *of)


# ---- layer norm ------------------------------------------------------------------------------------------------

def _ln_params(x, c, code, weight, bias, op):
    """The weight's dtype code; weight and bias are (C,) of x's type or float32, of one type."""
    wcode, index = code, x.get_device()
    if c > 1 << 30:
        _fail(op, f"{c} channels are more than 2^30")
    if weight is not None:
        wcode = _ln_param(x, c, weight, index, "weight", op)
    if bias is not None:
        bcode = _ln_param(x, c, bias, index, "bias", op)
        if weight is not None and bcode != wcode:
            _fail(op, "weight and bias must have the same type")
        wcode = bcode
    return wcode


def _ln_param(x, c, t, index, name, op):
    if t.shape != (c,) or t.get_device() != index or not t.is_contiguous() or (t.dtype is not x.dtype and t.dtype is not torch.float32):
        _fail(op, f"{name} must be a contiguous ({c},) tensor of type {x.dtype} or float32 on {x.device}")
    return _CODES[t.dtype]


def _ln_forward(x, rows, c, weight, bias, eps, keep):
    code = _code(x, "layer_norm", "x")
    wcode = _ln_params(x, c, code, weight, bias, "layer_norm")
    y = torch.empty_like(x)
    stats = mean = rstd = None
    if keep:
        stats = x.new_empty((2, rows), dtype=torch.float32)
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
    if rows > 0:
        _launch("layer_norm", lib.dc_layer_norm, x, x.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), mean, rstd, rows, c, code, wcode, eps)
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        rows, c = _rows(x, "layer_norm")
        y, stats = _ln_forward(x, rows, c, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.sizes = rows, c
        ctx.wtype = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        if not torch.is_grad_enabled():
            return (*_LayerNorm._backward(ctx, dy, x, weight, stats), None)
        with torch.no_grad():                                # create_graph
            grads = _LayerNorm._backward(ctx, dy, x, weight, stats)
        return (*_once("layer_norm", grads, dy, x, weight), None)

    @staticmethod
    def _backward(ctx, dy, x, weight, stats):
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        rows, c = ctx.sizes
        # saved-tensor hooks may bring x back in another layout (offloading to pinned memory loses that of a map)
        x = _like_rows(x, x)
        dy = _like_rows(dy, x)
        code, wtype = _CODES[x.dtype], ctx.wtype
        dx = torch.empty_like(x) if need_x else None
        dw = x.new_empty(c, dtype=wtype) if need_w else None
        db = x.new_empty(c, dtype=wtype) if need_b else None
        nbytes = _bytes_wanted("dc_layer_norm_backward_workspace_bytes", x.get_device(), rows, c, code)
        ws = x.new_empty(nbytes, dtype=torch.uint8)
        mean = stats.data_ptr()
        _launch("layer_norm_backward", lib.dc_layer_norm_backward, x, dy.data_ptr(), x.data_ptr(), _ptr(weight), mean, mean + 4 * rows, _ptr(dx), _ptr(dw),
                _ptr(db), rows, c, code, _CODES[wtype], ws.data_ptr(), nbytes)
        return dx, dw, db


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the channels, statistics and arithmetic in float32. ``weight`` and
    ``bias``: (C,) in x's type or float32, or None. Differentiable in x, weight and bias, once: gradients of the gradients are
    refused. Sums are added in an order that follows from the shape, the addresses' alignment (16 bytes, 4, less) and the GPU
    (``DC_GRID_SHARE`` included): where these are equal, equal inputs give equal bits. No reference counterpart."""
    _no_tangent("layer_norm", x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps)
    rows, c = _rows(x, "layer_norm")
    return _ln_forward(x, rows, c, weight, bias, eps, False)[0]


def _delta_map(x, name, weight, bias, op):
    """(pixels, channels, type code, weight's type code) of a feature map in the delta path."""
    _no_tangent(op, x, weight, bias)
    _check_feature(x, name)
    if x.dtype not in (torch.float32, torch.float16):
        _fail(op, f"unsupported dtype {x.dtype} (float32 and float16 only)")
    n, c, h, w = x.shape
    if c == 0:
        _fail(op, f"{name} has no channels")
    code = _CODES[x.dtype]
    return n * h * w, c, code, _ln_params(x, c, code, weight, bias, op)


def _layer_norm_delta_first(x, weight, bias, eps):
    """The norm of a whole first frame as ``prev_out`` of the delta form: bit for bit what ``layer_norm_delta`` computes for a pixel that
    does not change afterwards (``layer_norm`` may add a row's sums in another order)."""
    op = "layer_norm_delta"
    pixels, c, code, wcode = _delta_map(x, "x", weight, bias, op)
    y = torch.empty_like(x)
    _launch(op, lib.dc_layer_norm_delta_first, x, x.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), pixels, c, code, wcode, eps)
    return y


def layer_norm_delta(delta, mask, prev_in, prev_out, weight=None, bias=None, threshold=0.0, eps=1e-5, out=None, out_mask=None):
    """Layer norm over the channels of a (delta, mask) pair with its caches (no gradient): on masked pixels
    ``prev_in += delta`` and ``e = layer_norm(prev_in) - prev_out``; where any ``|e| > threshold`` the pixel stays in the mask,
    ``out = e`` and ``prev_out += e``; elsewhere the out-mask is 0 and ``out`` and ``prev_out`` keep what they hold.
    ``prev_in``: the accumulated input, ``prev_out``: the sum of what was handed on, both updated in place. ``out`` may be
    ``delta`` and ``out_mask`` may be ``mask``; new tensors where None. Before the first frame both caches are zeros, and the frame
    itself is the delta, every pixel masked. At most 8192 channels. Returns (out, out_mask). No reference counterpart."""
    op = "layer_norm_delta"
    _no_tangent(op, prev_in, prev_out)
    pixels, c, code, wcode = _delta_map(delta, "delta", weight, bias, op)
    _check_mask(mask, delta, "mask")
    _check_like(prev_in, delta, "prev_in")
    _check_like(prev_out, delta, "prev_out")
    if out is None:
        out = torch.empty_like(delta)
    else:
        _check_like(out, delta, "out")
    if out_mask is None:
        out_mask = torch.empty_like(mask)
    else:
        _check_mask(out_mask, delta, "out_mask")
    for t, name in ((mask, "mask"), (out_mask, "out_mask")):
        if t.device != delta.device or not t.is_contiguous():
            _fail(op, f"{name} must be contiguous and on {delta.device}")
    if len({t.data_ptr() for t in (delta, prev_in, prev_out)}) < 3 or out.data_ptr() in (prev_in.data_ptr(), prev_out.data_ptr()):
        if delta.numel() > 0:
            _fail(op, "delta, prev_in and prev_out must be three tensors, and out none of the caches")
    _launch(op, lib.dc_layer_norm_delta, delta, delta.data_ptr(), mask.data_ptr(), prev_in.data_ptr(), prev_out.data_ptr(), _ptr(weight), _ptr(bias),
            out.data_ptr(), out_mask.data_ptr(), pixels, c, code, wcode, float(threshold), eps)
    return out, out_mask


# ---- MXFP4 -----------------------------------------------------------------------------------------------------

def _mx4_shapes(rows, cols):
    nb = (cols + 31) // 32
    return (rows, 16 * nb), ((rows + 127) // 128, (nb + 3) // 4, 32, 4, 4)


def _packed_bytes(rows, cols):
    nb = (cols + 31) // 32
    return rows * nb * 16 + (rows + 127) // 128 * ((nb + 3) // 4) * 512


class MX4Tensor:
    """A packed rows x cols matrix. ``data``: uint8 (rows, 16 * nb), nb = ceil(cols / 32), two e2m1 codes a byte, the even
    column in the low half, zeros behind the last column. ``scales``: uint8 (ceil(rows / 128), ceil(nb / 4), 32, 4, 4), block b of
    row r at [r // 128, b // 4, r % 32, r % 128 // 32, b % 4] (what the tensor core reads); its entries for rows behind
    the last one are never looked at, those for blocks behind the last one must not be 255."""
    __slots__ = ("_data", "_scales", "_at", "shape")

    def __init__(self, data, scales, shape):
        rows, cols = shape
        want_data, want_scales = _mx4_shapes(rows, cols)
        if cols <= 0 or data.dtype != torch.uint8 or scales.dtype != torch.uint8 or data.shape != want_data or scales.shape != want_scales:
            raise RuntimeError(f"deltacnn_b200.MX4Tensor: a {rows} x {cols} matrix needs uint8 data {want_data} and scales {want_scales}")
        if not data.is_contiguous() or not scales.is_contiguous() or data.device != scales.device:
            raise RuntimeError("deltacnn_b200.MX4Tensor: data and scales must be contiguous and on one device")
        self._data, self._scales, self._at, self.shape = data, scales, None, (rows, cols)

    @classmethod
    def _empty(cls, rows, cols, like):
        """A new matrix in one allocation: the scales stand behind the codes, ``_at`` bytes into it."""
        q = cls.__new__(cls)
        q._at = rows * ((cols + 31) // 32) * 16
        q._data, q._scales, q.shape = like.new_empty(_packed_bytes(rows, cols), dtype=torch.uint8), None, (rows, cols)
        return q

    @property
    def data(self):
        return self._data if self._at is None else self._data[:self._at].view(_mx4_shapes(*self.shape)[0])

    @property
    def scales(self):
        return self._scales if self._at is None else self._data[self._at:].view(_mx4_shapes(*self.shape)[1])

    def _ptrs(self):
        p = self._data.data_ptr()
        return p, (self._scales.data_ptr() if self._at is None else p + self._at)

    def dequantize(self, dtype=torch.float32):
        return mx4_dequantize(self, dtype)


def _quantize(x, rows, cols, both):
    """(packed x, packed x^T or None)."""
    code = _code(x, "mx4_quantize", "x")
    q = MX4Tensor._empty(rows, cols, x)
    qt = MX4Tensor._empty(cols, rows, x) if both else None
    if rows > 0:
        _launch("mx4_quantize", lib.dc_mx4_quantize, x, x.data_ptr(), *q._ptrs(), *(qt._ptrs() if both else _NONE), None, rows, cols, code, 0, None, 0)
    return q, qt


_NONE = (None, None)


def mx4_quantize(x):
    """x packed along its channels: an ``MX4Tensor`` of rows x channels. Blocks of 32 values share the scale
    2^(floor(log2 max|v|) - 2); values are rounded to the nearest of +-{0, 1/2, 1, 3/2, 2, 3, 4, 6} times the scale (ties to
    even, saturating); a block with an infinity or a NaN becomes NaN. No gradient, no reference counterpart."""
    _no_tangent("mx4_quantize", x)
    rows, cols = _rows(x, "mx4_quantize")
    return _quantize(x, rows, cols, False)[0]


def mx4_quantize_both(x):
    """(packed x, packed x^T) from one read of x; the second is cols x rows with blocks along x's columns (what the products
    of a backward pass contract over)."""
    _no_tangent("mx4_quantize_both", x)
    rows, cols = _rows(x, "mx4_quantize_both")
    if rows == 0:
        _fail("mx4_quantize_both", "x has no rows")
    return _quantize(x, rows, cols, True)


def mx4_dequantize(q, dtype=torch.float32):
    """The values that an ``MX4Tensor`` stands for, as a (rows, cols) tensor."""
    op = "mx4_dequantize"
    rows, cols = q.shape
    if dtype not in _CODES:
        _fail(op, f"unsupported dtype {dtype} (float32, float16 and bfloat16 only)")
    if not q._data.is_cuda:
        _fail(op, "data must be a CUDA tensor (there is no CPU path)")
    out = q._data.new_empty((rows, cols), dtype=dtype)
    if rows > 0:
        _launch(op, lib.dc_mx4_dequantize, out, *q._ptrs(), out.data_ptr(), rows, cols, _CODES[dtype])
    return out


def _check_bias(op, bias, n, device):
    if bias is not None and (bias.shape != (n,) or not bias.is_contiguous() or bias.device != device or bias.dtype not in _CODES):
        _fail(op, f"bias must be a contiguous ({n},) tensor on {device}")


def mx4_matmul(a, b, bias=None, dtype=torch.float16, out=None):
    """``a @ b.T + bias`` of two packed matrices (m x k and n x k, a weight in nn.Linear's layout): products and sums in float32,
    one rounding to ``dtype``. ``bias``: (n,) or None. ``out``: a contiguous (m, n) tensor to write to."""
    op = "mx4_matmul"
    _no_tangent(op, bias)
    (m, k), (n, k2) = a.shape, b.shape
    if k != k2:
        _fail(op, f"the matrices have {k} and {k2} columns")
    code = _CODES.get(dtype)
    if code is None:
        _fail(op, f"unsupported dtype {dtype} (float32, float16 and bfloat16 only)")
    device = a._data.device
    if not a._data.is_cuda or b._data.device != device:
        _fail(op, "both matrices must be on one CUDA device (there is no CPU path)")
    _check_bias(op, bias, n, device)
    if out is None:
        out = a._data.new_empty((m, n), dtype=dtype)
    elif out.dtype != dtype or tuple(out.shape) != (m, n) or not out.is_contiguous() or out.device != device:
        _fail(op, f"out must be a contiguous ({m}, {n}) tensor of type {dtype} on {device}")
    if m > 0 and n > 0:
        _launch(op, lib.dc_mx4_matmul, out, *a._ptrs(), *b._ptrs(), _ptr(bias), out.data_ptr(), m, n, k, 0 if bias is None else _CODES[bias.dtype], code)
    return out


def _empty(like, shape, dtype):
    """A new tensor of rows: a 4-D one is a channels-last map. No view of another: what an autograd function returns has to be its
    own tensor, or nothing may write to it in place."""
    if len(shape) == 4:
        return torch.empty(shape, dtype=dtype, device=like.device, memory_format=torch.channels_last)
    return like.new_empty(shape, dtype=dtype)


def _result(x, rows, c):
    """A new tensor of x's type and shape with c channels."""
    if x.dim() == 2:
        return x.new_empty((rows, c))
    shape = x.shape
    return _empty(x, (shape[0], c, *shape[2:]) if len(shape) == 4 else (*shape[:-1], c), x.dtype)


@functools.lru_cache(maxsize=4096)
def _train_bytes(rows, cols, outs):
    """Bytes of the packed x^T and w^T that a backward pass reads, and of the packed x and w of the forward product."""
    return _packed_bytes(cols, rows), _packed_bytes(cols, outs), _packed_bytes(rows, cols) + _packed_bytes(outs, cols)


class _MX4Linear(torch.autograd.Function):
    """y = Q(x) Q(w)^T + b; dx = Q(dy) Q(w^T)^T, dw = Q(dy^T) Q(x^T)^T, db = sum dy: every operand is rounded along the axis that
    its product sums over, the rounding's own gradient is taken as 1. What is kept for the backward pass is 4-bit. The second
    result is empty: dx depends on the weight and dw on x, and it keeps the way to both without keeping either."""

    @staticmethod
    def forward(ctx, x, weight, bias, rows, cols):
        outs = weight.shape[0]
        need_x, need_w = ctx.needs_input_grad[:2]
        out = _result(x, rows, outs)
        codes = _CODES[x.dtype], _CODES[weight.dtype], 0 if bias is None else _CODES[bias.dtype]
        kept, x_at, w_at = None, None, None
        if rows > 0:
            # the packed x^T and w^T that the backward pass reads, in one piece
            x_bytes, w_bytes, nbytes = _train_bytes(rows, cols, outs)
            x_bytes, w_bytes = x_bytes if need_w else 0, w_bytes if need_x else 0
            x_at, w_at = 0 if need_w else None, x_bytes if need_x else None
            kept = x.new_empty(x_bytes + w_bytes, dtype=torch.uint8)
            ws = x.new_empty(nbytes, dtype=torch.uint8)
            at = kept.data_ptr()
            _launch("mx4_linear", lib.dc_mx4_linear_train, x, x.data_ptr(), weight.data_ptr(), _ptr(bias), out.data_ptr(), at if need_w else None,
                    at + x_bytes if need_x else None, rows, outs, cols, *codes, ws.data_ptr(), nbytes)
        ctx.plan = rows, cols, outs, x.shape, x.dtype, weight.dtype, None if bias is None else bias.dtype, codes, x_at, w_at
        origin = x.new_empty(0) if need_x and need_w else None
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(kept, origin)
        return out, origin

    @staticmethod
    def backward(ctx, dy, _):
        if dy is None:
            return None, None, None, None, None
        kept, origin = ctx.saved_tensors
        if not torch.is_grad_enabled():
            return (*_MX4Linear._backward(ctx, dy, kept), None, None)
        with torch.no_grad():                                # create_graph
            grads = _MX4Linear._backward(ctx, dy, kept)
        return (*_once("mx4_linear", grads, dy, origin), None, None)

    @staticmethod
    def _backward(ctx, dy, kept):
        need_x, need_w, need_b, _, _ = ctx.needs_input_grad
        rows, cols, outs, x_shape, x_dtype, w_dtype, b_dtype, codes, x_at, w_at = ctx.plan
        dy = _like_rows(dy, dy)
        dx = _empty(dy, x_shape, x_dtype) if need_x else None
        if rows == 0:
            return dx, dy.new_zeros((outs, cols), dtype=w_dtype) if need_w else None, dy.new_zeros(outs, dtype=b_dtype) if need_b else None
        dw = dy.new_empty((outs, cols), dtype=w_dtype) if need_w else None
        db = dy.new_empty(outs, dtype=b_dtype) if need_b else None
        at = kept.data_ptr()
        if at % 16:
            kept = kept.clone()                              # saved-tensor hooks may bring it back at any address
            at = kept.data_ptr()
        nbytes = _bytes_wanted("dc_mx4_linear_backward_workspace_bytes", dy.get_device(), rows, outs, cols)
        ws = dy.new_empty(nbytes, dtype=torch.uint8)
        _launch("mx4_linear_backward", lib.dc_mx4_linear_backward, dy, dy.data_ptr(), None if x_at is None else at + x_at, None if w_at is None else at + w_at,
                _ptr(dx), _ptr(dw), _ptr(db), rows, outs, cols, *codes, ws.data_ptr(), nbytes)
        return dx, dw, db


def mx4_linear(x, weight, bias=None):
    """Linear layer over the channels in MXFP4, result in x's type. ``weight``: an ``MX4Tensor`` of outputs x inputs (packed once,
    inference only), or a (outputs, inputs) tensor, which is packed in the call and, like x and ``bias``, gets a gradient from
    4-bit products (dx and dw have the types of x and weight; differentiable once)."""
    op = "mx4_linear"
    rows, cols = _rows(x, op)
    code = _code(x, op, "x")
    packed = isinstance(weight, MX4Tensor)
    _no_tangent(op, x, None if packed else weight, bias)
    outs, k = weight.shape
    if k != cols:
        _fail(op, f"x has {cols} channels, the weight {k} columns")
    _check_bias(op, bias, outs, x.device)
    grad = torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad) or (not packed and weight.requires_grad))
    if packed:
        if grad:
            _fail(op, "a packed weight is for inference: pass the unpacked weight to train, or call under torch.no_grad()")
        if weight._data.device != x.device:
            _fail(op, f"the weight must be on {x.device}")
    else:
        if not weight.is_contiguous() or weight.device != x.device or weight.dtype not in _CODES or outs == 0:
            _fail(op, f"weight must be a contiguous (outputs, {cols}) tensor on {x.device}")
        if grad:
            return _MX4Linear.apply(x, weight, bias, rows, cols)[0]
        weight = _quantize(weight, outs, cols, False)[0]
    out = _result(x, rows, outs)
    if rows > 0 and outs > 0:
        nbytes = _bytes_wanted("dc_mx4_linear_workspace_bytes", x.get_device(), rows, outs, cols)
        ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        _launch(op, lib.dc_mx4_linear, x, x.data_ptr(), *weight._ptrs(), _ptr(bias), out.data_ptr(), rows, outs, cols, code,
                0 if bias is None else _CODES[bias.dtype], _ptr(ws), nbytes)
    return out
