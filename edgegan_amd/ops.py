"""Operators over rows on torch tensors of the GPU: layer norm and its gradient, 8-bit quantisation and the product of 8-bit
integer matrices, distillation from a teacher's top logits.

They are for training and inference code beside the engine (a head behind the encoder's features, a recogniser that the classifier learns
from); the engine runs the same kernels where ``E_norm`` / ``G_norm`` / ``D_norm`` is 'layernorm', in ``EdgeGAN.set_teacher`` and in 8-bit inference.
A call works on the current stream of its tensors' device, allocates its results there with torch, waits for nothing, and may be
captured into a graph.  The last dimension is the row; the dimensions before it have to be one stride apart as if they were a single one (a slice of columns is fine, a transposed
view is not).  Every refusal raises EdgeGANLibError.  There is no autograd: results have no gradient history, whatever their inputs require, and the gradient calls are
explicit, as everywhere in this package.  A gradient that torch has expanded (of a sum: stride 0) has to be made contiguous first."""
from __future__ import annotations

import math
import sys
from typing import Optional, Tuple

import torch
from torch._C import _cuda_getCurrentRawStream as _stream   # torch.cuda.current_stream(device).cuda_stream without the object

from ._lib import EdgeGANLibError, load_library

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTS = {None: 0, 'none': 0, 'relu': 1, 'lrelu': 2}
_lib = None


def _library():
    """The library, on the HIP runtime that torch uses (two runtimes in a process share neither streams nor memory)."""
    global _lib
    if _lib is None:
        lib = load_library()
        if sys.platform == 'linux':
            with open('/proc/self/maps') as f:
                runtimes = {line.split()[-1] for line in f if 'libamdhip64' in line}
            if len(runtimes) > 1:
                raise EdgeGANLibError('the engine was loaded before torch and runs on another HIP runtime '
                                      f'({", ".join(sorted(runtimes))}): import torch or edgegan_amd.ops first')
        _lib = lib
    return _lib


def _refuse(what: str):
    raise EdgeGANLibError(what)


def _refuse_negated(x: torch.Tensor, name: str):
    """A view that torch negates when it is read: the imaginary part of a conjugate (never consecutive with more than one element)."""
    if x.is_neg():
        _refuse(f'{name}: a view that torch negates when it is read (resolve_neg makes a tensor of it)')


def _rows(x: torch.Tensor, name: str, types=_TYPES) -> Tuple[int, int, int]:
    """(rows, cols, elements between rows) of a GPU tensor of one of `types`."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        _refuse(f'{name}: a tensor on the GPU is required')
    if x.dtype not in types:
        _refuse(f'{name}: {x.dtype} is not one of {", ".join(str(t) for t in types)}')
    shape = x.shape
    n = len(shape)
    if n == 0:
        _refuse(f'{name}: at least one dimension is required')
    cols = shape[-1]
    try:
        consecutive = x.is_contiguous()
    except RuntimeError:
        _refuse(f'{name}: a strided tensor is required, not {x.layout}')
    if cols == 1 or not consecutive:
        _refuse_negated(x, name)
    if consecutive:
        return (shape[0] if n == 2 else 1 if n == 1 else math.prod(shape[:-1])), cols, cols
    stride = x.stride()
    if cols > 1 and stride[-1] != 1:
        _refuse(f'{name}: the last dimension has to be consecutive (stride {stride[-1]})')
    rows, ld = 1, cols
    for i in range(n - 2, -1, -1):
        if shape[i] == 1:
            continue
        if rows == 1:
            ld = stride[i]
        elif stride[i] != ld * rows:
            _refuse(f'{name}: dimensions {tuple(shape[:-1])} with strides {tuple(stride[:-1])} are not rows one stride apart')
        rows *= shape[i]
    if rows > 1 and ld < cols:
        _refuse(f'{name}: rows {ld} elements apart overlap')
    return rows, cols, ld


def _vector(v: Optional[torch.Tensor], n: int, name: str, device: int, dtype: torch.dtype) -> Optional[int]:
    """The address of a consecutive vector of n elements on that GPU (None: null)."""
    if v is None:
        return None
    if not isinstance(v, torch.Tensor) or v.get_device() != device:
        _refuse(f'{name}: a tensor on GPU {device} is required')
    if v.dtype != dtype:
        _refuse(f'{name}: {dtype} is required, not {v.dtype}')
    if n == 1:
        _refuse_negated(v, name)
    try:
        consecutive = v.is_contiguous()
    except RuntimeError:
        _refuse(f'{name}: a strided tensor is required, not {v.layout}')
    if v.numel() != n or not consecutive:
        _refuse(f'{name}: {n} consecutive elements are required, not {tuple(v.shape)} with strides {tuple(v.stride())}')
    return v.data_ptr()


def _like(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _empty(x: torch.Tensor, shape, dtype: torch.dtype) -> torch.Tensor:
    """A new consecutive tensor on x's GPU (with strides given torch allocates it in 1.2 us rather than 1.7)."""
    n = len(shape)
    if n == 1:
        return torch.empty_strided(shape, (1,), dtype=dtype, device=x.device)
    if n == 2 and shape[1]:
        return torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=x.device)
    return torch.empty(shape, dtype=dtype, device=x.device)


def _act(act) -> int:
    if not (act is None or isinstance(act, str)) or act not in _ACTS:
        _refuse(f'act: {act!r} is not one of {", ".join(repr(a) for a in _ACTS)}')
    return _ACTS[act]


def _number(v, name: str) -> float:
    if type(v) is float:
        return v
    if isinstance(v, (int, float)):
        try:
            return float(v)
        except OverflowError:
            _refuse(f'{name}: a number that a float holds is required')
    _refuse(f'{name}: a number is required, not {type(v).__name__}')


def _check(rc: int):
    if rc:
        raise EdgeGANLibError(_lib.eg_last_error(None).decode())


def _workspace(size: int, x: torch.Tensor) -> Tuple[Optional[torch.Tensor], Optional[int]]:
    if size < 0:
        _refuse('sizes out of range')
    if size == 0:
        return None, None
    w = _empty(x, (size,), torch.uint8)
    return w, w.data_ptr()


def _parameter_type(weight, bias, x) -> torch.dtype:
    """One type for both: that of x or f32."""
    t = x.dtype
    for p in (weight, bias):
        if isinstance(p, torch.Tensor):
            t = p.dtype
            break
    if t != x.dtype and t != torch.float32:
        _refuse(f'weight, bias: {x.dtype} or torch.float32 is required, not {t}')
    return t


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               act: Optional[str] = None, statistics: bool = False):
    """y = act((x - mean) rstd weight + bias) over the last dimension, in x's type (f32, bf16, f16); act: None, 'relu', 'lrelu' (slope 0.2).

    statistics: also returns mean and rstd (f32, one of each row), which layer_norm_backward needs."""
    lib = _lib or _library()
    rows, cols, ld = _rows(x, 'x')
    device, wtype = x.get_device(), _parameter_type(weight, bias, x)
    w, b = _vector(weight, cols, 'weight', device, wtype), _vector(bias, cols, 'bias', device, wtype)
    y = _like(x)
    mean = rstd = pm = pr = None
    if statistics:
        mean = _empty(x, x.shape[:-1], torch.float32)
        rstd = torch.empty_like(mean)
        pm, pr = mean.data_ptr(), rstd.data_ptr()
    _check(lib.eg_layer_norm(device, _stream(device), _TYPES[x.dtype], x.data_ptr(), ld, _TYPES[wtype], w, b, rows, cols, _number(eps, 'eps'), _act(act), y.data_ptr(), cols, pm, pr))
    return (y, mean, rstd) if statistics else y


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight: Optional[torch.Tensor] = None,
                        bias: Optional[torch.Tensor] = None, act: Optional[str] = None):
    """(dx, dweight, dbias) of layer_norm at x, with the statistics that it returned; dweight is None without a weight, dbias without a bias.

    Where the pre-activation is exactly 0 the derivative of 'lrelu' is its slope 0.2, that of 'relu' 0."""
    lib = _lib or _library()
    rows, cols, ld = _rows(x, 'x')
    device = x.get_device()
    if not isinstance(dy, torch.Tensor) or dy.get_device() != device or dy.dtype != x.dtype or dy.shape != x.shape:
        _refuse(f'dy: {x.dtype} of shape {tuple(x.shape)} on {x.device} is required')
    ldy = _rows(dy, 'dy')[2]
    m, r = _vector(mean, rows, 'mean', device, torch.float32), _vector(rstd, rows, 'rstd', device, torch.float32)
    if m is None or r is None:
        _refuse('mean, rstd: required')
    wtype = _parameter_type(weight, bias, x)
    w, b = _vector(weight, cols, 'weight', device, wtype), _vector(bias, cols, 'bias', device, wtype)
    dx = _like(x)
    dweight = dbias = keep = pw = pb = ws = None
    size = 0
    if weight is not None:
        dweight = torch.empty_like(weight)
        pw = dweight.data_ptr()
    if bias is not None:
        dbias = torch.empty_like(bias)
        pb = dbias.data_ptr()
    if pw or pb:
        size = lib.eg_layer_norm_workspace(rows, cols)
        keep, ws = _workspace(size, x)
    _check(lib.eg_layer_norm_backward(device, _stream(device), _TYPES[x.dtype], dy.data_ptr(), ldy, x.data_ptr(), ld, m, r, _TYPES[wtype], w, b, rows, cols, _act(act),
                                      dx.data_ptr(), cols, pw, pb, ws, size))
    return dx, dweight, dbias


def _norm_parameters(norm, cols, device):
    if norm is None:
        return 0, None, None, 1.0
    if not isinstance(norm, (tuple, list)) or len(norm) != 3:
        _refuse('norm: (weight or None, bias or None, eps) is required')
    return 1, _vector(norm[0], cols, 'norm weight', device, torch.float32), _vector(norm[1], cols, 'norm bias', device, torch.float32), _number(norm[2], 'eps')


def quantize_rows(x: torch.Tensor, norm=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale): q int8 of x's shape, scale f32 of each row = max |x| / 127; q = the whole number nearest to 127 x / max |x|, a tie to the even one.

    A row of zeros has scale 0; one with a NaN or an infinity has scale NaN.  norm = (weight, bias, eps): of layer_norm(x, weight, bias, eps) in the same pass
    (weight, bias f32 or None).  q's rows are a multiple of 16 bytes apart, the gap zeros: what int8_matmul reads fastest."""
    lib = _lib or _library()
    rows, cols, ld = _rows(x, 'x')
    device = x.get_device()
    on, g, b, eps = _norm_parameters(norm, cols, device)
    pitch = (cols + 15) // 16 * 16
    q = _empty(x, x.shape[:-1] + (pitch,), torch.int8)
    scale = _empty(x, x.shape[:-1], torch.float32)
    _check(lib.eg_quantize_rows(device, _stream(device), _TYPES[x.dtype], x.data_ptr(), ld, on, g, b, eps, rows, cols, q.data_ptr(), pitch, scale.data_ptr()))
    return (q if pitch == cols else q[..., :cols]), scale


_INT8 = (torch.int8,)


def _weight(weight, k, device) -> Tuple[int, int]:
    n, kw, ld = _rows(weight, 'weight', _INT8)
    if weight.dim() != 2 or weight.get_device() != device or kw != k:
        _refuse(f'weight: [n, {k}] on GPU {device} is required, not {tuple(weight.shape)} on {weight.device}')
    return n, ld


def int8_matmul(q: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """out[..., j] = (sum_k q[..., k] weight[j, k]) scale[...] weight_scale[j] + bias[j], the sum in 32-bit integers.

    q int8 [..., k] with a scale for each row, weight int8 [n, k] with a scale for each output channel (both as quantize_rows returns them; k <= 131071),
    bias f32 [n] or None; out in out_dtype (f32, bf16, f16)."""
    lib = _lib or _library()
    m, k, lda = _rows(q, 'q', _INT8)
    device = q.get_device()
    n, ldb = _weight(weight, k, device)
    if out_dtype not in _TYPES:
        _refuse(f'out_dtype: {out_dtype} is not one of {", ".join(str(t) for t in _TYPES)}')
    s, ws = _vector(scale, m, 'scale', device, torch.float32), _vector(weight_scale, n, 'weight_scale', device, torch.float32)
    b = _vector(bias, n, 'bias', device, torch.float32)
    if s is None or ws is None:
        _refuse('scale, weight_scale: required')
    out = _empty(q, q.shape[:-1] + (n,), out_dtype)
    _check(lib.eg_int8_matmul(device, _stream(device), q.data_ptr(), lda, s, weight.data_ptr(), ldb, ws, b, m, n, k, _TYPES[out_dtype], out.data_ptr(), n))
    return out


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, norm=None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """A linear layer in 8-bit integers: int8_matmul(*quantize_rows(x, norm), weight, weight_scale, bias), in x's type unless out_dtype says otherwise; for few rows
    and for short ones (64 values, without a norm) one launch."""
    lib = _lib or _library()
    m, k, ld = _rows(x, 'x')
    device = x.get_device()
    on, g, beta, eps = _norm_parameters(norm, k, device)
    n, ldw = _weight(weight, k, device)
    if out_dtype is None:
        out_dtype = x.dtype
    elif out_dtype not in _TYPES:
        _refuse(f'out_dtype: {out_dtype} is not one of {", ".join(str(t) for t in _TYPES)}')
    ws, b = _vector(weight_scale, n, 'weight_scale', device, torch.float32), _vector(bias, n, 'bias', device, torch.float32)
    if ws is None:
        _refuse('weight_scale: required')
    out = _empty(x, x.shape[:-1] + (n,), out_dtype)
    xt, ot, px, pw = _TYPES[x.dtype], _TYPES[out_dtype], x.data_ptr(), weight.data_ptr()
    size, keep, wp = 0, None, None
    if not lib.eg_int8_linear_in_one(xt, px, ld, on, g, beta, pw, ldw, m, n, k, ot, n):
        size = lib.eg_int8_linear_workspace(m, k)
        keep, wp = _workspace(size, x)
    _check(lib.eg_int8_linear(device, _stream(device), xt, px, ld, on, g, beta, eps, pw, ldw, ws, b, m, n, k, ot, out.data_ptr(), n, wp, size))
    return out


_F32 = (torch.float32,)
_INDEXES = {torch.int64: 8, torch.int32: 4}   # bytes


def distill_loss(logits: torch.Tensor, index: torch.Tensor, teacher: torch.Tensor, temperature: float = 1.0,
                 row_weight: Optional[torch.Tensor] = None, grad: bool = True):
    """(loss, dlogits): for each row w T^2 KL(softmax(teacher / T) || softmax(logits / T)) over the teacher's kept logits, and the gradient of
    the losses' sum (None with grad=False).

    logits [..., classes] (f32, bf16, f16; dlogits in the same type), index [..., top] int32 or int64 and teacher [..., top] f32 (top <= 1024), row_weight f32 [...]
    or None (1).  An index outside [0, classes) is padding; a row of weight 0 or without a kept logit has loss and gradient 0 whatever its logits hold."""
    lib = _lib or _library()
    rows, cols, ld = _rows(logits, 'logits')
    device, shape = logits.get_device(), logits.shape[:-1]
    if not isinstance(index, torch.Tensor) or not isinstance(teacher, torch.Tensor) or index.shape != teacher.shape or index.shape[:-1] != shape \
            or index.get_device() != device or teacher.get_device() != device:
        _refuse(f'index, teacher: both {tuple(shape)} + (top,) on {logits.device} are required')
    _, top, ldi = _rows(index, 'index', _INDEXES)
    ldt = _rows(teacher, 'teacher', _F32)[2]
    w = _vector(row_weight, rows, 'row_weight', device, torch.float32)
    loss = _empty(logits, shape, torch.float32)
    dlogits = pg = None
    if grad:
        dlogits = _like(logits)
        pg = dlogits.data_ptr()
    size = lib.eg_distill_loss_workspace(rows, cols, top)
    keep, ws = _workspace(size, logits)
    _check(lib.eg_distill_loss(device, _stream(device), _TYPES[logits.dtype], logits.data_ptr(), ld, _INDEXES[index.dtype], index.data_ptr(), ldi, teacher.data_ptr(), ldt,
                               w, rows, cols, top, _number(temperature, 'temperature'), loss.data_ptr(), pg, cols, ws, size))
    return loss, dlogits
