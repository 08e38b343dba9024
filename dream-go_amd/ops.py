"""Operators on device tensors, for predictors that are not the reference's own network (include/dgnn_ops.h, libdgnn_ops.so).

    dense(x, weight, bias, residual)     act(alpha1 * x W^T + alpha2 * residual + bias): the dense layer of the reference's heads
                                         (src/libdg_nn/layers/dense.rs:197-220) at any size, fp16 / bf16
    group_norm(x, num_groups, ...)       group norm over channels-last maps, skip input and activation included
    adjust_logits(logits, ...)           penalties for repeated tokens, biases, masks -- what pool/policy_helper.rs:87-134 does to a
                                         policy, on the device and in front of the soft-max

The tensors are torch tensors on one GPU.  A call enqueues its work on the current torch stream of THAT device, whatever the current
device is, and returns; it may be captured into a graph.  Errors are api.Error with the status codes of the C ABI; arguments are
checked before anything is enqueued.  The operators evaluate and are not differentiable: a tensor that requires grad is refused while
gradients are being recorded, and one with a forward-mode tangent always.  An `out` counts as changed in place.  There is no CPU fallback.

A predictor made of them goes behind the leaf pool and the search like any other (api.python_predictor): that boundary is host memory, so the
planes are copied to the device and value and policy back.
"""
import ctypes
import operator
import os
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import api

OPS_LIB_PATH = os.environ.get("DGNN_OPS_LIBRARY") or os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libdgnn_ops.so")

# every symbol include/dgnn_ops.h declares: (name, restype, argtypes).  Argument blocks travel as packed bytes (the struct formats below).
SYMBOLS = [
    ("dgnn_ops_last_hip_error", ctypes.c_int, []),
    ("dgnn_dense_workspace", ctypes.c_int, [ctypes.c_char_p, ctypes.POINTER(ctypes.c_int64)]),
    ("dgnn_dense", ctypes.c_int, [ctypes.c_int, ctypes.c_void_p, ctypes.c_char_p]),
    ("dgnn_group_norm_workspace", ctypes.c_int, [ctypes.c_char_p, ctypes.POINTER(ctypes.c_int64)]),
    ("dgnn_group_norm", ctypes.c_int, [ctypes.c_int, ctypes.c_void_p, ctypes.c_char_p]),
    ("dgnn_adjust_logits", ctypes.c_int, [ctypes.c_int, ctypes.c_void_p, ctypes.c_char_p]),
]

ACTIVATIONS = {"identity": 0, "relu": 1, "tanh": 2, "gelu": 3, "silu": 4}
_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_HALVES = {torch.float16: 0, torch.bfloat16: 1}
_INTEGERS = {torch.int32: 3, torch.int64: 4}

# dgnn_dense_args, dgnn_group_norm_args, dgnn_logits_args
_DENSE = struct.Struct("@6P8q2f4i")
_GROUP_NORM = struct.Struct("@6P11qf3i")
_LOGITS = struct.Struct("@10P8q3f4i4x")


def _load():
    if not os.path.exists(OPS_LIB_PATH):
        raise ImportError(f"{OPS_LIB_PATH} is missing: run `python dream-go_amd/build.py` (hipcc, gfx950). There is no CPU fallback.")
    lib = ctypes.CDLL(OPS_LIB_PATH, mode=ctypes.RTLD_LOCAL)     # (torch, imported above, has brought the HIP runtime both share)
    for name, restype, argtypes in SYMBOLS:
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    return lib


lib = _load()


def _fail(status, where):
    error = api.Error(status, where)
    if status == api.HIP_ERROR:
        error.hip_error = lib.dgnn_ops_last_hip_error()
        error.args = (f"{error.args[0]} (hipError_t {error.hip_error})",)
    raise error


def _refuse(where, why, status=api.BAD_ARGUMENT):
    raise api.Error(status, f"{where}: {why}")


def _explain(where, name, t, index, types):
    """Raises what is wrong with an operand that should live on device `index` (None: on any GPU) and have one of `types`."""
    if not isinstance(t, torch.Tensor):
        _refuse(where, f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        _refuse(where, f"{name} must be a tensor on a GPU, it is on {t.device}")
    if index is not None and t.get_device() != index:
        _refuse(where, f"{name} is on {t.device}, expected cuda:{index}")
    _refuse(where, f"{name} is {t.dtype}, expected {' or '.join(str(x) for x in types)}", api.UNSUPPORTED)


def _pointer(where, name, t, index, types):
    """The pointer of an operand; `types` is a dict or tuple of what it may be."""
    try:
        if t.get_device() == index and t.dtype in types:
            return t.data_ptr()
    except AttributeError:
        pass
    _explain(where, name, t, index, types)


def _first(where, name, t, types):
    """The device index of the first operand: it says which device the call is for."""
    try:
        index = t.get_device()
        if index >= 0 and t.dtype in types:
            return index
    except AttributeError:
        pass
    _explain(where, name, t, None, types)


def _records(*operands):
    """Whether gradients are being recorded and one of the operands asks for its own, or one has a forward-mode tangent (those are carried on under
    torch.no_grad() too)."""
    if torch.is_grad_enabled():
        for t in operands:
            if t is not None and t.requires_grad:
                return True
    if forward_ad._current_level >= 0:                          # inside a dual_level
        for t in operands:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                return True
    return False


def _no_grad(where):
    _refuse(where, "an operand requires grad or has a tangent: the operators evaluate only (torch.no_grad(), detach(), unpack_dual().primal)", api.UNSUPPORTED)


def _rows(where, name, t, rows, columns, broadcast=False):
    """The row stride of a [rows, columns] operand whose columns are contiguous; with `broadcast`, [columns] stands for every row."""
    shape = t.shape
    if shape == (rows, columns):
        row, column = t.stride()
    elif broadcast and (shape == (columns,) or shape == (1, columns)):
        row, column = 0, t.stride(-1)
    else:
        _refuse(where, f"{name} is {tuple(shape)}, expected {(rows, columns)}" + (f" or {(columns,)}" if broadcast else ""))
    if column != 1 and columns > 1:
        _refuse(where, f"{name} must be contiguous in its last dimension", api.UNSUPPORTED)
    return row if rows > 1 else columns


def _vector(where, name, t, length):
    if t.shape != (length,):
        _refuse(where, f"{name} is {tuple(t.shape)}, expected {(length,)}")
    if length > 1 and t.stride(0) != 1:
        _refuse(where, f"{name} must be contiguous", api.UNSUPPORTED)


def _flat(where, name, t, leading):
    """[..., columns] as [rows, columns] without a copy, or a refusal."""
    if t.dim() == 2:
        return t
    try:
        return t.view(leading, t.shape[-1])
    except RuntimeError:
        _refuse(where, f"{name}'s leading dimensions do not make rows of one stride", api.UNSUPPORTED)


def _number(where, name, value):
    """A number as the block takes it (rounded to fp32 there).  Of a tensor it is the value, so one that carries gradients is refused."""
    if isinstance(value, torch.Tensor) and _records(value):
        _no_grad(where)
    try:
        if isinstance(value, (str, bytes)):
            raise TypeError
        return float(value)
    except (TypeError, ValueError, OverflowError, RuntimeError):               # (RuntimeError: a tensor of more than one element)
        _refuse(where, f"{name} must be a number, got {type(value).__name__}")


def _activation(where, name):
    code = ACTIVATIONS.get(name) if isinstance(name, str) else None
    if code is None:
        _refuse(where, f"activation {name!r} is none of {', '.join(ACTIVATIONS)}")
    return code


# The current stream of a device as a handle; torch.cuda.current_stream makes an object of it first, which takes as long as a launch.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(index):
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def _launch(where, run, workspace, index, block, args):
    """One call; once more with work memory where it asks for some."""
    try:
        packed = block.pack(*args)
    except struct.error as error:
        _refuse(where, f"an argument is out of its type's range ({error})")
    stream = _stream(index)
    status = run(index, stream, packed)
    if status == 0:
        return
    if status == api.BAD_ARGUMENT and workspace is not None:
        need = ctypes.c_int64()
        if workspace(packed, need) == 0 and need.value:
            memory = torch.empty(need.value, dtype=torch.uint8, device=torch.device("cuda", index))
            status = run(index, stream, block.pack(*args[:5], memory.data_ptr(), need.value, *args[7:]))
            if status == 0:
                return
    _fail(status, where)


def dense(x, weight, bias=None, residual=None, *, alpha1=1.0, alpha2=1.0, activation="identity", out=None, out_dtype=None):
    """act(alpha1 * x @ weight.T + alpha2 * residual + bias), summed in fp32 and rounded once.

    x         [..., k] fp16 or bf16, contiguous in k; the leading dimensions are rows of one stride
    weight    [n, k] of x's type, contiguous in k: one row per output
    bias      [n] of x's type or fp32
    residual  [..., n] or [n] of the output's type; may be `out` itself
    out       where to put the result ([..., n], rows of one stride); allocated where None
    out_dtype x's type (default) or torch.float32
    """
    where = "dense"
    index = _first(where, "x", x, _HALVES)
    dtype = x.dtype
    code = _TYPES[dtype]
    pw = _pointer(where, "weight", weight, index, (dtype,))
    shape = x.shape
    if not shape or weight.dim() != 2 or shape[-1] != weight.shape[1]:
        _refuse(where, f"x {tuple(shape)} and weight {tuple(weight.shape)} do not multiply: expected [..., k] and [n, k]")
    n, k = weight.shape
    leading = shape[:-1]
    m = leading.numel()
    ldx = k if x.is_contiguous() else _rows(where, "x", _flat(where, "x", x, m), m, k)
    ldw = k if weight.is_contiguous() else _rows(where, "weight", weight, n, k)
    if out_dtype is None:
        out_dtype = dtype if not isinstance(out, torch.Tensor) else out.dtype
    if out_dtype is not dtype and out_dtype is not torch.float32:
        _refuse(where, f"out_dtype {out_dtype} is neither x's type nor torch.float32", api.UNSUPPORTED)
    pb = pz = ldz = 0
    bias_code = code
    if bias is not None:
        pb = _pointer(where, "bias", bias, index, (dtype, torch.float32))
        _vector(where, "bias", bias, n)
        bias_code = _TYPES[bias.dtype]
    if residual is not None:
        pz = _pointer(where, "residual", residual, index, (out_dtype,))
        if residual.dim() == 1:
            _vector(where, "residual", residual, n)
        elif residual.shape != (*leading, n):
            _refuse(where, f"residual is {tuple(residual.shape)}, expected {(*leading, n)} or {(n,)}")
        else:
            ldz = n if residual.is_contiguous() else _rows(where, "residual", _flat(where, "residual", residual, m), m, n)
    given = out is not None
    if not given:
        out = torch.empty((*leading, n), dtype=out_dtype, device=x.device)
        py, ldy = out.data_ptr(), n
    else:
        py = _pointer(where, "out", out, index, (out_dtype,))
        if out.shape != (*leading, n):
            _refuse(where, f"out is {tuple(out.shape)}, expected {(*leading, n)}")
        ldy = n if out.is_contiguous() else _rows(where, "out", _flat(where, "out", out, m), m, n)
    if _records(x, weight, bias, residual, out):
        _no_grad(where)
    if type(alpha1) is not float or type(alpha2) is not float:
        alpha1, alpha2 = _number(where, "alpha1", alpha1), _number(where, "alpha2", alpha2)
    _launch(where, lib.dgnn_dense, lib.dgnn_dense_workspace, index, _DENSE,
            (x.data_ptr(), pw, pb, pz, py, 0, 0, m, n, k, ldx, ldw, ldz, ldy, alpha1, alpha2, code, _TYPES[out_dtype], bias_code, _activation(where, activation)))
    if given:
        increment_version(out)      # what autograd has saved of it is not what it holds now
    return out


def _maps(where, name, t, shape):
    """(sample stride, position stride) of channels-last maps [n, ..., c] whose positions have one stride."""
    if t.shape != shape:
        _refuse(where, f"{name} is {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dim() != 3:
        try:
            t = t.view(shape[0], shape[1:-1].numel(), shape[-1])
        except RuntimeError:
            _refuse(where, f"{name}'s positions do not have one stride", api.UNSUPPORTED)
    if t.shape[2] > 1 and t.stride(2) != 1:
        _refuse(where, f"{name} must be contiguous in its channels, the last dimension", api.UNSUPPORTED)
    return t.stride(0), t.stride(1)


def group_norm(x, num_groups, weight=None, bias=None, residual=None, *, eps=1e-5, activation="identity", out=None):
    """act((x - mean) / sqrt(variance + eps) * weight + bias + residual) over channels-last maps.

    Mean and (biased) variance are those of a sample's group: all its positions x the group's channels, in fp32; one rounding at the end.

    x         [n, ..., c] fp16, bf16 or fp32, contiguous in c, the positions of one stride; num_groups divides c
    weight    [c] of x's type or fp32 (default 1);  bias: the same type as weight (default 0)
    residual  of x's shape and type
    out       of x's shape and type; may be x or residual itself.  Allocated where None
    """
    where = "group_norm"
    index = _first(where, "x", x, _TYPES)
    dtype, shape = x.dtype, x.shape
    if len(shape) < 2:
        _refuse(where, f"x is {tuple(shape)}, expected [n, ..., c]")
    n, c = shape[0], shape[-1]
    p = shape[1] if len(shape) == 3 else shape[1:-1].numel()
    x_n, x_p = (p * c, c) if x.is_contiguous() else _maps(where, "x", x, shape)
    if type(num_groups) is not int:
        try:
            num_groups = operator.index(num_groups)
        except TypeError:
            _refuse(where, f"num_groups must be a whole number, got {type(num_groups).__name__}")
    if num_groups < 1 or c % num_groups:
        _refuse(where, f"{num_groups} groups do not divide {c} channels")
    pw = pb = pz = z_n = z_p = 0
    affine = dtype
    if weight is not None:
        pw = _pointer(where, "weight", weight, index, (dtype, torch.float32))
        _vector(where, "weight", weight, c)
        affine = weight.dtype
    if bias is not None:
        pb = _pointer(where, "bias", bias, index, (dtype, torch.float32) if weight is None else (affine,))
        _vector(where, "bias", bias, c)
        affine = bias.dtype
    if residual is not None:
        pz = _pointer(where, "residual", residual, index, (dtype,))
        z_n, z_p = (p * c, c) if residual.is_contiguous() and residual.shape == shape else _maps(where, "residual", residual, shape)
    given = out is not None
    if not given:
        out = torch.empty_like(x) if x.is_contiguous() else torch.empty(shape, dtype=dtype, device=x.device)
        py, y_n, y_p = out.data_ptr(), p * c, c
    else:
        py = _pointer(where, "out", out, index, (dtype,))
        y_n, y_p = _maps(where, "out", out, shape)
    if _records(x, weight, bias, residual, out):
        _no_grad(where)
    _launch(where, lib.dgnn_group_norm, lib.dgnn_group_norm_workspace, index, _GROUP_NORM,
            (x.data_ptr(), pw, pb, pz, py, 0, 0, n, p, c, num_groups, x_n, x_p, z_n, z_p, y_n, y_p, eps if type(eps) is float else _number(where, "eps", eps), _TYPES[dtype], _TYPES[affine],
             _activation(where, activation)))
    if given:
        increment_version(out)      # what autograd has saved of it is not what it holds now
    return out


def _per_row(where, name, value, index, rows):
    """(pointer, value for all) of a penalty: one number, or fp32 [rows]."""
    if isinstance(value, torch.Tensor):
        p = _pointer(where, name, value, index, (torch.float32,))
        _vector(where, name, value, rows)
        return p, 1.0
    return 0, value if type(value) is float else _number(where, name, value)


def adjust_logits(logits, *, mask=None, bias=None, history=None, lengths=None, prompt_lengths=None,
                  repetition=1.0, presence=0.0, frequency=0.0, out=None):
    """Logits [b, v] with penalties for repeated tokens, a bias and a mask applied, in this order, in fp32:

        seen:   l = l / repetition where l > 0, l * repetition elsewhere
                l = l - frequency * count - (presence where count > 0)
                l = l + bias
        masked: l = -inf, whatever it was (a row whose mask leaves nothing is -inf throughout)

    logits          fp16, bf16 or fp32, contiguous in v
    mask            int32 [b, ceil(v / 32)], or [ceil(v / 32)] for all rows: bit v % 32 of word v // 32 set = token v is allowed
    bias            [b, v], or [v] for all rows; of the logits' type or fp32
    history         int32 or int64 [b, t]: the row's tokens, the first `lengths` of them (int32 [b], default t).  Tokens outside 0 .. v-1
                    are padding.  `seen` looks at all of them, `count` at those from `prompt_lengths` (int32 [b], default 0) on
    repetition, presence, frequency   a number, or fp32 [b]; repetition > 0.  Without history they do nothing
    out             [b, v] of the logits' type or fp32; may be logits itself.  Allocated (logits' type) where None
    """
    where = "adjust_logits"
    index = _first(where, "logits", logits, _TYPES)
    dtype = logits.dtype
    if logits.dim() != 2:
        _refuse(where, f"logits is {tuple(logits.shape)}, expected [b, v]")
    b, v = logits.shape
    ld_logits = v if logits.is_contiguous() else _rows(where, "logits", logits, b, v)
    pm = ld_mask = pb = ld_bias = ph = t = ld_history = pn = pp = repetitions = presences = frequencies = 0
    bias_code, history_code = _TYPES[dtype], 3
    if mask is not None:
        pm = _pointer(where, "mask", mask, index, (torch.int32,))
        ld_mask = _rows(where, "mask", mask, b, (v + 31) // 32, broadcast=True)
    if bias is not None:
        pb = _pointer(where, "bias", bias, index, (dtype, torch.float32))
        ld_bias = _rows(where, "bias", bias, b, v, broadcast=True)
        bias_code = _TYPES[bias.dtype]
    tensors = [t for t in (repetition, presence, frequency) if isinstance(t, torch.Tensor)]
    repetitions, repetition = _per_row(where, "repetition", repetition, index, b)
    presences, presence = _per_row(where, "presence", presence, index, b)
    frequencies, frequency = _per_row(where, "frequency", frequency, index, b)
    if history is not None:
        ph = _pointer(where, "history", history, index, _INTEGERS)
        if history.dim() != 2:
            _refuse(where, f"history is {tuple(history.shape)}, expected [b, t]")
        t = history.shape[1]
        ld_history = _rows(where, "history", history, b, t)
        history_code = _INTEGERS[history.dtype]
        if lengths is not None:
            pn = _pointer(where, "lengths", lengths, index, (torch.int32,))
            _vector(where, "lengths", lengths, b)
        if prompt_lengths is not None:
            pp = _pointer(where, "prompt_lengths", prompt_lengths, index, (torch.int32,))
            _vector(where, "prompt_lengths", prompt_lengths, b)
    elif lengths is not None or prompt_lengths is not None:
        _refuse(where, "lengths without history")
    given = out is not None
    if not given:
        out = torch.empty_like(logits) if logits.is_contiguous() else torch.empty((b, v), dtype=dtype, device=logits.device)
        po, ld_out, out_dtype = out.data_ptr(), v, dtype
    else:
        po = _pointer(where, "out", out, index, (dtype, torch.float32))
        ld_out, out_dtype = _rows(where, "out", out, b, v), out.dtype
    if _records(logits, bias, out) or (repetitions or presences or frequencies) and _records(*tensors):
        _no_grad(where)
    _launch(where, lib.dgnn_adjust_logits, None, index, _LOGITS,
            (logits.data_ptr(), po, pm, pb, ph if t else 0, pn, pp, repetitions, presences, frequencies, b, v, t, ld_logits, ld_out, ld_mask, ld_bias, ld_history,
             repetition, presence, frequency, _TYPES[dtype], _TYPES[out_dtype], bias_code, history_code))
    if given:
        increment_version(out)      # what autograd has saved of it is not what it holds now
    return out
