"""Operators on device tensors, for predictors that are not the reference's own network (include/dgnn_ops.h, libdgnn_ops.so).

    dense(x, weight, bias, residual)     act(alpha1 * x W^T + alpha2 * residual + bias): the dense layer of the reference's heads
                                         (src/libdg_nn/layers/dense.rs:197-220) at any size, fp16 / bf16
    group_norm(x, num_groups, ...)       group norm over channels-last maps, skip input and activation included
    adjust_logits(logits, ...)           penalties for repeated tokens, biases, masks -- what pool/policy_helper.rs:87-134 does to a
                                         policy, on the device and in front of the soft-max

The tensors are torch tensors on one GPU.  A call enqueues its work on the current torch stream of THAT device, whatever the current
device is, and returns; it may be captured into a graph.  Errors are api.Error with the status codes of the C ABI; arguments are
checked before anything is enqueued.  The operators evaluate and are not differentiable: a tensor that requires grad is refused while
gradients are being recorded.  There is no CPU fallback.

A predictor made of them goes behind the leaf pool and the search like any other (api.python_predictor).
"""
import ctypes
import os
import struct

import torch

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


def _tensor(where, name, t, device, types):
    """The pointer of an operand that lives on `device` and has one of `types`."""
    if not isinstance(t, torch.Tensor):
        _refuse(where, f"{name} must be a tensor, got {type(t).__name__}")
    if t.device != device:
        _refuse(where, f"{name} is on {t.device}, expected {device}")
    if t.dtype not in types:
        _refuse(where, f"{name} is {t.dtype}, expected {' or '.join(str(x) for x in types)}", api.UNSUPPORTED)
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(where, f"{name} requires grad: the operators evaluate only (torch.no_grad() or detach())", api.UNSUPPORTED)
    return t.data_ptr()


def _first(where, name, t, types):
    """The first operand: it says which device the call is for."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(where, f"{name} must be a tensor on a GPU")
    return _tensor(where, name, t, t.device, types)


def _rows(where, name, t, rows, columns, broadcast=False):
    """The row stride of a [rows, columns] operand whose columns are contiguous; with `broadcast`, [columns] stands for every row."""
    shape = t.shape
    if broadcast and (shape == (columns,) or shape == (1, columns)):
        if columns > 1 and t.stride(-1) != 1:
            _refuse(where, f"{name} must be contiguous in its last dimension", api.UNSUPPORTED)
        return 0
    if shape != (rows, columns):
        _refuse(where, f"{name} is {tuple(shape)}, expected {(rows, columns)}")
    if columns > 1 and t.stride(1) != 1:
        _refuse(where, f"{name} must be contiguous in its last dimension", api.UNSUPPORTED)
    return t.stride(0) if rows > 1 else columns


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


def _activation(where, name):
    code = ACTIVATIONS.get(name)
    if code is None:
        _refuse(where, f"activation {name!r} is none of {', '.join(ACTIVATIONS)}")
    return code


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


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
    px = _first(where, "x", x, (torch.float16, torch.bfloat16))
    device, dtype = x.device, x.dtype
    pw = _tensor(where, "weight", weight, device, (dtype,))
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        _refuse(where, f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not multiply: expected [..., k] and [n, k]")
    n, k = weight.shape
    leading = x.shape[:-1]
    m = leading.numel()
    ldx = _rows(where, "x", _flat(where, "x", x, m), m, k)
    ldw = _rows(where, "weight", weight, n, k)
    if out_dtype is None:
        out_dtype = dtype if out is None else out.dtype
    if out_dtype != dtype and out_dtype != torch.float32:
        _refuse(where, f"out_dtype {out_dtype} is neither x's type nor torch.float32", api.UNSUPPORTED)
    pb = pz = ldz = bias_type = 0
    if bias is not None:
        pb = _tensor(where, "bias", bias, device, (dtype, torch.float32))
        _vector(where, "bias", bias, n)
        bias_type = _TYPES[bias.dtype]
    else:
        bias_type = _TYPES[dtype]
    if residual is not None:
        pz = _tensor(where, "residual", residual, device, (out_dtype,))
        if residual.dim() == 1:
            _vector(where, "residual", residual, n)
        elif residual.shape[:-1] != leading:
            _refuse(where, f"residual is {tuple(residual.shape)}, expected {(*leading, n)} or {(n,)}")
        else:
            ldz = _rows(where, "residual", _flat(where, "residual", residual, m), m, n)
    if out is None:
        out = torch.empty(*leading, n, dtype=out_dtype, device=device)
        py, ldy = out.data_ptr(), n
    else:
        py = _tensor(where, "out", out, device, (out_dtype,))
        if out.shape != (*leading, n):
            _refuse(where, f"out is {tuple(out.shape)}, expected {(*leading, n)}")
        ldy = _rows(where, "out", _flat(where, "out", out, m), m, n)
    tail = (m, n, k, ldx, ldw, ldz, ldy, alpha1, alpha2, _TYPES[dtype], _TYPES[out_dtype], bias_type, _activation(where, activation))
    block = _DENSE.pack(px, pw, pb, pz, py, 0, 0, *tail)
    need = ctypes.c_int64()
    status = lib.dgnn_dense_workspace(block, need)
    if status:
        _fail(status, where)
    if need.value:
        workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
        block = _DENSE.pack(px, pw, pb, pz, py, workspace.data_ptr(), need.value, *tail)
    status = lib.dgnn_dense(device.index, _stream(device), block)
    if status:
        _fail(status, where)
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
    px = _first(where, "x", x, tuple(_TYPES))
    device, dtype, shape = x.device, x.dtype, x.shape
    if x.dim() < 2:
        _refuse(where, f"x is {tuple(shape)}, expected [n, ..., c]")
    n, c = shape[0], shape[-1]
    p = shape[1:-1].numel()
    x_n, x_p = _maps(where, "x", x, shape)
    num_groups = int(num_groups)
    if num_groups < 1 or c % num_groups:
        _refuse(where, f"{num_groups} groups do not divide {c} channels")
    pw = pb = pz = z_n = z_p = 0
    affine = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            q = _tensor(where, name, t, device, (dtype, torch.float32) if affine is None else (affine,))
            _vector(where, name, t, c)
            affine = t.dtype
            if name == "weight":
                pw = q
            else:
                pb = q
    if residual is not None:
        pz = _tensor(where, "residual", residual, device, (dtype,))
        z_n, z_p = _maps(where, "residual", residual, shape)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=device)
        py, y_n, y_p = out.data_ptr(), p * c, c
    else:
        py = _tensor(where, "out", out, device, (dtype,))
        y_n, y_p = _maps(where, "out", out, shape)
    tail = (n, p, c, num_groups, x_n, x_p, z_n, z_p, y_n, y_p, eps, _TYPES[dtype], _TYPES[affine or dtype], _activation(where, activation))
    block = _GROUP_NORM.pack(px, pw, pb, pz, py, 0, 0, *tail)
    need = ctypes.c_int64()
    status = lib.dgnn_group_norm_workspace(block, need)
    if status:
        _fail(status, where)
    if need.value:
        workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
        block = _GROUP_NORM.pack(px, pw, pb, pz, py, workspace.data_ptr(), need.value, *tail)
    status = lib.dgnn_group_norm(device.index, _stream(device), block)
    if status:
        _fail(status, where)
    return out


def _per_row(where, name, value, device, rows):
    """(pointer, value for all) of a penalty: one number, or fp32 [rows]."""
    if isinstance(value, torch.Tensor):
        p = _tensor(where, name, value, device, (torch.float32,))
        _vector(where, name, value, rows)
        return p, 1.0
    return 0, float(value)


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
    pl = _first(where, "logits", logits, tuple(_TYPES))
    device, dtype = logits.device, logits.dtype
    if logits.dim() != 2:
        _refuse(where, f"logits is {tuple(logits.shape)}, expected [b, v]")
    b, v = logits.shape
    ld_logits = _rows(where, "logits", logits, b, v)
    pm = ld_mask = pb = ld_bias = ph = t = ld_history = pn = pp = 0
    bias_type, history_type = _TYPES[dtype], 3
    if mask is not None:
        pm = _tensor(where, "mask", mask, device, (torch.int32,))
        ld_mask = _rows(where, "mask", mask, b, (v + 31) // 32, broadcast=True)
    if bias is not None:
        pb = _tensor(where, "bias", bias, device, (dtype, torch.float32))
        ld_bias = _rows(where, "bias", bias, b, v, broadcast=True)
        bias_type = _TYPES[bias.dtype]
    repetitions, repetition = _per_row(where, "repetition", repetition, device, b)
    presences, presence = _per_row(where, "presence", presence, device, b)
    frequencies, frequency = _per_row(where, "frequency", frequency, device, b)
    if history is not None:
        ph = _tensor(where, "history", history, device, tuple(_INTEGERS))
        if history.dim() != 2:
            _refuse(where, f"history is {tuple(history.shape)}, expected [b, t]")
        t = history.shape[1]
        ld_history = _rows(where, "history", history, b, t)
        history_type = _INTEGERS[history.dtype]
    for name, value in (("lengths", lengths), ("prompt_lengths", prompt_lengths)):
        if value is not None:
            if history is None:
                _refuse(where, f"{name} without history")
            q = _tensor(where, name, value, device, (torch.int32,))
            _vector(where, name, value, b)
            if name == "lengths":
                pn = q
            else:
                pp = q
    if t == 0:
        ph = 0
    if out is None:
        out = torch.empty(b, v, dtype=dtype, device=device)
        po, ld_out, out_dtype = out.data_ptr(), v, dtype
    else:
        po = _tensor(where, "out", out, device, (dtype, torch.float32))
        ld_out, out_dtype = _rows(where, "out", out, b, v), out.dtype
    block = _LOGITS.pack(pl, po, pm, pb, ph, pn, pp, repetitions, presences, frequencies, b, v, t, ld_logits, ld_out, ld_mask, ld_bias, ld_history,
                         repetition, presence, frequency, _TYPES[dtype], _TYPES[out_dtype], bias_type, history_type)
    status = lib.dgnn_adjust_logits(device.index, _stream(device), block)
    if status:
        _fail(status, where)
    return out
