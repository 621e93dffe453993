"""The training operators next to the environment step (libb3train.so,
include/b3x_train.h), over ctypes: log probabilities of actions and their
gradient, advantages, and the AdamW step.

Arguments are torch tensors on the current CUDA device; outputs are tensors of
the caller's that the call fills.  Every call only enqueues on `stream` (the
current stream by default), allocates nothing on the device and returns a
cudaError_t code: 0 success, 1 invalid arguments (types, shapes, strides or
devices that the call does not take), with nothing launched or written.  Memory
given to a call is in use on its stream until the work is done, as with any
kernel: a tensor that another stream made or will free has to be ordered by the
caller.  There is no CPU path: loading fails loudly when the library is
missing.

The header states each operator's formulas and what it does with masked rows,
actions that are none, terminals and lengths.
"""
import array
import ctypes
import operator
import os

import torch

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "_lib", "libb3train.so")

CUDA_SUCCESS = 0
CUDA_ERROR_INVALID_VALUE = 1
MAX_TOP = 32             # alternatives a row (B3X_TRAIN_MAX_TOP)
BLOCK = 256              # elements that share a scale of 8-bit moments (B3X_TRAIN_BLOCK)

_F32, _BF16, _F16, _E4M3, _U8 = range(5)
_FLOATS = {torch.float32: _F32, torch.bfloat16: _BF16, torch.float16: _F16}
_BYTES = {torch.uint8: _U8, torch.bool: _U8}

_Strides = ctypes.c_longlong * 11
_numel, _dense, _where, _pointer = (torch.Tensor.numel, torch.Tensor.is_contiguous, torch.Tensor.get_device,
                                    torch.Tensor.data_ptr)
_kind = operator.attrgetter("dtype")

_lib = None


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError("%s is not built; run python -m puffysics_b200.build" % LIB_PATH)
        L = ctypes.CDLL(LIB_PATH)
        vp, i, ll, f, d = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_double
        rows = [vp, i, ll, ll, ll, vp, ll, vp, i, f]
        L.b3x_train_logprob_gpu.argtypes = rows + [vp, vp, vp, i, vp, vp, vp]
        L.b3x_train_logprob_grad_gpu.argtypes = rows + [vp, vp, vp, vp, vp, ll, vp]
        L.b3x_train_advantage_gpu.argtypes = [ll, ll, vp, vp, i, vp, i, vp, vp, vp, vp, vp, f, f, vp]
        L.b3x_train_grad_norm_workspace_bytes.argtypes = []
        L.b3x_train_grad_norm_workspace_bytes.restype = ctypes.c_size_t
        L.b3x_train_grad_norm_gpu.argtypes = [i, vp, i, vp, d, vp, vp, ctypes.c_size_t, vp]
        L.b3x_train_adamw_gpu.argtypes = [i, vp, i, vp, i, vp, vp, vp, i, vp, vp, vp, ll, d, d, d, d, d, vp, i,
                                          ctypes.c_uint, vp]
        for name in ("logprob", "logprob_grad", "advantage", "grad_norm", "adamw"):
            getattr(L, "b3x_train_%s_gpu" % name).restype = ctypes.c_int
        _lib = L
    return _lib


_device = torch.cuda.current_device
# the current stream's handle without the object around it, which costs as much as a launch
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _s(stream, device):
    return _raw_stream(device) if stream is None else stream.cuda_stream


class _Refused(Exception):
    """An argument that a call does not take: the call returns cudaErrorInvalidValue."""


def _vec(t, n, device, dtype=torch.float32):
    """The pointer of a dense tensor of n elements, of this type, on the device; None for none."""
    if t is None:
        return None
    if t.dtype is dtype and t.dim() == 1 and t.numel() == n and t.is_contiguous() and t.get_device() == device:
        return t.data_ptr()
    raise _Refused


def _mat(t, rows, cols, device, dtype=torch.float32):
    """The same for (rows, cols)."""
    if t is None:
        return None
    if (t.dtype is dtype and t.dim() == 2 and t.size(1) == cols and t.size(0) == rows and t.is_contiguous()
            and t.get_device() == device):
        return t.data_ptr()
    raise _Refused


def _rows(logits, actions, mask):
    """The leading arguments of the two calls over rows of logits, and the device."""
    kind = _FLOATS.get(logits.dtype)
    if kind is None or logits.dim() != 2:
        raise _Refused
    rows, width = logits.shape
    row_stride, stride = logits.stride()
    device = logits.get_device()
    if device < 0 or (stride != 1 and width > 1) or device != _device():
        raise _Refused
    mask_at = None
    mask_stride = action_bytes = 0
    if actions is not None:
        action_bytes = 8 if actions.dtype is torch.int64 else 4
        actions = _vec(actions, rows, device, torch.int64 if action_bytes == 8 else torch.int32)
    if mask is not None:
        if (mask.dtype not in _BYTES or mask.dim() != 2 or mask.size(0) != rows or mask.size(1) != width
                or mask.get_device() != device):
            raise _Refused
        mask_stride, stride = mask.stride()
        if stride != 1 and width > 1:
            raise _Refused
        mask_at = mask.data_ptr()
    return logits.data_ptr(), kind, rows, width, row_stride, mask_at, mask_stride, actions, action_bytes, device


def logprob(logits, actions=None, logp=None, entropy=None, stats=None, top_ids=None, top_logp=None, mask=None,
            scale=1.0, stream=None):
    """Log probability of each row's action, entropy and most likely
    alternatives of (rows, width) logits (float32, bfloat16 or float16, rows at
    any stride).

    actions (rows,) int32 or int64; mask (rows, width) uint8 or bool, zero
    where an action is not allowed (rows at any stride; expand() one row for
    all).  Outputs, each optional: logp (rows,), entropy (rows,), stats
    (rows, 2) with the row's maximum and the log of its sum of exponentials
    above it (what logprob_grad takes), top_ids (rows, k) int32 with top_logp
    (rows, k), k up to 32; float32 where not said otherwise."""
    try:
        z, kind, rows, width, stride, mask, mask_stride, act, act_bytes, device = _rows(logits, actions, mask)
        top = 0
        if top_ids is not None or top_logp is not None:
            if top_ids is None or top_logp is None or top_ids.dim() != 2:
                return CUDA_ERROR_INVALID_VALUE
            top = top_ids.size(1)
            top_ids, top_logp = _mat(top_ids, rows, top, device, torch.int32), _mat(top_logp, rows, top, device)
        return lib().b3x_train_logprob_gpu(z, kind, rows, width, stride, mask, mask_stride, act, act_bytes, scale,
                                           _vec(logp, rows, device), _vec(entropy, rows, device),
                                           _mat(stats, rows, 2, device), top, top_ids, top_logp, _s(stream, device))
    except _Refused:
        return CUDA_ERROR_INVALID_VALUE


def logprob_grad(logits, stats, grad, actions=None, d_logp=None, entropy=None, d_entropy=None, mask=None, scale=1.0,
                 stream=None):
    """Gradient of sum(d_logp * logp) + sum(d_entropy * entropy) with respect
    to the logits, into grad (their shape and type, rows at any stride; the
    logits themselves to overwrite them), from the stats (and entropy, where
    d_entropy is given) that logprob wrote."""
    try:
        z, kind, rows, width, stride, mask, mask_stride, act, act_bytes, device = _rows(logits, actions, mask)
        if (grad.dtype is not logits.dtype or grad.dim() != 2 or grad.size(0) != rows or grad.size(1) != width
                or grad.get_device() != device or stats is None):
            return CUDA_ERROR_INVALID_VALUE
        grad_stride, one = grad.stride()
        if one != 1 and width > 1:
            return CUDA_ERROR_INVALID_VALUE
        return lib().b3x_train_logprob_grad_gpu(z, kind, rows, width, stride, mask, mask_stride, act, act_bytes, scale,
                                                _mat(stats, rows, 2, device), _vec(entropy, rows, device),
                                                _vec(d_logp, rows, device), _vec(d_entropy, rows, device),
                                                grad.data_ptr(), grad_stride, _s(stream, device))
    except _Refused:
        return CUDA_ERROR_INVALID_VALUE


def advantage(rewards, values, terminals, last_values, advantages, returns=None, gamma=0.99, lam=0.95, lengths=None,
              stream=None):
    """Generalised advantages and returns of a (steps, envs) rollout, any
    strides (pass .t() of arrays with one row per environment).

    rewards, advantages, returns float32; values and last_values (envs,)
    float32, bfloat16 or float16; terminals float32, uint8 or bool; lengths
    (envs,) int32, the steps that each environment has."""
    shape = rewards.shape
    kind, f32, device = _FLOATS.get(values.dtype), torch.float32, rewards.get_device()
    if (len(shape) != 2 or kind is None or rewards.dtype is not f32 or advantages.dtype is not f32
            or last_values.dtype is not values.dtype
            or (terminals.dtype is not f32 and terminals.dtype not in _BYTES)
            or values.shape != shape or terminals.shape != shape or advantages.shape != shape
            or last_values.shape != shape[1:] or device < 0 or device != _device()
            or values.get_device() != device or terminals.get_device() != device
            or last_values.get_device() != device or advantages.get_device() != device):
        return CUDA_ERROR_INVALID_VALUE
    if returns is not None and (returns.dtype is not f32 or returns.shape != shape or returns.get_device() != device):
        return CUDA_ERROR_INVALID_VALUE
    try:
        lengths = _vec(lengths, shape[1], device, torch.int32)
    except _Refused:
        return CUDA_ERROR_INVALID_VALUE
    strides = _Strides(*rewards.stride(), *values.stride(), *terminals.stride(), *last_values.stride(),
                       *advantages.stride(), *((0, 0) if returns is None else returns.stride()))
    return lib().b3x_train_advantage_gpu(shape[0], shape[1], rewards.data_ptr(), values.data_ptr(), kind,
                                         terminals.data_ptr(), _F32 if terminals.dtype is f32 else _U8,
                                         last_values.data_ptr(), lengths, advantages.data_ptr(),
                                         None if returns is None else returns.data_ptr(), strides,
                                         gamma, lam, _s(stream, device))


def _list(tensors, sizes, dtype, device):
    """Pointers of a list of dense tensors on the device, of one type and these
    element counts; None where they are not."""
    if (list(map(_numel, tensors)) != sizes or not all(map(_dense, tensors)) or {dtype} != {dtype, *map(_kind, tensors)}
            or {device} != {device, *map(_where, tensors)}):
        return None
    return array.array("Q", map(_pointer, tensors))


def _addr(a):
    return None if a is None else a.buffer_info()[0]


def grad_norm_workspace_bytes():
    return lib().b3x_train_grad_norm_workspace_bytes()


def grad_norm(grads, max_norm, out, workspace, stream=None):
    """Global 2-norm of a list of gradients into out[0], and the factor that
    clips them to max_norm into out[1] (out (2,) float32; NaN where the norm is
    not finite).  workspace: a uint8 tensor of grad_norm_workspace_bytes()."""
    device = _device()
    sizes = list(map(_numel, grads))
    dtype = grads[0].dtype if grads else torch.float32
    g = _list(grads, sizes, dtype, device) if dtype in _FLOATS else None
    if (g is None or out.dtype is not torch.float32 or out.shape != (2,) or not out.is_contiguous()
            or out.get_device() != device or workspace.dtype is not torch.uint8 or not workspace.is_contiguous()
            or workspace.get_device() != device):
        return CUDA_ERROR_INVALID_VALUE
    counts = array.array("q", sizes)   # named, so that it outlives the call
    return lib().b3x_train_grad_norm_gpu(len(sizes), _addr(g), _FLOATS[dtype], _addr(counts), max_norm,
                                         out.data_ptr(), workspace.data_ptr(), workspace.numel(), _s(stream, device))


def adamw(params, grads, exp_avg, exp_avg_sq, step, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01,
          scales=None, grad_scale=None, copies=None, seed=None, stream=None):
    """One AdamW step (step counts from 1) over lists of dense tensors, each
    list of one type: params float32 or bfloat16; grads float32, bfloat16 or
    float16; exp_avg and exp_avg_sq float32, or float8_e4m3fn (m and sqrt(v))
    with scales, a list of (ceil(numel / 256), 2) float32.

    weight_decay: a number, or a list with one for each tensor.  grad_scale: a
    float32 tensor of one element (grad_norm's out[1:]); where it is not finite
    the step changes nothing.  copies: bfloat16 tensors that get the new
    parameters.  seed: round 8-bit moments and bfloat16 parameters
    stochastically by this 32-bit number; None rounds to nearest."""
    n = len(params)
    if n == 0:
        return CUDA_SUCCESS if not len(grads) else CUDA_ERROR_INVALID_VALUE
    pt, gt, st = params[0].dtype, grads[0].dtype if len(grads) else None, exp_avg[0].dtype if len(exp_avg) else None
    if pt not in (torch.float32, torch.bfloat16) or gt not in _FLOATS or st not in (torch.float32, torch.float8_e4m3fn):
        return CUDA_ERROR_INVALID_VALUE
    device = _device()
    sizes = list(map(_numel, params))
    p, g = _list(params, sizes, pt, device), _list(grads, sizes, gt, device)
    m, v = _list(exp_avg, sizes, st, device), _list(exp_avg_sq, sizes, st, device)
    f8 = st is torch.float8_e4m3fn
    if p is None or g is None or m is None or v is None or f8 != (scales is not None):
        return CUDA_ERROR_INVALID_VALUE
    s = c = decays = None
    if f8:
        s = _list(scales, [(k + BLOCK - 1) // BLOCK * 2 for k in sizes], torch.float32, device)
        if s is None:
            return CUDA_ERROR_INVALID_VALUE
    if copies is not None:
        c = _list(copies, sizes, torch.bfloat16, device)
        if c is None:
            return CUDA_ERROR_INVALID_VALUE
    if isinstance(weight_decay, (list, tuple)):
        if len(weight_decay) != n:
            return CUDA_ERROR_INVALID_VALUE
        decays, weight_decay = array.array("f", weight_decay), 0.0
    if grad_scale is not None and (grad_scale.dtype is not torch.float32 or grad_scale.numel() != 1
                                   or grad_scale.get_device() != device):
        return CUDA_ERROR_INVALID_VALUE
    counts = array.array("q", sizes)
    return lib().b3x_train_adamw_gpu(n, _addr(p), _FLOATS[pt], _addr(g), _FLOATS[gt], _addr(m), _addr(v), _addr(s),
                                     _E4M3 if f8 else _F32, _addr(c), _addr(counts), _addr(decays), step, lr, beta1,
                                     beta2, eps, weight_decay,
                                     None if grad_scale is None else grad_scale.data_ptr(), seed is not None,
                                     (seed or 0) & 0xFFFFFFFF, _s(stream, device))
