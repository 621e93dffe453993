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


def _s(stream):
    return (torch.cuda.current_stream() if stream is None else stream).cuda_stream


def _here(t):
    """Whether a tensor is on the current CUDA device."""
    return t.is_cuda and t.get_device() == torch.cuda.current_device()


def _out(t, shape, dtype=torch.float32):
    """Whether an optional output has this shape and type, dense."""
    return t is None or (t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.is_cuda)


def _p(t):
    return None if t is None else t.data_ptr()


def _rows(logits, actions, mask):
    """The leading arguments of the two calls over rows of logits, or None."""
    if logits.dim() != 2 or logits.dtype not in _FLOATS or not _here(logits):
        return None
    rows, width = logits.shape
    if width > 1 and logits.stride(1) != 1:
        return None
    mask_stride = action_bytes = 0
    if actions is not None:
        action_bytes = 8 if actions.dtype is torch.int64 else 4 if actions.dtype is torch.int32 else 0
        if not action_bytes or actions.shape != (rows,) or not actions.is_contiguous() or not _here(actions):
            return None
    if mask is not None:
        if mask.dtype not in _BYTES or mask.shape != logits.shape or (width > 1 and mask.stride(1) != 1) or not _here(mask):
            return None
        mask_stride = mask.stride(0)
    return (_p(logits), _FLOATS[logits.dtype], rows, width, logits.stride(0), _p(mask), mask_stride, _p(actions),
            action_bytes)


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
    a = _rows(logits, actions, mask)
    if a is None:
        return CUDA_ERROR_INVALID_VALUE
    rows = a[2]
    top = 0
    if top_ids is not None or top_logp is not None:
        if top_ids is None or top_logp is None or top_ids.dim() != 2:
            return CUDA_ERROR_INVALID_VALUE
        top = top_ids.shape[1]
        if not _out(top_ids, (rows, top), torch.int32) or not _out(top_logp, (rows, top)):
            return CUDA_ERROR_INVALID_VALUE
    if not (_out(logp, (rows,)) and _out(entropy, (rows,)) and _out(stats, (rows, 2))):
        return CUDA_ERROR_INVALID_VALUE
    return lib().b3x_train_logprob_gpu(*a, scale, _p(logp), _p(entropy), _p(stats), top, _p(top_ids) if top else None,
                                       _p(top_logp) if top else None, _s(stream))


def logprob_grad(logits, stats, grad, actions=None, d_logp=None, entropy=None, d_entropy=None, mask=None, scale=1.0,
                 stream=None):
    """Gradient of sum(d_logp * logp) + sum(d_entropy * entropy) with respect
    to the logits, into grad (their shape and type, rows at any stride; the
    logits themselves to overwrite them), from the stats (and entropy, where
    d_entropy is given) that logprob wrote."""
    a = _rows(logits, actions, mask)
    if a is None:
        return CUDA_ERROR_INVALID_VALUE
    rows, width = a[2], a[3]
    if (grad.dtype is not logits.dtype or grad.shape != logits.shape or (width > 1 and grad.stride(1) != 1)
            or not _here(grad) or not _out(stats, (rows, 2)) or not _out(entropy, (rows,)) or not _out(d_logp, (rows,))
            or not _out(d_entropy, (rows,))):
        return CUDA_ERROR_INVALID_VALUE
    return lib().b3x_train_logprob_grad_gpu(*a, scale, _p(stats), _p(entropy), _p(d_logp), _p(d_entropy), _p(grad),
                                            grad.stride(0), _s(stream))


def advantage(rewards, values, terminals, last_values, advantages, returns=None, gamma=0.99, lam=0.95, lengths=None,
              stream=None):
    """Generalised advantages and returns of a (steps, envs) rollout, any
    strides (pass .t() of arrays with one row per environment).

    rewards, advantages, returns float32; values and last_values (envs,)
    float32, bfloat16 or float16; terminals float32, uint8 or bool; lengths
    (envs,) int32, the steps that each environment has."""
    shape = rewards.shape
    if (len(shape) != 2 or rewards.dtype is not torch.float32 or values.dtype not in _FLOATS
            or last_values.dtype is not values.dtype or advantages.dtype is not torch.float32
            or (terminals.dtype is not torch.float32 and terminals.dtype not in _BYTES)
            or values.shape != shape or terminals.shape != shape or advantages.shape != shape
            or last_values.shape != shape[1:]
            or not (_here(rewards) and _here(values) and _here(terminals) and _here(last_values) and _here(advantages))):
        return CUDA_ERROR_INVALID_VALUE
    if returns is not None and (returns.dtype is not torch.float32 or returns.shape != shape or not _here(returns)):
        return CUDA_ERROR_INVALID_VALUE
    if lengths is not None and (lengths.dtype is not torch.int32 or lengths.shape != shape[1:]
                                or not lengths.is_contiguous() or not _here(lengths)):
        return CUDA_ERROR_INVALID_VALUE
    strides = (ctypes.c_longlong * 11)(*rewards.stride(), *values.stride(), *terminals.stride(), *last_values.stride(),
                                       *advantages.stride(), *((0, 0) if returns is None else returns.stride()))
    return lib().b3x_train_advantage_gpu(shape[0], shape[1], _p(rewards), _p(values), _FLOATS[values.dtype],
                                         _p(terminals), _F32 if terminals.dtype is torch.float32 else _U8,
                                         _p(last_values), _p(lengths), _p(advantages), _p(returns), strides, gamma, lam,
                                         _s(stream))


def _list(tensors, sizes, dtype):
    """Pointers of a list of dense tensors on the current device, of one type
    and these element counts; None where they are not."""
    if len(tensors) != len(sizes):
        return None
    device = torch.cuda.current_device()
    for t, n in zip(tensors, sizes):
        if t.dtype is not dtype or t.numel() != n or not t.is_contiguous() or t.get_device() != device:
            return None
    return array.array("Q", [t.data_ptr() for t in tensors])


def _addr(a):
    return None if a is None else a.buffer_info()[0]


def grad_norm_workspace_bytes():
    return lib().b3x_train_grad_norm_workspace_bytes()


def grad_norm(grads, max_norm, out, workspace, stream=None):
    """Global 2-norm of a list of gradients into out[0], and the factor that
    clips them to max_norm into out[1] (out (2,) float32; NaN where the norm is
    not finite).  workspace: a uint8 tensor of grad_norm_workspace_bytes()."""
    sizes = array.array("q", [t.numel() for t in grads])
    dtype = grads[0].dtype if grads else torch.float32
    g = _list(grads, sizes, dtype) if dtype in _FLOATS else None
    if (g is None or not _out(out, (2,)) or out is None or not _here(out) or workspace.dtype is not torch.uint8
            or not workspace.is_contiguous() or not _here(workspace)):
        return CUDA_ERROR_INVALID_VALUE
    return lib().b3x_train_grad_norm_gpu(len(grads), _addr(g), _FLOATS[dtype], _addr(sizes), max_norm, _p(out),
                                         _p(workspace), workspace.numel(), _s(stream))


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
    sizes = array.array("q", [t.numel() for t in params])
    p, g = _list(params, sizes, pt), _list(grads, sizes, gt)
    m, v = _list(exp_avg, sizes, st), _list(exp_avg_sq, sizes, st)
    f8 = st is torch.float8_e4m3fn
    if p is None or g is None or m is None or v is None or f8 != (scales is not None):
        return CUDA_ERROR_INVALID_VALUE
    s = c = decays = None
    if f8:
        s = _list(scales, [(k + BLOCK - 1) // BLOCK * 2 for k in sizes], torch.float32)
        if s is None:
            return CUDA_ERROR_INVALID_VALUE
    if copies is not None:
        c = _list(copies, sizes, torch.bfloat16)
        if c is None:
            return CUDA_ERROR_INVALID_VALUE
    if isinstance(weight_decay, (list, tuple)):
        if len(weight_decay) != n:
            return CUDA_ERROR_INVALID_VALUE
        decays, weight_decay = array.array("f", weight_decay), 0.0
    if grad_scale is not None and (grad_scale.dtype is not torch.float32 or grad_scale.numel() != 1
                                   or not _here(grad_scale)):
        return CUDA_ERROR_INVALID_VALUE
    return lib().b3x_train_adamw_gpu(n, _addr(p), _FLOATS[pt], _addr(g), _FLOATS[gt], _addr(m), _addr(v), _addr(s),
                                     _E4M3 if f8 else _F32, _addr(c), _addr(sizes), _addr(decays), step, lr, beta1,
                                     beta2, eps, weight_decay, _p(grad_scale), seed is not None,
                                     (seed or 0) & 0xFFFFFFFF, _s(stream))
