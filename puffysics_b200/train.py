"""The training operators next to the environment step (libb3train.so,
include/b3x_train.h): log probabilities of actions and their gradient,
advantages, and the AdamW step.

Arguments are torch tensors on the current CUDA device; outputs are tensors of
the caller's that the call fills.  Every call only enqueues on `stream` (the
current stream by default), allocates nothing on the device and returns a
cudaError_t code: 0 success, 1 invalid arguments (types, shapes, strides or
devices that the call does not take), with nothing launched or written.  Memory
given to a call is in use on its stream until the work is done, as with any
kernel: a tensor that another stream made or will free has to be ordered by the
caller.  There is no CPU path: loading fails loudly when a library is missing.

The calls read and write memory and are not part of autograd: outputs carry no
graph and their version counters stay, so a loss made of logprob's outputs gives
the logits no gradient.  Take the derivatives by logp and entropy to
logprob_grad, and its result to backward() (examples/hover_train.py); and do not
let a call overwrite what autograd has saved, which it would not notice.

The checks are made in compiled code (csrc/b3x_train_py.cpp): made in Python
they took as long as a launch.

The header states each operator's formulas and what it does with masked rows,
actions that are none, terminals and lengths.
"""
import ctypes
import importlib.util
import os

import torch

from . import build

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "_lib", "libb3train.so")
PY_PATH = os.path.join(_PKG, "_lib", "b3train_py.so")

CUDA_SUCCESS = 0
CUDA_ERROR_INVALID_VALUE = 1
MAX_TOP = 32             # alternatives a row (B3X_TRAIN_MAX_TOP)
BLOCK = 256              # elements that share a scale of 8-bit moments (B3X_TRAIN_BLOCK)

_lib = _py = None


def lib():
    """The C-ABI library, for callers of its functions by themselves."""
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


def _binding():
    """The compiled functions that the ones below call."""
    global _py
    if _py is None:
        if not os.path.exists(PY_PATH):
            raise RuntimeError("%s is not built; run python -m puffysics_b200.build" % PY_PATH)
        if not build.train_py_current():
            raise RuntimeError("%s is not %s; run python -m puffysics_b200.build" % (PY_PATH, build.built_for()))
        spec = importlib.util.spec_from_file_location("b3train_py", PY_PATH)
        _py = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_py)
    return _py


# the current stream's handle without the object around it, which costs as much as a launch
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _place(stream):
    """The current device, and the handle of a stream (the current one by default)."""
    device = torch.cuda.current_device()
    return device, _raw_stream(device) if stream is None else stream.cuda_stream


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
    return _binding().logprob(logits, actions, logp, entropy, stats, top_ids, top_logp, mask, scale, *_place(stream))


def logprob_grad(logits, stats, grad, actions=None, d_logp=None, entropy=None, d_entropy=None, mask=None, scale=1.0,
                 stream=None):
    """Gradient of sum(d_logp * logp) + sum(d_entropy * entropy) with respect
    to the logits, into grad (their shape and type, rows at any stride; the
    logits themselves to overwrite them), from the stats (and entropy, where
    d_entropy is given) that logprob wrote."""
    return _binding().logprob_grad(logits, stats, grad, actions, d_logp, entropy, d_entropy, mask, scale, *_place(stream))


def advantage(rewards, values, terminals, last_values, advantages, returns=None, gamma=0.99, lam=0.95, lengths=None,
              stream=None):
    """Generalised advantages and returns of a (steps, envs) rollout, any
    strides (pass .t() of arrays with one row per environment).

    rewards, advantages, returns float32; values and last_values (envs,)
    float32, bfloat16 or float16; terminals float32, uint8 or bool; lengths
    (envs,) int32, the steps that each environment has."""
    return _binding().advantage(rewards, values, terminals, last_values, advantages, returns, gamma, lam, lengths,
                                *_place(stream))


def grad_norm_workspace_bytes():
    return lib().b3x_train_grad_norm_workspace_bytes()


def grad_norm(grads, max_norm, out, workspace, stream=None):
    """Global 2-norm of a list of gradients into out[0], and the factor that
    clips them to max_norm into out[1] (out (2,) float32; NaN where the norm is
    not finite).  workspace: a uint8 tensor of grad_norm_workspace_bytes()."""
    return _binding().grad_norm(grads, max_norm, out, workspace, *_place(stream))


def adamw(params, grads, exp_avg, exp_avg_sq, step, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01,
          scales=None, grad_scale=None, copies=None, seed=None, stream=None):
    """One AdamW step (step counts from 1) over lists of dense tensors, each
    list of one type: params float32 or bfloat16; grads float32, bfloat16 or
    float16; exp_avg and exp_avg_sq float32, or float8_e4m3fn (m and sqrt(v))
    with scales, a list of (ceil(numel / 256), 2) float32.

    weight_decay: a number, or a list with one for each tensor.  grad_scale: a
    float32 tensor of one element (grad_norm's out[1:]); where it is not finite
    the step changes nothing.  copies: bfloat16 tensors that get the new
    parameters rounded to nearest (also where bfloat16 parameters themselves are
    rounded stochastically).  seed: round 8-bit moments and bfloat16 parameters
    stochastically by this 32-bit number; None rounds to nearest."""
    return _binding().adamw(params, grads, exp_avg, exp_avg_sq, step, lr, beta1, beta2, eps, weight_decay, scales,
                            grad_scale, copies, seed, *_place(stream))
