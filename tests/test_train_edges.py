"""The training operators at values where 32-bit arithmetic can go wrong: large
negative fills, scales and eps near the ends of the floats, what is no number.
Tolerances are test_train.py's."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest
import torch

from puffysics_b200 import build, train
from test_train import (DT, E, H, INF, built, check_logprob, grad_oracle, host, make_adam, near, np_decode,  # noqa: F401
                        np_mix, np_pack, terms_of)


# ---- rows with stretches of a large negative value ---------------------------------------------
# (fill, scale): products with the scale whose 32-bit neighbours are whole numbers apart, from 8 to beyond the floats
FILLS = [(-1e7, 1.0), (-1e8, 1.0), (-1e9, 1.0), (-1e9, 1 / 0.6), (-1e9, 2.0), (-2e9, 1 / 1.2), (-2.5e9, 1.0), (-5e9, 1.4),
         (-5e9, 2.0), (-1e10, 0.7), (-1e10, 1.0), (-1e12, 1.0), (-1e12, 1 / 0.6), (-1e20, 1.0), (-1e30, 2.0), (-1e38, 1 / 0.6)]
# (rows, width): a warp a row that walks; a block a row in one turn and in several, few rows and many; clusters
FILLED = [("f32", 1200, 1100), ("bf16", 1200, 2500), ("f32", 40, 4096), ("bf16", 40, 9000), ("bf16", 640, 9000),
          ("f32", 160, 20000), ("bf16", 8, 131072), ("f32", 3, 300001), ("f32", 50, 400), ("bf16", 50, 30)]


def make_filled(rows, width, pad, dtype, fill, seed):
    """Ordinary logits beside stretches of `fill`: the first places, the last, all but one, every other stretch, all."""
    rng = np.random.default_rng(seed)
    z = rng.normal(0, 3, (rows, width))
    for r in range(rows):
        kind = r % 6
        if kind == 0:
            z[r, :(width * 3) // 20 + 1] = fill
        elif kind == 1:
            z[r, width // 2:] = fill
        elif kind == 2:
            z[r] = np.where(np.arange(width) == rng.integers(width), z[r], fill)
        elif kind == 3:
            z[r, (np.arange(width) // 97) % 2 == 0] = fill
        elif kind == 4:
            z[r] = fill
        else:
            z[r, rng.random(width) < 0.9] = fill
    store = torch.full((rows, width + pad), math.nan, dtype=DT[dtype])
    store[:, :width] = torch.from_numpy(z).to(DT[dtype])
    return store


def check_filled(dtype, rows, width, fill, scale, masked, seed):
    store = make_filled(rows, width, seed % 3, dtype, fill, seed)
    rng = np.random.default_rng(seed)
    actions = torch.from_numpy(rng.integers(0, width, rows))
    mask = torch.from_numpy((rng.random((rows, width)) < 0.8).astype(np.uint8)) if masked else None
    dev, act, dmask, out, want = check_logprob(store, width, actions, mask, scale, 0)
    g, h = rng.normal(0, 1, rows).astype(np.float32), rng.normal(0, 1, rows).astype(np.float32)
    grad = torch.full((rows, width), 7.0, device="cuda")
    assert train.logprob_grad(dev[:, :width].float(), out["stats"], grad, actions=act, mask=dmask, scale=scale,
                              d_logp=torch.from_numpy(g).cuda(), entropy=out["entropy"], d_entropy=torch.from_numpy(h).cuda()) == 0
    want_g, size = grad_oracle(store[:, :width].double().numpy(), want, actions.numpy(), mask, scale, g, h)
    n, total = terms_of(width), want["stats"][:, 1:]
    tol = size * E * 2 * (n + 80) * (1 + total) + np.abs(h[:, None]) * scale * np.exp(want["lp"]) * E * (n + 64) * (2 + 2 * total)
    near(grad.cpu().numpy(), want_g, tol * (1 + E) + np.abs(want_g) * E + 2.0 ** -149 + 1e-30)


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype,rows,width", FILLED)
def test_logprob_and_gradient_of_filled_rows(dtype, rows, width, masked):
    """A large negative value in the place of logits that are not allowed is a value like any other: log
    probabilities, entropy and gradient stay those of the formula, whichever threads' places are all filled."""
    some = FILLS if rows * width < 400000 else FILLS[FILLED.index((dtype, rows, width)) % 3 + masked::4]
    for k, (fill, scale) in enumerate(some):
        check_filled(dtype, rows, width, fill, scale, masked, k)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", [(1200, 2500), (40, 9000), (8, 131072)])
def test_logprob_of_filled_rows_in_half_precision(rows, width):
    """The same by the scale: -60,000 at 1e5, logits of some 1e-5 beside it."""
    scale = 1e5
    store = make_filled(rows, width, 1, "f32", -6e9, 1)
    store = (store.double() / scale).to(torch.float16)
    check_logprob(store, width, torch.from_numpy(np.random.default_rng(1).integers(0, width, rows)), None, scale, 0)


# ---- what is no number, far ahead ---------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("order", ["time", "env"])
@pytest.mark.parametrize("steps,envs", [(20, 5), (100, 64), (9000, 3), (4000, 40), (3000, 700), (300, 9000), (65536, 1)])
@pytest.mark.parametrize("gamma,lam", [(0.99, 0.95), (0.9, 0.1), (1.0, 1e-30), (-0.9, 0.1)])
def test_advantage_carries_nan_and_infinity_to_every_earlier_step(steps, envs, order, gamma, lam):
    """What is no number at a step reaches every step before it back to a terminal, however far and in every layout:
    a product of many gamma lam is below the floats, but it is not the 0 of a terminal."""
    def lay(x):
        return x.cuda() if order == "time" else x.t().contiguous().cuda().t()
    r, v, d = (torch.zeros((steps, envs)) for _ in range(3))
    r += 1
    r[steps - 1, 0::3] = math.nan
    r[steps - 1, 1::3] = INF
    cut = steps // 2
    d[cut, 1::3] = 1          # from the step after the terminal on
    adv = lay(torch.full((steps, envs), 7.0))
    assert train.advantage(lay(r), lay(v), lay(d), torch.zeros(envs, device="cuda"), adv, gamma=gamma, lam=lam) == 0
    got = adv.cpu()
    assert torch.isnan(got[:, 0::3]).all()
    assert torch.isinf(got[cut + 1:, 1::3]).all() and torch.isfinite(got[:cut + 1, 1::3]).all()
    assert torch.isfinite(got[:, 2::3]).all()


# ---- eps below the normal floats -----------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("state", ["f32", "f8"])
@pytest.mark.parametrize("eps", [1e-40, 2e-38, 1e-30])
def test_adamw_tiny_eps(eps, state):
    """eps below the normal floats: an element without a gradient stays where it is, one whose squared gradient is
    below the floats takes the formula's step."""
    n = 600
    p0 = np.random.default_rng(0).normal(0, 1, n).astype(np.float32)
    grads = np.zeros(n, np.float32)
    grads[300:400] = 1e-25 if state == "f32" else 0.0
    p, g = torch.from_numpy(p0.copy()).cuda(), torch.from_numpy(grads).cuda()
    kind = torch.float32 if state == "f32" else torch.float8_e4m3fn
    m, v = (torch.zeros(n, device="cuda").to(kind) for _ in range(2))
    sc = [torch.zeros((3, 2), device="cuda")] if state == "f8" else None
    lr = float(np.float32(eps)) * 1e20      # steps of about 1e-5
    assert train.adamw([p], [g], [m], [v], 1, lr, 0.9, 0.95, eps, 0.0, scales=sc) == 0
    mm = (grads * np.float32(1 - 0.9)).astype(np.float64)
    size = lr * (mm / (1 - 0.9)) / float(np.float32(eps))
    near(host(p), p0 - size, E * (4 * np.abs(p0) + 13 * np.abs(size)) + 1e-40)


# ---- scales near the ends of the floats ----------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("scale", [2.0 ** -140, 1e-30, 1e30, 3.0e38])
@pytest.mark.parametrize("dtype,rows,width", [("f32", 9, 5), ("f32", 9, 40), ("bf16", 9, 700), ("f32", 1200, 1100), ("f32", 9, 5000),
                                              ("bf16", 8, 131072)])
def test_logprob_of_any_finite_scale(dtype, rows, width, scale):
    """Scales near both ends of the floats: with 3e38 its product with log2(e) is beyond them.  Equal logits have
    probability 1 / width whatever the scale, and a row's lone largest logit has 1 at a large one."""
    z = torch.zeros((rows, width + 3), dtype=DT[dtype])
    z[1::3, width // 2] = 2.0
    z[2::3] = -1.5
    check_logprob(z, width, torch.full((rows,), width // 2), None, scale, 0)


# ---- views that torch negates lazily -------------------------------------------------------------
@pytest.mark.gpu
def test_lazily_negated_views_are_refused():
    """The imaginary part of a conjugate is a view whose memory holds the values with the other sign."""
    z = torch.view_as_complex(torch.ones((6, 4, 2), device="cuda"))
    neg = z.conj().imag
    assert neg.is_neg() and (neg == -1).all()
    plain, last, adv = torch.ones((6, 4), device="cuda"), torch.zeros(4, device="cuda"), torch.full((6, 4), 7.0, device="cuda")
    for at in range(3):
        args = [plain, plain.clone(), torch.zeros_like(plain)]
        args[at] = neg
        assert train.advantage(*args, last, adv) == 1
    assert train.advantage(plain, plain.clone(), torch.zeros_like(plain), last, neg) == 1
    assert (adv == 7).all() and (neg == -1).all()
    assert train.advantage(neg.resolve_neg(), plain, torch.zeros_like(plain), last, adv) == 0
    torch.cuda.synchronize()


# ---- square roots ------------------------------------------------------------------------------
SQRT = r"""
#include "b3x_train_common.cuh"
__global__ void compare(float up, int* bad) {   // all floats of [1, 4), times a power of 4
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < 1 << 24; i += gridDim.x * blockDim.x) {
        const float x = __uint_as_float(0x3F800000u + i) * up, y = __uint_as_float(0x3F800000u + ((i + 1) & 0xFFFFFF)) * up;
        const float2 r = b3t::unpack2(b3t::sqrt2(b3t::pack2(x, y)));
        if (r.x != sqrtf(x) || r.y != sqrtf(y)) atomicAdd(bad, 1);
    }
}
extern "C" __attribute__((visibility("default"))) int differing(float up, int* bad) {
    compare<<<1024, 256>>>(up, bad);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? (int)e : (int)cudaDeviceSynchronize();
}
"""


@pytest.mark.gpu
def test_square_roots_of_the_moments_are_those_of_sqrtf(tmp_path):
    """Every significand of two octaves, at both ends of the range and in between."""
    src, lib = tmp_path / "sqrt.cu", tmp_path / "libsqrt.so"
    src.write_text(SQRT)
    cmd = ([build.NVCC] + build.ARCH + ["-O3", "-std=c++17"] + build.PARITY
           + ["-Xcompiler", "-fPIC,-fvisibility=hidden", "-shared", "-cudart", "static", "-I" + os.path.join(build.ROOT, "include"),
              "-I" + os.path.join(build.PKG, "csrc"), str(src), "-o", str(lib)])
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr
    f = ctypes.CDLL(str(lib)).differing
    f.argtypes = [ctypes.c_float, ctypes.c_void_p]
    for up in (-96, -50, 0, 40, 98):
        bad = torch.zeros(1, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        assert f(2.0 ** up, bad.data_ptr()) == 0
        assert int(bad) == 0, up


# ---- AdamW: parameters of long lists, copies beside stochastic rounding ------------------------------
def low_bits(index, tensor, step, seed):
    """The 16 random bits that round a bfloat16 parameter, and the 32 of its moments."""
    M = np.uint64(0xFFFFFFFF)
    key = np_mix(np.array([(seed + tensor * 0x9E3779B1 + step * 0x6A09E667) & 0xFFFFFFFF], np.uint64))[0]
    bits = np_mix(((index & M) * np.uint64(0x9E3779B1) + (index >> np.uint64(32)) * np.uint64(0x6A09E667) + key) & M)
    return np_mix((bits + np.uint64(0x9E3779B1)) & M) & np.uint64(0xFFFF), bits


def check_rounded(got, want, tol, low=None):
    """bfloat16 numbers: the 32-bit result, within tol of want, plus its random bits and cut, or rounded to nearest.
    Either way a larger result never gives a smaller number."""
    def rounded(x):
        if low is None:
            return torch.from_numpy(x).float().to(torch.bfloat16).float().numpy()
        return ((x.astype(np.float32).view(np.uint32) + low.astype(np.uint32)) & np.uint32(0xFFFF0000)).view(np.float32)
    bad = np.isnan(want)      # an infinite gradient
    assert np.array_equal(np.isnan(got), bad)
    assert ((rounded(want - tol) <= got) & (got <= rounded(want + tol)) | bad).all()


@pytest.mark.gpu
@pytest.mark.parametrize("param,grad,state,seed", [("f32", "f32", "f32", None), ("f32", "bf16", "f8", 7), ("bf16", "bf16", "f32", 7),
                                                   ("bf16", "bf16", "f8", 7), ("bf16", "f16", "f8", None)])
def test_adamw_parameters_of_millions(param, grad, state, seed):
    """Chunks of several turns: parameters against the formula in 64 bits, from the moments in 32; copies are the
    32-bit results rounded to nearest, also where the parameters are rounded stochastically."""
    sizes, step = [10000001, 37, 300000], 3
    s = make_adam(sizes, param, grad, state, 3)
    before = {k: None if v is None else [host(t).copy() for t in v] for k, v in s.items() if k != "whole"}
    copies = [torch.zeros(n, dtype=torch.bfloat16, device="cuda") for n in sizes]
    decays = [0.1, 0.0, 0.2]
    assert train.adamw(s["params"], s["grads"], s["m"], s["v"], step, weight_decay=decays, scales=s["scales"], copies=copies,
                       seed=seed, **H) == 0
    b1, c1, b2, c2 = (np.float32(x) for x in (0.9, 1 - 0.9, 0.95, 1 - 0.95))
    for k, n in enumerate(sizes):
        g, m, v = before["grads"][k], before["m"][k], before["v"][k]
        if state == "f8":
            sc = before["scales"][k].repeat(256, 0)[:n]
            m, r = np_decode(m) * sc[:, 0], np_decode(v) * sc[:, 1]
            v = r * r
        m, v = (m * b1 + g * c1).astype(np.float64), (v * b2 + (g * g) * c2).astype(np.float64)
        p = before["params"][k].astype(np.float64)
        with np.errstate(invalid="ignore"):
            size = H["lr"] * (m / (1 - 0.9 ** step)) / (np.sqrt(v / (1 - 0.95 ** step)) + H["eps"])
        want = p * (1 - H["lr"] * np.float64(np.float32(decays[k]))) - size
        tol = E * (3 * np.abs(p) + 12 * np.abs(size) + np.abs(want)) + 1e-40
        got = host(s["params"][k])
        check_rounded(host(copies[k]), want, tol)
        if param == "f32":
            near(got, want, tol)
            assert torch.equal(copies[k], s["params"][k].to(torch.bfloat16))
        elif seed is None:
            assert torch.equal(copies[k].view(torch.int16), s["params"][k].view(torch.int16))
        else:
            check_rounded(got, want, tol, low_bits(np.arange(n, dtype=np.uint64), k, step, seed)[0])


@pytest.mark.gpu
def test_adamw_moments_and_parameters_beyond_32_bits():
    """The last elements of a tensor of 2^32 + 700: codes of sqrt(v) bit for bit, parameters by their random bits."""
    n, tail, seed, lr = (1 << 32) + 700, 1000, 11, 1e-2
    p, g = (torch.zeros(n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    sc = torch.zeros(((n + 255) // 256, 2), device="cuda")
    first = (n - tail) // 256 * 256
    g[first:] = torch.from_numpy(np.random.default_rng(0).normal(0, 1, n - first).astype(np.float32)).cuda()
    grads = host(g[first:])
    assert train.adamw([p], [g], [m], [v], 1, lr, scales=[sc], weight_decay=0.0, seed=seed) == 0
    low, bits = low_bits(np.arange(first, n, dtype=np.uint64), 0, 1, seed)
    root = np.sqrt((grads * grads) * np.float32(1 - 0.999))
    cv, sv = np_pack(root, bits >> np.uint64(16))
    cv = np.where((cv == 0) & (root > 0) & (sv.repeat(256)[:len(root)] > 0), 1, cv)
    assert np.array_equal(host(v[first:]), cv) and np.array_equal(host(sc[first // 256:, 1]), sv)
    mm = (grads * np.float32(1 - 0.9)).astype(np.float64)
    want = -lr * (mm / (1 - 0.9)) / (root.astype(np.float64) / math.sqrt(1 - 0.999) + 1e-8)
    check_rounded(host(p[first:]), want, 12 * E * np.abs(want) + 1e-40, low)
