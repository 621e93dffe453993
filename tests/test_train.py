"""The training operators (libb3train.so, puffysics_b200/train.py) against
their formulas in 64 bits.

Tolerances are worked out from the arithmetic, in units of e = 2^-24 (half the
spacing of 32-bit floats at 1): a sum of n terms in partial sums of `terms`
each, joined in a tree, is off by at most (terms + depth) e of the sum of
magnitudes; each elementary operation and each exponential adds a few e of its
result.  What the operators hold in 8 bits is compared bit for bit with the
same operations in numpy's 32 bits.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from puffysics_b200 import build, train

E = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF = math.inf


@pytest.fixture(scope="module", autouse=True)
def built():
    build.build()
    return train.lib()


# ---- logprob -------------------------------------------------------------------------------
PATTERNS = ("random", "equal", "nothing", "one", "lowest", "some lowest", "wide", "rising", "falling", "two values",
            "half -inf", "zeros of both signs")


def make_logits(rows, width, pad, dtype, seed):
    """(rows, width) logits with every pattern in turn, rows at a stride of width + pad, and NaN in between."""
    rng = np.random.default_rng(seed)
    low = torch.finfo(DT[dtype]).min
    z = rng.normal(0, 3, (rows, width))
    for r in range(rows):
        kind = PATTERNS[(r + seed) % len(PATTERNS)]
        if kind == "equal":
            z[r] = 1.5
        elif kind == "nothing":
            z[r] = -INF
        elif kind == "one":
            z[r] = -INF
            z[r, rng.integers(width)] = -2.0
        elif kind == "lowest":
            z[r] = low
        elif kind == "some lowest":
            z[r, rng.random(width) < 0.5] = low
        elif kind == "wide":
            z[r] = rng.normal(0, 3000, width)
        elif kind == "rising":
            z[r] = np.linspace(-20, 20, width)
        elif kind == "falling":
            z[r] = np.linspace(20, -20, width)
        elif kind == "two values":
            z[r] = rng.integers(0, 2, width)
        elif kind == "half -inf":
            z[r, rng.random(width) < 0.5] = -INF
        elif kind == "zeros of both signs":
            z[r] = np.where(rng.random(width) < 0.5, -0.0, 0.0)
    store = torch.full((rows, width + pad), math.nan, dtype=DT[dtype])
    store[:, :width] = torch.from_numpy(z).to(DT[dtype])
    return store


def logprob_oracle(z, actions, mask, scale, top):
    """The definitions, row by row, in 64 bits."""
    z = z.astype(np.float64)
    if mask is not None:
        z = np.where(mask != 0, z, -INF)
    rows, width = z.shape
    out = dict(logp=np.zeros(rows), entropy=np.zeros(rows), stats=np.zeros((rows, 2)), lp=np.full((rows, width), -INF),
               top_ids=np.full((rows, top), -1), top_logp=np.full((rows, top), -INF))
    for r in range(rows):
        m = z[r].max()
        out["stats"][r, 0] = m
        if m > -INF:
            d = (z[r] - m) * scale
            total = np.log(np.exp(d).sum())
            lp = d - total
            out["lp"][r] = lp
            out["stats"][r, 1] = total
            p = np.exp(lp)
            out["entropy"][r] = -(p[p > 0] * lp[p > 0]).sum()
            order = np.lexsort((np.arange(width), -z[r]))[:top]
            order = order[z[r][order] > -INF]
            out["top_ids"][r, :len(order)] = order
            out["top_logp"][r, :len(order)] = lp[order]
        if 0 <= actions[r] < width:
            out["logp"][r] = out["lp"][r, actions[r]]
    return out


def near(got, want, tol):
    got = np.asarray(got, np.float64)
    with np.errstate(over="ignore"):
        want32 = want.astype(np.float32)
    assert not np.isnan(got).any()
    fine = np.isfinite(want32)
    assert np.array_equal(np.isfinite(got), fine)
    assert np.array_equal(got[~fine], want32[~fine])
    off = np.abs(got[fine] - want[fine])
    bad = off > np.broadcast_to(tol, want.shape)[fine]
    assert not bad.any(), (off[bad][:5], np.broadcast_to(tol, want.shape)[fine][bad][:5])


def terms_of(width):
    """Terms of one partial sum: at least 32 partial sums for short rows, 128 and more for long ones."""
    return max(32, width // 128)


def outputs(rows, top):
    f = dict(dtype=torch.float32, device="cuda")
    out = dict(logp=torch.full((rows,), 7.0, **f), entropy=torch.full((rows,), 7.0, **f), stats=torch.full((rows, 2), 7.0, **f))
    if top:
        out["top_ids"] = torch.full((rows, top), 77, dtype=torch.int32, device="cuda")
        out["top_logp"] = torch.full((rows, top), 7.0, **f)
    return out


def check_logprob(store, width, actions, mask, scale, top, stream=None):
    rows = store.shape[0]
    dev = store.cuda()
    out = outputs(rows, top)
    act = actions.cuda()
    dmask = None if mask is None else mask.cuda()
    torch.cuda.synchronize()
    assert train.logprob(dev[:, :width], act, mask=dmask, scale=scale, stream=stream, **out) == 0
    torch.cuda.synchronize()
    want = logprob_oracle(store[:, :width].double().numpy(), actions.numpy(), None if mask is None else mask.numpy(), scale, top)
    got = {k: v.cpu().numpy() for k, v in out.items()}
    n = terms_of(width)
    logp = np.where(np.isfinite(want["logp"]), np.abs(want["logp"]), 0)
    total = want["stats"][:, 1]
    near(got["logp"], want["logp"], E * (n + 64 + 4 * logp))
    # H = log s - t / s: each sum is off by (n + 64) e, t / s by that of log s - H, exponents by e |d|
    near(got["entropy"], want["entropy"], E * (n + 64) * (1 + 2 * total))
    near(got["stats"][:, 0], want["stats"][:, 0], 0.0)
    near(got["stats"][:, 1], total, E * (n + 64 + total))
    if top:
        assert np.array_equal(got["top_ids"], want["top_ids"])
        t = np.where(np.isfinite(want["top_logp"]), np.abs(want["top_logp"]), 0)
        near(got["top_logp"], want["top_logp"], E * (n + 64 + 4 * t))
    return dev, act, dmask, out, want


WIDTHS = [1, 2, 3, 7, 8, 9, 16, 17, 21, 31, 32, 33, 64, 65, 127, 128, 255, 256, 257, 500, 1000, 1023, 1024, 1025, 2047,
          2048, 4096, 4099, 16384, 16391]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("width", WIDTHS)
def test_logprob_against_the_formula(width, dtype):
    k = WIDTHS.index(width)
    rows, pad, top = (24, 13, 37)[k % 3], (0, 1, 8, 5)[k % 4], (20, 1, 32, 0, 5)[k % 5]
    store = make_logits(rows, width, pad, dtype, k)
    rng = np.random.default_rng(k)
    actions = torch.from_numpy(rng.integers(0, width, rows))
    actions[0], actions[1] = -1, width
    if k % 2:
        actions = actions.to(torch.int32)
    check_logprob(store, width, actions, None, 1.0, top)
    mask = torch.from_numpy((rng.random((rows, width)) < 0.7).astype(np.uint8))
    mask[2] = 0
    store[:, :width][mask == 0] = math.nan if k % 2 else 60000.0      # masked places hold anything
    store[3] = torch.where(torch.isnan(store[3]), store[3], torch.full_like(store[3], 2.0))
    check_logprob(store, width, actions, mask if k % 2 else mask.bool(), 0.7, top)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,pad,dtype,top", [
    (1, 131072, 0, "bf16", 20), (3, 131075, 0, "bf16", 32), (12, 50001, 3, "f16", 5), (12, 70001, 0, "f32", 20),
    (150, 50001, 0, "bf16", 1), (700, 9000, 1, "bf16", 20), (1, 600001, 0, "f32", 32), (24, 40000, 0, "bf16", 0)])
def test_logprob_long_rows(rows, width, pad, dtype, top):
    store = make_logits(rows, width, pad, dtype, rows + width)
    check_logprob(store, width, torch.from_numpy(np.random.default_rng(1).integers(0, width, rows)), None, 1.0, top)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,top", [(100003, 3, 3), (40000, 9, 0), (5000, 200, 5)])
def test_logprob_many_rows(rows, width, top):
    store = torch.from_numpy(np.random.default_rng(3).normal(0, 2, (rows, width)).astype(np.float32))
    check_logprob(store, width, torch.from_numpy(np.random.default_rng(1).integers(0, width, rows)), None, 1.0, top)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [5, 300, 5000])
def test_logprob_one_mask_row_for_all_and_one_logit_row_for_all(width):
    rows = 9
    store = make_logits(rows, width, 0, "f32", 4)
    one = torch.from_numpy((np.random.default_rng(2).random(width) < 0.5).astype(np.uint8))
    one[0] = 1
    actions = torch.zeros(rows, dtype=torch.int64)
    dev, out, ref = store.cuda(), outputs(rows, 5), outputs(rows, 5)
    mask = one.cuda()[None].expand(rows, width)
    assert mask.stride(0) == 0
    assert train.logprob(dev, actions.cuda(), mask=mask, **out) == 0
    assert train.logprob(dev, actions.cuda(), mask=mask.contiguous(), **ref) == 0
    assert all(torch.equal(out[k], ref[k]) for k in out)
    same = dev[:1].expand(rows, width)
    assert train.logprob(same, actions.cuda(), **out) == 0
    assert train.logprob(same.contiguous(), actions.cuda(), **ref) == 0
    assert all(torch.equal(out[k], ref[k]) for k in out)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [4, 100, 3001])
def test_logprob_nan_and_infinity(width):
    z = torch.zeros((4, width))
    z[0, 1] = math.nan
    z[1, 2] = INF
    z[2, 0], z[2, 3] = INF, INF
    dev, out = z.cuda(), outputs(4, 2)
    assert train.logprob(dev, torch.zeros(4, dtype=torch.int64, device="cuda"), **out) == 0
    for k in ("logp", "entropy"):
        assert torch.isnan(out[k][:3]).all() and torch.isfinite(out[k][3]), k
    assert torch.isnan(out["stats"][0]).all() and (out["stats"][1:3, 0] == INF).all() and torch.isnan(out["stats"][1:3, 1]).all()
    assert out["top_ids"].tolist() == [[0, 2], [2, 0], [0, 3], [0, 1]]
    grad = torch.full((4, width), 7.0, device="cuda")
    ones = torch.ones(4, device="cuda")
    assert train.logprob_grad(dev, out["stats"], grad, actions=torch.zeros(4, dtype=torch.int64, device="cuda"), d_logp=ones,
                              entropy=out["entropy"], d_entropy=ones) == 0
    assert torch.isnan(grad[:3]).all() and torch.isfinite(grad[3]).all()


@pytest.mark.gpu
def test_logprob_single_outputs_and_no_actions():
    store = make_logits(30, 45, 0, "f32", 0)
    actions = torch.zeros(30, dtype=torch.int64)
    dev, act, _, out, _ = check_logprob(store, 45, actions, None, 1.0, 5)
    for keys in (("logp",), ("entropy",), ("stats",), ("top_ids", "top_logp")):
        one = {k: v for k, v in outputs(30, 5).items() if k in keys}
        assert train.logprob(dev, act if "logp" in keys else None, **one) == 0
        assert all(torch.equal(one[k], out[k]) for k in keys)


def grad_oracle(z, want, actions, mask, scale, g, h):
    lp, rows = want["lp"], len(z)
    p = np.exp(lp)
    got, size = np.zeros_like(lp), np.zeros_like(lp)
    for r in range(rows):
        on = lp[r] > -INF
        a = actions[r]
        gr = g[r] if 0 <= a < z.shape[1] and on[a] else 0.0
        x = np.where(on, lp[r], 0.0)
        got[r] = -p[r] * (gr + h[r] * (np.where(p[r] > 0, x, 0.0) + want["entropy"][r]))
        # the size of what is summed, each off by a few e, and p by (3 |log p| + n) e
        size[r] = p[r] * (abs(gr) + abs(h[r]) * (np.where(p[r] > 0, -x, 0.0) + want["entropy"][r]))
        size[r] *= 3 * np.where(p[r] > 0, -x, 0.0) + 1
        if gr:
            got[r, a] += gr
            size[r, a] += abs(gr)
    return got * scale, size * scale


GRAD = [(33, 1, 0, "f32"), (33, 3, 0, "f32"), (24, 21, 2, "bf16"), (24, 64, 0, "f16"), (24, 257, 0, "bf16"), (24, 1000, 8, "f32"),
        (24, 4099, 1, "f16"), (36, 50001, 7, "bf16"), (24, 16384, 0, "bf16"), (24, 9001, 0, "f32")]


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("rows,width,pad,dtype", GRAD)
def test_logprob_grad_against_the_formula(rows, width, pad, dtype, masked):
    store = make_logits(rows, width, pad, dtype, 5)
    rng = np.random.default_rng(width)
    actions = torch.from_numpy(rng.integers(0, width, rows))
    actions[0], actions[1] = -100, width + 5
    mask = None
    scale = 1.0
    if masked:
        mask = torch.from_numpy((rng.random((rows, width)) < 0.7).astype(np.uint8))
        store[:, :width][mask == 0] = math.nan
        scale = 1.7
    dev, act, dmask, out, want = check_logprob(store, width, actions, mask, scale, 0)
    g, h = rng.normal(0, 1, rows).astype(np.float32), rng.normal(0, 1, rows).astype(np.float32)
    dg, dh = torch.from_numpy(g).cuda(), torch.from_numpy(h).cuda()
    place = torch.full((rows, width + pad + 3), 7.0, dtype=DT[dtype], device="cuda")
    grad = place[:, :width]
    args = dict(actions=act, mask=dmask, scale=scale)
    n = terms_of(width)
    z32, grad32 = dev[:, :width].float(), torch.full((rows, width), 7.0, device="cuda")
    for use_g, use_h in ((True, True), (True, False), (False, True)):
        want_g, size = grad_oracle(store[:, :width].double().numpy(), want, actions.numpy(), mask, scale,
                                   g if use_g else 0 * g, h if use_h else 0 * h)
        more = dict(d_logp=dg if use_g else None, entropy=out["entropy"] if use_h else None, d_entropy=dh if use_h else None, **args)
        assert train.logprob_grad(z32, out["stats"], grad32, **more) == 0
        total = want["stats"][:, 1:]
        # stats and entropy come rounded: their own (n + 64) e go into p and into log p + H
        tol = size * E * 2 * (n + 80) * (1 + total) + np.abs(h[:, None]) * scale * np.exp(want["lp"]) * E * (n + 64) * (2 + 2 * total)
        near(grad32.cpu().numpy(), want_g, tol * (1 + E) + np.abs(want_g) * E + 2.0 ** -149 + 1e-30)
        # the other types: the same values, rounded once
        assert train.logprob_grad(dev[:, :width], out["stats"], grad, **more) == 0
        assert torch.equal(grad, grad32.to(DT[dtype]))
        assert (place[:, width:] == 7).all()
    # over the logits themselves: the same bits
    both = dict(d_logp=dg, entropy=out["entropy"], d_entropy=dh, **args)
    assert train.logprob_grad(dev[:, :width], out["stats"], grad, **both) == 0
    own = dev.clone()
    assert train.logprob_grad(own[:, :width], out["stats"], own[:, :width], **both) == 0
    assert torch.equal(own[:, :width], grad)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [3, 40, 400])
def test_logprob_grad_against_differences(width):
    """Central differences of the operator itself, step d = 2^-6: off by d^2 / 6 of a third derivative (at most 8
    of |g| + |h| (1 + H) for softmax sums) and by rounding, 4 (n + 64) e (1 + log width) / d."""
    rows, d = 6, 2.0 ** -6
    rng = np.random.default_rng(width)
    z = torch.from_numpy(rng.normal(0, 1, (rows, width)).astype(np.float32)).cuda()
    act = torch.from_numpy(rng.integers(0, width, rows)).cuda()
    g, h = (torch.from_numpy(rng.normal(0, 1, rows).astype(np.float32)).cuda() for _ in range(2))

    def value(x, actions, gg, hh):
        out = outputs(len(x), 0)
        assert train.logprob(x, actions, **out) == 0
        return gg.double() * out["logp"].double() + hh.double() * out["entropy"].double(), out
    _, out = value(z, act, g, h)
    grad = torch.empty_like(z)
    assert train.logprob_grad(z, out["stats"], grad, actions=act, d_logp=g, entropy=out["entropy"], d_entropy=h) == 0
    pick = range(width) if width <= 40 else range(0, width, 37)
    tol = (d * d / 6 * 8 + 4 * (64 + 64) * E * (1 + math.log(width)) / d) * (g.abs() + h.abs() * (1 + math.log(width))).double()
    for j in pick:
        step = torch.zeros_like(z)
        step[:, j] = d
        diff = (value(z + step, act, g, h)[0] - value(z - step, act, g, h)[0]) / (2 * d)
        assert ((diff - grad[:, j].double()).abs() <= tol).all(), j


# ---- advantage -----------------------------------------------------------------------------
def advantage_oracle(r, v, d, last, lengths, gamma, lam):
    T, N = r.shape
    adv, ret, tol = np.zeros((T, N)), np.zeros((T, N)), np.zeros((T, N))
    for n in range(N):
        L = T if lengths is None else min(max(int(lengths[n]), 0), T)
        ahead, after, s, k = 0.0, last[n] if L else 0.0, 0.0, 0.0
        for t in range(L - 1, -1, -1):
            on = d[t, n] == 0
            a = gamma * lam if on else 0.0
            delta = r[t, n] + (gamma * after if on else 0.0) - v[t, n]
            size = abs(r[t, n]) + (abs(gamma * after) if on else 0.0) + abs(v[t, n])
            ahead = delta + (a * ahead if on else 0.0)
            # a term k steps ahead has passed k products: off by (k + 8) e of its size
            k = abs(a) * (k + s)
            s = size + abs(a) * s
            adv[t, n], ret[t, n], tol[t, n] = ahead, ahead + v[t, n], 2 * E * (k + 8 * s)
            after = v[t, n]
    return adv, ret, tol


SHAPES = [(1, 1), (1, 37), (2, 1), (5, 3), (17, 33), (64, 40), (65, 31), (128, 7), (300, 130), (513, 2), (1025, 5), (2500, 1), (9000, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["time", "env", "every other"])
@pytest.mark.parametrize("steps,envs", SHAPES)
def test_advantage_against_the_recurrence(steps, envs, order):
    k = SHAPES.index((steps, envs))
    vt = ("f32", "bf16", "f16")[k % 3]
    rng = np.random.default_rng(k)
    r = rng.normal(0, 1, (steps, envs)).astype(np.float32)
    v = torch.from_numpy(rng.normal(5, 2, (steps, envs)).astype(np.float32)).to(DT[vt])
    d = rng.random((steps, envs)) < 0.05
    last = torch.from_numpy(rng.normal(5, 2, envs).astype(np.float32)).to(DT[vt])
    lengths = rng.integers(-1, steps + 2, envs).astype(np.int32) if k % 2 else None

    def lay(x):
        x = x.cuda()
        if order == "time":
            return x.contiguous()
        if order == "env":
            return x.t().contiguous().t()
        big = torch.zeros((2 * x.shape[0] + 1, 3 * x.shape[1] + 2), dtype=x.dtype, device="cuda")
        big[1::2][:, 2::3] = x
        return big[1::2][:, 2::3]
    vo = v.clone()
    ro = r.copy()
    if lengths is not None:     # what lies beyond an environment's end is of no matter
        for n in range(envs):
            L = min(max(int(lengths[n]), 0), steps)
            ro[L:, n], vo[L:, n] = math.nan, math.nan
    dt = torch.from_numpy(d.astype(np.float32)) if k % 4 < 2 else torch.from_numpy(d)
    adv, ret = lay(torch.full((steps, envs), 7.0)), lay(torch.full((steps, envs), 7.0))
    lens = None if lengths is None else torch.from_numpy(lengths).cuda()
    args = [lay(torch.from_numpy(ro)), lay(vo), lay(dt), last.cuda()]
    for gamma, lam in ((0.99, 0.95), (1.0, 1.0), (0.9, 0.0)):
        assert train.advantage(*args, adv, ret, gamma=gamma, lam=lam, lengths=lens) == 0
        g32, a32 = float(np.float32(gamma)), float(np.float32(np.float32(gamma) * np.float32(lam)))
        want_a, want_r, tol = advantage_oracle(r.astype(np.float64), v.double().numpy(), d, last.double().numpy(), lengths, g32, a32 / g32)
        near(adv.cpu().numpy(), want_a, tol)
        near(ret.cpu().numpy(), want_r, tol + E * np.abs(want_r))
    only = lay(torch.full((steps, envs), 7.0))
    assert train.advantage(*args, only, gamma=0.9, lam=0.0, lengths=lens) == 0
    assert torch.equal(only, adv)


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [4, 70, 3000])
def test_advantage_takes_nothing_from_beyond_a_terminal(steps):
    """NaN and infinity after a terminal, in values and in the last value, stay there."""
    r = torch.ones((steps, 6), device="cuda")
    v = torch.full((steps, 6), 2.0, device="cuda")
    d = torch.zeros((steps, 6), device="cuda")
    last = torch.tensor([math.nan, INF, 1.0, 1.0, 1.0, 1.0], device="cuda")
    d[steps - 1, :2] = 1
    cut = steps // 2
    v[cut, 2], r[cut, 3], v[cut, 4] = math.nan, INF, -INF
    d[cut - 1, 2:5] = 1
    adv = torch.empty((steps, 6), device="cuda")
    assert train.advantage(r, v, d, last, adv, gamma=0.9, lam=0.9) == 0
    assert torch.isfinite(adv[:, :2]).all() and torch.isfinite(adv[:, 5]).all()
    assert torch.isfinite(adv[:cut, 2:5]).all()
    assert torch.isnan(adv[cut, 2]) and adv[cut, 3] == INF and adv[cut, 4] == INF


# ---- adamw ---------------------------------------------------------------------------------
SIZES = [1, 3, 255, 256, 257, 2048, 2049, 5000, 70000, 0, 128]
H = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8)


def np_mix(x):
    M = np.uint64(0xFFFFFFFF)
    x = x ^ (x >> np.uint64(16))
    x = (x * np.uint64(0x85A308D3)) & M
    x = x ^ (x >> np.uint64(13))
    x = (x * np.uint64(0x243F6A89)) & M
    return x ^ (x >> np.uint64(16))


def np_hash(n, tensor, step, seed):
    M = 0xFFFFFFFF
    key = np_mix(np.array([(seed + tensor * 0x9E3779B1 + step * 0x6A09E667) & M], np.uint64))[0]
    return np_mix((np.arange(n, dtype=np.uint64) * np.uint64(0x9E3779B1) + key) & np.uint64(M))


def np_decode(codes):
    c = codes.astype(np.uint32)
    y = ((c & 0x7F) << 20).view(np.float32) * np.float32(2.0 ** 120)
    return np.where(c & 0x80, -y, y)


def np_pack(x, bits):
    """e4m3 codes and scales of the formula, in 32 bits."""
    n = len(x)
    b = np.pad(x, (0, -n % 256)).reshape(-1, 256)
    most = np.abs(b).max(1)
    ok = most >= np.float32(2.0 ** -100)
    with np.errstate(divide="ignore"):
        scale = np.where(ok, most / np.float32(448), np.float32(0))
        inverse = np.where(ok, np.float32(448) / most, np.float32(0))
    y = (b * inverse[:, None]).reshape(-1)[:n].astype(np.float32)
    w = (np.abs(y) * np.float32(2.0 ** -120)).view(np.uint32)
    w = w + ((bits.astype(np.uint32) << 4 | 8) if bits is not None else 0x7FFFF + ((w >> 20) & 1)).astype(np.uint32)
    c = np.minimum(w >> 20, 0x7E)
    return np.where(y < 0, c | 0x80, c).astype(np.uint8), scale.astype(np.float32)


def make_adam(sizes, param, grad, state, seed, offset=0):
    """Lists of tensors, `offset` elements into larger ones."""
    rng = np.random.default_rng(seed)

    def put(x, dtype):
        t = torch.full((len(x) + offset + 4,), 9.0, dtype=torch.float32).to(dtype).cuda()
        t[offset:offset + len(x)] = torch.from_numpy(x).to(dtype).cuda() if dtype is not torch.uint8 else torch.from_numpy(x).cuda()
        s["whole"].append(t)
        return t[offset:offset + len(x)]
    s = dict(params=[], grads=[], m=[], v=[], scales=[] if state == "f8" else None, whole=[])
    for n in sizes:
        s["params"].append(put(rng.normal(0, 1, n).astype(np.float32), DT[param]))
        s["grads"].append(put((rng.normal(0, 1, n) * np.exp(rng.normal(0, 2, n))).astype(np.float32), DT[grad]))
        m = (rng.normal(0, 0.1, n) * np.exp(rng.normal(0, 1, n))).astype(np.float32)
        v = ((rng.normal(0, 1, n) * np.exp(rng.normal(0, 2, n))) ** 2).astype(np.float32)
        if n > 600:
            m[256:512] = 0
            v[256:512] = 0
            s["grads"][-1][256:512] = 0     # a block that has seen no gradient
        if state == "f32":
            s["m"].append(put(m, torch.float32))
            s["v"].append(put(v, torch.float32))
        else:
            (cm, sm), (cv, sv) = np_pack(m, None), np_pack(np.sqrt(v), None)
            s["m"].append(put(cm, torch.uint8).view(torch.float8_e4m3fn))
            s["v"].append(put(cv, torch.uint8).view(torch.float8_e4m3fn))
            s["scales"].append(torch.from_numpy(np.stack((sm, sv), 1)).cuda())
    return s


def host(t):
    return t.view(torch.uint8).cpu().numpy() if t.dtype is torch.float8_e4m3fn else t.float().cpu().numpy()


ADAM = [("f32", "f32", "f32"), ("f32", "bf16", "f32"), ("bf16", "bf16", "f32"), ("bf16", "f16", "f32"), ("f32", "f32", "f8"),
        ("f32", "f16", "f8"), ("bf16", "bf16", "f8"), ("bf16", "f32", "f8")]


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("seed", [None, 99])
@pytest.mark.parametrize("param,grad,state", ADAM)
def test_adamw_against_the_formula(param, grad, state, seed, offset):
    """m and v in 32 bits (and the codes and scales of 8-bit moments, bit for bit), the parameters in 64 bits: off by
    e for each of p's two operations and by a few e of the step taken, then by its own rounding."""
    s = make_adam(SIZES, param, grad, state, 1, offset)
    before = {k: None if v is None else [host(t).copy() for t in v] for k, v in s.items()}
    copies = [torch.zeros(n, dtype=torch.bfloat16, device="cuda") for n in SIZES]
    decays = [0.1 * (k % 3) for k in range(len(SIZES))]
    gs = torch.tensor([3.0, 0.37], device="cuda")
    step = 3
    if param == "bf16":
        s["wide"] = [t.float() for t in s["params"]]
        other = [[t.clone() for t in s[x]] if s[x] is not None else None for x in ("m", "v", "scales")]
        assert train.adamw(s["wide"], s["grads"], other[0], other[1], step, weight_decay=decays, scales=other[2],
                           grad_scale=gs[1:], seed=seed, **H) == 0
    assert train.adamw(s["params"], s["grads"], s["m"], s["v"], step, weight_decay=decays, scales=s["scales"],
                       grad_scale=gs[1:], copies=copies, seed=seed, **H) == 0
    b1, c1, b2, c2 = (np.float32(x) for x in (0.9, 1 - 0.9, 0.95, 1 - 0.95))
    for k, n in enumerate(SIZES):
        g = before["grads"][k] * np.float32(0.37)
        if state == "f32":
            m, v = before["m"][k], before["v"][k]
        else:
            sc = before["scales"][k].repeat(256, 0)[:n]
            m, r = np_decode(before["m"][k]) * sc[:, 0], np_decode(before["v"][k]) * sc[:, 1]
            v = r * r
        m = m * b1 + g * c1
        v = v * b2 + (g * g) * c2
        root = np.sqrt(v)
        assert m.dtype == v.dtype == np.float32
        if state == "f32":
            assert np.array_equal(host(s["m"][k]), m) and np.array_equal(host(s["v"][k]), v)
        else:
            bits = np_hash(n, k, step, seed) if seed is not None else None
            cm, sm = np_pack(m, None if bits is None else bits & np.uint64(0xFFFF))
            cv, sv = np_pack(root, None if bits is None else bits >> np.uint64(16))
            cv = np.where((cv == 0) & (root > 0) & (sv.repeat(256)[:n] > 0), 1, cv)
            assert np.array_equal(host(s["scales"][k]), np.stack((sm, sv), 1))
            assert np.array_equal(host(s["m"][k]), cm) and np.array_equal(host(s["v"][k]), cv)
        m, v, p = m.astype(np.float64), v.astype(np.float64), before["params"][k].astype(np.float64)
        step_size = H["lr"] * (m / (1 - 0.9 ** step)) / (np.sqrt(v / (1 - 0.95 ** step)) + H["eps"])
        want = p * (1 - H["lr"] * np.float64(np.float32(decays[k]))) - step_size
        tol = E * (3 * np.abs(p) + 12 * np.abs(step_size) + np.abs(want)) + 1e-40
        if param == "f32":
            near(host(s["params"][k]), want, tol)
            assert torch.equal(copies[k], s["params"][k].to(torch.bfloat16))
            continue
        # bf16 parameters: what 32-bit ones would be, rounded
        wide = s["wide"][k]
        near(host(wide), want, tol)
        assert torch.equal(copies[k], wide.to(torch.bfloat16))
        if seed is None:
            assert torch.equal(s["params"][k], copies[k])
        else:
            low = np_mix((np_hash(n, k, step, seed) + np.uint64(0x9E3779B1)) & np.uint64(0xFFFFFFFF)) & np.uint64(0xFFFF)
            x = (host(wide).view(np.uint32) + low.astype(np.uint32)) & np.uint32(0xFFFF0000)
            assert np.array_equal(host(s["params"][k]), x.view(np.float32))
    for t in s["whole"]:       # nothing beside a tensor is written
        assert (t[:offset] == 9).all() and (t[-4:] == 9).all()


@pytest.mark.gpu
def test_adamw_many_tensors_and_plain_arguments():
    """More tensors than one launch takes, no decay list, copies or scale."""
    sizes = [int(x) for x in np.random.default_rng(0).integers(1, 3000, 700)]
    s = make_adam(sizes, "f32", "f32", "f32", 2)
    p0, g, m0, v0 = ([host(t).copy() for t in s[k]] for k in ("params", "grads", "m", "v"))
    assert train.adamw(s["params"], s["grads"], s["m"], s["v"], 1, weight_decay=0.0, **H) == 0
    for k in range(len(sizes)):
        m = m0[k] * np.float32(0.9) + g[k] * np.float32(1 - 0.9)
        v = v0[k] * np.float32(0.95) + (g[k] * g[k]) * np.float32(1 - 0.95)
        assert np.array_equal(host(s["m"][k]), m) and np.array_equal(host(s["v"][k]), v)
        size = H["lr"] * (m.astype(np.float64) / (1 - 0.9)) / (np.sqrt(v.astype(np.float64) / (1 - 0.95)) + H["eps"])
        near(host(s["params"][k]), p0[k].astype(np.float64) - size, E * (4 * np.abs(p0[k]) + 13 * np.abs(size)))


@pytest.mark.gpu
def test_adamw_stochastic_rounding_has_no_bias():
    """The mean of many roundings of one value: 2^16 elements, each rounding spread over one spacing d at most, so
    the mean is within 5 d / sqrt(12 * 65536) of the value but for chance of 1e-6 (d / 2 for a value midway)."""
    n = 1 << 16
    p = torch.full((n,), 1.0 + 2.0 ** -9 + 2.0 ** -10, dtype=torch.bfloat16, device="cuda")
    p.fill_(1.0)
    zero = [torch.zeros(n, device="cuda") for _ in range(3)]
    # p (1 - lr decay) with lr decay = -3/8 of the spacing 2^-7 above 1
    assert train.adamw([p], zero[:1], zero[1:2], zero[2:], 1, lr=1.0, weight_decay=-0.375 * 2.0 ** -7, seed=5) == 0
    assert set(p.unique().tolist()) == {1.0, 1.0 + 2.0 ** -7}
    assert abs(float(p.double().mean()) - (1 + 0.375 * 2.0 ** -7)) < 5 * 0.5 * 2.0 ** -7 / math.sqrt(n)
    again, other = torch.ones_like(p), torch.ones_like(p)
    assert train.adamw([again], zero[:1], zero[1:2], zero[2:], 1, lr=1.0, weight_decay=-0.375 * 2.0 ** -7, seed=5) == 0
    assert train.adamw([other], zero[:1], zero[1:2], zero[2:], 2, lr=1.0, weight_decay=-0.375 * 2.0 ** -7, seed=5) == 0
    assert torch.equal(again, p) and not torch.equal(other, p)


@pytest.mark.gpu
def test_adamw_eight_bit_moments_follow_a_decaying_average():
    """1000 steps of beta2 = 0.999, each block's largest element kept in place by its gradient and the others without
    one: rounded to nearest a code could never leave its place; rounded stochastically the mean of sqrt(v) falls by
    0.999^500.  A step moves a code by 0.0005 r of its spacing d = 8, a variance of at most 0.0005 r d; 1000 of them
    leave the mean of 65280 elements with a deviation of 0.08, 0.13% of the 63 that are expected: within 1%."""
    n = 1 << 16
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    m = torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    v = torch.full((n,), 100.0, device="cuda").to(torch.float8_e4m3fn)
    v.view(torch.uint8)[::256] = 0x7E       # one large element a block holds the scale
    g[::256] = 448.0
    sc = torch.ones((n // 256, 2), device="cuda")
    for t in range(1, 1001):
        assert train.adamw([p], [g], [m], [v], t, 1e-3, beta2=0.999, scales=[sc], seed=3) == 0
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[::256] = False
    r = v.double() * sc[:, 1].double().repeat_interleave(256)
    start = float(torch.tensor(100.0).to(torch.float8_e4m3fn).double())
    assert abs(float(r[keep].mean()) / (start * 0.999 ** 500) - 1) < 0.01


@pytest.mark.gpu
@pytest.mark.parametrize("grad", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("sizes", [[], [0], [1], SIZES, [100000] * 3, [7] * 700])
def test_grad_norm(grad, sizes):
    rng = np.random.default_rng(1)
    store = [torch.from_numpy(rng.normal(0, 1, n + 1).astype(np.float32)).to(DT[grad]).cuda() for n in sizes]
    grads = [t[k % 2:k % 2 + n] for k, (t, n) in enumerate(zip(store, sizes))]
    want = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
    ws = torch.full((train.grad_norm_workspace_bytes(),), 255, dtype=torch.uint8, device="cuda")
    out = torch.full((2,), 7.0, device="cuda")
    for limit in (0.5, 1e9, INF):
        assert train.grad_norm(grads, limit, out, ws) == 0
        norm, factor = out.tolist()
        assert abs(norm - want) <= 2 * E * want
        assert abs(factor - min(1.0, limit / (want + 1e-6))) <= 6 * E
    if sum(sizes) > 5:
        grads[-1][0] = INF
        assert train.grad_norm(grads, 1.0, out, ws) == 0
        assert out[0] == INF and torch.isnan(out[1])
        s = make_adam([300], "f32", "f32", "f32", 1)
        old = [t.clone() for k in ("params", "m", "v") for t in s[k]]
        assert train.adamw(s["params"], s["grads"], s["m"], s["v"], 1, grad_scale=out[1:], **H) == 0
        assert all(torch.equal(a, b) for a, b in zip(old, [t for k in ("params", "m", "v") for t in s[k]]))


@pytest.mark.gpu
def test_grad_norm_of_large_and_small_gradients():
    """Squares beyond 32 bits' range do not overflow or vanish."""
    ws = torch.empty(train.grad_norm_workspace_bytes(), dtype=torch.uint8, device="cuda")
    out = torch.empty(2, device="cuda")
    for x in (1e30, 1e-30):
        assert train.grad_norm([torch.full((1000,), x, device="cuda")], 1.0, out, ws) == 0
        assert abs(float(out[0]) / (x * math.sqrt(1000)) - 1) < 1e-6


# ---- all -----------------------------------------------------------------------------------
@pytest.mark.gpu
def test_same_bits_again_and_on_another_stream():
    z = make_logits(40, 20001, 0, "bf16", 3).cuda()
    act = torch.arange(40, device="cuda")
    T, N = 3000, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    r, v, last = torch.randn((T, N), generator=g, device="cuda"), torch.randn((T, N), generator=g, device="cuda"), torch.randn(N, generator=g, device="cuda")
    d = (torch.rand((T, N), generator=g, device="cuda") < 0.02).float()
    grads = [torch.randn(n, generator=g, device="cuda") for n in (5, 100000, 33)]
    got = []
    for k in range(3):
        stream = torch.cuda.Stream() if k else torch.cuda.current_stream()
        out = outputs(40, 20)
        more = dict(grad=torch.empty_like(z), adv=torch.empty_like(r), norm=torch.empty(2, device="cuda"),
                    ws=torch.empty(train.grad_norm_workspace_bytes(), dtype=torch.uint8, device="cuda"))
        ones = torch.ones(40, device="cuda")
        torch.cuda.synchronize()
        assert train.logprob(z, act, stream=stream, **out) == 0
        assert train.logprob_grad(z, out["stats"], more["grad"], actions=act, d_logp=ones, entropy=out["entropy"],
                                  d_entropy=ones, stream=stream) == 0
        assert train.advantage(r, v, d, last, more["adv"], stream=stream) == 0
        assert train.grad_norm(grads, 1.0, more["norm"], more["ws"], stream=stream) == 0
        stream.synchronize()
        got.append([t.cpu() for t in (*out.values(), more["grad"], more["adv"], more["norm"])])
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
def test_refusals_write_nothing():
    f = dict(device="cuda")
    z, act = torch.zeros((4, 6), **f), torch.zeros(4, dtype=torch.int64, **f)
    out = outputs(4, 3)
    bad = [dict(logits=z.double()), dict(logits=z[0]), dict(logits=z.t()), dict(actions=act[:3]), dict(actions=act.float()),
           dict(actions=None), dict(mask=torch.ones((4, 5), dtype=torch.uint8, **f)), dict(mask=torch.ones((4, 6), **f)),
           dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=INF), dict(logp=torch.zeros(5, **f)),
           dict(logp=torch.zeros(4, dtype=torch.float64, **f)), dict(entropy=torch.zeros(8, **f)[::2]), dict(stats=torch.zeros((4, 3), **f)),
           dict(top_ids=None), dict(top_logp=None), dict(top_ids=torch.zeros((4, 3), dtype=torch.int64, **f)),
           dict(top_ids=torch.zeros((4, 33), dtype=torch.int32, **f), top_logp=torch.zeros((4, 33), **f)),
           dict(logits=z.cpu()), dict(actions=act.cpu()), dict(logits=torch.zeros((4, 0), **f)),
           dict(logits=z, logp=None, entropy=None, stats=None, top_ids=None, top_logp=None)]
    for change in bad:
        args = dict(logits=z, actions=act, **out)
        args.update(change)
        assert train.logprob(**args) == 1, change.keys()
    grad, ones = torch.full((4, 6), 7.0, **f), torch.ones(4, **f)
    good = dict(logits=z, stats=out["stats"], grad=grad, actions=act, d_logp=ones, entropy=ones, d_entropy=ones)
    for change in (dict(grad=grad.half()), dict(grad=grad[:3]), dict(grad=grad[:1].expand(4, 6)), dict(actions=None), dict(entropy=None),
                   dict(d_logp=ones[:2]), dict(stats=ones), dict(logits=z.half()), dict(scale=0.0), dict(grad=torch.zeros((6, 4), **f).t())):
        assert train.logprob_grad(**dict(good, **change)) == 1, change.keys()
    r = torch.zeros((5, 3), **f)
    adv = torch.full((5, 3), 7.0, **f)
    good = dict(rewards=r, values=r.clone(), terminals=r.clone(), last_values=torch.zeros(3, **f), advantages=adv)
    for change in (dict(rewards=r.double()), dict(values=r[:4]), dict(values=r.bfloat16()), dict(terminals=r.half()), dict(terminals=r.int()),
                   dict(last_values=torch.zeros(5, **f)), dict(advantages=adv[:, :1].expand(5, 3)), dict(advantages=r), dict(returns=adv),
                   dict(lengths=torch.zeros(3, dtype=torch.int64, **f)), dict(lengths=torch.zeros(5, dtype=torch.int32, **f)),
                   dict(gamma=math.nan), dict(lam=INF), dict(rewards=r.cpu())):
        assert train.advantage(**dict(good, **change)) == 1, change.keys()
    s = make_adam([10, 20], "f32", "f32", "f32", 1)
    t = make_adam([10, 20], "f32", "f32", "f8", 1)
    old = [x.clone() for x in s["params"]]
    good = dict(params=s["params"], grads=s["grads"], exp_avg=s["m"], exp_avg_sq=s["v"], step=1, lr=0.1)
    for change in (dict(params=[x.half() for x in s["params"]]), dict(grads=s["grads"][:1]), dict(grads=[s["grads"][0], s["grads"][1].half()]),
                   dict(grads=[s["grads"][0], s["grads"][1][:5]]), dict(exp_avg=t["m"]), dict(exp_avg=t["m"], exp_avg_sq=t["v"]),
                   dict(scales=t["scales"]), dict(exp_avg=t["m"], exp_avg_sq=t["v"], scales=t["scales"][:1]), dict(step=0), dict(lr=math.nan),
                   dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0), dict(eps=INF), dict(weight_decay=INF), dict(weight_decay=[0.1]),
                   dict(grad_scale=torch.zeros(2, **f)), dict(copies=[torch.zeros(10, **f), torch.zeros(20, **f)]), dict(grads=[]),
                   dict(params=[torch.zeros((5, 4), **f).t(), s["params"][1]]), dict(grads=[x.cpu() for x in s["grads"]])):
        assert train.adamw(**dict(good, **change)) == 1, change.keys()
    ws, n2 = torch.zeros(train.grad_norm_workspace_bytes(), dtype=torch.uint8, **f), torch.full((2,), 7.0, **f)
    for a in ((s["grads"], 0.0, n2, ws), (s["grads"], -1.0, n2, ws), (s["grads"], math.nan, n2, ws), (s["grads"], 1.0, n2, ws[:-1]),
              (s["grads"], 1.0, n2, ws.float()), (s["grads"], 1.0, n2[:1], ws), ([x.double() for x in s["grads"]], 1.0, n2, ws)):
        assert train.grad_norm(*a) == 1
    torch.cuda.synchronize()
    assert all((out[k] == (77 if k == "top_ids" else 7)).all() for k in out)
    assert (grad == 7).all() and (adv == 7).all() and (n2 == 7).all() and all(torch.equal(a, b) for a, b in zip(old, s["params"]))


@pytest.mark.gpu
def test_nothing_to_do_succeeds():
    f = dict(device="cuda")
    assert train.logprob(torch.zeros((0, 5), **f), logp=torch.zeros(0, **f), actions=torch.zeros(0, dtype=torch.int64, **f)) == 0
    assert train.logprob_grad(torch.zeros((0, 5), **f), torch.zeros((0, 2), **f), torch.zeros((0, 5), **f)) == 0
    for shape in ((0, 4), (4, 0)):
        e = torch.zeros(shape, **f)
        assert train.advantage(e, e, e, torch.zeros(shape[1], **f), e) == 0
    assert train.adamw([], [], [], [], 1, 0.1) == 0
    z = torch.zeros(0, **f)
    assert train.adamw([z], [z], [z], [z], 1, 0.1) == 0


def test_exports_and_argument_checks_need_no_device(built):
    L = built
    n, one = None, ctypes.c_void_p(64)
    assert L.b3x_train_grad_norm_workspace_bytes() % 8 == 0
    # rows == 0 succeeds without pointers; everything else wrong is refused before a launch
    assert L.b3x_train_logprob_gpu(n, 0, 0, 5, 5, n, 0, n, 0, 1.0, n, n, n, 0, n, n, n) == 0
    ok = [one, 0, 2, 5, 5, n, 0, one, 8, 1.0, one, n, n, 0, n, n, n]
    for at, bad in ((0, n), (0, ctypes.c_void_p(66)), (1, 3), (1, -1), (2, -1), (3, 0), (3, 1 << 31), (4, -5), (8, 2), (9, 0.0),
                    (7, ctypes.c_void_p(68)), (7, n), (10, ctypes.c_void_p(66)), (10, n), (13, 33), (13, -1), (13, 1)):
        args = list(ok)
        args[at] = bad
        assert L.b3x_train_logprob_gpu(*args) == 1, at
    ok = [one, 0, 2, 5, 5, n, 0, one, 8, 1.0, one, one, one, one, one, 5, n]
    for at, bad in ((0, n), (10, n), (11, n), (14, n), (15, 4), (15, 6), (14, ctypes.c_void_p(66)), (7, n)):
        args = list(ok)
        args[at] = bad
        assert L.b3x_train_logprob_grad_gpu(*args) == 1, at
    two = ctypes.c_void_p(4096)
    st = (ctypes.c_longlong * 11)(3, 1, 3, 1, 3, 1, 1, 3, 1, 3, 1)
    ok = [5, 3, one, one, 0, one, 0, one, n, two, n, st, 0.9, 0.9, n]
    for at, bad in ((0, -1), (1, -1), (2, n), (3, n), (4, 3), (5, n), (6, 1), (7, n), (9, n), (9, one), (10, two), (11, n),
                    (11, (ctypes.c_longlong * 11)(3, 1, 3, 1, 3, 1, 1, 2, 1, 3, 1)), (11, (ctypes.c_longlong * 11)(-3, 1, 3, 1, 3, 1, 1, 3, 1, 3, 1)),
                    (12, math.nan), (13, INF)):
        args = list(ok)
        args[at] = bad
        assert L.b3x_train_advantage_gpu(*args) == 1, at
    assert L.b3x_train_advantage_gpu(0, 3, n, n, 0, n, 0, n, n, n, n, n, 0.9, 0.9, n) == 0
    ptr, sizes = (ctypes.c_void_p * 1)(64), (ctypes.c_longlong * 1)(10)
    none, neg = (ctypes.c_void_p * 1)(0), (ctypes.c_longlong * 1)(-1)
    ok = [1, ptr, 0, ptr, 0, ptr, ptr, n, 0, n, sizes, n, 1, 0.1, 0.9, 0.99, 1e-8, 0.0, n, 0, 0, n]
    for at, bad in ((0, -1), (1, n), (1, none), (2, 2), (3, none), (4, 3), (5, none), (6, n), (8, 3), (8, 1), (9, (ctypes.c_void_p * 1)(65)),
                    (10, neg), (10, n), (12, 0), (13, math.inf), (14, 1.0), (15, 1.0), (16, -1.0), (17, math.nan), (18, ctypes.c_void_p(66))):
        args = list(ok)
        args[at] = bad
        assert L.b3x_train_adamw_gpu(*args) == 1, at
    assert L.b3x_train_adamw_gpu(0, n, 0, n, 0, n, n, n, 0, n, n, n, 1, 0.1, 0.9, 0.99, 1e-8, 0.0, n, 0, 0, n) == 0
    for args in ((1, ptr, 0, sizes, 0.0, one, one, 1 << 20, n), (1, none, 0, sizes, 1.0, one, one, 1 << 20, n), (1, ptr, 0, sizes, 1.0, n, one, 1 << 20, n),
                 (1, ptr, 0, sizes, 1.0, one, one, 8, n), (1, ptr, 3, sizes, 1.0, one, one, 1 << 20, n), (1, ptr, 0, neg, 1.0, one, one, 1 << 20, n)):
        assert L.b3x_train_grad_norm_gpu(*args) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("eight_bit", [False, True])
def test_hover_training_learns(eight_bit):
    """The example's loop: a policy that began at random holds its height far better after 40 iterations (a step's
    reward is at most 1, and 0 at two metres' error)."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "hover_train.py")
    spec = importlib.util.spec_from_file_location("hover_train", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    got = module.run(envs=1024, iterations=40, eight_bit=eight_bit)
    assert all(math.isfinite(x) for x in got)
    assert sum(got[-4:]) / 4 > sum(got[1:8]) / 7 + 0.3, got


# ---- more rows, longer lists, larger offsets -------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("rows,width,pad,dtype,top", [
    (1300, 700, 1, "f32", 20), (1300, 2500, 0, "bf16", 32), (1200, 5001, 2, "f16", 5), (1200, 1100, 0, "bf16", 0),
    (700, 3000, 0, "bf16", 20), (700, 1500, 3, "f32", 1)])
def test_logprob_more_rows_than_blocks(rows, width, pad, dtype, top, masked):
    store = make_logits(rows, width, pad, dtype, width)
    rng = np.random.default_rng(rows)
    mask = torch.from_numpy((rng.random((rows, width)) < 0.6).astype(np.uint8)) if masked else None
    check_logprob(store, width, torch.from_numpy(rng.integers(0, width, rows)), mask, 1.3, top)


@pytest.mark.gpu
def test_logprob_offsets_beyond_32_bits():
    """Rows 1.5e9 elements apart: the last one begins beyond 2^31 elements."""
    stride, width = 1500000000, 1003
    store = torch.empty(2 * stride + width, dtype=torch.bfloat16, device="cuda")
    z = torch.as_strided(store, (3, width), (stride, 1))
    z.copy_(torch.from_numpy(np.random.default_rng(0).normal(0, 2, (3, width))))
    out, ref = outputs(3, 20), outputs(3, 20)
    act = torch.tensor([0, 5, 1002], device="cuda")
    dense = z.contiguous()
    for a, o in ((z, out), (dense, ref)):
        assert train.logprob(a, act, **o) == 0
    for k in out:
        if k in ("top_ids",):
            assert torch.equal(out[k], ref[k])
        else:
            assert (out[k] - ref[k]).abs().max() <= 64 * E * (1 + ref[k].abs().max())
    ones = torch.ones(3, device="cuda")
    want = torch.empty_like(dense)
    assert train.logprob_grad(dense, out["stats"], want, actions=act, d_logp=ones, entropy=out["entropy"], d_entropy=ones) == 0
    assert train.logprob_grad(z, out["stats"], z, actions=act, d_logp=ones, entropy=out["entropy"], d_entropy=ones) == 0
    assert torch.equal(z, want)


def advantage_many(r, v, d, last, gamma, lam):
    """advantage_oracle for all environments at once, all of full length."""
    T, N = r.shape
    adv, tol = np.zeros((T, N)), np.zeros((T, N))
    ahead, after, s, k = np.zeros(N), last, np.zeros(N), np.zeros(N)
    for t in range(T - 1, -1, -1):
        on = d[t] == 0
        a = np.where(on, gamma * lam, 0.0)
        ahead = r[t] + np.where(on, gamma * after, 0.0) - v[t] + a * ahead
        k = a * (k + s)
        s = np.abs(r[t]) + np.where(on, np.abs(gamma * after), 0.0) + np.abs(v[t]) + a * s
        adv[t], tol[t], after = ahead, 2 * E * (k + 8 * s), v[t]
    return adv, tol


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["time", "env"])
@pytest.mark.parametrize("steps,envs", [(64, 4096), (300, 5000), (127, 20001), (3, 70000), (2000, 700)])
def test_advantage_of_many_environments(steps, envs, order):
    rng = np.random.default_rng(steps)
    r, v = (rng.normal(0, 1, (steps, envs)).astype(np.float32) for _ in range(2))
    d = (rng.random((steps, envs)) < 0.02).astype(np.float32)
    last = rng.normal(0, 1, envs).astype(np.float32)

    def lay(x):
        x = torch.from_numpy(x).cuda()
        return x if order == "time" else x.t().contiguous().t()
    adv, ret = lay(np.zeros_like(r)), lay(np.zeros_like(r))
    assert train.advantage(lay(r), lay(v), lay(d), torch.from_numpy(last).cuda(), adv, ret, gamma=0.99, lam=0.95) == 0
    g32 = float(np.float32(0.99))
    a32 = float(np.float32(np.float32(0.99) * np.float32(0.95)))
    want, tol = advantage_many(*(x.astype(np.float64) for x in (r, v, d, last)), g32, a32 / g32)
    near(adv.cpu().numpy(), want, tol)
    near(ret.cpu().numpy(), want + v, tol + E * np.abs(want + v))


@pytest.mark.gpu
def test_advantage_offsets_beyond_32_bits():
    """Steps 1.1e9 elements apart."""
    stride = 1100000000
    store = torch.empty(2 * stride + 8, device="cuda")
    r = torch.as_strided(store, (3, 5), (stride, 1))
    r.copy_(torch.arange(15.0).view(3, 5))
    dense = r.contiguous()
    v, d, last = torch.ones((3, 5), device="cuda"), torch.zeros((3, 5), device="cuda"), torch.zeros(5, device="cuda")
    got, want = torch.empty((3, 5), device="cuda"), torch.empty((3, 5), device="cuda")
    assert train.advantage(r, v, d, last, got) == 0 and train.advantage(dense, v, d, last, want) == 0
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("state", ["f32", "f8"])
def test_adamw_of_millions(state):
    """Chunks of several turns: the same bits as the plain formula where it is held in 8 bits, in 32 for m and v."""
    sizes = [10000001, 37, 300000]
    s = make_adam(sizes, "f32", "f32", state, 3)
    before = {k: None if v is None else [host(t).copy() for t in v] for k, v in s.items() if k != "whole"}
    ws, norm = torch.empty(train.grad_norm_workspace_bytes(), dtype=torch.uint8, device="cuda"), torch.empty(2, device="cuda")
    assert train.grad_norm(s["grads"], INF, norm, ws) == 0
    want = math.sqrt(sum(float((g.double() ** 2).sum()) for g in s["grads"]))
    assert abs(float(norm[0]) - want) <= 2 * E * want and float(norm[1]) == 1.0
    assert train.adamw(s["params"], s["grads"], s["m"], s["v"], 3, weight_decay=0.0, scales=s["scales"], seed=7, **H) == 0
    b1, c1, b2, c2 = (np.float32(x) for x in (0.9, 1 - 0.9, 0.95, 1 - 0.95))
    for k, n in enumerate(sizes):
        g = before["grads"][k]
        if state == "f32":
            m, v = before["m"][k], before["v"][k]
        else:
            sc = before["scales"][k].repeat(256, 0)[:n]
            m, r = np_decode(before["m"][k]) * sc[:, 0], np_decode(before["v"][k]) * sc[:, 1]
            v = r * r
        m, v = m * b1 + g * c1, v * b2 + (g * g) * c2
        if state == "f32":
            assert np.array_equal(host(s["m"][k]), m) and np.array_equal(host(s["v"][k]), v)
        else:
            bits = np_hash(n, k, 3, 7)
            root = np.sqrt(v)
            cm, sm = np_pack(m, bits & np.uint64(0xFFFF))
            cv, sv = np_pack(root, bits >> np.uint64(16))
            cv = np.where((cv == 0) & (root > 0) & (sv.repeat(256)[:n] > 0), 1, cv)
            assert np.array_equal(host(s["scales"][k]), np.stack((sm, sv), 1))
            assert np.array_equal(host(s["m"][k]), cm) and np.array_equal(host(s["v"][k]), cv)


@pytest.mark.gpu
def test_adamw_elements_beyond_32_bits():
    """A tensor of 2^32 + 700 elements (34 GB with its gradient and moments): the last ones as any others."""
    n, tail = (1 << 32) + 700, 1000
    p, g = (torch.zeros(n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    sc = torch.zeros(((n + 255) // 256, 2), device="cuda")
    first = (n - tail) // 256 * 256
    grads = (np.random.default_rng(0).normal(0, 1, n - first)).astype(np.float32)
    g[first:] = torch.from_numpy(grads).cuda()
    grads = host(g[first:])
    assert train.adamw([p], [g], [m], [v], 1, 1e-2, scales=[sc], weight_decay=0.0, seed=11) == 0
    M = np.uint64(0xFFFFFFFF)
    i = np.arange(first, n, dtype=np.uint64)
    key = np_mix(np.array([(11 + 0x6A09E667) & 0xFFFFFFFF], np.uint64))[0]
    bits = np_mix(((i & M) * np.uint64(0x9E3779B1) + (i >> np.uint64(32)) * np.uint64(0x6A09E667) + key) & M)
    mm = grads * np.float32(1 - 0.9)
    cm, sm = np_pack(mm, bits & np.uint64(0xFFFF))
    assert np.array_equal(host(m[first:]), cm) and np.array_equal(host(sc[first // 256:, 0]), sm)
    assert (p[:1000] == 0).all() and (p[first:] != 0).any()
