"""What the training operators (puffysics_b200/train.py) are measured on.

listed() names the cases, draw() gives others of the same ranges, prepare()
makes a case's inputs on the GPU and run() is one pass: with `own` false the
operator in elementary torch operations in 32 bits, with `own` true the
framework's call.  exact() computes the same from the definitions in 64 bits.

The operators are those between an environment batch and its next policy:
  logprob       log probability of the action taken in each row of logits, the
                row's entropy, and its most likely alternatives
  logprob_grad  their gradient with respect to the logits
  advantage     generalised advantages and returns of a rollout
  adamw         one AdamW step over a list of tensors, moments in 32 bits or in
                8, behind a clip of the gradients' global norm
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256              # elements that share a scale where moments are held in 8 bits
E4M3_MAX = 448.0
GAMMA, LAM = 0.99, 0.95
LR, BETA1, BETA2, EPS, DECAY = 3e-4, 0.9, 0.95, 1e-8, 0.01
FIRST_STEP, SEED = 100, 12345
M32 = 0xFFFFFFFF


# ---- cases -------------------------------------------------------------------------------
def listed():
    return [
        # one step of the hover batch: 4,096 environments, three thrust levels; the smallest calls
        dict(name="logprob hover step", op="logprob", rows=4096, width=3, pad=0, dtype="f32", top=0, mask=False),
        # nine joint actions of 16,384 chains, each discretised to 21 levels, greedy action beside the sampled one,
        # levels beyond a joint's limit masked
        dict(name="logprob joint levels", op="logprob", rows=147456, width=21, pad=0, dtype="f32", top=1, mask=True),
        # answering: a few sequences, one token each, twenty alternatives; latency
        dict(name="logprob decode 8", op="logprob", rows=8, width=131072, pad=0, dtype="bf16", top=20, mask=False),
        # scoring with an odd vocabulary (rows at every alignment), padded rows, masked tokens, half precision
        dict(name="logprob odd vocabulary", op="logprob", rows=2048, width=50001, pad=6, dtype="f16", top=5, mask=True),
        # scoring a long batch: the largest
        dict(name="logprob score 4096", op="logprob", rows=4096, width=131072, pad=0, dtype="bf16", top=20, mask=False),
        # the hover rollout's update: 64 steps of 4,096 environments at once
        dict(name="grad hover rollout", op="logprob_grad", rows=262144, width=3, pad=0, dtype="f32", mask=False),
        # a token policy's update, odd vocabulary
        dict(name="grad odd vocabulary", op="logprob_grad", rows=4096, width=50001, pad=7, dtype="bf16", mask=False),
        # the hover rollout as the environment writes it, one row of environments per step
        dict(name="advantage hover rollout", op="advantage", steps=64, envs=4096, order="time", values="f32", ragged=False),
        # long sequences of tokens, each of its own length, one sequence after the other in memory, bf16 values
        dict(name="advantage sequences", op="advantage", steps=8191, envs=1024, order="env", values="bf16", ragged=True),
        # the hover policy: eight small tensors, clip and step; latency
        dict(name="adamw hover policy", op="adamw", layers=0, width=128, param="f32", grad="f32", state="f32", copy=False, clip=True),
        # mixed precision: 32-bit parameters and moments, bf16 gradients, bf16 copies for the next forward pass
        dict(name="adamw mixed", op="adamw", layers=8, width=2048, param="f32", grad="bf16", state="f32", copy=True, clip=True),
        # everything small: bf16 parameters and gradients, 8-bit moments, odd sizes
        dict(name="adamw 8 bit", op="adamw", layers=8, width=2047, param="bf16", grad="bf16", state="f8", copy=False, clip=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprob", "logprob", "logprob_grad", "advantage", "adamw"])
    if op in ("logprob", "logprob_grad"):
        width = _log(rng, 2, 200000)
        most = (1 << 29) if op == "logprob" else (1 << 27)
        rows = _log(rng, 1, min(262144, most // width))
        case = dict(op=op, rows=rows, width=width, pad=rng.choice([0, 0, 1, 8, 13]),
                    dtype=rng.choice(["f32", "bf16", "f16"]), mask=rng.random() < 0.25)
        if op == "logprob":
            case["top"] = rng.choice([0, 1, 5, 20, 32])
        return case
    if op == "advantage":
        steps = _log(rng, 1, 65536)
        return dict(op=op, steps=steps, envs=_log(rng, 1, min(65536, (1 << 23) // steps)), order=rng.choice(["time", "env"]),
                    values=rng.choice(["f32", "bf16"]), ragged=rng.random() < 0.5)
    state = rng.choice(["f32", "f8"])
    return dict(op=op, layers=rng.randint(0, 6), width=_log(rng, 17, 2048), param=rng.choice(["f32", "bf16"]),
                grad=rng.choice(["f32", "bf16", "f16"]), state=state, copy=False, clip=state == "f32" and rng.random() < 0.5)


def _shapes(case):
    """Element counts of the tensors that an adamw case updates."""
    w = case["width"]
    got = [3 * w, w, w * w, w, 3 * w, 3, w, 1]          # a policy of two hidden layers with a value head
    for _ in range(case["layers"]):
        got += [w * w, w, 2 * w * w, 2 * w, 2 * w * w]
    return got


# ---- inputs ------------------------------------------------------------------------------
def _rows(case, g):
    """(rows, width) logits with a row stride of width + pad, as a policy head gives them: most near zero, a
    few tokens well above; the mask of allowed tokens or None, with one row that allows nothing; the actions."""
    rows, width, dt = case["rows"], case["width"], DTYPES[case["dtype"]]
    store = torch.empty((rows, width + case["pad"]), dtype=dt, device="cuda")
    part = max(1, (1 << 26) // (width + case["pad"]))
    for r in range(0, rows, part):
        block = store[r:r + part]
        x = torch.randn(block.shape, generator=g, device="cuda")
        x = x * 2 + (x > 2.5) * 4
        block.copy_(x)
    mask = None
    if case["mask"]:
        chance = torch.rand((rows, width), generator=g, device="cuda")
        actions = torch.where(chance < 0.8, chance, torch.zeros((), device="cuda")).argmax(1)  # one that is allowed
        mask = (chance < 0.8).to(torch.uint8)
        if rows > 8:
            mask[rows // 2] = 0
    else:
        actions = torch.randint(0, width, (rows,), generator=g, device="cuda")
    return store[:, :width], mask, actions


def _f32_rows(state, r, part):
    x = state["logits"][r:r + part].float()
    if state["mask"] is not None:
        x = torch.where(state["mask"][r:r + part] != 0, x, torch.full((), -math.inf, device="cuda"))
    return x


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=dict(case))
    if case["op"] in ("logprob", "logprob_grad"):
        rows, width = case["rows"], case["width"]
        s["logits"], s["mask"], s["actions"] = _rows(case, g)
        s["scale"] = 1.0
        f = dict(dtype=torch.float32, device="cuda")
        if case["op"] == "logprob":
            s["logp"], s["entropy"], s["stats"] = torch.empty(rows, **f), torch.empty(rows, **f), torch.empty((rows, 2), **f)
            if case["top"]:
                s["top_ids"] = torch.empty((rows, case["top"]), dtype=torch.int32, device="cuda")
                s["top_logp"] = torch.empty((rows, case["top"]), **f)
        else:
            # what the forward pass of the same step left behind
            s["stats"], s["entropy"] = torch.empty((rows, 2), **f), torch.empty(rows, **f)
            part = max(1, (1 << 26) // width)
            for r in range(0, rows, part):
                m, logsum, lp = _softmax(_f32_rows(s, r, part), s["scale"])
                s["stats"][r:r + part] = torch.stack((m, logsum), 1)
                s["entropy"][r:r + part] = _entropy(lp)
            s["d_logp"] = torch.randn(rows, generator=g, device="cuda") / rows
            s["d_entropy"] = torch.full((rows,), -0.01 / rows, device="cuda")
            s["grad"] = torch.empty_strided(s["logits"].shape, s["logits"].stride(), dtype=s["logits"].dtype, device="cuda")
    elif case["op"] == "advantage":
        T, N = case["steps"], case["envs"]

        def two(x):  # (steps, envs) whichever runs fastest in memory
            return x if case["order"] == "time" else x.t().contiguous().t()
        s["rewards"] = two(1 - torch.rand((T, N), generator=g, device="cuda"))
        s["values"] = two((torch.randn((T, N), generator=g, device="cuda") * 3 + 10).to(DTYPES[case["values"]]))
        s["terminals"] = two((torch.rand((T, N), generator=g, device="cuda") < 1 / 128).float())
        s["last_values"] = (torch.randn(N, generator=g, device="cuda") * 3 + 10).to(DTYPES[case["values"]])
        s["lengths"] = torch.randint(T // 2, T + 1, (N,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
        s["advantages"], s["returns"] = two(torch.empty((T, N), device="cuda")), two(torch.empty((T, N), device="cuda"))
    else:
        counts = _shapes(case)
        at, total = [], 0
        for n in counts:  # each tensor at an aligned place of one buffer, as an allocator gives them
            at.append(total)
            total += (n + 511) // 512 * 512

        def views(buffer):
            return [buffer[a:a + n] for a, n in zip(at, counts)]
        used = torch.zeros(total, dtype=torch.bool, device="cuda")
        for v in views(used):
            v.fill_(True)

        def normal(std):
            return torch.where(used, torch.randn(total, generator=g, device="cuda") * std, torch.zeros((), device="cuda"))
        s["at"], s["counts"], s["step"] = at, counts, FIRST_STEP
        s["all_params"] = normal(0.02).to(DTYPES[case["param"]])
        # gradients of very different size from element to element, as they are
        s["all_grads"] = (normal(1e-3) * torch.exp(normal(1.0))).to(DTYPES[case["grad"]])
        m, v = normal(1e-4), (normal(1e-3) * torch.exp(normal(1.0))).square()
        if case["state"] == "f32":
            s["all_m"], s["all_v"], s["all_scales"] = m, v, None
        else:  # the buffer's places are multiples of BLOCK, so one pass packs all tensors
            (qm, sm), (qr, sr) = _pack(m, None), _pack(v.sqrt(), None)
            s["all_m"], s["all_v"], s["all_scales"] = qm, qr, torch.stack((sm, sr), 1).contiguous()
        s["copies"] = None
        s["all_copies"] = torch.zeros(total, dtype=torch.bfloat16, device="cuda") if case["copy"] else None
        for name in ("params", "grads", "m", "v"):
            s[name] = views(s["all_" + name])
        if case["copy"]:
            s["copies"] = views(s["all_copies"])
        s["scales"] = None if s["all_scales"] is None else [s["all_scales"][a // BLOCK:a // BLOCK + (n + BLOCK - 1) // BLOCK]
                                                            for a, n in zip(at, counts)]
        s["norm"] = torch.zeros(2, device="cuda")
        s["workspace"] = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
        # the gradients' norm is about 1e-3 e sqrt(n): half of it, so that the clip is at work
        s["max_norm"] = 0.5e-3 * math.e * math.sqrt(sum(counts))
    return s


# ---- plain forms -------------------------------------------------------------------------
def _softmax(x, scale):
    """Row maximum, log of the sum of exp(scale (x - maximum)), and log probabilities."""
    m = x.amax(1)
    d = (x - torch.where(m == -math.inf, torch.zeros_like(m), m)[:, None]) * scale
    total = torch.exp(d).sum(1)
    logsum = torch.where(m == -math.inf, torch.zeros_like(m), torch.log(total))
    return m, logsum, d - logsum[:, None]


def _entropy(lp):
    p = torch.exp(lp)
    return -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)


def _plain_logprob(s):
    c = s["case"]
    x = _f32_rows(s, 0, c["rows"])
    m, logsum, lp = _softmax(x, s["scale"])
    out = dict(logp=torch.gather(lp, 1, s["actions"][:, None])[:, 0], entropy=_entropy(lp), stats=torch.stack((m, logsum), 1))
    if c["top"]:
        k = min(c["top"], c["width"])
        # one whole number a token that orders by value, and by lowest index where values tie
        bits = (x + 0.0).view(torch.int32).to(torch.int64)
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        key = (bits << 32) + (M32 - torch.arange(c["width"], device="cuda"))
        ids = M32 - (torch.topk(key, k, 1).values & M32)
        top = torch.gather(lp, 1, ids)
        ids = torch.where(top == -math.inf, torch.full_like(ids, -1), ids).to(torch.int32)
        out["top_ids"] = torch.nn.functional.pad(ids, (0, c["top"] - k), value=-1)
        out["top_logp"] = torch.nn.functional.pad(top, (0, c["top"] - k), value=-math.inf)
    return out


def _plain_logprob_grad(s):
    x = _f32_rows(s, 0, s["case"]["rows"])
    m, logsum = s["stats"][:, 0], s["stats"][:, 1]
    lp = (x - torch.where(m == -math.inf, torch.zeros_like(m), m)[:, None]) * s["scale"] - logsum[:, None]
    p = torch.exp(lp)
    zero = torch.zeros((), device="cuda")
    taken = torch.gather(lp, 1, s["actions"][:, None])
    g = torch.where(taken > -math.inf, s["d_logp"][:, None], zero)
    d = -p * (g + s["d_entropy"][:, None] * (torch.where(p > 0, lp, zero) + s["entropy"][:, None]))
    d = d.scatter_add(1, s["actions"][:, None], g) * s["scale"]
    return dict(grad=d.to(s["logits"].dtype))


def _plain_advantage(s):
    r, v, d = s["rewards"], s["values"].float(), s["terminals"]
    T = r.shape[0]
    t = torch.arange(T, device="cuda")[:, None]
    length = s["lengths"] if s["lengths"] is not None else torch.full((r.shape[1],), T, device="cuda")
    inside = t < length
    after = torch.cat((v[1:], v[:1]))
    after = torch.where(t == length - 1, s["last_values"].float(), after)
    live = (d == 0) & inside
    zero = torch.zeros((), device="cuda")
    b = torch.where(inside, r + GAMMA * torch.where(live, after, zero) - v, zero)
    a = torch.where(live & (t < length - 1), GAMMA * LAM, 0.0)
    k = 1
    while k < T:  # A[t] = b[t] + a[t] A[t + 1], twice as far with each pass
        pad = torch.zeros((k, r.shape[1]), device="cuda")
        b = b + a * torch.cat((b[k:], pad))
        a = a * torch.cat((a[k:], pad))
        k *= 2
    return dict(advantages=b, returns=torch.where(inside, b + v, zero))


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x85A308D3) & M32
    x = x ^ (x >> 13)
    x = (x * 0x243F6A89) & M32
    return x ^ (x >> 16)


def _hash(n, tensor, step):
    """32 random bits for each element of a tensor: a whole number in the place of a generator's state."""
    key = _mix((SEED + tensor * 0x9E3779B1 + step * 0x6A09E667) & M32)
    i = torch.arange(n, device="cuda")
    return _mix(((i & M32) * 0x9E3779B1 + (i >> 32) * 0x6A09E667 + key) & M32)


def _pack(x, bits):
    """x as e4m3 with a scale for each BLOCK (448 stands for the block's largest), rounded by 16 random bits
    an element, or to nearest where there are none."""
    n = x.numel()
    blocks = torch.nn.functional.pad(x, (0, -n % BLOCK)).view(-1, BLOCK)
    most = blocks.abs().amax(1)
    ok = most >= 2.0 ** -100
    scale = torch.where(ok, most / E4M3_MAX, torch.zeros_like(most))
    inverse = torch.where(ok, E4M3_MAX / most, torch.zeros_like(most))
    y = (blocks * inverse[:, None]).view(-1)[:n]
    word = (y.abs() * 2.0 ** -120).view(torch.int32)
    word = word + (((bits.to(torch.int32) << 4) | 8) if bits is not None else 0x7FFFF + ((word >> 20) & 1))
    code = torch.clamp(word >> 20, max=0x7E)
    return torch.where(y < 0, code | 0x80, code).to(torch.uint8).view(torch.float8_e4m3fn), scale


def _unpack(q, scale):
    return q.float() * scale.repeat_interleave(BLOCK)[:q.numel()]


def _plain_adamw(s):
    c = s["case"]
    factor = torch.ones((), device="cuda")
    if c["clip"]:
        norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
        factor = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
        s["norm"].copy_(torch.stack((norm, factor)))
    t = s["step"]
    lr1, root2 = LR / (1 - BETA1 ** t), 1 / math.sqrt(1 - BETA2 ** t)
    for k in range(len(s["params"])):
        p, m, v = s["params"][k], s["m"][k], s["v"][k]
        g = s["grads"][k].float() * factor
        if c["state"] == "f8":
            new_m, r = _unpack(m, s["scales"][k][:, 0]), _unpack(v, s["scales"][k][:, 1])
            new_v = r * r
        else:
            new_m, new_v = m, v
        new_m = new_m * BETA1 + g * (1 - BETA1)
        new_v = new_v * BETA2 + (g * g) * (1 - BETA2)
        root = torch.sqrt(new_v)
        x = p.float() * (1 - LR * DECAY) - (new_m / (root * root2 + EPS)) * lr1
        if c["state"] == "f8":
            bits = _hash(p.numel(), k, t)
            qm, sm = _pack(new_m, bits & 0xFFFF)
            qr, sr = _pack(root, bits >> 16)
            # an element that has seen a gradient keeps the smallest step above zero: a moment never divides by eps alone
            qr = torch.where((qr.view(torch.uint8) == 0) & (root > 0) & (sr > 0).repeat_interleave(BLOCK)[:p.numel()],
                             torch.ones((), dtype=torch.uint8, device="cuda"), qr.view(torch.uint8))
            m.view(torch.uint8).copy_(qm.view(torch.uint8))
            v.view(torch.uint8).copy_(qr)
            s["scales"][k].copy_(torch.stack((sm, sr), 1))
        else:
            m.copy_(new_m)
            v.copy_(new_v)
        if c["param"] == "bf16":
            low = _mix((_hash(p.numel(), k, t) + 0x9E3779B1) & M32) & 0xFFFF
            x = ((x.view(torch.int32) + low.to(torch.int32)) & -65536).view(torch.float32)
        p.copy_(x)
        if c["copy"]:
            s["copies"][k].copy_(x)
    return _adamw_outputs(s)


def _adamw_outputs(s):
    out = dict(params=s["all_params"], m=s["all_m"], v=s["all_v"])
    if s["all_scales"] is not None:
        out["scales"] = s["all_scales"]
    if s["copies"] is not None:
        out["copies"] = s["all_copies"]
    if s["case"]["clip"]:
        out["norm"] = s["norm"]
    return out


# ---- one pass ----------------------------------------------------------------------------
def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        out = {"logprob": _plain_logprob, "logprob_grad": _plain_logprob_grad, "advantage": _plain_advantage,
               "adamw": _plain_adamw}[op](s)
        if op == "adamw":
            s["step"] += 1
        return out
    from puffysics_b200 import train
    if op == "logprob":
        rc = train.logprob(s["logits"], s["actions"], logp=s["logp"], entropy=s["entropy"], stats=s["stats"],
                           top_ids=s.get("top_ids"), top_logp=s.get("top_logp"), mask=s["mask"], scale=s["scale"])
        out = {k: s[k] for k in ("logp", "entropy", "stats", "top_ids", "top_logp") if k in s}
    elif op == "logprob_grad":
        rc = train.logprob_grad(s["logits"], s["stats"], s["grad"], actions=s["actions"], d_logp=s["d_logp"],
                                entropy=s["entropy"], d_entropy=s["d_entropy"], mask=s["mask"], scale=s["scale"])
        out = dict(grad=s["grad"])
    elif op == "advantage":
        rc = train.advantage(s["rewards"], s["values"], s["terminals"], s["last_values"], s["advantages"], s["returns"],
                             gamma=GAMMA, lam=LAM, lengths=s["lengths"])
        out = dict(advantages=s["advantages"], returns=s["returns"])
    else:
        rc = 0
        if c["clip"]:
            rc = train.grad_norm(s["grads"], s["max_norm"], s["norm"], s["workspace"])
        rc = rc or train.adamw(s["params"], s["grads"], s["m"], s["v"], s["step"], LR, BETA1, BETA2, EPS, DECAY,
                               scales=s["scales"], grad_scale=s["norm"][1:] if c["clip"] else None, copies=s["copies"],
                               seed=SEED)
        s["step"] += 1
        out = _adamw_outputs(s)
    if rc:
        raise RuntimeError("%s: error %d" % (op, rc))
    return out


# ---- what a pass cannot do without ---------------------------------------------------------
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] in ("logprob", "logprob_grad"):
        n, rows = case["rows"] * case["width"], case["rows"]
        read = n * (size[case["dtype"]] + int(case["mask"]))
        if case["op"] == "logprob":
            return dict(bytes=read + rows * (8 + 16 + 8 * case["top"]), flops=7 * n)
        return dict(bytes=read + n * size[case["dtype"]] + rows * (8 + 20), flops=8 * n)
    if case["op"] == "advantage":
        n = case["steps"] * case["envs"]
        return dict(bytes=n * (16 + size[case["values"]]) + case["envs"] * (size[case["values"]] + 4 * int(case["ragged"])), flops=8 * n)
    n = sum(_shapes(case))
    one = 2 * size[case["param"]] + size[case["grad"]] + (16 if case["state"] == "f32" else 4 + 16 / BLOCK) + 2 * int(case["copy"])
    return dict(bytes=n * one, flops=(14 + 2 * int(case["clip"])) * n)


# ---- the definitions in 64 bits --------------------------------------------------------------
def _exact_rows(s, r, part):
    z = s["logits"][r:r + part].to(torch.float64)
    if s["mask"] is not None:
        z[s["mask"][r:r + part] == 0] = -math.inf
    log_p = z * s["scale"]
    log_p -= torch.logsumexp(log_p, 1, keepdim=True)
    log_p[torch.isnan(log_p)] = -math.inf               # a row that allows nothing
    return z, log_p


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprob":
        out = dict(logp=[], entropy=[], stats=[], top_logp=[])
        part = max(1, (1 << 26) // case["width"])
        for r in range(0, case["rows"], part):
            z, log_p = _exact_rows(s, r, part)
            top = z.max(1).values
            total = torch.exp((z - top[:, None]) * s["scale"]).sum(1)
            out["stats"].append(torch.stack((top, torch.where(top == -math.inf, torch.zeros_like(top), total.log())), 1))
            out["logp"].append(log_p[torch.arange(len(z), device="cuda"), s["actions"][r:r + part]])
            out["entropy"].append(torch.special.entr(log_p.exp()).sum(1))
            if case["top"]:
                k = min(case["top"], case["width"])
                best = torch.sort(log_p, 1, descending=True).values[:, :k] if case["width"] < 1024 else torch.topk(log_p, k, 1).values
                out["top_logp"].append(torch.cat((best, torch.full((len(z), case["top"] - k), -math.inf, device="cuda", dtype=best.dtype)), 1))
        out = {k: torch.cat(v) if v else None for k, v in out.items()}
        if not case["top"]:
            del out["top_logp"]
        else:
            out["top_ids"] = None
        return out
    if case["op"] == "logprob_grad":
        got = torch.empty((case["rows"], case["width"]), dtype=torch.float64, device="cuda")
        part = max(1, (1 << 26) // case["width"])
        for r in range(0, case["rows"], part):
            _, log_p = _exact_rows(s, r, part)
            p = log_p.exp()
            entropy = torch.special.entr(p).sum(1, keepdim=True)
            a = s["actions"][r:r + part]
            row = torch.arange(len(p), device="cuda")
            g = s["d_logp"][r:r + part].double() * (p[row, a] > 0)
            h = s["d_entropy"][r:r + part].double()
            d = torch.special.entr(p) * h[:, None] - p * (g[:, None] + h[:, None] * entropy)
            d[row, a] += g
            got[r:r + part] = d * s["scale"]
        return dict(grad=got)
    if case["op"] == "advantage":
        r, v, d, last = (s[k].double().cpu().numpy() for k in ("rewards", "values", "terminals", "last_values"))
        T, N = r.shape
        import numpy as np
        length = s["lengths"].cpu().numpy() if s["lengths"] is not None else np.full(N, T)
        adv, ret = np.zeros((T, N)), np.zeros((T, N))
        ahead, value = np.zeros(N), np.zeros(N)
        for t in range(T - 1, -1, -1):
            starts = t == length - 1
            ahead, value = np.where(starts, 0.0, ahead), np.where(starts, last, value)
            on = 1.0 - d[t]
            ahead = r[t] + GAMMA * on * value - v[t] + GAMMA * LAM * on * ahead
            value = v[t]
            inside = t < length
            adv[t], ret[t] = np.where(inside, ahead, 0), np.where(inside, ahead + value, 0)
        return dict(advantages=adv, returns=ret)
    # one step; what is held in fewer bits than 32 has no value in 64
    t = s["step"]
    out = dict(params=s["all_params"].double(), m=None, v=None)
    grads = s["all_grads"].double()
    norm = torch.linalg.vector_norm(grads)
    if case["clip"]:
        factor = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
        grads *= factor
        out["norm"] = torch.stack((norm, torch.full_like(norm, factor)))
    if case["state"] == "f32":
        m, v = s["all_m"].double(), s["all_v"].double()
    else:
        scale = s["all_scales"].double().repeat_interleave(BLOCK, 0)
        m, v = s["all_m"].double() * scale[:, 0], (s["all_v"].double() * scale[:, 1]) ** 2
    m.lerp_(grads, 1 - BETA1)
    v.mul_(BETA2).addcmul_(grads, grads, value=1 - BETA2)
    step = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    out["params"] = out["params"] * (1 - LR * DECAY) - LR * step
    if case["state"] == "f32":
        out["m"], out["v"] = m, v
    else:
        out["scales"] = torch.stack([x.view(-1, BLOCK).abs().amax(1) / E4M3_MAX for x in (m, v.sqrt())], 1)
    if case["copy"]:
        out["copies"] = out["params"]
    return out
