"""Trains a policy on the hover environment: the environment's step and the
training operators on one stream, nothing copied to the host between them.

    python examples/hover_train.py [--envs 4096] [--iterations 40]

Each iteration rolls the batch out for 64 steps (puffysics_b200/hover_env.py
writes rewards and terminals into the rollout's rows, train.logprob the log
probability of each action), turns rewards and terminals into advantages and
returns (train.advantage), and goes over the rollout a few times in shuffled
eighths: a clipped surrogate of the new and old log probabilities with an
entropy bonus, whose derivatives train.logprob_grad turns into gradients of the
logits, torch's backward pass through the network's two layers, a clip of the
gradients' norm (train.grad_norm) and a step (train.adamw), with moments in 32
or 8 bits.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from puffysics_b200 import build, hover_env, train  # noqa: E402

LEVELS = 3               # thrust levels: none, one, two


def check(rc):
    if rc != 0:
        raise RuntimeError("CUDA error %d" % rc)


class Policy(torch.nn.Module):
    def __init__(self, width=64):
        super().__init__()
        self.body = torch.nn.Sequential(torch.nn.Linear(hover_env.OBS, width), torch.nn.Tanh(),
                                        torch.nn.Linear(width, width), torch.nn.Tanh())
        self.logits, self.value = torch.nn.Linear(width, LEVELS), torch.nn.Linear(width, 1)

    def forward(self, obs):
        h = self.body(obs)
        return self.logits(h), self.value(h)[:, 0]


class AdamW:
    """Parameters with their moments; step() clips and updates from their .grad."""

    def __init__(self, params, lr, max_norm, eight_bit=False):
        self.params, self.lr, self.max_norm, self.t = [p.data for p in params], lr, max_norm, 0
        self.owners = list(params)
        kind = dict(dtype=torch.float8_e4m3fn if eight_bit else torch.float32, device="cuda")
        self.m, self.v = ([torch.zeros(p.shape, **kind) for p in self.params] for _ in range(2))
        self.scales = [torch.zeros(((p.numel() + train.BLOCK - 1) // train.BLOCK, 2), device="cuda")
                       for p in self.params] if eight_bit else None
        self.norm = torch.zeros(2, device="cuda")
        self.workspace = torch.empty(train.grad_norm_workspace_bytes(), dtype=torch.uint8, device="cuda")

    def step(self):
        self.t += 1
        grads = [p.grad for p in self.owners]
        check(train.grad_norm(grads, self.max_norm, self.norm, self.workspace))
        check(train.adamw(self.params, grads, self.m, self.v, self.t, self.lr, weight_decay=0.0, scales=self.scales,
                          grad_scale=self.norm[1:], seed=1 if self.scales else None))


def run(envs=4096, iterations=40, steps=64, epochs=3, parts=8, lr=1e-3, clip=0.2, bonus=0.003, eight_bit=False, seed=1,
        report=None):
    """Mean reward a step of each iteration's rollout."""
    build.build()
    torch.manual_seed(seed)
    f = dict(dtype=torch.float32, device="cuda")
    policy = Policy().cuda()
    optimiser = AdamW(list(policy.parameters()), lr, 0.5, eight_bit)
    state = torch.zeros((envs, hover_env.env_bytes()), dtype=torch.uint8, device="cuda")
    obs, now = torch.empty((steps, envs, hover_env.OBS), **f), torch.empty((envs, hover_env.OBS), **f)
    rewards, terminals, values, old = (torch.empty((steps, envs), **f) for _ in range(4))
    actions = torch.empty((steps, envs), dtype=torch.int64, device="cuda")
    advantages, returns = torch.empty((steps, envs), **f), torch.empty((steps, envs), **f)
    check(hover_env.init(state, seed))
    check(hover_env.reset(state, now, rewards[0], terminals[0]))
    got = []
    for iteration in range(iterations):
        with torch.no_grad():
            for t in range(steps):
                obs[t] = now
                logits, values[t] = policy(now)
                # the largest of logits and Gumbel noise is a sample
                actions[t] = (logits - torch.log(-torch.log(torch.rand_like(logits)))).argmax(1)
                check(train.logprob(logits, actions[t], logp=old[t]))
                check(hover_env.step(state, actions[t].float(), now, rewards[t], terminals[t]))
            last = policy(now)[1]
        check(train.advantage(rewards, values, terminals, last, advantages, returns, gamma=0.99, lam=0.95))
        flat = [x.reshape(steps * envs, *x.shape[2:]) for x in (obs, actions, old, advantages, returns)]
        for _ in range(epochs):
            for rows in torch.randperm(steps * envs, device="cuda").chunk(parts):
                o, a, lp0, adv, ret = (x[rows] for x in flat)
                n = len(rows)
                adv = (adv - adv.mean()) / (adv.std() + 1e-6)
                logits, value = policy(o)
                lp, entropy, stats = torch.empty(n, **f), torch.empty(n, **f), torch.empty((n, 2), **f)
                check(train.logprob(logits.detach(), a, logp=lp, entropy=entropy, stats=stats))
                ratio = torch.exp(lp - lp0)
                held = ((ratio > 1 + clip) & (adv > 0)) | ((ratio < 1 - clip) & (adv < 0))
                d_logp = torch.where(held, 0.0, -adv * ratio) / n
                d_entropy = torch.full((n,), -bonus / n, **f)
                d_logits = torch.empty_like(logits)
                check(train.logprob_grad(logits.detach(), stats, d_logits, actions=a, d_logp=d_logp, entropy=entropy,
                                         d_entropy=d_entropy))
                policy.zero_grad(set_to_none=True)
                torch.autograd.backward([logits, value], [d_logits, 0.5 * (value.detach() - ret) / n])
                optimiser.step()
        got.append(rewards.mean())
        if report:
            report(iteration, got[-1])
    return [float(x) for x in got]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--envs", type=int, default=4096)
    ap.add_argument("--iterations", type=int, default=40)
    ap.add_argument("--eight-bit", action="store_true", help="moments in 8 bits")
    a = ap.parse_args()
    run(a.envs, a.iterations, eight_bit=a.eight_bit, report=lambda k, r: print("iteration %3d  mean reward %.4f" % (k, float(r))))
