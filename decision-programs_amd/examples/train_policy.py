#!/usr/bin/env python3
"""Trains boosted trees as a policy: actions, advantages, clipped policy loss, preferences.

A table of situations, episodes of STEPS rows each, in which one action is right; the right
action pays 1.  Every batch samples actions from the trees' margins, turns rewards into advantages
(a reverse linear recurrence) and boosts a few rounds with the gradient and hessian of the clipped
policy loss, with a KL term to the policy that the batch began with.  Then two samples of every
episode are compared, and more rounds are boosted from the preference loss of the better one.

    python decision-programs_amd/examples/train_policy.py
"""
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import torch  # noqa: E402
from dpgbdt import Booster, DMatrix, ops  # noqa: E402

STEPS, FEATURES, ACTIONS = 8, 6, 4
GAMMA, LAMBDA = 0.9, 0.8


def sample(margin, generator):
    """An action of every row, by its probability (the largest of margin + Gumbel noise)."""
    u = torch.rand(margin.shape, generator=generator, device=margin.device)
    return (margin - torch.log(-torch.log(u.clamp(1e-20, 1.0 - 1e-7)))).argmax(1)


def advantages(ws, reward, episodes):
    """Discounted sums of what a step paid beyond its batch's mean, to the episode's end."""
    value = (reward - reward.mean()).view(episodes, STEPS, 1)
    gate = torch.full_like(value, GAMMA * LAMBDA)
    states, _ = ops.linear_recurrence(ws, gate, value, reverse=True)
    a = states.reshape(-1)
    return (a - a.mean()) / (a.std() + 1e-6)


def train(episodes=512, batches=10, rounds=4, preference_rounds=6, seed=0, device="cuda"):
    """-> mean rewards: of the first sample, after the policy loss, after the preferences."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    n = episodes * STEPS
    x = torch.randn((n, FEATURES), generator=g, device=device)
    right = (x[:, 0] > 0).long() + 2 * (x[:, 1] + 0.3 * x[:, 2] > 0).long()
    ws = ops.Workspace()
    trees = Booster({"objective": "multi:softprob", "num_class": ACTIONS, "max_depth": 4,
                     "eta": 0.3, "base_score": 0.5})
    matrix = DMatrix(x, torch.zeros(n, device=device))
    margin = torch.zeros((n, ACTIONS), device=device)
    done, rewards = 0, []

    def boost(out):
        nonlocal margin, done
        trees.boost(matrix, done, out.grad, out.hess)
        done += 1
        margin = trees.predict(x, margin=True).view(n, ACTIONS)

    for _ in range(batches):
        action = sample(margin, g)
        reward = (action == right).float()
        rewards.append(reward.mean().item())
        old, _ = ops.action_logprobs(ws, margin, action)
        advantage = advantages(ws, reward, episodes)
        for _ in range(rounds):
            boost(ops.policy_loss(ws, margin, action, old, advantage, reference=old, kl=0.02,
                                  entropy=0.005, hessian=True))
    after_policy = (sample(margin, g) == right).float().mean().item()

    # Two samples of every episode; the one that is paid more comes first.
    both = torch.stack([sample(margin, g), sample(margin, g)], 1).view(episodes, STEPS, 2)
    paid = (both == right.view(episodes, STEPS, 1)).sum(1)
    first = paid.argmax(1)[:, None, None].expand(episodes, STEPS, 1)
    order = torch.cat([both.gather(2, first), both.gather(2, 1 - first)], 2)  # [E, STEPS, 2]
    action = order.transpose(1, 2).reshape(-1)  # sequences: better, worse, better, worse ...
    same = paid[:, 0] == paid[:, 1]
    action = torch.where(same[:, None].expand(episodes, 2 * STEPS).reshape(-1), -1, action)
    sequences = torch.arange(2 * episodes + 1, device=device) * STEPS
    rows = torch.arange(n, device=device).view(episodes, 1, STEPS).expand(episodes, 2, STEPS)
    rows = rows.reshape(-1)
    reference, _ = ops.action_logprobs(ws, margin[rows], action)
    for _ in range(preference_rounds):
        out = ops.preference_loss(ws, margin[rows], action, sequences, reference=reference,
                                  beta=0.5, hessian=True)
        # a situation's two rows go into one
        add = torch.zeros_like(margin)
        boost(out._replace(grad=add.index_add(0, rows, out.grad),
                           hess=add.index_add(0, rows, out.hess)))
    after_preferences = (sample(margin, g) == right).float().mean().item()
    return rewards[0], after_policy, after_preferences


if __name__ == "__main__":
    print("mean reward: %.3f at first, %.3f after the policy loss, %.3f after the preferences"
          % train())
