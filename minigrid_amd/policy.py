"""A policy for the batched environments, and what a rollout of one leaves: ActorCritic (layers from `ops.linear`) and Trajectory (advantages and loss from
`ops.advantages` and `ops.policy_loss`).  `MiniGridVecEnv.rollout(policy=...)` runs the one and returns the other."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import ops


class ActorCritic(torch.nn.Module):
    """Logits of the seven actions and the value of an observation: image bytes -> hidden (tanh) -> `layers` residual layers (gelu) -> one head whose last
    column is the value.  A policy for `MiniGridVecEnv.rollout`: called with an observation as `step` returns it (the dictionary, or the image)."""

    def __init__(self, image_shape, hidden: int = 256, layers: int = 1, actions: int = 7, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        k = math.prod(image_shape)
        make = lambda n, m, gain: torch.nn.Parameter((torch.randn(n, m, device=device) * (gain / math.sqrt(m))).to(dtype))
        self.actions, self.pixels = int(actions), k
        # (the bytes of an observation are 0..10, about 2 in the mean square)
        self.w_in, self.b_in = make(hidden, k, 0.5), torch.nn.Parameter(torch.zeros(hidden, dtype=dtype, device=device))
        self.w = torch.nn.ParameterList([make(hidden, hidden, 0.5) for _ in range(layers)])
        self.b = torch.nn.ParameterList([torch.nn.Parameter(torch.zeros(hidden, dtype=dtype, device=device)) for _ in range(layers)])
        self.w_out, self.b_out = make(actions + 1, hidden, 0.1), torch.nn.Parameter(torch.zeros(actions + 1, dtype=dtype, device=device))

    def forward(self, obs):
        image = obs["image"] if isinstance(obs, dict) else obs
        lead = image.shape[:-3]
        h = ops.linear(image.reshape(-1, self.pixels), self.w_in, self.b_in, activation="tanh")
        for w, b in zip(self.w, self.b):
            h = ops.linear(h, w, b, activation="gelu", residual=h)
        out = ops.linear(h, self.w_out, self.b_out)
        return out[:, :self.actions].unflatten(0, lead), out[:, self.actions].float().unflatten(0, lead)


@dataclass
class Trajectory:
    """`steps` x `envs` transitions.  image, direction, mission_id: the observation a step was taken on; action, log_prob: what was drawn there; value: what
    the policy thought of it; reward, terminated, truncated: what the step returned; done: whether an episode ended in the step before the first;
    last_value: of the observation behind the last step."""
    image: torch.Tensor
    direction: torch.Tensor
    mission_id: torch.Tensor
    action: torch.Tensor
    log_prob: torch.Tensor
    value: torch.Tensor
    reward: torch.Tensor
    terminated: torch.Tensor
    truncated: torch.Tensor
    done: torch.Tensor
    last_value: torch.Tensor
    autoreset_mode: str
    final_value: Optional[torch.Tensor] = None

    def advantages(self, gamma: float = 0.99, lam: float = 0.95):
        """(advantage, return, valid) of the rollout: `ops.advantages`.  In the same_step mode a truncated step is bootstrapped from final_value, and counts as worth
        0 without it."""
        next_step = self.autoreset_mode == "next_step"
        return ops.advantages(self.reward, self.value, self.last_value, self.terminated, self.truncated, gamma=gamma, lam=lam,
                              autoreset_mode=self.autoreset_mode, done=self.done if next_step else None, final_value=None if next_step else self.final_value)

    def loss(self, logits, advantage, mask=None, *, index: Optional[torch.Tensor] = None, ref_log_prob=None, **kw):
        """`ops.policy_loss` of new logits for all transitions, or for those at `index` of the flattened (steps x envs) -- a minibatch; advantage, mask and
        ref_log_prob are (steps, envs) either way.  In the next_step mode mask is `advantages`' valid: without it the rows that only reset count too."""
        pick = (lambda t: t) if index is None else (lambda t: None if t is None else t.reshape(-1)[index])
        return ops.policy_loss(logits, pick(self.action), pick(self.log_prob), pick(advantage), mask=pick(mask), ref_log_prob=pick(ref_log_prob), **kw)
