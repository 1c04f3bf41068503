r"""Switch-Transformer top-1 gate: uniform jitter added to the logits in training, per-expert capacity,
balance loss over the surviving tokens (behaviour of fmoe/gates/switch_gate.py:12-59)."""
import torch

from .naive_gate import NaiveGate
from .utils import balance_loss_kernel_applies, capacity_of, limit_by_capacity
from ..functions import balance_loss


class SwitchGate(NaiveGate):
    def __init__(self, d_model, num_expert, world_size, topk=1, switch_eps=0.1,
                 capacity=(1.2, 2.4)):
        if topk != 1:
            raise AssertionError("topk should be 1 in switch")
        super().__init__(d_model, num_expert, world_size, top_k=1)
        self.switch_eps = switch_eps
        self.capacity = capacity

    def forward(self, inp):
        logits = self.gate(inp)
        if self.training:
            # uniform in [1-eps, 1+eps], ADDED to the logits as in switch_gate.py:30-34
            eps = self.switch_eps
            logits = logits + (1.0 - eps + 2 * eps * torch.rand_like(logits))
        logits = logits.float()
        prob = torch.softmax(logits, dim=-1)   # the loss needs every expert's probability
        top1_score, top1_idx = prob.max(dim=-1, keepdim=True)
        top1_score = top1_score.to(inp.dtype)

        cap = capacity_of(self.capacity, self.training, inp.shape[0])
        top1_idx = limit_by_capacity(top1_idx, self.num_expert, self.world_size, cap)[2]

        # fraction of the surviving tokens per expert x summed probability per expert, both over
        # the number of survivors (switch_gate.py:46-58)
        if balance_loss_kernel_applies(logits):
            self.set_loss(balance_loss(logits, top1_idx, per="slot")[0])
            return top1_idx, top1_score
        kept = top1_idx[top1_idx >= 0]
        fraction = torch.bincount(kept, minlength=self.tot_expert).to(torch.float) / kept.numel()
        prob_sum = prob.sum(dim=0) / kept.numel()
        self.set_loss((fraction * prob_sum).sum() * self.tot_expert)
        return top1_idx, top1_score
