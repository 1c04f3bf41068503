r"""Capacity helpers of the gates (fmoe/gates/utils.py:9-26), and when their balance loss is the kernel's."""
import math
import os

import torch

from .. import fmoe_native
from ..functions import _attach_route, _route_launch, count_by_gate, nothing_watches


def limit_by_capacity(topk_idx, num_expert, world_size, capacity):
    r"""Caps every expert at ``capacity`` slots and rewrites the gate indices of the
    slots that do not fit to -1 (slots with the lowest flat index win).
    Returns ``(new_local_expert_count, new_global_expert_count, pruned_idx)``.
    The reference unpacks three values from ``count_by_gate``'s five
    (fmoe/gates/utils.py:14); the five-tuple is what is used here.

    The indices that stay are routed on the way, out of the routing that the gate's kernels left on ``topk_idx`` (or made
    here); it rides on ``pruned_idx`` to the layer."""
    with torch.no_grad():
        if (world_size == 1 and topk_idx.is_cuda and topk_idx.dtype == torch.int64 and topk_idx.numel() > 0
                and 1 <= num_expert <= 1024 and 0 <= int(capacity) < 1 << 31):
            counts, _pos, slot_to_row, table = _route_launch(topk_idx, num_expert, with_table=True)
            new_lec, pruned, pos, slot_to_row, table = fmoe_native.limit_route(topk_idx.contiguous(), counts, slot_to_row, table,
                                                                               capacity)
            _attach_route(pruned, num_expert, new_lec, pos, slot_to_row, table)
            return new_lec, new_lec, pruned
        cap = torch.full((num_expert,), int(capacity), dtype=torch.int32, device=topk_idx.device)
        _pos, _lec, _all_ec, gec, _all_gec = count_by_gate(topk_idx, num_expert, world_size,
                                                           require_pos=False)
        new_gec = fmoe_native.limit_by_capacity(gec, cap, num_expert, world_size)
        new_lec = new_gec  # one worker: nothing to exchange
        pruned = fmoe_native.prune_gate_by_capacity(topk_idx.contiguous(), new_lec.to(torch.int32),
                                                    num_expert, world_size)
    return new_lec, new_gec, pruned


def capacity_of(rates, training, n_tokens):
    r"""Slots an expert may take: ``rates = (train, eval)`` factors of the token count, rounded up
    (fmoe/gates/gshard_gate.py:36-37, switch_gate.py:40-41)."""
    return math.ceil(rates[0 if training else 1] * n_tokens)


def balance_loss_kernel_applies(logits):
    r"""Whether a gate's balance loss over ``logits`` is :func:`~fastermoe_amd.functions.balance_loss`, which reads nothing on the host (boolean
    indexing and ``torch.bincount`` do): GPU tensors that it takes, unless ``FMOE_BALANCE_LOSS_KERNEL=0`` keeps the torch operators or something has to see them."""
    return (logits.is_cuda and logits.dim() == 2 and logits.shape[0] > 0 and fmoe_native.balance_loss_supported(logits.shape[1], logits.dtype)
            and os.environ.get("FMOE_BALANCE_LOSS_KERNEL", "1") != "0" and nothing_watches(logits))
