r"""MoE feed-forward block of a transformer (fmoe/transformer.py)."""
import os

import torch
import torch.nn as nn

from . import _lib, fmoe_native
from .functions import (MOEExpertMLP, MOEExpertMLPCheckpointed, MOERoutedGatedMLP, MOERoutedMLP, MOERoutedMLPCheckpointed,
                        _gate_activation_code, _no_hooks, add_layer_norm, gated_mlp, layer_call, layer_norm, linear_int8,
                        nothing_watches, quantize_rows)
from .gates import NaiveGate
from .layers import FMoE, FMoELinear


class _Expert(nn.Module):
    r"""All experts of a worker as two grouped linears around an activation
    (fmoe/transformer.py:10-30).  ``act_checkpoint`` (or ``FMOE_ACT_CHECKPOINT=1``): a training step keeps what its backward needs of
    the activation in 8 bits."""

    act_checkpoint = False

    def __init__(self, num_expert, d_model, d_hidden, activation, rank=0, bias=True):
        super().__init__()
        self.htoh4 = FMoELinear(num_expert, d_model, d_hidden, bias=bias, rank=rank)
        self.h4toh = FMoELinear(num_expert, d_hidden, d_model, bias=bias, rank=rank)
        self.activation = activation
        if os.environ.get("FMOE_ACT_CHECKPOINT", "0") == "1":
            self.act_checkpoint = True

    def _saves(self, inp):
        """Whether a backward through these experts may come."""
        return torch.is_grad_enabled() and (inp.requires_grad or any(
            p is not None and p.requires_grad for p in (self.htoh4.weight, self.htoh4.bias, self.h4toh.weight, self.h4toh.bias)))

    def _checkpoints(self, inp):
        r"""Whether this step keeps its activations in 8 bits; an error where it is to and cannot."""
        if not self.act_checkpoint or not inp.is_cuda or not self._saves(inp):
            return False
        if self._epilogue_activation() is None:
            raise NotImplementedError(f"act_checkpoint takes GELU, ReLU or no activation, got {self.activation!r}")
        if not fmoe_native.act_checkpoint_supported(inp.dtype):
            raise NotImplementedError(f"act_checkpoint does not take {inp.dtype}")
        return True

    def forward(self, inp, fwd_expert_count):
        # GELU (exact), ReLU or no activation: one autograd node with the activation in the GEMM
        # epilogues (FMOE_EXPERT_EPILOGUE=0 keeps the three modules apart, as the reference runs them)
        code = self._epilogue_activation()
        if self._checkpoints(inp):
            return MOEExpertMLPCheckpointed.apply(inp, fwd_expert_count, self.htoh4.weight, self.htoh4.bias,
                                                  self.h4toh.weight, self.h4toh.bias, code)
        # (float64 keeps torch's activation: the epilogue's GELU is evaluated in single precision)
        if (code is not None and inp.is_cuda and inp.dtype in (torch.float32, torch.bfloat16, torch.float16)
                and os.environ.get("FMOE_EXPERT_EPILOGUE", "1") != "0"):
            return MOEExpertMLP.apply(inp, fwd_expert_count, self.htoh4.weight, self.htoh4.bias,
                                      self.h4toh.weight, self.h4toh.bias, code)
        x = self.htoh4(inp, fwd_expert_count)
        x = self.activation(x)
        return self.h4toh(x, fwd_expert_count)

    def routed_forward(self, inp, pos_buf, slot_to_row, counts_dev, top_k, table=None):
        r"""The experts over token rows ``inp [N, d_model]`` routed by ``pos_buf`` / ``slot_to_row`` /
        ``counts_dev`` (the device tensors of the routing call, and ``table``, the segment table of the
        counts, where the call made one), without any of them being read on the host: returns the
        experts' output in expert-sorted order, one row per slot, or ``None`` when this shape or
        activation needs the module-by-module path."""
        if not self._device_tables_apply(inp):
            return None
        code = self._epilogue_activation()
        if table is None:
            table = fmoe_native.segment_table(counts_dev, pos_buf.numel())
        params = (self.htoh4.weight, self.htoh4.bias, self.h4toh.weight, self.h4toh.bias)
        if self._checkpoints(inp):
            return MOERoutedMLPCheckpointed.apply(inp, *params, pos_buf, slot_to_row, table, top_k, code)
        return MOERoutedMLP.apply(inp, *params, pos_buf, slot_to_row, table, top_k, code, self._saves(inp))

    def routed_layer(self, inp, gate_w, gate_b, score, routing, top_k):
        r"""The layer's output from its input as one call: with the gate's linear layer ``gate_w``, ``gate_b`` inside it, or
        over the ``score`` and ``routing`` (``pos_buf``, ``slot_to_row`` and the segment table) of a gate outside.  ``None``
        where that call does not apply: a subclass, replaced linears, another activation, tensors or sizes that it does not
        take, activations that are kept in 8 bits, or somebody who watches the operators."""
        first, second = self._modules.get("htoh4"), self._modules.get("h4toh")
        if type(self) is not _Expert or type(first) is not FMoELinear or type(second) is not FMoELinear:
            return None
        try:
            params = [linear._parameters[name] for linear in (first, second) for name in ("weight", "bias")]
        except KeyError:   # (parametrised, or a view that a sharding wrapper put there)
            return None
        if self.act_checkpoint and self._checkpoints(inp):
            return None
        code = self._epilogue_activation()
        if code is None or params[0] is None or params[2] is None or not nothing_watches(inp, *(t for t in (gate_w, gate_b, score, *params) if t is not None)):
            return None
        if gate_w is None:
            gate = _lib.GATE_ROUTED
        elif fmoe_native.gate_linear_supported(inp.shape[1], gate_w.shape[0], top_k, inp.dtype):
            gate = _lib.GATE_LINEAR
        else:
            gate = _lib.GATE_LOGITS
        return layer_call(inp, gate_w, gate_b, score, *params, routing, top_k, code, gate)

    def unchunked_is_faster(self, inp, n_slots):
        r"""Whether :meth:`routed_forward` beats the chunked pipeline: where both linears run on the persistent
        kernel and nobody asks for a number of chunks.  The pipeline hides the row permutes behind the
        products of its chunks, but needs the counts on the host and pays every chunk's last round of tiles."""
        if "FMOE_FUSE_GRAN" in os.environ or not self._device_tables_apply(inp):
            return False
        n_expert, d_hidden, d_model = self.htoh4.weight.shape
        code = self._epilogue_activation()
        return (fmoe_native.linear_dev_reads_rows(n_slots, n_expert, d_model, d_hidden, inp.dtype, code, code == _lib.ACT_GELU)
                and fmoe_native.linear_dev_reads_rows(n_slots, n_expert, d_hidden, d_model, inp.dtype))

    def _device_tables_apply(self, inp):
        r"""Whether the products over a device table take these tensors.  They want whole 16-byte chunks on
        16-byte boundaries, in the sizes and in where the tensors begin: parameters that are views into one flat
        buffer, or rows that begin inside another tensor, go the module's or the pipeline's way instead."""
        d_hidden, d_model = self.htoh4.weight.shape[1:]
        return (self._epilogue_activation() is not None and inp.is_cuda
                and inp.dtype in (torch.float32, torch.bfloat16, torch.float16)
                and self.htoh4.weight.dtype == inp.dtype and self.h4toh.weight.dtype == inp.dtype
                and os.environ.get("FMOE_EXPERT_EPILOGUE", "1") != "0"
                and os.environ.get("FMOE_DEVICE_TABLES", "1") != "0"
                and fmoe_native.linear_dev_supported(d_model, d_hidden, inp.dtype)
                and all(t is None or t.data_ptr() % 16 == 0 for t in
                        (inp, self.htoh4.weight, self.htoh4.bias, self.h4toh.weight, self.h4toh.bias)))

    def _epilogue_activation(self):
        from .fused_functions import _activation_code
        try:
            return _activation_code(self.activation)
        except NotImplementedError:
            return None


def _gate_code_or_none(activation):
    """The code of an activation that the kernels of gated experts and of experts in 8 bits have."""
    try:
        return _gate_activation_code(activation)
    except NotImplementedError:
        return None


def _is_its_product(linear):
    """Whether calling ``linear`` is :class:`FMoELinear`'s product of its parameters (or parametrised tensors) and nothing else: no module in its
    place, no ``forward`` or hook of its own."""
    return (isinstance(linear, FMoELinear) and type(linear).forward is FMoELinear.forward and "forward" not in linear.__dict__
            and not (linear._forward_hooks or linear._forward_pre_hooks or linear._backward_hooks or linear._backward_pre_hooks))


class _GatedExpert(_Expert):
    r"""All experts of a worker as gated blocks, ``h4toh(act(g) * u)`` with ``[g u] = htoh4(x)``: ``htoh4`` has ``2 * d_hidden`` outputs, the
    gate's first.  With SiLU, exact GELU, ReLU or no activation one call each way (:func:`fastermoe_amd.functions.gated_mlp`), else, or
    where a linear was replaced or has hooks or the call does not take the sizes, the modules one by one."""

    def __init__(self, num_expert, d_model, d_hidden, activation, rank=0, bias=True):
        super().__init__(num_expert, d_model, d_hidden, activation, rank=rank, bias=bias)
        self.htoh4 = FMoELinear(num_expert, d_model, 2 * d_hidden, bias=bias, rank=rank)

    def _checkpoints(self, inp):
        if self.act_checkpoint and inp.is_cuda and self._saves(inp):
            raise NotImplementedError("act_checkpoint does not take gated experts")
        return False

    def _one_call(self, inp):
        """The activation's code where the block is one call, else ``None``."""
        if not (inp.is_cuda and os.environ.get("FMOE_EXPERT_EPILOGUE", "1") != "0"
                and _is_its_product(self.htoh4) and _is_its_product(self.h4toh)
                and fmoe_native.gated_mlp_supported(inp.dtype, *self.h4toh.weight.shape[1:])
                and all(p is None or p.dtype == inp.dtype for linear in (self.htoh4, self.h4toh) for p in (linear.weight, linear.bias))):
            return None
        return _gate_code_or_none(self.activation)

    def forward(self, inp, fwd_expert_count):
        code = self._one_call(inp)
        self._checkpoints(inp)
        if code is not None:
            return gated_mlp(inp, fwd_expert_count, self.htoh4.weight, self.htoh4.bias, self.h4toh.weight, self.h4toh.bias, code)
        gate, linear = self.htoh4(inp, fwd_expert_count).chunk(2, dim=1)
        x = self.activation(gate) if self.activation is not None else gate
        return self.h4toh((x * linear).contiguous(), fwd_expert_count)

    def routed_forward(self, inp, pos_buf, slot_to_row, counts_dev, top_k, table=None):
        code = self._one_call(inp)
        if code is None or os.environ.get("FMOE_DEVICE_TABLES", "1") == "0":
            return None
        self._checkpoints(inp)
        if table is None:
            table = fmoe_native.segment_table(counts_dev, pos_buf.numel())
        return MOERoutedGatedMLP.apply(inp, self.htoh4.weight, self.htoh4.bias, self.h4toh.weight, self.h4toh.bias, pos_buf, slot_to_row, table,
                                       top_k, code, self._saves(inp))

    def routed_layer(self, inp, gate_w, gate_b, score, routing, top_k):
        return None

    def unchunked_is_faster(self, inp, n_slots):
        return True   # (the pipeline has no gated experts)


class _Int8Expert(nn.Module):
    r"""The experts of ``experts`` for inference, their weights in 8-bit integers with a scale to each output channel and their rows rounded to the same as they come (:func:`fastermoe_amd.functions.linear_int8`).
    Biases stay as they are."""

    act_checkpoint = False

    def __init__(self, experts):
        super().__init__()
        if type(experts) not in (_Expert, _GatedExpert):
            raise TypeError(f"only this package's own experts are held in 8 bits, got {type(experts).__name__}")
        self.activation, self.gated = experts.activation, isinstance(experts, _GatedExpert)
        if _gate_code_or_none(self.activation) is None:
            raise NotImplementedError(f"experts in 8 bits take SiLU, GELU, ReLU or no activation, got {self.activation!r}")
        for name in ("htoh4", "h4toh"):
            if not _is_its_product(getattr(experts, name)):
                raise TypeError(f"{name} is not just its product, and only that is held in 8 bits: it was replaced, or has a forward or hooks of its own")
        for name in ("htoh4", "h4toh"):
            linear = getattr(experts, name)
            q, scale = quantize_rows(linear.weight)
            halves = 2 if self.gated and name == "htoh4" else 1
            if not fmoe_native.linear_int8_supported(q.shape[2], q.shape[1] // halves, halves == 2, linear.weight.dtype):
                raise NotImplementedError(f"{name} of {tuple(q.shape)} is beyond the sizes of products in 8 bits for {linear.weight.dtype} rows")
            self.register_buffer(name + "_weight", q)
            self.register_buffer(name + "_scale", scale)
            self.register_buffer(name + "_bias", None if linear.bias is None else linear.bias.detach())

    def _apply(self, fn, recurse=True):
        # (scales are float32 and rows lie whole 16 bytes apart, whatever type or device the layer moves to)
        scales = {name: self._buffers[name] for name in ("htoh4_scale", "h4toh_scale")}
        super()._apply(fn, recurse)
        for name, scale in scales.items():
            if self._buffers[name].dtype != torch.float32:
                self._buffers[name] = scale.to(self._buffers[name].device)
        for name in ("htoh4_weight", "h4toh_weight"):
            self._buffers[name] = fmoe_native.int8_layout(self._buffers[name])
        return self

    def _product(self, inp, table, name, activation, gated, expert_count=None, **rows):
        bias = getattr(self, name + "_bias")
        return linear_int8(inp, expert_count, getattr(self, name + "_weight"), getattr(self, name + "_scale"),
                           None if bias is None else bias.to(inp.dtype), activation, gated, table, **rows)

    def _inference_only(self, inp):
        if torch.is_grad_enabled() and inp.requires_grad:
            raise NotImplementedError("experts in 8 bits have no gradients: call the layer under torch.no_grad()")

    def forward(self, inp, fwd_expert_count):
        self._inference_only(inp)
        with torch.no_grad():
            mid = self._product(inp, None, "htoh4", self.activation, self.gated, fwd_expert_count)
            return self._product(mid, None, "h4toh", None, False, fwd_expert_count)

    def routed_forward(self, inp, pos_buf, slot_to_row, counts_dev, top_k, table=None):
        self._inference_only(inp)
        with torch.no_grad():
            if table is None:
                table = fmoe_native.segment_table(counts_dev, pos_buf.numel())
            mid = self._product(inp, table, "htoh4", self.activation, self.gated, row_index=pos_buf, index_div=top_k)
            return self._product(mid, table, "h4toh", None, False)

    def routed_layer(self, inp, gate_w, gate_b, score, routing, top_k):
        return None

    def unchunked_is_faster(self, inp, n_slots):
        return True   # (the pipeline has no products in 8 bits)

    def _checkpoints(self, inp):
        return False


def _gen_policy(alpha):
    r"""Shadowing policy factory (fmoe/transformer.py:33-87).  Shadowing copies
    experts between workers; with one worker the policy selects nothing."""

    def _no_policy(all_experts_count, all_global_expert_count, num_expert, world_size, d_model, fused):
        return all_experts_count.new_zeros(world_size, num_expert, dtype=bool)

    return _no_policy


class FMoETransformerMLP(FMoE):
    r"""``Linear(d_model, d_hidden) -> activation -> Linear(d_hidden, d_model)`` per
    expert, any leading input shape (fmoe/transformer.py:89-139)."""

    _expert_class = _Expert

    def __init__(self, num_expert=32, d_model=1024, d_hidden=4096, world_size=1, mp_group=None,
                 moe_group=None, activation=torch.nn.GELU(), gate=NaiveGate, top_k=2,
                 expert_dp_comm="none", gate_hook=None, bias=True, mask=None, mask_dict=None):
        super().__init__(num_expert=num_expert, d_model=d_model, gate=gate, top_k=top_k,
                         world_size=world_size, mp_group=mp_group, moe_group=moe_group,
                         gate_hook=gate_hook, mask=mask, policy_fn=_gen_policy(d_hidden / d_model),
                         mask_dict=mask_dict)
        self.experts = self._expert_class(num_expert, d_model, d_hidden, activation, rank=self.mp_rank, bias=bias)
        self.mark_parallel_comm(expert_dp_comm)

    def forward(self, inp: torch.Tensor):
        if inp.dim() == 2 and inp.shape[1] == self.d_model:
            return super().forward(inp)
        original_shape = inp.shape
        inp = inp.reshape(-1, self.d_model)
        output = super().forward(inp)
        return output.reshape(original_shape)

    @property
    def act_checkpoint(self):
        r"""Whether a training step keeps what its backward needs of the experts' activations in 8 bits (off; ``FMOE_ACT_CHECKPOINT=1``
        turns it on): the same output, a quarter of the memory, gradients made where the numbers kept are.  The fused pipeline
        (``enable_fuse``) stands back for it."""
        return getattr(self.experts, "act_checkpoint", False)

    @act_checkpoint.setter
    def act_checkpoint(self, on):
        if not isinstance(self.experts, _Expert):
            raise AttributeError("act_checkpoint is a matter of this package's own experts")
        self.experts.act_checkpoint = bool(on)


    def quantize_experts(self):
        r"""Holds the experts in 8-bit integers from here on, for inference: weights with a scale to each output channel, rows rounded with a scale of their own
        as they come, exact sums.  Half of the memory of 16-bit weights, and half of the bytes that a decoding step reads.  The experts have no
        parameters afterwards; calls that would need their gradients raise.  Experts of another class, or with linears that were replaced or have hooks,
        are refused.  Returns the layer."""
        self.experts = _Int8Expert(self.experts)
        return self


def _gated_defaults(args, kwargs):
    """A layer's arguments, with SiLU where no activation is named (it is the seventh)."""
    return kwargs if len(args) > 6 or "activation" in kwargs else dict(kwargs, activation=nn.SiLU())


class FMoEGatedMLP(FMoETransformerMLP):
    r""":class:`FMoETransformerMLP` with gated experts (not in the reference): ``h4toh(activation(g) * u)`` with ``[g u] = htoh4(x)``, ``htoh4`` with
    ``2 * d_hidden`` outputs, the gate's first.  ``activation`` is SiLU unless given.  The pipeline of ``enable_fuse`` stands back for gated experts."""

    _expert_class = _GatedExpert

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **_gated_defaults(args, kwargs))


class FMoEPositionwiseFF(FMoETransformerMLP):
    r"""The layer in a transformer block, with the layer norm and the residual around it (``CustomizedMoEPositionwiseFF``,
    examples/transformer-xl/mem_transformer.py:379-409): ``x + layer(norm(x))`` with ``pre_lnorm``, else ``norm(x + layer(x))``, with dropout on
    the layer's output.  ``gated``: with gated experts, as :class:`FMoEGatedMLP` has them.  Further arguments are those of :class:`FMoETransformerMLP`."""

    def __init__(self, *args, pre_lnorm=False, dropout=0.0, gated=False, **kwargs):
        if gated:
            self._expert_class = _GatedExpert
        super().__init__(*args, **(_gated_defaults(args, kwargs) if gated else kwargs))
        self.layer_norm = nn.LayerNorm(self.d_model)
        self.pre_lnorm = pre_lnorm
        self.dropout = nn.Dropout(dropout)

    def _norm_kernel_applies(self, *tensors):
        """Whether calling ``layer_norm`` is the kernel on its parameters and nothing else."""
        norm, first = self.layer_norm, tensors[0]
        return (type(norm) is nn.LayerNorm and _no_hooks(norm) and norm.normalized_shape == (self.d_model,) and first.is_cuda
                and first.shape[-1:] == norm.normalized_shape and fmoe_native.layer_norm_supported(first.dtype) and not torch.is_autocast_enabled()
                and all(t.dtype == first.dtype and t.device == first.device and t.shape == first.shape for t in tensors)
                and all(p is None or (p.device == first.device and p.dtype in (first.dtype, torch.float32) and p.is_contiguous())
                        for p in (norm.weight, norm.bias))
                and (norm.weight is None or norm.bias is None or norm.weight.dtype == norm.bias.dtype))

    def forward(self, inp):
        norm = self.layer_norm
        if self.pre_lnorm:
            x = layer_norm(inp, norm.weight, norm.bias, norm.eps) if self._norm_kernel_applies(inp) else norm(inp)
            return inp + self.dropout(super().forward(x))
        out = self.dropout(super().forward(inp))
        if self._norm_kernel_applies(out, inp):
            return add_layer_norm(out, inp, norm.weight, norm.bias, norm.eps)[0]
        return norm(inp + out)
