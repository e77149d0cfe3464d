"""Activations in 8 bits for the backward pass: `checkpoint_pack` / `checkpoint_unpack`, and the gradients of the two operators at such a
checkpoint of their input.  A layer differentiated the ordinary way keeps its input, its output and a workspace; with a checkpoint
it keeps one byte per input value and 8 (float64: 16) per group, and computes the rest again.  The gradients are those of the operator at
the values that the checkpoint stands for, which lie within half a step, 1 / 504 of the range of a group, of the input (in a group whose
range is below 252 of the type's smallest normal number all values become its lowest one).

The reference has no counterpart: its graphs keep every activation (HUJI-Deep/simnets-tf python/simnets/ops/mex.py:47-81 takes the op's
input and output into the gradient ops)."""
import math

import torch

from .. import _lib
from .. import _torch_glue
from .mex import _attrs as _mex_attrs, mex_plan
from .similarity import _attrs as _sim_attrs, similarity_plan_of_shape

GROUPS = (32, 64, 128, 256)


def check_group(group):
    """`group` as a group length of a checkpoint (a ValueError if it is none)."""
    if isinstance(group, bool) or group not in GROUPS:
        raise ValueError("a checkpoint's group must be one of %s, got %r" % (list(GROUPS), group))
    return int(group)


class Checkpoint(object):
    """An activation in 8 bits: `codes` (uint8, one per value in memory order), `ranges` ([groups, 2]: lowest value and step of every
    `group` consecutive values, in the type of the values) and the activation's `shape`."""

    __slots__ = ("codes", "ranges", "shape", "group")

    def __init__(self, codes, ranges, shape, group=128):
        self.group = check_group(group)
        self.shape = tuple(int(s) for s in shape)
        n = math.prod(self.shape)
        if any(s < 0 for s in self.shape):
            raise ValueError("a checkpoint's shape must not be negative, got %s" % (self.shape,))
        if codes.dtype != torch.uint8:
            raise TypeError("codes must be uint8, got %s" % codes.dtype)
        _torch_glue.dtype_code(ranges)
        if codes.numel() != n or tuple(ranges.shape) != (-(-n // self.group), 2):
            raise ValueError("a checkpoint of %s in groups of %d has %d codes and %d ranges, got %d and %s"
                             % (self.shape, self.group, n, -(-n // self.group), codes.numel(), tuple(ranges.shape)))
        if codes.device != ranges.device:
            raise RuntimeError("codes and ranges must be on the same device")
        self.codes, self.ranges = _torch_glue.plain(codes), _torch_glue.plain(ranges)

    @classmethod
    def _packed(cls, codes, ranges, shape, group):
        """What the library has packed itself: nothing to check."""
        self = cls.__new__(cls)
        self.codes, self.ranges, self.shape, self.group = codes, ranges, tuple(shape), group
        return self

    @property
    def dtype(self):
        """Type of the values."""
        return self.ranges.dtype

    @property
    def device(self):
        return self.codes.device

    def nbytes(self):
        return self.codes.numel() + self.ranges.numel() * self.ranges.element_size()


def checkpoint_pack(input, group=128):
    """A `Checkpoint` of a float32 or float64 CUDA tensor.  Infinities and NaN are kept as such; NaN entries and infinities do not count
    towards a group's range.  Not differentiable: `mex_checkpointed` and `similarity_checkpointed` are."""
    group = check_group(group)
    codes, ranges = _lib.ops().checkpoint_pack(input, group)
    return Checkpoint._packed(codes, ranges, input.shape, group)


def checkpoint_unpack(checkpoint):
    """The activation that a checkpoint stands for."""
    return _lib.ops().checkpoint_unpack(checkpoint.codes, checkpoint.ranges, list(checkpoint.shape), checkpoint.group)


def _four(checkpoint):
    if len(checkpoint.shape) != 4:
        raise ValueError("the checkpoint of an operator's input must be 4-D, got %s" % (checkpoint.shape,))
    return checkpoint.shape


def mex_checkpoint_backward(checkpoint, offsets, output_grad, num_instances, flags=0, pooled=False, doff_out=None, **attrs):
    """(input_grad, offsets_grad) of the `Mex` op at a checkpoint of its input; the output is computed again.  `pooled`, FLAG_ACCUMULATE
    with `doff_out`, and `attrs` as in `mex_backward`.  Sums are in FP32; abi.FLAG_MEX_CHECKPOINT_TENSORCORE (which `mex_checkpointed` and the
    layers set) lets blocks of more than 128 taps take the tensor-core kernels of the ordinary gradients, with their accuracy."""
    plan = mex_plan(_four(checkpoint), checkpoint.dtype, num_instances, _mex_attrs(**attrs))
    return _lib.ops().mex_checkpoint_backward(plan, checkpoint.codes, checkpoint.ranges, checkpoint.group, offsets, output_grad, flags, pooled, doff_out)


def similarity_checkpoint_backward(checkpoint, templates, weights, output_grad, flags=0, out=None, **attrs):
    """(input_grad, templates_grad, weights_grad) of the `Similarity` op at a checkpoint of its input.  `out`, `flags` and `attrs` as in
    `similarity_parameters_grad`."""
    plan = similarity_plan_of_shape(_four(checkpoint), checkpoint.dtype, templates, weights, _sim_attrs(**attrs))
    dt, dw = out if out is not None else (None, None)
    return _lib.ops().sim_checkpoint_backward(plan, checkpoint.codes, checkpoint.ranges, checkpoint.group, templates, weights, output_grad, flags, dt, dw)


def mex_checkpointed_with_plan(plan_of, input, offsets, group, layer_ws=None, fwd_flags=0, op_flags=0, sum_pool2=False, grad_sink=None):
    """`mex_with_plan` (on the plan `plan_of(input)`) that keeps a checkpoint of `input` for its gradients."""
    def call(x, o, sink=None):
        plan, apply = plan_of(x), _lib.ops().mex_checkpoint_apply
        if sum_pool2 and (plan.height_out % 2 or plan.width_out % 2):
            return torch.nn.functional.avg_pool2d(apply(plan, x, o, group, layer_ws, fwd_flags, op_flags, False, sink), 2) * 4.0
        return apply(plan, x, o, group, layer_ws, fwd_flags, op_flags, sum_pool2, sink)

    if _torch_glue.is_tracing():            # (its gradients go through autograd, also to the `.grad` that a sink stands for)
        return _torch_glue.recorded(call, input, offsets)
    return call(input, offsets, grad_sink)


def similarity_checkpointed_with_plan(plan_of, input, templates, weights, group, flags=0, extrema=None, grad_sinks=None):
    """The differentiable Similarity op on the plan `plan_of(input, templates, weights)`, keeping a checkpoint of `input`."""
    up, down = extrema if extrema is not None else (None, None)

    def call(x, t, w, sinks=None):
        dt, dw = sinks if sinks is not None else (None, None)
        return _lib.ops().sim_checkpoint_apply(plan_of(x, t, w), x, t, w, group, flags, up or 0, down or 0, dt, dw)

    if _torch_glue.is_tracing():
        return _torch_glue.recorded(call, input, templates, weights)
    return call(input, templates, weights, grad_sinks)


def mex_checkpointed(input, offsets, num_instances, group=128, sum_pool2=False, **attrs):
    """`mex(...)` (with sum_pool2=True `mex_sum_pool2(...)`), differentiable (once), keeping its input in 8 bits and nothing else."""
    group, attrs = check_group(group), _mex_attrs(**{k: v for k, v in attrs.items() if k != "name"})
    _torch_glue.dtype_code(input)
    return mex_checkpointed_with_plan(lambda x: mex_plan(x.shape, x.dtype, num_instances, attrs), input, offsets, group, sum_pool2=sum_pool2)


def similarity_checkpointed(input, templates, weights, group=128, **attrs):
    """`similarity(...)`, differentiable (once), keeping its input in 8 bits and its parameters."""
    group, attrs = check_group(group), _sim_attrs(**{k: v for k, v in attrs.items() if k != "name"})
    return similarity_checkpointed_with_plan(lambda x, t, w: similarity_plan_of_shape(tuple(x.shape), x.dtype, t, w, attrs), input, templates, weights, group)
