"""Operators of deep stacks with large outputs, on CUDA ``torch`` tensors.

    new, normed, stats = residual_norm(stream, branch, gate=gate, post_weight=wp, pre_weight=wn)
    out, packed = activate_and_pack(preact, "gelu")
    loss, lse = vocab_cross_entropy(normed, weight, targets)

Each has an explicit gradient (``residual_norm_backward``, ``packed_activation_backward``,
``vocab_cross_entropy_backward``): like the layers of this package, and unlike torch's own functions,
they record nothing for automatic differentiation, and their results carry no history.

Tensors are float32 or bfloat16, all of a call alike, on one device.  Leading dimensions are free and count as
rows, as far as one stride describes them; the last dimension is contiguous.  Work is enqueued on torch's current
stream of the tensors' device; results and workspaces come from torch's allocator, so that calls can be
captured into CUDA graphs and made on several streams at once.  Nothing waits for the GPU.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional

from . import _lib
from .layer import ACT_IDS, Activation

BLOCK = 128  # elements of a row that share a scale
_NORMS = {"rms": 0, "layer": 1}


def _torch():
    import torch
    return torch


def _stream(torch, device):
    """The handle of torch's current stream; without the Stream object around it where torch offers that (7 us less)."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device.index) if raw is not None else torch.cuda.current_stream(device).cuda_stream


class _Call:
    """What the tensors of one call have in common: type and device, taken from the first.  (Few and cheap
    steps: a call for one token is bound by the host.)"""
    __slots__ = ("torch", "name", "first", "dtype", "device", "type")

    def __init__(self, name, first_name, first):
        torch = self.torch = _torch()
        self.name = name
        if not isinstance(first, torch.Tensor):
            raise TypeError(f"{name}: {first_name} has to be a torch tensor, not {type(first).__name__}")
        self.first, self.dtype, self.device = first, first.dtype, first.device
        if self.dtype is torch.bfloat16:
            self.type = 1
        elif self.dtype is torch.float32:
            self.type = 0
        else:
            raise TypeError(f"{name}: {first_name} is {first.dtype}; float32 and bfloat16 are supported")
        if not first.is_cuda:
            raise ValueError(f"{name}: {first_name} is on {first.device}; there is no CPU path")

    def tensor(self, label, t, dtype=None):
        if not isinstance(t, self.torch.Tensor):
            raise TypeError(f"{self.name}: {label} has to be a torch tensor, not {type(t).__name__}")
        if t.dtype is not (dtype or self.dtype):
            raise TypeError(f"{self.name}: {label} is {t.dtype}, {dtype or self.dtype} is needed")
        if t.device != self.device:
            raise ValueError(f"{self.name}: {label} is on {t.device}, the call on {self.device}")
        return t

    def matrix(self, label, t, shape=None):
        """(rows, width, row stride) of a tensor whose leading dimensions one stride describes."""
        found = self.tensor(label, t).shape
        if shape is not None and found != shape:
            raise ValueError(f"{self.name}: {label} is {tuple(found)}, {tuple(shape)} is needed")
        if len(found) < 2:
            raise ValueError(f"{self.name}: {label} needs two dimensions at least, it has {t.dim()}")
        width = found[-1]
        rows = found[0] if len(found) == 2 else math.prod(found[:-1])
        if t.is_contiguous():
            return rows, width, max(width, 1)
        if width > 1 and t.stride(-1) != 1:
            raise ValueError(f"{self.name}: the last dimension of {label} has to be contiguous")
        try:
            stride = t.view(rows, width).stride(0)
        except RuntimeError:
            raise ValueError(f"{self.name}: no one stride describes the rows of {label}: make it contiguous") from None
        return rows, width, max(width, 1) if rows <= 1 else stride

    def vector(self, label, t, width):
        if t is None:
            return None
        if self.tensor(label, t).shape != (width,) or not t.is_contiguous():
            raise ValueError(f"{self.name}: {label} has to be a contiguous vector of {width}")
        return t.data_ptr()

    def empty(self, shape, dtype=None):
        return self.first.new_empty(shape, dtype=dtype or self.dtype)

    def like(self, t, dtype=None):
        """An empty contiguous tensor of t's shape, in the call's type."""
        if t.is_contiguous():  # (half the time of the general form)
            return self.torch.empty_like(t) if dtype is None else self.torch.empty_like(t, dtype=dtype)
        return self.empty(t.shape, dtype)

    def run(self, function, *args, workspace=None, call=None):
        """function(stream, *args) on torch's current stream of the tensors' device; ``workspace(call, size)`` tells
        first how much the call needs."""
        cuda = self.torch.cuda
        if cuda.current_device() != self.device.index:
            with cuda.device(self.device):
                return self.run(function, *args, workspace=workspace, call=call)
        if call is not None:
            if workspace is not None:
                size = ctypes.c_size_t()
                _lib.check(workspace(size))
                held = self.empty(size.value, self.torch.uint8)  # (its memory is reused in stream order)
                call.workspace, call.workspace_bytes = held.data_ptr(), size.value
            args = (ctypes.byref(call),)
        _lib.check(function(_stream(self.torch, self.device), *args))


# ------------------------------------------------------------------------------ vocabulary loss
class VocabGradients(NamedTuple):
    hidden: object
    weight: object
    bias: Optional[object]


def _vocab_call(call, hidden, weight, targets, bias, scale, ignore_index):
    rows, width, hidden_stride = call.matrix("hidden", hidden)
    vocab, weight_width, weight_stride = call.matrix("weight", weight)
    if weight.dim() != 2 or weight_width != width:
        raise ValueError(f"{call.name}: weight is {tuple(weight.shape)}, (vocabulary, {width}) is needed")
    if call.tensor("targets", targets, call.torch.int64).shape != hidden.shape[:-1]:
        raise ValueError(f"{call.name}: targets is {tuple(targets.shape)}, {tuple(hidden.shape[:-1])} is needed")
    targets = targets.contiguous()
    c = _lib.VocabCe(rows=rows, width=width, vocab=vocab, hidden_stride=hidden_stride, weight_stride=weight_stride,
                     type=call.type, scale=scale, ignore_index=ignore_index, hidden=hidden.data_ptr(),
                     weight=weight.data_ptr(), bias=call.vector("bias", bias, vocab), targets=targets.data_ptr())
    return c, targets


def vocab_cross_entropy(hidden, weight, targets, bias=None, *, scale: float = 1.0, ignore_index: int = -100):
    """Softmax cross entropy of ``hidden`` [..., width] against a vocabulary ``weight`` [vocab, width], without
    ever keeping the logits ``scale * hidden @ weight.T + bias``.

    Returns ``(loss, lse)``, float32 of ``targets``' shape: the loss of every row and the logarithm of its sum of
    exponentials, which ``vocab_cross_entropy_backward`` needs.  Rows whose target (int64) is ``ignore_index`` or
    outside the vocabulary are ignored: both are 0, whatever the row holds."""
    call = _Call("vocab_cross_entropy", "hidden", hidden)
    c, targets = _vocab_call(call, hidden, weight, targets, bias, scale, ignore_index)
    lib = _lib.load()
    loss, lse = call.like(targets, call.torch.float32), call.like(targets, call.torch.float32)
    c.loss, c.lse = loss.data_ptr(), lse.data_ptr()
    call.run(lib.dpc_vocab_ce_forward, call=c,
             workspace=lambda size: lib.dpc_vocab_ce_workspace(ctypes.byref(c), 0, ctypes.byref(size)))
    return loss, lse


def vocab_cross_entropy_backward(grad_loss, hidden, weight, targets, lse, bias=None, *, scale: float = 1.0,
                                 ignore_index: int = -100) -> VocabGradients:
    """Gradients of ``vocab_cross_entropy`` with respect to hidden, weight and bias (None without one), in
    their type.  ``grad_loss``: float32, the gradient of every row's loss, or one value for all rows; ``lse``
    as the forward call returned it."""
    call = _Call("vocab_cross_entropy_backward", "hidden", hidden)
    torch = call.torch
    c, targets = _vocab_call(call, hidden, weight, targets, bias, scale, ignore_index)
    lib = _lib.load()
    if call.tensor("lse", lse, torch.float32).shape != targets.shape:
        raise ValueError(f"{call.name}: lse is {tuple(lse.shape)}, {tuple(targets.shape)} is needed")
    call.tensor("grad_loss", grad_loss, torch.float32)
    if grad_loss.numel() != 1 and grad_loss.shape != targets.shape:
        raise ValueError(f"{call.name}: grad_loss is {tuple(grad_loss.shape)}, {tuple(targets.shape)} or one value is needed")
    one = grad_loss.numel() == 1 or (grad_loss.numel() > 1 and not any(grad_loss.stride()))
    grad_loss, lse = grad_loss if one else grad_loss.contiguous(), lse.contiguous()
    d_hidden, d_weight = call.like(hidden), call.like(weight)
    d_bias = None if bias is None else call.like(bias)
    c.lse, c.grad_loss, c.grad_stride = lse.data_ptr(), grad_loss.data_ptr(), 0 if one else 1
    c.d_hidden, c.d_hidden_stride = d_hidden.data_ptr(), c.width
    c.d_weight, c.d_weight_stride = d_weight.data_ptr(), c.width
    c.d_bias = None if bias is None else d_bias.data_ptr()
    call.run(lib.dpc_vocab_ce_backward, call=c,
             workspace=lambda size: lib.dpc_vocab_ce_workspace(ctypes.byref(c), 1, ctypes.byref(size)))
    return VocabGradients(d_hidden, d_weight, d_bias)


# ------------------------------------------------------------------------------ residual norms
class ResidualNormGradients(NamedTuple):
    stream: object
    branch: Optional[object]
    gate: Optional[object]
    post_weight: Optional[object]
    post_bias: Optional[object]
    pre_weight: Optional[object]
    pre_bias: Optional[object]


def _norm_call(call, like, branch, norm, post_norm, post_weight, post_bias, gate, stream_scale, branch_scale,
               pre_weight, pre_bias, eps):
    if norm not in _NORMS:
        raise ValueError(f"{call.name}: norm {norm!r} is none of {sorted(_NORMS)}")
    rows, width, stride = call.matrix("the residual stream", like)
    post_norm = post_weight is not None or post_bias is not None if post_norm is None else bool(post_norm)
    c = _lib.ResidualNorm(rows=rows, width=width, groups=1, type=call.type, norm=_NORMS[norm], post_norm=post_norm,
                          stream_scale=stream_scale, branch_scale=branch_scale, eps=eps,
                          post_weight=call.vector("post_weight", post_weight, width),
                          post_bias=call.vector("post_bias", post_bias, width),
                          pre_weight=call.vector("pre_weight", pre_weight, width),
                          pre_bias=call.vector("pre_bias", pre_bias, width), stream_stride=stride,
                          new_stream_stride=stride)
    if branch is not None:
        c.branch_stride = call.matrix("branch", branch, like.shape)[2]
        c.branch = branch.data_ptr()
    elif post_norm or gate is not None or stream_scale != 1.0:
        raise ValueError(f"{call.name}: without a branch there is no gate, post norm or stream scale")
    if gate is not None:
        table = call.tensor("gate", gate)
        table = table[None] if table.dim() == 1 else table
        c.groups, gate_width, c.gate_stride = call.matrix("gate", table)
        if rows == 0 and c.groups == 0:
            c.groups = 1  # no sequences, each with a gate of its own
        if gate_width != width or c.groups < 1 or rows % c.groups:
            raise ValueError(f"{call.name}: gate is {tuple(gate.shape)}; its last dimension has to be {width}, and "
                             f"its rows have to divide {rows}")
        c.gate = gate.data_ptr()
    if rows == 0:  # empty tensors have no addresses: the presence of each operand is what counts
        c.branch = None if branch is None else 16
        c.gate = None if gate is None else 16
    return c


def residual_norm(stream, branch=None, *, norm: str = "rms", post_norm: Optional[bool] = None, post_weight=None,
                  post_bias=None, gate=None, stream_scale: float = 1.0, branch_scale: float = 1.0, pre_weight=None,
                  pre_bias=None, eps: float = 1e-6):
    """The end of one residual block and the norm before the next, in one pass:

        new_stream = stream_scale * stream + branch_scale * gate * (norm(branch) * post_weight + post_bias)
        normed = norm(new_stream) * pre_weight + pre_bias

    ``stream`` and ``branch`` [..., width]; ``norm``: "rms" or "layer"; ``post_norm=False`` (the default without
    post weights) takes the branch as it is.  ``gate``: [width], or [groups, width] (also [..., width]) for as many equal
    runs of rows, e.g. one of a sequence.  Without a branch (before the first block) new_stream is ``stream`` itself.

    Returns ``(new_stream, normed, stats)``; ``stats`` (float32 [..., 4]: mean and 1/deviation of the branch and of the new stream)
    goes to ``residual_norm_backward`` with ``new_stream`` and ``branch``."""
    call = _Call("residual_norm", "stream", stream)
    c = _norm_call(call, stream, branch, norm, post_norm, post_weight, post_bias, gate, stream_scale, branch_scale,
                   pre_weight, pre_bias, eps)
    lib = _lib.load()
    c.stream = stream.data_ptr()
    new_stream = stream if branch is None else call.like(stream)
    normed = call.like(stream)
    stats = call.empty((*stream.shape[:-1], 4), call.torch.float32)
    if branch is not None:
        c.new_stream, c.new_stream_stride = new_stream.data_ptr(), c.width
    c.normed, c.normed_stride, c.stats = normed.data_ptr(), c.width, stats.data_ptr()
    call.run(lib.dpc_residual_norm_forward, call=c)
    return new_stream, normed, stats


def residual_norm_backward(d_normed, d_stream, new_stream, branch, stats, *, norm: str = "rms",
                           post_norm: Optional[bool] = None, post_weight=None, post_bias=None, gate=None,
                           stream_scale: float = 1.0, branch_scale: float = 1.0, pre_weight=None,
                           pre_bias=None) -> ResidualNormGradients:
    """Gradients of ``residual_norm`` from those of ``normed`` and of the new stream (``d_stream``; None where nothing
    else reads it), with the tensors and options of the forward call.  What was not given has None."""
    call = _Call("residual_norm_backward", "new_stream", new_stream)
    c = _norm_call(call, new_stream, branch, norm, post_norm, post_weight, post_bias, gate, stream_scale, branch_scale,
                   pre_weight, pre_bias, 0.0)
    lib, shape, width = _lib.load(), new_stream.shape, c.width
    c.new_stream = new_stream.data_ptr()
    c.d_normed_stride = call.matrix("d_normed", d_normed, shape)[2]
    c.d_normed = d_normed.data_ptr()
    if d_stream is not None:
        c.d_new_stream_stride = call.matrix("d_stream", d_stream, shape)[2]
        c.d_new_stream = d_stream.data_ptr()
    if tuple(call.tensor("stats", stats, call.torch.float32).shape) != (*shape[:-1], 4) or not stats.is_contiguous():
        raise ValueError(f"{call.name}: stats has to be the tensor that residual_norm returned")
    c.stats = stats.data_ptr()
    d_in = call.like(new_stream)
    c.d_stream, c.d_stream_stride = d_in.data_ptr(), width
    d_branch = None if branch is None else call.like(branch)
    if branch is not None:
        c.d_branch, c.d_branch_stride = (d_branch.data_ptr() if c.rows else 16), width
    d_gate = None if gate is None else call.like(gate)
    if gate is not None:
        c.d_gate, c.d_gate_stride = d_gate.data_ptr(), width
    vectors = {}
    for label, t in (("post_weight", post_weight), ("post_bias", post_bias), ("pre_weight", pre_weight),
                     ("pre_bias", pre_bias)):
        vectors[label] = None if t is None else call.like(t)
        if t is not None:
            setattr(c, "d_" + label, vectors[label].data_ptr())
    call.run(lib.dpc_residual_norm_backward, call=c,
             workspace=lambda size: lib.dpc_residual_norm_workspace(ctypes.byref(c), ctypes.byref(size)))
    return ResidualNormGradients(stream=d_in, branch=d_branch, gate=d_gate, **vectors)


# ------------------------------------------------------------------------------ packed activations
def _activation(name, activation):
    key = activation.to_string() if isinstance(activation, Activation) else activation
    if key not in ACT_IDS:
        raise ValueError(f"{name}: activation {activation!r} is none of {sorted(ACT_IDS)}")
    return ACT_IDS[key]


class PackedActivations:
    """A tensor [..., width] in 8 bits: ``codes`` (int8, its shape) and ``scales`` (float32 [..., ceil(width / 128)]);
    the value of an element is its code times its block's scale."""

    def __init__(self, codes, scales):
        torch = _torch()
        if not torch.is_tensor(codes) or codes.dtype != torch.int8 or codes.dim() < 2 or not codes.is_contiguous():
            raise ValueError("PackedActivations: codes has to be a contiguous int8 tensor [..., width]")
        shape = (*codes.shape[:-1], -(-codes.shape[-1] // BLOCK))
        if not torch.is_tensor(scales) or scales.dtype != torch.float32 or tuple(scales.shape) != shape or \
                not scales.is_contiguous() or scales.device != codes.device:
            raise ValueError(f"PackedActivations: scales has to be a contiguous float32 tensor {shape} beside the codes")
        self.codes, self.scales = codes, scales

    @property
    def shape(self):
        return self.codes.shape

    def unpack(self, dtype=None):
        """The values, in ``dtype`` (float32 or bfloat16; default float32)."""
        torch = _torch()
        out = torch.empty(self.shape, dtype=dtype or torch.float32, device=self.codes.device)
        call = _Call("PackedActivations.unpack", "the result", out)
        _packed_backward(call, self, ACT_IDS["linear"], None, None, out)
        return out


def _packed_backward(call, packed, act, d_out, d_preact, out):
    lib = _lib.load()
    width = packed.shape[-1]
    rows = math.prod(packed.shape[:-1])
    stride = 0 if d_out is None else call.matrix("d_out", d_out, packed.shape)[2]
    call.run(lib.dpc_packed_activation_backward, call.type, act, rows, width, packed.codes.data_ptr(),
             packed.scales.data_ptr(), None if d_out is None else d_out.data_ptr(), stride,
             None if d_preact is None else d_preact.data_ptr(), width, None if out is None else out.data_ptr(), width)


def activate_and_pack(preact, activation):
    """``(f(preact), packed)``: a layer's activation (a name such as "gelu", or an ``Activation``), with the
    pre-activation [..., width] kept in 8 bits for ``packed_activation_backward``.  Every 128 neighbours of the last dimension share
    a scale, so an element is off by 1/254 of its block's largest at most; a block with nothing of 2^-100 or larger becomes zeros, one with
    an infinity or a NaN becomes NaN."""
    call = _Call("activate_and_pack", "preact", preact)
    act = _activation(call.name, activation)
    rows, width, stride = call.matrix("preact", preact)
    if width < 1:
        raise ValueError(f"{call.name}: preact has no columns")
    lib = _lib.load()
    out, codes = call.like(preact), call.like(preact, call.torch.int8)
    scales = call.empty((*preact.shape[:-1], -(-width // BLOCK)), call.torch.float32)
    call.run(lib.dpc_activate_and_pack, call.type, act, rows, width, preact.data_ptr(), stride, out.data_ptr(), width,
             codes.data_ptr(), scales.data_ptr())
    return out, PackedActivations(codes, scales)


def packed_activation_backward(d_out, packed, activation, *, recompute: bool = False):
    """``(d_preact, out)`` from the gradient of the activation's output: ``d_out * f'(x)`` at the kept x and, with
    ``recompute``, ``f(x)`` again (else None), which the next layer's weight gradient reads."""
    call = _Call("packed_activation_backward", "d_out", d_out)
    act = _activation(call.name, activation)
    if not isinstance(packed, PackedActivations):
        raise TypeError(f"{call.name}: packed is a {type(packed).__name__}, not PackedActivations")
    call.tensor("packed", packed.codes, call.torch.int8)
    d_preact = call.like(d_out)
    out = call.like(d_out) if recompute else None
    _packed_backward(call, packed, act, d_out, d_preact, out)
    return d_preact, out
