"""Differentiable layers whose result for one sample does not depend on who shares its batch.

* ``group_norm``     — group normalisation + residual add + activation, channels last, one affine pair for everybody or
  one per client (ops/csrc/groupnorm_{fwd,bwd}.hip); the normalisation of federated models whose clients' data differ, and of
  differentially private ones, which a batch statistic would leak
* ``client_dropout`` — dropout from a counter-based generator keyed by the client, drawn again in the backward pass
  instead of stored (ops/csrc/dropout.hip)
* ``rope_axes``      — rotary positions with several axes for image and video tokens: no table whose length ties the
  parameters to one image size (ops/csrc/rope.hip)

CUDA tensors run the hand-written kernels (fp32, bf16 or fp16; anything else raises), CPU tensors, tensors wrapped by
``torch.func`` transforms, tensor subclasses that define their operations, those with a forward-mode tangent, and calls that
are traced or run under a dispatch mode the oracles of ``reference.py``.  Arguments are checked alike on both.  The gradients are
first-order: differentiating them again raises.  As with any operator, a backward pass is captured into a graph with no
eager graph of the same leaves alive: what that one left on the leaves belongs to its stream.  The autograd nodes are C++
(csrc/autograd.cpp): both passes run without the interpreter.
"""
import functools
import math
from ctypes import c_float

import torch
from torch.autograd import forward_ad

import blades_amd.ops as _ops

from . import reference as ref

_ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
_KINDS = ("elem", "channel", "sample")
_P_END = 1.0 - 2.0 ** -25  # rounds to 1 in 32 bits from here
_POS = (torch.int64, torch.float32)
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_wrapped = torch._C._functorch.is_functorch_wrapped_tensor
_PLAIN = (torch.Tensor, torch.nn.Parameter)
_loaded = None


def _tangent(t) -> bool:
    """Does ``t`` carry a forward-mode tangent?  The nodes of csrc/autograd.cpp know reverse mode alone."""
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def _nodes():
    global _loaded
    if _loaded is None:
        _loaded = _ops._h().autograd()
    return _loaded


def _recorded() -> bool:
    """Is somebody listening to the operations (``torch.jit.trace``, ``make_fx``, fake tensors, selective checkpoints)?  Of a
    kernel launched by address they would see the allocations alone."""
    return torch._C._is_tracing() or torch._C._len_torch_dispatch_stack() > 0


def _wrapper(t) -> bool:
    """A tensor subclass that defines its operations itself (and may have no memory of its own)."""
    return type(t) not in _PLAIN and torch._C._dispatch_keys(t).has(torch._C.DispatchKey.Python)


def _elementary(t) -> bool:
    """Must ``t`` go through operations that PyTorch sees?"""
    return _wrapped(t) or _wrapper(t) or _tangent(t)


def _own_kernel(name: str, t: torch.Tensor, *others) -> bool:
    if not t.is_cuda or _ops._FORCE_REFERENCE or _recorded() or _elementary(t):
        return False
    for o in others:
        if o is not None and _elementary(o):
            return False
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name}: CUDA tensors must be fp32, bf16 or fp16, got {t.dtype}")
    return True


def group_norm(x, groups: int, weight=None, bias=None, eps: float = 1e-5, act: str = "none", residual=None):
    """``act(group_norm(x) * weight + bias + residual)``.

    ``x [N, C, *]``, read channels last (other layouts are copied); ``weight`` / ``bias`` ``[C]``, or ``[K, C]``: one row
    for each of K clients that own N / K consecutive samples (their gradients then come per client).  ``act``: none, relu,
    gelu (erf) or silu.  Statistics, products and sums are 32-bit, the result is rounded once.  On the GPU a group has
    at most 2048 channels (1024 where C or an address rules out accesses of four), the layer at most 2^24 channels, fewer than
    2^24 samples and fewer than 2^30 pixels."""
    if x.dim() < 2 or not x.is_floating_point():
        raise ValueError(f"group_norm: expected a floating-point tensor [N, C, *], got {x.dtype} {tuple(x.shape)}")
    N, C = x.shape[0], x.shape[1]
    groups, eps = int(groups), float(eps)
    if groups < 1 or C < 1 or C % groups:
        raise ValueError(f"group_norm: {C} channels do not divide into {groups} groups")
    if act not in _ACTS:
        raise ValueError(f"group_norm: act must be one of {tuple(_ACTS)}, got {act!r}")
    if not eps >= 0.0:
        raise ValueError(f"group_norm: eps must not be negative, got {eps}")
    for t in (weight, bias):
        if t is None:
            continue
        if t.dim() not in (1, 2) or t.shape[-1] != C or not t.is_floating_point() or t.device != x.device or (
                t.dim() == 2 and (t.shape[0] < 1 or N % t.shape[0])):
            raise ValueError(f"group_norm: weight and bias must be floating-point [{C}] or [clients, {C}] tensors on {x.device}, "
                             f"the clients dividing {N} samples, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if weight is not None and bias is not None and weight.shape != bias.shape:
        raise ValueError(f"group_norm: weight {tuple(weight.shape)} and bias {tuple(bias.shape)} must be shared or per client "
                         f"alike")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"group_norm: residual must match x ({x.dtype} {tuple(x.shape)}), got {residual.dtype} "
                         f"{tuple(residual.shape)} on {residual.device}")
    if not _own_kernel("group_norm", x, weight, bias, residual) or x.numel() == 0:
        return ref.group_norm(x, groups, weight, bias, eps, act, residual)
    return _nodes().group_norm(x, groups, weight, bias, eps, _ACTS[act], residual)


def client_dropout(x, uids, seed: int, tag, layer: int, p: float, kind: str = "elem", layout: str = "major", scale=None):
    """``x`` with every element (``kind`` "elem"), channel ("channel"; elements for 1-D and 2-D inputs) or sample
    ("sample") dropped with probability ``p`` and the kept ones times ``scale`` (None: 1 / (1 - p)).

    ``layout`` "major": ``x [K * B, C, *]``, client k owning B consecutive samples; "inner": ``x [B, K * C, *]``, client k
    owning C consecutive channels.  ``uids``: int64 ``[K]``, the clients' keys (0-d: one client).  A client's draws depend
    on (seed, uid, tag, layer) and on the position inside its own share alone — not on K, the memory layout or the
    device — and equal ``client_dropout_mult``'s.  ``tag``: an int, or a 1-element int64 tensor that the kernel reads when it
    runs; changing that tensor between a forward pass and its backward pass raises."""
    if not x.is_floating_point() or x.dim() < 1:
        raise ValueError(f"client_dropout: expected a floating-point tensor, got {x.dtype} {tuple(x.shape)}")
    if kind not in _KINDS or layout not in ("major", "inner"):
        raise ValueError(f"client_dropout: kind must be one of {_KINDS}, layout major or inner, got {kind!r}, {layout!r}")
    p = float(p)
    if not 0.0 <= p < _P_END:
        raise ValueError(f"client_dropout: need 0 <= p < 1 in 32 bits, got {p}")
    K, by_value = uids.numel(), not torch.is_tensor(tag)
    if uids.dtype != torch.int64 or uids.dim() > 1 or K < 1 or uids.device != x.device:
        raise ValueError("client_dropout: uids must be an int64 vector (or scalar) of clients on x's device")
    if not by_value and (tag.dtype != torch.int64 or tag.numel() != 1 or tag.device != x.device):
        raise ValueError("client_dropout: tag must be an int or a 1-element int64 tensor on x's device")
    inner = layout == "inner"
    if inner and x.dim() < 2:
        raise ValueError("client_dropout: layout inner needs [B, K * C, *]")
    if x.shape[1 if inner else 0] % K:
        raise ValueError(f"client_dropout: {tuple(x.shape)} does not divide among {K} clients (layout {layout})")
    if x.numel() == 0:
        return x.clone()
    if not _own_kernel("client_dropout", x, uids, None if by_value else tag):
        return ref.client_dropout(x, uids, seed, tag, layer, p, kind, layout, scale)
    if uids.dim() == 0 or not uids.is_contiguous():
        uids = uids.reshape(-1).contiguous()
    least, times = _draw(p)
    code = 0 if kind == "elem" or (kind == "channel" and x.dim() <= 2) else 1 if kind == "channel" else 2
    return _nodes().client_dropout(x, uids, None if by_value else tag, int(tag) & 0xFFFFFFFF if by_value else 0,
                                   int(seed) & (2 ** 64 - 1), (2 + 256 * int(layer)) & 0xFFFFFFFF, least, times if scale is None else float(scale), code,
                                   inner)


@functools.lru_cache(maxsize=256)
def _draw(p: float):
    """(smallest 24-bit draw that is kept, 1 / (1 - p)): p rounded to 32 bits, as draws are compared with it, and the quotient
    rounded to 32 bits once (from a rounded 1 - p it would be off by 1e-6 of itself at p = 0.99)."""
    return math.ceil(c_float(p).value * 16777216.0), c_float(1.0 / (1.0 - p)).value


def rope_axes(x, pos, axes, base: float = 10000.0, slots=None):
    """Rotary positions with one section of the head dimension per axis.

    ``x [R, N, H, D]`` (queries or keys), or ``[R, N, S, H, D]``, the packed projection, whose first ``slots`` slots (None:
    all) are turned and whose others are copied.  ``axes``: even widths of the sections, one per axis, together at most D
    (the rest of the head passes through).  ``pos``: int64 or fp32 positions, ``[N, A]`` shared by the samples or
    ``[R, N, A]``.  Pair (2i, 2i + 1) of a section d wide is turned by ``pos * base ** (-2 i / d)``; angles are 64-bit.
    D is even, at most 256; at most 8 axes; on the GPU S * H is at most 10^9."""
    if x.dim() not in (4, 5) or not x.is_floating_point():
        raise ValueError(f"rope_axes: expected a floating-point [R, N, H, D] or [R, N, S, H, D] tensor, got {x.dtype} "
                         f"{tuple(x.shape)}")
    axes, base = tuple(int(a) for a in axes), float(base)
    D, S = x.shape[-1], x.shape[2] if x.dim() == 5 else 1
    if not axes or len(axes) > 8 or any(a < 2 or a % 2 for a in axes) or sum(axes) > D or D % 2 or D > 256:
        raise ValueError(f"rope_axes: 1 to 8 even sections that fit an even head dimension of at most 256 are needed, got "
                         f"{axes} for {D}")
    slots = S if slots is None else int(slots)
    if not 0 <= slots <= S:
        raise ValueError(f"rope_axes: slots must lie in 0 .. {S}, got {slots}")
    if not 0.0 < base < float("inf"):
        raise ValueError(f"rope_axes: base must be positive and finite, got {base}")
    shape = pos.shape
    if pos.dtype not in _POS or shape[-2:] != (x.shape[1], len(axes)) or len(shape) > 3 or (
            len(shape) == 3 and shape[0] != x.shape[0]) or pos.device != x.device or pos.requires_grad:
        raise ValueError(f"rope_axes: pos must be int64 or fp32 [{x.shape[1]}, {len(axes)}] or [{x.shape[0]}, {x.shape[1]}, "
                         f"{len(axes)}] on {x.device} without a gradient, got {pos.dtype} {tuple(shape)} on {pos.device}")
    if not _own_kernel("rope_axes", x, pos):
        return ref.rope_axes(x, pos, axes, base, slots)
    return _nodes().rope_axes(x, pos, axes, base, slots)
