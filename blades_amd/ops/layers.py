"""Differentiable layers whose result for one sample does not depend on who shares its batch.

* ``group_norm``     — group normalisation + residual add + activation, channels last, one affine pair for everybody or
  one per client (ops/csrc/groupnorm.hip); the normalisation of federated models whose clients' data differ, and of
  differentially private ones, which a batch statistic would leak
* ``client_dropout`` — dropout from a counter-based generator keyed by the client, drawn again in the backward pass
  instead of stored (ops/csrc/dropout.hip)
* ``rope_axes``      — rotary positions with several axes for image and video tokens: no table whose length ties the
  parameters to one image size (ops/csrc/rope.hip)

CUDA tensors run the hand-written kernels (fp32, bf16 or fp16; anything else raises), CPU tensors and tensors wrapped by
``torch.func`` transforms the oracles of ``reference.py``.  Arguments are checked alike on both.  The gradients are
first-order: a second backward pass raises.
"""
import torch
from torch.autograd.function import once_differentiable

import blades_amd.ops as _ops

from . import reference as ref

_ACTS = ("none", "relu", "gelu", "silu")
_KINDS = ("elem", "channel", "sample")
_P_END = 1.0 - 2.0 ** -25  # rounds to 1 in 32 bits from here
_POS = (torch.int64, torch.float32)
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_wrapped = torch._C._functorch.is_functorch_wrapped_tensor
_grad_mode = torch.is_grad_enabled
_kernels = None


def _h():
    global _kernels
    if _kernels is None:
        _kernels = _ops._h()
    return _kernels


def _own_kernel(name: str, t: torch.Tensor) -> bool:
    if not t.is_cuda or _ops._FORCE_REFERENCE or _wrapped(t):
        return False
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name}: CUDA tensors must be fp32, bf16 or fp16, got {t.dtype}")
    return True


def _first_order(backward):
    """A backward that must not be differentiated again.  torch's wrapper for that costs 6 us a call; it is only needed
    while a graph of the backward pass is being built."""
    guarded = once_differentiable(backward)

    def call(ctx, gy):
        return guarded(ctx, gy) if _grad_mode() else backward(ctx, gy)

    return call


class _GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, cfg):
        groups, eps, act = cfg
        w, b = _affine(weight), _affine(bias)
        clients = _clients(w, b)
        y, stats, gate, plan = _h().group_norm_forward(x, groups, w, b, eps, act, residual, clients, True, True)
        lead = None  # the types of affine vectors that are not fp32
        if w is not None and weight.dtype != w.dtype or b is not None and bias.dtype != b.dtype:
            lead = (None if weight is None else weight.dtype, None if bias is None else bias.dtype)
        ctx.cfg = (groups, act, clients, plan, lead)
        # the gate stands in for the residual; without one z is computed again, from x and a smooth activation's residual
        ctx.save_for_backward(x, w, b, stats, residual if act in ("gelu", "silu") else None, gate)
        return y

    @staticmethod
    @_first_order
    def backward(ctx, gy):
        x, w, b, stats, res, gate = ctx.saved_tensors
        groups, act, clients, plan, lead = ctx.cfg
        nx, nw, nb, nr, _ = ctx.needs_input_grad
        dw = torch.empty(w.shape, device=x.device) if nw else None
        db = torch.empty(b.shape, device=x.device) if nb else None
        dx, dres = _kernels.group_norm_backward(x, gy, groups, w, b, stats, plan, act, res, gate, clients, nx,
                                                nr and act != "none", dw, db, x.shape[1], None, False, True)
        if nr and act == "none":
            dres = gy
        if lead is not None:
            dw = dw if dw is None else dw.to(lead[0])
            db = db if db is None else db.to(lead[1])
        return dx, dw, db, dres, None


def _affine(t):
    if t is None:
        return None
    t = t.detach()
    if t.dtype != torch.float32:
        t = t.to(torch.float32)
    return t if t.stride(-1) == 1 else t.contiguous()


def _clients(*affine):
    for t in affine:
        if t is not None and t.dim() == 2:
            return t.shape[0]
    return 1


def _needs_grad(*tensors) -> bool:
    if _grad_mode():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def group_norm(x, groups: int, weight=None, bias=None, eps: float = 1e-5, act: str = "none", residual=None):
    """``act(group_norm(x) * weight + bias + residual)``.

    ``x [N, C, *]``, read channels last (other layouts are copied); ``weight`` / ``bias`` ``[C]``, or ``[K, C]``: one row
    for each of K clients that own N / K consecutive samples (their gradients then come per client).  ``act``: none, relu,
    gelu (erf) or silu.  Statistics, products and sums are 32-bit, the result is rounded once.  A group has at most 2048
    channels on the GPU (1024 where C or an address rules out accesses of four)."""
    if x.dim() < 2 or not x.is_floating_point():
        raise ValueError(f"group_norm: expected a floating-point tensor [N, C, *], got {x.dtype} {tuple(x.shape)}")
    N, C = x.shape[0], x.shape[1]
    groups, eps = int(groups), float(eps)
    if groups < 1 or C < 1 or C % groups:
        raise ValueError(f"group_norm: {C} channels do not divide into {groups} groups")
    if act not in _ACTS:
        raise ValueError(f"group_norm: act must be one of {_ACTS}, got {act!r}")
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
    if not _own_kernel("group_norm", x) or x.numel() == 0:
        return ref.group_norm(x, groups, weight, bias, eps, act, residual)
    if _needs_grad(x, weight, bias, residual):
        return _GroupNormFn.apply(x, weight, bias, residual, (groups, eps, act))
    w, b = _affine(weight), _affine(bias)
    return _h().group_norm_forward(x, groups, w, b, eps, act, residual, _clients(w, b), False, True)[0]


class _ClientDropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, uids, tag, cfg):
        h = _h()
        x, plan = h.dropout_plan(x, uids, *cfg)
        # the ids and the tag are saved, so that changing them between the two passes raises instead of drawing another mask
        if type(tag) is int:
            ctx.save_for_backward(uids)
            ctx.run = (plan, x.stride(), cfg, tag)
        else:
            ctx.save_for_backward(uids, tag)
            ctx.run = (plan, x.stride(), cfg, None)
        return h.dropout_launch(x, uids, tag, plan)

    @staticmethod
    @_first_order
    def backward(ctx, gy):
        plan, stride, cfg, tag = ctx.run
        if tag is None:
            uids, tag = ctx.saved_tensors
        else:
            (uids,) = ctx.saved_tensors
        if gy.stride() != stride:
            gy, plan = _h().dropout_plan(gy, uids, *cfg)
        return _kernels.dropout_launch(gy, uids, tag, plan), None, None, None


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
    if not _own_kernel("client_dropout", x):
        return ref.client_dropout(x, uids, seed, tag, layer, p, kind, layout, scale)
    cfg = (int(seed), int(layer), p, kind, layout, None if scale is None else float(scale))  # (dropout_plan's)
    if uids.dim() == 0 or not uids.is_contiguous():
        uids = uids.reshape(-1).contiguous()
    if by_value:
        tag = int(tag)
    if x.requires_grad and _grad_mode():
        return _ClientDropoutFn.apply(x, uids, tag, cfg)
    x, plan = _h().dropout_plan(x, uids, *cfg)
    return _kernels.dropout_launch(x, uids, tag, plan)


class _RopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, cfg):
        ctx.save_for_backward(pos)
        ctx.cfg = cfg
        return _h().rope_axes(x, pos, *cfg, False, None, True)

    @staticmethod
    @_first_order
    def backward(ctx, gy):
        return _h().rope_axes(gy, ctx.saved_tensors[0], *ctx.cfg, True, None, True), None, None


def rope_axes(x, pos, axes, base: float = 10000.0, slots=None):
    """Rotary positions with one section of the head dimension per axis.

    ``x [R, N, H, D]`` (queries or keys), or ``[R, N, S, H, D]``, the packed projection, whose first ``slots`` slots (None:
    all) are turned and whose others are copied.  ``axes``: even widths of the sections, one per axis, together at most D
    (the rest of the head passes through).  ``pos``: int64 or fp32 positions, ``[N, A]`` shared by the samples or
    ``[R, N, A]``.  Pair (2i, 2i + 1) of a section d wide is turned by ``pos * base ** (-2 i / d)``; angles are 64-bit.
    D is even, at most 256; at most 8 axes."""
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
    if not _own_kernel("rope_axes", x):
        return ref.rope_axes(x, pos, axes, base, slots)
    if x.requires_grad and _grad_mode():
        return _RopeFn.apply(x, pos, (axes, base, slots))
    return _h().rope_axes(x, pos, axes, base, slots, False, None, True)
