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

from . import reference as ref

_ACTS = ("none", "relu", "gelu", "silu")
_KINDS = ("elem", "channel", "sample")


def _own_kernel(t: torch.Tensor) -> bool:
    from blades_amd import ops

    return t.is_cuda and not ops._FORCE_REFERENCE and not torch._C._functorch.is_functorch_wrapped_tensor(t)


def _h():
    from blades_amd import ops

    return ops._h()


class _GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, groups, eps, act):
        h = _h()
        ctx.lead = [None if t is None else (t.dtype, t.dim()) for t in (weight, bias)]
        w, b = (None if t is None else t.detach().to(torch.float32) for t in (weight, bias))
        w, b = (t if t is None or t.stride(-1) == 1 else t.contiguous() for t in (w, b))
        clients = next((t.shape[0] for t in (w, b) if t is not None and t.dim() == 2), 1)
        grad = any(ctx.needs_input_grad)
        y, stats, gate = h.group_norm_forward(x, groups, w, b, eps, act, residual, clients, want_gate=grad)
        # the gate stands in for the residual; without a ReLU or a residual z is computed again from x
        keep = residual if gate is None and act in ("gelu", "silu") else None
        ctx.cfg = (groups, act, clients, gate[1] if gate is not None else 0)
        ctx.has_res = residual is not None
        ctx.save_for_backward(x, w, b, stats, keep, gate[0] if gate is not None else None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, w, b, stats, res, gate = ctx.saved_tensors
        groups, act, clients, gvec = ctx.cfg
        nx, nw, nb, nr = ctx.needs_input_grad[:4]
        C = x.shape[1]
        dw = torch.empty(clients, C, device=x.device) if nw else None
        db = torch.empty(clients, C, device=x.device) if nb else None
        dx, dres = _h().group_norm_backward(
            x, gy, groups, w, b, stats, act, res, (gate, gvec) if gate is not None else None, clients, want_dx=nx,
            want_dres=nr and act != "none", dweight=dw, dbias=db, ld=C)
        if nr and act == "none":
            dres = gy

        def as_leaf(t, lead):
            return None if t is None else t.reshape(t.shape if lead[1] == 2 else (C,)).to(lead[0])

        return dx, as_leaf(dw, ctx.lead[0]), as_leaf(db, ctx.lead[1]), dres if nr else None, None, None, None


def group_norm(x, groups: int, weight=None, bias=None, eps: float = 1e-5, act: str = "none", residual=None):
    """``act(group_norm(x) * weight + bias + residual)``.

    ``x [N, C, *]``, read channels last (other layouts are copied); ``weight`` / ``bias`` ``[C]``, or ``[K, C]``: one row
    for each of K clients that own N / K consecutive samples (their gradients then come per client).  ``act``: none, relu,
    gelu (erf) or silu.  Statistics, products and sums are 32-bit, the result is rounded once.  A group has at most 2048
    channels on the GPU (1024 where C or an address rules out 16-byte accesses)."""
    if x.dim() < 2 or not x.is_floating_point():
        raise ValueError(f"group_norm: expected a floating-point tensor [N, C, *], got {x.dtype} {tuple(x.shape)}")
    N, C = x.shape[0], x.shape[1]
    groups = int(groups)
    if groups < 1 or C < 1 or C % groups:
        raise ValueError(f"group_norm: {C} channels do not divide into {groups} groups")
    if act not in _ACTS:
        raise ValueError(f"group_norm: act must be one of {_ACTS}, got {act!r}")
    if not eps >= 0.0:
        raise ValueError(f"group_norm: eps must not be negative, got {eps}")
    rows = set()
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dim() not in (1, 2) or t.shape[-1] != C or not t.is_floating_point() or t.device != x.device:
            raise ValueError(f"group_norm: {name} must be a floating-point [{C}] or [clients, {C}] tensor on {x.device}, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")
        rows.add(t.shape[0] if t.dim() == 2 else 0)
    if len(rows) > 1 or any(k and N % k for k in rows) or (rows and N and 0 in [t.shape[0] for t in (weight, bias)
                                                                              if t is not None and t.dim() == 2]):
        raise ValueError(f"group_norm: weight and bias must be shared or both per client, with {N} samples a multiple of the "
                         f"clients")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"group_norm: residual must match x ({x.dtype} {tuple(x.shape)}), got {residual.dtype} "
                         f"{tuple(residual.shape)}")
    if not _own_kernel(x) or x.numel() == 0:
        return ref.group_norm(x, groups, weight, bias, eps, act, residual)
    return _GroupNormFn.apply(x, weight, bias, residual, groups, float(eps), act)


class _ClientDropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, uids, tag, cfg):
        ctx.cfg, ctx.int_tag = cfg, not torch.is_tensor(tag)
        # (saved, so that changing the ids or the tag between the two passes raises instead of redrawing another mask)
        ctx.save_for_backward(uids, *([] if ctx.int_tag else [tag]))
        ctx.tag = tag if ctx.int_tag else None
        seed, layer, p, kind, layout, scale = cfg
        return _h().client_dropout(x, uids, seed, tag, layer, p, kind, layout, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        uids = ctx.saved_tensors[0]
        tag = ctx.tag if ctx.int_tag else ctx.saved_tensors[1]
        seed, layer, p, kind, layout, scale = ctx.cfg
        return _h().client_dropout(gy, uids, seed, tag, layer, p, kind, layout, scale), None, None, None


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
    if not 0.0 <= float(p) < 1.0:
        raise ValueError(f"client_dropout: need 0 <= p < 1, got {p}")
    if uids.dtype != torch.int64 or uids.dim() > 1 or uids.numel() < 1 or uids.device != x.device:
        raise ValueError("client_dropout: uids must be an int64 vector (or scalar) of clients on x's device")
    if torch.is_tensor(tag) and (tag.dtype != torch.int64 or tag.numel() != 1 or tag.device != x.device):
        raise ValueError("client_dropout: tag must be an int or a 1-element int64 tensor on x's device")
    K = uids.numel()
    if layout == "inner" and x.dim() < 2:
        raise ValueError("client_dropout: layout inner needs [B, K * C, *]")
    if x.shape[0 if layout == "major" else 1] % K:
        raise ValueError(f"client_dropout: {tuple(x.shape)} does not divide among {K} clients (layout {layout})")
    if not _own_kernel(x):
        if x.numel() == 0:
            return x.clone()
        return ref.client_dropout(x, uids, seed, tag, layer, p, kind, layout, scale)
    return _ClientDropoutFn.apply(x, uids.reshape(-1).contiguous(), tag,
                                  (int(seed), int(layer), float(p), kind, layout, None if scale is None else float(scale)))


class _RopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, axes, base, slots):
        ctx.save_for_backward(pos)
        ctx.cfg = (axes, base, slots)
        return _h().rope_axes(x, pos, axes, base, slots)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        (pos,) = ctx.saved_tensors
        axes, base, slots = ctx.cfg
        return _h().rope_axes(gy, pos, axes, base, slots, inverse=True), None, None, None, None


def rope_axes(x, pos, axes, base: float = 10000.0, slots=None):
    """Rotary positions with one section of the head dimension per axis.

    ``x [R, N, H, D]`` (queries or keys), or ``[R, N, S, H, D]``, the packed projection, whose first ``slots`` slots (None:
    all) are turned and whose others are copied.  ``axes``: even widths of the sections, one per axis, together at most D
    (the rest of the head passes through).  ``pos``: int64 or fp32 positions, ``[N, A]`` shared by the samples or
    ``[R, N, A]``.  Pair (2i, 2i + 1) of a section d wide is turned by ``pos * base ** (-2 i / d)``; angles are 64-bit.
    D is even, at most 256 on the GPU; at most 8 axes."""
    if x.dim() not in (4, 5) or not x.is_floating_point():
        raise ValueError(f"rope_axes: expected a floating-point [R, N, H, D] or [R, N, S, H, D] tensor, got {x.dtype} "
                         f"{tuple(x.shape)}")
    axes = tuple(int(a) for a in axes)
    D, S = x.shape[-1], x.shape[2] if x.dim() == 5 else 1
    if not axes or len(axes) > 8 or any(a < 2 or a % 2 for a in axes) or sum(axes) > D or D % 2 or D > 256:
        raise ValueError(f"rope_axes: 1 to 8 even sections that fit an even head dimension of at most 256 are needed, got "
                         f"{axes} for {D}")
    if slots is not None and not 0 <= int(slots) <= S:
        raise ValueError(f"rope_axes: slots must lie in 0 .. {S}, got {slots}")
    if not float(base) > 0.0:
        raise ValueError(f"rope_axes: base must be positive, got {base}")
    want = (x.shape[1], len(axes))
    if pos.dtype not in (torch.int64, torch.float32) or tuple(pos.shape) not in (want, (x.shape[0],) + want) \
            or pos.device != x.device or pos.requires_grad:
        raise ValueError(f"rope_axes: pos must be int64 or fp32 {list(want)} or {[x.shape[0], *want]} on {x.device} without a "
                         f"gradient, got {pos.dtype} {tuple(pos.shape)} on {pos.device}")
    slots = S if slots is None else int(slots)
    if not _own_kernel(x):
        return ref.rope_axes(x, pos, axes, float(base), slots)
    return _RopeFn.apply(x, pos, axes, float(base), slots)
