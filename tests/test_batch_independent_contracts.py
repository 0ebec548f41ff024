"""What callers may ask of group norm, client-keyed dropout and rotary positions besides their values."""
import pytest
import torch
from torch.autograd import forward_ad

from blades_amd import ops
from blades_amd.ops import reference as ref

U32 = 2.0 ** -24  # half a step of fp32, relative


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    import importlib
    importlib.import_module("blades_amd.ops._hip")  # must load: no fallback on GPU
    return torch.device("cuda")


def last(t):
    """The same values, stored channels last."""
    return t.movedim(1, -1).contiguous().movedim(-1, 1)


def layers(device, dt=torch.float32):
    """An input and, by name, (function of a list of differentiable tensors, those tensors)."""
    g = torch.Generator().manual_seed(5)
    x, r = (last(torch.randn(6, 8, 4, 4, generator=g)).to(device=device, dtype=dt) for _ in range(2))
    w, b = ((1 + 0.3 * torch.randn(3, 8, generator=g)).to(device=device, dtype=dt) for _ in range(2))
    uids, tag = torch.arange(3, device=device), torch.ones(1, dtype=torch.int64, device=device)
    pos = torch.arange(8, device=device).unsqueeze(1)
    return {
        "group_norm": (lambda t: ops.group_norm(t[0], 2, t[1], t[2], act="gelu", residual=t[3]), [x, w, b, r]),
        "dropout": (lambda t: ops.client_dropout(t[0], uids, 1, tag, 0, 0.5), [x]),
        "dropout by value": (lambda t: ops.client_dropout(t[0], uids, 1, 7, 0, 0.25, kind="channel"), [x]),
        "rotary": (lambda t: ops.rope_axes(t[0], pos, (4,)), [x]),
    }


LAYERS = ["group_norm", "dropout", "dropout by value", "rotary"]


@pytest.mark.gpu
@pytest.mark.parametrize("name", LAYERS)
def test_forward_mode_tangents(dev, name):
    """A dual tensor's tangent goes through every layer, whichever argument carries it, as in 64 bits on the CPU; without a
    tangent the kernels run as ever."""
    f, args = layers(dev)[name]
    f64, args64 = layers("cpu", torch.float64)[name]
    plain = f(args)
    for i in range(len(args)):
        d = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)

        def tangent(fn, a, v):
            with forward_ad.dual_level():
                assert a is args64 or torch.equal(fn(a), plain)
                y = fn([forward_ad.make_dual(t, v) if j == i else t for j, t in enumerate(a)])
                return forward_ad.unpack_dual(y).tangent

        want, got = tangent(f64, args64, d), tangent(f, args, d.float().to(dev))
        assert got is not None
        # fewer than 512 half steps (the sums of a group of 64 and under 30 roundings in a row), each of at most the
        # largest term: (1 + |x of a unit spread|)^2 <= 25 of the largest tangent
        assert float((got.cpu().double() - want).abs().max()) <= 512 * U32 * 25 * max(1.0, float(want.abs().max()))


@pytest.mark.gpu
def test_engine_dropout_forward_mode(dev):
    from blades_amd.engine.layers import ClientDropout, DropContext

    ctx = DropContext(3, dev)
    ctx.set(torch.tensor([7, 1], device=dev), "major")
    m = ClientDropout(0.5, "elem", 2, ctx).train()
    x, d = torch.randn(4, 6, device=dev), torch.randn(4, 6, device=dev)
    with forward_ad.dual_level():
        y = m(forward_ad.make_dual(x, d))
        assert torch.equal(forward_ad.unpack_dual(y).tangent, torch.where(m(x) != 0, 2 * d, 0 * d))
