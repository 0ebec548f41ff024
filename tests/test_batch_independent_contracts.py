"""What callers may ask of group norm, client-keyed dropout and rotary positions besides their values."""
import pytest
import torch
from torch import nn
from torch.autograd import forward_ad

from blades_amd import ops
from blades_amd.ops import reference as ref
from tests.test_engine_paths import build, one_round_updates

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


class Doubled(torch.Tensor):
    """A subclass without memory of its own: stands for twice the tensor inside."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, strides=t.stride(), dtype=t.dtype, device=t.device)

    def __init__(self, t):
        self.t = t

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        def full(a):
            return a.t * 2 if isinstance(a, Doubled) else a

        return func(*torch.utils._pytree.tree_map(full, args), **torch.utils._pytree.tree_map(full, kwargs or {}))


class Tagged(torch.Tensor):
    """A subclass that leaves the operations alone."""


def test_who_must_see_the_operations():
    from torch.fx.experimental.proxy_tensor import make_fx

    from blades_amd.ops import layers as mod

    t = torch.zeros(2, 3)
    assert not mod._elementary(t) and not mod._elementary(torch.nn.Parameter(t)) and not mod._recorded()
    assert not mod._elementary(t.as_subclass(Tagged)) and mod._elementary(Doubled(t))
    seen = []

    def probe(a):
        seen.append(mod._recorded())
        return a + 1

    torch.jit.trace(probe, (t,), check_trace=False)
    make_fx(probe)(t)
    make_fx(probe, tracing_mode="fake")(t)
    assert len(seen) >= 3 and all(seen) and not mod._recorded()


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["trace", "fx", "fake"])
@pytest.mark.parametrize("name", LAYERS)
@pytest.mark.filterwarnings("ignore")
def test_recorded_calls(dev, name, how):
    """A recorded layer computes other inputs' results (not the memory its allocations find), and recording works on tensors
    without memory."""
    from torch.fx.experimental.proxy_tensor import make_fx

    f, args = layers(dev)[name]

    def g(*a):
        return f(a)

    rec = torch.jit.trace(g, tuple(args), check_trace=False) if how == "trace" else make_fx(
        g, tracing_mode="real" if how == "fx" else "fake", _allow_non_fake_inputs=True)(*args)
    new = [2 * a + 1 for a in args]
    want, got = f(new), rec(*new)
    # two fp32 forms of the same values, each within 512 half steps of (1 + |x of a unit spread|) <= 5 times a slope of 1.13
    assert float((got - want).abs().max()) <= 2 * 512 * U32 * 5 * 1.13 * max(1.0, float(want.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("name", LAYERS)
def test_tensor_subclasses(dev, name):
    f, args = layers(dev)[name]
    plain = f([2 * args[0]] + args[1:])
    assert torch.equal(f([(2 * args[0]).as_subclass(Tagged)] + args[1:]).as_subclass(torch.Tensor), plain)
    got = f([Doubled(args[0])] + args[1:])
    assert float((got - plain).abs().max()) <= 2 * 512 * U32 * 5 * 1.13 * max(1.0, float(plain.abs().max()))


# ---------------------------------------------------------------------------------------------------------------
# digits
@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act,far", [("gelu", 12.0), ("silu", 80.0)])
@pytest.mark.parametrize("C,groups", [(4096, 16), (4095, 15)])
def test_activations_keep_their_digits(dev, act, far, C, groups, dt):
    """Relative to the value, in the tails too.  A zero weight makes every channel's pre-activation its bias, exactly.

    GELU, u a half step: the exponent z^2 / 2 is rounded twice and its factor once (1.25 z^2 u of e^(-z^2/2)), 2^x is off by
    2 u, the reciprocal and its argument by 3 u, the polynomial by 3 u (fit) and 4 u (sums of up to twice the result), the
    three products by 3 u: (16 + 1.5 z^2) u of the normal integral; within one standard deviation less than 9 u.  The
    density: (4 + 1.25 z^2) u.  SiLU: 2^x and the reciprocal 2 u each, sums and products 4 u, 12 u with a margin; 16-bit
    outputs |z| u more for the exponent.  Its slope s (1 + z (1 - s)) has these of s and of z s."""
    z = torch.linspace(-far, far, C)
    half, least = torch.finfo(dt).eps / 2, torch.finfo(dt).tiny * torch.finfo(dt).eps / 2
    z64 = z.double()
    if act == "gelu":
        cdf, pdf = 0.5 * torch.special.erfc(-z64 / 2 ** 0.5), torch.exp(-z64 * z64 / 2) / (2 * torch.pi) ** 0.5
        y, off = z64 * cdf, (16 + 1.5 * z64 * z64) * U32 * (z64 * cdf).abs()
        slope, soff = cdf + z64 * pdf, (16 + 1.5 * z64 * z64) * U32 * (cdf + (z64 * pdf).abs())
    else:
        s, more = torch.sigmoid(z64), 0.0 if dt == torch.float32 else 2 * z64.abs()
        y, off = z64 * s, (12 + more) * U32 * (z64 * s).abs()
        slope, soff = s * (1 + z64 * (1 - s)), (24 + 2 * more) * U32 * s * (1 + z64.abs())
    x = torch.randn(1, C, 3, device=dev).to(dt)
    res = torch.zeros(1, C, 3, device=dev, dtype=dt).requires_grad_(True)
    got = ops.group_norm(last(x), groups, torch.zeros(C, device=dev), z.to(dev), act=act, residual=last(res))
    (g,) = torch.autograd.grad(got, res, torch.ones_like(got))
    for a, want, tol in ((got, y, off), (g, slope, soff)):
        err = (a[0].detach().double().cpu() - want.unsqueeze(1)).abs()
        assert bool((err <= (tol + half * want.abs() + least).unsqueeze(1)).all()), float((err / want.abs().unsqueeze(1)).max())


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_activations_of_infinities(dev, act):
    """An infinity or NaN that the residual brings: as torch's activations of it in 64 bits (its 32-bit GELU on the CPU makes
    an infinity NaN)."""
    vals = torch.tensor([float("inf"), float("-inf"), float("nan"), 200.0, -200.0, 3e38, -3e38, 0.0])
    x, w = torch.randn(1, 8, 4, device=dev), torch.zeros(8, device=dev)
    res = vals.reshape(1, 8, 1).expand(1, 8, 4).contiguous()
    got = ops.group_norm(last(x), 2, w, w, act=act, residual=last(res.to(dev))).cpu()
    F = torch.nn.functional
    want = {"none": lambda t: t, "relu": F.relu, "gelu": F.gelu, "silu": F.silu}[act](res.double()).float()
    torch.testing.assert_close(got, want, rtol=16 * U32, atol=torch.finfo(torch.float32).tiny, equal_nan=True)


def check_scale(device, p):
    y = ops.client_dropout(torch.ones(4000, device=device), torch.arange(1, device=device), 1, 1, 0, p)
    kept = y[y != 0]
    assert kept.numel() > 0 and bool((kept.double() * (1.0 - p) - 1.0).abs().max() <= U32 * (1 + 2 * U32))


SCALES = [0.1, 0.3, 0.6, 0.701, 0.8, 0.9, 0.99, 0.999]


@pytest.mark.parametrize("p", SCALES)
def test_dropout_scale_is_rounded_once_cpu(p):
    check_scale("cpu", p)


@pytest.mark.gpu
@pytest.mark.parametrize("p", SCALES)
def test_dropout_scale_is_rounded_once(dev, p):
    check_scale(dev, p)


@pytest.mark.gpu
@pytest.mark.parametrize("C,groups", [(8, 2), (6, 3)])
@pytest.mark.parametrize("where", ["residual", "bias"])
@pytest.mark.parametrize("pixels", [9, 200 * 211])  # in a workgroup's registers, in chunks
def test_a_nan_passes_the_relu_both_ways(dev, where, pixels, C, groups):
    """What is NaN in front of a ReLU comes out NaN, and its gradient passes, as torch has it."""
    grads = []
    for device, dt in (("cpu", torch.float64), (dev, torch.float32)):
        g = torch.Generator().manual_seed(0)
        x, r, gy = (torch.randn(2, C, pixels, generator=g) for _ in range(3))
        b, w = torch.zeros(C), torch.ones(C)
        r[0, 3, 5] = b[4] = float("nan")
        leaves = [t.to(device=device, dtype=dt).requires_grad_(True) for t in (x, w, b if where == "bias" else 0 * w)]
        res = r.to(device=device, dtype=dt).requires_grad_(True) if where == "residual" else None
        y = ops.group_norm(last(leaves[0]), groups, leaves[1], leaves[2], act="relu", residual=None if res is None else last(res))
        assert bool(y[:, 4].isnan().all()) if where == "bias" else int(y.isnan().sum()) == 1
        grads.append([t.double().cpu() for t in torch.autograd.grad(
            y, leaves + ([res] if res is not None else []), gy.to(device=device, dtype=dt))])
    want, got = grads
    if where == "residual":
        assert float(want[3][0, 3, 5]) != 0.0 and torch.equal(got[3][0, 3, 5], want[3][0, 3, 5])
        assert torch.equal(got[3].isnan(), want[3].isnan())
    else:
        # every gate of that channel is open: its sum of 2 * pixels gradients, of magnitude 0.8 on average
        assert abs(float(got[2][4] - want[2][4])) <= 512 * U32 * 2 * pixels and abs(float(want[2][4])) > 0.1
    for a, b in zip(got, want):
        assert torch.equal(a.isnan(), b.isnan())


# ---------------------------------------------------------------------------------------------------------------
# the engine's modules
class Tapped(nn.Module):
    """Calls, slices and walks the children of a Sequential besides running it."""

    def __init__(self):
        super().__init__()
        self.body = nn.Sequential(nn.Conv2d(3, 8, 1), nn.GroupNorm(2, 8), nn.SiLU(), nn.Conv2d(8, 8, 1), nn.GroupNorm(4, 8),
                                  nn.ReLU())

    def forward(self, x):
        h = self.body[1](self.body[0](x))  # in front of the activation
        a = self.body[2](h) + 3 * h
        b = self.body[:2](x)
        c = self.body[0:5:4](x)            # the convolution and the second norm
        d = x
        for m in self.body:
            d = m(d)
        return torch.cat([a, b, c, d, self.body(x)], 1)


class TappedPool(nn.Module):
    """The same with a pool behind the activation."""

    def __init__(self):
        super().__init__()
        self.body = nn.Sequential(nn.Conv2d(3, 8, 1), nn.GroupNorm(2, 8), nn.ReLU(), nn.MaxPool2d(2), nn.Conv2d(8, 8, 1),
                                  nn.ReLU(), nn.MaxPool2d(2, 1))

    def forward(self, x):
        h = self.body[1](self.body[0](x))
        r = self.body[2](h)
        p = self.body[3](r - 0.5)  # the pool alone
        q = self.body[5](self.body[4](p))
        return [h, r, p, q, self.body[6](q - 0.5), self.body[4:6](p), self.body(x)]


def test_a_models_own_use_of_a_pool():
    from blades_amd.engine.fused import GradSink, build_template

    net, sink = TappedPool(), GradSink()
    sink.Kc = 2
    tmpl = build_template(net, sink)
    x = torch.randn(4, 3, 6, 6)
    with torch.no_grad():
        for a, b in zip(tmpl(x), net(x)):
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)


def test_a_models_own_use_of_a_sequentials_children():
    from blades_amd.engine.fused import GradSink, build_template

    net, sink = Tapped(), GradSink()
    sink.Kc = 2
    tmpl = build_template(net, sink)
    x = torch.randn(4, 3, 5, 5)
    with torch.no_grad():
        torch.testing.assert_close(tmpl(x), net(x), rtol=1e-5, atol=1e-5)


class Tied(nn.Module):
    """One group norm in several places, with and without an activation behind it."""

    def __init__(self):
        super().__init__()
        gn = nn.GroupNorm(2, 8)
        self.body = nn.Sequential(nn.Conv2d(3, 8, 1), gn, nn.Conv2d(8, 8, 1), gn, nn.Conv2d(8, 8, 1), gn, nn.SiLU())
        self.fc = nn.Linear(8, 10)

    def forward(self, x):
        return self.fc(self.body(x).mean((2, 3)))


def test_a_group_norm_in_several_places(data_root):
    """Its gradients are the sum over the places."""
    a, b = build(data_root, Tied, "fused"), build(data_root, Tied, "vmap")
    assert a.engine.fused is not None and b.engine.fused is None
    Ua, Ub = one_round_updates(a)[0], one_round_updates(b)[0]
    # two fp32 paths of under 100 operations in a chain, each off by under 16 half steps of its scale
    assert float(((Ua - Ub).norm(dim=1) / Ub.norm(dim=1)).max()) < 1e-4


def test_a_group_norm_with_a_forward_of_its_own_keeps_it():
    """A subclass may compute something else: the fused executor leaves its model to the general path."""
    from blades_amd.engine.fused import supports

    class NormAct(nn.GroupNorm):
        def forward(self, x):
            return torch.tanh(super().forward(x))

    assert supports(nn.Sequential(nn.Conv2d(3, 8, 1), nn.GroupNorm(2, 8)))
    assert not supports(nn.Sequential(nn.Conv2d(3, 8, 1), NormAct(2, 8)))


def test_a_residual_block_without_a_norm_argument():
    """Blocks written for (in_planes, planes, stride) build a ResNet as they did before there was a choice of norm."""
    from blades_amd.models.resnet import BasicBlock, ResNet

    class Block(BasicBlock):
        def __init__(self, in_planes, planes, stride=1):
            super().__init__(in_planes, planes, stride)

    net = ResNet(Block, [1, 1, 1, 1])
    assert net(torch.randn(2, 3, 32, 32)).shape == (2, 10)
    with pytest.raises(TypeError):
        ResNet(Block, [1, 1, 1, 1], norm="group")


def test_an_attention_from_before_rotary_positions():
    """Pickled by an earlier version: no position module, and none is asked for."""
    from blades_amd.engine.fused import GradSink, PCAttention
    from blades_amd.models.cctnets.layers import Attention

    new = Attention(16, 2).eval()
    old = Attention(16, 2).eval()
    old.load_state_dict(new.state_dict())
    del old.rope
    x = torch.randn(2, 5, 16)
    with torch.no_grad():
        assert torch.equal(old(x), new(x)) and PCAttention(old, GradSink()).rope is None


@pytest.mark.gpu
def test_evaluation_stores_nothing_for_a_backward_pass(dev, monkeypatch):
    from blades_amd.engine.fused import GradSink, PCGroupNorm

    h, asked = ops._h(), []
    forward = h.group_norm_forward

    def spy(*a, **k):
        out = forward(*a, **k)
        asked.append((k["for_backward"], out[1] is not None or out[2] is not None))
        return out

    monkeypatch.setattr(h, "group_norm_forward", spy)
    sink = GradSink()
    sink.Kc = 1
    m = PCGroupNorm(nn.GroupNorm(2, 8).to(dev), sink)
    x = torch.randn(2, 8, 3, 3, device=dev)
    with torch.no_grad():
        y = m(x, residual=x, relu=True)
    z = m(x, residual=x, relu=True)
    assert asked == [(False, False), (True, True)] and torch.equal(y, z) and z.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("name", LAYERS)
def test_poisoned_buffers(dev, name):
    """Asked for poisoned buffers, the nodes fill every one they allocate, in both passes, and the results stay."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from blades_amd.ops import layers as mod

    class Log(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.empty, self.filled = 0, 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.empty += func.overloadpacket in (torch.ops.aten.empty, torch.ops.aten.empty_like)
            self.filled += func.overloadpacket is torch.ops.aten.fill_
            return func(*args, **(kwargs or {}))

    nodes, (f, args) = mod._nodes(), layers(dev)[name]
    big = [last(torch.randn(2, 24, 130, 121, device=dev)) for _ in range(2)]  # a group norm in chunks: workspaces

    def run():
        leaves = [a.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for a in args]
        y = f(leaves)
        out = [y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))]
        if name == "group_norm":
            x = big[0].requires_grad_(True)
            y = ops.group_norm(x, 1, act="relu", residual=big[1])
            out += [y.detach(), *torch.autograd.grad(y, x, big[1])]
        return out

    plain = run()
    try:
        nodes.poison(True)
        assert all(torch.equal(a, b) for a, b in zip(run(), plain))
        with pytest.MonkeyPatch.context() as m, Log() as log:
            m.setattr(mod, "_recorded", lambda: False)  # (the kernels, though somebody is listening)
            run()
    finally:
        nodes.poison(False)
    assert log.filled == log.empty >= (13 if name == "group_norm" else 2), (log.filled, log.empty)


@pytest.mark.gpu
def test_more_samples_than_a_group_norm_takes(dev):
    """Refused by the function, in words that name the limit; the engine's layer falls back to the oracle."""
    from blades_amd.engine.fused import GradSink, PCGroupNorm

    x = torch.zeros(1 << 24, 4, device=dev, dtype=torch.bfloat16)
    x[-1] = torch.tensor([1.0, 3.0, -2.0, 2.0])
    with pytest.raises(ValueError, match="samples"):
        ops.group_norm(x, 2)
    assert not ops._h().group_norm_supported(x, 2) and ops._h().group_norm_supported(x[1:], 2)
    with pytest.raises(ValueError, match="2048 channels"):
        ops.group_norm(torch.zeros(2, 2056, device=dev), 1)
    assert not ops._h().group_norm_supported(torch.zeros(2, 2056, device=dev), 1)
    sink = GradSink()
    sink.Kc = 1
    y = PCGroupNorm(nn.GroupNorm(2, 4, eps=0.0, affine=False), sink)(x)
    assert y[-1].tolist() == [-1.0, 1.0, -1.0, 1.0]


@pytest.mark.gpu
def test_sizes_past_32_bits_are_refused(dev):
    """Counts that an int of the plan would cut to a few channels or slots, leaving the rest of the output unwritten."""
    with pytest.raises(ValueError, match="channels"):
        ops.group_norm(torch.empty(1, 2 ** 32 + 4, device=dev, dtype=torch.float16), 1)
    assert not ops._h().group_norm_supported(torch.empty(1, 2 ** 32 + 4, device=dev, dtype=torch.float16), 1)
    pos = torch.zeros(1, 1, dtype=torch.int64, device=dev)
    one = torch.zeros(1, 1, 1, 1, 2, device=dev, dtype=torch.float16)
    for shape in ((1, 1, 2 ** 32 + 1, 1, 2), (1, 1, 1, 2 ** 32 + 1, 2)):
        with pytest.raises(ValueError):
            ops.rope_axes(one.expand(shape), pos, (2,))
        with pytest.raises(ValueError):
            ops._h().rope_axes(one.expand(shape), pos, (2,))


def test_group_norm_plan_bounds_samples_times_chunks():
    """The affine sums count a client's samples times chunks in 31 bits: below 2^24 + 2048 for every layer the plan takes (read
    off the backward pass's workspace: samples x chunks x C entries of 8 bytes, and at most one per sample and group)."""
    import ctypes
    import random

    from blades_amd.ops import build

    if not build.HIP_LIB.exists():
        pytest.skip("kernels are not built")
    lib = ctypes.CDLL(str(build.HIP_LIB))
    lib.blades_group_norm_plan_size.restype = ctypes.c_long
    buf, ws = ctypes.create_string_buffer(lib.blades_group_norm_plan_size()), (ctypes.c_long * 2)()
    L, I, rng, taken = ctypes.c_long, ctypes.c_int, random.Random(1), 0
    for _ in range(4000):
        C = int(2 ** rng.uniform(0, 12))
        G = rng.choice([g for g in range(1, C + 1) if C % g == 0])
        N, P = (int(2 ** rng.uniform(0, e)) for e in (24, 30))
        dt = rng.randrange(3)
        if lib.blades_group_norm_plan(buf, L(N), L(P), I(C), I(G), ctypes.c_float(1e-5), I(0), I(N), L(0), L(0), I(dt),
                                      I(1 if C % 4 else 4), ws) == 0:
            taken += 1
            assert ws[1] // (8 * C) < (1 << 24) + 2048 + N  # (the means: at most N x G <= N x C entries)
    assert taken > 2000


# ---------------------------------------------------------------------------------------------------------------
# builds that fit together
def test_the_nodes_and_the_kernels_share_one_interface():
    """Both libraries are made from one header, depend on it, and refuse a partner of another build."""
    import ctypes
    import importlib

    from blades_amd.ops import build

    abi = build.CSRC / "layers_abi.h"
    for name in ("autograd.cpp", "groupnorm_fwd.hip", "groupnorm_bwd.hip", "dropout.hip", "rope.hip"):
        assert abi in build._headers(build.CSRC / name), name
    if not build.AUTOGRAD_LIB.exists():
        pytest.skip("nodes are not built")
    nodes = importlib.import_module("blades_amd.ops._autograd")
    other = ctypes.CFUNCTYPE(ctypes.c_long)(lambda: 1)
    with pytest.raises(RuntimeError, match="another build"):
        nodes.entries([ctypes.cast(other, ctypes.c_void_p).value] * 9)


def test_objects_depend_on_their_command(tmp_path, monkeypatch):
    """A changed flag, source or header makes a target stale; another folder does not."""
    import os

    from blades_amd.ops import build

    monkeypatch.setattr(build, "HERE", tmp_path)
    src, out = tmp_path / "a.hip", tmp_path / "a.o"
    cmd = ["hipcc", "-O3", str(src), "-o", str(out)]
    src.write_text("")
    assert build._stale(out, [src], cmd)
    out.write_text("")
    assert build._stale(out, [src], cmd)  # made by nobody knows what
    build._made(out, cmd)
    assert not build._stale(out, [src], cmd)
    assert build._stale(out, [src], cmd + ["-Xclang", "-packed-fp32-ops"])
    os.utime(src, (out.stat().st_mtime + 5,) * 2)
    assert build._stale(out, [src], cmd)
    moved = tmp_path / "moved"
    moved.mkdir()
    (moved / "_build").mkdir()
    (moved / "_build" / "a.o.cmd").write_text((tmp_path / "_build" / "a.o.cmd").read_text())
    (moved / "a.hip").write_text("")
    (moved / "a.o").write_text("")
    monkeypatch.setattr(build, "HERE", moved)
    assert not build._stale(moved / "a.o", [moved / "a.hip"], ["hipcc", "-O3", moved / "a.hip", "-o", moved / "a.o"])


def viewing(norm):
    class Viewing(nn.Module):
        """Flattens maps of several pixels with ``view``, which asks for channels first."""

        def __init__(self):
            super().__init__()
            self.conv, self.norm, self.fc = nn.Conv2d(3, 8, 3, stride=4), norm(), nn.Linear(8 * 64, 10)

        def forward(self, x):
            x = nn.functional.silu(self.norm(self.conv(x)))
            return self.fc(x.view(x.size(0), -1))

    return Viewing


@pytest.mark.gpu
@pytest.mark.parametrize("first", ["train", "evaluate"])
@pytest.mark.parametrize("nb", [1, 2])
@pytest.mark.parametrize("norm", [nn.Identity, lambda: nn.GroupNorm(2, 8)], ids=["none", "group"])
def test_a_model_that_views_its_maps_channels_first(data_root, norm, nb, first):
    """The fused executor, channels last throughout, hands it to the general ones."""
    from tests.test_batch_independent_models import gpu_copy

    a = build(data_root, viewing(norm), "vmap", nb=nb, lr=0.05)
    g = gpu_copy(a, "auto")
    assert g.engine.fused is not None
    want = a.engine.evaluate(a.server.theta)
    if first == "evaluate":
        got = g.engine.evaluate(g.server.theta)
        assert g.engine.fused is None and abs(got["ce_loss"] - want["ce_loss"]) < 1e-4
    Ug, Ua = one_round_updates(g)[0].cpu(), one_round_updates(a)[0]
    # two fp32 paths of under 100 operations in a chain, each off by under 16 half steps of its scale, over two steps
    assert float(((Ug - Ua).norm(dim=1) / Ua.norm(dim=1)).max()) < 4e-4
    assert "layout" in g.engine.fused_pc_error
    got, want = g.engine.evaluate(g.server.theta), a.engine.evaluate(a.server.theta)
    assert abs(got["ce_loss"] - want["ce_loss"]) < 1e-3


# ---------------------------------------------------------------------------------------------------------------
# rotary positions
def through(device, dt):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 1, 2, 24, generator=g).to(dt)
    x[..., 12::3] = float("inf")
    x[..., 13::3] = float("nan")
    x[..., 14::3] = -0.0
    x[0, 0, 0, 0, 20:] = torch.tensor([torch.finfo(dt).tiny / 2, -torch.finfo(dt).tiny / 4, -0.0, -torch.finfo(dt).max])
    x = x.to(device).requires_grad_(True)
    pos = torch.arange(1, 4, device=device).unsqueeze(1)
    y = ops.rope_axes(x, pos, (10,))
    return x.detach(), y.detach(), torch.autograd.grad(y, x, x.detach())[0]


def bits(t):
    return t.contiguous().view(torch.int32 if t.element_size() == 4 else torch.int16)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_the_rest_of_the_head_passes_through_cpu(dt):
    x, y, dx = through("cpu", dt)
    assert torch.equal(bits(y[..., 10:]), bits(x[..., 10:])) and bool(torch.isfinite(y[..., :10]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_the_rest_of_the_head_passes_through(dev, dt):
    """Bit for bit, both ways: an infinity does not reach its neighbour, a zero keeps its sign."""
    x, y, dx = through(dev, dt)
    assert torch.equal(bits(y[..., 10:]), bits(x[..., 10:])) and torch.equal(bits(dx[..., 10:]), bits(x[..., 10:]))
    assert bool(torch.isfinite(y[..., :10]).all())
    z = x.clone()
    ops._h().rope_axes(z, torch.arange(1, 4, device=dev).unsqueeze(1), (10,), out=z)
    assert torch.equal(bits(z), bits(y))


# ---------------------------------------------------------------------------------------------------------------
# what a model does with an output
@pytest.mark.gpu
@pytest.mark.parametrize("spatial", [(), (5,), (4, 3), (1, 1), (2, 3, 4)])
def test_outputs_may_be_changed_in_place(dev, spatial):
    """As those of any operator: an in-place activation or residual add behind the layer, in the engine's module too."""
    from blades_amd.engine.fused import GradSink, PCGroupNorm

    sink = GradSink()
    sink.Kc = 1
    m = PCGroupNorm(nn.GroupNorm(2, 8, affine=False), sink)
    x = torch.randn(3, 8, *spatial, device=dev)
    for f in (lambda t: ops.group_norm(t, 2), m, lambda t: ops.client_dropout(t, torch.zeros((), dtype=torch.int64, device=dev),
                                                                           1, 1, 0, 0.5)):
        a, b = (x.clone().requires_grad_(True) for _ in range(2))
        y = f(a)
        y.mul_(3).add_(a)
        z = f(b) * 3 + b
        assert torch.equal(y, z)
        gy = torch.randn_like(x)
        assert torch.equal(torch.autograd.grad(y, a, gy)[0], torch.autograd.grad(z, b, gy)[0])
    t = torch.randn(2, 5, 3, 2, 8, device=dev, requires_grad=True)
    y = ops.rope_axes(t, torch.arange(5, device=dev).unsqueeze(1), (4,), slots=2)
    y.mul_(2)
    y.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("name", LAYERS)
def test_gradients_without_memory_are_refused(dev, name):
    """A wrapper subclass as gradient, a batch of gradients: raised, nothing launched on their addresses."""
    f, args = layers(dev)[name]
    leaves = [a.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for a in args]
    y = f(leaves)
    gy = torch.ones_like(y)
    want = torch.autograd.grad(y, leaves, gy, retain_graph=True)
    with pytest.raises(RuntimeError, match="memory of their own"):
        torch.autograd.grad(y, leaves, Doubled(gy), retain_graph=True)
    with pytest.raises(RuntimeError, match="memory of their own"):
        torch.autograd.grad(y, leaves, torch.stack([gy, gy]), is_grads_batched=True, retain_graph=True)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, gy), want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", LAYERS)
def test_a_gradients_tangent_is_refused(dev, name):
    """Forward over reverse with the tangent behind the layer: a second derivative, which raises as the others do."""
    f, args = layers(dev)[name]
    leaves = [a.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for a in args]
    y = f(leaves)
    gy = torch.ones_like(y)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y, leaves, forward_ad.make_dual(gy, gy), retain_graph=True)
        torch.autograd.grad(y, leaves, gy)


def test_an_installed_host_library_is_loaded_not_built(tmp_path, monkeypatch):
    """A package without a record of how it was built (a wheel) loads its library as it is."""
    import os
    import subprocess

    from blades_amd.ops import build

    lib, src = tmp_path / "libblades_host.so", tmp_path / "csrc" / "host.cpp"
    src.parent.mkdir()
    src.write_text("")
    lib.write_text("")
    for name, value in (("HERE", tmp_path), ("CSRC", src.parent), ("HOST_LIB", lib)):
        monkeypatch.setattr(build, name, value)
    monkeypatch.setattr(subprocess, "check_call", lambda cmd: built.append(cmd))
    built = []
    os.utime(lib, (src.stat().st_mtime + 5,) * 2)
    assert build.host_lib() == lib and not built
    os.utime(src, (lib.stat().st_mtime + 5,) * 2)
    assert build.host_lib() == lib and len(built) == 1
