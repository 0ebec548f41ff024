"""Group norm with activation, client-keyed dropout without a stored mask, rotary positions with several axes: the public
functions against their definitions in 64 bits (CPU and GPU), gradients, refusals, layouts, streams and captured graphs."""
import math
import os

import pytest
import torch
import torch.nn.functional as F

from blades_amd import ops
from blades_amd.ops import reference as ref

U32 = 2.0 ** -24  # half a step of fp32, relative


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    import importlib
    importlib.import_module("blades_amd.ops._hip")  # must load: no fallback on GPU
    return torch.device("cuda")


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(11)


def half_step(dt):
    return torch.finfo(dt).eps / 2


def subnormal(dt):
    """Half a step below the smallest normal value, absolute: there the step stays eps * tiny (fp16: 2^-24, so a value of
    2^-17 may be off by 2^-25, which is 2^-8 of it)."""
    return torch.finfo(dt).tiny * torch.finfo(dt).eps / 2


def last(t):
    """The same values, stored channels last."""
    return t.movedim(1, -1).contiguous().movedim(-1, 1)


# ---------------------------------------------------------------------------------------------------------------
# group norm
def gn64(x, groups, w, b, eps, act, res, gy):
    """Value, pre-activation and gradients by the formulas, in 64 bits, one client at a time."""
    N, C = x.shape[:2]
    K = w.shape[0] if w is not None and w.dim() == 2 else 1
    x64, g64 = x.double(), gy.double()
    xs = x64.reshape(N, groups, -1)
    mean = xs.mean(2, keepdim=True)
    rstd = 1.0 / torch.sqrt(((xs - mean) ** 2).mean(2, keepdim=True) + eps)
    xhat = ((xs - mean) * rstd).reshape(N, C, -1)
    gam = torch.ones(K, C, dtype=torch.float64) if w is None else w.double().reshape(K, C)
    bet = torch.zeros(K, C, dtype=torch.float64) if b is None else b.double().reshape(K, C)
    gam, bet = (t.to(x.device).repeat_interleave(N // K, 0).unsqueeze(-1) for t in (gam, bet))
    z = xhat * gam + bet
    if res is not None:
        z = z + res.double().reshape(N, C, -1)
    if act == "relu":
        y, slope = z.clamp_min(0), (z > 0).double()
    elif act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        y, slope = z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    elif act == "silu":
        s = torch.sigmoid(z)
        y, slope = z * s, s * (1 + z * (1 - s))
    else:
        y, slope = z, torch.ones_like(z)
    g = g64.reshape(N, C, -1) * slope
    gg = (g * gam).reshape(N, groups, -1)
    xg = xhat.reshape(N, groups, -1)
    dx = rstd * (gg - gg.mean(2, keepdim=True) - xg * (gg * xg).mean(2, keepdim=True))
    A, B = g.sum(2).reshape(K, N // K, C), (g * xhat).sum(2).reshape(K, N // K, C)
    absum = (g.abs() * (1 + xhat.abs())).sum(2).reshape(K, N // K, C).sum(1)
    return {"y": y.reshape(x.shape), "z": z.reshape(x.shape), "dx": dx.reshape(x.shape), "dw": B.sum(1), "db": A.sum(1),
            "dres": g.reshape(x.shape), "absum": absum, "xhat": xhat, "rstd": rstd, "gg": gg}


def gn_inputs(N, C, spatial, groups, K, act, res, dt, device, seed=0, affine=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(N, C, *spatial, generator=g) * 1.5 + torch.randn(C, generator=g).reshape(1, C, *[1] * len(spatial)))
    x = x.to(dt).to(device)
    w = b = None
    if affine:
        lead = (K, C) if K else (C,)
        w = (1 + 0.3 * torch.rand(*lead, generator=g)).to(device)
        b = (0.3 * torch.randn(*lead, generator=g)).to(device)
    r = torch.randn(N, C, *spatial, generator=g).to(dt).to(device) if res else None
    gy = torch.randn(N, C, *spatial, generator=g).to(dt).to(device)
    if act == "relu":  # keep every gate clear of its border: within rounding of it either gradient is right
        for _ in range(3):
            near = gn64(x, groups, w, b, 1e-5, act, r, gy)["z"].abs() < 1e-3
            if r is not None:
                r = torch.where(near, r + 0.25, r)
            else:
                x = torch.where(near, x + 0.25, x)
        assert float(gn64(x, groups, w, b, 1e-5, act, r, gy)["z"].abs().min()) > 2e-4
    return x, w, b, r, gy


def gn_check(got, want, dt, K):
    """Tolerances.  Sums of a group add at most 64 values in a row and then at most 2^10 partial ones in trees and teams
    (16 more in a row), so a mean is off by at most 80 u of mean|x|, about 4 standard deviations at most here (offsets of
    the channels): 320 u of a standard deviation; the square root of the variance by 80 u relative; subtraction, two
    products and the sums with beta and the residual by 8 u of at most 8: under 512 u of (1 + max|xhat|) in all.  The
    slopes of the activations are at most 1.13, their second derivatives 0.8.  The input gradient has two such means more:
    512 u of rstd * max|g gamma| * (1 + max|xhat|)^2, twice.  The affine sums: 512 u of sum |g| (1 + |xhat|).  An output is
    rounded once more to its type."""
    u, h = 512 * U32, half_step(dt)
    xm = float(want["xhat"].abs().max())
    gm = float(want["gg"].abs().max())

    def near(name, bound):
        a, b = got[name].double(), want[name].reshape(got[name].shape)
        assert bool(((a - b).abs() <= bound + h * b.abs() * (name in ("y", "dx", "dres")) + subnormal(dt)).all()), \
            (name, float((a - b).abs().max()))

    near("y", 2 * u * (1 + xm) * 1.3)
    if "dx" in got:
        rs = want["rstd"].expand(*want["gg"].shape).reshape(got["dx"].shape)
        near("dx", 2 * u * rs * max(gm, 1.0) * (1 + xm) ** 2)
    for n in ("dw", "db"):
        if n in got:
            near(n, 2 * u * want["absum"].reshape(got[n].shape) * (1 + xm))
    if "dres" in got:
        near("dres", 2 * u * (1 + xm) * float(want["dres"].abs().max()))


def gn_run(x, groups, w, b, r, gy, act, eps=1e-5):
    leaves = {"dx": x, "dw": w, "db": b, "dres": r}
    leaves = {k: v.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for k, v in leaves.items()
              if v is not None}
    y = ops.group_norm(leaves["dx"], groups, leaves.get("dw"), leaves.get("db"), eps=eps, act=act,
                       residual=leaves.get("dres"))
    grads = torch.autograd.grad(y, list(leaves.values()), gy)
    return {"y": y.detach(), **dict(zip(leaves, grads))}


GN_CASES = [  # N, C, spatial, groups, clients, act, residual
    (1, 64, (32, 32), 32, 0, "relu", False),
    (6, 30, (9, 7), 10, 3, "relu", True),      # three channels a group
    (4, 32, (5, 5), 32, 0, "silu", False),     # instance norm
    (5, 512, (4, 4), 32, 5, "relu", True),
    (3, 48, (7, 1), 2, 0, "gelu", True),
    (2, 64, (33, 31), 4, 2, "none", True),
    (4, 40, (), 5, 2, "relu", False),          # no pixels: [N, C]
    (3, 10, (13,), 5, 0, "silu", True),
    (2, 6, (3, 4, 5), 3, 0, "relu", False),
    (2, 1, (4, 9), 1, 0, "gelu", False),       # one channel
    (2, 7952, (3, 2), 16, 0, "none", False),   # 497 channels a group: no 16-byte slab
    (3, 2048, (2, 2), 1, 0, "relu", True),     # the widest group
    (130, 8, (1, 2), 1, 65, "relu", False),
]


@pytest.mark.parametrize("N,C,spatial,groups,K,act,res", [c for c in GN_CASES])
def test_group_norm_formulas_cpu(N, C, spatial, groups, K, act, res):
    x, w, b, r, gy = gn_inputs(N, C, spatial, groups, K, act, res, torch.float32, "cpu")
    gn_check(gn_run(x, groups, w, b, r, gy, act), gn64(x, groups, w, b, 1e-5, act, r, gy), torch.float32, K)


def test_group_norm_matches_torch_and_differences_cpu():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 12, 3, 5, generator=g, dtype=torch.float64)
    w, b = torch.rand(12, generator=g, dtype=torch.float64) + 0.5, torch.randn(12, generator=g, dtype=torch.float64)
    torch.testing.assert_close(ops.group_norm(x, 4, w, b), F.group_norm(x, 4, w, b), rtol=1e-12, atol=1e-12)
    wk = torch.stack([w, 2 * w])
    torch.testing.assert_close(ops.group_norm(x, 4, wk, torch.stack([b, b]))[2:], F.group_norm(x, 4, 2 * w, b)[2:],
                               rtol=1e-12, atol=1e-12)
    leaves = [t.requires_grad_(True) for t in (x, wk.clone(), torch.stack([b, -b]), torch.randn_like(x))]
    assert torch.autograd.gradcheck(lambda a, c, d, e: ops.group_norm(a, 4, c, d, act="gelu", residual=e), leaves)


def test_layers_on_nothing_cpu():
    w = torch.ones(8, requires_grad=True)
    y = ops.group_norm(torch.empty(0, 8, 4, 4), 2, w)
    assert y.shape == (0, 8, 4, 4) and torch.equal(torch.autograd.grad(y.sum(), w)[0], torch.zeros(8))
    assert ops.group_norm(torch.empty(3, 8, 0), 2).shape == (3, 8, 0)
    assert ops.client_dropout(torch.empty(0, 8), torch.arange(2), 1, 1, 0, 0.5).shape == (0, 8)
    assert ops.rope_axes(torch.empty(0, 3, 2, 8), torch.zeros(3, 1), (8,)).shape == (0, 3, 2, 8)
    assert ops.rope_axes(torch.empty(2, 0, 2, 8), torch.zeros(0, 1), (8,)).shape == (2, 0, 2, 8)


@pytest.mark.parametrize("kw,args", [
    ({}, (torch.zeros(4), 1)), ({}, (torch.zeros(2, 4, dtype=torch.int64), 1)), ({}, (torch.zeros(2, 4), 3)),
    ({}, (torch.zeros(2, 4), 0)), ({"act": "tanh"}, (torch.zeros(2, 4), 2)), ({"eps": -1.0}, (torch.zeros(2, 4), 2)),
    ({"eps": float("nan")}, (torch.zeros(2, 4), 2)), ({"weight": torch.ones(3)}, (torch.zeros(2, 4), 2)),
    ({"weight": torch.ones(3, 4), "bias": torch.ones(3, 4)}, (torch.zeros(2, 4), 2)),
    ({"weight": torch.ones(2, 4), "bias": torch.ones(4)}, (torch.zeros(2, 4), 2)),
    ({"residual": torch.zeros(2, 5)}, (torch.zeros(2, 4), 2)),
    ({"residual": torch.zeros(2, 4, dtype=torch.float64)}, (torch.zeros(2, 4), 2)),
])
def test_group_norm_refusals(kw, args):
    with pytest.raises(ValueError):
        ops.group_norm(*args, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,C,spatial,groups,K,act,res", GN_CASES + [
    (3, 64, (112, 112), 8, 3, "relu", True),    # a sample is cut into chunks
    (2, 24, (130, 121), 1, 0, "silu", False),
    (2, 15, (150, 150), 5, 2, "gelu", True),
    (9, 64, (32, 32), 32, 3, "relu", False),
    (600, 16, (4, 4), 4, 200, "relu", True),
])
def test_group_norm_kernels(dev, N, C, spatial, groups, K, act, res, dt):
    x, w, b, r, gy = gn_inputs(N, C, spatial, groups, K, act, res, dt, dev)
    got = gn_run(last(x), groups, w, b, None if r is None else last(r), last(gy), act)
    gn_check(got, gn64(x, groups, w, b, 1e-5, act, r, gy), dt, K)
    assert got["y"].dtype == dt and got["dx"].dtype == dt
    again = gn_run(last(x), groups, w, b, None if r is None else last(r), last(gy), act)
    assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.gpu
@pytest.mark.parametrize("act,res", [("relu", True), ("relu", False), ("gelu", True), ("none", False)])
def test_group_norm_layouts_and_addresses(dev, act, res):
    """Plain layouts, sliced batches, addresses off 16 bytes, an expanded gradient, missing affine vectors."""
    x, w, b, r, gy = gn_inputs(5, 32, (6, 5), 8, 0, act, res, torch.float32, dev)
    want = gn64(x, 8, w, b, 1e-5, act, r, gy)
    gn_check(gn_run(x, 8, w, b, r, gy, act), want, torch.float32, 0)  # NCHW

    def off(t):  # the same values one element into a buffer
        buf = torch.empty(t.numel() + 1, device=dev)
        v = buf[1:].view(t.shape[0], *t.shape[2:], t.shape[1]).movedim(-1, 1)
        v.copy_(t)
        return v

    for xo, ro, go in ((off, last, last), (last, off, last), (last, last, off)):
        xx, rr = xo(x).requires_grad_(True), None if r is None else ro(r)
        y = ops.group_norm(xx, 8, w, b, act=act, residual=rr)
        gn_check({"y": y.detach(), "dx": torch.autograd.grad(y, xx, go(gy))[0]}, want, torch.float32, 0)
    big = torch.cat([last(x), last(x)])
    gn_check({"y": ops.group_norm(last(big)[5:], 8, w, b, act=act, residual=None if r is None else last(r))}, want,
             torch.float32, 0)
    one = torch.ones(1, device=dev).expand(x.shape)
    xx = last(x).requires_grad_(True)
    ops.group_norm(xx, 8, w, b, act=act, residual=r).sum().backward()
    gn_check({"y": want["y"].float(), "dx": xx.grad}, gn64(x, 8, w, b, 1e-5, act, r, one), torch.float32, 0)
    bare = gn64(x, 8, None, None, 1e-5, "none", None, gy)
    gn_check({"y": ops.group_norm(last(x), 8)}, bare, torch.float32, 0)


@pytest.mark.gpu
def test_group_norm_only_the_gradients_asked_for(dev):
    x, w, b, r, gy = gn_inputs(4, 16, (5, 4), 4, 2, "relu", True, torch.float32, dev)
    want = gn64(x, 4, w, b, 1e-5, "relu", r, gy)
    for asked in ("dx", "dw", "db", "dres"):
        leaves = {"dx": x, "dw": w, "db": b, "dres": r}
        leaf = leaves[asked] = leaves[asked].clone().requires_grad_(True)
        y = ops.group_norm(leaves["dx"], 4, leaves["dw"], leaves["db"], act="relu", residual=leaves["dres"])
        gn_check({"y": y.detach(), asked: torch.autograd.grad(y, leaf, gy)[0]}, want, torch.float32, 2)
    xx = x.clone().requires_grad_(True)
    (g1,) = torch.autograd.grad(ops.group_norm(xx, 4, w, b).square().sum(), xx, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g1.sum(), xx)


@pytest.mark.gpu
def test_group_norm_special_values(dev):
    """A constant group, a large offset, and an infinity or NaN, which stays in its own group of its own sample."""
    x = torch.randn(3, 8, 6, 6, device=dev)
    x[0, :4] = 3.25
    y = ops.group_norm(last(x), 2)
    assert torch.equal(y[0, :4], torch.zeros_like(y[0, :4]))
    for bad in (float("inf"), float("nan")):
        z = x.clone()
        z[1, 5, 2, 2] = bad
        y2 = ops.group_norm(last(z), 2, act="relu")
        assert bool(y2[1, 4:].isnan().any()) and bool(torch.isfinite(y2[1, :4]).all())
        assert torch.equal(y2[0], torch.relu(y[0])) and torch.equal(y2[2], torch.relu(y[2]))
    # offset 1000 at spread 1: the variance keeps its digits (squares around the mean, not their difference); the mean
    # itself is rounded to fp32, 2^-15 of a standard deviation, and x - mean is exact
    far = x + 1000.0
    want = gn64(far, 2, None, None, 1e-5, "none", None, far)["y"]
    got = ops.group_norm(last(far), 2)
    assert float((got.double() - want)[1:].abs().max()) < 80 * U32 * 1000 * 1.1
    assert ops.group_norm(torch.empty(0, 8, 4, 4, device=dev), 2).shape == (0, 8, 4, 4)


@pytest.mark.gpu
def test_group_norm_refusals_gpu(dev):
    with pytest.raises(ValueError):
        ops.group_norm(torch.zeros(2, 4, device=dev, dtype=torch.float64), 2)
    with pytest.raises(ValueError):  # a group wider than a workgroup's slab
        ops.group_norm(torch.zeros(2, 2056, device=dev), 1)
    with pytest.raises(ValueError):
        ops.group_norm(torch.zeros(2, 4, device=dev), 2, weight=torch.ones(4))


# ---------------------------------------------------------------------------------------------------------------
# client-keyed dropout
def drop_mask(uids, shape, seed, tag, layer, p, kind, layout):
    """Multipliers by walking the definition: client by client, value by value (CPU, 64 bits)."""
    K = uids.numel()
    B, C = (shape[0] // K, shape[1] if len(shape) > 1 else 1) if layout == "major" else (shape[0], shape[1] // K)
    tail = list(shape[2:])
    keep = [1] * (1 + len(tail)) if kind == "sample" else [C] + ([1] * len(tail) if kind == "channel" and tail else tail)
    m = ref.client_dropout_mult(uids.cpu(), B * math.prod(keep), seed, int(tag), layer, p).double() != 0
    m = m.reshape(K, B, *keep).expand(K, B, C, *tail)
    m = m if layout == "major" else m.transpose(0, 1)
    return m.reshape(shape).double() / (1 - p)


DROP_CASES = [  # shape per client and sample, clients, batch
    ((128,), 6, 8), ((7,), 3, 5), ((1,), 1, 1), ((13, 9), 4, 3), ((64, 32), 2, 4), ((5, 7, 3), 3, 2), ((64, 6, 6), 2, 5),
    ((3, 32, 32), 2, 2), ((65, 9, 30), 2, 2), ((130, 1, 1), 2, 3), ((8, 2, 2), 33, 1), ((2, 300, 40), 1, 2),
    ((64, 6, 6), 30, 40), ((6, 50, 70), 2, 3), ((512, 2, 2), 40, 1), ((16, 8), 5, 300),
]


@pytest.mark.parametrize("kind", ["elem", "channel", "sample"])
@pytest.mark.parametrize("layout", ["major", "inner"])
@pytest.mark.parametrize("shape,K,B", DROP_CASES)
def test_client_dropout_cpu(shape, K, B, layout, kind):
    full = (K * B,) + shape if layout == "major" else (B, K * shape[0]) + shape[1:]
    uids = torch.arange(K) * 7 + 3
    x = torch.randn(full).requires_grad_(True)
    y = ops.client_dropout(x, uids, 12345678901, 5, 2, 0.3, kind, layout)
    m = drop_mask(uids, full, 12345678901, 5, 2, 0.3, kind, layout)
    # the scale and the product are each rounded once to fp32
    torch.testing.assert_close(y.detach().double(), x.detach().double() * m, rtol=4 * U32, atol=0)
    gy = torch.randn(full)
    torch.testing.assert_close(torch.autograd.grad(y, x, gy)[0].double(), gy.double() * m, rtol=4 * U32, atol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["elem", "channel", "sample"])
@pytest.mark.parametrize("layout", ["major", "inner"])
@pytest.mark.parametrize("shape,K,B", DROP_CASES)
def test_client_dropout_kernels(dev, shape, K, B, layout, kind, dt):
    full = (K * B,) + shape if layout == "major" else (B, K * shape[0]) + shape[1:]
    uids = (torch.arange(K) * 7 + 3).to(dev)
    tag = torch.tensor([41], device=dev)
    m = drop_mask(uids, full, 98765432109, 41, 3, 0.3, kind, layout).to(dev)
    x, gy = torch.randn(full).to(dt).to(dev), torch.randn(full).to(dt).to(dev)
    forms = [lambda t: t] + ([last] if len(full) == 4 else [])
    for f in forms:
        xx = f(x).requires_grad_(True)
        y = ops.client_dropout(xx, uids, 98765432109, tag, 3, 0.3, kind, layout)
        (dx,) = torch.autograd.grad(y, xx, f(gy))
        for a, src in ((y.detach(), x), (dx, gy)):
            assert torch.equal(a != 0, (src.double() * m).to(dt) != 0)
            torch.testing.assert_close(a.double(), src.double() * m, rtol=4 * U32 + half_step(dt), atol=subnormal(dt))
        assert torch.equal(y, ops.client_dropout(f(x), uids, 98765432109, 41, 3, 0.3, kind, layout))  # tag by value


@pytest.mark.gpu
def test_client_dropout_equals_the_stored_multipliers(dev):
    """fp32: bit for bit x * client_dropout_mult, with an odd share per client, views and addresses off 16 bytes."""
    uids, tag = torch.tensor([5, 900, 17], device=dev), torch.tensor([77], device=dev)
    for n in (1, 3, 4, 37, 4096, 100003):
        x = torch.randn(3 * n + 1, device=dev)[1:].reshape(3, n)
        m = ops.client_dropout_mult(uids, n, 11, tag, 4, 0.1)
        assert torch.equal(ops.client_dropout(x, uids, 11, tag, 4, 0.1), x * m)
    assert torch.equal(ops.client_dropout(x, uids, 11, tag, 4, 0.0), x)
    half = ops.client_dropout(x, uids, 11, tag, 4, 0.1, scale=0.5)
    assert torch.equal(half, x * (m != 0) * 0.5)
    assert torch.equal(ops.client_dropout(x.t(), uids, 11, tag, 4, 0.1, layout="inner"),
                       ops.client_dropout(x.t().contiguous(), uids, 11, tag, 4, 0.1, layout="inner"))
    x[1, 5] = float("inf")
    assert ops.client_dropout(x, uids, 11, tag, 4, 0.1, scale=0.0).isnan().sum() == 1  # 0 * inf, as multiplied
    assert ops.client_dropout(x[:0], uids, 11, tag, 4, 0.1).shape == (0, n)
    one = ops.client_dropout(x[:1], uids[1], 11, tag, 4, 0.1)  # a 0-d id: one client
    assert torch.equal(one, ops.client_dropout(x[:1], uids[1:2], 11, tag, 4, 0.1))


@pytest.mark.gpu
def test_client_dropout_changed_tag_raises(dev):
    x = torch.randn(4, 8, device=dev, requires_grad=True)
    uids, tag = torch.arange(2, device=dev), torch.ones(1, dtype=torch.int64, device=dev)
    y = ops.client_dropout(x, uids, 1, tag, 0, 0.5)
    tag.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()


@pytest.mark.parametrize("x,uids,kw", [
    (torch.zeros(4, 2, dtype=torch.int64), torch.arange(2), {}), (torch.zeros(5, 2), torch.arange(2), {}),
    (torch.zeros(4, 3), torch.arange(2), {"layout": "inner"}), (torch.zeros(4), torch.arange(2), {"layout": "inner"}),
    (torch.zeros(4, 2), torch.arange(2), {"kind": "row"}), (torch.zeros(4, 2), torch.arange(2), {"layout": "outer"}),
    (torch.zeros(4, 2), torch.arange(2), {"p": 1.0}), (torch.zeros(4, 2), torch.arange(2), {"p": 1 - 2.0 ** -25}), (torch.zeros(4, 2), torch.arange(2), {"p": -0.1}),
    (torch.zeros(4, 2), torch.arange(2), {"p": float("nan")}), (torch.zeros(4, 2), torch.zeros(2), {}),
    (torch.zeros(4, 2), torch.zeros(0, dtype=torch.int64), {}), (torch.zeros(4, 2), torch.zeros(2, 1, dtype=torch.int64), {}),
    (torch.zeros(4, 2), torch.arange(2), {"tag": torch.zeros(2, dtype=torch.int64)}),
    (torch.zeros(4, 2), torch.arange(2), {"tag": torch.zeros(1)}),
])
def test_client_dropout_refusals(x, uids, kw):
    with pytest.raises(ValueError):
        ops.client_dropout(x, uids, 1, kw.pop("tag", 1), 0, kw.pop("p", 0.5), **kw)


# ---------------------------------------------------------------------------------------------------------------
# rotary positions
def rope64(x, pos, axes, base, slots, sign=1.0):
    """Pair by pair as complex numbers, in 64 bits."""
    ang, D = [], x.shape[-1]
    for a, d in enumerate(axes):
        ang.append(pos[..., a:a + 1].double() * torch.pow(torch.tensor(base, dtype=torch.float64, device=pos.device),
                                                          -torch.arange(0, d, 2, device=pos.device).double() / d))
    ang = sign * torch.cat(ang + [torch.zeros(*pos.shape[:-1], (D - sum(axes)) // 2, dtype=torch.float64,
                                              device=pos.device)], -1).unsqueeze(-2)
    z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], D // 2, 2).contiguous())
    if x.dim() == 5:
        ang = ang.unsqueeze(-3) * (torch.arange(x.shape[2], device=x.device) < slots).double().reshape(-1, 1, 1)
    return torch.view_as_real(z * torch.polar(torch.ones_like(ang), ang)).flatten(-2)


def rope_near(got, x, want, dt, far=0):
    """sin and cos are off by at most 2 u (their angle, at most pi / 4 after reduction, is rounded once, then the
    polynomial's rounding); the two products and their sum add 2 u: 4 u (|a| + |b|) and the output's half step.  A far
    angle has the 64-bit rounding of its frequency (the power and its factor: 3 half steps of 2^-53) and of its product (1)
    on either side, 8 * 2^-53 of itself together, and a position's angle is at most the position."""
    pairs = x.double().abs().reshape(*x.shape[:-1], -1, 2).sum(-1, keepdim=True).expand(*x.shape[:-1], -1, 2).flatten(-2)
    assert bool(((got.double() - want).abs() <= (4 * U32 + 8 * far * 2.0 ** -53) * pairs + half_step(dt) * want.abs() + subnormal(dt)).all()), \
        float((got.double() - want).abs().max())


ROPE_CASES = [  # R, N, S, H, D, axes, slots, per sample, farthest, float positions
    (3, 64, 3, 2, 64, (32, 32), 2, False, 0, False),
    (2, 1, 1, 6, 64, (16, 24, 24), None, True, 10 ** 6, False),
    (1, 1, 1, 1, 2, (2,), None, False, 3, False),
    (5, 17, 3, 3, 20, (4, 10), 2, True, 2 ** 31, False),      # pass-through dimensions, D % 8 != 0
    (2, 9, 2, 1, 14, (14,), 1, False, 50, True),
    (2, 50, 1, 12, 128, (32, 48, 40), None, False, 4000, True),
    (1, 3, 4, 2, 256, (2, 4, 6, 8, 10, 12, 14, 200), 0, True, 9, False),
]


def rope_inputs(case, dt, device):
    R, N, S, H, D, axes, slots, per, far, flt = case
    g = torch.Generator().manual_seed(N)
    shape = (R, N, S, H, D) if slots is not None or S > 1 else (R, N, H, D)
    x = torch.randn(*shape, generator=g).to(dt).to(device)
    pos = torch.randint(0, far + 1, (R, N, len(axes)) if per else (N, len(axes)), generator=g) if far else \
        torch.stack([torch.arange(N) // 8, torch.arange(N) % 8], -1)
    pos = (pos.float() * 0.37 - 5) if flt else pos
    return x, pos.to(device), axes, slots, S if slots is None else slots


@pytest.mark.parametrize("case", ROPE_CASES)
def test_rope_axes_cpu(case):
    x, pos, axes, slots, s = rope_inputs(case, torch.float32, "cpu")
    x.requires_grad_(True)
    y = ops.rope_axes(x, pos, axes, slots=slots)
    rope_near(y.detach(), x.detach(), rope64(x.detach(), pos, axes, 10000.0, s), torch.float32, case[8])
    gy = torch.randn_like(x)
    rope_near(torch.autograd.grad(y, x, gy)[0], gy, rope64(gy, pos, axes, 10000.0, s, -1.0), torch.float32, case[8])


def test_rope_axes_differences_cpu():
    x = torch.randn(2, 5, 3, 2, 12, dtype=torch.float64, requires_grad=True)
    pos = torch.randint(0, 40, (2, 5, 2))
    assert torch.autograd.gradcheck(lambda t: ops.rope_axes(t, pos, (4, 6), slots=2), (x,))
    # relative: a shift of both positions leaves every product of a turned query and key as it was
    q, k = torch.randn(1, 1, 1, 16).double(), torch.randn(1, 1, 1, 16).double()

    def dot(a, b):
        return float((ops.rope_axes(q, torch.tensor([a]), (8, 8)) * ops.rope_axes(k, torch.tensor([b]), (8, 8))).sum())

    assert abs(dot([3, 9], [5, 2]) - dot([103, 59], [105, 52])) < 1e-10


@pytest.mark.parametrize("shape,pos,axes,kw", [
    ((2, 3, 8), torch.zeros(3, 1, dtype=torch.int64), (8,), {}), ((2, 3, 1, 8), torch.zeros(3, 1, dtype=torch.int64), (3,), {}),
    ((2, 3, 1, 8), torch.zeros(3, 1, dtype=torch.int64), (10,), {}), ((2, 3, 1, 8), torch.zeros(3, 1, dtype=torch.int64), (), {}),
    ((2, 3, 1, 8), torch.zeros(3, 2, dtype=torch.int64), (8,), {}), ((2, 3, 1, 8), torch.zeros(4, 1, dtype=torch.int64), (8,), {}),
    ((2, 3, 1, 8), torch.zeros(3, 1, dtype=torch.float64), (8,), {}), ((2, 3, 1, 7), torch.zeros(3, 1, dtype=torch.int64), (4,), {}),
    ((2, 3, 1, 8), torch.zeros(3, 1, dtype=torch.int64), (8,), {"slots": 2}),
    ((2, 3, 1, 8), torch.zeros(3, 1, dtype=torch.int64), (8,), {"base": 0.0}),
    ((2, 3, 1, 8), torch.zeros(1, 3, 1, dtype=torch.int64), (8,), {}),
    ((2, 3, 1, 258), torch.zeros(3, 1, dtype=torch.int64), (8,), {}),
    ((2, 3, 1, 18), torch.zeros(3, 9, dtype=torch.int64), (2,) * 9, {}),
])
def test_rope_axes_refusals(shape, pos, axes, kw):
    with pytest.raises(ValueError):
        ops.rope_axes(torch.zeros(shape), pos, axes, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", ROPE_CASES)
def test_rope_axes_kernel(dev, case, dt):
    x, pos, axes, slots, s = rope_inputs(case, dt, dev)
    x.requires_grad_(True)
    y = ops.rope_axes(x, pos, axes, slots=slots)
    xd = x.detach()
    rope_near(y.detach(), xd, rope64(xd, pos, axes, 10000.0, s), dt, case[8])
    gy = torch.randn_like(xd)
    rope_near(torch.autograd.grad(y, x, gy)[0], gy, rope64(gy, pos, axes, 10000.0, s, -1.0), dt, case[8])
    if xd.dim() == 5 and s < xd.shape[2]:
        assert torch.equal(y[:, :, s:], xd[:, :, s:])
    h = ops._h()
    z = xd.clone()
    assert h.rope_axes(z, pos, axes, slots=slots, out=z) is z and torch.equal(z, y)  # in place


@pytest.mark.gpu
def test_rope_axes_strides(dev):
    """Heads in front of tokens, a slice of the packed projection, an expanded batch, odd addresses."""
    pos = torch.randint(0, 99, (7, 2), device=dev)
    x = torch.randn(3, 4, 7, 32, device=dev)
    want = rope64(x.transpose(1, 2), pos, (16, 16), 100.0, 1)
    rope_near(ops.rope_axes(x.transpose(1, 2), pos, (16, 16), base=100.0), x.transpose(1, 2), want, torch.float32)
    qkv = torch.randn(3, 7, 3, 4, 32, device=dev)
    rope_near(ops.rope_axes(qkv[:, :, 1], pos, (16, 16)), qkv[:, :, 1], rope64(qkv[:, :, 1], pos, (16, 16), 10000.0, 1),
              torch.float32)
    e = torch.randn(1, 7, 4, 32, device=dev).expand(5, 7, 4, 32)
    rope_near(ops.rope_axes(e, pos, (16, 16)), e, rope64(e, pos, (16, 16), 10000.0, 1), torch.float32)
    for shift in (1, 2):
        o = torch.randn(7 * 4 * 32 + 4, device=dev)[shift:shift + 7 * 4 * 32].view(1, 7, 4, 32)
        rope_near(ops.rope_axes(o, pos, (16, 16)), o, rope64(o, pos, (16, 16), 10000.0, 1), torch.float32)
    assert ops.rope_axes(x[:0].transpose(1, 2), pos, (16, 16)).shape == (0, 7, 4, 32)
    with pytest.raises(ValueError):
        ops._h().rope_axes(e, pos, (16, 16), out=e)


# ---------------------------------------------------------------------------------------------------------------
# together: a convolutional block's norm, its dropout and a rotary attention's projection, as a training step runs them
def together(x, w, b, qkv, uids, tag, pos):
    y = ops.group_norm(x, 8, w, b, act="relu")
    y = ops.client_dropout(y, uids, 7, tag, 0, 0.25, kind="channel")
    y = ops.group_norm(y, 4, act="silu", residual=x)
    y = ops.client_dropout(y, uids, 7, tag, 1, 0.1)
    t = y.flatten(2).transpose(1, 2) @ qkv  # [R, tokens, 3 * 2 * 12]
    t = ops.rope_axes(t.reshape(t.shape[0], -1, 3, 2, 12), pos, (6, 6), slots=2)
    q, k, v = t.permute(2, 0, 3, 1, 4)
    a = torch.softmax((q.unsqueeze(-2) * k.unsqueeze(-3)).sum(-1) * 0.25, -1)
    return (a.unsqueeze(-1) * v.unsqueeze(-3)).sum(-2)


def together_inputs(device, seed=3):
    g = torch.Generator().manual_seed(seed)
    x = last(torch.randn(6, 32, 4, 4, generator=g)).to(device)
    w, b = (1 + 0.2 * torch.rand(3, 32, generator=g)).to(device), (0.2 * torch.randn(3, 32, generator=g)).to(device)
    qkv = (0.2 * torch.randn(32, 72, generator=g)).to(device)
    pos = torch.stack([torch.arange(16) // 4, torch.arange(16) % 4], -1).to(device)
    return x, w, b, qkv, torch.tensor([4, 9, 2], device=device), torch.tensor([seed], device=device), pos


def together_step(args):
    leaves = [t.detach().requires_grad_(True) for t in args[:4]]
    out = together(*leaves, *args[4:])
    return [out.detach()] + list(torch.autograd.grad(out.square().sum(), leaves))


def test_layers_together_differences_cpu():
    """The chain's gradient against central differences, in 64 bits (smooth where no gate is within a step of its border)."""
    args = together_inputs("cpu")
    args = [t.double() if t.is_floating_point() else t for t in args]
    got = together_step(args)
    g = torch.Generator().manual_seed(0)
    for i in range(4):
        d = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        h = 1e-7

        def at(s):
            a = list(args)
            a[i] = args[i] + s * h * d
            return float(together(*a).square().sum())

        want, have = (at(1) - at(-1)) / (2 * h), float((got[1 + i] * d).sum())
        # differences: rounding 2^-52 * |f| / h and a third-order term h^2
        assert abs(want - have) <= 1e-5 * max(1.0, abs(have), abs(float(got[0].square().sum())))


@pytest.mark.gpu
def test_layers_together_gpu_matches_64_bits(dev):
    args = together_inputs("cpu")
    want = together_step([t.double() if t.is_floating_point() else t for t in args])
    got = together_step([t.to(dev) for t in args])
    for a, b in zip(got, want):
        # relative to the largest entry: a chain of under 30 roundings of 512 u each (see gn_check), slopes of order 1
        assert float((a.cpu().double() - b).abs().max()) <= 30 * 512 * U32 * max(1.0, float(b.abs().max()))


@pytest.mark.gpu
def test_layers_on_another_stream_and_in_a_graph(dev):
    """A side stream's result equals the default stream's; a captured forward and backward pass follows new inputs and a
    new tag over several replays with eager work in between."""
    args = [t.to(dev) for t in together_inputs("cpu")]
    want = together_step(args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = together_step(args)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = [t.clone(memory_format=torch.preserve_format) for t in args]
    with torch.cuda.stream(s):
        for _ in range(2):
            together_step(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = together_step(static)
    for seed in (3, 5, 6, 3):
        new = [t.to(dev) for t in together_inputs("cpu", seed)]
        for t, n in zip(static, new):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        eager = together_step(new)
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.gpu
def test_layers_under_functorch_transforms_use_the_oracle(dev):
    from torch.func import grad, vmap

    x = torch.randn(3, 4, 8, 2, 2, device=dev)
    w = torch.rand(3, 8, device=dev)

    def loss(w1, x1):
        return ops.group_norm(x1, 2, w1, act="silu").square().sum()

    g0 = grad(lambda w1: loss(w1, x[0]))(w[0])  # only the weight is wrapped
    got = vmap(grad(loss))(w, x)
    torch.testing.assert_close(got[0], g0, rtol=1e-4, atol=1e-4)
    wl = w.clone().requires_grad_(True)
    ops.group_norm(x.reshape(12, 8, 2, 2), 2, wl, act="silu").square().sum().backward()
    torch.testing.assert_close(got, wl.grad, rtol=1e-4, atol=1e-4)


def layer_calls(dev):
    x = last(torch.randn(6, 8, 4, 4)).to(dev)
    uids, tag = torch.arange(3, device=dev), torch.ones(1, dtype=torch.int64, device=dev)
    pos = torch.arange(8, device=dev).unsqueeze(1)
    return x, [lambda t: ops.group_norm(t, 2, act="gelu"), lambda t: ops.client_dropout(t, uids, 1, tag, 0, 0.5),
               lambda t: ops.client_dropout(t, uids, 1, 7, 0, 0.5), lambda t: ops.rope_axes(t, pos, (4,))]


@pytest.mark.gpu
def test_layers_autograd_contract(dev):
    """A second backward pass needs retain_graph, a second differentiation raises, a changed input raises, and gradients
    reach a graph in front of the layer."""
    x, calls = layer_calls(dev)
    for f in calls:
        a = x.clone(memory_format=torch.preserve_format).requires_grad_(True)
        y = f(a)
        gy = torch.randn_like(y)
        g1 = torch.autograd.grad(y, a, gy, retain_graph=True)[0]
        assert torch.equal(torch.autograd.grad(y, a, gy)[0], g1)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, a, gy)
        (g2,) = torch.autograd.grad(f(a), a, gy, create_graph=True)
        assert torch.equal(g2, g1)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g2.sum(), a)
        torch.testing.assert_close(torch.autograd.grad(f(a * 1.0), a, gy)[0], g1)
        with torch.no_grad():
            z = f(a)
        assert not z.requires_grad and torch.equal(z, y)
        with torch.inference_mode():
            assert torch.equal(f(x), y)
    a = x.clone(memory_format=torch.preserve_format).requires_grad_(True)
    b = a * 1.0
    y = ops.group_norm(b, 2)
    with torch.no_grad():
        b.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()
    # the same tensor as input and residual, and as a layer's only leaf twice
    a = x.clone(memory_format=torch.preserve_format).requires_grad_(True)
    ops.group_norm(a, 2, act="silu", residual=a).sum().backward()
    c = x.double().cpu().requires_grad_(True)
    ops.group_norm(c, 2, act="silu", residual=c).sum().backward()
    assert float((a.grad.cpu().double() - c.grad).abs().max()) <= 2 * 512 * U32 * 40


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["contiguous", "host", "shifted"])
def test_saved_tensors_that_move(dev, how):
    """Saved tensors may come back from hooks with other strides, from the host, or at other addresses."""
    def unpack(t):
        if how == "host":
            return t.to(dev)
        if how == "contiguous" or t.dim() == 0:
            return t
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=dev)[1:].view(t.shape)  # off by one element
        return buf.copy_(t)

    def pack(t):
        return t.cpu() if how == "host" else t.contiguous().clone()

    K, C = 3, 16
    rows = torch.randn(K, 5 * C, device=dev)  # per-client affine vectors inside longer rows
    x = last(torch.randn(6, C, 5, 5, device=dev))
    r = last(torch.randn(6, C, 5, 5, device=dev))
    gy = torch.randn(6, C, 5, 5, device=dev)
    uids, tag = torch.arange(3, device=dev), torch.ones(1, dtype=torch.int64, device=dev)
    pos = torch.arange(C, device=dev).unsqueeze(1)

    def grads():
        out = []
        for act in ("none", "relu", "gelu"):
            leaves = [t.detach().requires_grad_(True) for t in (x, rows[:, C:2 * C], rows[:, 3 * C:4 * C], r)]
            a, w, b, s = leaves
            assert w.stride(0) == 5 * C
            out += torch.autograd.grad(ops.group_norm(a, 4, w, b, act=act, residual=s), leaves, gy)
        shared = rows[0, :C].detach().requires_grad_(True)
        out += torch.autograd.grad(ops.group_norm(x, 4, shared.expand(K, C), None, act="silu"), shared, gy)
        a = x.detach().requires_grad_(True)
        out += torch.autograd.grad(ops.client_dropout(a, uids, 1, tag, 0, 0.5), a, gy)
        a = torch.empty_like(gy[..., :4]).copy_(gy[..., :4]).requires_grad_(True)
        return out + list(torch.autograd.grad(ops.rope_axes(a, pos, (4,)), a, gy[..., :4]))

    want = grads()
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        got = grads()
    for g, w in zip(got, want):
        assert torch.equal(g, w)


@pytest.mark.gpu
def test_saved_tensors_that_change_are_refused(dev):
    x, calls = layer_calls(dev)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.reshape(-1)[:1].clone()):
        for f in calls:
            a = x.clone(memory_format=torch.preserve_format).requires_grad_(True)
            y = f(a)
            with pytest.raises(RuntimeError, match="saved tensor"):
                y.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "silu"])
def test_group_norm_gradient_at_any_address(dev, act):
    """Groups of more than 1024 channels need accesses of four: a gradient at an odd address is brought in line."""
    x = last(torch.randn(2, 2048, 3, device=dev)).requires_grad_(True)
    gy = torch.randn(2 * 3 * 2048 + 1, device=dev)[1:].view(2, 3, 2048).movedim(-1, 1)
    y = ops.group_norm(x, 1, act=act)
    (g1,) = torch.autograd.grad(y, x, gy, retain_graph=True)
    (g2,) = torch.autograd.grad(y, x, last(gy.clone()))
    assert gy.data_ptr() % 16 and torch.equal(g1, g2)


@pytest.mark.gpu
def test_layers_from_two_threads_and_streams(dev):
    """Calls from two threads on two streams at once give what one gives alone."""
    import threading

    x, calls = layer_calls(dev)
    x = x.repeat(50, 1, 1, 1).contiguous(memory_format=torch.channels_last)

    def work(out):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(s):
            for _ in range(20):
                a = x.detach().requires_grad_(True)
                res = []
                for f in calls[:3]:
                    y = f(a)
                    res += [y.detach(), torch.autograd.grad(y, a, x)[0]]
                out[:] = res
        s.synchronize()

    torch.cuda.synchronize()
    want, outs = [], [[], []]
    work(want)
    threads = [threading.Thread(target=work, args=(o,)) for o in outs]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for o in outs:
        assert len(o) == len(want) and all(torch.equal(p, q) for p, q in zip(o, want))


@pytest.mark.gpu
def test_layers_many_small_samples(dev):
    """More samples than a grid of workgroups holds at once, one pixel each; offsets stay right to the last row."""
    N = (1 << 22) + 5
    x = torch.randn(N, 8, device=dev)
    y = ops.group_norm(x, 2, act="relu")
    for rows in (slice(0, 3), slice(N - 3, N), slice((1 << 21) - 2, (1 << 21) + 2)):
        want = gn64(x[rows], 2, None, None, 1e-5, "relu", None, x[rows])["y"]
        assert float((y[rows].double() - want).abs().max()) <= 2 * 512 * U32 * 4


@pytest.mark.gpu
def test_layers_past_32_bit_offsets(dev):
    """Tensors of more than 2^32 bytes and 2^31 elements: the last samples are right."""
    R = (1 << 31) // (64 * 384) + 64
    x = torch.ones(R, 64, 3, 2, 64, device=dev, dtype=torch.bfloat16)
    x[-2:] = torch.randn(2, 64, 3, 2, 64, device=dev).to(torch.bfloat16)
    pos = torch.stack([torch.arange(64, device=dev) // 8, torch.arange(64, device=dev) % 8], -1)
    y = ops.rope_axes(x, pos, (32, 32), slots=2)
    rope_near(y[-2:], x[-2:], rope64(x[-2:], pos, (32, 32), 10000.0, 2), torch.bfloat16)
    del y
    v = x.view(-1)[: ((1 << 31) + 4096 * 8) // 64 * 64]
    uids = torch.tensor([3, 8], device=dev)
    a = v[: v.numel() // 2 * 2].view(2, -1)
    y = ops.client_dropout(a, uids, 9, 4, 1, 0.25)
    n = a.shape[1]
    m = ref.client_dropout_mult(uids[1:].cpu(), 4, 9, 4, 1, 0.25)  # the start of the second client's share
    assert torch.equal((y[1, :4] != 0).cpu(), (a[1, :4].cpu() * m[0].to(torch.bfloat16)) != 0)
    tail = ref._philox4x32(*(torch.tensor([t]) for t in ((n - 4) >> 2, 8, 4, 2 + 256)), 9, 0)
    keep = torch.tensor([(int(w) >> 8) * 2.0 ** -24 >= 0.25 for w in tail])
    want = torch.where(keep, a[1, -4:].cpu().double() / 0.75, torch.zeros(4, dtype=torch.float64))
    torch.testing.assert_close(y[1, -4:].cpu().double(), want, rtol=half_step(torch.bfloat16) + 4 * U32, atol=0)
    del y, a, v
    N = (1 << 31) // (64 * 1024) + 3
    x = x.view(-1)[: N * 65536].view(N, 32, 32, 64).permute(0, 3, 1, 2)
    x[-2:] = torch.randn(2, 64, 32, 32, device=dev).to(torch.bfloat16)
    y = ops.group_norm(x, 32, act="silu")
    want = gn64(x[-2:], 32, None, None, 1e-5, "silu", None, x[-2:])
    assert bool(((y[-2:].double() - want["y"]).abs() <= 4 * 512 * U32 * 8 + half_step(torch.bfloat16) * want["y"].abs()).all())


@pytest.mark.parametrize("N,P,C,G", [(12693514, 109, 387, 43), (4780147, 238, 327, 109), (1 << 19, 256, 2048, 64),
                                     (48, 12544, 64, 8)])
def test_group_norm_plan_counts_every_grid(N, P, C, G):
    """A launch's threads are counted in 32 bits, and the kernels that join chunks have 256 per (sample, group): read off the
    plan's workspace, which holds one entry of 8 bytes per sample of a piece, chunk and group."""
    import ctypes

    from blades_amd.ops import build

    if not os.path.exists(build.HIP_LIB):
        pytest.skip("kernels are not built")
    lib = ctypes.CDLL(build.HIP_LIB)
    lib.blades_group_norm_plan_size.restype = ctypes.c_long
    buf, ws = ctypes.create_string_buffer(lib.blades_group_norm_plan_size()), (ctypes.c_long * 2)()
    L, I = ctypes.c_long, ctypes.c_int

    def plan(n, p, c, g):
        return lib.blades_group_norm_plan(buf, L(n), L(p), I(c), I(g), ctypes.c_float(1e-5), I(0), I(n), L(0), L(0), I(1),
                                          I(1 if c % 4 else 4), ws)

    assert plan(N, P, C, G) == 0
    # the backward pass's is N x chunks x C entries and at most N x G for the means
    chunks = max(1, -(-ws[1] // (N * C * 8)) - 1)
    assert ws[0] // (8 * chunks) * 256 < 1 << 32
    assert plan(1, 1, (1 << 24) + 4, 1 << 22) != 0 and plan(1 << 24, 1, 4, 1) != 0
