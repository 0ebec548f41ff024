"""Cases of the batch-independent training layers: group norm with an activation (channels last), client-keyed dropout
whose mask is recomputed instead of stored, and rotary positions with several axes.

Every case is one pass of a layer: forward, or forward and backward.  ``own`` false: elementary torch operations in
32 bits (64 for Philox words' products, far angles); true: the package's kernels."""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
_DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    gn = {"op": "group_norm", "dtype": "float32", "act": "relu", "residual": False, "train": True, "clients": 0}
    dr = {"op": "dropout", "dtype": "float32", "kind": "elem", "layout": "major", "p": 0.1}
    ro = {"op": "rope", "dtype": "float32", "slots": 2, "packed": 3, "train": True, "per_sample": False, "far": 0}
    return [
        # one CIFAR-sized image through the first stage of a ResNet: evaluation of a single sample, latency
        {**gn, "name": "gn_one_image", "n": 1, "c": 64, "h": 32, "w": 32, "groups": 32, "train": False},
        # first ResNet stage of a training chunk: 32 clients x 64 samples, each client with weights of its own
        {**gn, "name": "gn_stage1_train", "n": 2048, "c": 64, "h": 32, "w": 32, "groups": 32, "clients": 32},
        # end of a residual block of the last stage: norm, shortcut and ReLU in one, weights shared by the clients
        {**gn, "name": "gn_stage4_residual", "n": 2048, "c": 512, "h": 4, "w": 4, "groups": 32, "residual": True},
        # second stage in the bf16 compute mode, smooth activation
        {**gn, "name": "gn_stage2_bf16", "n": 2048, "c": 128, "h": 16, "w": 16, "groups": 32, "dtype": "bfloat16",
         "act": "silu", "clients": 32},
        # convolutional tokenizer of a 224-pixel transformer (7x7 / stride 2): an image no longer fits a workgroup
        {**gn, "name": "gn_tokenizer_224", "n": 48, "c": 64, "h": 112, "w": 112, "groups": 8, "act": "gelu"},
        # odd everything: three channels a group, 9 x 7 maps
        {**gn, "name": "gn_odd", "n": 50, "c": 30, "h": 9, "w": 7, "groups": 10, "residual": True},
        # hidden layer of the MNIST MLP, 60 clients x 64 samples: latency
        {**dr, "name": "drop_mlp", "clients": 60, "batch": 64, "c": 128, "h": 0, "w": 0, "p": 0.2},
        # token activations of the compact transformer, 32 clients x 64 samples x 64 tokens x 128
        {**dr, "name": "drop_tokens", "clients": 32, "batch": 64, "c": 64, "h": 128, "w": 0},
        # whole channels of the convolutional network's last feature maps (channels last, bf16)
        {**dr, "name": "drop_channels_bf16", "clients": 60, "batch": 64, "c": 64, "h": 6, "w": 6, "kind": "channel",
         "p": 0.25, "dtype": "bfloat16"},
        # one token for each of 32 requests, far along its axes: latency
        {**ro, "name": "rope_one_token", "r": 32, "n": 1, "heads": 6, "dim": 64, "axes": "32,32", "train": False,
         "per_sample": True, "far": 100000},
        # q and k of the packed projection of the compact image transformer: 2048 images of 8 x 8 tokens
        {**ro, "name": "rope_images", "r": 2048, "n": 64, "heads": 2, "dim": 64, "axes": "32,32"},
        # video: 16 frames of 14 x 14 patches, each clip with a start time of its own
        {**ro, "name": "rope_video_bf16", "r": 8, "n": 3136, "heads": 6, "dim": 64, "axes": "16,24,24",
         "per_sample": True, "far": 5000, "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("group_norm", "group_norm", "dropout", "rope"))
    dtype = rng.choice(("float32", "float32", "bfloat16"))
    if op == "group_norm":
        groups = rng.choice((1, 2, 4, 5, 8, 10, 16, 32))
        c = groups * _log(rng, 1, max(1, 512 // groups))
        h, w = _log(rng, 2, 112), _log(rng, 2, 112)
        while h * w * (c // groups) < 16:
            h += 1
        most = 2048 * 64 * 1024 * 2 // (3 * c * h * w)
        clients = _log(rng, 2, 32) if most >= 2 and rng.random() < 0.5 else 0
        n = _log(rng, 1, max(1, min(2048, most)))
        if clients:
            clients = min(clients, n)
            n -= n % clients
        return {"op": op, "dtype": dtype, "n": n, "c": c, "h": h, "w": w, "groups": groups, "clients": clients,
                "act": rng.choice(("none", "relu", "relu", "gelu", "silu")), "residual": rng.random() < 0.4,
                "train": rng.random() < 0.8}
    if op == "dropout":
        clients, kind = _log(rng, 1, 64), rng.choice(("elem", "elem", "channel", "sample"))
        c, h, w = rng.choice(((_log(rng, 1, 2000), 0, 0), (_log(rng, 1, 200), _log(rng, 1, 400), 0),
                              (_log(rng, 1, 256), _log(rng, 1, 32), _log(rng, 1, 32))))
        batch = _log(rng, 1, max(1, min(256, 2048 * 64 * 128 // (clients * c * max(h, 1) * max(w, 1)))))
        return {"op": op, "dtype": dtype, "clients": clients, "batch": batch, "c": c, "h": h, "w": w, "kind": kind,
                "layout": rng.choice(("major", "major", "inner")) if not h or w else "major",
                "p": round(rng.uniform(0.02, 0.8), 3)}
    axes = [2 * _log(rng, 1, 16) for _ in range(rng.choice((1, 2, 2, 3)))]
    dim = sum(axes) + 2 * rng.choice((0, 0, 0, 1, 4))
    heads, packed = _log(rng, 1, 12), rng.choice((1, 3, 3))
    n = _log(rng, 1, 4096)
    r = _log(rng, 1, max(1, min(2048, 2048 * 64 * 3 * 128 // (n * heads * dim * packed))))
    return {"op": op, "dtype": dtype, "r": r, "n": n, "heads": heads, "dim": dim, "axes": ",".join(map(str, axes)),
            "packed": packed, "slots": 2 if packed == 3 else 1, "per_sample": rng.random() < 0.4,
            "far": rng.choice((0, 1000, 1000000)), "train": rng.random() < 0.7}


# ---------------------------------------------------------------------------------------------------------------
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _pre64(x, res, w, b, groups):
    """The value in front of the activation, in 64 bits (prepare only)."""
    n, c, h, wd = x.shape
    x64 = x.double().permute(0, 2, 3, 1).reshape(n, h * wd, groups, c // groups)
    var, mean = torch.var_mean(x64, dim=(1, 3), unbiased=False, keepdim=True)
    z = ((x64 - mean) * (var + EPS).rsqrt()).reshape(n, h, wd, c).permute(0, 3, 1, 2)
    k = w.shape[0] if w.dim() == 2 else 1
    z = z.reshape(k, n // k, c, h, wd) * w.double().reshape(k, 1, c, 1, 1) + b.double().reshape(k, 1, c, 1, 1)
    z = z.reshape(n, c, h, wd)
    return z if res is None else z + res.double()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DT[case["dtype"]]
    if case["op"] == "group_norm":
        n, c, h, w, k = (case[i] for i in ("n", "c", "h", "w", "clients"))
        # what a convolution leaves: channels of their own spread and offset
        x = _randn(g, n, h, w, c) * (0.5 + torch.rand(c, generator=g, device="cuda")) + 0.5 * _randn(g, c)
        x = x.to(dt).permute(0, 3, 1, 2)
        res = _randn(g, n, h, w, c).to(dt).permute(0, 3, 1, 2) if case["residual"] else None
        lead = (k, c) if k else (c,)
        wt = 1.0 + 0.25 * torch.rand(*lead, generator=g, device="cuda")
        bs = 0.3 * _randn(g, *lead)
        if case["act"] == "relu":
            # A ReLU's gate within rounding of its border is decided by the last bit: such an element (one in ten
            # thousand) is moved off it, so that every way of computing the layer has the same gradient.
            for _ in range(2):
                near = _pre64(x, res, wt, bs, case["groups"]).abs() < 1e-4
                if res is not None:
                    res = torch.where(near, res + 0.0625, res)
                else:
                    x = torch.where(near, x + 0.0625, x)
        x = x.contiguous(memory_format=torch.channels_last)
        st = {"case": case, "x": x, "w": wt, "b": bs, "res": None, "gy": None}
        if res is not None:
            st["res"] = res.contiguous(memory_format=torch.channels_last)
        if case["train"]:
            st["gy"] = _randn(g, n, h, w, c).to(dt).permute(0, 3, 1, 2)
            for t in ("x", "w", "b", "res"):
                if st[t] is not None:
                    st[t].requires_grad_(True)
        return st
    if case["op"] == "dropout":
        k, b, c, h, w = (case[i] for i in ("clients", "batch", "c", "h", "w"))
        lead = (k * b, c) if case["layout"] == "major" else (b, k * c)
        if w:
            x = _randn(g, lead[0], h, w, lead[1]).to(dt).permute(0, 3, 1, 2)
            gy = _randn(g, lead[0], h, w, lead[1]).to(dt).permute(0, 3, 1, 2)
        else:
            shape = lead + ((h,) if h else ())
            x, gy = _randn(g, *shape).to(dt), _randn(g, *shape).to(dt)
        return {"case": case, "x": x.requires_grad_(True), "gy": gy, "key": 1000003 * int(seed) + 17, "layer": 3,
                "uids": torch.randperm(1000, generator=g, device="cuda")[:k],
                "tag": torch.randint(1, 100000, (1,), generator=g, device="cuda")}
    r, n, heads, dim, s = (case[i] for i in ("r", "n", "heads", "dim", "packed"))
    axes = [int(a) for a in case["axes"].split(",")]
    shape = (r, n, 3, heads, dim) if s == 3 else (r, n, heads, dim)
    grid = [max(1, round(n ** (1.0 / len(axes))))] * len(axes)
    t = torch.arange(n, device="cuda")
    cols = []
    for e in reversed(grid[1:]):  # row-major walk over the axes, the first one unbounded
        cols.append(t % e)
        t = t // e
    pos = torch.stack([t] + cols[::-1], dim=-1)
    if case["per_sample"]:
        pos = pos.unsqueeze(0) + torch.randint(0, case["far"] + 1, (r, 1, len(axes)), generator=g, device="cuda")
    elif case["far"]:
        pos = pos + torch.randint(0, case["far"] + 1, (1, len(axes)), generator=g, device="cuda")
    st = {"case": case, "x": _randn(g, *shape).to(dt), "pos": pos, "axes": axes, "gy": None}
    if case["train"]:
        st["gy"] = _randn(g, *shape).to(dt)
        st["x"].requires_grad_(True)
    return st


# ---------------------------------------------------------------------------------------------------------------
def _act(z, act):
    """(activation, its derivative)."""
    if act == "relu":
        on = (z > 0).float()
        return z * on, on
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    return z, None


def _plain_group_norm(st):
    case, x = st["case"], st["x"]
    n, c, h, w = x.shape
    groups, dt = case["groups"], x.dtype
    k = case["clients"] or 1
    # channels innermost, as they lie: [client, sample, pixel, group, channel of the group]
    xl = x.permute(0, 2, 3, 1).float().reshape(k, n // k, h * w, groups, c // groups)
    gamma = st["w"].reshape(k, 1, 1, groups, c // groups)
    beta = st["b"].reshape(k, 1, 1, groups, c // groups)
    d = xl - xl.mean(dim=(2, 4), keepdim=True)
    rstd = (d.square().mean(dim=(2, 4), keepdim=True) + EPS).rsqrt()
    xhat = d * rstd
    z = xhat * gamma + beta
    if st["res"] is not None:
        z = z + st["res"].permute(0, 2, 3, 1).float().reshape(z.shape)
    y, slope = _act(z, case["act"])

    def out(t):
        return t.reshape(n, h, w, c).permute(0, 3, 1, 2).to(dt)

    if st["gy"] is None:
        return {"y": out(y)}
    g = st["gy"].permute(0, 2, 3, 1).float().reshape(z.shape)
    g = g if slope is None else g * slope
    dxhat = g * gamma
    dx = rstd * (dxhat - dxhat.mean(dim=(2, 4), keepdim=True) - xhat * (dxhat * xhat).mean(dim=(2, 4), keepdim=True))
    got = {"y": out(y), "dx": out(dx), "dw": (g * xhat).sum(dim=(1, 2)).reshape(st["w"].shape),
           "db": g.sum(dim=(1, 2)).reshape(st["b"].shape)}
    if st["res"] is not None:
        got["dres"] = out(g)
    return got


def _philox(c0, c1, c2, c3, key):
    """Philox4x32-10 (Salmon et al., SC'11) on int64 tensors holding 32-bit words."""
    mask = 0xFFFFFFFF
    k0, k1 = key & mask, (key >> 32) & mask
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & mask) ^ c1 ^ k0, p1 & mask, ((p0 >> 32) & mask) ^ c3 ^ k1, p0 & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack((c0, c1, c2, c3), dim=-1)


def _plain_dropout(st):
    case, x = st["case"], st["x"]
    k, b, c, p = case["clients"], case["batch"], case["c"], case["p"]
    tail = list(x.shape[2:])
    # the dimensions a mask value is drawn for: all of them, (sample, channel), or the sample alone
    keep = [b] if case["kind"] == "sample" else [b, c] if case["kind"] == "channel" and tail else [b, c] + tail
    n = math.prod(keep)
    block = torch.arange((n + 3) // 4, device=x.device).unsqueeze(0) + torch.zeros_like(st["uids"]).unsqueeze(1)
    words = _philox(block, st["uids"].unsqueeze(1) + torch.zeros_like(block), st["tag"] + torch.zeros_like(block),
                    torch.full_like(block, 2 + 256 * st["layer"]), st["key"])
    u = (words >> 8).reshape(k, -1)[:, :n].float() * (1.0 / 16777216.0)
    m = ((u >= p).float() * (1.0 / (1.0 - p))).reshape([k] + keep)
    m = m.reshape([k] + keep + [1] * (2 + len(tail) - len(keep)))
    if case["layout"] == "inner":
        m = m.transpose(0, 1)  # [batch, client, channel, ...]
        shape = [b, k, c] + tail
    else:
        shape = [k, b, c] + tail
    y = (x.float().reshape(shape) * m).reshape(x.shape)
    dx = (st["gy"].float().reshape(shape) * m).reshape(x.shape)
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype)}


def _plain_rotate(x, pos, axes, slots, sign):
    half = [torch.arange(a // 2, device=x.device, dtype=torch.float64) * (-2.0 / a) for a in axes]
    freq = 10000.0 ** torch.cat(half)
    axis = torch.repeat_interleave(torch.arange(len(axes), device=x.device),
                                   torch.tensor([a // 2 for a in axes], device=x.device))
    angle = pos.double()[..., axis] * freq  # [(sample,) token, pair]: far positions need the 64 bits
    cos, sin = torch.cos(angle).float().unsqueeze(-2), (sign * torch.sin(angle)).float().unsqueeze(-2)
    xf = x.float()
    if x.dim() == 5:
        cos, sin = cos.unsqueeze(-3), sin.unsqueeze(-3)
        part, rest = xf[:, :, :slots], xf[:, :, slots:]
    else:
        part, rest = xf, None
    rot = sum(axes)
    a, b = part[..., 0:rot:2], part[..., 1:rot:2]
    turned = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    turned = torch.cat((turned, part[..., rot:]), dim=-1)
    return (turned if rest is None else torch.cat((turned, rest), dim=2)).to(x.dtype)


def run(state):
    case = state["case"]
    if own:
        from blades_amd import ops

        if case["op"] == "group_norm":
            y = ops.group_norm(state["x"], case["groups"], state["w"], state["b"], eps=EPS, act=case["act"],
                               residual=state["res"])
            if state["gy"] is None:
                return {"y": y}
            names = ["x", "w", "b"] + (["res"] if state["res"] is not None else [])
            grads = torch.autograd.grad(y, [state[i] for i in names], state["gy"])
            return {"y": y, **{"d" + i: t for i, t in zip(names, grads)}}
        if case["op"] == "dropout":
            y = ops.client_dropout(state["x"], state["uids"], state["key"], state["tag"], state["layer"], case["p"],
                                   kind=case["kind"], layout=case["layout"])
            return {"y": y, "dx": torch.autograd.grad(y, state["x"], state["gy"])[0]}
        y = ops.rope_axes(state["x"], state["pos"], state["axes"], slots=case["slots"])
        if state["gy"] is None:
            return {"y": y}
        return {"y": y, "dx": torch.autograd.grad(y, state["x"], state["gy"])[0]}
    with torch.no_grad():
        if case["op"] == "group_norm":
            return _plain_group_norm(state)
        if case["op"] == "dropout":
            return _plain_dropout(state)
        got = {"y": _plain_rotate(state["x"], state["pos"], state["axes"], case["slots"], 1.0)}
        if state["gy"] is not None:
            got["dx"] = _plain_rotate(state["gy"], state["pos"], state["axes"], case["slots"], -1.0)
        return got


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "group_norm":
        e = case["n"] * case["c"] * case["h"] * case["w"]
        fwd, both = (3, 6) if case["residual"] else (2, 4)  # x (res) y; and gy dx (dres)
        cost = {"none": 0, "relu": 1, "gelu": 12, "silu": 6}[case["act"]]
        return {"bytes": e * size * (both if case["train"] else fwd),
                "flops": e * (8 + cost + (14 + cost if case["train"] else 0))}
    if case["op"] == "dropout":
        e = case["clients"] * case["batch"] * case["c"] * max(case["h"], 1) * max(case["w"], 1)
        draws = {"elem": e, "sample": case["clients"] * case["batch"],
                 "channel": case["clients"] * case["batch"] * case["c"] if case["h"] else e}[case["kind"]]
        return {"bytes": 4 * e * size, "flops": 2 * e + 20 * draws}
    e = case["r"] * case["n"] * case["packed"] * case["heads"] * case["dim"]
    turned = e // case["packed"] * case["slots"]
    passes = 2 if case["train"] else 1
    return {"bytes": passes * 2 * e * size, "flops": passes * 3 * turned}


# ---------------------------------------------------------------------------------------------------------------
def _exact_group_norm(st):
    """The definition differentiated by autograd, in 64 bits."""
    case = st["case"]
    x, w, b = (st[i].detach().double().requires_grad_(True) for i in ("x", "w", "b"))
    res = None if st["res"] is None else st["res"].detach().double().requires_grad_(True)
    n, c = x.shape[:2]
    flat = x.reshape(n, case["groups"], -1)
    var, mean = torch.var_mean(flat, dim=2, unbiased=False, keepdim=True)
    z = ((flat - mean) / torch.sqrt(var + EPS)).reshape(x.shape)
    each = (lambda t: t.reshape(1, c)) if w.dim() == 1 else (lambda t: t.repeat_interleave(n // t.shape[0], dim=0))
    z = z * each(w)[:, :, None, None] + each(b)[:, :, None, None]
    if res is not None:
        z = z + res
    if case["act"] == "relu":
        y = torch.clamp_min(z, 0.0)
    elif case["act"] == "gelu":
        y = z * torch.special.ndtr(z)
    elif case["act"] == "silu":
        y = z * torch.sigmoid(z)
    else:
        y = z
    if st["gy"] is None:
        return {"y": y.detach()}
    names, leaves = ["dx", "dw", "db"], [x, w, b]
    if res is not None:
        names, leaves = names + ["dres"], leaves + [res]
    return {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, leaves, st["gy"].double())))}


def _exact_words(uid, tag, c3, key, blocks):
    """The same generator on numpy's unsigned words: [blocks, 4]."""
    m = np.uint64(0xFFFFFFFF)
    s = np.uint64(32)
    c = [np.arange(blocks, dtype=np.uint64)] + [np.full(blocks, v & 0xFFFFFFFF, np.uint64) for v in (uid, tag, c3)]
    k0, k1 = key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s) ^ c[1] ^ np.uint64(k0), b & m, (a >> s) ^ c[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return np.stack(c, axis=1)


def _exact_dropout(st):
    case = st["case"]
    k, b, c = case["clients"], case["batch"], case["c"]
    tail = tuple(st["x"].shape[2:])
    one = (1,) * len(tail)
    value = {"sample": (1,) + one, "channel": (c,) + one, "elem": (c,) + tail}[case["kind"]]  # of one sample
    per = math.prod(value)
    if k * b * per > 4e7:
        return None
    least = int(math.ceil(float(np.float32(case["p"])) * 2 ** 24))  # a 24-bit draw below it is dropped
    masks = []
    for uid in st["uids"].tolist():
        words = _exact_words(uid, int(st["tag"]), 2 + 256 * st["layer"], st["key"], (b * per + 3) // 4)
        masks.append((words >> np.uint64(8)).reshape(-1)[: b * per] >= least)
    m = torch.from_numpy(np.stack(masks)).cuda().double() / (1.0 - case["p"])
    m = m.reshape((k, b) + value).expand((k, b, c) + tail)
    m = m.permute(1, 0, *range(2, m.dim())) if case["layout"] == "inner" else m
    m = m.reshape(st["x"].shape)
    return {"y": st["x"].detach().double() * m, "dx": st["gy"].double() * m}


def _exact_rope(st):
    """Each pair as a complex number times exp(i angle), in 64 bits."""
    case, axes = st["case"], st["axes"]
    x = st["x"].detach()
    angles = []
    for j, a in enumerate(axes):
        f = torch.exp(-math.log(10000.0) * torch.arange(0, a, 2, device=x.device, dtype=torch.float64) / a)
        angles.append(st["pos"][..., j: j + 1].double() * f)
    angle = torch.cat(angles, dim=-1).unsqueeze(-2)
    rot = sum(axes)

    def turn(t, way):
        out = t.double().clone()
        part = out[:, :, : case["slots"]] if t.dim() == 5 else out
        ang = angle.unsqueeze(-3) if t.dim() == 5 else angle
        pairs = torch.view_as_complex(part[..., :rot].reshape(*part.shape[:-1], rot // 2, 2).contiguous())
        pairs = pairs * torch.polar(torch.ones_like(ang), way * ang)
        part[..., :rot] = torch.view_as_real(pairs).flatten(-2)
        return out

    got = {"y": turn(x, 1.0)}
    if st["gy"] is not None:
        got["dx"] = turn(st["gy"], -1.0)
    return got


def exact(case, seed):
    st = prepare(case, seed)
    return {"group_norm": _exact_group_norm, "dropout": _exact_dropout, "rope": _exact_rope}[case["op"]](st)
