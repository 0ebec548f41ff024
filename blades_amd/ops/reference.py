"""Plain-PyTorch fp32 reference ("oracle") of every update-matrix primitive.

Each function here defines the numerical contract of the HIP kernel with the
same name in ``csrc/`` (see ``blades_amd/ops/__init__.py`` for the dispatch).
They run on any device; on CPU they are what the non-GPU test tier executes,
and on the GPU test tier they are what each kernel is compared against.

``U`` is always the ``[K, Dl]`` fp32 update matrix (row = client, column =
parameter coordinate; ``Dl`` is the local column shard).  ``mask`` is an
optional ``[K]`` tensor; rows with ``mask == 0`` do not take part.
"""
import math
from typing import Optional, Tuple

import torch


def _maskf(U, mask):
    if mask is None:
        return None
    return mask.to(device=U.device, dtype=torch.float32)


def weighted_col_sum(U: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """``out[j] = sum_i w[i] * U[i, j]``."""
    return torch.mv(U.t(), w.to(U.dtype))


def col_mean(U: torch.Tensor, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    if mask is None:
        return U.mean(dim=0)
    m = _maskf(U, mask)
    return weighted_col_sum(U, m / m.sum())


def col_mean_std(U, mask=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Column mean and *unbiased* std over the selected rows
    (``torch.std`` default, reference ``alie_adversary.py:29-30``)."""
    if mask is not None:
        U = U[_maskf(U, mask) > 0]
    return U.mean(dim=0), U.std(dim=0)


def col_min_max(U, mask=None):
    if mask is not None:
        U = U[_maskf(U, mask) > 0]
    return U.min(dim=0).values, U.max(dim=0).values


def col_median(U, mask=None) -> torch.Tensor:
    """Mean of lower and upper median (reference ``aggregators.py:12-16``)."""
    if mask is not None:
        U = U[_maskf(U, mask) > 0]
    upper = U.median(dim=0).values
    lower = (-U).median(dim=0).values
    return (upper - lower) / 2


def col_trimmed_mean(U, b: int, mask=None) -> torch.Tensor:
    """Mean after dropping the ``b`` largest and ``b`` smallest per column
    (reference ``aggregators.py:40-48``)."""
    if mask is not None:
        U = U[_maskf(U, mask) > 0]
    n = U.shape[0]
    if n <= 2 * b:
        raise ValueError("Not enough inputs to compute trimmed mean")
    if b == 0:
        return U.mean(dim=0)
    s = torch.sort(U, dim=0).values
    return s[b: n - b].sum(dim=0) / (n - 2 * b)


def row_stats(U: torch.Tensor, valid_cols: Optional[int] = None):
    """Per-row ``(sum of squares [K] f32, counts [K,3] i64 of >0, <0, ==0)``
    over the first ``valid_cols`` columns (the rest is shard padding)."""
    if valid_cols is not None and valid_cols < U.shape[1]:
        U = U[:, :valid_cols]
    sq = (U * U).sum(dim=1)
    pos = (U > 0).sum(dim=1)
    neg = (U < 0).sum(dim=1)
    zero = (U == 0).sum(dim=1)
    return sq, torch.stack([pos, neg, zero], dim=1).to(torch.int64)


def row_sqnorm(U):
    return (U * U).sum(dim=1)


def sqdist_to(U: torch.Tensor, m: torch.Tensor) -> torch.Tensor:
    """``out[i] = sum_j (U[i,j] - m[j])^2`` (partial over the local columns)."""
    d = U - m.unsqueeze(0)
    return (d * d).sum(dim=1)


def row_dot(U: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """``out[i] = sum_j U[i,j] * v[j]`` (partial over the local columns)."""
    return torch.mv(U, v.to(U.dtype))


def gram(U: torch.Tensor) -> torch.Tensor:
    """``U @ U.T`` in fp32 (partial over the local columns)."""
    return U @ U.t()


def gram_batched(S: torch.Tensor) -> torch.Tensor:
    """``S[b] @ S[b].T`` for a stack ``[B, K, n]``."""
    return torch.bmm(S, S.transpose(1, 2))


_M64 = (1 << 64) - 1


def _splitmix64(z: int) -> int:
    z = (z + 0x9E3779B97F4A7C15) & _M64
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & _M64
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & _M64
    return z ^ (z >> 31)


def sample_distinct(D: int, n: int, iters: int, seed: int) -> torch.Tensor:
    """``iters`` sets of ``n`` distinct ids in ``[0, D)``: set ``it`` is the image of ``0..n-1`` under a keyed
    pseudo-random permutation of ``[0, D)`` (balanced Feistel network, eight rounds, cycle walking).  The same numbers as
    ops/csrc/colgather.hip::sample_distinct_kernel, bit for bit.  int64 ``[iters, n]``."""
    import numpy as np

    if not (1 <= n <= D <= (1 << 40) and iters >= 1):
        raise ValueError("sample_distinct: need 1 <= n <= D <= 2^40")
    b = 2
    while (1 << b) < D:
        b += 1
    b += b & 1
    h = b // 2
    mask = np.uint32((1 << h) - 1)
    out = np.empty((iters, n), dtype=np.int64)

    def mix32(x):
        x = x ^ (x >> np.uint32(16))
        x = x * np.uint32(0x85EBCA6B)
        x = x ^ (x >> np.uint32(13))
        x = x * np.uint32(0xC2B2AE35)
        return x ^ (x >> np.uint32(16))

    with np.errstate(over="ignore"):
        for it in range(iters):
            keys = [np.uint32(_splitmix64((seed + 0x632BE59BD9B4E019 * (it * 8 + r + 1)) & _M64) & 0xFFFFFFFF)
                    for r in range(8)]
            x = np.arange(n, dtype=np.uint64)
            todo = np.ones(n, dtype=bool)
            for _ in range(512):
                cur = x[todo]
                L = (cur >> np.uint64(h)).astype(np.uint32)
                R = cur.astype(np.uint32) & mask
                for r in range(8):
                    L, R = R, L ^ (mix32(R + keys[r]) & mask)
                cur = (L.astype(np.uint64) << np.uint64(h)) | R.astype(np.uint64)
                x[todo] = cur
                todo = x >= np.uint64(D)
                if not todo.any():
                    break
            x = np.where(todo, x % np.uint64(D), x)
            out[it] = x.astype(np.int64)
    return torch.from_numpy(out)


def gather_center_cols(U: torch.Tensor, idx: torch.Tensor) -> torch.Tensor:
    """``out[i, k, j] = U[k, idx[i, j]] - mean_k U[k, idx[i, j]]``: ``[iters, K, n]``."""
    iters, n = idx.shape
    S = U.index_select(1, idx.reshape(-1)).view(U.shape[0], iters, n)
    S = S - S.mean(dim=0, keepdim=True)
    return S.permute(1, 0, 2).contiguous()


def row_scale_(U: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """In-place ``U[i, :] *= s[i]``."""
    U.mul_(s.to(U.dtype).unsqueeze(1))
    return U


def set_rows_(U: torch.Tensor, rows: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """In-place ``U[rows[r], :] = v`` (``v`` is ``[Dl]`` or ``[len(rows), Dl]``)."""
    U[rows] = v
    return U


def alie_forge_(U, benign_mask, mal_rows, z: float, sign: Optional[torch.Tensor] = None):
    """Fused ALIE: ``v = mean + z * std * sign`` over benign rows, written
    into every row of ``mal_rows``; returns ``v``."""
    mean, std = col_mean_std(U, benign_mask)
    if sign is not None:
        std = std * sign
    v = mean + z * std
    if mal_rows.numel():
        U[mal_rows] = v
    return v


def ipm_forge_(U, benign_mask, mal_rows, scale: float):
    v = -scale * col_mean(U, benign_mask)
    if mal_rows.numel():
        U[mal_rows] = v
    return v


def server_step_(theta, buf, agg, lr: float, momentum: float, first: bool):
    """Fused server SGD on a flat slice (reference ``server.py:109-130``):
    ``g = -agg; buf = g if first else momentum*buf + g; theta -= lr*buf``
    (``torch.optim.SGD`` with dampening 0, no nesterov, no weight decay)."""
    if momentum != 0.0:
        if first:
            buf.copy_(agg).neg_()
        else:
            buf.mul_(momentum).sub_(agg)
        theta.sub_(buf, alpha=lr)
    else:
        theta.add_(agg, alpha=lr)
    return theta


def client_sgd_step_(W, G, M, lr: float, momentum: float, first: bool,
                     gscale: Optional[torch.Tensor] = None):
    """Fused per-client SGD on the replica matrix ``W[Kc, D]``.

    ``g = G * gscale[row]`` (sign flip / clip coefficient), momentum buffer
    ``M`` as ``torch.optim.SGD``; ``W -= lr * g``."""
    g = G if gscale is None else G * gscale.unsqueeze(1)
    if momentum != 0.0:
        if first:
            M.copy_(g)
        else:
            M.mul_(momentum).add_(g)
        W.sub_(M, alpha=lr)
    else:
        W.sub_(g, alpha=lr)
    return W


# ---------------------------------------------------------------------------
# Counter-based RNG (Philox4x32-10).  Values depend only on (seed, stream,
# global element index), so a sharded run draws exactly the numbers a
# single-GPU run draws for the same coordinates.
# ---------------------------------------------------------------------------
_M0, _M1 = 0xD2511F53, 0xCD9E8D57
_W0, _W1 = 0x9E3779B9, 0xBB67AE85
_MASK = 0xFFFFFFFF


def _philox4x32(c0, c1, c2, c3, k0: int, k1: int):
    """Vectorised Philox4x32-10 on int64 tensors holding uint32 values."""
    for _ in range(10):
        p0 = c0 * _M0
        p1 = c2 * _M1
        hi0, lo0 = (p0 >> 32) & _MASK, p0 & _MASK
        hi1, lo1 = (p1 >> 32) & _MASK, p1 & _MASK
        c0, c1, c2, c3 = (hi1 ^ c1 ^ k0) & _MASK, lo1, (hi0 ^ c3 ^ k1) & _MASK, lo0
        k0 = (k0 + _W0) & _MASK
        k1 = (k1 + _W1) & _MASK
    return c0, c1, c2, c3


def philox_uniform(n: int, seed: int, stream: int, offset: int = 0, device="cpu"):
    """``n`` uniforms in [0,1): element ``e = offset + i`` uses counter
    ``(e//4 lo, e//4 hi, stream, 0)``, lane ``e % 4``, key from ``seed``;
    ``u = (x >> 8) * 2^-24``."""
    e = torch.arange(offset, offset + n, dtype=torch.int64, device=device)
    blk = e >> 2
    c0, c1 = blk & _MASK, (blk >> 32) & _MASK
    c2 = torch.full_like(c0, stream & _MASK)
    c3 = torch.zeros_like(c0)
    r = _philox4x32(c0, c1, c2, c3, seed & _MASK, (seed >> 32) & _MASK)
    lane = e & 3
    x = torch.where(lane == 0, r[0], torch.where(lane == 1, r[1], torch.where(lane == 2, r[2], r[3])))
    return ((x >> 8).to(torch.float32)) * (1.0 / 16777216.0)


def adaptive_forge(mean, mn, mx, seed: int, stream: int, offset: int, b: float = 2.0):
    """Fang et al. attack vector (reference blades/adversaries/adaptive_adversary.py:32-65) from the benign column
    mean / min / max and one Philox uniform per (global) coordinate."""
    u = philox_uniform(mean.numel(), seed, stream, offset, device=mean.device)
    s = torch.sign(mean)
    out = torch.zeros_like(mean)
    out = torch.where((s == -1) & (mx > 0), mx * (1 + u * (b - 1)), out)
    out = torch.where((s == -1) & (mx < 0), mx * (1 + u * (1 / b - 1)), out)
    out = torch.where((s == 1) & (mn > 0), mn * (1 / b + u * (1 - 1 / b)), out)
    out = torch.where((s == 1) & (mn < 0), mn * (b + u * (1 - b)), out)
    return torch.where(s == 0, mean, out)


def perm_keys(n: int, seed: int, stream: int, offset: int, d_valid_end: int, device="cpu"):
    """Unique int64 sort keys of a random permutation of the coordinates: (31 Philox bits : 32-bit global index);
    padding coordinates (global index >= ``d_valid_end``) get the largest key."""
    e = torch.arange(offset, offset + n, dtype=torch.int64, device=device)
    blk = e >> 2
    c0, c1 = blk & _MASK, (blk >> 32) & _MASK
    r = _philox4x32(c0, c1, torch.full_like(c0, stream & _MASK), torch.zeros_like(c0), seed & _MASK,
                    (seed >> 32) & _MASK)
    lane = e & 3
    x = torch.where(lane == 0, r[0], torch.where(lane == 1, r[1], torch.where(lane == 2, r[2], r[3])))
    keys = ((x >> 1) << 32) | (e & _MASK)
    return torch.where(e < d_valid_end, keys, torch.full_like(keys, 0x7FFFFFFFFFFFFFFF))


def signguard_forge(keys, thresholds, seed: int, stream: int, offset: int):
    u = philox_uniform(keys.numel(), seed, stream, offset, device=keys.device)
    return torch.where(keys < thresholds[0], u, torch.where(keys < thresholds[1], -u, torch.zeros_like(u)))


def client_dropout_mult(uids, n: int, seed: int, tag, layer: int, p: float):
    """``[len(uids), n]`` dropout multipliers (0 or 1/(1-p)), keyed by client: element ``e`` of client ``uid``
    uses lane ``e % 4`` of Philox counter ``(e//4, uid, tag, 2 + 256*layer)``.  ``tag`` (int or 1-element int64
    tensor) identifies the round / local step.  ``uids`` may be a 0-dim tensor (one client, e.g. under vmap):
    the result is then ``[n]``."""
    single = uids.dim() == 0
    u2 = uids.reshape(-1, 1)
    e = torch.arange(n, dtype=torch.int64, device=uids.device).unsqueeze(0)
    c0 = ((e >> 2) & _MASK) + torch.zeros_like(u2)
    c1 = (u2 & _MASK) + torch.zeros_like(e)
    t = tag.to(uids.device).reshape(1, 1) if torch.is_tensor(tag) else torch.tensor([[int(tag)]], device=uids.device)
    c2 = (t & _MASK) + torch.zeros_like(c0)
    c3 = torch.full_like(c0, (2 + 256 * int(layer)) & _MASK)
    r = _philox4x32(c0, c1, c2, c3, seed & _MASK, (seed >> 32) & _MASK)
    lane = e & 3
    x = torch.where(lane == 0, r[0], torch.where(lane == 1, r[1], torch.where(lane == 2, r[2], r[3])))
    u = ((x >> 8).to(torch.float32)) * (1.0 / 16777216.0)
    m = (u >= p).to(torch.float32) * (1.0 / (1.0 - p))
    return m[0] if single else m


def philox_normal(n: int, seed: int, stream: int, offset: int = 0, mean=0.0, std=1.0, device="cpu"):
    """Box–Muller on Philox words: element ``e`` uses counter ``(e//2, stream, 1)``
    words (0,1) for even ``e`` (cos branch) and (2,3) for odd ``e`` (sin of the
    second pair) — every element is an independent draw."""
    e = torch.arange(offset, offset + n, dtype=torch.int64, device=device)
    blk = e >> 1
    c0, c1 = blk & _MASK, (blk >> 32) & _MASK
    c2 = torch.full_like(c0, stream & _MASK)
    c3 = torch.ones_like(c0)
    r = _philox4x32(c0, c1, c2, c3, seed & _MASK, (seed >> 32) & _MASK)
    odd = (e & 1).bool()
    a = torch.where(odd, r[2], r[0])
    b = torch.where(odd, r[3], r[1])
    u1 = ((a >> 8).to(torch.float32) + 1.0) * (1.0 / 16777216.0)  # (0,1]
    u2 = (b >> 8).to(torch.float32) * (1.0 / 16777216.0)
    rad = torch.sqrt(-2.0 * torch.log(u1))
    z = rad * torch.cos(6.283185307179586 * u2)
    return z * std + mean


def add_normal_rows_(U, rows, seed: int, stream: int, col_offset: int, d_total: int,
                     mean: float, std: float, overwrite: bool):
    """Rows ``rows[r]`` of ``U`` get (``overwrite``) or are incremented by
    N(mean,std) noise; element ``(global_row_id g, global column c)`` uses the
    Philox index ``g * d_total + c`` so the draw is shard-independent.
    ``rows`` is ``[R,2]`` int64: (local row, global row id)."""
    Dl = U.shape[1]
    for lr_, g in rows.tolist():
        z = philox_normal(Dl, seed, stream, offset=g * d_total + col_offset, mean=mean, std=std,
                          device=U.device)
        if overwrite:
            U[lr_] = z
        else:
            U[lr_] += z
    return U


def power_iteration_top(G: torch.Tensor, iters: int = 8) -> torch.Tensor:
    """Top eigenvector of a symmetric PSD ``[K,K]`` matrix.

    Repeated squaring (``A <- A A / ||A A||_F``, 6 times: A ∝ G^64) followed by
    ``iters`` plain power steps with ``G``; deterministic start vector.  K x K
    work only (K = number of clients), library GEMMs."""
    K = G.shape[0]
    v = torch.full((K,), 1.0 / K ** 0.5, dtype=G.dtype, device=G.device)
    v = v + torch.arange(K, device=G.device, dtype=G.dtype) * (1e-3 / K)
    nrm = torch.linalg.matrix_norm(G)
    A = G / nrm.clamp_min(1e-30)
    for _ in range(6):
        A = A @ A
        A = A / torch.linalg.matrix_norm(A).clamp_min(1e-30)
    v = A @ v
    v = v / v.norm().clamp_min(1e-30)
    for _ in range(iters):
        w = G @ v
        v = w / w.norm().clamp_min(1e-30)
    return v


def ce_topk(logits: torch.Tensor, labels: torch.Tensor, ks=(1,)) -> torch.Tensor:
    """float64 ``[1 + len(ks)]``: summed cross-entropy, then the number of samples whose target class is among
    the ``k`` best logits (ties go to the lower class index) for every ``k`` in ``ks``
    (reference metrics: ``fllib/tasks/task.py:104-121``)."""
    lg = logits.float().reshape(-1, logits.shape[-1])
    y = labels.reshape(-1).long()
    ce = torch.nn.functional.cross_entropy(lg, y, reduction="sum").double()
    ly = lg.gather(1, y[:, None])
    cls = torch.arange(lg.shape[1], device=lg.device)[None, :]
    rank = ((lg > ly) | ((lg == ly) & (cls < y[:, None]))).sum(1)
    hits = [(rank < int(k)).sum().double() for k in ks]
    return torch.stack([ce] + hits)


def mha(qkv, B: int, scale: float, uids=None, tag=0, seed: int = 0, layer: int = 0, p: float = 0.0):
    """Oracle of ops/csrc/mha.hip: ``qkv [R, N, 3, H, hd]`` (client-major samples, ``B`` per client) ->
    ``softmax(q k^T * scale)``, client-keyed dropout on the ``[B, H, N, N]`` probabilities of each client
    (``client_dropout_mult``), ``@ v`` -> ``[R, N, H * hd]``.  Differentiable (plain torch ops)."""
    R, N, _, H, hd = qkv.shape
    q, k, v = qkv.permute(2, 0, 3, 1, 4)  # [R, H, N, hd]
    attn = ((q @ k.transpose(-2, -1)) * scale).softmax(dim=-1)
    if uids is not None and p > 0.0:
        m = client_dropout_mult(uids, B * H * N * N, seed, tag, layer, p)  # [Kc, B*H*N*N]
        attn = attn * m.reshape(R, H, N, N).to(attn.dtype)
    return (attn @ v).transpose(1, 2).reshape(R, N, H * hd)


def shuffle_keys(uids, epochs, lens, nmax: int, seed: int):
    """``[rows, nmax]`` float64 sort keys of the device batch sampler: position ``pos`` of client ``uid`` in epoch
    ``ep`` -> the word pair of Philox counter ``(pos, uid, ep, 7)`` as a signed 64-bit integer / 2^64, in [-0.5, 0.5); positions past the
    client's shard length get 2.0 (sort last)."""
    rows = uids.numel()
    pos = torch.arange(nmax, dtype=torch.int64, device=uids.device).unsqueeze(0).expand(rows, -1)
    uid = uids.reshape(-1, 1).expand_as(pos)
    ep = epochs.reshape(-1, 1).expand_as(pos)
    w = _philox4x32(pos, uid & _MASK, ep & _MASK, torch.full_like(pos, 7), seed & _MASK, (seed >> 32) & _MASK)
    keys = (w[0] * 4294967296 + w[1]).double() / float(2 ** 64)
    return keys.masked_fill(pos >= lens.reshape(-1, 1), 2.0)


def group_norm(x, groups: int, weight=None, bias=None, eps: float = 1e-5, act: str = "none", residual=None):
    """Oracle of ops/csrc/groupnorm_fwd.hip: ``act(group_norm(x) * weight + bias + residual)`` for ``x [N, C, *]``;
    ``weight`` / ``bias`` ``[C]``, or ``[K, C]`` for K clients of N / K consecutive samples each.  32-bit arithmetic
    (64 for 64-bit inputs), rounded once.  Differentiable (plain torch ops)."""
    acc = torch.float64 if x.dtype == torch.float64 else torch.float32
    N, C = x.shape[0], x.shape[1]
    tail = [1] * (x.dim() - 2)
    xf = x.to(acc).reshape(N, groups, (C // groups) * math.prod(x.shape[2:]))
    d = xf - xf.mean(dim=2, keepdim=True)
    z = (d * torch.rsqrt(d.square().mean(dim=2, keepdim=True) + eps)).reshape(x.shape)

    def per_sample(t):
        t = t.to(acc)
        return t.reshape(1, C, *tail) if t.dim() == 1 else t.repeat_interleave(int(N // t.shape[0]), dim=0).reshape(N, C, *tail)

    if weight is not None:
        z = z * per_sample(weight)
    if bias is not None:
        z = z + per_sample(bias)
    if residual is not None:
        z = z + residual.to(acc)
    F = torch.nn.functional
    y = {"none": lambda t: t, "relu": F.relu, "gelu": F.gelu, "silu": F.silu}[act](z)
    return y.to(x.dtype)


def client_dropout(x, uids, seed: int, tag, layer: int, p: float, kind: str = "elem", layout: str = "major", scale=None):
    """Oracle of ops/csrc/dropout.hip: ``x`` times the multipliers of ``client_dropout_mult``, laid over the elements,
    channels or samples of every client's share of the batch.  Differentiable."""
    uids = uids.reshape(-1)
    Kc = uids.numel()
    keep = 1 if kind == "sample" else (2 if kind == "channel" and x.dim() > 2 else x.dim())
    if layout == "major":
        B, C = int(x.shape[0] // Kc), int(x.shape[1]) if x.dim() > 1 else 1
        lead = [Kc, B]
    else:
        B, C = int(x.shape[0]), int(x.shape[1] // Kc)
        lead = [B, Kc]
    value = [1 if i >= keep else (C if i == 1 else int(d)) for i, d in enumerate(x.shape)][1:]  # draws of one sample
    n = B
    for d in value:
        n *= d
    m = client_dropout_mult(uids, n, seed, tag, layer, p)
    if scale is not None:
        m = (m != 0).to(m.dtype) * scale
    m = m.reshape([Kc, B] + value)
    m = (m if layout == "major" else m.transpose(0, 1))
    acc = torch.float64 if x.dtype == torch.float64 else torch.float32
    xs = x.to(acc).reshape(lead + [C] * (x.dim() > 1) + list(x.shape[2:]))
    return (xs * m.to(acc)).reshape(x.shape).to(x.dtype)


def rope_axes(x, pos, axes, base: float = 10000.0, slots=None, inverse: bool = False):
    """Oracle of ops/csrc/rope.hip: rotary positions with one section of the head dimension per axis.
    ``x [R, N, H, D]``, or ``[R, N, S, H, D]`` whose first ``slots`` slots are turned; ``pos [N, A]`` or ``[R, N, A]``.
    Angles in 64 bits, products in 32.  Differentiable."""
    acc = torch.float64 if x.dtype == torch.float64 else torch.float32
    dev = x.device
    freq = torch.cat([float(base) ** (torch.arange(a // 2, dtype=torch.float64, device=dev) * (-2.0 / a)) for a in axes])
    axis = torch.cat([torch.full((a // 2,), i, dtype=torch.int64, device=dev) for i, a in enumerate(axes)])
    angle = pos.to(dev).double()[..., axis] * freq
    cos, sin = angle.cos().to(acc).unsqueeze(-2), angle.sin().to(acc).unsqueeze(-2)
    sin = -sin if inverse else sin
    part, rest = x, None
    if x.dim() == 5:
        cos, sin = cos.unsqueeze(-3), sin.unsqueeze(-3)
        if slots is not None and slots < x.shape[2]:
            part, rest = x[:, :, :slots], x[:, :, slots:]
    rot = 2 * freq.numel()
    pf = part.to(acc)
    a, b = pf[..., 0:rot:2], pf[..., 1:rot:2]
    y = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2).to(x.dtype)
    y = torch.cat((y, part[..., rot:]), dim=-1)
    return y if rest is None else torch.cat((y, rest), dim=2)
