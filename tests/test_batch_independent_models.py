"""Group norm, client-keyed dropout and rotary positions inside the models and the engine: the execution paths agree on the
update matrix, on the CPU and on the GPU, eager and replayed."""
import copy

import pytest
import torch
from torch import nn

from blades_amd.models.catalog import ModelCatalog
from tests.test_engine_paths import build, one_round_updates


class NormNet(nn.Module):
    """Smooth everywhere (no gate can tip between two roundings): group norms with folded and separate activations, with
    and without an affine pair, channel and element dropout."""

    def __init__(self):
        super().__init__()
        act = nn.SiLU()
        self.body = nn.Sequential(
            nn.Conv2d(3, 32, 3, padding=1), nn.GroupNorm(8, 32), act,
            nn.Conv2d(32, 64, 3, stride=2, padding=1), nn.GroupNorm(16, 64), nn.GELU(), nn.Dropout2d(0.1),
            nn.Conv2d(64, 64, 3, stride=2, padding=1), nn.GroupNorm(1, 64, affine=False), act)
        self.last = nn.GroupNorm(4, 64)
        self.drop = nn.Dropout(0.2)
        self.fc = nn.Linear(64, 10)

    def forward(self, x):
        x = self.last(self.body(x).mean(dim=(2, 3)))
        return self.fc(self.drop(x))


ROTARY = {"type": "cvt_2_4_32", "positional_embedding": "rotary"}
GROUPED = {"type": "resnet10", "norm": "group"}


def rel_rows(U, V):
    return (U.cpu() - V.cpu()).norm(dim=1) / V.cpu().norm(dim=1)


# Relative error of a client's update between two correct fp32 paths: fewer than 100 operations in a chain, each off by
# under 16 half steps (2^-24) of its scale: 1e-4.
SMOOTH = 1e-4


@pytest.mark.parametrize("model", [NormNet, ROTARY])
def test_fused_equals_vectorised_cpu(data_root, model):
    a, b = build(data_root, model, "fused"), build(data_root, model, "vmap")
    assert a.engine.fused is not None and b.engine.fused is None
    Ua, ta = one_round_updates(a)
    Ub, tb = one_round_updates(b)
    assert float(rel_rows(Ua, Ub).max()) < SMOOTH
    assert float((ta - tb).norm() / tb.norm()) < SMOOTH


def test_fused_equals_vectorised_group_norm_resnet_cpu(data_root):
    a, b = build(data_root, GROUPED, "fused"), build(data_root, GROUPED, "vmap")
    Ua, _ = one_round_updates(a)
    Ub, _ = one_round_updates(b)
    rel = rel_rows(Ua, Ub)
    # rows without a ReLU gate within rounding of its border agree to rounding, the others to the weight of the gate's pixel
    assert int((rel < SMOOTH).sum()) * 2 >= rel.numel() and float(rel.max()) < 2e-2, rel


def test_folding_follows_the_positions_not_the_instances():
    """One activation module in several places: each group norm takes only the activation directly behind it."""
    from blades_amd.engine.fused import GradSink, PCGroupNorm, build_template, supports

    relu, silu = nn.ReLU(), nn.SiLU()
    net = nn.Sequential(relu, nn.Conv2d(3, 8, 1), nn.GroupNorm(2, 8), relu, silu, nn.GroupNorm(4, 8), silu)
    assert supports(net)
    sink = GradSink()
    tmpl = build_template(net, sink)
    assert [m.act for m in tmpl.modules() if isinstance(m, PCGroupNorm)] == ["relu", "silu"]
    sink.Kc = 2
    x = torch.randn(4, 3, 5, 5)
    with torch.no_grad():
        torch.testing.assert_close(tmpl(x), net(x), rtol=1e-5, atol=1e-5)


def test_catalog_options():
    net = ModelCatalog.get_model(GROUPED)
    assert not any(isinstance(m, nn.BatchNorm2d) for m in net.modules())
    plain = ModelCatalog.get_model("resnet10")
    assert [(n, p.shape) for n, p in net.named_parameters()] == [(n, p.shape) for n, p in plain.named_parameters()]
    x = torch.randn(4, 3, 32, 32)
    with torch.no_grad():  # a sample's output does not depend on its batch (up to the convolutions' summation order)
        torch.testing.assert_close(net(x)[:1], net(x[:1]), rtol=1e-4, atol=1e-5)
    assert ModelCatalog.get_model({"type": "resnet18", "norm": "group", "norm_groups": 16}).bn1.num_groups == 16
    for bad in ({"type": "resnet10", "norm": "layer"},):
        with pytest.raises(ValueError):
            ModelCatalog.get_model(bad)
    for bad in ({"type": "resnet", "norm": "group"}, {"type": "nothing"}, {}):
        with pytest.raises(NotImplementedError):
            ModelCatalog.get_model(bad)


def test_rotary_transformer():
    from blades_amd.models.cctnets.layers import RotaryGrid, TransformerClassifier

    torch.manual_seed(0)
    net = ModelCatalog.get_model(ROTARY).eval()
    assert not any("positional" in n for n, _ in net.named_parameters()) and not list(net.state_dict().keys() & {"pos"})
    blocks = net.classifier.blocks
    assert blocks[0].self_attn.rope is blocks[1].self_attn.rope and blocks[0].self_attn.rope.pos.shape == (64, 2)
    assert blocks[0].self_attn.rope.pos[9].tolist() == [1, 1]
    # positions matter: patch embeddings in another order give the same logits without them (64 bits: up to 1e-12), and
    # others with them (small weights at the start: by 1e-5 or so)
    cls = net.classifier.double()
    tok = torch.randn(2, 64, 128, dtype=torch.float64)
    perm = torch.randperm(64)
    with torch.no_grad():
        assert float((cls(tok) - cls(tok[:, perm])).abs().max()) > 1e-8
        for b in blocks:
            b.self_attn.rope = None
        assert float((cls(tok) - cls(tok[:, perm])).abs().max()) < 1e-12
    # models of other image sizes share every parameter
    small, large = (ModelCatalog.get_model({**ROTARY, "img_size": s}) for s in (32, 64))
    assert [(n, p.shape) for n, p in small.named_parameters()] == [(n, p.shape) for n, p in large.named_parameters()]
    cls = TransformerClassifier(seq_pool=False, embedding_dim=32, num_layers=1, num_heads=2, positional_embedding="rotary",
                                sequence_length=6, token_grid=(2, 3), num_classes=4)
    assert cls.blocks[0].self_attn.rope.pos.tolist() == [[0, 0], [1, 1], [1, 2], [1, 3], [2, 1], [2, 2], [2, 3]]
    assert cls(torch.randn(3, 6, 32)).shape == (3, 4)
    with pytest.raises(ValueError):
        TransformerClassifier(embedding_dim=32, num_layers=1, num_heads=2, positional_embedding="rotary", sequence_length=6)
    with pytest.raises(ValueError):
        RotaryGrid((2, 2), 2)


# ---------------------------------------------------------------------------------------------------------------
def gpu_copy(algo, mode="fused", amp="fp32"):
    cfg = copy.deepcopy(algo.config)
    cfg._is_frozen = False
    cfg.device, cfg.amp_dtype, cfg.execution_mode = "cuda", amp, mode
    g = cfg.build()
    g.server.theta.copy_(algo.server.theta.cuda())
    return g


@pytest.mark.gpu
@pytest.mark.parametrize("model", [NormNet, ROTARY])
def test_fused_gpu_matches_vectorised_cpu(data_root, model):
    a = build(data_root, model, "vmap")
    g = gpu_copy(a)
    assert g.engine.fused is not None
    Ug, _ = one_round_updates(g)
    Ua, _ = one_round_updates(a)
    rel = rel_rows(Ug, Ua)
    assert float(rel.max()) < SMOOTH, rel


@pytest.mark.gpu
@pytest.mark.parametrize("model", [NormNet, ROTARY])
def test_local_steps_gpu_match_vectorised_cpu(data_root, model):
    """Two local steps: each client's own affine pair, read in place from its weight row."""
    a = build(data_root, model, "vmap", nb=2, lr=0.05)
    g = gpu_copy(a, "auto")
    Ug, _ = one_round_updates(g)
    assert g.engine.fused_pc, g.engine.fused_pc_error
    Ua, _ = one_round_updates(a)
    rel = rel_rows(Ug, Ua)
    assert float(rel.max()) < 4 * SMOOTH, rel  # the second step starts from weights that differ by the first one's error


@pytest.mark.gpu
def test_group_norm_resnet_gpu_matches_cpu(data_root):
    a = build(data_root, GROUPED, "fused")
    g = gpu_copy(a)
    Ug, _ = one_round_updates(g)
    Ua, _ = one_round_updates(a)
    rel = rel_rows(Ug, Ua)
    assert int((rel < SMOOTH).sum()) * 2 >= rel.numel() and float(rel.max()) < 2e-2, rel
    acc = g.evaluate() if hasattr(g, "evaluate") else None
    assert acc is None or all(v == v for v in acc.values() if isinstance(v, float))


@pytest.mark.gpu
@pytest.mark.parametrize("model", [NormNet, ROTARY])
def test_bf16_mode(data_root, model):
    a = build(data_root, model, "vmap")
    g = gpu_copy(a, amp="bf16")
    Ug, _ = one_round_updates(g)
    Ua, _ = one_round_updates(a)
    cos = torch.nn.functional.cosine_similarity(Ug.cpu().double(), Ua.double(), dim=1)
    # activations and gradients are rounded to 2^-9 of themselves at about 30 places in a row, independently: 30^0.5 2^-8
    # = 2 % of a row, cosine 1 - 0.02^2 / 2; with a margin of ten for rows whose gradient is small against its terms
    assert float(cos.min()) > 0.98, cos


@pytest.mark.gpu
@pytest.mark.parametrize("nb", [1, 3])
@pytest.mark.parametrize("model", [NormNet, ROTARY, GROUPED])
def test_graph_replay_matches_eager(tmp_path, model, nb):
    from tests.test_engine_gpu import _run

    kw = dict(rounds=6, nb=nb, lr=0.05)
    th_e, loss_e, eng_e = _run(tmp_path, "0", "cifar10", model, "ALIEAdversary", **kw)
    th_g, loss_g, eng_g = _run(tmp_path, "1", "cifar10", model, "ALIEAdversary", **kw)
    assert eng_e.graph_replays == 0 and eng_g.graph_replays >= 3, getattr(eng_g, "_graph_error", None)
    assert loss_g == loss_e and torch.equal(th_g, th_e)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,shape", [("elem", (12, 40)), ("channel", (12, 8, 6, 6)), ("sample", (12, 10, 16)),
                                        ("channel", (12, 9))])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["major", "inner"])
def test_engine_dropout_equals_its_stored_multipliers(kind, shape, dt, layout):
    """The engine's dropout layer gives, bit for bit, the product with client_dropout_mult's multipliers of the
    activations' type."""
    from blades_amd import ops
    from blades_amd.engine.layers import ClientDropout, DropContext

    dev = torch.device("cuda")
    ctx = DropContext(3, dev)
    ctx.set(torch.tensor([7, 1, 30], device=dev), layout)
    ctx.set_tag(19)
    m = ClientDropout(0.3, kind, 2, ctx).train()
    full = shape if layout == "major" else (4, 3 * shape[1]) + shape[2:]
    g = torch.Generator().manual_seed(0)
    x = torch.randn(full, generator=g).to(dt).to(dev)
    B, C = 4, shape[1]
    keep = [1] * (len(shape) - 1) if kind == "sample" else [C] + [1] * (len(shape) - 2) if kind == "channel" and len(
        shape) > 2 else list(shape[1:])
    n = B
    for d in keep:
        n *= d
    mult = ops.client_dropout_mult(ctx.uids, n, ctx.seed, ctx.tag, 2, 0.3).reshape([3, B] + keep).expand(3, B, *shape[1:])
    mult = mult if layout == "major" else mult.transpose(0, 1)
    assert torch.equal(m(x), x * mult.reshape(full).to(dt))
